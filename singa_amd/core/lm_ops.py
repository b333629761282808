"""Operators of language models over core tensors: rotary positions with the
norm of every head, losses over the log-probabilities of given tokens, and the
AdamW step.

The functions check their arguments on the host (the kernels trust them), and
submit one named operation each, so that they run eagerly or become a node of
the recorded step.  The reference has none of them.
"""
import math

import numpy as np

from . import dtypes
from .tensor_core import Contiguous, Tensor, _one_device, _submit

_FLOATS = (dtypes.kFloat32, dtypes.kFloat16, dtypes.kBFloat16)


def _refuse(condition, message, *args):
    if condition:
        raise ValueError(message % args if args else message)


def _float_operand(what, t):
    if t._dtype not in _FLOATS:
        raise TypeError("%s is float32, float16 or bfloat16, got %s" %
                        (what, dtypes.name(t._dtype)))


def _int_operand(what, t):
    if t._dtype != dtypes.kInt:
        raise TypeError("%s is int32, got %s" % (what, dtypes.name(t._dtype)))


def _rows_contiguous(t):
    """A strided view whose last dimension is contiguous passes as it is."""
    return t if t._stride and (t._stride[-1] == 1 or t._shape[-1] == 1) \
        else Contiguous(t)


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------
class RotaryHandle(object):
    """What a rotary embedding is made of, apart from its inputs.

    head_dim:    channels of a head (even, at most 1024)
    rotary_dim:  the first so many of them turn (even, at most 512; all of
                 them by default), the others pass through
    base:        pair i turns by base^(-2 i / rotary_dim) for each position
    layout:      "half" pairs channel i with i + rotary_dim / 2,
                 "interleaved" pairs 2 i with 2 i + 1
    scaling:     for contexts longer than the trained one; None or
                 ("linear", factor): every frequency is divided by the factor;
                 ("base", factor): the base grows so that the slowest pair
                     turns factor times slower and the fastest as before,
                     base * factor^(R / (R - 2));
                 ("ramp", factor, length[, low, high]): a pair that makes n
                     turns over the trained length keeps its frequency for
                     n >= high (32), is divided by the factor for n <= low (1)
                     and goes from one to the other linearly in n between;
                     its amplitude is 1 + 0.1 log(factor)
    amplitude:   the rotated channels are multiplied by it (default 1, or the
                 scaling's own)

    ``frequencies`` (float64, radians for each position) and ``amplitude`` are
    what came of it."""

    def __init__(self, head_dim, rotary_dim=None, base=10000.0, layout="half",
                 scaling=None, amplitude=None):
        self.head_dim = int(head_dim)
        self.rotary_dim = self.head_dim if rotary_dim is None \
            else int(rotary_dim)
        D, R = self.head_dim, self.rotary_dim
        _refuse(D < 2 or D > 1024 or D % 2,
                "head_dim is even, from 2 to 1024, got %d", D)
        _refuse(R < 2 or R > min(D, 512) or R % 2,
                "rotary_dim is even, from 2 to min(head_dim, 512), got %d", R)
        _refuse(layout not in ("half", "interleaved"),
                "layout is 'half' or 'interleaved', got %r", layout)
        base = float(base)
        _refuse(not (math.isfinite(base) and base >= 1.0),
                "base is a finite number from 1, got %r", base)
        self.layout = layout
        own_amplitude = 1.0
        kind, values = None, ()
        if scaling is not None:
            kind, values = scaling[0], [float(v) for v in scaling[1:]]
            counts = {"linear": (1,), "base": (1,), "ramp": (2, 4)}.get(kind)
            _refuse(counts is None or len(values) not in counts,
                    "scaling is ('linear', factor), ('base', factor) or "
                    "('ramp', factor, length[, low, high]), got %r",
                    (scaling,))
            _refuse(not all(math.isfinite(v) for v in values) or
                    values[0] < 1.0,
                    "a scaling factor is a finite number from 1, got %r",
                    (scaling,))
        if kind == "base":
            _refuse(R == 2, "one pair has no base to scale")
            base *= values[0] ** (R / (R - 2.0))
        f = base ** (-np.arange(0, R, 2, dtype=np.float64) / R)
        if kind == "linear":
            f = f / values[0]
        elif kind == "ramp":
            factor, length = values[:2]
            low, high = values[2:] or (1.0, 32.0)
            _refuse(length <= 0 or not high > low,
                    "a ramp has a positive length and high > low, got %r",
                    (scaling,))
            turns = length * f / (2 * math.pi)
            keep = np.clip((turns - low) / (high - low), 0.0, 1.0)
            f = f * (keep + (1.0 - keep) / factor)
            own_amplitude = 1.0 + 0.1 * math.log(factor)
        self.frequencies = f
        self.amplitude = own_amplitude if amplitude is None \
            else float(amplitude)
        _refuse(not math.isfinite(self.amplitude),
                "amplitude is a finite number, got %r", amplitude)
        # turns for each position as fractions of 2^64 (base >= 1: below 2^62)
        self._turns = np.array(
            [round(math.ldexp(v / (2 * math.pi), 64)) for v in f], np.uint64)


def _check_rotary(handle, xs, scales, positions):
    _refuse(not 1 <= len(xs) <= 2, "rotary takes one or two tensors")
    lead = xs[0]
    for x in xs:
        _float_operand("a rotary operand", x)
        _refuse(x.nDim() != 4 or x._shape[-1] != handle.head_dim,
                "a rotary operand is (batch, sequence, heads, %d), got %s",
                handle.head_dim, tuple(x._shape))
        _refuse(x._shape[:2] != lead._shape[:2] or x._dtype != lead._dtype,
                "queries and keys share batch, sequence and type: %s %s, "
                "%s %s", tuple(lead._shape), dtypes.name(lead._dtype),
                tuple(x._shape), dtypes.name(x._dtype))
    B, S = lead._shape[:2]
    _refuse(B * S > 0x7fffffff, "more than 2^31 - 1 tokens in one call")
    _refuse(any(x._shape[2] > 65536 for x in xs), "more than 65536 heads")
    if scales:
        _refuse(len(scales) != len(xs), "one scale for each tensor")
        for w in scales:
            _refuse(w._shape != [handle.head_dim] or w._dtype != lead._dtype,
                    "a scale is (%d,) of the operands' type, got %s %s",
                    handle.head_dim, tuple(w._shape), dtypes.name(w._dtype))
    if positions is not None:
        _int_operand("positions", positions)
        _refuse(positions._shape not in ([S], [B, S]),
                "positions are (%d,) or (%d, %d), got %s", S, B, S,
                tuple(positions._shape))


def _rotary(name, handle, xs, scales, positions, eps, dys):
    """Shared body: forward without ``dys``, else backward.  Returns
    (outputs, scale gradients)."""
    _check_rotary(handle, xs, scales, positions)
    eps = float(eps)
    _refuse(not eps >= 0.0, "eps is a number from 0, got %r", eps)
    dev, n = xs[0]._dev, len(xs)
    back = dys is not None
    if back:
        for x, g in zip(xs, dys):
            _refuse(g._shape != x._shape or g._dtype != x._dtype,
                    "a gradient of %s %s for an output of %s %s",
                    tuple(g._shape), dtypes.name(g._dtype), tuple(x._shape),
                    dtypes.name(x._dtype))
        dys = [_rows_contiguous(g) for g in dys]
    # the backward pass of a rotation alone does not need its input
    inputs = [] if back and not scales else [_rows_contiguous(x) for x in xs]
    grads = dys if back else []
    scales = [Contiguous(w) for w in scales]
    ys = [Tensor(x._shape, dev, x._dtype) for x in xs]
    dws = [Tensor([handle.head_dim], dev, w._dtype) for w in scales] \
        if back else []
    at = [positions] if positions is not None else []
    reads = inputs + grads + scales + at
    counts = (len(inputs), len(grads), len(scales), len(at), len(ys),
              len(dws))

    def body(*ts):
        parts, k = [], 0
        for c in counts:
            parts.append([t.view() for t in ts[k:k + c]])
            k += c
        x, g, w, p, y, dw = parts
        ts[0]._dev.math.rotary(handle, x, g, w, p[0] if p else None, y, dw,
                               eps)

    _one_device(name, dev, reads)
    _submit(dev, name, body, reads, ys + dws)
    return ys, dws


def RotaryForward(handle, xs, scales=(), positions=None, eps=1e-6):
    """Turn the heads of one or two (B, S, H, D) tensors by their positions,
    after the root-mean-square norm of each head when ``scales`` (one (D,)
    tensor for each) are given.  positions: int32 (S,) or (B, S), any value;
    0 .. S - 1 without.  Returns the list of turned tensors."""
    return _rotary("RotaryForward", handle, list(xs), list(scales), positions,
                   eps, None)[0]


def RotaryBackward(handle, dys, xs, scales=(), positions=None, eps=1e-6):
    """-> (gradients of xs, gradients of scales)."""
    return _rotary("RotaryBackward", handle, list(xs), list(scales), positions,
                   eps, list(dys))


# ---------------------------------------------------------------------------
# losses over the log-probabilities of given tokens
# ---------------------------------------------------------------------------
LOSS_LOG_PROB, LOSS_PREFERENCE, LOSS_POLICY = 0, 1, 2


class TokenLoss(object):
    """One loss over the labels' log-probabilities: its constants, and what its
    forward pass keeps for the backward pass."""

    def __init__(self, mode, x, label, ref=None, old=None, adv=None,
                 weight=None, beta=0.0, smoothing=0.0, clip=(0.0, 0.0),
                 kl=0.0):
        _float_operand("logits", x)
        _int_operand("a label", label)
        _refuse(x.nDim() < 1 or x._shape[:-1] != label._shape,
                "logits %s need labels %s, got %s", tuple(x._shape),
                tuple(x._shape[:-1]), tuple(label._shape))
        _refuse(x._shape[-1] < 1, "an empty vocabulary")
        self.mode = mode
        self.pairs = self.seq = 0
        if mode == LOSS_PREFERENCE:
            _refuse(x.nDim() != 3 or x._shape[0] % 2 or x.Size() == 0,
                    "preference logits are (2 pairs, sequence, vocabulary), "
                    "the chosen ones first, got %s", tuple(x._shape))
            self.pairs, self.seq = x._shape[0] // 2, x._shape[1]
        for what, t in (("reference", ref), ("old", old), ("advantages", adv),
                        ("weights", weight)):
            if t is not None:
                _float_operand(what, t)
                _refuse(t._shape != label._shape,
                        "%s have the labels' shape %s, got %s", what,
                        tuple(label._shape), tuple(t._shape))
        _one_device("a token loss", x._dev,
                    [t for t in (label, ref, old, adv, weight)
                     if t is not None])
        self.x, self.label = Contiguous(x), Contiguous(label)
        self.extra = [t if t is None else
                      Contiguous(t.AsType(dtypes.kFloat32))
                      for t in (ref, old, adv, weight)]
        self.consts = (float(beta), float(smoothing), 1.0 - float(clip[0]),
                       1.0 + float(clip[1]), float(kl))
        self.V = x._shape[-1]
        self.rows = x.Size() // self.V

    def forward(self):
        """-> the loss (1,) or, for the log-probabilities, (labels' shape);
        float32."""
        dev, rows, f32 = self.x._dev, self.rows, dtypes.kFloat32
        logp = self.mode == LOSS_LOG_PROB
        value = Tensor(self.label._shape, dev, f32)
        # of each row the largest logit and the log of the sum relative to it,
        # then the derivative (policy), then what rows' derivatives are
        # multiplied by (policy: one number, preference: one for each pair)
        n = {LOSS_LOG_PROB: 2 * rows, LOSS_PREFERENCE: 2 * rows + self.pairs,
             LOSS_POLICY: 3 * rows + 1}[self.mode]
        self.saved = Tensor([n], dev, f32)
        loss = value if logp else Tensor([1], dev, f32)
        given = [t for t in self.extra if t is not None]
        here = [t is not None for t in self.extra]
        ins = [self.x, self.label] + given
        spec = (self.mode, rows, self.V, self.pairs, self.seq, self.consts)

        def body(*ts):
            rest = iter(t.flat() for t in ts[2:2 + len(given)])
            extra = [next(rest) if h else None for h in here]
            val, saved = ts[2 + len(given)], ts[3 + len(given)]
            ts[0]._dev.math.token_loss_fwd(
                spec, ts[0].flat(), ts[1].flat(), extra, val.flat(),
                saved.flat(), None if logp else ts[-1].flat())

        outs = [value, self.saved] + ([] if logp else [loss])
        _submit(dev, "TokenLossForward", body, ins, outs)
        return loss

    def backward(self, dy):
        """dy: a float or a one-element tensor; for the log-probabilities a
        tensor of the labels' shape.  -> the gradient of the logits."""
        dev, logp = self.x._dev, self.mode == LOSS_LOG_PROB
        scale, dys = 1.0, []
        if isinstance(dy, Tensor):
            _refuse(dy.Size() != (self.rows if logp else 1),
                    "a gradient of %s for a loss of %s", tuple(dy._shape),
                    tuple(self.label._shape) if logp else (1,))
            dys = [Contiguous(dy.AsType(dtypes.kFloat32))]
        else:
            _refuse(logp, "log-probabilities need a gradient tensor")
            scale = float(dy)
        dx = Tensor(self.x._shape, dev, self.x._dtype)
        weight = [self.extra[3]] if self.extra[3] is not None else []
        spec = (self.mode, self.rows, self.V, self.pairs, self.seq)

        def body(*ts):
            w = ts[3].flat() if weight else None
            g = ts[3 + len(weight)].flat() if dys else None
            ts[0]._dev.math.token_loss_bwd(spec, ts[0].flat(), ts[1].flat(),
                                           ts[2].flat(), w, g, scale,
                                           ts[-1].flat())

        reads = [self.x, self.label, self.saved] + weight + dys
        _one_device("TokenLossBackward", dev, reads)
        _submit(dev, "TokenLossBackward", body, reads, [dx])
        return dx


# ---------------------------------------------------------------------------
# AdamW
# ---------------------------------------------------------------------------
ADAMW_BLOCK = 256       # values that share the scale of an 8-bit state


def AdamWUpdateMulti(params, grads, masters, state1, state2, scales1, scales2,
                     hypers, state_bits=32, scale=1.0, seed=0):
    """One AdamW step for a list of parameters of one type (one graph node,
    one launch for every 48 tensors).  masters: float32 copies of 16-bit
    parameters, or None.  state_bits 32: state1 / state2 are the float32
    moments; 8: int32 words of four e4m3 codes of the first moment and of the
    root of the second, in whole blocks of 256 values, with float32 scales1 /
    scales2 for each block.  hypers = (lr, weight_decay, epsilon, beta_1,
    beta_2, step): one-element float32 tensors."""
    n, dev = len(params), params[0]._dev
    grads = [g if g._dtype == p._dtype else g.AsType(p._dtype)
             for p, g in zip(params, grads)]
    lists = [list(params), [Contiguous(g) for g in grads],
             list(masters or ()), list(state1), list(state2),
             list(scales1 or ()), list(scales2 or ())]
    for p in params:
        _refuse(not p.is_contiguous(), "AdamW steps contiguous parameters")
    scale, seed, state_bits = float(scale), int(seed), int(state_bits)
    written = [i for i in (0, 2, 3, 4, 5, 6) if lists[i]]
    reads = [t for ts in lists for t in ts] + list(hypers)
    sizes = [len(ts) for ts in lists]

    def body(*ts):
        # the outputs stand behind the inputs: for a recorded step they are
        # the same blocks
        parts, k = [], 0
        for c in sizes:
            parts.append([t.flat() for t in ts[k:k + c]])
            k += c
        hyp = [t.flat() for t in ts[k:k + len(hypers)]]
        ts[0]._dev.math.adamw_update_multi(
            [t.Size() for t in ts[:n]], *parts, *hyp, state_bits, scale, seed)

    _one_device("AdamWUpdateMulti", dev, reads)
    _submit(dev, "AdamWUpdateMulti", body, reads,
            [t for i in written for t in lists[i]])
    return params
