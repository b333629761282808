"""Operators of language models over core tensors: rotary positions with the
norm of every head, losses over the log-probabilities of given tokens, and the
AdamW step.

The functions check their arguments on the host (the kernels trust them), and
submit one named operation each, so that they run eagerly or become a node of
the recorded step.  The reference has none of them.
"""
import itertools
import math
import operator

import numpy as np

from . import dtypes
from .. import _rt
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
        self.turns_address = self._turns.ctypes.data
        self.half = layout == "half"

    def __setstate__(self, state):
        # a copy has a table of its own: the original's may be gone
        self.__dict__.update(state)
        self._turns = self._turns.copy()
        self.turns_address = self._turns.ctypes.data


def _described(t):
    return "%s %s" % (tuple(t._shape), dtypes.name(t._dtype))


def _check_rotary(handle, xs, scales, positions):
    _refuse(not 1 <= len(xs) <= 2, "rotary takes one or two tensors")
    lead, D = xs[0], handle.head_dim
    B, S = lead._shape[:2] if lead.nDim() == 4 else (0, 0)
    for x in xs:
        _float_operand("a rotary operand", x)
        shape = x._shape
        if len(shape) != 4 or shape[3] != D:
            raise ValueError("a rotary operand is (batch, sequence, heads, "
                             "%d), got %s" % (D, tuple(shape)))
        if shape[0] != B or shape[1] != S or x._dtype != lead._dtype:
            raise ValueError("queries and keys share batch, sequence and "
                             "type: %s, %s" % (_described(lead),
                                               _described(x)))
        _refuse(not 1 <= shape[2] <= 65536, "1 to 65536 heads, got %d",
                shape[2])
    _refuse(B * S > 1 << 30, "more than 2^30 tokens in one call")
    if scales:
        _refuse(len(scales) != len(xs), "one scale for each tensor")
        for w in scales:
            if w._shape != [D] or w._dtype != lead._dtype:
                raise ValueError("a scale is (%d,) of the operands' type, got "
                                 "%s" % (D, _described(w)))
    if positions is not None:
        _int_operand("positions", positions)
        if positions._shape != [S] and positions._shape != [B, S]:
            raise ValueError("positions are (%d,) or (%d, %d), got %s" %
                             (S, B, S, tuple(positions._shape)))


def _rotary(name, handle, xs, scales, positions, eps, dys):
    """Shared body: forward without ``dys``, else backward.  Returns
    (outputs, scale gradients)."""
    _check_rotary(handle, xs, scales, positions)
    eps = float(eps)
    _refuse(not eps >= 0.0, "eps is a number from 0, got %r", eps)
    dev, back = xs[0]._dev, dys is not None
    if back:
        for x, g in zip(xs, dys):
            if g._shape != x._shape or g._dtype != x._dtype:
                raise ValueError("a gradient of %s for an output of %s" %
                                 (_described(g), _described(x)))
        dys = [_rows_contiguous(g) for g in dys]
    # the backward pass of a rotation alone does not need its input
    inputs = [] if back and not scales else [_rows_contiguous(x) for x in xs]
    grads = dys if back else []
    scales = [Contiguous(w) for w in scales]
    ys = [Tensor(x._shape, dev, x._dtype) for x in xs]
    dws = [Tensor(w._shape, dev, w._dtype) for w in scales] if back else []
    at = [positions] if positions is not None else []
    reads = inputs + grads + scales + at
    _one_device(name, dev, reads)
    if xs[0].Size() == 0:
        for w in dws:      # sums over nothing
            w.SetFloatValue(0.0)
    elif not dev.graph_enabled():
        dev.math.rotary(handle, inputs, grads, scales, positions, ys, dws, eps)
    else:
        ends = []
        for group in (inputs, grads, scales, at, ys):
            ends.append((ends[-1] if ends else 0) + len(group))

        def body(*ts):
            i, g, w, p, y = ends
            dev.math.rotary(handle, ts[:i], ts[i:g], ts[g:w],
                            ts[w] if p > w else None, ts[p:y], ts[y:], eps)

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
        shape = label._shape
        if len(x._shape) < 2 or x._shape[:-1] != shape:
            raise ValueError("logits %s need labels %s, got %s" % (
                tuple(x._shape), tuple(x._shape[:-1]), tuple(shape)))
        self.V = x._shape[-1]
        _refuse(self.V < 1, "an empty vocabulary")
        self.mode = mode
        self.pairs = self.seq = 0
        if mode == LOSS_PREFERENCE:
            if len(x._shape) != 3 or shape[0] % 2 or not all(shape):
                raise ValueError(
                    "preference logits are (2 pairs, sequence, vocabulary), "
                    "the chosen ones first, got %s" % (tuple(x._shape),))
            self.pairs, self.seq = shape[0] // 2, shape[1]
        given = []
        for what, t in (("reference", ref), ("old", old), ("advantages", adv),
                        ("weights", weight)):
            if t is not None:
                _float_operand(what, t)
                if t._shape != shape:
                    raise ValueError("%s have the labels' shape %s, got %s" % (
                        what, tuple(shape), tuple(t._shape)))
                if t._dtype != dtypes.kFloat32:
                    t = t.AsType(dtypes.kFloat32)
                t = Contiguous(t)
            given.append(t)
        self.extra = given
        self.x, self.label = Contiguous(x), Contiguous(label)
        _one_device("a token loss", x._dev, [self.label] +
                    [t for t in given if t is not None])
        self.consts = (float(beta), float(smoothing), 1.0 - float(clip[0]),
                       1.0 + float(clip[1]), float(kl))
        self.rows = 1
        for n in shape:
            self.rows *= n

    def forward(self):
        """-> the loss (1,) or, for the log-probabilities, (labels' shape);
        float32."""
        dev, rows, f32 = self.x._dev, self.rows, dtypes.kFloat32
        logp = self.mode == LOSS_LOG_PROB
        # kept of each row: the largest logit, the log of the sum relative to
        # it, the row's result (unless that is the output), its derivative
        # (policy); then what rows' derivatives are multiplied by (policy: one
        # number, preference: one for each pair)
        n = {LOSS_LOG_PROB: 2 * rows, LOSS_PREFERENCE: 3 * rows + self.pairs,
             LOSS_POLICY: 4 * rows + 1}[self.mode]
        self.saved = Tensor([n], dev, f32)
        loss = Tensor(self.label._shape if logp else [1], dev, f32)
        given = [t for t in self.extra if t is not None]
        here = [t is not None for t in self.extra]
        ins = [self.x, self.label] + given
        spec = (self.mode, rows, self.V, self.pairs, self.seq, self.consts)

        def body(*ts):
            flat = [t._storage() for t in ts]
            rest = iter(flat[2:])
            extra = [next(rest) if h else None for h in here]
            dev.math.token_loss_fwd(spec, flat[0], flat[1], extra, flat[-2],
                                    flat[-1])

        if self.rows or not logp:
            _submit(dev, "TokenLossForward", body, ins, [self.saved, loss])
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
            flat = [t._storage() for t in ts]
            dev.math.token_loss_bwd(spec, *flat[:3],
                                    flat[3] if weight else None,
                                    flat[-2] if dys else None, scale, flat[-1])

        reads = [self.x, self.label, self.saved] + weight + dys
        _one_device("TokenLossBackward", dev, reads)
        if self.rows:
            _submit(dev, "TokenLossBackward", body, reads, [dx])
        return dx


# ---------------------------------------------------------------------------
# AdamW
# ---------------------------------------------------------------------------
ADAMW_BLOCK = 256       # values that share the scale of an 8-bit state


_typed = operator.attrgetter("_dtype")
_held_in = operator.attrgetter("_block")
_placed = operator.attrgetter("_dev")


class AdamWGroup(object):
    """Parameters of one type, contiguous, and their states.  states: lists of
    the parameters' (m, v) -- float32, of the parameter's shape -- or, with 8
    bits, (m, r, m_scale, r_scale): int32 words of four e4m3 codes of the first
    moment and of the root of the second, in whole blocks of 256 values, and a
    float32 scale for each block; behind them, when ``mixed``, the float32
    master copies of 16-bit parameters.  It holds while every tensor in it
    keeps its block and storage (``holding``: parameters, then each list of
    states)."""

    def __init__(self, params, states, mixed):
        self.params, self.states = params, states
        self.mixed = bool(mixed)
        self.dev, self.dtype = params[0]._dev, params[0]._dtype
        n = len(params)
        # the tensors of a launch are stepped side by side
        _refuse(len(set(map(id, map(_held_in, params)))) != n,
                "a parameter twice in one step")
        self.members = [*params, *itertools.chain(*states)]
        _one_device("AdamWUpdateMulti", self.dev, self.members)
        self.sizes = [p.Size() for p in params]
        self.strides = [p._stride for p in params]
        storage = [t._storage() for t in self.members]
        self.columns = [storage[i:i + n] for i in range(0, len(storage), n)]
        self.holding = _rt.Holding(list(map(_held_in, self.members)))
        self.addresses = [[t.data_ptr() for t in c] for c in self.columns]


def AdamWUpdateMulti(group, grads, hypers, state_bits=32, scale=1.0, seed=0):
    """One AdamW step of an AdamWGroup (one graph node, one launch for every
    48 parameters).  hypers = (lr, weight_decay, epsilon, beta_1, beta_2,
    step): one-element float32 tensors."""
    dev, n = group.dev, len(group.params)
    if {group.dtype} != set(map(_typed, grads)):
        grads = [g.AsType(group.dtype) for g in grads]
    grads = [g if g._stride == s else Contiguous(g)
             for g, s in zip(grads, group.strides)]
    if {dev} != set(map(_placed, itertools.chain(grads, hypers))):
        _one_device("AdamWUpdateMulti", dev, [*grads, *hypers])
    scale, seed, state_bits = float(scale), int(seed), int(state_bits)
    if not dev.graph_enabled():
        flat = _rt.storages(list(map(_held_in, itertools.chain(grads, hypers))))
        if any(map(operator.is_, flat, itertools.repeat(None))):
            flat = [t._storage() for t in itertools.chain(grads, hypers)]
        dev.math.adamw_update_multi(
            group.sizes, group.columns, flat[:n], group.mixed, flat[n:],
            state_bits, scale, seed, group.addresses)
        return
    sizes, mixed = group.sizes, group.mixed

    def body(*ts):
        # the outputs stand behind the inputs: they are the same blocks
        flat = [t._storage() for t in ts[:len(group.members) + n + 6]]
        grads, flat = flat[:n], flat[n:]
        dev.math.adamw_update_multi(
            sizes, [flat[i:i + n] for i in range(0, len(flat) - 6, n)], grads,
            mixed, flat[-6:], state_bits, scale, seed)

    _submit(dev, "AdamWUpdateMulti", body, [*grads, *group.members, *hypers],
            group.members)
