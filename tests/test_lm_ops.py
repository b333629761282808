"""Rotary positions with head norms, losses over token log-probabilities and
AdamW against plain float64 evaluations, on the host and on the MI355X.

Tolerances count roundings: half a step of the result's type, relative to it
(fp32 2^-24, fp16 2^-11, bf16 2^-8), plus a number of float32 roundings of the
intermediate values, each at most 2^-24 of the values' scale."""
import copy
import gc
import math
import pickle
import weakref

import numpy as np
import pytest
import torch

import test_dist
from singa_amd import _rt, autograd, device, layer, model, opt, singa_wrap, tensor
from singa_amd.utils import checkpoint

E32 = 2.0 ** -24
HALF = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
# half of the smallest step of the type (float16 loses small gradients)
LEAST = {"float32": 0.0, "float16": 2.0 ** -25, "bfloat16": 0.0}
CODE = {"float32": tensor.float32, "float16": tensor.float16,
        "bfloat16": tensor.bfloat16}
TORCH = {"float32": torch.float32, "float16": torch.float16,
         "bfloat16": torch.bfloat16}
DTYPES = sorted(CODE)


@pytest.fixture(autouse=True)
def _training():
    autograd.training = True
    yield
    autograd.training = False


def rounded(x, dtype):
    """float64 values that the type holds."""
    return x.to(TORCH[dtype]).double()


def put(dev, x, dtype="float32", **kw):
    """A tensor on dev holding the float64 (or integer) torch tensor x."""
    if not x.is_floating_point():
        return tensor.Tensor(device=dev, data=x.numpy().astype(np.int32),
                             requires_grad=False)
    t = tensor.Tensor(device=dev, data=x.numpy().astype(np.float32))
    if dtype != "float32":
        t = t.as_type(CODE[dtype])
    for k, v in dict(requires_grad=True, **kw).items():
        setattr(t, k, v)
    return t


def got(t):
    """float64 torch tensor of a Tensor or core tensor."""
    if not isinstance(t, tensor.Tensor):
        t = tensor.from_raw_tensor(t)
    return torch.from_numpy(np.asarray(tensor.to_numpy(t), np.float64))


def check(t, want, dtype="float32", scale=0.0):
    """|t - want| <= half a step of the type + scale (a tensor or number)."""
    have = got(t).reshape(want.shape)
    room = HALF[dtype] * want.abs() + LEAST[dtype] + scale
    off = (have - want).abs()
    same = (have == want) | (torch.isnan(have) & torch.isnan(want))
    assert bool((same | (off <= room)).all()), \
        "off by %g where %g is allowed" % (
            float(off[~same].max()), float((off - room)[~same].max()))


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed),
                       dtype=torch.float64)


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------
def turn64(x, handle, positions, back=False):
    R = handle.rotary_dim
    f = torch.from_numpy(handle.frequencies)
    angle = positions.double().unsqueeze(-1).unsqueeze(-1) * f
    z = torch.polar(torch.full_like(angle, handle.amplitude), angle)
    if back:
        z = z.conj()
    y = x.clone()
    a, b = ((slice(0, R // 2), slice(R // 2, R)) if handle.layout == "half"
            else (slice(0, R, 2), slice(1, R, 2)))
    p = torch.complex(x[..., a].contiguous(), x[..., b].contiguous()) * z
    y[..., a], y[..., b] = p.real, p.imag
    return y


def rotary64(x, w, handle, positions, eps):
    if w is None:
        return turn64(x, handle, positions)
    r = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    return turn64(x * r * w, handle, positions)


def rotary_grad64(g, x, w, handle, positions, eps):
    """(dx, dw, sum of the magnitudes that dw adds up)"""
    g = turn64(g, handle, positions, back=True)
    if w is None:
        return g, None, None
    r = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    xh = x * r
    terms = g * xh
    g = g * w
    return r * (g - xh * (g * xh).mean(-1, keepdim=True)), \
        terms.sum((0, 1, 2)), terms.abs().sum((0, 1, 2))


ROTARY = [
    # B, S, H, K, D, R, layout, scaling, norm, positions
    (2, 9, 4, 2, 64, None, "half", None, True, "one"),
    (1, 1, 8, 1, 128, None, "half", ("ramp", 16.0, 8192), True, "far"),
    (3, 7, 3, 3, 80, 40, "interleaved", ("linear", 4.0), True, "each"),
    (2, 5, 1, 1, 2, None, "half", None, False, None),
    (2, 5, 1, 2, 6, 2, "interleaved", None, True, "negative"),
    (1, 33, 12, 4, 96, 32, "interleaved", ("base", 4.0), False, "far"),
    (1, 3, 5, 2, 256, 64, "half", None, True, None),
    (1, 2, 2, 1, 1024, 512, "half", None, True, "far"),
    (1, 2, 2, 1, 1022, 510, "interleaved", None, True, "far"),
    (1, 1300, 2, 1, 10, 6, "half", None, True, "each"),
    (2, 600, 7, 5, 32, 30, "half", None, True, None),
]


def rotary_inputs(case, dtype, seed=0):
    B, S, H, K, D, R, layout, scaling, norm, where = case
    handle = singa_wrap.RotaryHandle(D, R, layout=layout, scaling=scaling)
    gen = torch.Generator().manual_seed(seed)
    positions = {
        None: None, "one": torch.arange(S) + 5,
        "each": torch.randint(0, 5000, (B, S), generator=gen),
        "negative": -torch.arange(S) * 1000,
        "far": torch.randint((1 << 31) - 4096, (1 << 31) - 1, (B, S),
                             generator=gen)}[where]
    data = [rounded(1.5 * normal(seed + i, B, S, h, D), dtype)
            for i, h in enumerate((H, K, H, K))]
    scales = [rounded(1 + 0.2 * normal(seed + 9 + i, D), dtype)
              for i in range(2)] if norm else []
    at = torch.arange(S) if positions is None else positions
    return handle, positions, at, data, scales


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", ROTARY, ids=lambda c: "x".join(map(str, c[:6])))
def test_rotary(dev, case, dtype):
    handle, positions, at, (q, k, dq, dk), scales = rotary_inputs(case, dtype)
    eps = 1e-6
    op = autograd.Rotary(handle, None if positions is None
                         else put(dev, positions), norm=bool(scales), eps=eps)
    ys = op(*[put(dev, x, dtype) for x in [q, k] + scales])
    grads = op.backward(*[put(dev, x, dtype).data for x in (dq, dk)])
    assert len(ys) == 2 and len(grads) == 2 + len(scales)
    # an angle is good to 2^-24 half turns (pi of them), sine and cosine to two
    # roundings; a head's mean of squares to log2 of its width, the products to
    # a few more
    steps = (12 + 2 * math.log2(handle.head_dim)) * E32 * handle.amplitude
    for i, (x, g) in enumerate(((q, dq), (k, dk))):
        w = scales[i] if scales else None
        want = rotary64(x, w, handle, at, eps)
        check(ys[i], want, dtype, steps * float(want.abs().max()))
        dx, dw, mass = rotary_grad64(g, x, w, handle, at, eps)
        check(grads[i], dx, dtype, steps * float(dx.abs().max()) * 2)
        if scales:
            # terms good to `steps`, added in trees over at most a few rows
            check(grads[2 + i], dw, dtype, 2 * (steps + 32 * E32) * mass)


def test_rotary_gradient_is_the_difference(dev):
    case = (1, 3, 2, 1, 12, 8, "half", ("ramp", 4.0, 64), True, "each")
    handle, positions, at, (q, k, dq, dk), scales = rotary_inputs(case,
                                                                  "float32")
    op = autograd.Rotary(handle, put(dev, positions), norm=True)
    op(*[put(dev, x) for x in [q, k] + scales])
    grads = [got(g) for g in op.backward(put(dev, dq).data, put(dev, dk).data)]

    def loss(q, k, wq, wk):
        return (rotary64(q, wq, handle, at, 1e-6) * dq).sum() + \
            (rotary64(k, wk, handle, at, 1e-6) * dk).sum()

    args = [q, k] + scales
    for i, x in enumerate(args):
        for at_ in (0, x.numel() // 2, x.numel() - 1):
            h = torch.zeros_like(x).view(-1)
            h[at_] = 1e-5
            h = h.view(x.shape)
            up = loss(*[a + h if j == i else a for j, a in enumerate(args)])
            down = loss(*[a - h if j == i else a for j, a in enumerate(args)])
            slope = float(up - down) / 2e-5
            # central difference: 1e-10 of curvature, 2^-52 / 1e-5 of rounding
            assert abs(slope - float(grads[i].view(-1)[at_])) < \
                1e-6 + 64 * E32 * float(grads[i].abs().max())


def test_rotary_views_and_one_tensor(dev):
    """(batch, heads, sequence, dim) seen as (batch, sequence, heads, dim), a
    tensor whose rows are not contiguous, and one tensor alone."""
    handle = singa_wrap.RotaryHandle(24, 16)
    x = rounded(normal(3, 2, 5, 7, 24), "float32")        # B, H, S, D
    want = rotary64(x.transpose(1, 2), None, handle, torch.arange(7), 0)
    t = put(dev, x).transpose((0, 2, 1, 3))
    check(autograd.rotary(handle, t), want, scale=16 * E32 * 6)
    # the last dimension strided: copied first
    t = put(dev, x.transpose(2, 3).contiguous()).transpose((0, 3, 1, 2))
    check(autograd.rotary(handle, t), want, scale=16 * E32 * 6)
    w = rounded(1 + 0.1 * normal(5, 24), "float32")
    check(autograd.rotary(handle, t, scale=put(dev, w), eps=0.5),
          rotary64(x.transpose(1, 2), w, handle, torch.arange(7), 0.5),
          scale=24 * E32 * 6)


def test_rotary_through_the_tape(dev):
    """Gradients reach the leaves through autograd.backward; an output that
    nothing uses counts as zero."""
    handle = singa_wrap.RotaryHandle(8)
    q, k = normal(1, 2, 3, 4, 8), normal(2, 2, 3, 2, 8)
    wq, wk = 1 + 0.1 * normal(3, 8), 1 + 0.1 * normal(4, 8)
    q, k, wq, wk = (rounded(v, "float32") for v in (q, k, wq, wk))
    leaves = [put(dev, v, stores_grad=True) for v in (q, k, wq, wk)]
    for which in (0, 1):
        y = autograd.rotary_qk(handle, leaves[0], leaves[1], None, leaves[2],
                               leaves[3])
        target = put(dev, torch.zeros(y[which].shape, dtype=torch.float64))
        target.requires_grad = False
        grads = {id(p): got(g) for p, g in autograd.backward(
            autograd.mse_loss(y[which], target))}
        x, w = ((q, wq), (k, wk))[which]
        y64 = rotary64(x, w, handle, torch.arange(3), 1e-6)
        dx, dw, mass = rotary_grad64(2 * y64 / y64.numel(), x, w, handle,
                                     torch.arange(3), 1e-6)
        have = [grads[id(t)] for t in leaves]
        # dx is the small rest of terms as large as dy
        assert (have[which] - dx).abs().max() <= 64 * E32 * y64.abs().max()
        assert ((have[2 + which] - dw).abs() <= 64 * E32 * mass).all()
        assert not have[1 - which].any() and not have[3 - which].any()


def test_rotary_zero_rows_and_empty(dev):
    handle = singa_wrap.RotaryHandle(8)
    x = torch.zeros(1, 2, 3, 8, dtype=torch.float64)
    w = torch.ones(8, dtype=torch.float64)
    op = autograd.Rotary(handle, norm=True, eps=1e-6)
    y = op(put(dev, x), put(dev, w))[0]
    assert not got(y).any()
    g = normal(1, 1, 2, 3, 8)
    dx, dw = op.backward(put(dev, g).data)
    want = turn64(rounded(g, "float32"), handle, torch.arange(2), True) * 1e3
    check(dx, want, scale=16 * E32 * 4e3)
    assert not got(dw).any()
    none = tensor.Tensor((2, 0, 3, 8), dev)
    y = autograd.rotary(handle, none)
    assert y.shape == (2, 0, 3, 8)
    op = autograd.Rotary(handle, norm=True)
    op(none, put(dev, w))
    dx, dw = op.backward(none.data)
    assert dx.shape() == [2, 0, 3, 8] and not got(dw).any()


def test_rotary_scalings():
    D = 32
    i = np.arange(0, D, 2)
    plain = 10000.0 ** (-i / D)
    f = lambda **kw: singa_wrap.RotaryHandle(D, **kw).frequencies  # noqa: E731
    np.testing.assert_allclose(f(), plain, rtol=1e-14)
    np.testing.assert_allclose(f(scaling=("linear", 8)), plain / 8, rtol=1e-14)
    stretched = f(scaling=("base", 8))
    np.testing.assert_allclose(stretched[0], plain[0], rtol=1e-14)
    np.testing.assert_allclose(stretched[-1], plain[-1] / 8, rtol=1e-12)
    h = singa_wrap.RotaryHandle(D, scaling=("ramp", 8, 4096))
    turns = 4096 * plain / (2 * np.pi)
    np.testing.assert_allclose(h.frequencies[turns >= 32], plain[turns >= 32])
    np.testing.assert_allclose(h.frequencies[turns <= 1],
                               plain[turns <= 1] / 8)
    assert np.all(np.diff(h.frequencies) < 0)
    assert abs(h.amplitude - (1 + 0.1 * math.log(8))) < 1e-15
    assert singa_wrap.RotaryHandle(D, scaling=("ramp", 8, 4096),
                                   amplitude=1.0).amplitude == 1.0


def test_rotary_refusals(cpu_dev):
    H = singa_wrap.RotaryHandle
    for bad in (dict(head_dim=7), dict(head_dim=0), dict(head_dim=1026),
                dict(head_dim=8, rotary_dim=3), dict(head_dim=8, rotary_dim=10),
                dict(head_dim=1024, rotary_dim=514),
                dict(head_dim=8, layout="other"), dict(head_dim=8, base=0.5),
                dict(head_dim=8, base=float("nan")),
                dict(head_dim=8, scaling=("none", 2.0)),
                dict(head_dim=8, scaling=("linear",)),
                dict(head_dim=8, scaling=("linear", 0.5)),
                dict(head_dim=2, scaling=("base", 2.0)),
                dict(head_dim=8, scaling=("ramp", 2.0)),
                dict(head_dim=8, scaling=("ramp", 2.0, 64, 8, 8)),
                dict(head_dim=8, amplitude=float("inf"))):
        with pytest.raises(ValueError):
            H(**bad)
    h = H(8)

    def t(*shape, dtype=tensor.float32):
        return tensor.Tensor(shape, cpu_dev, dtype)

    x = t(2, 3, 4, 8)
    for call, error in (
            (lambda: autograd.rotary(h, t(2, 3, 8)), ValueError),
            (lambda: autograd.rotary(h, t(2, 3, 4, 6)), ValueError),
            (lambda: autograd.rotary(h, t(2, 3, 0, 8)), ValueError),
            (lambda: autograd.rotary(h, t(2, 3, 4, 8, dtype=tensor.int32)),
             TypeError),
            (lambda: autograd.rotary(h, x, t(3)), TypeError),
            (lambda: autograd.rotary(h, x, t(4, dtype=tensor.int32)),
             ValueError),
            (lambda: autograd.rotary(h, x, t(3, 2, dtype=tensor.int32)),
             ValueError),
            (lambda: autograd.rotary(h, x, scale=t(4)), ValueError),
            (lambda: autograd.rotary(h, x, scale=t(8, dtype=tensor.float16)),
             ValueError),
            (lambda: autograd.rotary(h, x, scale=t(8), eps=-1.0), ValueError),
            (lambda: autograd.rotary(h, x, scale=t(8), eps=float("nan")),
             ValueError),
            (lambda: autograd.rotary_qk(h, x, t(2, 4, 4, 8)), ValueError),
            (lambda: autograd.rotary_qk(h, x, t(2, 3, 4, 8,
                                                dtype=tensor.float16)),
             ValueError),
            (lambda: autograd.rotary_qk(h, x, x, q_scale=t(8)), ValueError),
            (lambda: autograd.Rotary(h)(x, x, x), ValueError),
            (lambda: autograd.Rotary(h, norm=True)(x), ValueError)):
        with pytest.raises(error):
            call()
    op = autograd.Rotary(h)
    op(x)
    with pytest.raises(ValueError):
        op.backward(t(2, 3, 4, 4).data)


# ---------------------------------------------------------------------------
# losses over token log-probabilities
# ---------------------------------------------------------------------------
def logits(seed, dtype, *shape):
    return rounded(3 * normal(seed, *shape), dtype)


def labels(seed, V, *shape, ignore=0.3):
    gen = torch.Generator().manual_seed(seed)
    t = torch.randint(0, V, shape, generator=gen)
    return torch.where(torch.rand(shape, generator=gen) < ignore,
                       torch.full_like(t, -1), t)


def log_prob64(x, t):
    V = x.shape[-1]
    used = (t >= 0) & (t < V)
    at = torch.where(used, t, torch.zeros_like(t)).unsqueeze(-1)
    lp = torch.log_softmax(x, -1).gather(-1, at).squeeze(-1)
    return torch.where(used, lp, torch.zeros_like(lp)), used


def rows_room(V):
    """Relative error of a row's probabilities: exponents of up to about 30 at
    one rounding each, products, and sums of up to V / 64 terms in a row."""
    return (64 + V / 64) * E32


def check_dx(have, c, x, t, used, dtype, room):
    """The gradient c (1[label] - softmax), c good to `room` relative."""
    V = x.shape[-1]
    p = torch.softmax(x, -1)
    p = torch.where(used.unsqueeze(-1), p, torch.zeros_like(p))
    at = torch.where(used, t, torch.zeros_like(t)).unsqueeze(-1)
    one = torch.zeros_like(p).scatter_(-1, at, 1.0)
    one = torch.where(used.unsqueeze(-1), one, torch.zeros_like(one))
    c = torch.where(used, c, torch.zeros_like(c)).unsqueeze(-1)
    check(have, c * (one - p), dtype,
          c.abs() * (rows_room(V) * p + room * (one + p)))
    # what is ignored is exactly zero
    assert not got(have).view(p.shape)[~used].any()


VOCABS = [1, 2, 63, 997, 4096, 4097, 50257]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", VOCABS)
def test_token_log_prob(dev, V, dtype):
    for shape in ((1,), (3, 5)):
        x, t = logits(V, dtype, *shape, V), labels(V + 1, V, *shape)
        t.view(-1)[0] = V - 1
        dy = rounded(normal(7, *shape), "float32")
        op = autograd.TokenLogProb(put(dev, t))
        y = op(put(dev, x, dtype))[0]
        want, used = log_prob64(x, t)
        assert y.dtype == tensor.float32 and y.shape == shape
        check(y, want, scale=rows_room(V) + 4 * E32 * 12)
        dx = op.backward(put(dev, dy).data)
        check_dx(dx, dy, x, t, used, dtype, 4 * E32)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 7, 300, 700])
def test_token_log_prob_pieces(gpu_dev, rows):
    """Few rows over a long vocabulary are cut into pieces; the cut falls
    anywhere, also where the rows are not aligned."""
    V = 20011
    x, t = logits(rows, "float16", rows, V), labels(rows, V, rows)
    t[0] = 0
    dy = rounded(normal(7, rows), "float32")
    op = autograd.TokenLogProb(put(gpu_dev, t))
    y = op(put(gpu_dev, x, "float16"))[0]
    want, used = log_prob64(x, t)
    check(y, want, scale=rows_room(V) + 4 * E32 * 14)
    check_dx(op.backward(put(gpu_dev, dy).data), dy, x, t, used, "float16",
             4 * E32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_token_log_prob_long_rows(gpu_dev, dtype):
    """Rows that eight waves share, and a gradient that is stored past the
    caches (over 128 MB)."""
    rows, V = (700, 50257) if dtype == "float32" else (1400, 50257)
    x, t = logits(rows, dtype, rows, V), labels(rows, V, rows)
    dy = rounded(normal(7, rows), "float32")
    op = autograd.TokenLogProb(put(gpu_dev, t))
    y = op(put(gpu_dev, x, dtype))[0]
    want, used = log_prob64(x, t)
    check(y, want, scale=rows_room(V) + 4 * E32 * 14)
    check_dx(op.backward(put(gpu_dev, dy).data), dy, x, t, used, dtype,
             4 * E32)


def preference64(x, t, ref, beta, smooth):
    lp, used = log_prob64(x, t)
    a = torch.where(used, lp - ref, torch.zeros_like(lp)).sum(-1)
    P = len(a) // 2
    z = beta * (a[:P] - a[P:])
    F = torch.nn.functional
    return ((1 - smooth) * F.softplus(-z) + smooth * F.softplus(z)).mean()


def policy64(x, t, old, adv, w, ref, clip, kl):
    lp, used = log_prob64(x, t)
    w = torch.ones_like(lp) if w is None else w
    used = used & (w != 0)
    zero = torch.zeros_like(lp)
    r = torch.exp(torch.where(used, lp - old, zero))
    each = -torch.minimum(r * adv, r.clamp(1 - clip[0], 1 + clip[1]) * adv)
    if kl:
        d = torch.where(used, ref - lp, zero)
        each = each + kl * (torch.exp(d) - d - 1)
    w = torch.where(used, w, zero)
    total = w.sum()
    return torch.where(used, w * each, zero).sum() / \
        (total if float(total) > 0 else 1.0)


def loss_and_coefficients(fn, x, t):
    """The loss in 64 bits, and its derivative for each log-probability: the
    gradient of logit t[r] is c (1 - p)."""
    x = x.clone().requires_grad_()
    y = fn(x)
    g, = torch.autograd.grad(y, x)
    return y.detach(), g


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("P,S,V", [(1, 1, 2), (1, 33, 997), (3, 7, 130),
                                   (17, 5, 65), (2, 40, 5000)])
def test_preference_loss(dev, P, S, V, dtype):
    x = logits(S, dtype, 2 * P, S, V)
    t = labels(V, V, 2 * P, S)
    t[0] = -1                       # a sequence of which nothing is left
    ref = rounded(log_prob64(x, t)[0] + 0.3 * normal(5, 2 * P, S), "float32")
    for beta, smooth, dy in ((0.1, 0.0, 1.0), (2.0, 0.25, -3.0)):
        op = autograd.PreferenceLoss(put(dev, t), put(dev, ref), beta, smooth)
        y = op(put(dev, x, dtype))[0]
        want, g = loss_and_coefficients(
            lambda v: preference64(v, t, ref, beta, smooth), x, t)
        assert y.dtype == tensor.float32 and y.shape == (1,)
        # z is beta times a sum over 2 S log-probabilities
        off = beta * 2 * S * (rows_room(V) + 16 * E32)
        check(y, want.reshape(1), scale=off + 8 * E32)
        dx = op.backward(dy)
        p = torch.softmax(x, -1)
        most = abs(dy) * beta / P
        check(dx, dy * g, dtype, most * (rows_room(V) + 2 * off + 16 * E32) *
              (p + (g != 0)))
        assert not got(dx).view(g.shape)[t < 0].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,V,weighted,kl", [
    (1, 2, False, 0.0), (9, 31, True, 0.05), (130, 997, True, 0.0),
    (40, 5001, False, 0.2), (2500, 64, True, 0.1)])
def test_policy_loss(dev, N, V, weighted, kl, dtype):
    x, t = logits(N, dtype, N, V), labels(V, V, N)
    if N == 1:
        t[0] = 1
    lp, used = log_prob64(x, t)
    f32 = lambda v: rounded(v, "float32")  # noqa: E731
    old, ref = f32(lp + 0.3 * normal(5, N)), f32(lp + 0.2 * normal(6, N))
    adv = f32(normal(8, N))
    w = f32(torch.rand(N, dtype=torch.float64,
                       generator=torch.Generator().manual_seed(1))) \
        if weighted else None
    if weighted:
        w[::4] = 0.0
    # away from the corners of the clip, where the derivative jumps
    r = torch.exp(lp - old)
    near = ((r - 0.8).abs() < 1e-3) | ((r - 1.28).abs() < 1e-3)
    old = torch.where(near, f32(old + 0.01), old)
    op = autograd.PolicyLoss(put(dev, t), put(dev, old), put(dev, adv),
                             None if w is None else put(dev, w), put(dev, ref),
                             clip=(0.2, 0.28), kl=kl)
    y = op(put(dev, x, dtype))[0]
    want, g = loss_and_coefficients(
        lambda v: policy64(v, t, old, adv, w, ref, (0.2, 0.28), kl), x, t)
    most = float(adv.abs().max()) * 4 + 4 * kl
    room = rows_room(V) + 32 * E32
    check(y, want.reshape(1), scale=most * room)
    dx = op.backward(2.0)
    p = torch.softmax(x, -1)
    total = 1.0 if w is None else float(w[used].sum())
    total = (float(used.sum()) if w is None else total) or 1.0
    weight = torch.ones(N, dtype=torch.float64) if w is None else w
    c = 2 * most * weight.unsqueeze(-1) / total
    check(dx, 2 * g, dtype, 4 * room * c * (p + (g != 0)))
    out = ~used if w is None else ~used | (w == 0)
    assert not got(dx)[out].any()


@pytest.mark.parametrize("V", [40, 5000])
def test_loss_gradients_are_the_differences(dev, V):
    P, S = 1, 3
    x, t = logits(1, "float32", 2 * P, S, V), labels(2, V, 2 * P, S, ignore=0)
    lp = log_prob64(x, t)[0]
    ref = rounded(lp + 0.2 * normal(3, 2 * P, S), "float32")
    old = rounded(lp + 0.05 * normal(4, 2 * P, S), "float32")
    adv = rounded(normal(5, 2 * P, S), "float32")
    for op, fn in (
            (autograd.PreferenceLoss(put(dev, t), put(dev, ref), 0.5, 0.1),
             lambda v: preference64(v, t, ref, 0.5, 0.1)),
            (autograd.PolicyLoss(put(dev, t), put(dev, old), put(dev, adv),
                                 reference=put(dev, ref), kl=0.1),
             lambda v: policy64(v, t, old, adv, None, ref, (0.2, 0.2), 0.1))):
        op(put(dev, x))
        dx = got(op.backward(1.0)).view(x.shape)
        for b, s in ((0, 0), (1, 2)):
            for v in (int(t[b, s]), (int(t[b, s]) + 1) % V):
                h = torch.zeros_like(x)
                h[b, s, v] = 1e-5
                slope = float(fn(x + h) - fn(x - h)) / 2e-5
                assert abs(slope - float(dx[b, s, v])) < 1e-7 + 200 * E32


@pytest.mark.parametrize("V", [37, 5003])
@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_and_infinite_logits(dev, V, dtype):
    """Ignored rows may hold anything; a vocabulary entry of minus infinity or
    of the type's lowest value has probability 0; a row of nothing else, NaN
    and plus infinity give NaN, and only to their own row."""
    low = float(torch.finfo(TORCH[dtype]).min)
    x = logits(3, dtype, 8, V)
    t = torch.tensor([-1, V, 3, 3, 3, 3, 3, -(1 << 31)])
    x[0], x[1, ::2], x[7] = float("nan"), float("inf"), -float("inf")
    x[2, V // 2:], x[3, V // 2:] = -float("inf"), low
    x[4] = -float("inf")
    x[5, 1], x[6, 2] = float("nan"), float("inf")
    op = autograd.TokenLogProb(put(dev, t))
    y = got(op(put(dev, x, dtype))[0])
    dx = got(op.backward(put(dev, torch.ones(8, dtype=torch.float64)).data))
    dx = dx.view(8, V)
    want, used = log_prob64(x, t)
    assert not y[[0, 1, 7]].any() and not dx[[0, 1, 7]].any()
    assert torch.isnan(y[4:7]).all() and torch.isnan(dx[5]).all()
    assert ((y[2:4] - want[2:4]).abs() <= rows_room(V) + 64 * E32).all()
    assert torch.isfinite(dx[2:4]).all() and not dx[2:4, V // 2:].any()
    # every entry the lowest value: uniform, not NaN
    x = torch.full((1, V), low, dtype=torch.float64)
    y = got(autograd.token_log_prob(put(dev, x, dtype),
                                    put(dev, torch.tensor([0]))))
    # x[label] - maximum is 0 exactly
    assert abs(float(y) + math.log(V)) <= (rows_room(V) + 16 * E32)
    # a label of probability 0
    x = logits(4, dtype, 2, 1, V)
    x[0, 0, 1] = -float("inf")
    op = autograd.PreferenceLoss(
        put(dev, torch.tensor([[1], [0]])),
        put(dev, torch.zeros(2, 1, dtype=torch.float64)), 0.5)
    assert float(got(op(put(dev, x, dtype))[0])) == float("inf")
    dx = got(op.backward(1.0)).view(2, V)
    assert abs(float(dx[0, 1]) + 0.5) < 1e-6 and torch.isfinite(dx).all()


@pytest.mark.parametrize("V", [37, 5003])
def test_logits_far_from_zero(dev, V):
    """Only differences of logits count: a row around 2^20 (whose float32
    neighbours are an eighth apart) and one of the lowest values."""
    x = logits(3, "float32", 3, V)
    x[0] = rounded(x[0] + 2.0 ** 20, "float32")
    x[1] = float(torch.finfo(torch.float32).min)
    t = torch.tensor([1, 2, 3])
    dy = rounded(normal(4, 3), "float32")
    op = autograd.TokenLogProb(put(dev, t))
    check(op(put(dev, x))[0], log_prob64(x, t)[0],
          scale=rows_room(V) + 64 * E32)
    check_dx(op.backward(put(dev, dy).data), dy, x, t, t >= 0, "float32",
             4 * E32)


def test_nothing_takes_part(dev):
    x = put(dev, torch.full((2, 3, 9), float("nan"), dtype=torch.float64))
    t = put(dev, torch.full((2, 3), -1))
    z = put(dev, torch.zeros(2, 3, dtype=torch.float64))
    nan = put(dev, torch.full((2, 3), float("nan"), dtype=torch.float64))
    op = autograd.PreferenceLoss(t, nan)
    assert abs(float(got(op(x)[0])) - math.log(2)) < 2 * E32
    assert not got(op.backward(1.0)).any()
    for w, lab in ((None, t), (z, put(dev, torch.zeros(2, 3).long()))):
        op = autograd.PolicyLoss(lab, nan, nan, w, nan, kl=0.1)
        assert float(got(op(x)[0])) == 0.0
        assert not got(op.backward(1.0)).any()
    none, no = tensor.Tensor((0, 5), dev), tensor.Tensor((0,), dev)
    op = autograd.TokenLogProb(tensor.Tensor((0,), dev, tensor.int32))
    assert op(none)[0].shape == (0,)
    assert op.backward(no.data).shape() == [0, 5]
    op = autograd.PolicyLoss(tensor.Tensor((0,), dev, tensor.int32), no, no)
    assert float(got(op(none)[0])) == 0.0
    assert op.backward(1.0).shape() == [0, 5]


def test_losses_through_the_tape(dev):
    """A loss that is scaled and added to another, over strided logits."""
    V = 23
    x, t = logits(1, "float32", 2, 3, V), labels(2, V, 2, 3)
    ref = rounded(normal(3, 2, 3), "float32")
    leaf = put(dev, x.transpose(1, 2).contiguous(), stores_grad=True)
    flat = autograd.transpose(leaf, (0, 2, 1))
    loss = autograd.preference_loss(flat, put(dev, t), put(dev, ref), 0.5)
    two = tensor.Tensor(device=dev, data=np.array([2.0], np.float32),
                        requires_grad=False)
    total = autograd.add(autograd.mul(loss, two), autograd.policy_loss(
        flat, put(dev, t), put(dev, ref), put(dev, ref)))
    (p, g), = autograd.backward(total)
    assert p is leaf
    _, want = loss_and_coefficients(
        lambda v: 2 * preference64(v, t, ref, 0.5, 0) +
        policy64(v, t, ref, ref, None, None, (0.2, 0.2), 0), x, t)
    assert (got(g).transpose(1, 2) - want).abs().max() < \
        64 * E32 * (2 + float(torch.exp(-ref).max()) * 4)


def test_loss_refusals(cpu_dev):
    def t(*shape, dtype=tensor.float32):
        return tensor.Tensor(shape, cpu_dev, dtype)

    i32 = dict(dtype=tensor.int32)
    x = t(4, 3, 9)
    lab, f = t(4, 3, **i32), t(4, 3)
    for call, error in (
            (lambda: autograd.token_log_prob(t(4, 3, 9, **i32), lab),
             TypeError),
            (lambda: autograd.token_log_prob(x, f), TypeError),
            (lambda: autograd.token_log_prob(x, t(3, 4, **i32)), ValueError),
            (lambda: autograd.token_log_prob(t(4, 0), t(4, **i32)),
             ValueError),
            (lambda: autograd.token_log_prob(t(9), t(**i32)), ValueError),
            (lambda: autograd.preference_loss(x, lab, t(4)), ValueError),
            (lambda: autograd.preference_loss(x, lab, lab), TypeError),
            (lambda: autograd.preference_loss(t(3, 3, 9), t(3, 3, **i32),
                                              t(3, 3)), ValueError),
            (lambda: autograd.preference_loss(t(0, 3, 9), t(0, 3, **i32),
                                              t(0, 3)), ValueError),
            (lambda: autograd.preference_loss(t(12, 9), t(12, **i32), t(12)),
             ValueError),
            (lambda: autograd.preference_loss(x, lab, f, smoothing=1.5),
             ValueError),
            (lambda: autograd.policy_loss(x, lab, f, t(4)), ValueError),
            (lambda: autograd.policy_loss(x, lab, f, f, clip=(1.5, 0.2)),
             ValueError),
            (lambda: autograd.policy_loss(x, lab, f, f, clip=-0.1),
             ValueError),
            (lambda: autograd.policy_loss(x, lab, f, f, kl=0.1), ValueError)):
        with pytest.raises(error):
            call()
    op = autograd.TokenLogProb(lab)
    op(x)
    for bad in (1.0, t(4).data):
        with pytest.raises(ValueError):
            op.backward(bad)


# ---------------------------------------------------------------------------
# AdamW
# ---------------------------------------------------------------------------
HYPER = dict(lr=0.01, beta_1=0.9, beta_2=0.99, epsilon=1e-8, weight_decay=0.1)
F32 = {k: float(np.float32(v)) for k, v in HYPER.items()}
SHAPES = [(3,), (1,), (256,), (17, 31), (255,), (257,), (64, 64), (4097,),
          (5, 7, 11)]


def adamw64(p, g, m, v, t):
    """One step from float64 states; -> p, m, v."""
    h = F32
    m = h["beta_1"] * m + (1 - h["beta_1"]) * g
    v = h["beta_2"] * v + (1 - h["beta_2"]) * g * g
    u = (m / (1 - h["beta_1"] ** t)) / (
        torch.sqrt(v / (1 - h["beta_2"] ** t)) + h["epsilon"])
    return p - h["lr"] * h["weight_decay"] * p - h["lr"] * u, m, v


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("master", [True, False])
def test_adamw_32(dev, dtype, master):
    o = opt.AdamW(**HYPER, master_weights=master)
    start = [rounded(normal(i, *s), dtype) for i, s in enumerate(SHAPES)]
    params = [put(dev, p, dtype) for p in start]
    for i, p in enumerate(params):
        p.name = "w%d" % i
    p64 = list(start)
    m64 = [torch.zeros_like(p) for p in start]
    v64 = [torch.zeros_like(p) for p in start]
    float_step = dtype == "float32" or master
    for step in range(1, 4):
        scale = 0.5 if step == 2 else 1.0
        grads = [rounded(normal(10 * step + i, *s), dtype)
                 for i, s in enumerate(SHAPES)]
        grads[0][0] = 0.0
        o.apply_many([(p, put(dev, g, dtype)) for p, g in zip(params, grads)],
                     scale)
        o.step()
        for i, g in enumerate(grads):
            p64[i], m64[i], v64[i] = adamw64(p64[i], g * scale, m64[i],
                                             v64[i], step)
            # per step: three roundings of the moments, some sixteen of the
            # update (at most about lr / 0.1), two of the parameter
            room = step * (16 * E32 * F32["lr"] * 10 + 3 * E32 *
                           p64[i].abs().max())
            check(o.m["w%d" % i], m64[i], scale=4 * E32 * step * 4)
            check(o.v["w%d" % i], v64[i], scale=4 * E32 * step * 16)
            if dtype != "float32" and master:
                check(o.masters["w%d" % i], p64[i], scale=room)
            if not float_step:      # rounded at every step
                room = room + step * HALF[dtype] * p64[i].abs().max()
            check(params[i], p64[i], dtype, room)


def codes64(words, scales):
    """The numbers that the 8-bit states stand for, and the codes alone."""
    c = torch.from_numpy(np.asarray(tensor.to_numpy(words)).astype(np.int32))
    c = c.view(torch.uint8).view(torch.float8_e4m3fn).float().double()
    s = got(scales)
    return (c.view(-1, 256) * s.view(-1, 1)).view(-1), c.view(-1, 256), s


def noise16(n, step, seed):
    """16 + 16 bits for each value: Philox4x32-10 in unsigned arithmetic."""
    u, low, half = np.uint64, np.uint64(0xffffffff), np.uint64(32)
    q = np.arange((n + 3) // 4, dtype=np.uint64)
    c = [q & low, q >> half, np.full_like(q, step), np.zeros_like(q)]
    k = [seed & 0xffffffff, seed >> 32]
    for _ in range(10):
        a, b = u(0xD2511F53) * c[0], u(0xCD9E8D57) * c[2]
        c = [(b >> half) ^ c[1] ^ u(k[0]), b & low,
             (a >> half) ^ c[3] ^ u(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xffffffff,
             (k[1] + 0xBB67AE85) & 0xffffffff]
    out = torch.from_numpy(np.stack(c, 1).reshape(-1)[:n].astype(np.int64))
    return (out & 0xffff).double() / 65536, (out >> 16).double() / 65536


def check_codes(codes, scales, x, u, keep):
    """Codes of the values x (float64): the stochastic rounding of x / scale.
    Where x / scale + u is within its error of a whole number of steps (x good
    to 8 roundings of at most 16 steps) either neighbour will do."""
    n = x.numel()
    pad = torch.zeros(codes.numel() - n, dtype=torch.float64)
    x, u = torch.cat([x, pad]).view(-1, 256), torch.cat([u, pad]).view(-1, 256)
    top = x.abs().amax(1)
    assert ((scales - top / 448).abs() <= 8 * E32 * top / 448).all()
    t = x.abs() * torch.where(top > 0, 448 / top, torch.zeros_like(top))[:, None]
    unit = torch.exp2(torch.floor(torch.log2(t.clamp_min(2.0 ** -6))) - 3)
    lo, hi = (torch.floor(t / unit + u + e) * unit for e in
              (-128 * E32, 128 * E32))
    if keep:
        lo, hi = (torch.where(t > 0, v.clamp_min(2.0 ** -9), v)
                  for v in (lo, hi))
    lo, hi = (torch.where(t > 0, v, torch.zeros_like(v)).clamp_max(448)
              for v in (lo, hi))
    c = codes.abs()
    assert ((c == lo) | (c == hi)).all()
    assert (torch.sign(codes)[c > 0] == torch.sign(x)[c > 0]).all()
    # rarely either
    assert float((lo != hi).double().mean()) < 0.01


@pytest.mark.parametrize("dtype", DTYPES)
def test_adamw_8(dev, dtype):
    o = opt.AdamW(**HYPER, state_bits=8, seed=77)
    start = [rounded(normal(i, *s), dtype) for i, s in enumerate(SHAPES)]
    params = [put(dev, p, dtype) for p in start]
    for i, p in enumerate(params):
        p.name = "w%d" % i
    for step in range(1, 4):
        # magnitudes over many binades, zeros among them
        grads = [rounded(normal(10 * step + i, *s) *
                         torch.exp(2 * normal(99 + i, *s)), dtype)
                 for i, s in enumerate(SHAPES)]
        grads[3][2] = 0.0
        before = []
        for i, s in enumerate(SHAPES):
            n, key = math.prod(s), "w%d" % i
            if step == 1:
                before.append([torch.zeros(n, dtype=torch.float64)] * 2)
            else:
                before.append([codes64(a[key], b[key])[0][:n] for a, b in
                               ((o.m, o.m_scale), (o.r, o.r_scale))])
        held = [got(o.masters["w%d" % i]) if dtype != "float32" and step > 1
                else got(p) for i, p in enumerate(params)]
        o.apply_many([(p, put(dev, g, dtype)) for p, g in zip(params, grads)])
        o.step()
        for i, g in enumerate(grads):
            key, n = "w%d" % i, g.numel()
            m, r = before[i]
            p64, m, v = adamw64(held[i].view(-1), g.view(-1), m, r * r, step)
            room = 16 * E32 * F32["lr"] * 10 + 3 * E32 * p64.abs()
            check(params[i], p64.view(g.shape), dtype, room.view(g.shape))
            um, ur = noise16(n, step - 1, 77)
            _, c, s = codes64(o.m[key], o.m_scale[key])
            check_codes(c, s, m, um, False)
            _, c, s = codes64(o.r[key], o.r_scale[key])
            check_codes(c, s, torch.sqrt(v), ur, True)
            assert not c.view(-1)[n:].any()


def test_adamw_8_bad_gradients_stay_alone(dev):
    """An infinite or NaN gradient spoils its own element only."""
    g = normal(1, 600)
    clean = rounded(g, "float32")
    g = clean.clone()
    g[3], g[300], g[301] = float("nan"), float("inf"), -float("inf")
    runs = []
    for grad in (clean, g):
        o = opt.AdamW(**HYPER, state_bits=8)
        p = put(dev, normal(2, 600))
        p.name = "w"
        for _ in range(2):
            o.apply_many([(p, put(dev, grad))])
            o.step()
        runs.append((got(p), codes64(o.m["w"], o.m_scale["w"])[0][:600],
                     codes64(o.r["w"], o.r_scale["w"])[0][:600]))
    good = torch.ones(600, dtype=torch.bool)
    good[[3, 300, 301]] = False
    for a, b in zip(*runs):
        assert torch.isfinite(b[good]).all() and torch.isnan(b[~good]).any()
    # and the others are stepped as without it, up to their scale's largest
    assert (runs[0][0][good] - runs[1][0][good]).abs().max() < 0.02


def test_adamw_8_rounding_keeps_the_mean(dev):
    """The second moment's root moves by less than a code's step: rounded to
    the nearest it would stand still; stochastically it follows on average."""
    n = 4096
    o = opt.AdamW(lr=0.0, beta_2=0.99, weight_decay=0.0, state_bits=8)
    p = put(dev, torch.zeros(n, dtype=torch.float64))
    p.name = "w"
    g = torch.full((n,), 0.5, dtype=torch.float64)
    g[::256] = 1.0                   # every block's largest
    for _ in range(60):
        o.apply_many([(p, put(dev, g))])
        o.step()
    r = codes64(o.r["w"], o.r_scale["w"])[0]
    rest = torch.ones(n, dtype=torch.bool)
    rest[::256] = False
    want = 0.5 * math.sqrt(1 - 0.99 ** 60)
    # 3840 values, each within a step (an eighth) or two of the mean: the
    # mean's own deviation is under a quarter of a percent
    assert abs(float(r[rest].mean()) / want - 1) < 0.02


def test_adamw_schedule_states_and_masters(dev):
    """A schedule is followed; states carried over continue bit for bit."""
    lr = opt.ExponentialDecay(0.1, 1, 0.5)
    for bits in (32, 8):
        def fresh(states=None):
            o = opt.AdamW(lr=lr, state_bits=bits, seed=5)
            p = put(dev, normal(1, 700), "float16")
            p.name = "w"
            if states:
                p.copy_from_numpy(states["p"])
                o.set_states(states)
            return o, p

        grads = [put(dev, normal(10 + i, 700), "float16") for i in range(4)]
        o, p = fresh()
        for g in grads[:2]:
            o.apply_many([(p, g)])
            o.step()
        saved = {k: {n: tensor.from_numpy(tensor.to_numpy(t))
                     for n, t in v.items()} if isinstance(v, dict) else v
                 for k, v in o.get_states().items()}
        saved["p"] = tensor.to_numpy(p)
        o2, p2 = fresh(saved)
        for g in grads[2:]:
            for a, b in ((o, p), (o2, p2)):
                a.apply_many([(b, g)])
                a.step()
        assert abs(float(got(o.lr_value)) - 0.1 / 16) < 1e-6
        assert (got(p) == got(p2)).all()
        assert (got(o.masters["w"]) == got(o2.masters["w"])).all()
        for name in o.state_names:
            a, b = getattr(o, name)["w"], getattr(o2, name)["w"]
            assert (tensor.to_numpy(a) == tensor.to_numpy(b)).all()
        # a 16-bit parameter is its master, rounded
        assert (got(p) == rounded(got(o.masters["w"]), "float16")).all()


def test_adamw_follows_its_tables(dev):
    """A step reads the states that the tables hold now: masters dropped or
    overwritten, states loaded in place or put in anew."""
    o = opt.AdamW(lr=0.1, weight_decay=0.0)
    p, g = put(dev, normal(1, 300), "float16"), put(dev, normal(2, 300),
                                                    "float16")
    p.name = "w"
    o.apply_many([(p, g)])
    o.forget_masters()
    p.copy_from_numpy(np.full(300, 5.0, np.float16))
    o.apply_many([(p, g)])
    assert (got(p) - 5.0).abs().max() < 0.5
    p.copy_from_numpy(np.full(300, -5.0, np.float16))
    o.sync_masters({"w": p})
    o.apply_many([(p, g)])
    assert (got(p) + 5.0).abs().max() < 0.5
    zero = put(dev, torch.zeros(300, dtype=torch.float64))
    for fresh in (False, True):
        o.apply_many([(p, g)])
        if fresh:
            o.m["w"] = zero.clone()
        else:
            o.set_states(dict(o.get_states(), m={"w": zero}))
        o.apply_many([(p, g)])
        check(o.m["w"], got(g) * 0.1, scale=4 * E32)
    # a state moved or converted under the optimizer's hands
    o.v["w"].to_type(tensor.float16)
    with pytest.raises(ValueError):
        o.apply_many([(p, g)])
    o.v["w"] = zero.clone()
    o.apply_many([(p, g)])
    # a parameter that grew has states of the wrong size
    p.data.Resize([400])
    p.shape = (400,)
    with pytest.raises(ValueError):
        o.apply_many([(p, put(dev, normal(2, 400), "float16"))])
    # another tensor in the parameter's place: the same name, its own state
    q = put(dev, normal(1, 20))
    q.name = "w"
    o.apply_many([(q, put(dev, normal(2, 20)))])
    assert got(o.m["w"]).numel() == 300 and len(o.m) == 2


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_large_step(gpu_dev, bits):
    """Large enough to go past the caches; whole chunks and a ragged end."""
    o = opt.AdamW(**HYPER, state_bits=bits, seed=9)
    n = [5_000_003, 4_100_000]
    start = [rounded(normal(i, k), "float32") for i, k in enumerate(n)]
    grads = [rounded(normal(9 + i, k), "float32") for i, k in enumerate(n)]
    params = [put(gpu_dev, p) for p in start]
    for i, p in enumerate(params):
        p.name = "w%d" % i
    o.apply_many([(p, put(gpu_dev, g)) for p, g in zip(params, grads)])
    for i, g in enumerate(grads):
        zero = torch.zeros_like(g)
        p64, m, v = adamw64(start[i], g, zero, zero, 1)
        check(params[i], p64, scale=16 * E32 * F32["lr"] * 10 +
              3 * E32 * p64.abs())
        key = "w%d" % i
        if bits == 32:
            check(o.m[key], m, scale=16 * E32)
            check(o.v[key], v, scale=64 * E32)
            continue
        um, ur = noise16(n[i], 0, 9)
        for words, scales, x, u, keep in (
                (o.m, o.m_scale, m, um, False),
                (o.r, o.r_scale, torch.sqrt(v), ur, True)):
            _, c, s = codes64(words[key], scales[key])
            check_codes(c, s, x, u, keep)


def test_adamw_refusals(cpu_dev):
    with pytest.raises(ValueError):
        opt.AdamW(state_bits=4)
    with pytest.raises(ValueError):
        opt.AdamW(weight_decay=-1.0)
    p = put(cpu_dev, normal(1, 300))
    p.name = "w"
    g = put(cpu_dev, normal(2, 300))
    a, b = opt.AdamW(), opt.AdamW(state_bits=8)
    for o in (a, b):
        o.apply_many([(p, g)])
    with pytest.raises(ValueError):
        opt.AdamW(state_bits=8).set_states(a.get_states())
    with pytest.raises(ValueError):
        opt.AdamW().set_states(b.get_states())
    states = b.get_states()
    states["m"] = {"w": tensor.Tensor((3,), cpu_dev, tensor.int32)}
    o = opt.AdamW(state_bits=8)
    o.set_states(states)
    with pytest.raises(ValueError):
        o.apply_many([(p, g)])
    # one launch steps its tensors side by side: the same memory only once
    for twice in (p, p.copy()):
        with pytest.raises(ValueError):
            opt.AdamW().apply_many([(p, g), (twice, g)])
    q = put(cpu_dev, normal(1, 4, 5)).transpose()
    q.name = "q"
    with pytest.raises(ValueError):
        opt.AdamW().apply_many([(q, put(cpu_dev, normal(1, 5, 4)))])


# ---------------------------------------------------------------------------
# together: one step of preference tuning of a small decoder
# ---------------------------------------------------------------------------
class Decoder(model.Model):
    """One layer: embedding, normed rotary attention (causal), read-out."""

    def __init__(self, vocab, heads=2, dim=64):
        super().__init__()
        self.heads, self.dim = heads, dim
        self.emb = layer.Embedding(vocab, heads * dim)
        self.q, self.k, self.v = (layer.Linear(heads * dim, bias=False)
                                  for _ in range(3))
        self.rope = layer.RotaryQK(norm=True)
        self.out = layer.Linear(vocab, bias=False)
        self.loss = layer.PreferenceLoss(beta=0.5)

    def forward(self, ids, mask):
        x = self.emb(ids)
        B, S = ids.shape
        q, k, v = (autograd.reshape(f(x), (B, S, self.heads, self.dim))
                   for f in (self.q, self.k, self.v))
        q, k = self.rope(q, k)
        y = autograd.attention(autograd.transpose(q, (0, 2, 1, 3)),
                               autograd.transpose(k, (0, 2, 3, 1)),
                               autograd.transpose(v, (0, 2, 1, 3)), mask,
                               self.dim ** -0.5)
        return self.out(y)

    def train_one_batch(self, ids, t, ref, mask):
        logits = self.forward(ids, mask)
        loss = self.loss(logits, t, ref)
        self.optimizer(loss)
        return logits, loss


def decoder64(w, ids, t, ref, S, handle, beta=0.5):
    B = len(ids)
    x = w["emb.W"][ids]
    q, k, v = ((x @ w["%s.W" % n]).view(B, S, 2, 64) for n in "qkv")
    q = rotary64(q, w["rope.q_scale"], handle, torch.arange(S), 1e-6)
    k = rotary64(k, w["rope.k_scale"], handle, torch.arange(S), 1e-6)
    q, k, v = (z.transpose(1, 2) for z in (q, k, v))
    a = (q @ k.transpose(2, 3)) / 8.0
    a = a.masked_fill(torch.ones(S, S).triu(1).bool(), -float("inf"))
    y = (torch.softmax(a, -1) @ v).transpose(1, 2).reshape(B, S, 128)
    return preference64(y @ w["out.W"], t, ref, beta, 0.0)


@pytest.mark.parametrize("use_graph", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
def test_preference_tuning_step(dev, use_graph, bits):
    """Rotary, attention, preference loss and AdamW as a program runs them,
    eagerly and as a recorded (on the GPU: captured) step that is replayed;
    gradients, through the first step's moments, against float64."""
    P, S, V = 2, 9, 53
    gen = torch.Generator().manual_seed(0)
    ids = torch.randint(0, V, (2 * P, S), generator=gen)
    t, ref = labels(1, V, 2 * P, S), rounded(-4 + normal(2, 2 * P, S),
                                             "float32")
    mask = torch.full((S, S), -1e9, dtype=torch.float64).triu(1)
    tx, tt = put(dev, ids), put(dev, t)
    tr, tm = put(dev, ref), put(dev, mask)
    tr.requires_grad = tm.requires_grad = False
    tm = tm.reshape((1, 1, S, S))
    tm.requires_grad = False
    m = Decoder(V)
    m.compile([tx, tm], is_train=True, use_graph=use_graph, sequential=False)
    params = m.get_params()
    for i, (name, p) in enumerate(sorted(params.items())):
        w = normal(50 + i, *p.shape) * (0.3 if len(p.shape) == 2 else 0.1)
        p.copy_from_numpy((w + (len(p.shape) == 1)).numpy()
                          .astype(np.float32))
    start = {n: got(p).requires_grad_() for n, p in params.items()}
    o = opt.AdamW(lr=0.01, state_bits=bits)
    m.set_optimizer(o)
    handle = singa_wrap.RotaryHandle(64)
    bare = {n.split("Decoder.")[-1]: p for n, p in start.items()}
    want = decoder64(bare, ids, t, ref, S, handle)
    grads = dict(zip(start, torch.autograd.grad(want, list(start.values()))))
    losses = []
    for step in range(4):
        _, loss = m(tx, tt, tr, tm)
        losses.append(float(got(loss)))
        if step == 0:
            # float32 products of 128 terms behind each other
            assert abs(losses[0] - float(want.detach())) < 1e-4
            for n, p in params.items():
                g = grads[n]
                if bits == 32:
                    have = got(o.m[p.name]) / (1 - F32["beta_1"])
                else:
                    have = codes64(o.m[p.name], o.m_scale[p.name])[0]
                    have = have[:g.numel()].view(g.shape) / 0.1
                # 8 bits: a step (an eighth) of the value, the least code
                room = 2e-4 * g.abs().max() + 1e-7
                if bits == 8:
                    room = room + g.abs() / 8 + g.abs().max() * 2.0 ** -17
                assert ((have - g).abs() <= room).all(), n
    first = {n: got(p) for n, p in params.items()}
    # the same program again gives the same result, replayed or not
    for n, p in params.items():
        p.copy_from_numpy(start[n].detach().numpy().astype(np.float32))
    dev.EnableGraph(False)
    o2 = opt.AdamW(lr=0.01, state_bits=bits)
    m.graph_mode = False
    autograd.training = True
    for step in range(4):
        loss = m.loss(m.forward(tx, tm), tt, tr)
        o2(loss)
        # the embedding's and the products' sums may be added in another order
        assert abs(float(got(loss)) - losses[step]) < 1e-3
    assert losses[-1] == losses[-1]
    if bits == 32:
        for n, p in params.items():
            assert (got(p) - first[n]).abs().max() < 0.02


@pytest.mark.gpu
def test_another_stream(gpu_dev):
    """The operators run on the stream that is current."""
    handle = singa_wrap.RotaryHandle(64)
    x = rounded(normal(1, 2, 50, 4, 64), "float32")
    s = torch.cuda.Stream()
    t = put(gpu_dev, x)
    lg, lab = logits(2, "float32", 30, 5000), labels(3, 5000, 30)
    tl, tt = put(gpu_dev, lg), put(gpu_dev, lab)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        y = autograd.rotary(handle, t)
        z = autograd.token_log_prob(tl, tt)
    s.synchronize()
    check(y, rotary64(x, None, handle, torch.arange(50), 0), scale=24 * E32 * 6)
    check(z, log_prob64(lg, lab)[0], scale=rows_room(5000) + 64 * E32)


@pytest.mark.gpu
def test_offsets_beyond_32_bits(gpu_dev):
    """More than 2^31 values in one tensor: its first and last rows."""
    if torch.cuda.mem_get_info()[0] < 100 << 30:
        pytest.skip("needs 100 GB of device memory")

    def raw(*shape, dtype=tensor.bfloat16):
        t = tensor.Tensor(shape, gpu_dev, dtype)
        return t, t.data.view()

    # losses
    V, rows = 50257, 43000
    x, vx = raw(rows, V)
    t, vt = raw(rows, dtype=tensor.int32)
    dy, vd = raw(rows, dtype=tensor.float32)
    vx.zero_()
    vt.fill_(-1)
    vd.fill_(0.5)
    ends = [0, 1, rows - 2, rows - 1]
    some = logits(1, "bfloat16", 4, V)
    lab = torch.tensor([3, V - 1, 0, V - 1])
    vx[ends] = some.to(vx)
    vt[ends] = lab.to(vt)
    op = autograd.TokenLogProb(t)
    y = op(x)[0].data.view()
    want, used = log_prob64(some, lab)
    assert ((y[ends].double().cpu() - want).abs() <=
            rows_room(V) + 64 * E32).all()
    dx = op.backward(dy.data).view()
    check_dx(tensor.Tensor(device=device.get_default_device(),
                           data=dx[ends].float().cpu().numpy()),
             torch.full((4,), 0.5, dtype=torch.float64), some, lab, used,
             "bfloat16", 4 * E32)
    assert not dx[2:rows - 2].any()
    del x, vx, dx, op
    # rotary: 2^31 + 2^13 values
    S, H, D = (1 << 19) + 2, 32, 128
    handle = singa_wrap.RotaryHandle(D)
    x, vx = raw(1, S, H, D)
    vx.fill_(1.0)
    y = autograd.rotary(handle, x).data.view()
    for s in (0, 1, S - 2, S - 1):
        want = turn64(torch.ones(1, 1, 1, D, dtype=torch.float64), handle,
                      torch.tensor([s]))
        off = (y[0, s].double().cpu() - want[0, 0]).abs()
        assert (off <= HALF["bfloat16"] * want[0, 0].abs() + 24 * E32).all()
    del x, vx, y
    # AdamW, 8 bits: the last of 2^31 + 300 elements
    n = (1 << 31) + 300
    p, vp = raw(n)
    g, vg = raw(n)
    vp.fill_(1.0)
    vg.fill_(0.25)
    p.name = "w"
    o = opt.AdamW(lr=0.5, weight_decay=0.0, state_bits=8, master_weights=False)
    o.apply_many([(p, g)])
    # every first step is lr long: 1 - 0.5
    for part in (vp[:300], vp[(1 << 31) - 5:]):
        assert ((part.double() - 0.5).abs() <= HALF["bfloat16"]).all()
    words = o.m["w"].data.view()
    # the largest of every block is its scale times 448, code 0x7e; where the
    # product falls a rounding short and the noise is 0 (of 2^16) the code below
    whole = (words == 0x7e7e7e7e).sum().item()
    assert n // 4 * (1 - 2.0 ** -13) < whole <= n // 4


@pytest.mark.gpu
def test_operands_of_another_device_are_refused(gpu_dev, cpu_dev):
    h = singa_wrap.RotaryHandle(8)
    x = tensor.Tensor((1, 2, 3, 8), gpu_dev)
    lg = tensor.Tensor((2, 9), gpu_dev)
    lab = tensor.Tensor((2,), gpu_dev, tensor.int32)
    f = tensor.Tensor((2,), cpu_dev)
    for call in (
            lambda: autograd.rotary(h, x, tensor.Tensor((2,), cpu_dev,
                                                        tensor.int32)),
            lambda: autograd.rotary(h, x, scale=tensor.Tensor((8,), cpu_dev)),
            lambda: autograd.token_log_prob(lg, tensor.Tensor(
                (2,), cpu_dev, tensor.int32)),
            lambda: autograd.policy_loss(lg, lab, f, f),
            lambda: opt.AdamW().apply_many([(lg, tensor.Tensor((2, 9),
                                                               cpu_dev))])):
        with pytest.raises(ValueError):
            call()


@pytest.mark.gpu
def test_many_rows(gpu_dev):
    """More rows than one launch takes, and sums over more than one workgroup
    adds up."""
    N, V = (1 << 22) + 5, 3
    x, t = logits(1, "float16", N, V), labels(2, V, N)
    x[-5:], t[-5:] = x[:5], torch.tensor([0, 1, 2, -1, 1])
    lp, used = log_prob64(x, t)
    old = rounded(lp + 0.1 * normal(3, N), "float32")
    adv = rounded(normal(4, N), "float32")
    tx, tt = put(gpu_dev, x, "float16"), put(gpu_dev, t)
    op = autograd.TokenLogProb(tt)
    check(op(tx)[0], lp, scale=rows_room(V) + 64 * E32)
    check_dx(op.backward(put(gpu_dev, adv).data), adv, x, t, used, "float16",
             4 * E32)
    op = autograd.PolicyLoss(tt, put(gpu_dev, old), put(gpu_dev, adv))
    want, g = loss_and_coefficients(
        lambda v: policy64(v, t, old, adv, None, None, (0.2, 0.2), 0.0), x, t)
    # each token's term good to a few roundings of at most |r A|
    check(op(tx)[0], want.reshape(1), scale=float((4 * adv.abs()).mean()) *
          (rows_room(V) + 32 * E32))
    dx = got(op.backward(float(N))).view(N, V)
    room = HALF["float16"] * (N * g).abs() + 2.0 ** -25 + \
        4 * adv.abs().unsqueeze(-1) * 64 * (rows_room(V) + 32 * E32)
    assert ((dx - N * g).abs() <= room).all()
    # 2 x 2100 sequences of 9: a workgroup for each
    P, S = 2100, 9
    x, t = x[:2 * P * S].view(2 * P, S, V), t[:2 * P * S].view(2 * P, S)
    ref = rounded(lp[:2 * P * S].view(2 * P, S) + 0.3 * normal(5, 2 * P, S),
                  "float32")
    op = autograd.PreferenceLoss(put(gpu_dev, t), put(gpu_dev, ref), 0.5, 0.1)
    y = op(put(gpu_dev, x, "float16"))[0]
    want, g = loss_and_coefficients(
        lambda v: preference64(v, t, ref, 0.5, 0.1), x, t)
    off = 0.5 * 2 * S * (rows_room(V) + 16 * E32)
    check(y, want.reshape(1), scale=off + 8 * E32)
    dx = got(op.backward(float(P))).view(2 * P, S, V)
    assert ((dx - P * g).abs() <= HALF["float16"] * (P * g).abs() +
            2.0 ** -25 + 0.5 * (rows_room(V) + 2 * off + 32 * E32)).all()


@pytest.mark.gpu
def test_results_repeat(gpu_dev):
    """No atomics: the same call gives the same bits."""
    handle = singa_wrap.RotaryHandle(128)
    q = rounded(normal(1, 2, 700, 8, 128), "bfloat16")
    w = rounded(1 + 0.1 * normal(2, 128), "bfloat16")
    x, t = logits(3, "bfloat16", 6, 50, 5001), labels(4, 5001, 6, 50)
    ref = rounded(normal(5, 6, 50), "float32")
    runs = []
    for _ in range(3):
        op = autograd.Rotary(handle, norm=True)
        op(put(gpu_dev, q, "bfloat16"), put(gpu_dev, w, "bfloat16"))
        a = op.backward(put(gpu_dev, q, "bfloat16").data)
        op = autograd.PreferenceLoss(put(gpu_dev, t), put(gpu_dev, ref))
        y = op(put(gpu_dev, x, "bfloat16"))[0]
        runs.append([got(v) for v in (*a, y, op.backward(1.0))])
    for other in runs[1:]:
        for a, b in zip(runs[0], other):
            assert torch.equal(a, b)


def test_devices_agree_on_the_handle(cpu_dev):
    """The fixed-point turns hold the frequencies to 2^-52."""
    h = singa_wrap.RotaryHandle(64, scaling=("ramp", 8.0, 4096))
    turns = h._turns.astype(np.float64) / 2.0 ** 64
    np.testing.assert_allclose(turns * 2 * np.pi, h.frequencies, rtol=1e-14)
    assert device.get_default_device() is cpu_dev


def test_handle_copies_own_their_turns(cpu_dev):
    """A copied or unpickled handle addresses its own table."""
    h = singa_wrap.RotaryHandle(64, 32, layout="interleaved",
                                scaling=("linear", 4.0))
    for other in (copy.copy(h), copy.deepcopy(h),
                  pickle.loads(pickle.dumps(h))):
        assert other.turns_address == other._turns.ctypes.data
        assert (other._turns == h._turns).all()
        assert (other.half, other.rotary_dim) == (h.half, h.rotary_dim)


def test_adamw_lets_go_of_replaced_parameters(dev):
    """What a step kept of a parameter that is gone is dropped by the next
    step that looks states up; one that lives keeps its own."""
    o = opt.AdamW(lr=0.1)
    stays = put(dev, normal(1, 40))
    o.apply_many([(stays, put(dev, normal(2, 40)))])
    gone = []
    for _ in range(4):
        p = put(dev, normal(1, 300))
        p.name = "w"
        o.apply_many([(p, put(dev, normal(2, 300)))])
        gone.append(weakref.ref(p.data))
        del p
        gc.collect()
    # the last one stays until something else is looked up
    assert [r() is None for r in gone] == [True] * 3 + [False]
    q = put(dev, normal(1, 20))
    o.apply_many([(q, put(dev, normal(2, 20)))])
    gc.collect()
    assert gone[-1]() is None and len(o._groups) == 2
    # both of those live: the same group is found again
    found = dict(o._groups)
    o.apply_many([(stays, put(dev, normal(2, 40)))])
    assert all(o._groups[k] is v for k, v in found.items())


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_empty_parameters(dev, bits):
    """Parameters of no elements among others are stepped over."""
    for order in ((0, 700), (700, 0), (0, 0, 700, 0, 5), (0,)):
        o = opt.AdamW(lr=0.1, state_bits=bits)
        alone = opt.AdamW(lr=0.1, state_bits=bits)
        a, b = [], []
        for i, n in enumerate(order):
            g = put(dev, normal(10 + i, n))
            p, q = put(dev, normal(i, n)), put(dev, normal(i, n))
            a.append((p, g))
            if n:
                b.append((q, g))
        for _ in range(2):
            o.apply_many(a)
            alone.apply_many(b)
            o.step()
            alone.step()
        for (p, _), (q, _) in zip([e for e in a if e[0].size()], b):
            assert (got(p) == got(q)).all()


def test_rotary_layer_amplitude(dev):
    """The layer takes the handle's amplitude."""
    q, k = (put(dev, normal(s, 1, 3, 2, 8)) for s in (1, 2))
    plain = layer.RotaryQK()(q, k)
    twice = layer.RotaryQK(amplitude=2.0)(q, k)
    for a, b in zip(plain, twice):
        assert (got(b) == 2.0 * got(a)).all()


@pytest.mark.parametrize("use_graph", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_resumes_from_a_checkpoint(dev, use_graph, bits, tmp_path):
    """Steps after a restored checkpoint are those of the run that wrote it,
    bit for bit: in the model that went on (whose recorded step keeps reading
    the same tensors), and in a new one."""

    class Net(model.Model):

        def __init__(self):
            super().__init__()
            self.fc = layer.Linear(33)
            self.loss = layer.MeanSquareError()

        def forward(self, x):
            return self.fc(x)

        def train_one_batch(self, x, y):
            out = self.forward(x)
            loss = self.loss(out, y)
            self.optimizer(loss)
            return out, loss

    x, y = put(dev, normal(1, 8, 20), "float16"), put(dev, normal(2, 8, 33),
                                                      "float16")
    x.requires_grad = y.requires_grad = False

    def fresh():
        m = Net()
        m.compile([x], is_train=True, use_graph=use_graph, sequential=False)
        for i, p in enumerate(p for _, p in sorted(m.get_params().items())):
            p.copy_from_numpy((normal(5 + i, *p.shape) * 0.3).numpy()
                              .astype(np.float16))
        o = opt.AdamW(lr=0.01, state_bits=bits, seed=3)
        m.set_optimizer(o)
        return m, o

    def end(m, o):
        tables = [getattr(o, n) for n in o.state_names] + [o.masters]
        return [tensor.to_numpy(p) for _, p in sorted(m.get_params().items())
                ] + [tensor.to_numpy(t) for table in tables
                     for _, t in sorted(table.items())]

    files = checkpoint.CheckpointManager(str(tmp_path))
    m, o = fresh()
    for _ in range(3):
        m(x, y)
    files.save(m, 3, o)
    for _ in range(3):
        m(x, y)
    want = end(m, o)
    assert len(want) == 2 * (2 + (2 if bits == 32 else 4))
    # (a device holds one recorded step, whatever the optimizer: the model
    # that goes on first, as compiling another replaces its step)
    for make in (lambda: (m, o), fresh):
        again = make()
        assert files.restore(*again)["step"] == 3
        for _ in range(3):
            again[0](x, y)
        for a, b in zip(want, end(*again)):
            assert a.dtype == b.dtype and (a == b).all()


def _ranks_step(rank, world, holder, bits, use_graph):
    """Parameters of test_dist's perceptron after four AdamW steps, on a part
    of its samples (or alone on all of them)."""
    dev = device.get_default_device()
    # epsilon of the gradients' size: a step then moves with a gradient
    # smoothly, and sums in another order stay small
    o = opt.AdamW(lr=0.01, epsilon=0.1, state_bits=bits)
    if world > 1:
        o = opt.DistOpt(o, nccl_id=holder, local_rank=rank, world_size=world)
    x, y = test_dist._data()
    n = len(x) // world
    x, y = (tensor.Tensor(device=dev, data=v[rank * n:(rank + 1) * n])
            for v in (x, y))
    m = test_dist._make_model()
    m.set_optimizer(o)
    m.compile([x], is_train=True, use_graph=use_graph, sequential=True)
    test_dist._init(m)
    for _ in range(4):
        m(x, y, "plain", None)
    return {k: tensor.to_numpy(v) for k, v in m.get_params().items()}


@pytest.mark.parametrize("bits,use_graph", [(32, False), (8, False),
                                            (8, True)])
def test_adamw_two_ranks(cpu_dev, bits, use_graph):
    """Ranks stay equal to the bit, also where states are rounded at random
    (the same bits for the same place), and 32-bit states give what one
    process gives on all samples: gradients are sums of 16 terms below 8, off
    by 16 2^-24 8 < 1e-5, a step moves by lr / epsilon = 0.1 of that for each
    moment, four steps by less than 1e-5 in all."""
    res = test_dist._spawn(_ranks_step, args=(bits, use_graph))
    for k, v in res[0].items():
        assert (v == res[1][k]).all()
    if bits == 32:
        for k, v in _ranks_step(0, 1, None, bits, use_graph).items():
            assert np.abs(v - res[0][k]).max() < 1e-5


def test_blocks_and_their_storage_are_recognised(cpu_dev):
    """The native list of an optimizer's blocks tells every change of one."""
    cores = [put(cpu_dev, normal(i, 5)).data for i in range(3)]
    blocks = [c._block for c in cores]
    stored = _rt.storages(blocks + [None])
    assert stored[3] is None
    assert all(s is c._storage() for s, c in zip(stored, cores))
    held = _rt.Holding(blocks)
    assert held.same(list(blocks))
    assert not held.same(blocks[:2]) and not held.same(blocks + blocks[:1])
    assert not held.same([blocks[1], blocks[0], blocks[2]])
    assert not held.same([None] * 3)
    # another tensor in the block's place, the old one back, none
    was = blocks[1].data
    blocks[1].data = was.clone()
    assert not held.same(blocks)
    blocks[1].data = was
    assert held.same(blocks)
    blocks[1].free_data()
    assert not held.same(blocks) and _rt.storages(blocks)[1] is None
    # the blocks live as long as they are held
    alone = _rt.Holding([cpu_dev.NewBlock(8)])
    gc.collect()
    assert not alone.same(blocks[:1])
    with pytest.raises((RuntimeError, TypeError)):
        _rt.Holding([1])
    with pytest.raises((RuntimeError, TypeError)):
        _rt.storages(["block"])


def test_adamw_gradient_that_was_never_written(dev):
    """Allocated on first use, as by every operator."""
    for bits in (32, 8):
        o, p = opt.AdamW(lr=0.1, weight_decay=0.0, state_bits=bits), put(
            dev, normal(1, 300))
        g = tensor.Tensor((300,), dev)
        assert g.data._block.data is None
        o.apply_many([(p, g)])
        assert g.data._block.data is not None
