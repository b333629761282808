"""Timing cases of the operators that a decoder is fine-tuned with: rotary
positions of queries and keys (with the norm of every head in the same pass),
losses over the log-probabilities of given tokens (token log-probabilities,
the paired preference loss, the clipped policy loss), and the AdamW step over
many tensors with states in 32 or in 8 bits.

``run`` computes a case either in its plain form -- elementary torch
operations -- or, with ``own`` set, through ``singa_amd``'s operators.

Formulas
  rotary   f_i = base^(-2i/R) for pair i of the first R channels, rescaled for
           long contexts; x' = x / sqrt(mean(x^2) + eps) * scale over the head
           (where it is normed), then pair i turns by the angle position * f_i.
  losses   lp = x[label] - log sum exp(x); a label outside the vocabulary is
           ignored.  preference: -mean over pairs of
           (1-s) log sigmoid(z) + s log sigmoid(-z), z = beta * (chosen -
           rejected) of sum(lp - reference).  policy: sum of w * (-min(r A,
           clip(r) A) + kl * (exp(d) - d - 1)) / sum of w with r = exp(lp - old)
           and d = reference - lp.
  AdamW    m = b1 m + (1-b1) g, v = b2 v + (1-b2) g^2,
           p = p - lr wd p - lr (m / (1-b1^t)) / (sqrt(v / (1-b2^t)) + eps).
           8 bits: m and sqrt(v) are kept in e4m3, a float scale for each 256
           values (their largest becomes 448), rounded stochastically with
           Philox4x32-10 bits: counter (element / 4, step), key seed; the word
           of an element gives its low 16 bits to m and its high 16 to sqrt(v).
"""
import math

import numpy as np
import torch

own = False

_DTYPES = {"float32": torch.float32, "float16": torch.float16,
           "bfloat16": torch.bfloat16}
_BYTES = {"float32": 4, "float16": 2, "bfloat16": 2}
_BLOCK = 256                  # values that share the scale of an 8-bit state
_LR, _B1, _B2, _EPS, _WD = (float(np.float32(v)) for v in
                            (2e-5, 0.9, 0.999, 1e-8, 0.01))
_SEED, _STEP = 1234, 100      # of the stochastic rounding; steps done before


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one new token for each of 16 sequences of a server, far positions
        # with the long-context ramp: latency alone counts
        dict(name="rotary decode", kind="rotary", batch=16, seq=1, heads=32,
             kv_heads=8, dim=128, rot=128, layout="half", scaling="ramp",
             norm=True, far=True, backward=False, dtype="bfloat16"),
        # a training step's queries and keys of one decoder layer, grouped heads
        dict(name="rotary train 2x4096", kind="rotary", batch=2, seq=4096,
             heads=32, kv_heads=8, dim=128, rot=128, layout="half",
             scaling="none", norm=True, far=False, backward=True,
             dtype="bfloat16"),
        # BERT-base's heads (12 of 64, sequences of 256, batch 32) with rotary
        # positions on half of each head, no norm
        dict(name="rotary train bert heads", kind="rotary", batch=32, seq=256,
             heads=12, kv_heads=12, dim=64, rot=32, layout="interleaved",
             scaling="base", norm=False, far=False, backward=True,
             dtype="float16"),
        # float32 fine-tuning of a head width that is no power of two, ragged
        # length, packed sequences whose positions start again
        dict(name="rotary train odd", kind="rotary", batch=3, seq=1021,
             heads=10, kv_heads=5, dim=80, rot=40, layout="interleaved",
             scaling="linear", norm=True, far=True, backward=True,
             dtype="float32"),
        # scoring the next token of 8 sequences over a large vocabulary: few
        # rows, so the vocabulary axis itself has to be split
        dict(name="log-prob few rows", kind="logprob", rows=8, vocab=131071,
             backward=False, dtype="float32"),
        # a character-sized model's preference pair: the smallest call
        dict(name="preference small", kind="preference", pairs=1, seq=33,
             vocab=997, backward=True, dtype="float32"),
        # preference tuning over the vocabulary of GPT-2 (odd, so rows start
        # unaligned): four pairs of 1024 tokens
        dict(name="preference 4x1024 gpt", kind="preference", pairs=4,
             seq=1024, vocab=50257, backward=True, dtype="bfloat16"),
        # policy optimisation over BERT's vocabulary, a third of the tokens
        # masked, with the divergence from a frozen model
        dict(name="policy 4096 bert", kind="policy", rows=4096, vocab=30522,
             kl=0.05, backward=True, dtype="float16"),
        # a small perceptron's eight tensors: launches and dispatch
        dict(name="adamw small", kind="adamw", vocab=129, width=64, ffn=172,
             layers=1, bits=32, dtype="float32"),
        # a 140 M parameter decoder in float32
        dict(name="adamw 32 decoder", kind="adamw", vocab=50257, width=1024,
             ffn=2816, layers=8, bits=32, dtype="float32"),
        # the same in bfloat16 with float32 masters and 8-bit states
        dict(name="adamw 8 decoder bf16", kind="adamw", vocab=50257,
             width=1024, ffn=2816, layers=8, bits=8, dtype="bfloat16"),
        # float32 weights of odd sizes with 8-bit states
        dict(name="adamw 8 odd", kind="adamw", vocab=10007, width=500,
             ffn=1333, layers=4, bits=8, dtype="float32"),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo),
                                                          math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rotary", "logprob", "preference", "policy", "adamw"])
    dtype = rng.choice(sorted(_DTYPES))
    if kind == "rotary":
        dim = rng.choice([32, 48, 64, 80, 96, 128, 192, 256])
        kv = rng.randint(1, 16)
        group = rng.choice([1, 1, 2, 4, 5, 8])
        seq = 1 if rng.random() < 0.25 else _log_uniform(rng, 2, 8192)
        room = 1 << 26            # values of the queries
        batch = _log_uniform(rng, 1, max(1, min(
            64, room // (seq * kv * group * dim))))
        return dict(kind=kind, batch=batch, seq=seq, heads=kv * group,
                    kv_heads=kv, dim=dim,
                    rot=rng.choice([dim, dim, dim // 2, 2 * (dim // 8)]),
                    layout=rng.choice(["half", "interleaved"]),
                    scaling=rng.choice(["none", "linear", "base", "ramp"]),
                    norm=rng.random() < 0.6, far=rng.random() < 0.5,
                    backward=seq > 1 and rng.random() < 0.8, dtype=dtype)
    if kind == "adamw":
        width = 4 * _log_uniform(rng, 8, 256) + 4 * rng.randint(0, 1)
        return dict(kind=kind, vocab=_log_uniform(rng, 50, 50257),
                    width=width, ffn=_log_uniform(rng, 40, 2816),
                    layers=rng.randint(1, 7), bits=rng.choice([8, 32]),
                    dtype=dtype)
    vocab = _log_uniform(rng, 100, 160000)
    most = 350_000_000 // (vocab * (2 if dtype == "float32" else 1))
    if kind == "preference":
        pairs = _log_uniform(rng, 1, 8)
        return dict(kind=kind, pairs=pairs,
                    seq=_log_uniform(rng, 1, max(2, min(2048, most // (2 * pairs)))),
                    vocab=vocab, backward=True, dtype=dtype)
    case = dict(kind=kind, rows=_log_uniform(rng, 1, max(2, min(16384, most))),
                vocab=vocab, backward=rng.random() < 0.75, dtype=dtype)
    if kind == "policy":
        case.update(kl=rng.choice([0.0, 0.05]), backward=True)
    return case


def _weights(case):
    """Shapes of a decoder's parameters: embedding, then for each layer two
    norms, four projections (a quarter of the key and value heads), the two
    head norms and the three matrices of a gated feed-forward block."""
    w, f = case["width"], case["ffn"]
    layer = [(w,), (w, w), (w, w // 4), (w, w // 4), (w, w), (64,), (64,),
             (w,), (w, f), (w, f), (f, w)]
    return [(case["vocab"], w)] + layer * case["layers"] + [(w,)]


def work(case):
    size, kind = _BYTES[case["dtype"]], case["kind"]
    if kind == "rotary":
        n = case["batch"] * case["seq"] * case["dim"] * (case["heads"] +
                                                         case["kv_heads"])
        small = 4 * case["batch"] * case["seq"]
        # forward: x in, y out; backward: dy (and x, where it was normed) in,
        # dx out
        if not case["backward"]:
            return {"bytes": 2 * n * size + small, "flops": 8 * n}
        return {"bytes": (5 if case["norm"] else 4) * n * size + 2 * small,
                "flops": 24 * n}
    if kind == "adamw":
        n = sum(math.prod(s) for s in _weights(case))
        state = 8 if case["bits"] == 32 else 2 + 8 / _BLOCK
        master = 0 if size == 4 else 8       # read and written
        # gradient in; parameter out (and in, where it is its own master)
        here = size + (size if master else 2 * size) + master + 2 * state
        return {"bytes": n * here, "flops": 16 * n}
    rows = case["rows"] if "rows" in case else 2 * case["pairs"] * case["seq"]
    n = rows * case["vocab"]
    # logits in; backward: logits in again, since a loss over all tokens is
    # known only after the last of them, and their gradient out
    return {"bytes": n * size * (3 if case["backward"] else 1) + 16 * rows,
            "flops": n * (8 if case["backward"] else 4)}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def prepare(case, seed):
    g = torch.Generator(device=_device())
    g.manual_seed(int(seed))
    make = {"rotary": _prepare_rotary, "adamw": _prepare_adamw}.get(
        case["kind"], _prepare_loss)
    return make(case, g, _DTYPES[case["dtype"]])


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=g.device)


def _wrap(x):
    """A singa_amd tensor over the memory of a torch tensor."""
    from singa_amd import device, tensor
    from singa_amd.core import dtypes
    dev = device.create_cuda_gpu_on(0) if x.is_cuda else \
        device.get_default_device()
    t = tensor.Tensor(tuple(x.shape), dev, dtypes.from_torch(x.dtype),
                      requires_grad=x.is_floating_point(),
                      stores_grad=x.is_floating_point())
    t.data.block().data = x.reshape(-1)
    return t


def _scaling(case):
    return {"none": None, "linear": ("linear", 4.0), "base": ("base", 4.0),
            "ramp": ("ramp", 16.0, 8192)}[case["scaling"]]


def _prepare_rotary(case, g, dt):
    B, S, H, K, D = (case[k] for k in ("batch", "seq", "heads", "kv_heads",
                                       "dim"))
    s = dict(case=case)
    for name, heads in (("q", H), ("k", K)):
        s[name] = (_normal(g, B, S, heads, D) * 1.5).to(dt)
        s["d" + name] = _normal(g, B, S, heads, D).to(dt)
        s[name + "_scale"] = (1 + 0.2 * _normal(g, D)).to(dt)
    if case["far"]:
        # every sequence is somewhere in a context of up to a million tokens
        start = torch.randint(0, 1 << 20, (B, 1), generator=g, device=g.device)
        at = torch.arange(S, device=g.device)
        # and begins again in its middle
        s["positions"] = (torch.where(at < (S + 1) // 2, at + start,
                                      at - (S + 1) // 2)).to(torch.int32)
    else:
        s["positions"] = torch.arange(S, device=g.device, dtype=torch.int32)
    if own:
        from singa_amd import autograd, singa_wrap
        autograd.training = True
        s["handle"] = singa_wrap.RotaryHandle(
            D, case["rot"], base=10000.0, layout=case["layout"],
            scaling=_scaling(case))
        for name in ("q", "k", "dq", "dk", "q_scale", "k_scale", "positions"):
            s[name] = _wrap(s[name])
    return s


def _prepare_loss(case, g, dt):
    V = case["vocab"]
    if case["kind"] == "preference":
        shape = (2 * case["pairs"], case["seq"])
    else:
        shape = (case["rows"],)
    n = math.prod(shape)
    x = torch.empty(n, V, dtype=dt, device=g.device)
    labels = torch.randint(0, V, (n,), generator=g, device=g.device)
    some = max(1, (1 << 26) // V)
    lp = torch.empty(n, device=g.device)
    for a in range(0, n, some):
        part = 2.0 * _normal(g, min(some, n - a), V)
        rows = torch.arange(part.shape[0], device=g.device)
        part[rows, labels[a:a + some]] += 6.0    # mostly what the model expects
        part = part.to(dt)
        x[a:a + some] = part
        part = part.float()
        lp[a:a + some] = part[rows, labels[a:a + some]] - \
            torch.logsumexp(part, -1)
    # prompts and padding are ignored
    skip = torch.rand(n, generator=g, device=g.device) < 0.3
    if case["kind"] != "logprob" and n > 2:
        labels = torch.where(skip, -1, labels)
    s = dict(case=case, x=x.view(*shape, V), t=labels.view(shape).to(torch.int32),
             reference=(lp + 0.05 * _normal(g, n)).view(shape),
             old=(lp + 0.15 * _normal(g, n)).view(shape),
             advantages=_normal(g, n).view(shape),
             weights=(0.5 + torch.rand(n, generator=g,
                                       device=g.device)).view(shape),
             dy=_normal(g, n).view(shape))
    if own:
        from singa_amd import autograd
        autograd.training = True
        for name in ("x", "t", "reference", "old", "advantages", "weights",
                     "dy"):
            s[name] = _wrap(s[name])
    return s


def _prepare_adamw(case, g, dt):
    shapes = _weights(case)
    sizes = np.array([math.prod(s) for s in shapes])
    room = -(-sizes // _BLOCK) * _BLOCK      # every tensor starts a block
    starts = np.concatenate([[0], np.cumsum(room)])
    n = int(starts[-1])
    # zero between the tensors, where nothing reads or writes
    where = torch.zeros(n, dtype=torch.bool, device=g.device)
    for a, k in zip(starts, sizes):
        where[int(a):int(a) + int(k)] = True
    grad = (0.01 * _normal(g, n) * where).to(dt)
    scale = torch.exp(_normal(g, n // _BLOCK, 1))    # blocks differ in size
    m = (0.004 * _normal(g, n // _BLOCK, _BLOCK) * scale).view(-1) * where
    v = ((0.01 * _normal(g, n // _BLOCK, _BLOCK) * scale) ** 2 + 1e-8).view(-1) \
        * where
    master = 0.02 * _normal(g, n) * where
    s = dict(case=case, n=n, g=grad, step=_STEP, p=master.to(dt))
    if dt != torch.float32:
        s["master"] = master
    if case["bits"] == 32:
        s["m"], s["v"] = m, v
    else:
        at = torch.from_numpy(np.concatenate(
            [np.arange(r // _BLOCK) for r in room]) * (_BLOCK // 4))
        # of each 4 values: their number within their tensor
        s["group"] = (at.to(g.device)[:, None] +
                      torch.arange(_BLOCK // 4, device=g.device)).view(-1)
        for name, x in (("m", m), ("r", torch.sqrt(v))):
            x = x.view(-1, _BLOCK)
            s[name + "_scale"] = x.abs().amax(1) / 448.0
            s[name] = (x / s[name + "_scale"].clamp_min(1e-30)[:, None]).clamp(
                -448, 448).to(torch.float8_e4m3fn).view(-1)
    if own:
        s.update(_own_adamw(case, s, shapes, starts))
    return s


def _own_adamw(case, s, shapes, starts):
    from singa_amd import opt
    o = opt.AdamW(lr=_LR, beta_1=_B1, beta_2=_B2, epsilon=_EPS,
                  weight_decay=_WD, state_bits=case["bits"], seed=_SEED)
    pairs, states = [], {"step_counter": float(_STEP)}

    def keep(table, name, x):
        states.setdefault(table, {})[name] = _wrap(x)

    for i, shape in enumerate(shapes):
        a, k = int(starts[i]), math.prod(shape)
        b, e = a // _BLOCK, int(starts[i + 1])
        p, g = _wrap(s["p"][a:a + k].view(shape)), \
            _wrap(s["g"][a:a + k].view(shape))
        p.name = name = "weight%d" % i
        pairs.append((p, g))
        if "master" in s:
            keep("masters", name, s["master"][a:a + k].view(shape))
        if case["bits"] == 32:
            keep("m", name, s["m"][a:a + k].view(shape))
            keep("v", name, s["v"][a:a + k].view(shape))
        else:
            for table in ("m", "r"):
                keep(table, name, s[table][a:e].view(torch.int32))
                keep(table + "_scale", name, s[table + "_scale"][b:e // _BLOCK])
    o.set_states(states)
    return dict(opt=o, pairs=pairs)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    kind = s["case"]["kind"]
    if kind == "rotary":
        return _run_rotary(s) if own else _plain_rotary(s)
    if kind == "adamw":
        return _run_adamw(s) if own else _plain_adamw(s)
    return _run_loss(s) if own else _plain_loss(s)


def _out(*named):
    """Results of the framework as torch tensors (no copy)."""
    return {k: t.view() for k, t in named}


def _run_rotary(s):
    from singa_amd import autograd
    case = s["case"]
    scales = (s["q_scale"], s["k_scale"]) if case["norm"] else ()
    op = autograd.Rotary(s["handle"], s["positions"], norm=case["norm"],
                         eps=1e-6)
    q, k = op(s["q"], s["k"], *scales)
    out = _out(("q", q.data), ("k", k.data))
    if case["backward"]:
        grads = op.backward(s["dq"].data, s["dk"].data)
        out.update(_out(*zip(("dq", "dk", "dq_scale", "dk_scale"), grads)))
    return out


def _run_loss(s):
    from singa_amd import autograd
    case = s["case"]
    if case["kind"] == "logprob":
        op = autograd.TokenLogProb(s["t"])
    elif case["kind"] == "preference":
        op = autograd.PreferenceLoss(s["t"], s["reference"], beta=0.1,
                                     smoothing=0.05)
    else:
        op = autograd.PolicyLoss(s["t"], s["old"], s["advantages"],
                                 weights=s["weights"], reference=s["reference"],
                                 clip=(0.2, 0.28), kl=case["kl"])
    y = op(s["x"])[0]
    out = _out(("y", y.data))
    if case["backward"]:
        dy = s["dy"].data if case["kind"] == "logprob" else 1.0
        out.update(_out(("dx", op.backward(dy))))
    return out


def _run_adamw(s):
    s["opt"].apply_many(s["pairs"])
    s["opt"].step()
    return _state(s)


def _state(s):
    return {k: s[k] for k in ("p", "master", "m", "v", "r", "m_scale",
                              "r_scale") if k in s}


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _frequencies(case):
    """Angle of one position for each pair, float64, and the amplitude."""
    R, scaling = case["rot"], _scaling(case)
    i = torch.arange(0, R, 2, dtype=torch.float64, device=_device())
    base, amplitude = 10000.0, 1.0
    if scaling and scaling[0] == "base":
        base = base * scaling[1] ** (R / max(1, R - 2))
    f = torch.exp(-i / R * math.log(base))
    if scaling and scaling[0] == "linear":
        f = f / scaling[1]
    if scaling and scaling[0] == "ramp":
        _, factor, length = scaling
        turns = length * f / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        f = f * (keep + (1 - keep) / factor)
        amplitude = 0.1 * math.log(factor) + 1.0
    return f, amplitude


def _turn(case, x, cos, sin):
    R = case["rot"]
    r = x[..., :R]
    if case["layout"] == "half":
        a, b = r[..., :R // 2], r[..., R // 2:]
        r = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([r, x[..., R:]], -1)


def _plain_rotary(s):
    case, eps = s["case"], 1e-6
    dt = _DTYPES[case["dtype"]]
    f, amplitude = _frequencies(case)
    angle = s["positions"].double().unsqueeze(-1) * f
    cos = (amplitude * torch.cos(angle)).float().unsqueeze(-2)   # (.., S, 1, R/2)
    sin = (amplitude * torch.sin(angle)).float().unsqueeze(-2)
    out = {}

    def one(name):
        x, w = s[name].float(), s[name + "_scale"].float()
        rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
        normed = x * rstd * w if case["norm"] else x
        out[name] = _turn(case, normed, cos, sin).to(dt)
        if not case["backward"]:
            return
        g = _turn(case, s["d" + name].float(), cos, -sin)
        if not case["norm"]:
            out["d" + name] = g.to(dt)
            return
        xhat = x * rstd
        out["d" + name + "_scale"] = (g * xhat).double().sum((0, 1, 2)).to(dt)
        g = g * w
        out["d" + name] = (rstd * (g - xhat * (g * xhat).mean(
            -1, keepdim=True))).to(dt)

    one("q")
    one("k")
    return out


def _log_sigmoid(z):
    return -(torch.clamp(-z, min=0) + torch.log1p(torch.exp(-z.abs())))


def _token_loss(s, lp, used):
    """The loss of these log-probabilities and its derivative for each."""
    case, zero = s["case"], torch.zeros_like(lp)
    if case["kind"] == "preference":
        P, beta, smooth = case["pairs"], 0.1, 0.05
        ratio = torch.where(used, lp - s["reference"], zero).sum(-1)
        z = beta * (ratio[:P] - ratio[P:])
        loss = -((1 - smooth) * _log_sigmoid(z) +
                 smooth * _log_sigmoid(-z)).mean()
        dz = (smooth * torch.sigmoid(z) -
              (1 - smooth) * torch.sigmoid(-z)) * beta / P
        c = torch.cat([dz, -dz]).unsqueeze(-1).expand_as(lp)
        return loss, torch.where(used, c, zero)
    ratio = torch.exp(lp - s["old"])
    A, w = s["advantages"], torch.where(used, s["weights"], zero)
    total = w.sum()
    total = torch.where(total > 0, total, torch.ones_like(total))
    plain, cut = ratio * A, ratio.clamp(1 - 0.2, 1 + 0.28) * A
    d = s["reference"] - lp
    each = -torch.minimum(plain, cut) + case["kl"] * (torch.exp(d) - d - 1)
    c = torch.where(plain <= cut, -plain, zero) + \
        case["kl"] * (1 - torch.exp(d))
    return torch.where(used, w * each, zero).sum() / total, \
        torch.where(used, w * c, zero) / total


def _plain_loss(s):
    case, V = s["case"], s["case"]["vocab"]
    x = s["x"].float()
    used = (s["t"] >= 0) & (s["t"] < V)
    label = torch.where(used, s["t"], 0).long().unsqueeze(-1)
    top = x.amax(-1, keepdim=True)
    x = x - top
    norm = torch.log(torch.exp(x).sum(-1, keepdim=True))
    # from here on a value for each token, and sums over all of them
    lp = (x.gather(-1, label).double() - norm.double()).squeeze(-1)
    lp = torch.where(used, lp, 0.0)
    if case["kind"] == "logprob":
        y, c = lp, torch.where(used, s["dy"].double(), 0.0)
    else:
        s64 = dict(s, **{k: s[k].double() for k in
                         ("reference", "old", "advantages", "weights")})
        y, c = _token_loss(s64, lp, used)
        y = y.reshape(1)
    out = {"y": y.float()}
    if case["backward"]:
        c = c.float().unsqueeze(-1)
        dx = -c * torch.exp(x - norm)
        out["dx"] = dx.scatter_add_(-1, label, c).to(s["x"].dtype)
    return out


_LOW = 0xFFFFFFFF


def _random_words(group, step):
    """The four words of Philox4x32-10 for each counter (group, step)."""
    c = [group & _LOW, group >> 32, torch.full_like(group, step),
         torch.zeros_like(group)]
    k = [_SEED & _LOW, _SEED >> 32]
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [((b >> 32) & _LOW) ^ c[1] ^ k[0], b & _LOW,
             ((a >> 32) & _LOW) ^ c[3] ^ k[1], a & _LOW]
        k = [(k[0] + 0x9E3779B9) & _LOW, (k[1] + 0xBB67AE85) & _LOW]
    return torch.stack(c, -1).view(-1)


def _to_e4m3(x, noise, keep):
    """Codes and block scales of x; noise in [0, 1) decides the rounding."""
    top = x.view(-1, _BLOCK).abs().amax(1, keepdim=True)
    inv = torch.where(top > 0, 448.0 / top, torch.zeros_like(top))
    t = (x.view(-1, _BLOCK) * inv).view(-1)
    size = t.abs()
    # the binade of each value as a power of two: its exponent bits alone
    unit = (size.clamp_min(2.0 ** -6).view(torch.int32) & 0x7F800000).view(
        torch.float32) * 0.125
    size = torch.floor(size / unit + noise) * unit
    if keep:      # what is divided by does not round to zero
        size = torch.where(t > 0, size.clamp_min(2.0 ** -9), size)
    size = size.clamp_max(448.0)
    return torch.copysign(size, t).to(torch.float8_e4m3fn), (top / 448.0).view(-1)


def _plain_adamw(s):
    t = s["step"] + 1
    g, p = s["g"].float(), s.get("master", s["p"])
    if s["case"]["bits"] == 32:
        m, v = s["m"], s["v"]
    else:
        m = (s["m"].float().view(-1, _BLOCK) * s["m_scale"][:, None]).view(-1)
        r = (s["r"].float().view(-1, _BLOCK) * s["r_scale"][:, None]).view(-1)
        v = r * r
    keep1, keep2 = (float(np.float32(1) - np.float32(b)) for b in (_B1, _B2))
    m = _B1 * m + keep1 * g
    v = _B2 * v + keep2 * (g * g)
    c1, c2 = (1 / (1 - b ** t) for b in (_B1, _B2))
    p = p - float(np.float32(_LR) * np.float32(_WD)) * p
    p = p - _LR * ((m * c1) / (torch.sqrt(v * c2) + _EPS))
    if "master" in s:
        s["master"] = p
    s["p"] = p.to(s["g"].dtype)
    if s["case"]["bits"] == 32:
        s["m"], s["v"] = m, v
    else:
        words = _random_words(s["group"], s["step"])
        s["m"], s["m_scale"] = _to_e4m3(m, (words & 0xFFFF).float() / 65536,
                                        False)
        s["r"], s["r_scale"] = _to_e4m3(torch.sqrt(v),
                                        (words >> 16).float() / 65536, True)
    s["step"] = t
    return _state(s)


# ---------------------------------------------------------------------------
# 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["kind"] == "rotary":
        return _exact_rotary(case, s)
    return _exact_adamw(case, s) if case["kind"] == "adamw" else \
        _exact_loss(case, s)


def _exact_rotary(case, s):
    R, D, scaling = case["rot"], case["dim"], _scaling(case)
    base, f, amplitude = 10000.0, [], 1.0
    if scaling and scaling[0] == "base":
        base *= scaling[1] ** (R / max(1, R - 2))
    for i in range(R // 2):
        w = base ** (-2.0 * i / R)
        if scaling and scaling[0] == "linear":
            w /= scaling[1]
        if scaling and scaling[0] == "ramp":
            share = (scaling[2] * w / (2 * math.pi) - 1.0) / 31.0
            share = min(1.0, max(0.0, share))
            w = share * w + (1.0 - share) * w / scaling[1]
            amplitude = 1.0 + 0.1 * math.log(scaling[1])
        f.append(w)
    f = torch.tensor(f, dtype=torch.float64, device=_device())
    # the rotation as a product with a complex number of that amplitude
    turn = torch.polar(torch.full((), amplitude, dtype=torch.float64,
                                  device=f.device),
                       s["positions"].double()[..., None, None] * f)
    first = torch.arange(R // 2, device=f.device) * \
        (1 if case["layout"] == "half" else 2)
    second = first + (R // 2 if case["layout"] == "half" else 1)

    def turned(x, by):
        z = torch.complex(x[..., first], x[..., second]) * by
        y = x.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return y

    out = {}
    for name in ("q", "k"):
        x, w = s[name].double(), s[name + "_scale"].double()
        length = torch.sqrt(x.square().sum(-1, keepdim=True) / D + 1e-6)
        unit = x / length
        out[name] = turned(unit * w if case["norm"] else x, turn)
        if case["backward"]:
            g = turned(s["d" + name].double(), turn.conj())
            if case["norm"]:
                out["d%s_scale" % name] = (g * unit).flatten(0, 2).sum(0)
                g = g * w
                g = (g - unit * (g * unit).sum(-1, keepdim=True) / D) / length
            out["d" + name] = g
    return out


def _exact_loss(case, s):
    V = case["vocab"]
    t = s["t"].reshape(-1).long()
    x = s["x"].reshape(-1, V)
    used = (t >= 0) & (t < V)
    rows = torch.arange(len(t), device=x.device)
    some = max(1, (1 << 27) // V)
    pieces = [(a, x[a:a + some].double()) for a in range(0, len(t), some)]
    total = torch.cat([torch.logsumexp(p, -1) for _, p in pieces])
    lp = x[rows, t.clamp(0, V - 1)].double() - total
    lp = torch.where(used, lp, 0.0).requires_grad_()
    if case["kind"] == "logprob":
        y, c = lp, torch.where(used, s["dy"].double(), 0.0)
    else:
        each = {k: s[k].double().reshape(-1) for k in
                ("reference", "old", "advantages", "weights")}
        d = lp - each["reference"]
        if case["kind"] == "preference":
            side = torch.where(used, d, 0.0).view(2, case["pairs"], -1).sum(-1)
            z = 0.1 * (side[0] - side[1])
            y = (0.95 * torch.nn.functional.softplus(-z) +
                 0.05 * torch.nn.functional.softplus(z)).mean()
        else:
            r, A = torch.exp(lp - each["old"]), each["advantages"]
            gain = torch.where(A >= 0, r.clamp(max=1.28), r.clamp(min=0.8)) * A
            w = torch.where(used, each["weights"], 0.0)
            y = (w * (case["kl"] * (torch.expm1(-d) + d) - gain)).sum()
            y = y / w.sum() if float(w.sum()) > 0 else y
        c, = torch.autograd.grad(y, lp)      # of the scalar loss only
        y = y.reshape(1)
    out = {"y": y.detach().view(s["t"].shape if case["kind"] == "logprob"
                                else (1,))}
    if case["backward"]:
        dx = torch.cat([-c[a:a + len(p), None] * torch.exp(
            p - total[a:a + len(p), None]) for a, p in pieces])
        dx[rows, t.clamp(0, V - 1)] += torch.where(used, c, 0.0)
        out["dx"] = dx.view(s["x"].shape)
    return out


def _exact_adamw(case, s):
    n = s["n"]
    g = s["g"].double()
    p = s.get("master", s["p"]).double()

    def blocks(x, scale):
        return (x.double().view(-1, _BLOCK) * scale.double()[:, None]).view(-1)

    if case["bits"] == 32:
        m, v = s["m"].double(), s["v"].double()
    else:
        m = blocks(s["m"], s["m_scale"])
        v = blocks(s["r"], s["r_scale"]).square()
    m = m + (1 - _B1) * (g - m)
    v = v + (1 - _B2) * (g * g - v)
    t = _STEP + 1
    p = (1 - _LR * _WD) * p - _LR * (m / -math.expm1(t * math.log(_B1))) / (
        torch.sqrt(v / -math.expm1(t * math.log(_B2))) + _EPS)
    out = {"p": p}
    if "master" in s:
        out["master"] = p
    if case["bits"] == 32:
        out.update(m=m, v=v)
        return out
    # the random words on the host, in unsigned 64-bit arithmetic
    group = s["group"].cpu().numpy().astype(np.uint64)
    c = [group & np.uint64(_LOW), group >> np.uint64(32),
         np.full(len(group), _STEP, np.uint64), np.zeros(len(group), np.uint64)]
    key = [_SEED & _LOW, _SEED >> 32]
    half, low = np.uint64(32), np.uint64(_LOW)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> half) ^ c[1] ^ np.uint64(key[0]), b & low,
             (a >> half) ^ c[3] ^ np.uint64(key[1]), a & low]
        key = [(key[0] + 0x9E3779B9) & _LOW, (key[1] + 0xBB67AE85) & _LOW]
    words = torch.from_numpy(np.stack(c, 1).reshape(-1).astype(np.int64)).to(
        g.device)
    for name, x, bits in (("m", m, words % 65536),
                          ("r", torch.sqrt(v), words // 65536)):
        x = x.view(-1, _BLOCK)
        top = x.abs().max(1, keepdim=True).values
        t = (x * torch.where(top > 0, 448.0 / top, 0.0)).view(n)
        power = (torch.frexp(t.abs()).exponent - 1).clamp(min=-6) - 3
        steps = torch.floor(torch.ldexp(t.abs(), -power) +
                            bits.double() / 65536.0)
        if name == "r":
            steps = torch.where((t > 0) & (steps < 1), 1.0, steps)
        out[name] = (torch.sign(t) * torch.ldexp(steps, power)).clamp(-448, 448)
        out[name + "_scale"] = top.view(-1) / 448.0
    return out
