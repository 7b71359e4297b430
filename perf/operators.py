"""Timed workloads of the decoder's attention operators: rotary positions, attention with its gradient, and attention of
new tokens over a cache.

A case names the sizes (batch B, queries S, keys T, query heads H, key/value heads G, head size d), the element type and what is
asked: "rotary" turns q and k by their positions, "attend" is softmax attention; with ``train`` the pass returns the gradients of
its inputs too.  Tensors are in GPU memory before a pass, q, k and v as views of one packed projection or of a cache, as in a
decoder.  ``run`` computes the operators from elementary operations in 32 bits; with ``own`` it calls the package.

The keys of sequence b are the first lengths[b] of T; query i stands at position starts[b] + i and sees the keys up to its
own position.  A query that sees no key gives zeros.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}

DEFAULTS = dict(
    train=False,          # gradients too
    ragged=False,         # sequences of different lengths in one batch (padded, or caches filled to different marks)
    part=1.0,             # rotary: share of the head that turns
    interleaved=False,    # rotary: pairs (2i, 2i+1) instead of (i, i + R/2)
    scaling="none",       # rotary: "none", "linear", "base" or "parts" for contexts past the trained one
    far=0,                # rotary: positions start here
)
BASE, FACTOR, TRAINED = 10000.0, 8.0, 4096


def _case(name, op, B, S, T, H, G, d, dtype, **options):
    return dict(DEFAULTS, name=name, op=op, B=B, S=S, T=T, H=H, G=G, d=d, dtype=dtype, **options)


def listed():
    return [
        # one new token of each of 16 sequences that generate together: launches and host time
        _case("rotary_step_bf16", "rotary", 16, 1, 1, 16, 16, 64, "bf16", ragged=True, far=700),
        # the benchmark's decoder: a training step's turn of q and k
        _case("rotary_train_bf16", "rotary", 16, 1024, 1024, 16, 16, 64, "bf16", train=True),
        # a long prompt past the trained context: shared key heads, half of the head turned, pairs side by side
        _case("rotary_long_f16", "rotary", 1, 50001, 50001, 16, 4, 128, "f16", part=0.5, interleaved=True, scaling="parts",
              far=90000),
        # a unit-test sized training step: latency
        _case("train_tiny_f32", "attend", 2, 100, 100, 4, 2, 32, "f32", train=True),
        # the benchmark's decoder: 16 sequences of 1024, 16 heads of 64
        _case("train_decoder_bf16", "attend", 16, 1024, 1024, 16, 16, 64, "bf16", train=True),
        # the same model in single precision on a small batch
        _case("train_decoder_f32", "attend", 2, 1024, 1024, 16, 16, 64, "f32", train=True),
        # a padded batch of odd lengths, heads of 80, fp16
        _case("train_padded_f16", "attend", 6, 1717, 1717, 8, 2, 80, "f16", train=True, ragged=True),
        # one long sequence with shared key heads: the largest call
        _case("train_long_bf16", "attend", 1, 8192, 8192, 16, 4, 128, "bf16", train=True),
        # a prompt's next piece of odd length against what the cache holds
        _case("prefill_bf16", "attend", 2, 1003, 5003, 16, 4, 128, "bf16", ragged=True),
        # one sequence generating with a short cache: the smallest call
        _case("decode_1_bf16", "attend", 1, 1, 1024, 16, 16, 64, "bf16"),
        # 48 sequences generating together, caches filled to different marks
        _case("decode_48_bf16", "attend", 48, 1, 8192, 16, 4, 128, "bf16", ragged=True),
        # one sequence with a very long cache
        _case("decode_long_f16", "attend", 1, 1, 131071, 16, 2, 128, "f16"),
    ]


def _spread(rng: random.Random, lo: int, hi: int) -> int:
    """An integer of [lo, hi], its logarithm evenly spread."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng: random.Random):
    kind = rng.choice(("rotary", "train", "train", "prefill", "decode", "decode"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    G = rng.choice((1, 2, 4, 8))
    H = G * rng.choice((1, 2, 4, 8))
    d = rng.choice((32, 64, 64, 80, 96, 128, 128))
    B = _spread(rng, 1, 64)
    c = dict(DEFAULTS, op="attend", B=B, H=H, G=G, d=d, dtype=dtype)
    if kind == "rotary":
        c.update(op="rotary", S=max(1, min(_spread(rng, 1, 65536), 50001 * 20 * 128 // (B * (H + G) * d))),
                 train=rng.random() < 0.5, part=rng.choice((1.0, 0.5, 0.25)), interleaved=rng.random() < 0.5,
                 scaling=rng.choice(("none", "linear", "base", "parts")), far=_spread(rng, 1, 1 << 20),
                 ragged=rng.random() < 0.3)
        c["T"] = c["S"]
        return c
    # no more pairs of query and key than the largest listed case; single precision has a sixteenth of the matrix rate
    most = 16 * 8192 * 8192 // (16 if dtype == "f32" else 1)
    c["ragged"] = rng.random() < 0.5
    if kind == "train":
        S = max(1, min(_spread(rng, 16, 8192), math.isqrt(most // (B * H))))
        c.update(S=S, T=S, train=True)
    elif kind == "prefill":
        S = max(1, min(_spread(rng, 2, 4096), math.isqrt(most // (B * H))))
        c.update(S=S, T=max(S, min(S + _spread(rng, 1, 30000), most // (B * H * S), 48 * 8192 * 4 * 128 // (B * G * d))))
    else:
        c.update(S=1, T=min(_spread(rng, 16, 131071), 48 * 8192 * 4 * 128 // (B * G * d)))
    return c


def _turned(c):
    """Elements of a head that turn: even, two at least."""
    return max(2, int(c["d"] * c["part"]) // 2 * 2)


def _theta(c):
    """Angle per position of every pair, radians, and the factor on the turned values."""
    R = _turned(c)
    base, scaling = BASE, c["scaling"]
    if scaling == "base" and R > 2:
        base *= FACTOR ** (R / (R - 2))
    th = [base ** (-2 * i / R) for i in range(R // 2)]
    if scaling == "linear":
        th = [t / FACTOR for t in th]
    if scaling == "parts":
        # pairs that turn 32 times or more within the trained context stay, those that turn once or less are stretched
        keep = [min(1.0, max(0.0, (TRAINED * t / (2 * math.pi) - 1) / 31)) for t in th]
        th = [t * (s + (1 - s) / FACTOR) for t, s in zip(th, keep)]
    return th, (1 + 0.1 * math.log(FACTOR) if scaling == "parts" else 1.0)


def prepare(case, seed):
    c = case
    dt, dev = DTYPES[c["dtype"]], "cuda"
    g = torch.Generator(dev).manual_seed(seed)
    B, S, T, H, G, d = (c[n] for n in "BSTHGd")

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32).mul_(scale).to(dt)
    st = dict(case=c)
    if c["op"] == "rotary" or S == T:                   # one packed projection
        qkv = normal(B, S, H + 2 * G, d)
        st["q"], st["k"], st["v"] = qkv[:, :, :H], qkv[:, :, H:H + G], qkv[:, :, H + G:]
    else:                                               # new queries and a cache
        st["q"], st["k"], st["v"] = normal(B, S, H, d), normal(B, T, G, d), normal(B, T, G, d)
    if c["op"] == "rotary":
        start = torch.full((B, 1), c["far"], device=dev)
        if c["ragged"]:
            start = start + torch.randint(0, 4000, (B, 1), generator=g, device=dev)
        st["positions"] = (start + torch.arange(S, device=dev)).contiguous()
        if c["train"]:
            st["gq"], st["gk"] = normal(B, S, H, d), normal(B, S, G, d)
    else:
        st["lengths"] = st["starts"] = None
        if c["ragged"]:
            low = max(S, T // 2) if not c["train"] else max(1, T // 4)
            st["lengths"] = torch.randint(low, T + 1, (B,), generator=g, device=dev, dtype=torch.int32)
            if not c["train"]:                          # the queries are the last of what their cache holds
                st["starts"] = st["lengths"] - S
        if c["train"]:
            st["go"] = normal(B, S, H, d)
    if c["train"]:
        for n in ("q", "k") if c["op"] == "rotary" else ("q", "k", "v"):
            st[n].requires_grad_()
    if own and c["op"] == "rotary":
        from analog_moe_amd.rotary import Rotary
        st["rotary"] = Rotary(_turned(c), base=BASE, interleaved=c["interleaved"], scaling=c["scaling"], factor=FACTOR,
                              trained_context=TRAINED).to(dev)
    elif c["op"] == "rotary":
        st["theta"] = torch.tensor(_theta(c)[0], dtype=torch.float64, device=dev)
    return st


def run(state):
    c = state["case"]
    if own:
        return _run_rotary(state) if c["op"] == "rotary" else _run_attention(state)
    with torch.no_grad():
        return _plain_rotary(state) if c["op"] == "rotary" else _plain_attention(state)


# ------------------------------------------------------------------------------ the package
def _run_rotary(st):
    if not st["case"]["train"]:
        with torch.no_grad():
            return st["rotary"](st["q"], st["k"], positions=st["positions"])
    q, k = st["rotary"](st["q"], st["k"], positions=st["positions"])
    return (q.detach(), k.detach(), *torch.autograd.grad((q, k), (st["q"], st["k"]), (st["gq"], st["gk"])))


def _run_attention(st):
    from analog_moe_amd.attention import attention
    if not st["case"]["train"]:
        with torch.no_grad():
            return attention(st["q"], st["k"], st["v"], lengths=st["lengths"], starts=st["starts"])
    out = attention(st["q"], st["k"], st["v"], lengths=st["lengths"], starts=st["starts"])
    return (out.detach(), *torch.autograd.grad(out, (st["q"], st["k"], st["v"]), st["go"]))


# ------------------------------------------------------------------------------ the plain forms
def _turn(x, cos, sin, R, interleaved):
    """x [B, S, heads, d] with its first R elements turned; cos, sin [B, S, 1, R / 2] in 32 bits."""
    f = x.float()
    a, b = (f[..., 0:R:2], f[..., 1:R:2]) if interleaved else (f[..., :R // 2], f[..., R // 2:R])
    u, w = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((u, w), -1).flatten(-2) if interleaved else torch.cat((u, w), -1)
    return torch.cat((turned, f[..., R:]), -1).to(x.dtype)


def _plain_rotary(st):
    c = st["case"]
    R, il, size = _turned(c), c["interleaved"], _theta(c)[1]
    angle = st["positions"].double()[..., None, None] * st["theta"]      # far positions: 32 bits lose the angle
    cos, sin = (size * torch.cos(angle)).float(), (size * torch.sin(angle)).float()
    out = _turn(st["q"], cos, sin, R, il), _turn(st["k"], cos, sin, R, il)
    if c["train"]:
        out += _turn(st["gq"], cos, -sin, R, il), _turn(st["gk"], cos, -sin, R, il)
    return out


def _heads_first(x, groups):
    """[B, S, heads, d] -> [B, groups, heads / groups * S, d] in 32 bits."""
    B, S, H, d = x.shape
    return x.float().permute(0, 2, 1, 3).reshape(B, groups, H // groups * S, d)


def _heads_last(x, S, dtype):
    B, G, rows, d = x.shape
    return x.reshape(B, G * (rows // S), S, d).permute(0, 2, 1, 3).to(dtype).contiguous()


def _plain_attention(st):
    c = st["case"]
    S, T, G, d = (c[n] for n in "STGd")
    dt, dev = st["q"].dtype, st["q"].device
    key = torch.arange(T, device=dev)
    at = torch.arange(S, device=dev) + (T - S)
    if st["starts"] is not None:
        at = st["starts"][:, None] + torch.arange(S, device=dev)
    seen = key <= at.reshape(-1, S, 1)                                    # [B or 1, S, T]
    k, v = _heads_first(st["k"], G), _heads_first(st["v"], G)
    if st["lengths"] is not None:
        held = key < st["lengths"][:, None]
        seen = seen & held[:, None]
        k, v = (torch.where(held[:, None, :, None], t, 0.0) for t in (k, v))
    seen = seen[:, None].repeat(1, 1, c["H"] // G, 1)                     # [.., 1, heads of a group * S, T]
    q = _heads_first(st["q"], G)
    scale = 1 / math.sqrt(d)
    p = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(scale)
    p.masked_fill_(~seen, float("-inf"))
    top = p.amax(-1, keepdim=True)
    p.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(torch.where(total == 0, 1.0, total))
    o = torch.matmul(p, v)
    out = _heads_last(o, S, dt)
    if not c["train"]:
        return out
    go = _heads_first(st["go"], G)
    dv = torch.matmul(p.transpose(2, 3), go)
    ds = torch.matmul(go, v.transpose(2, 3).contiguous())
    ds.sub_((go * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq, dk = torch.matmul(ds, k), torch.matmul(ds.transpose(2, 3), q)
    return out, _heads_last(dq, S, dt), _heads_last(dk, T, dt), _heads_last(dv, T, dt)


# ------------------------------------------------------------------------------ what a pass cannot do without
def _marks(c, seed=0):
    """Expected keys a sequence holds, and pairs of query and key that see each other, per sequence and head."""
    S, T = c["S"], c["T"]
    held = T if not c["ragged"] else ((T + max(S, T // 2)) / 2 if not c["train"] else (T + max(1, T // 4)) / 2)
    if c["train"]:
        return held, held * (held + 1) / 2 + (S - held) * held
    return held, S * (held - (S - 1) / 2)


def work(case):
    c = case
    size = 4 if c["dtype"] == "f32" else 2
    B, S, T, H, G, d = (c[n] for n in "BSTHGd")
    if c["op"] == "rotary":
        passes = 2 if c["train"] else 1
        n = B * S * (H + G)
        return {"bytes": passes * (2 * n * d * size + 8 * B * S), "flops": passes * 3 * n * _turned(c)}
    held, pairs = _marks(c)
    rows, keys = B * S * H * d * size, B * held * G * d * size
    if c["train"]:      # q, k, v, gradient of the output in; output, three gradients out
        return {"bytes": 4 * rows + 2 * keys + 2 * B * T * G * d * size, "flops": 14 * B * H * pairs * d}
    return {"bytes": 2 * rows + 2 * keys, "flops": 4 * B * H * pairs * d}


# ------------------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return _exact_rotary(case, st) if case["op"] == "rotary" else _exact_attention(case, st)


def _exact_rotary(c, st):
    """Pairs as complex numbers times e^(i angle), or e^(-i angle) for a gradient."""
    th, size = _theta(c)
    R = _turned(c)
    angle = st["positions"].to(torch.float64)[:, :, None, None] * torch.tensor(th, dtype=torch.float64, device="cuda")
    unit = torch.polar(torch.full_like(angle, size), angle)

    def turn(x, w):
        y = x.to(torch.float64)
        pairs = y[..., :R].unflatten(-1, (R // 2, 2) if c["interleaved"] else (2, R // 2))
        if not c["interleaved"]:
            pairs = pairs.transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * w)
        if not c["interleaved"]:
            z = z.transpose(-1, -2)
        y = y.clone()
        y[..., :R] = z.flatten(-2)
        return y
    out = [turn(st["q"], unit), turn(st["k"], unit)]
    if c["train"]:
        out += [turn(st["gq"], unit.conj()), turn(st["gk"], unit.conj())]
    return tuple(out)


def _exact_attention(c, st):
    """Sequence by sequence and head by head, on the keys that a sequence holds."""
    B, S, T, H, G, d = (c[n] for n in "BSTHGd")
    f64 = dict(dtype=torch.float64, device="cuda")
    out, dq = torch.zeros(B, S, H, d, **f64), torch.zeros(B, S, H, d, **f64)
    dk, dv = torch.zeros(B, T, G, d, **f64), torch.zeros(B, T, G, d, **f64)
    lengths = [T] * B if st["lengths"] is None else st["lengths"].tolist()
    starts = [T - S] * B if st["starts"] is None else st["starts"].tolist()
    for b in range(B):
        n = lengths[b]
        hidden = torch.arange(n, device="cuda") > (starts[b] + torch.arange(S, device="cuda"))[:, None]
        for h in range(H):
            j = h // (H // G)
            q, k, v = st["q"][b, :, h].double(), st["k"][b, :n, j].double(), st["v"][b, :n, j].double()
            w = torch.softmax((q @ k.T / d ** 0.5).masked_fill(hidden, -math.inf), -1)
            w = w.masked_fill(hidden, 0.0)                     # (a row that sees nothing: zeros, not NaN)
            out[b, :, h] = w @ v
            if c["train"]:
                g = st["go"][b, :, h].double()
                dv[b, :n, j] += w.T @ g
                s = g @ v.T
                s = w * (s - (w * s).sum(-1, keepdim=True)) / d ** 0.5
                dq[b, :, h] = s @ k
                dk[b, :n, j] += s.T @ q
    return (out, dq, dk, dv) if c["train"] else out
