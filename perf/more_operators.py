"""Timed workloads of the decoder's other operators: layer norm of a residual stream with its gradient, attention of sequences
that continue one prompt, and the choice of the next token.

A case names the operator and its sizes.  "norm": rows of D elements; with ``residual`` the sum of a sublayer's output and the
stream is formed (rounded to the type, returned) and normalised; with ``train`` the pass returns all gradients too.  "shared":
N prompts of up to P keys, each continued by R sequences that hold up to T keys of their own; S queries a sequence, H heads over G
key heads of d elements.  "sample": B rows of V logits, one number of [0, 1) for each, and the settings of the draw.  Tensors are
in GPU memory before a pass.  ``run`` computes the operators from elementary operations; with ``own`` it calls the package.

A draw: tokens rank by their logits, the lower index first among equals; each weighs exp((logit - largest) / temperature).
Kept are the first top_k (0: all), of these the shortest run from the top with at least top_p of their weight, of these what weighs
min_p of the largest or more.  The token is the first, in the order of the indices, up to which the kept ones weigh more than u times
all of them.  Temperature 0: the largest logit.  Not-a-numbers count as minus infinity; a row of nothing else gives -1.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-5


def _norm(name, rows, D, dtype, residual=True, train=True):
    return dict(name=name, op="norm", rows=rows, D=D, dtype=dtype, residual=residual, train=train)


def _shared(name, N, R, S, P, T, H, G, d, dtype, ragged=True):
    return dict(name=name, op="shared", N=N, R=R, S=S, P=P, T=T, H=H, G=G, d=d, dtype=dtype, ragged=ragged)


def _sample(name, B, V, dtype, spread=2.5, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mixed=False, masked=False):
    return dict(name=name, op="sample", B=B, V=V, dtype=dtype, spread=spread, temperature=temperature, top_k=top_k, top_p=top_p,
                min_p=min_p, mixed=mixed, masked=masked)


def listed():
    return [
        # one new token of each of 16 sequences, the benchmark's model width: launches and host time
        _norm("norm_step_bf16", 16, 1024, "bf16", train=False),
        # the benchmark's decoder: a training step's 16 x 1024 tokens
        _norm("norm_train_bf16", 16384, 1024, "bf16"),
        # an odd number of tokens of a width that is no whole number of 16-byte chunks, no stream to add to
        _norm("norm_ragged_f16", 5003, 412, "f16", residual=False),
        # a wide model in single precision
        _norm("norm_wide_f32", 4096, 8192, "f32"),
        # four answers to a short prompt, the benchmark's heads: the smallest call
        _shared("shared_4_bf16", 1, 4, 1, 500, 64, 16, 16, 64, "bf16"),
        # 64 answers to one long document, some hundred tokens in
        _shared("shared_64_bf16", 1, 64, 1, 30001, 1024, 16, 4, 128, "bf16"),
        # prompts of different lengths, eight answers each, five proposed tokens checked at once; heads of 80
        _shared("shared_check_f16", 3, 8, 5, 4000, 300, 8, 2, 80, "f16"),
        # four prompts with 64 answers each: the largest call
        _shared("shared_256_bf16", 4, 64, 1, 8192, 512, 32, 8, 128, "bf16"),
        # one sequence, the benchmark's vocabulary
        _sample("sample_1_bf16", 1, 8000, "bf16", temperature=0.8, top_p=0.9),
        # a serving batch in which every request has settings of its own, some tokens forbidden
        _sample("sample_mixed_bf16", 64, 50001, "bf16", mixed=True, masked=True),
        # many rows of the benchmark's vocabulary without truncation, as rollouts for training draw them
        _sample("sample_full_f32", 2048, 8000, "f32"),
        # a large batch over a large vocabulary, flat rows of which many tokens are kept
        _sample("sample_256_f32", 256, 130001, "f32", spread=1.5, temperature=1.2, top_k=60000, top_p=0.95),
    ]


def _spread(rng: random.Random, lo: int, hi: int) -> int:
    """An integer of [lo, hi], its logarithm evenly spread."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng: random.Random):
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    op = rng.choice(("norm", "shared", "sample"))
    if op == "norm":
        D = _spread(rng, 8, 16384)
        c = _norm("", max(1, min(_spread(rng, 1, 65536), 4096 * 8192 // D)), D, dtype, rng.random() < 0.6, rng.random() < 0.7)
    elif op == "shared":
        G = rng.choice((1, 2, 4, 8))
        H = G * rng.choice((1, 2, 4, 8))
        d = rng.choice((32, 64, 64, 80, 96, 128, 128))
        N, R, S = _spread(rng, 1, 8), _spread(rng, 1, 64), rng.choice((1, 1, 1, 2, 5, 16))
        # no more pairs of query and key than the largest listed case (single precision has a sixteenth of the matrix rate), no
        # more bytes of keys and values
        f32 = dtype == "f32"
        most, keys = 256 * 32 * 128 * 6500 // (8 if f32 else 1), 3 * (8192 + 64 * 512) * 8 * 128 // (2 if f32 else 1)
        P = max(1, min(_spread(rng, 16, 65536), most // (N * R * S * H * d) // 2, keys // (N * G * d) // 2))
        T = max(S, min(_spread(rng, 1, 4096), most // (N * R * S * H * d) // 2, keys // (N * R * G * d) // 2))
        c = _shared("", N, R, S, P, T, H, G, d, dtype, rng.random() < 0.6)
    else:
        V = _spread(rng, 50, 260000)
        c = _sample("", max(1, min(_spread(rng, 1, 2048), 256 * 130001 // V)), V, dtype, rng.choice((0.5, 1.5, 2.5, 4.0)),
                    rng.choice((0.0, 0.6, 0.8, 1.0, 1.0, 1.3)), rng.choice((0, 0, 0, 1, 20, 50, _spread(rng, 1, V))),
                    rng.choice((1.0, 1.0, 0.5, 0.9, 0.95)), rng.choice((0.0, 0.0, 0.02, 0.1)), rng.random() < 0.3, rng.random() < 0.3)
    del c["name"]
    return c


def prepare(case, seed):
    c = case
    dt, dev = DTYPES[c["dtype"]], "cuda"
    g = torch.Generator(dev).manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32).mul_(scale).to(dt)

    def choose(values, n, dtype):
        return torch.tensor(values, dtype=dtype, device=dev)[torch.randint(0, len(values), (n,), generator=g, device=dev)]
    st = dict(case=c)
    if c["op"] == "norm":
        rows, D = c["rows"], c["D"]
        # a stream with some channels that are far larger than the others, off their mean
        channel = torch.randn(D, generator=g, device=dev).mul_(1.5).exp_()
        stream = torch.randn(rows, D, generator=g, device=dev).add_(0.3).mul_(channel).to(dt)
        st["x"], st["r"] = (normal(rows, D, scale=0.5), stream) if c["residual"] else (stream, None)
        st["w"], st["b"] = (torch.randn(D, generator=g, device=dev).mul_(0.2).add_(1).to(dt), normal(D, scale=0.1))
        if c["train"]:
            st["gy"] = normal(rows, D)
            st["gs"] = normal(rows, D) if c["residual"] else None
            for n in ("x", "r", "w", "b"):
                if st[n] is not None:
                    st[n].requires_grad_()
    elif c["op"] == "shared":
        N, R, S, P, T, H, G, d = (c[n] for n in "NRSPTHGd")
        B = N * R
        st["q"] = normal(B, S, H + 2 * G, d)[:, :, :H]                   # a view of the packed projection
        st["pk"], st["pv"], st["k"], st["v"] = normal(N, P, G, d), normal(N, P, G, d), normal(B, T, G, d), normal(B, T, G, d)
        st["held"] = torch.randint(max(1, P // 2), P + 1, (N,), generator=g, device=dev) if c["ragged"] else None
        st["lengths"] = torch.randint(max(S, T // 2), T + 1, (B,), generator=g, device=dev) if c["ragged"] else None
        st["starts"] = st["lengths"] - S if c["ragged"] else None        # the queries are the last of what their cache holds
    else:
        B, V = c["B"], c["V"]
        x = torch.randn(B, V, generator=g, device=dev).mul_(c["spread"])
        # a few likely tokens in every row
        at = torch.randint(0, V, (B, 5), generator=g, device=dev)
        x.scatter_add_(1, at, torch.rand(B, 5, generator=g, device=dev).mul_(3 * c["spread"]))
        if c["masked"]:
            x.masked_fill_(torch.rand(B, V, generator=g, device=dev) < 0.2, -math.inf)
        st["logits"] = x.to(dt)
        st["u"] = torch.rand(B, generator=g, device=dev)
        st["how"] = {n: c[n] for n in ("temperature", "top_k", "top_p", "min_p")}
        if c["mixed"]:
            st["how"] = dict(temperature=choose((0.0, 0.7, 1.0, 1.0, 1.3), B, torch.float32),
                             top_k=choose((0, 0, 1, 40, 1000), B, torch.int64),
                             top_p=choose((1.0, 0.95, 0.5), B, torch.float32), min_p=choose((0.0, 0.0, 0.05, 0.1), B, torch.float32))
    return st


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _run_norm, "shared": _run_shared, "sample": _run_sample}[op](state)
    with torch.no_grad():
        return {"norm": _plain_norm, "shared": _plain_shared, "sample": _plain_sample}[op](state)


# ------------------------------------------------------------------------------ the package
def _run_norm(st):
    from analog_moe_amd.norm import layer_norm
    if not st["case"]["train"]:
        with torch.no_grad():
            return layer_norm(st["x"], st["w"], st["b"], EPS, residual=st["r"])
    if st["r"] is None:
        y = layer_norm(st["x"], st["w"], st["b"], EPS)
        return (y.detach(), *torch.autograd.grad(y, (st["x"], st["w"], st["b"]), st["gy"]))
    y, s = layer_norm(st["x"], st["w"], st["b"], EPS, residual=st["r"])
    return (y.detach(), s.detach(), *torch.autograd.grad((y, s), (st["x"], st["r"], st["w"], st["b"]), (st["gy"], st["gs"])))


def _run_shared(st):
    from analog_moe_amd.attention import shared_attention
    with torch.no_grad():
        return shared_attention(st["q"], st["k"], st["v"], st["pk"], st["pv"], lengths=st["lengths"], starts=st["starts"],
                                prefix_lengths=st["held"])


def _run_sample(st):
    from analog_moe_amd.sampling import sample
    return sample(st["logits"], st["u"], **st["how"], want_logprob=True)


# ------------------------------------------------------------------------------ the plain forms
def _plain_norm(st):
    dt = st["x"].dtype
    s = st["x"] if st["r"] is None else (st["x"].float() + st["r"].float()).to(dt)
    f, w = s.float(), st["w"].float()
    d = f - f.mean(-1, keepdim=True)
    inv = torch.rsqrt((d * d).mean(-1, keepdim=True) + EPS)
    h = d * inv
    y = (h * w + st["b"].float()).to(dt)
    out = (y,) if st["r"] is None else (y, s)
    if not st["case"]["train"]:
        return out if len(out) > 1 else y
    gy = st["gy"].float()
    gh = gy * w
    dx = (gh - gh.mean(-1, keepdim=True) - h * (gh * h).mean(-1, keepdim=True)) * inv
    if st["gs"] is not None:
        dx = dx + st["gs"].float()
    dx = dx.to(dt)
    grads = (dx,) if st["r"] is None else (dx, dx)
    return (*out, *grads, (gy * h).sum(0).to(dt), gy.sum(0).to(dt))


def _plain_shared(st):
    c = st["case"]
    N, R, S, P, T, H, G, d = (c[n] for n in "NRSPTHGd")
    B, dev, q = N * R, st["q"].device, st["q"].float()
    rep = H // G
    # rows of a key head: [N, G, R * rep * S, d] against the prompt, [B, G, rep * S, d] against a sequence's own keys
    own_q = q.permute(0, 2, 1, 3).reshape(B, G, rep * S, d)
    all_q = own_q.reshape(N, R, G, rep * S, d).transpose(1, 2).reshape(N, G, R * rep * S, d)
    pk, pv, k, v = (st[n].float().permute(0, 2, 1, 3) for n in ("pk", "pv", "k", "v"))
    in_prompt = torch.arange(P, device=dev) < (torch.full((N, 1), P, device=dev) if st["held"] is None else st["held"][:, None])
    held = torch.arange(T, device=dev) < (torch.full((B, 1), T, device=dev) if st["lengths"] is None else st["lengths"][:, None])
    at = (torch.full((B, 1), T - S, device=dev) if st["starts"] is None else st["starts"][:, None]) + torch.arange(S, device=dev)
    seen = held[:, None] & (torch.arange(T, device=dev) <= at[..., None])                      # [B, S, T]
    scale = 1 / math.sqrt(d)
    s1 = torch.matmul(all_q, pk.transpose(2, 3).contiguous()).mul_(scale)
    s1.masked_fill_(~in_prompt[:, None, None], -math.inf)
    s1 = s1.reshape(N, G, R, rep * S, P).transpose(1, 2).reshape(B, G, rep * S, P)
    s2 = torch.matmul(own_q, k.transpose(2, 3).contiguous()).mul_(scale)
    s2.masked_fill_(~seen[:, None].repeat(1, 1, rep, 1), -math.inf)
    top = torch.maximum(s1.amax(-1, keepdim=True), s2.amax(-1, keepdim=True))
    top = torch.where(top == -math.inf, 0.0, top)
    p1, p2 = s1.sub_(top).exp_(), s2.sub_(top).exp_()
    total = p1.sum(-1, keepdim=True) + p2.sum(-1, keepdim=True)
    pv, v = torch.where(in_prompt[:, None, :, None], pv, 0.0), torch.where(held[:, None, :, None], v, 0.0)
    o1 = torch.matmul(p1.reshape(N, R, G, rep * S, P).transpose(1, 2).reshape(N, G, R * rep * S, P), pv.contiguous())
    o1 = o1.reshape(N, G, R, rep * S, d).transpose(1, 2).reshape(B, G, rep * S, d)
    o = (o1 + torch.matmul(p2, v.contiguous())) / torch.where(total == 0, 1.0, total)
    return o.reshape(B, H, S, d).transpose(1, 2).to(st["q"].dtype).contiguous()


def _column(v, like):
    """A setting as [B, 1] in 64 bits, of the 32-bit number that a call is given."""
    if isinstance(v, torch.Tensor):
        return v.double()[:, None]
    return torch.tensor(v, dtype=torch.float32, device=like.device).double().expand(like.shape[0], 1)


def _plain_sample(st):
    x = st["logits"].double()                       # values next to a border: 32 bits would choose other tokens
    x = torch.where(torch.isnan(x), -math.inf, x)
    how = {n: _column(v, x) for n, v in st["how"].items()}
    greedy = how["temperature"] <= 0
    value, index = torch.sort(x, dim=-1, descending=True, stable=True)
    top = value[:, :1]
    w = torch.exp((value - top) / torch.where(greedy, 1.0, how["temperature"]))
    w = torch.where(greedy | (top == math.inf), (value == top).double(), w)
    rank = torch.arange(x.shape[1], device=x.device)
    k = torch.where(how["top_k"] <= 0, float(x.shape[1]), how["top_k"])
    w = torch.where(rank < torch.where(greedy, 1.0, k), w, 0.0)
    run_of = torch.cumsum(w, -1)
    before = torch.cat((torch.zeros_like(top), run_of[:, :-1]), -1)
    keep = (before < how["top_p"] * run_of[:, -1:]) | (how["top_p"] >= 1) | (rank == 0)
    w = torch.where(keep & (w >= how["min_p"]), w, 0.0)
    w = torch.zeros_like(w).scatter_(1, index, w)
    run_of = torch.cumsum(w, -1)
    total = run_of[:, -1:]
    token = (run_of <= st["u"].double()[:, None] * total).sum(-1, keepdim=True).clamp_(max=x.shape[1] - 1)
    logprob = torch.log(w.gather(1, token) / total)
    none = top == -math.inf
    return torch.where(none, -1, token)[:, 0], torch.where(none, -math.inf, logprob)[:, 0].float()


# ------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    size = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "norm":
        n, more = c["rows"] * c["D"], 2 if c["residual"] else 1
        tensors = 2 * more                                               # in and out
        flops = 9 * n
        if c["train"]:      # gradients in, the normalised rows again, one gradient out
            tensors += more + 2
            flops += 14 * n
        return {"bytes": tensors * n * size + 4 * c["D"] * size, "flops": flops}
    if c["op"] == "shared":
        N, R, S, P, T, H, G, d = (c[n] for n in "NRSPTHGd")
        p, t = ((P + max(1, P // 2)) / 2, (T + max(S, T // 2)) / 2) if c["ragged"] else (P, T)
        pairs = N * R * H * S * (p + t - (S - 1) / 2)
        return {"bytes": (2 * N * R * S * H * d + 2 * (N * p + N * R * t) * G * d) * size, "flops": 4 * pairs * d}
    return {"bytes": c["B"] * (c["V"] * size + 16), "flops": 4 * c["B"] * c["V"]}


# ------------------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "shared": _exact_shared, "sample": _exact_sample}[case["op"]](case, st)


def _exact_norm(c, st):
    """Through the mean and the variance as functions of the row: their derivatives, not the shortened formula."""
    D = c["D"]
    x = st["x"].double() if st["r"] is None else (st["x"].double() + st["r"].double()).to(st["x"].dtype).double()
    w, b = st["w"].double(), st["b"].double()
    mean = x.sum(-1, keepdim=True) / D
    var = (x - mean).square().sum(-1, keepdim=True) / D + EPS
    y = (x - mean) / var.sqrt() * w + b
    out = [y] if st["r"] is None else [y, x]
    if c["train"]:
        g = st["gy"].double()
        a = g * w
        d_var = -(a * (x - mean)).sum(-1, keepdim=True) / (2 * var * var.sqrt())
        d_mean = -a.sum(-1, keepdim=True) / var.sqrt()
        dx = a / var.sqrt() + d_var * 2 * (x - mean) / D + d_mean / D
        if st["gs"] is not None:
            dx = dx + st["gs"].double()
        out += [dx] if st["r"] is None else [dx, dx]
        out += [(g * (x - mean) / var.sqrt()).sum(0), g.sum(0)]
    return tuple(out) if len(out) > 1 else y


def _exact_shared(c, st):
    """Sequence by sequence over the keys that it sees, its prompt's and its own one after the other."""
    N, R, S, P, T, H, G, d = (c[n] for n in "NRSPTHGd")
    out = torch.zeros(N * R, S, H, d, dtype=torch.float64, device="cuda")
    held = [P] * N if st["held"] is None else st["held"].tolist()
    lengths = [T] * (N * R) if st["lengths"] is None else st["lengths"].tolist()
    starts = [T - S] * (N * R) if st["starts"] is None else st["starts"].tolist()
    for b in range(N * R):
        n, t = held[b // R], lengths[b]
        keys = torch.cat((st["pk"][b // R, :n], st["k"][b, :t])).double().transpose(0, 1).repeat_interleave(H // G, 0)
        values = torch.cat((st["pv"][b // R, :n], st["v"][b, :t])).double().transpose(0, 1).repeat_interleave(H // G, 0)
        hidden = torch.arange(t, device="cuda") > (starts[b] + torch.arange(S, device="cuda"))[:, None]
        hidden = torch.cat((torch.zeros(S, n, dtype=torch.bool, device="cuda"), hidden), 1)
        s = torch.matmul(st["q"][b].double().transpose(0, 1), keys.transpose(1, 2).contiguous()) / d ** 0.5
        out[b] = torch.matmul(torch.softmax(s.masked_fill(hidden, -math.inf), -1).nan_to_num(0.0), values).transpose(0, 1)
    return out


def _exact_sample(c, st):
    """Row by row on the host."""
    x, u = st["logits"].double().cpu().numpy(), st["u"].double().cpu().numpy()
    B, V = x.shape
    how = {n: v.double().cpu().numpy() if isinstance(v, torch.Tensor) else np.full(B, np.float32(v), dtype=np.float64)
           for n, v in st["how"].items()}
    token, logprob = np.full(B, -1, dtype=np.int64), np.full(B, -np.inf)
    for i in range(B):
        row = np.where(np.isnan(x[i]), -np.inf, x[i])
        top = row.max()
        if top == -np.inf:
            continue
        if how["temperature"][i] <= 0:
            token[i], logprob[i] = int(np.argmax(row)), 0.0
            continue
        w = (row == top).astype(np.float64) if top == np.inf else np.exp((row - top) / how["temperature"][i])
        order = np.argsort(-row, kind="stable")
        k = int(how["top_k"][i])
        order = order[:k] if k > 0 else order
        if how["top_p"][i] < 1:
            sums = np.cumsum(w[order])
            order = order[:1 + int(np.searchsorted(sums[:-1], how["top_p"][i] * sums[-1], side="left"))]
        order = np.sort(order[w[order] >= how["min_p"][i]])
        sums = np.cumsum(w[order])
        j = min(int(np.searchsorted(sums, u[i] * sums[-1], side="right")), len(order) - 1)
        token[i], logprob[i] = order[j], math.log(w[order[j]] / sums[-1])
    return torch.from_numpy(token), torch.from_numpy(logprob)
