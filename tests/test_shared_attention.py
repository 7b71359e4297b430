"""Attention of sequences that share a prefix against its formula in 64 bits: the kernels' source on the CPU, and the built library on
the GPU."""
import pytest
import torch

from analog_moe_amd import attention as A
from oracle import attention_oracle as O
from tests.test_attention import DT, _on_gpu, marks
from tests.test_emu_kernels import emu_ops  # noqa: F401


def test_a_gpu_is_needed():
    t = torch.zeros(2, 1, 1, 8)
    with pytest.raises(RuntimeError, match="GPU"):
        A.shared_attention(t, t, t, t[:1], t[:1])


def inputs(N, R, S, P, T, H, G, d, dtype, seed=0, layout="own", gain=1.0):
    """q, k, v, prefix_k, prefix_v of N prefixes with R sequences each."""
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: (torch.randn(*s, generator=g) * gain).to(DT[dtype])                   # noqa: E731
    B = N * R
    if layout == "odd":
        return (n(B, S, H, d + 3)[..., 1:d + 1], n(B, T, G, d + 5)[..., 2:d + 2], n(B, T, G, d + 1)[..., :d], n(N, P, G, d + 1)[..., 1:],
                n(N, P, G, d + 3)[..., 3:])
    if layout == "cache":                                 # a packed projection's queries, caches with room, a prefix among others
        return (n(B, S, H + 2 * G, d)[:, :, :H], n(B, T + 9, G, d)[:, :T], n(B, T + 2, G, d)[:, :T], n(N + 2, P + 7, G, d)[1:N + 1, :P],
                n(N + 1, P + 3, G, d)[1:, 3:])
    if layout == "heads":
        return (n(B, H, S, d).transpose(1, 2), n(B, G, T, d).transpose(1, 2), n(B, G, T, d).transpose(1, 2), n(N, G, P, d).transpose(1, 2),
                n(N, G, P, d).transpose(1, 2))
    if layout == "one":                                   # every sequence's own keys are the same memory, and so are the prefixes
        return (n(1, S, H, d).expand(B, S, H, d), n(1, T, G, d).expand(B, T, G, d), n(1, T, G, d).expand(B, T, G, d),
                n(1, P, G, d).expand(N, P, G, d), n(1, P, G, d).expand(N, P, G, d))
    return n(B, S, H, d), n(B, T, G, d), n(B, T, G, d), n(N, P, G, d), n(N, P, G, d)


def formula(q, k, v, pk, pv, lengths=None, starts=None, prefix_lengths=None, causal=True, scale=None):
    """(out, bound): query by query, over its prefix and its own keys in one row."""
    B, S, H, d = q.shape
    T, N, P = k.shape[1], pk.shape[0], pk.shape[1]
    out, bound = torch.empty(B, S, H, d, dtype=torch.float64), torch.empty(B, S, H, d, dtype=torch.float64)
    for b in range(B):
        n = P if prefix_lengths is None else min(max(int(prefix_lengths[b // (B // N)]), 0), P)
        t = T if lengths is None else min(max(int(lengths[b]), 0), T)
        first = T - S if starts is None else int(starts[b])
        keys, values = (torch.cat((x[b // (B // N), :n], y[b, :t]))[None] for x, y in ((pk, k), (pv, v)))
        for i in range(S):
            at = n + max(first + i, -1) if causal else n + t
            (o,), (e,) = O.attention(q[b:b + 1, i:i + 1], keys, values, starts=torch.tensor([at]), scale=scale)
            out[b, i], bound[b, i] = o[0, 0], e[0, 0]
    return out, bound


def check(tensors, device="cpu", rows=None, **how):
    """rows: (sequences, queries) that are looked at, None for all."""
    to = lambda t: t if device == "cpu" or not isinstance(t, torch.Tensor) else _on_gpu(t)          # noqa: E731
    got = A.shared_attention_forward(*map(to, tensors), **{n: to(t) for n, t in how.items()})
    again = A.shared_attention_forward(*map(to, tensors), **{n: to(t) for n, t in how.items()})
    assert torch.equal(got, again) and got.shape == tensors[0].shape and got.is_contiguous() and torch.isfinite(got).all()
    want, bound = formula(*tensors, **how)
    worst = ((got.cpu().double() - want).abs() / bound).max().item() if want.numel() else 0.0
    assert worst <= 1.0, worst
    return got


CASES = {
    # N, R, S, P, T, H, G, d, dtype, layout, options
    "one": (1, 1, 1, 1, 1, 1, 1, 8, "f32", "own", {}),
    "few": (1, 4, 1, 150, 40, 4, 4, 64, "bf16", "own", {}),
    "few_f32": (2, 3, 1, 70, 33, 4, 2, 32, "f32", "cache", dict(lengths=[33, 1, 0, 7, 20, 33], starts=[32, 0, -1, 6, 19, 32], prefix_lengths=[70, 13])),
    "rows_64": (1, 20, 1, 300, 20, 4, 2, 64, "bf16", "cache", dict(prefix_lengths=[257])),
    "rows_64_f16": (2, 6, 2, 200, 9, 8, 2, 96, "f16", "heads", {}),
    "rows_many": (1, 21, 2, 190, 5, 8, 2, 64, "f16", "own", {}),
    "rows_many_128": (1, 33, 1, 130, 3, 4, 1, 128, "bf16", "own", {}),
    "rows_many_f32": (2, 9, 1, 77, 10, 8, 1, 40, "f32", "own", dict(prefix_lengths=[0, 50])),
    "check": (2, 2, 5, 90, 21, 4, 2, 80, "f16", "cache", dict(lengths=[21, 5, 12, 20], starts=[16, 0, 7, 15], prefix_lengths=[90, 31])),
    "prompts": (1, 2, 40, 70, 60, 2, 1, 64, "bf16", "own", {}),
    "prompts_full": (1, 2, 35, 40, 50, 2, 2, 64, "f16", "own", dict(causal=False, lengths=[50, 11])),
    "odd": (2, 3, 1, 45, 13, 3, 1, 13, "bf16", "odd", {}),
    "odd_rows": (1, 40, 1, 70, 5, 2, 2, 20, "f32", "odd", dict(prefix_lengths=[69])),
    "same_memory": (2, 3, 1, 60, 20, 2, 1, 64, "bf16", "one", {}),
    "no_own": (2, 2, 1, 60, 0, 2, 1, 64, "bf16", "own", {}),
    "no_prefix": (1, 3, 1, 0, 50, 2, 1, 64, "bf16", "own", {}),
    "nothing": (1, 2, 2, 0, 0, 2, 1, 64, "f32", "own", {}),
    "sees_nothing": (2, 2, 1, 40, 30, 2, 1, 64, "f16", "own", dict(lengths=[0, 30, 30, 0], starts=[0, -1, -5, 3], prefix_lengths=[0, 7])),
    "each_alone": (4, 1, 1, 40, 30, 2, 1, 64, "bf16", "own", {}),
    "scale": (1, 3, 1, 40, 30, 2, 1, 64, "bf16", "own", dict(scale=0.9)),
    "past_the_end": (1, 2, 1, 40, 30, 2, 1, 64, "bf16", "own", dict(lengths=[99, -4], starts=[10 ** 6, 5], prefix_lengths=[1000])),
}


def options(o):
    return {n: marks(x, torch.int64 if n == "starts" else torch.int32) if n in ("lengths", "starts", "prefix_lengths") else x for n, x in o.items()}


@pytest.mark.parametrize("name", list(CASES))
def test_emulated(emu_ops, name):
    *sizes, dtype, layout, o = CASES[name]
    check(inputs(*sizes, dtype, seed=len(name), layout=layout), **options(o))


def test_queries_that_see_nothing_give_zeros(emu_ops):
    t = inputs(2, 2, 1, 40, 30, 2, 1, 64, "bf16")
    out = A.shared_attention(*t, lengths=marks([0, 30, 0, 30]), starts=marks([0, -1, 5, 29]), prefix_lengths=marks([0, 0]))
    assert not out[:3].any() and out[3].any()


def poisoned(device="cpu"):
    q, k, v, pk, pv = inputs(2, 3, 2, 130, 70, 4, 2, 64, "bf16", seed=1)
    n, t = [101, 0], [70, 3, 64, 9, 2, 33]
    how = dict(lengths=marks(t).to(device), starts=marks([x - 2 for x in t]).to(device), prefix_lengths=marks(n, torch.int64).to(device))
    q, k, v, pk, pv = (x.to(device) for x in (q, k, v, pk, pv))
    want = A.shared_attention(q, k, v, pk, pv, **how)
    for b in range(6):
        k[b, t[b]:], v[b, t[b]:] = float("nan"), float("inf")
    for b in range(2):
        pk[b, n[b]:], pv[b, n[b]:] = float("inf"), float("nan")
    assert torch.equal(A.shared_attention(q, k, v, pk, pv, **how), want)


def test_what_lies_behind_the_keys_is_not_read(emu_ops):
    poisoned()


@pytest.mark.gpu
def test_gpu_what_lies_behind_the_keys_is_not_read():
    poisoned("cuda")


def test_like_attention_over_both(emu_ops):
    """The same as attention over copies of the prefix with the own keys behind, to the rounding of either."""
    q, k, v, pk, pv = inputs(2, 3, 1, 50, 20, 4, 2, 64, "f32", seed=4)
    got = A.shared_attention(q, k, v, pk, pv)
    keys, values = (torch.cat((x.repeat_interleave(3, 0), y), 1) for x, y in ((pk, k), (pv, v)))
    assert (got - A.attention_forward(q, keys, values)[0]).abs().max() < 2.0 ** -18


def test_scores_far_from_zero(emu_ops):
    """Parts whose largest scores are far apart, and far from zero: the prefix takes all, the own keys take all."""
    q, k, v, pk, pv = inputs(1, 2, 1, 90, 40, 2, 2, 64, "f32", seed=6, gain=100.0)
    check((q, k, v * 0.01, pk * 30, pv * 0.01))
    check((q, k * 30, v * 0.01, pk, pv * 0.01))


def test_no_sequences(emu_ops):
    t = torch.empty(0, 1, 2, 64)
    p = torch.empty(2, 5, 2, 64)
    assert A.shared_attention(t, t, t, p, p).shape == (0, 1, 2, 64)
    q = torch.empty(2, 0, 2, 64)
    k = torch.empty(2, 3, 2, 64)
    assert A.shared_attention(q, k, k, p, p).shape == (2, 0, 2, 64)


def test_refusals(emu_ops):
    q, k, v, pk, pv = inputs(2, 2, 1, 10, 6, 4, 2, 16, "f32")
    for bad in ((q, k, v, pk[:, :, :1], pv[:, :, :1]), (q, k, v, pk, pv[:, :5]), (q, k, v, pk[..., :8], pv[..., :8]), (q, k, v, pk[0], pv[0]),
                (q, k, v, pk[:0], pv[:0]), (q[:3], k[:3], v[:3], pk, pv), (q, k[:2], v[:2], pk, pv)):
        with pytest.raises(ValueError):
            A.shared_attention(*bad)
    for how in (dict(lengths=marks([1, 2])), dict(prefix_lengths=marks([1, 2, 3, 4])), dict(scale=0.0), dict(scale=float("nan"))):
        with pytest.raises(ValueError):
            A.shared_attention(q, k, v, pk, pv, **how)
    with pytest.raises(TypeError):
        A.shared_attention(q, k, v, pk.half(), pv.half())
    with pytest.raises(TypeError):
        A.shared_attention(q, k, v, pk, pv, prefix_lengths=torch.ones(2))
    with pytest.raises(RuntimeError, match="no gradient"):
        A.shared_attention(q, k, v, pk.requires_grad_(), pv)


def test_library_refuses(emu_ops):
    from analog_moe_amd import _abi
    lib = emu_ops.get_lib()
    q, k, v, pk, pv = inputs(2, 2, 1, 10, 6, 4, 2, 16, "f32")
    ws, p = torch.zeros(1 << 16), q.data_ptr()

    def call(ws_at=ws.data_ptr(), size=1 << 18, **o):
        f = dict(dtype=0, B=4, S=1, T=6, P=10, N=2, H=4, G=2, d=16, causal=1, scale=0.25)
        for name, t in (("q", q), ("k", k), ("v", v), ("pk", pk), ("pv", pv)):
            f.update({name: t.data_ptr(), name + "b": t.stride(0), name + "s": t.stride(1), name + "h": t.stride(2)})
        f.update(l=0, l64=0, m=0, m64=0, held=0, held64=0, out=p)
        f.update(o)
        return lib.amoe_attention_shared_fwd(_abi.SHARED_ATTN_ARGS.pack(*f.values()), ws_at, size, None)
    out = torch.zeros_like(q)
    assert call(out=out.data_ptr()) == 0 and call(B=0, q=0) == 0
    for o in (dict(dtype=5), dict(B=-1), dict(P=-1), dict(N=-1), dict(G=0), dict(scale=0.0), dict(pkb=-1), dict(kh=1 << 41)):
        assert call(**o) == -1, o
    assert call(N=3) == call(H=5) == call(N=0) == -3
    assert call(q=0) == call(pk=0) == call(pv=0) == call(k=0) == call(out=0) == call(ws_at=None) == -2
    assert call(q=p + 2) == call(out=p + 1) == call(held=ws.data_ptr() + 2) == call(ws_at=ws.data_ptr() + 4) == -4
    assert call(size=64) == -5
    assert call(d=129) == call(P=1 << 29) == call(S=1 << 22) == -6
    assert lib.amoe_attention_shared_fwd(None, None, 0, None) == -2


def test_operator_on_meta():
    m = dict(device="meta")
    q, k, p = torch.empty(4, 1, 4, 16, **m), torch.empty(4, 6, 2, 16, **m), torch.empty(2, 9, 2, 16, **m)
    assert torch.ops.amoe.attention_shared(q, k, k, p, p, None, None, None, True, None).shape == q.shape


# ------------------------------------------------------------------------------ on the GPU
GPU_CASES = dict(CASES, **{
    "long": (1, 4, 1, 9001, 300, 4, 4, 64, "bf16", "own", {}),
    "long_64": (1, 16, 1, 5003, 130, 8, 2, 128, "bf16", "cache", dict(prefix_lengths=[5001])),
    "long_many": (2, 40, 1, 3001, 65, 8, 2, 128, "f16", "own", dict(prefix_lengths=[3001, 1777])),
    "long_many_f32": (1, 40, 1, 2001, 65, 8, 2, 64, "f32", "own", {}),
    "long_80": (3, 8, 5, 2000, 90, 8, 2, 80, "f16", "own", dict(prefix_lengths=[2000, 1, 999])),
    "long_odd": (1, 50, 1, 1501, 33, 4, 2, 45, "bf16", "odd", {}),
    "many_parts": (1, 2, 1, 60001, 100, 2, 1, 64, "f16", "own", {}),
    "long_prompts": (2, 2, 150, 700, 300, 4, 2, 128, "bf16", "own", {}),
})


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(GPU_CASES))
def test_gpu(name):
    *sizes, dtype, layout, o = GPU_CASES[name]
    check(inputs(*sizes, dtype, seed=len(name), layout=layout), "cuda", **options(o))


@pytest.mark.gpu
def test_gpu_offsets_past_32_bits():
    """Prefixes and own keys 2^32 bytes and more apart."""
    q, k, v, pk, pv = inputs(2, 2, 1, 40, 9, 2, 1, 64, "bf16", seed=2)

    def far(t):
        step = 3 << 29
        out = torch.empty(step * (t.shape[0] - 1) + t[0].numel(), dtype=t.dtype, device="cuda").as_strided(t.shape, (step, 64, 64, 1))
        return out.copy_(t)
    got = A.shared_attention(q.cuda(), far(k), far(v), far(pk), far(pv))
    assert torch.equal(got, A.shared_attention(*(t.cuda() for t in (q, k, v, pk, pv))))


@pytest.mark.gpu
def test_gpu_stream_graph_and_compile():
    q, k, v, pk, pv = (t.cuda() for t in inputs(2, 30, 1, 1001, 90, 4, 2, 64, "bf16"))
    lengths, held = torch.full((60,), 50, device="cuda"), torch.tensor([1001, 400], dtype=torch.int32, device="cuda")

    def work():
        return A.shared_attention(q, k, v, pk, pv, lengths=lengths, starts=lengths - 1, prefix_lengths=held)
    want = work().clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = work()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(want, got)
    assert torch.equal(torch.compile(work, fullgraph=True, backend="aot_eager")(), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for step in range(3):
        q.mul_(1.5)
        lengths.add_(13)
        held.sub_(100)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(work(), out), step
