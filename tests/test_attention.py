"""Attention of the decoder against its formula in 64 bits: the kernels' source on the CPU, and the built library on the GPU."""
import pytest
import torch

from analog_moe_amd import attention as A
from oracle import attention_oracle as O
from tests.test_emu_kernels import emu_ops  # noqa: F401

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def inputs(B, S, T, H, G, d, dtype, seed=0, layout="own", gain=1.0):
    """q, k, v, go.  layout: "own" tensors, "packed" views of one projection, "heads" first, "odd" offsets, "cache" with room."""
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: (torch.randn(*s, generator=g) * gain).to(DT[dtype])          # noqa: E731
    if layout == "packed":
        w = n(B, S, H + 2 * G, d)
        q, k, v = w[:, :, :H], w[:, :, H:H + G], w[:, :, H + G:]
    elif layout == "heads":
        q, k, v = n(B, H, S, d).transpose(1, 2), n(B, G, T, d).transpose(1, 2), n(B, G, T, d).transpose(1, 2)
    elif layout == "odd":
        q, k, v = n(B, S, H, d + 3)[..., 1:d + 1], n(B, T, G, d + 5)[..., 2:d + 2], n(B, T, G, d + 1)[..., :d]
    elif layout == "cache":
        q, k, v = n(B, S, H, d), n(B, T + 37, G, d)[:, :T], n(B, T + 5, G, d)[:, :T]
    elif layout == "shared":                  # one sequence's keys for the whole batch, one head's queries for all heads
        q, k, v = n(B, S, 1, d).expand(B, S, H, d), n(1, T, G, d).expand(B, T, G, d), n(1, T, G, d).expand(B, T, G, d)
    else:
        q, k, v = n(B, S, H, d), n(B, T, G, d), n(B, T, G, d)
    return q, k, v, n(B, S, H, d)


def marks(x, dtype=torch.int32):
    return None if x is None else torch.tensor(x, dtype=dtype)


def compare(got, want, bounds, what):
    for name, a, w, b in zip(("out", "dq", "dk", "dv"), got, want, bounds):
        a = a.cpu()
        assert a.shape == w.shape and torch.isfinite(a).all(), (what, name)
        worst = ((a.double() - w).abs() / b).max().item() if a.numel() else 0.0
        assert worst <= 1.0, (what, name, worst)


def check(q, k, v, go, lengths=None, starts=None, causal=True, scale=None, device="cpu"):
    kw = dict(lengths=lengths, starts=starts, causal=causal, scale=scale)
    want, bounds = O.attention(q, k, v, go, **kw)
    to = lambda t: None if t is None else t if device == "cpu" else _on_gpu(t)          # noqa: E731
    q, k, v, go, lengths, starts = map(to, (q, k, v, go, lengths, starts))
    out, lse, rest = A.attention_forward(q, k, v, lengths, starts, causal, scale, want_lse=True)
    plain, *none = A.attention_forward(q, k, v, lengths, starts, causal, scale)
    assert none == [None, None] and torch.equal(plain, out)
    assert rest is None if q.dtype == torch.float32 else (rest.abs() <= out.abs() * torch.finfo(q.dtype).eps + torch.finfo(q.dtype).tiny).all()
    compare((out, *A.attention_backward(go, q, k, v, out, lse, None, lengths, starts, causal, scale)), want, bounds, kw)
    grads = A.attention_backward(go, q, k, v, out, lse, rest, lengths, starts, causal, scale)
    compare((out, *grads), want, bounds, kw)
    again = A.attention_backward(go, q, k, v, out, lse, rest, lengths, starts, causal, scale)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    seen = O.visible(q.shape[0], q.shape[1], k.shape[1], causal, None if lengths is None else lengths.cpu(),
                     None if starts is None else starts.cpu()).any(-1)
    assert not out.cpu()[~seen].any() and not grads[0].cpu()[~seen].any()


def _on_gpu(t):
    """The tensor on the GPU with the strides that it has here."""
    base = t._base if t._base is not None else t
    flat = torch.empty(base.untyped_storage().nbytes() // base.element_size(), dtype=base.dtype, device="cuda")
    flat.copy_(torch.empty(0, dtype=base.dtype).set_(base.untyped_storage(), 0, (flat.numel(),), (1,)))
    return flat.as_strided(t.shape, t.stride(), t.storage_offset())


CASES = {
    # B, S, T, H, G, d, dtype, layout, options
    "one_token": (1, 1, 1, 1, 1, 8, "f32", "own", {}),
    "f32_small": (2, 40, 40, 2, 1, 32, "f32", "packed", {}),
    "bf16_two_tiles": (1, 70, 140, 2, 1, 64, "bf16", "own", {}),
    "f16_96": (1, 33, 70, 1, 1, 80, "f16", "heads", {}),
    "bf16_128": (1, 20, 66, 2, 2, 128, "bf16", "cache", {}),
    "odd_head": (1, 35, 35, 2, 1, 13, "bf16", "odd", {}),
    "odd_head_f32": (2, 9, 21, 2, 2, 103, "f32", "odd", {}),
    "shared": (2, 34, 34, 2, 1, 64, "bf16", "shared", {}),
    "full": (2, 17, 50, 2, 2, 64, "f16", "own", dict(causal=False, lengths=[50, 31])),
    "lengths": (3, 40, 40, 2, 1, 64, "bf16", "own", dict(lengths=[40, 0, 7])),
    "starts": (3, 5, 90, 2, 2, 64, "f32", "own", dict(lengths=[90, 33, 12], starts=[85, 28, -3])),
    "rows_see_nothing": (1, 40, 20, 1, 1, 64, "bf16", "own", {}),
    "scale": (1, 33, 33, 1, 1, 64, "bf16", "own", dict(scale=0.7)),
    "step": (2, 1, 300, 4, 2, 64, "bf16", "cache", dict(lengths=[300, 129], starts=[299, 128])),
    "step_96_f16": (1, 1, 200, 8, 1, 96, "f16", "own", {}),
    "step_odd": (1, 2, 150, 3, 1, 20, "f32", "odd", {}),
    "no_keys": (2, 3, 0, 2, 1, 64, "f32", "own", {}),
}


def options(o):
    return {n: marks(x) if n in ("lengths", "starts") else x for n, x in o.items()}


@pytest.mark.parametrize("name", list(CASES))
def test_emulated(emu_ops, name):
    *sizes, dtype, layout, o = CASES[name]
    check(*inputs(*sizes, dtype, layout=layout, seed=len(name)), **options(o))


def test_few_rows_in_parts(emu_ops, monkeypatch):
    """Rows over a long axis are worked on in parts, joined by a second kernel; also where a part holds no key."""
    q, k, v, _ = inputs(1, 1, 700, 2, 1, 64, "bf16", seed=3)
    lib = emu_ops.get_lib()
    args = A._Call(q, k, v, None, None, True, 0.125).pack(q, None, None)
    assert lib.amoe_attention_fwd_workspace(args) == 6 * 2 * 66 * 4
    for n in (700, 130, 128, 1, 0):
        kw = dict(lengths=marks([n]), starts=marks([n - 1], torch.int64))
        (want,), (bound,) = O.attention(q, k, v, **kw)
        out, lse, _ = A.attention_forward(q, k, v, **kw, want_lse=True)
        assert b"attn_join" in lib_last(lib)
        compare((out,), (want,), (bound,), n)
        assert torch.isinf(lse).all() == (n == 0)


def lib_last(lib):
    import ctypes
    lib.amoe_emu_last_kernel.restype = ctypes.c_char_p
    return lib.amoe_emu_last_kernel()


def behind_the_keys(device, sizes):
    for d in sizes:
        q, k, v, go = (t.to(device) for t in inputs(2, 6, 50, 2, 1, d, "bf16"))
        lengths, starts = marks([19, 33]).to(device), marks([13, 27]).to(device)
        want = A.attention_forward(q, k, v, lengths, starts)[0]
        k, v = k.clone(), v.clone()
        for b, n in enumerate((19, 33)):
            k[b, n:], v[b, n:] = float("nan"), float("inf")
        out, lse, rest = A.attention_forward(q, k, v, lengths, starts, want_lse=True)
        assert torch.equal(out, want)
        dq, dk, dv = A.attention_backward(go, q, k, v, out, lse, rest, lengths, starts)
        assert all(torch.isfinite(t).all() for t in (dq, dk, dv))
        assert not dk[0, 19:].any() and not dv[1, 33:].any()


def test_what_lies_behind_the_keys_is_not_read(emu_ops):
    behind_the_keys("cpu", (64, 13))


@pytest.mark.gpu
def test_gpu_what_lies_behind_the_keys_is_not_read():
    # (not a number everywhere first: nothing that a workgroup finds in its LDS may get into results either)
    nan = torch.full((64, 256, 8, 128), float("nan"), dtype=torch.bfloat16, device="cuda")
    for d in (128, 96, 80, 64, 48, 13):
        out, lse, rest = A.attention_forward(nan, nan, nan, want_lse=True)
        A.attention_backward(nan, nan, nan, nan, out, lse, rest)
        behind_the_keys("cuda", (d,))


def test_marks_outside_the_tensors(emu_ops):
    """Lengths past T are T, below 0 none; starts of any size only say what is seen."""
    q, k, v, _ = inputs(2, 3, 20, 1, 1, 64, "f32")
    big = 2 ** 62
    out = A.attention_forward(q, k, v, marks([big, -5], torch.int64), marks([big, big], torch.int64))[0]
    want = A.attention_forward(q, k, v, marks([20, 0]), causal=False)[0]
    assert torch.equal(out, want) and not out[1].any()
    assert not A.attention_forward(q, k, v, None, marks([-big, -4], torch.int64))[0].any()


def test_no_sequences_no_queries(emu_ops):
    for B, S, T in ((0, 3, 4), (2, 0, 5), (0, 0, 0)):
        q, k, v, go = inputs(B, S, T, 2, 1, 32, "bf16")
        left = A.attention_forward(q, k, v, want_lse=True)
        dq, dk, dv = A.attention_backward(go, q, k, v, *left)
        assert left[0].shape == q.shape == dq.shape and dk.shape == k.shape and not dk.any() and not dv.any()


def test_strides_of_single_elements(emu_ops):
    """How far apart the only sequence, token or head is from the next says nothing."""
    q, k, v, go = inputs(1, 1, 40, 1, 1, 64, "bf16")
    want = A.attention_forward(q, k, v)[0]
    odd = lambda t, st: torch.empty(0, dtype=t.dtype).set_(t.contiguous().untyped_storage(), 0, t.shape, st)          # noqa: E731
    assert torch.equal(A.attention_forward(odd(q, (7, 3, 1, 1)), odd(k, (5, 64, 3, 1)), odd(v, (1, 64, 9, 1)))[0], want)


def test_fp16_gradients_of_any_size(emu_ops):
    """The score gradients of fp16 tensors are held at a scale of their own: small and large gradients keep their accuracy."""
    for gain in (2.0 ** -9, 1.0, 2.0 ** 9):
        q, k, v, go = inputs(1, 40, 40, 2, 1, 64, "f16", seed=5)
        check(q, k, v, (go.float() * gain).half())


def test_refusals(emu_ops):
    q, k, v, go = inputs(2, 4, 6, 4, 2, 32, "f32")
    f = A.attention_forward
    for bad in (lambda: f(q[0], k, v), lambda: f(q, k[:1], v[:1]), lambda: f(q, k, v[:, :5]), lambda: f(q, k[..., :16], v[..., :16]),
                lambda: f(q[:, :, :3], k, v), lambda: f(q, k, v, marks([6])), lambda: f(q, k, v, None, marks([[1, 2]])),
                lambda: f(q, k, v, scale=0.0), lambda: f(q, k, v, scale=float("inf")), lambda: f(q, k, v, scale=float("nan")),
                lambda: f(*(torch.zeros(1, 1, 1, 129) for _ in range(3))), lambda: f(*(torch.zeros(1, 1, 1, 0) for _ in range(3))),
                lambda: f(q[:, :, :0], k, v), lambda: f(q, k[:, :, :0], v[:, :, :0])):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: f(q.double(), k, v), lambda: f(q, k.bfloat16(), v), lambda: f(q, k, v, torch.tensor([1.0, 2.0]))):
        with pytest.raises(TypeError):
            bad()
    out, lse, _ = f(q, k, v, want_lse=True)
    b = A.attention_backward
    for bad in (lambda: b(go[:, :3], q, k, v, out, lse), lambda: b(go, q, k, v, out, lse[:, :, :3]), lambda: b(go.half(), q, k, v, out, lse),
                lambda: b(go, q, k, v, out, lse.half()), lambda: b(go, q, k, v, out, lse, out[:1])):
        with pytest.raises(ValueError):
            bad()


def test_library_refuses_what_it_cannot_address(emu_ops):
    """Argument errors of the C entry points come back as codes, nothing is launched."""
    from analog_moe_amd import _abi
    lib = emu_ops.get_lib()
    q, k, v, go = inputs(1, 2, 3, 2, 1, 32, "f32")
    out, lse = torch.empty_like(q), torch.empty(1, 2, 2)
    good = list(_abi.ATTN_ARGS.unpack(A._Call(q, k, v, None, None, True, 0.5).pack(out, lse, None, go, (1 << 20,) * 3)))

    def fwd(**change):
        a = list(good)
        for i, x in change.items():
            a[int(i[1:])] = x
        return lib.amoe_attention_fwd(_abi.ATTN_ARGS.pack(*a), None, 0, None)
    assert fwd() == 0
    assert fwd(_0=7) == fwd(_1=-1) == fwd(_6=0) == fwd(_8=-1.0) == fwd(_8=float("nan")) == fwd(_10=-8) == -1
    assert fwd(_9=0) == fwd(_13=0) == fwd(_17=0) == fwd(_25=0) == -2
    assert fwd(_4=3, _5=2) == -3
    assert fwd(_9=good[9] + 2) == fwd(_21=good[9] + 2) == fwd(_26=good[26] + 1) == -4
    assert fwd(_6=129) == fwd(_2=2 ** 28 + 1) == fwd(_1=2 ** 31, _4=2 ** 20) == fwd(_1=2 ** 22, _2=1000) == -6
    assert lib.amoe_attention_bwd(_abi.ATTN_ARGS.pack(*good), None, 0, None) == -2
    assert lib.amoe_attention_bwd(_abi.ATTN_ARGS.pack(*good), lse.data_ptr(), 4, None) == -5
    assert lib.amoe_attention_fwd(None, None, 0, None) == -2


def test_autograd(emu_ops):
    q, k, v, go = inputs(2, 20, 20, 2, 1, 32, "f32", layout="packed")
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    out = A.attention(q, k, v)
    want, bounds = O.attention(q.detach(), k.detach(), v.detach(), go)
    compare((out.detach(), *torch.autograd.grad(out, (q, k, v), go)), want, bounds, "autograd")
    out = A.attention(q, k.detach(), v.detach())
    compare((out.detach(), *torch.autograd.grad(out, q, go)), want[:2], bounds[:2], "queries only")
    out = A.attention(q.detach(), k.detach(), v)
    compare(torch.autograd.grad(out, v, go), want[3:], bounds[3:], "values only")
    # a gradient of stride zero, and of the gradient: refused
    (g,) = torch.autograd.grad(A.attention(q, k, v).sum(), q, create_graph=True)
    compare((g.detach(),), O.attention(q.detach(), k.detach(), v.detach(), torch.ones_like(go))[0][1:2],
            O.attention(q.detach(), k.detach(), v.detach(), torch.ones_like(go))[1][1:2], "ones")
    with pytest.raises(RuntimeError, match="differentiable once"):
        (g.sum() + q.sum()).backward()
    with torch.no_grad():
        assert torch.equal(A.attention(q, k, v), A.attention_forward(q, k, v)[0])


def test_watched_calls(emu_ops):
    """Forward-mode derivatives and function transforms are refused, a trace computes anew (as for the expert layer)."""
    from torch.autograd import forward_ad
    q, k, v, _ = inputs(1, 4, 4, 1, 1, 16, "f32")
    with torch.no_grad(), forward_ad.dual_level(), pytest.raises(NotImplementedError):
        A.attention(forward_ad.make_dual(q, q), k, v)
    with torch.no_grad(), pytest.raises(RuntimeError):
        torch.func.vmap(lambda x: A.attention(x, k, v))(q[None])
    with torch.no_grad():
        traced = torch.jit.trace(lambda x: A.attention(x, k, v), (q,), check_trace=False)
        assert torch.equal(traced(k), A.attention(k, k, v))


def test_gradients_are_differences(emu_ops):
    """dq, dk and dv against central differences of the loss sum(out * go): step h, error h^2 * third derivative + 2^-24 / h."""
    q, k, v, go = inputs(1, 5, 7, 2, 1, 16, "f32", seed=11)
    grads = A.attention_backward(go, q, k, v, *A.attention_forward(q, k, v, want_lse=True))
    h = 2.0 ** -7
    loss = lambda a: (A.attention_forward(*a)[0].double() * go.double()).sum().item()          # noqa: E731
    for n, index in ((0, (0, 3, 1, 2)), (0, (0, 0, 0, 0)), (1, (0, 2, 0, 5)), (1, (0, 6, 0, 1)), (2, (0, 1, 0, 9)), (2, (0, 4, 0, 0))):
        at = []
        for sign in (1, -1):
            a = [t.clone() for t in (q, k, v)]
            a[n][index] += sign * h
            at.append(loss(a))
        assert abs((at[0] - at[1]) / (2 * h) - grads[n][index].item()) < 2e-3, (n, index)


# ------------------------------------------------------------------------------ on the GPU
GPU_CASES = {
    "f32": (2, 300, 300, 4, 2, 64, "f32", "packed", {}),
    "f32_128": (1, 257, 400, 4, 1, 128, "f32", "own", {}),
    "f32_96": (1, 129, 129, 2, 2, 72, "f32", "heads", {}),
    "bf16_64": (3, 515, 515, 4, 4, 64, "bf16", "packed", dict(lengths=[515, 77, 0])),
    "bf16_96": (2, 260, 333, 4, 2, 96, "bf16", "heads", {}),
    "bf16_128": (1, 1027, 1027, 4, 1, 128, "bf16", "packed", {}),
    "f16_64": (2, 383, 383, 2, 1, 64, "f16", "packed", {}),
    "f16_128": (1, 640, 640, 2, 2, 128, "f16", "cache", {}),
    "f16_80": (2, 515, 515, 4, 1, 80, "f16", "packed", dict(lengths=[515, 200])),
    "bf16_32": (2, 200, 200, 8, 2, 32, "bf16", "packed", {}),
    "odd_bf16": (2, 200, 231, 3, 1, 103, "bf16", "odd", {}),
    "odd_f32": (1, 140, 140, 2, 2, 33, "f32", "odd", {}),
    "odd_f16": (1, 140, 300, 2, 2, 1, "f16", "odd", {}),
    "shared": (4, 140, 140, 4, 2, 64, "bf16", "shared", {}),
    "full": (2, 130, 500, 2, 1, 64, "bf16", "own", dict(causal=False, lengths=[500, 129])),
    "early_rows_see_nothing": (2, 300, 100, 2, 1, 64, "bf16", "own", {}),
    "prefill": (2, 61, 3100, 4, 2, 128, "bf16", "cache", dict(lengths=[3100, 2000], starts=[3039, 1939])),
    "prefill_f32": (1, 50, 2100, 4, 2, 64, "f32", "cache", {}),
    "step": (5, 1, 4000, 8, 2, 128, "bf16", "cache", dict(lengths=[4000, 1, 0, 127, 2049], starts=[3999, 0, -1, 126, 2048])),
    "step_f16": (1, 1, 20000, 4, 4, 64, "f16", "own", {}),
    "step_f32": (2, 1, 5000, 32, 1, 128, "f32", "own", {}),
    "step_odd": (2, 1, 700, 6, 2, 45, "bf16", "odd", {}),
    "four_steps": (2, 4, 1500, 16, 2, 96, "bf16", "own", {}),
    "many_heads_share": (1, 3, 300, 64, 1, 64, "f16", "own", {}),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(GPU_CASES))
def test_gpu(name):
    *sizes, dtype, layout, o = GPU_CASES[name]
    check(*inputs(*sizes, dtype, layout=layout, seed=len(name)), **options(o), device="cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_gpu_large_scores(dtype):
    """Scores of some hundreds: the maximum is taken out before the exponential, nothing overflows."""
    q, k, v, go = inputs(1, 200, 200, 2, 1, 64, dtype, seed=2, gain=4.0)
    check(q, k, v, go, scale=0.5 if dtype == "f32" else 0.25, device="cuda")


@pytest.mark.gpu
def test_gpu_offsets_past_32_bits():
    """Heads first, and a cache whose sequences lie further apart than 32 bits of bytes reach."""
    T = 1100000
    k = torch.zeros(2, 8, T, 128, dtype=torch.bfloat16, device="cuda")           # 2.2 GB a sequence
    k.view(-1)[::3] = 1.0
    q = torch.zeros(2, 1, 8, 128, dtype=torch.bfloat16, device="cuda")
    kt = k.transpose(1, 2)
    n, at = 300, T - 300
    k[1, 7, at:] = torch.randn(n, 128, generator=torch.Generator().manual_seed(0)).bfloat16().cuda()
    q[1, 0, 7] = 1.0
    out = A.attention_forward(q, kt[:, at:], kt[:, at:])[0]
    (want,), (bound,) = O.attention(q[1:, :, 7:].cpu(), kt[1:, at:, 7:].cpu(), kt[1:, at:, 7:].cpu())
    compare((out[1:, :, 7:],), (want,), (bound,), "far")


@pytest.mark.gpu
def test_gpu_stream_and_graph():
    """On another stream than the default one, and captured: every replay computes from what its inputs hold then."""
    q, k, v, go = (t.cuda() for t in inputs(2, 1, 3000, 8, 2, 64, "bf16"))
    q2, k2, v2, go2 = (t.cuda() for t in inputs(1, 260, 260, 2, 1, 64, "bf16"))
    lengths = torch.tensor([3000, 100], dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()

    def work():
        left = A.attention_forward(q2, k2, v2, want_lse=True)
        return (A.attention_forward(q, k, v, lengths, lengths - 1)[0], left[0], *A.attention_backward(go2, q2, k2, v2, *left))
    want = [t.clone() for t in work()]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = work()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = work()
    for step in range(3):
        q.mul_(0.5)
        q2.add_(0.25)
        lengths.add_(7)
        lengths.clamp_(max=3000)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(work(), held)), step


@pytest.mark.gpu
def test_gpu_autograd_and_compile():
    q, k, v, go = inputs(2, 150, 150, 4, 2, 64, "bf16", layout="packed")
    want, bounds = O.attention(q, k, v, go)
    leaf = [t.cuda().requires_grad_() for t in (q, k, v)]
    for f in (A.attention, torch.compile(lambda q, k, v: A.attention(q, k, v), fullgraph=True, backend="aot_eager")):
        out = f(*leaf)
        compare((out.detach(), *torch.autograd.grad(out, leaf, go.cuda())), want, bounds, f)
    with torch.no_grad():
        assert torch.equal(f(*leaf), A.attention_forward(*leaf)[0])
