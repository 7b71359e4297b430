"""Rotary positions against their formula in 64 bits: the kernel's source on the CPU, and the built library on the GPU."""
import pytest
import torch

from analog_moe_amd import rotary as R
from oracle import attention_oracle as O
from tests.test_attention import DT, _on_gpu
from tests.test_emu_kernels import emu_ops  # noqa: F401


def inputs(B, S, H, G, d, dtype, layout="own", seed=0):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g).to(DT[dtype])          # noqa: E731
    if layout == "packed":
        w = n(B, S, H + 2 * G, d)
        return w[:, :, :H], w[:, :, H:H + G]
    if layout == "heads":
        return n(B, H, S, d).transpose(1, 2), n(B, G, S, d).transpose(1, 2)
    if layout == "odd":
        return n(B, S, H, d + 3)[..., 1:d + 1], n(B, S, G, d + 1)[..., :d]
    return n(B, S, H, d), n(B, S, G, d)


def places(kind, B, S):
    g = torch.Generator().manual_seed(S)
    if kind is None:
        return None, torch.arange(S).expand(B, S)
    if kind == "one":
        p = torch.randint(0, 1 << 20, (S,), generator=g)
        return p, p.expand(B, S)
    if kind == "each32":
        p = torch.randint(-(1 << 20), 1 << 20, (B, S), generator=g, dtype=torch.int32)
        return p, p.long()
    p = torch.randint(0, 1 << 20, (S, B), generator=g).t()              # (any strides)
    return p, p


def check(sizes, dtype, layout, kind, device="cpu", start=0, **how):
    B, S, _, _, d = sizes
    dim = how.pop("dim", d)
    q, k = inputs(*sizes, dtype, layout, seed=d + S)
    given, at = places(kind, B, S)
    r = R.Rotary(dim, **how)
    theta = R._angles(dim, how.get("base", 10000.0), how.get("scaling", "none"), how.get("factor", 1.0), how.get("trained_context"))
    if device == "cuda":
        r, q, k, given = r.to(torch.bfloat16).cuda(), _on_gpu(q), _on_gpu(k), None if given is None else _on_gpu(given)
        assert r.turns.dtype == torch.int64
    with torch.no_grad():
        turned = r(q, k, given, start)
    back = R.rotate(*turned, r.turns, given, start, r.interleaved, r.size, inverse=True)
    for x, y, z in zip((q, k), turned, back):
        for a, b, inv in ((x, y, False), (y, z, True)):
            want, bound = O.rotary(a.cpu(), theta, at + start, r.interleaved, r.size, inv)
            assert b.shape == a.shape and b.is_contiguous()
            err = (b.cpu().double() - want).abs()
            assert (err <= bound).all(), (err / bound.clamp_min(1e-300)).max()


CASES = {
    "halves": ((2, 5, 3, 1, 64), "bf16", "packed", "each", {}),
    "halves_f16": ((1, 9, 2, 2, 32), "f16", "heads", None, {}),
    "side_by_side": ((2, 4, 2, 1, 64), "f32", "own", "one", dict(interleaved=True)),
    "part": ((1, 7, 4, 2, 128), "bf16", "own", "each32", dict(dim=64, base=500000.0)),
    "part_side_by_side": ((1, 6, 2, 1, 96), "f16", "packed", "each", dict(dim=48, interleaved=True)),
    "odd": ((2, 3, 2, 1, 13), "bf16", "odd", "each", dict(dim=10)),
    "odd_side_by_side": ((2, 3, 2, 1, 7), "f32", "odd", "one", dict(dim=2, interleaved=True)),
    "linear": ((1, 5, 1, 1, 64), "f32", "own", "each", dict(scaling="linear", factor=4.0)),
    "base": ((1, 5, 1, 1, 64), "f32", "own", "each", dict(scaling="base", factor=4.0)),
    "parts": ((1, 5, 1, 1, 128), "f32", "own", "each", dict(scaling="parts", factor=8.0, trained_context=2048)),
    "one_token": ((1, 1, 1, 1, 2), "f32", "own", None, {}),
    "from": ((2, 3, 2, 2, 64), "bf16", "own", None, dict(start=999999)),
}


@pytest.mark.parametrize("name", list(CASES))
def test_emulated(emu_ops, name):
    sizes, dtype, layout, kind, how = CASES[name]
    check(sizes, dtype, layout, kind, **how)


GPU_CASES = dict(CASES, **{
    "many": ((3, 1001, 16, 4, 64), "bf16", "packed", "each", {}),
    "many_f16": ((1, 3001, 8, 8, 128), "f16", "own", None, dict(dim=64, interleaved=True, start=500000)),
    "many_f32": ((2, 517, 6, 2, 80), "f32", "heads", "each32", dict(scaling="parts", factor=16.0, trained_context=4096)),
    "many_odd": ((2, 517, 3, 1, 103), "bf16", "odd", "each", dict(dim=102)),
    "one_each": ((64, 1, 32, 8, 128), "bf16", "own", "each", {}),
    "wide": ((1, 40, 1, 1, 2048), "bf16", "own", "each", {}),
})


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(GPU_CASES))
def test_gpu(name):
    sizes, dtype, layout, kind, how = GPU_CASES[name]
    check(sizes, dtype, layout, kind, device="cuda", **how)


def test_far_positions_keep_their_angle(emu_ops):
    """The angle is an integer product modulo one revolution: 2^40 positions on, a pair that turns 1 / 2^k revolutions per
    position stands where it stood."""
    q, k = inputs(1, 4, 1, 1, 8, "f32")
    turns = torch.tensor([2 ** 54, 2 ** 40, 2 ** 30, 2 ** 24], dtype=torch.int64)
    near, far = (R.rotate(q, k, turns, torch.arange(4) + at) for at in (5, 5 + 2 ** 40))
    assert torch.equal(near[0], far[0]) and torch.equal(near[1], far[1])


def test_scalings():
    """What each scaling promises of the fastest and the slowest pair."""
    plain = R._angles(64, 10000.0, "none", 1.0, None)
    assert plain[0] == 1.0 and abs(plain[-1] - 10000.0 ** (-62 / 64)) < 1e-18
    assert R._angles(64, 10000.0, "linear", 4.0, None) == [t / 4 for t in plain]
    grown = R._angles(64, 10000.0, "base", 4.0, None)
    assert grown[0] == 1.0 and abs(grown[-1] / plain[-1] - 0.25) < 1e-12
    parts = R._angles(64, 10000.0, "parts", 4.0, 1000)
    assert parts[0] == plain[0] and abs(parts[-1] / plain[-1] - 0.25) < 1e-12
    assert all(a <= b and a >= b / 4 - 1e-18 for a, b in zip(parts, plain))
    for scaling in R.SCALINGS:
        assert R.Rotary(2, scaling=scaling, factor=2.0, trained_context=9).turns.tolist()[0] > 0


def test_into_a_cache_and_in_place(emu_ops):
    q, k = inputs(2, 3, 2, 1, 64, "bf16")
    r = R.Rotary(64)
    with torch.no_grad():
        want = r(q, k, start=4)
        cache = torch.zeros(2, 10, 1, 64, dtype=torch.bfloat16)
        r(q, k, start=4, out=(q, cache[:, 4:7]))
    assert torch.equal(q, want[0]) and torch.equal(cache[:, 4:7], want[1])
    assert not cache[:, :4].any() and not cache[:, 7:].any()


def test_gradient(emu_ops):
    q, k = (t.requires_grad_() for t in inputs(1, 5, 2, 1, 32, "f32"))
    gq, gk = inputs(1, 5, 2, 1, 32, "f32", seed=4)
    r = R.Rotary(16, scaling="parts", factor=4.0, trained_context=100)
    out = r(q, k, start=3)
    dq, dk = torch.autograd.grad(out, (q, k), (gq, gk), retain_graph=True)
    # the operator is linear and its gradient its transpose: <A x, g> = <x, A' g>; 160 products of fp32 results that are
    # off by 9 * 2^-24 of |a| + |b| at most
    for x, y, g, dx in ((q, out[0], gq, dq), (k, out[1], gk, dk)):
        a, b = (y.double() * g.double()).sum(), (x.double() * dx.double()).sum()
        assert abs(a - b) < 40 * 2.0 ** -24 * (x.abs().double().sum() * g.abs().max())
    (only,) = torch.autograd.grad(r(q, k.detach(), start=3)[0].sum(), q)
    assert torch.equal(only, R.rotate(torch.ones_like(q), k, r.turns, None, 3, False, r.size, True)[0])
    # differentiable as often as wanted: the gradient is linear in gq, its derivative the turn itself
    gq, gk = gq.requires_grad_(), gk.requires_grad_()
    dq, _ = torch.autograd.grad(r(q, k, start=3), (q, k), (gq, gk), create_graph=True)
    (back,) = torch.autograd.grad(dq, gq, q.detach())
    assert torch.equal(back, R.rotate(q, k, r.turns, None, 3, False, r.size)[0])
    with pytest.raises(RuntimeError):
        r(q, k, out=(torch.empty_like(q), torch.empty_like(k)))


def test_watched_calls(emu_ops):
    from torch.autograd import forward_ad
    q, k = inputs(1, 4, 1, 1, 16, "f32")
    r = R.Rotary(16)
    with torch.no_grad(), forward_ad.dual_level(), pytest.raises(NotImplementedError):
        r(forward_ad.make_dual(q, q), k)
    with torch.no_grad(), pytest.raises(RuntimeError):
        torch.func.vmap(lambda x: r(x, k)[0])(q[None])


def test_refusals(emu_ops):
    for bad in (dict(dim=0), dict(dim=3), dict(dim=2050), dict(dim=8, base=0.5), dict(dim=8, factor=0.5), dict(dim=8, base=float("inf")),
                dict(dim=8, scaling="other"), dict(dim=8, scaling="parts"), dict(dim=8, factor=float("nan"))):
        with pytest.raises(ValueError):
            R.Rotary(**bad)
    q, k = inputs(2, 3, 2, 1, 8, "f32")
    t = R.Rotary(8).turns
    at = torch.arange(3)
    for bad in (lambda: R.rotate(q[0], k, t), lambda: R.rotate(q, k[:, :2], t), lambda: R.rotate(q, k[..., :4], t),
                lambda: R.rotate(q, k, R.Rotary(10).turns), lambda: R.rotate(q, k, t[:0]), lambda: R.rotate(q, k, t, at[:2]),
                lambda: R.rotate(q, k, t, at, 1), lambda: R.rotate(q, k, t, at[None]),
                lambda: R.rotate(q, k, t, out=(q[:1], k)), lambda: R.rotate(q, k, t, out=(q.half(), k)),
                lambda: R.rotate(q, k, t, out=(q[:, :, :1].expand_as(q), k))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: R.rotate(q.double(), k.double(), t), lambda: R.rotate(q, k.half(), t), lambda: R.rotate(q, k, t.float()),
                lambda: R.rotate(q, k, t, at.float()), lambda: R.rotate(q, k, t.repeat(2)[::2])):
        with pytest.raises(TypeError):
            bad()


def test_library_refuses(emu_ops):
    from analog_moe_amd import _abi
    lib = emu_ops.get_lib()
    x = torch.zeros(1, 2, 2, 8)
    t = R.Rotary(8).turns
    good = [0, 1, 2, 2, 2, 8, 8, 0, 0, 1.0, t.data_ptr(), 0, 0, 0, 0, 0] + [x.data_ptr(), *x.stride()[:3]] * 4

    def call(**change):
        a = list(good)
        for i, v in change.items():
            a[int(i[1:])] = v
        return lib.amoe_rotary(_abi.ROTARY_ARGS.pack(*a), None)
    assert call() == 0 and call(_1=0) == 0 and call(_3=0, _16=0) == 0
    assert call(_0=5) == call(_1=-1) == call(_6=7) == call(_6=10) == call(_6=0) == call(_17=-1) == -1
    assert call(_10=0) == call(_16=0) == call(_28=0) == -2
    assert call(_10=t.data_ptr() + 4) == call(_16=x.data_ptr() + 2) == call(_11=t.data_ptr() + 1) == -4
    assert call(_5=4096, _6=4096) == call(_1=2 ** 30, _2=2 ** 20) == call(_1=2 ** 30, _3=256) == -6
    assert lib.amoe_rotary(None, None) == -2


@pytest.mark.gpu
def test_gpu_stream_graph_and_compile():
    r = R.Rotary(64).cuda()
    q, k = (t.cuda() for t in inputs(2, 300, 4, 2, 64, "bf16"))
    at = torch.arange(300, device="cuda")
    with torch.no_grad():
        want = r(q, k, at)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = r(q, k, at)
        torch.cuda.current_stream().wait_stream(side)
        assert all(map(torch.equal, want, got))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = r(q, k, at)
        for _ in range(3):
            at.add_(300)
            graph.replay()
            torch.cuda.synchronize()
            assert all(map(torch.equal, r(q, k, at), held))
    leaf = [t.requires_grad_() for t in (q, k)]
    f = torch.compile(lambda q, k: r(q, k, at), fullgraph=True, backend="aot_eager")
    for g in (r(*leaf, at), f(*leaf)):
        grads = torch.autograd.grad(g, leaf, (q.detach(), k.detach()))
        assert all(map(torch.equal, grads, R.rotate(q.detach(), k.detach(), r.turns, at, inverse=True)))
