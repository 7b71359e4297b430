"""Layer norm against its formula in 64 bits: the kernels' source on the CPU, and the built library on the GPU."""
import pytest
import torch
from torch import nn

from analog_moe_amd import norm as N
from oracle import norm_oracle as O
from tests.test_attention import DT, _on_gpu
from tests.test_emu_kernels import emu_ops  # noqa: F401


def test_a_gpu_is_needed():
    with pytest.raises(RuntimeError, match="GPU"):
        N.layer_norm(torch.zeros(2, 8))


def inputs(rows, D, dtype, residual=True, wdtype=None, layout="own", seed=0, off=0.3, size=1.0):
    """x, residual, w, b, gy, gs.  layout: "own" tensors, "part" of wider rows, "odd" offsets, "every" second row, "spread" gradients of
    one element; the stream has channels that are larger than others and is `off` of its spread from zero."""
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)                                          # noqa: E731

    def place(t):
        t = t.to(DT[dtype])
        if layout == "part":
            return torch.cat((t, torch.full((rows, 24), float("nan")).to(t)), 1)[:, :D]
        if layout == "odd":
            return torch.cat((torch.full((rows, 3), float("nan")).to(t), t, t[:, :2]), 1)[:, 3:3 + D]
        if layout == "every":
            return torch.stack((t, t + float("nan")), 1).reshape(2 * rows, D)[::2]
        return t
    stream = (n(rows, D) + off) * (n(D) * 0.7).exp() * size
    x, r = (place(n(rows, D) * 0.5 * size), place(stream)) if residual else (place(stream), None)
    wt = DT[wdtype or dtype]
    w, b = (n(D) * 0.3 + 1).to(wt), (n(D) * 0.2).to(wt)
    gy, gs = place(n(rows, D)), place(n(rows, D)) if residual else None
    if layout == "spread":
        gy = torch.tensor(0.75).to(DT[dtype]).expand(rows, D)
    return x, r, w, b, gy, gs


def compare(got, want, dtype, what):
    for name, t in got.items():
        value, bound = want[name]
        t = t.cpu()
        assert t.shape == value.shape and torch.isfinite(t).all(), (what, name)
        bound = bound + O.rounding(value, t.dtype)
        worst = ((t.double() - value).abs() / bound).max().item() if t.numel() else 0.0
        assert worst <= 1.0, (what, name, worst)


def check(x, r, w, b, gy, gs, eps=1e-5, device="cpu"):
    s = x if r is None else (x.float() + r.float()).to(x.dtype)
    want = O.layer_norm(s, w, b, eps, gy, gs)
    to = lambda t: None if t is None else t if device == "cpu" else _on_gpu(t)          # noqa: E731
    x, r, w, b, gy, gs = map(to, (x, r, w, b, gy, gs))
    y, left, stats = N.layer_norm_forward(x, w, b, eps, r, want_stats=True)
    assert (left is None) == (r is None) and (r is None or torch.equal(left.cpu(), s))
    assert torch.equal(y, N.layer_norm_forward(x, w, b, eps, r)[0])
    grads = N.layer_norm_backward(gy, x if r is None else left, w, b, stats, gs)
    got = dict(y=y, dx=grads[0])
    got.update({n: t for n, t in zip(("dw", "db"), grads[1:]) if t is not None})
    compare(got, want, x.dtype, tuple(x.shape))
    again = N.layer_norm_backward(gy, x if r is None else left, w, b, stats, gs)
    assert all(a is c or torch.equal(a, c) for a, c in zip(grads, again))
    if device == "cpu" and x.shape[1] > 600:             # (the host build takes seconds for each)
        return
    for wants in ((True, False, False), (False, True, False), (False, False, True)):
        part = N.layer_norm_backward(gy, x if r is None else left, w, b, stats, gs, *wants)
        for a, c, there in zip(part, grads, wants):
            assert (a is None) == (not there or c is None) and (a is None or torch.equal(a, c))


CASES = {
    # rows, D, dtype, options of inputs
    "one": (1, 8, "f32", {}),
    "one_element": (3, 1, "f32", {}),
    "tiny_bf16": (21, 64, "bf16", {}),
    "tiny_odd_f16": (35, 13, "f16", dict(layout="odd")),
    "wave_bf16": (9, 512, "bf16", dict(residual=False)),
    "wave_f32": (6, 256, "f32", {}),
    "two_bf16": (5, 1024, "bf16", dict(wdtype="f32")),
    "ragged_f16": (6, 412, "f16", dict(residual=False)),
    "odd_bf16": (5, 727, "bf16", dict(layout="odd")),
    "part_bf16": (9, 1000, "bf16", dict(layout="part", wdtype="f32")),
    "every_f32": (9, 96, "f32", dict(layout="every")),
    "spread_f16": (9, 96, "f16", dict(layout="spread")),
    "four_f32": (3, 1021, "f32", dict(layout="odd")),
    "four_bf16": (3, 2048, "bf16", {}),
    "group_f32": (2, 2801, "f32", dict(layout="odd")),
    "far_f32": (4, 300, "f32", dict(off=5000.0, residual=False)),
    "large_bf16": (4, 300, "bf16", dict(size=1e4)),
    "small_f32": (4, 300, "f32", dict(size=1e-4)),
}


@pytest.mark.parametrize("name", list(CASES))
def test_emulated(emu_ops, name):
    rows, D, dtype, o = CASES[name]
    check(*inputs(rows, D, dtype, seed=len(name), **o))


def test_without_weights(emu_ops):
    x, r, w, b, gy, gs = inputs(5, 40, "bf16")
    check(x, r, None, None, gy, gs)
    check(x, r, w, None, gy, gs)
    check(x, r, None, b.float(), gy, gs, eps=0.0)


def test_rows_of_one_value(emu_ops):
    """No spread: h is 0 whatever the value, y the bias, and the gradient that of the formula (inv = 1 / sqrt(eps))."""
    x = torch.full((3, 48), 7.3)
    x[1] = 0.0
    x[2] = -3e4
    _, _, w, b, gy, _ = inputs(3, 48, "f32")
    y, _, stats = N.layer_norm_forward(x, w, b, want_stats=True)
    assert torch.equal(y, b.expand(3, 48))
    check(x, None, w, b, gy, None)


def check_large_rows(cases, device="cpu"):
    """Rows of one value of 2e36 (no spread, so nothing overflows), at widths that leave lanes without columns: h is 0, y the bias, and what lanes
    without columns hold adds nothing."""
    to = lambda t: t if device == "cpu" else _on_gpu(t)                                   # noqa: E731
    for D, dtype in cases:
        x = torch.full((3, D), 2e36).bfloat16().to(DT[dtype])        # (8 bits: sums of 2^15 of them are exact in fp32)
        x[1] = -x[1]
        _, _, w, b, gy, _ = inputs(3, D, dtype, seed=D)
        _, _, stats = N.layer_norm_forward(to(x), to(w), to(b), want_stats=True)
        assert torch.equal(stats[:, 0].cpu(), x[:, 0].float()) and not stats[:, 1].any(), (D, dtype)
        check(x, None, w, b, gy, None, device=device)


def test_large_rows_of_one_value(emu_ops):
    check_large_rows([(9, "f32"), (16, "f32"), (100, "f32"), (9, "bf16"), (12, "bf16"), (16, "bf16"), (100, "bf16")])


def test_large_sums(emu_ops):
    """Rows whose sum no float holds, of one value and of small differences."""
    check_large_rows([(512, "f32"), (1000, "bf16")])
    x = torch.full((2, 300), -2.0 ** 126)
    x[1, ::2] = 2.0 ** 126
    y, _, stats = N.layer_norm_forward(x[:1], want_stats=True)
    assert not y.any() and stats[0, 0] == -2.0 ** 126
    # (differences whose squares are past the floats' range, as documented: no spread is too large for the mean)
    assert N.layer_norm_forward(x, want_stats=True)[2][1, 0] == 0


@pytest.mark.gpu
def test_gpu_large_rows():
    check_large_rows([(D, t) for D in (9, 16, 100, 412, 1024, 4096, 8192, 16384, 32768) for t in ("f32", "bf16")], "cuda")


def test_no_rows(emu_ops):
    x, w = torch.empty(0, 5, 16), torch.ones(16, requires_grad=True)
    assert N.layer_norm(x).shape == (0, 5, 16)
    y = N.layer_norm(x.requires_grad_(), w)
    gx, gw = torch.autograd.grad(y.sum(), (x, w))
    assert gx.shape == x.shape and not gw.any()


def test_rows_that_are_not_numbers_stay_alone(emu_ops):
    x, r, w, b, gy, gs = inputs(9, 64, "bf16")
    clean = N.layer_norm_forward(x, w, b, residual=r)[0]
    x = x.clone()
    x[4, 7], x[8, 0] = float("nan"), float("inf")
    y = N.layer_norm_forward(x, w, b, residual=r)[0]
    keep = [i for i in range(9) if i not in (4, 8)]
    assert torch.equal(y[keep], clean[keep]) and y[4].isnan().all() and y[8].isnan().all()


def test_strides_and_dimensions(emu_ops):
    x, r, w, b, _, _ = inputs(12, 32, "f32")
    want, s = N.layer_norm(x, w, b, residual=r)
    y, s3 = N.layer_norm(x.reshape(3, 4, 32), w, b, residual=r.reshape(3, 4, 32))
    assert torch.equal(y.reshape(12, 32), want) and torch.equal(s3.reshape(12, 32), s)
    y, _ = N.layer_norm(x.t().contiguous().t(), w, b, residual=r.reshape(4, 3, 32).transpose(0, 1).contiguous().transpose(0, 1).reshape(12, 32))
    assert torch.equal(y, want)
    assert torch.equal(N.layer_norm(x[3], w, b), N.layer_norm(x, w, b)[3])
    row = x[5].expand(7, 32)
    assert torch.equal(N.layer_norm(row, w, b), N.layer_norm(row.clone(), w, b))
    wide = torch.randn(2 * 32)
    assert torch.equal(N.layer_norm(x, wide[::2], b), N.layer_norm(x, wide[::2].contiguous(), b))


def test_types_of_the_summands(emu_ops):
    """A 16-bit sublayer's output on a float32 stream, as under autocast: both in the wider type."""
    x, r, w, b, gy, gs = inputs(5, 48, "bf16", wdtype="f32")
    r = r.float().requires_grad_()
    x = x.clone().requires_grad_()
    y, s = N.layer_norm(x, w, b, residual=r)
    assert y.dtype == s.dtype == torch.float32 and torch.equal(s.detach(), x.detach().float() + r.detach())
    gx, gr = torch.autograd.grad((y, s), (x, r), (gy.float(), gs.float()))
    assert gx.dtype == torch.bfloat16 and torch.equal(gr.to(torch.bfloat16), gx)


def test_autograd(emu_ops):
    x, r, w, b, gy, gs = (t.requires_grad_() for t in inputs(7, 40, "f32"))
    want = O.layer_norm((x + r).detach(), w.detach(), b.detach(), 1e-5, gy.detach(), gs.detach())
    y, s = N.layer_norm(x, w, b, residual=r)
    gx, gr, gw, gb = torch.autograd.grad((y, s), (x, r, w, b), (gy.detach(), gs.detach()))
    compare(dict(y=y.detach(), dx=gx, dw=gw, db=gb), want, x.dtype, "both")
    assert torch.equal(gx, gr)
    # the sum alone is used, the norm alone is used, one of four is wanted
    y, s = N.layer_norm(x, w, b, residual=r)
    gx, gw = torch.autograd.grad(s, (x, w), gs.detach())
    assert torch.equal(gx, gs) and not gw.any()
    y, s = N.layer_norm(x, w.detach(), b.detach(), residual=r)
    (gr,) = torch.autograd.grad(y, r, gy.detach())
    compare(dict(dx=gr), O.layer_norm((x + r).detach(), w.detach(), b.detach(), 1e-5, gy.detach()), x.dtype, "norm alone")
    y, _ = N.layer_norm(x.detach(), w, b.detach(), residual=r.detach())
    (gw,) = torch.autograd.grad(y, w, gy.detach())
    compare(dict(dw=gw), want, x.dtype, "weight alone")
    # leaves' gradients are tensors of their own
    y, s = N.layer_norm(x, w, b, residual=r)
    (y * 2 + s).sum().backward()
    assert x.grad.data_ptr() != r.grad.data_ptr() and torch.equal(x.grad, r.grad)
    (gx,) = torch.autograd.grad(N.layer_norm(x, w, b).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        (gx.sum() + x.sum()).backward()
    with torch.no_grad():
        assert torch.equal(N.layer_norm(x, w, b), N.layer_norm_forward(x, w, b)[0])


def test_watched_calls(emu_ops):
    from torch.autograd import forward_ad
    x, r, w, b, _, _ = inputs(4, 16, "f32")
    with torch.no_grad(), forward_ad.dual_level(), pytest.raises(NotImplementedError):
        N.layer_norm(forward_ad.make_dual(x, x), w, b)
    with torch.no_grad(), pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: N.layer_norm(t, w, b))(x[None])
    with torch.no_grad():
        traced = torch.jit.trace(lambda t: N.layer_norm(t, w, b, residual=r)[0], (x,), check_trace=False)
        assert torch.equal(traced(r), N.layer_norm(r, w, b, residual=r)[0])


def test_gradients_are_differences(emu_ops):
    """Against central differences of the loss sum(y * gy + s * gs) with step h: the formula's own difference says what the step
    does, and the two losses are off by what the bounds allow y."""
    x, r, w, b, gy, gs = inputs(3, 24, "f32", seed=2)
    y, s, stats = N.layer_norm_forward(x, w, b, residual=r, want_stats=True)
    grads = N.layer_norm_backward(gy, s, w, b, stats, gs)
    h = 2.0 ** -6

    def loss(x, w, b):
        y, s, _ = N.layer_norm_forward(x, w, b, residual=r)
        return (y.double() * gy.double() + s.double() * gs.double()).sum().item()

    def formula(x, w, b):
        y, off = O.layer_norm(x + r, w, b)["y"]
        s = (x + r).double()
        off = ((off + O.rounding(y, torch.float32)) * gy.double().abs() + 2.0 ** -24 * (s * gs.double()).abs()).sum().item()
        return (y * gy.double() + s * gs.double()).sum().item(), off
    for n, index in ((0, (0, 3)), (0, (2, 23)), (1, (0,)), (1, (17,)), (2, (5,)), (2, (23,))):
        got, want, off = [], [], 0.0
        for sign in (1, -1):
            a = [t.clone() for t in (x, w, b)]
            a[n][index] += sign * h
            got.append(loss(*a))
            f, o = formula(*a)
            want.append(f)
            off += o
        step = abs((want[0] - want[1]) / (2 * h) - O.layer_norm(s, w, b, 1e-5, gy, gs)[("dx", "dw", "db")[n]][0][index].item())
        g = O.layer_norm(s, w, b, 1e-5, gy, gs)[("dx", "dw", "db")[n]][1][index].item()
        assert abs((got[0] - got[1]) / (2 * h) - grads[n][index].item()) <= off / (2 * h) + step + g + 1e-6, (n, index)


def test_module(emu_ops):
    """Parameters and state dict of nn.LayerNorm, its values to the type's rounding."""
    m, like = N.LayerNorm(48, eps=1e-3), nn.LayerNorm(48, eps=1e-3)
    with torch.no_grad():
        like.weight.mul_(1.5)
        like.bias.add_(0.25)
    m.load_state_dict(like.state_dict())
    x, r, _, _, _, _ = inputs(6, 48, "f32")
    assert (m(x) - like(x)).abs().max() <= 2.0 ** -18 * like(x).abs().max()
    y, s = m(x, r)
    assert torch.equal(s, x + r) and torch.equal(y, m(x + r))
    assert N.LayerNorm(8, bias=False).bias is None and N.LayerNorm(8, elementwise_affine=False).weight is None
    with pytest.raises(ValueError):
        N.LayerNorm(0)


def test_types_of_the_module(emu_ops):
    """Autocast changes nothing, and parameters of a 16-bit module do not go with a float32 stream."""
    x, r, _, _, _, _ = inputs(5, 48, "bf16")
    m = N.LayerNorm(48)
    with torch.autocast("cpu", torch.bfloat16):
        assert m(x).dtype == torch.bfloat16 and m(x.float()).dtype == torch.float32 and m(x, r.float())[0].dtype == torch.float32
        assert torch.equal(m(x), N.layer_norm(x, m.weight, m.bias))
    m = m.bfloat16()
    assert m(x, r)[0].dtype == torch.bfloat16
    with pytest.raises(TypeError):
        m(x, r.float())


def test_refusals(emu_ops):
    x, r, w, b, gy, _ = inputs(4, 16, "bf16")
    for bad in (dict(weight=w[:8]), dict(bias=b.reshape(1, 16)), dict(residual=r[:2]), dict(eps=-1.0), dict(eps=float("nan")),
                dict(eps=float("inf"))):
        with pytest.raises(ValueError):
            N.layer_norm(x, **bad)
    with pytest.raises(ValueError):
        N.layer_norm(torch.zeros(2, 32769))
    with pytest.raises(ValueError):
        N.layer_norm(torch.zeros(2, 0))
    with pytest.raises(ValueError):
        N.layer_norm(torch.tensor(1.0))
    for bad in (dict(weight=w.half()), dict(weight=w.double()), dict(weight=w, bias=b.float())):
        with pytest.raises(TypeError):
            N.layer_norm(x, **bad)
    with pytest.raises(TypeError):
        N.layer_norm(x.double())
    _, _, stats = N.layer_norm_forward(x, w, b, want_stats=True)
    for args in ((gy[:2], x, w, b, stats), (gy.float(), x, w, b, stats), (gy, x, w, b, stats[:3]), (gy, x, w, b, stats.double())):
        with pytest.raises(ValueError):
            N.layer_norm_backward(*args)


def test_library_refuses(emu_ops):
    """The C entries by themselves: sizes, missing and odd pointers, a workspace that is too small.  Nothing is launched."""
    from analog_moe_amd import _abi
    lib = emu_ops.get_lib()
    x, w = torch.zeros(4, 16), torch.zeros(16)
    stats = torch.zeros(4, 3)
    p = x.data_ptr()

    def call(which="fwd", ws=None, n=0, **k):
        f = dict(dtype=0, wdtype=0, rows=4, D=16, eps=1e-5, x=p, ldx=16, w=w.data_ptr(), b=0, stats=stats.data_ptr(), r=0, ldr=0, y=p, s=0,
                 gy=p, ldgy=16, gs=0, ldgs=0, dx=p, dw=0, db=0)
        f.update(k)
        args = _abi.NORM_ARGS.pack(*f.values())
        return lib.amoe_layer_norm_fwd(args, None) if which == "fwd" else lib.amoe_layer_norm_bwd(args, ws, n, None)
    assert call() == 0 and call("bwd") == 0 and call(rows=0, x=0) == 0
    for k in (dict(dtype=3), dict(wdtype=1), dict(rows=-1), dict(D=0), dict(eps=-1.0), dict(eps=float("nan")), dict(ldx=-1)):
        assert call(**k) == -1, k
    assert call(D=32769) == call(rows=1 << 31) == call(rows=1 << 28) == call(rows=1 << 26, D=512, ldx=512) == call(rows=1 << 22, D=20000, ldx=20000) == -6
    assert call(x=0) == call(y=0) == call(r=p) == call(s=p) == -2 and call("bwd", gy=0) == call("bwd", stats=0) == -2
    assert call(x=p + 2) == call(w=w.data_ptr() + 1) == call(stats=stats.data_ptr() + 2) == -4
    dw = torch.zeros(16)
    assert call("bwd", dw=dw.data_ptr()) == -2
    ws = torch.zeros(4096)
    assert call("bwd", ws.data_ptr(), 8, dw=dw.data_ptr()) == -5
    assert call("bwd", ws.data_ptr() + 2, 8192, dw=dw.data_ptr()) == -4
    assert call("bwd", ws.data_ptr(), 8192, dw=dw.data_ptr()) == 0
    assert call("bwd", rows=0, dw=dw.data_ptr()) == -1
    assert lib.amoe_layer_norm_fwd(None, None) == -2


def test_operators_on_meta():
    x = torch.empty(3, 5, 16, device="meta", dtype=torch.bfloat16, requires_grad=True)
    r = torch.empty(3, 5, 16, device="meta", dtype=torch.bfloat16, requires_grad=True)
    w = torch.empty(16, device="meta", requires_grad=True)
    y, s, stats = torch.ops.amoe.layer_norm_fwd(x, r, w, None, 1e-5)
    assert y.shape == s.shape == x.shape and stats.shape == (15, 3) and stats.dtype == torch.float32
    gx, gr, gw = torch.autograd.grad((y, s), (x, r, w), (torch.empty_like(y), torch.empty_like(s)))
    assert gx.shape == gr.shape == x.shape and gw.shape == (16,) and gw.dtype == torch.float32
    y, s, _ = torch.ops.amoe.layer_norm_fwd(x, None, None, None, 1e-5)
    assert s.numel() == 0 and torch.autograd.grad(y.sum(), x)[0].shape == x.shape


# ------------------------------------------------------------------------------ on the GPU
GPU_CASES = dict(CASES, **{
    "group_bf16": (3, 4096, "bf16", {}),
    "wide_f16": (2, 5001, "f16", dict(residual=False)),
    "many_bf16": (3001, 1024, "bf16", {}),
    "many_f32": (2003, 512, "f32", dict(layout="part")),
    "many_f16": (5003, 412, "f16", dict(residual=False)),
    "many_tiny": (20011, 62, "bf16", {}),
    "many_odd": (777, 1131, "f16", dict(layout="odd")),
    "group_many": (1025, 4096, "bf16", dict(wdtype="f32")),
    "group_four": (300, 8192, "f16", {}),
    "group_four_f32": (300, 4096, "f32", {}),
    "wide_bf16": (601, 16384, "bf16", {}),
    "wide_odd": (40, 12345, "bf16", dict(layout="odd")),
    "wide_f32": (130, 8192, "f32", {}),
    "wider_f32": (33, 16384, "f32", {}),
    "widest_bf16": (20, 32768, "bf16", {}),
    "widest_f32": (20, 32768, "f32", {}),
    "widest_odd_f32": (5, 32767, "f32", dict(layout="odd")),
})


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(GPU_CASES))
def test_gpu(name):
    rows, D, dtype, o = GPU_CASES[name]
    check(*inputs(rows, D, dtype, seed=len(name), **o), device="cuda")


@pytest.mark.gpu
def test_gpu_offsets_past_32_bits():
    """Rows of one element each 2^26 apart: the last ones lie past 2^32 bytes, and past 2^32 elements in 16 bits."""
    rows, D, ld = 70, 24, 1 << 26
    base = torch.empty((rows - 1) * ld + D, dtype=torch.bfloat16, device="cuda")
    x = base.as_strided((rows, D), (ld, 1))
    own, _, w, b, gy, _ = inputs(rows, D, "bf16", residual=False)
    x.copy_(own)
    y, _, stats = N.layer_norm_forward(x, w.cuda(), b.cuda(), want_stats=True)
    grads = N.layer_norm_backward(gy.cuda(), x, w.cuda(), b.cuda(), stats)
    compare(dict(y=y, dx=grads[0], dw=grads[1], db=grads[2]), O.layer_norm(own, w, b, 1e-5, gy), x.dtype, "far")


@pytest.mark.gpu
def test_gpu_stream_and_graph():
    """On another stream than the default one, and captured: every replay computes from what its inputs hold then."""
    x, r, w, b, gy, gs = (t.cuda() for t in inputs(601, 1024, "bf16"))
    side = torch.cuda.Stream()

    def work():
        y, s, stats = N.layer_norm_forward(x, w, b, residual=r, want_stats=True)
        return (y, s, *N.layer_norm_backward(gy, s, w, b, stats, gs))
    want = [t.clone() for t in work()]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = work()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = work()
    for step in range(3):
        x.mul_(0.5)
        gy.add_(0.25)
        w.add_(0.125)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(work(), held)), step


@pytest.mark.gpu
def test_gpu_autograd_and_compile():
    x, r, w, b, gy, gs = inputs(150, 256, "bf16")
    want = O.layer_norm((x.float() + r.float()).to(x.dtype), w, b, 1e-5, gy, gs)
    leaf = [t.cuda().requires_grad_() for t in (x, r, w, b)]

    def plain(x, r, w, b):
        return N.layer_norm(x, w, b, residual=r)
    for f in (plain, torch.compile(plain, fullgraph=True, backend="aot_eager")):
        y, s = f(*leaf)
        gx, gr, gw, gb = torch.autograd.grad((y, s), leaf, (gy.cuda(), gs.cuda()))
        compare(dict(y=y.detach(), dx=gx, dw=gw, db=gb), want, x.dtype, f)
        assert torch.equal(gx, gr)
