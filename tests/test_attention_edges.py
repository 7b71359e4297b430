"""Attention where its numbers leave the ordinary range: the kernels' source on the CPU, and the built library on the GPU."""
import math

import pytest
import torch

from analog_moe_amd import attention as A
from oracle import attention_oracle as O
from tests.test_attention import DT, compare, inputs
from tests.test_emu_kernels import emu_ops  # noqa: F401


def one_hot(q, k, causal, scale):
    """[B, H, S] the key with a row's largest score, and whether it takes the whole row: the others then have less than 2^-127 of
    it, whatever the roundings of a score (d + 8 of 2^-24 of sum|q k|, of both of them) may do."""
    B, S, H, d = q.shape
    T, G = k.shape[1:3]
    Q, K = q.double().transpose(1, 2), k.double().transpose(1, 2).repeat_interleave(H // G, 1)
    s = Q @ K.transpose(2, 3) * scale
    size = Q.abs() @ K.abs().transpose(2, 3) * scale
    if causal:
        hidden = torch.arange(T) > torch.arange(S)[:, None] + T - S
        s, size = s.masked_fill(hidden, -math.inf), size.masked_fill(hidden, 0.0)
    two, top = s.topk(2, dim=-1)
    return top[..., 0], two[..., 0] - two[..., 1] > 2 * (d + 8) * 2.0 ** -24 * size.amax(-1) + 127 * math.log(2)


FAR = {
    # B, S, T, H, G, d, dtype, size of q and k, scale, causal
    "rows_f32": (1, 128, 128, 2, 1, 64, "f32", 1e5, None, True),
    "rows_bf16": (1, 128, 128, 2, 2, 64, "bf16", 1e5, None, False),
    "rows_bf16_128": (1, 70, 300, 2, 1, 128, "bf16", 1e6, None, True),
    "rows_f16": (1, 96, 200, 2, 1, 80, "f16", 1e4, None, True),
    "edges_f32": (1, 40, 90, 1, 1, 13, "f32", 1e9, None, True),
    "scale_f32": (1, 40, 90, 1, 1, 64, "f32", 1.0, 1e30, True),
    "step_f32": (2, 1, 300, 4, 2, 64, "f32", 1e7, None, True),
    "step_f16": (1, 2, 700, 4, 1, 96, "f16", 1e4, 1.0, True),
    "step_bf16": (1, 1, 500, 2, 1, 128, "bf16", 1e10, None, True),
}


def far_inputs(name):
    *sizes, dtype, size, scale, causal = FAR[name]
    q, k, v, go = inputs(*sizes, dtype, seed=len(name))
    q, k = ((t.float() * size).to(DT[dtype]) for t in (q, k))
    return q, k, v, go, causal, 1 / math.sqrt(sizes[5]) if scale is None else scale


def check_far_forward(name, device="cpu"):
    q, k, v, _, causal, scale = far_inputs(name)
    top, sure = one_hot(q, k, causal, scale)
    assert sure.double().mean() > 0.9
    out = A.attention_forward(*(t.to(device) for t in (q, k, v)), causal=causal, scale=scale)[0].cpu().double().transpose(1, 2)
    V = v.double().transpose(1, 2).repeat_interleave(q.shape[2] // k.shape[2], 1)
    want = V.gather(2, top[..., None].expand(-1, -1, -1, v.shape[3]))
    assert torch.isfinite(out).all()
    # the one probability, its sum and their quotient: 4 roundings of fp32 (others add nothing), and one to the type
    bound = (4 * 2.0 ** -24 + torch.finfo(q.dtype).eps / 2) * want.abs()
    assert ((out - want).abs() <= bound)[sure].all()
    assert (out.abs().amax(-1) > 0).all()                # no row is lost, whatever its scores


@pytest.mark.parametrize("name", list(FAR))
def test_far_scores(emu_ops, name):
    """Scores of any finite size: the largest one's probability is 1, however far it is from zero."""
    check_far_forward(name)


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(FAR))
def test_gpu_far_scores(name):
    check_far_forward(name, "cuda")


def test_scales_that_leave_the_kernels_numbers(emu_ops):
    """The kernels take scale and scale * log2(e) as normal floats: what is none of those is refused, the last ones that are work."""
    q, k, v, _ = inputs(1, 40, 40, 1, 1, 64, "f32")
    for scale in (1e-50, 1e-46, 2.0 ** -127, 1.8e38, 3e38, 1e300, -1.0):
        with pytest.raises(ValueError):
            A.attention_forward(q, k, v, scale=scale)
    lib = emu_ops.get_lib()
    out = torch.empty_like(q)
    for scale, code in ((1e-46, -1), (2.0 ** -127, -1), (2.0 ** -126, 0), (2.0 ** 127, 0), (3e38, -1)):
        call = A._Call(q, k, v, None, None, True, 0.5)
        call.head = (*call.head[:8], scale, *call.head[9:])
        assert lib.amoe_attention_fwd(call.pack(out, None, None), None, 0, None) == code, scale
    # scores of no size at all: the mean of what a row sees (40 terms, their sum, a quotient: 42 roundings)
    out = A.attention_forward(q, k, v, scale=2.0 ** -126)[0].double()
    n = torch.arange(1, 41)[:, None, None]
    assert ((out - v.double().cumsum(1) / n).abs() <= 48 * 2.0 ** -24 * v.double().abs().cumsum(1) / n).all()
    # and of the largest: scores have to stay finite themselves
    q, k = q * 2.0 ** -20, k * 2.0 ** -20
    top, sure = one_hot(q, k, True, 2.0 ** 127)
    out = A.attention_forward(q, k, v, scale=2.0 ** 127)[0].transpose(1, 2)
    want = v.transpose(1, 2).gather(2, top[..., None].expand(-1, -1, -1, 64))
    assert sure.all() and ((out - want).abs() <= 4 * 2.0 ** -24 * want.abs()).all()


def check_far_backward(name, device="cpu"):
    q, k, v, go, causal, scale = far_inputs(name)
    B, S, H, d = q.shape
    T, G = k.shape[1:3]
    top, sure = one_hot(q, k, causal, scale)
    Q, K, V = (t.double().transpose(1, 2).repeat_interleave(H // t.shape[2], 1) for t in (q, k, v))
    for held in (go, torch.where(sure.transpose(1, 2)[..., None], go, torch.zeros_like(go))):
        args = [t.to(device) for t in (held, q, k, v)]
        left = A.attention_forward(*args[1:], causal=causal, scale=scale, want_lse=True)
        grads = A.attention_backward(*args, *left, causal=causal, scale=scale)
        assert all(torch.isfinite(t).all() for t in grads)
    dq, dk, dv = (t.cpu().double().transpose(1, 2) for t in grads)
    # a row that one key takes hands its gradient to that key's value, and to q and k nothing: what dP - delta leaves there is
    # two sums of d products, 2 (d + 2) roundings, and their rounding to the type
    u, e, tiny = torch.finfo(q.dtype).eps / 2, 2.0 ** -24, torch.finfo(q.dtype).smallest_normal
    g = held.double().transpose(1, 2)
    at = top[..., None].expand(-1, -1, -1, d)
    ds = (2 * (d + 2) * e * (g.abs() * V.abs().gather(2, at)).sum(-1, keepdim=True) + tiny) * (1 + 2 * u)

    def to_keys(x):
        return torch.zeros(B, H, T, d, dtype=torch.float64).scatter_add_(2, at, x).reshape(B, G, H // G, T, d).sum(2)
    want, size = to_keys(g), to_keys(g.abs())
    assert ((dv - want).abs() <= u * want.abs() + (S * H // G + 8) * e * size + tiny).all()
    assert (dq.abs() <= 1.01 * scale * ds * K.abs().gather(2, at) + tiny).all()
    assert (dk.abs() <= 1.01 * scale * to_keys(ds * Q.abs()) + tiny).all()


@pytest.mark.parametrize("name", list(FAR))
def test_far_gradients(emu_ops, name):
    check_far_backward(name)


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(FAR))
def test_gpu_far_gradients(name):
    check_far_backward(name, "cuda")


SHIFTED = {
    # S, T, H, G, d, dtype, how far all scores of a row are from zero: 15 * size^2
    "f32": (70, 140, 2, 1, 16, "f32", 32),
    "f32_split": (2, 300, 2, 2, 16, "f32", 100),
    "f32_128": (40, 70, 1, 1, 128, "f32", 64),
    "bf16": (70, 140, 2, 1, 16, "bf16", 256),
    "bf16_128": (33, 130, 2, 1, 128, "bf16", 256),
    "f16": (70, 140, 2, 1, 16, "f16", 256),
    "f16_96": (20, 90, 1, 1, 96, "f16", 512),
    "odd_bf16": (40, 66, 1, 1, 17, "bf16", 256),
}


def check_shifted(name, device="cpu"):
    S, T, H, G, d, dtype, size = SHIFTED[name]
    _, _, v, go = inputs(1, S, T, H, G, d, dtype, seed=len(name))
    q, k = torch.zeros(1, S, H, d), torch.zeros(1, T, G, d)
    q[..., :15] = k[..., :15] = size
    q[:, 1::3, :, :15] = 0.0                              # (every third row is near, among those that are far)
    q[..., 15] = (-1.0) ** torch.arange(S)[:, None]
    k[..., 15] = torch.randint(0, 8, (1, T, G), generator=torch.Generator().manual_seed(0)).float()
    q, k = q.to(DT[dtype]), k.to(DT[dtype])
    for kw in ({}, dict(lengths=torch.tensor([T - 1]), starts=torch.tensor([-1]))):
        want, bounds = O.attention(q, k, v, go, scale=1.0, exact_scores=True, **kw)
        on = [t.to(device) for t in (q, k, v, go)]
        how = dict(scale=1.0, **{n: t.to(device) for n, t in kw.items()})
        out, lse, rest = A.attention_forward(*on[:3], want_lse=True, **how)
        compare((out, *A.attention_backward(on[3], *on[:3], out, lse, rest, **how)), want, bounds, name)


@pytest.mark.parametrize("name", list(SHIFTED))
def test_rows_far_from_zero(emu_ops, name):
    """Scores that differ by some units, all of them far from zero: as exact as their differences are."""
    check_shifted(name)


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(SHIFTED))
def test_gpu_rows_far_from_zero(name):
    check_shifted(name, "cuda")


EQUAL_VALUES = {
    # B, S, T, H, G, d, dtype, size of q
    "rows_bf16": (1, 70, 140, 2, 1, 64, "bf16", 1.0),
    "rows_f16": (2, 70, 140, 2, 1, 64, "f16", 1.0),
    "rows_f32": (1, 40, 90, 2, 1, 64, "f32", 1.0),
    "peaked_bf16_128": (1, 40, 300, 2, 2, 128, "bf16", 20.0),
    "peaked_f16_80": (1, 33, 200, 2, 1, 80, "f16", 20.0),
    "far_bf16": (1, 40, 140, 1, 1, 64, "bf16", 2000.0),
    "edges_bf16": (1, 40, 90, 1, 1, 13, "bf16", 3.0),
    "step_bf16": (2, 1, 700, 4, 2, 64, "bf16", 1.0),
    "step_f16": (1, 2, 500, 4, 1, 96, "f16", 5.0),
}


def check_equal_values(name, device="cpu"):
    *sizes, dtype, size = EQUAL_VALUES[name]
    B, S, T, H, G, d = sizes
    q, k, v, go = inputs(*sizes, dtype, seed=3)
    q = (q.float() * size).to(q.dtype)
    v = v[:, :1].expand(B, T, G, d)
    on = [t.to(device) for t in (q, k, v, go)]
    out, lse, rest = A.attention_forward(*on[:3], want_lse=True)
    want = v[:, :1].repeat_interleave(H // G, 2).expand(B, S, H, d)
    e = 2.0 ** -24
    # two sums of T terms, in other orders, and half a step of the subnormal numbers where rest is one
    off = 2 * (T + 4) * e * want.double().abs() + torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps / 2
    have = out.cpu().double() + (0 if rest is None else rest.cpu().double())
    assert ((have - want.double()).abs() <= off).all()
    if dtype != "f32":
        assert torch.equal(out.cpu(), want)                               # (what is off by less than half a step rounds back)
    # dP is the same for all keys and delta that number: what is left of dS are the roundings of d products, twice, and out's
    dq = A.attention_backward(on[3], *on[:3], out, lse, rest)[0].cpu().double()
    g = go.double().abs()
    ds = (g * (2 * (d + 2) * e * want.double().abs() + 2 * off)).sum(-1, keepdim=True) + torch.finfo(q.dtype).smallest_normal
    big = k.double().abs().amax(1, keepdim=True).repeat_interleave(H // G, 2)
    assert (dq.abs() <= 1.01 / math.sqrt(d) * ds * big + torch.finfo(q.dtype).smallest_normal).all()


@pytest.mark.parametrize("name", list(EQUAL_VALUES))
def test_equal_values(emu_ops, name):
    """Whatever the probabilities are rounded to, the sum that divides them counts the same numbers: a mean of equal values is
    that value, and q has no gradient."""
    check_equal_values(name)


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(EQUAL_VALUES))
def test_gpu_equal_values(name):
    check_equal_values(name, "cuda")


def check_tail(dtype, S, device="cpu"):
    """A long tail of keys with 2^-22 of the largest probability: as fp16 operands subnormal numbers, which the sum has to count as
    the product does.  Both are a mean of equal values."""
    T, d = 4000, 64
    q, k, v = torch.zeros(1, S, 2, d), torch.zeros(1, T, 1, d), torch.ones(1, T, 1, d)
    q[..., 0] = 1.0
    k[0, 1:, 0, 0] = -15.25
    v[..., ::2] = 3.0
    q, k, v = (t.to(DT[dtype]).to(device) for t in (q, k, v))
    out, _, rest = A.attention_forward(q, k, v, causal=False, scale=1.0, want_lse=True)
    have = (out.double() + (0 if rest is None else rest.double())).cpu()
    want = v[:, :1].double().cpu().expand_as(have)
    # a lane adds half the keys two by two, the product 16 at a time
    assert ((have - want).abs() <= (T / 4 + T / 16 + 16) * 2.0 ** -24 * want).all()
    # with other values in the tail: a thousandth of them arrives
    v[:, 1:] = 0.0
    have = A.attention_forward(q, k, v, causal=False, scale=1.0)[0].double().cpu()
    tail = (T - 1) * math.exp(-15.25)
    off = torch.finfo(q.dtype).eps / 2 + 2.0 ** -11 * tail + 2.0 ** -13
    assert 9e-4 < tail and ((have - want / (1 + tail)).abs() <= off * want).all()


@pytest.mark.parametrize("dtype, S", [("f16", 1), ("f16", 40), ("bf16", 1)])
def test_tail(emu_ops, dtype, S):
    check_tail(dtype, S)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, S", [("f16", 1), ("f16", 300), ("bf16", 1), ("bf16", 300)])
def test_gpu_tail(dtype, S):
    check_tail(dtype, S, "cuda")


def check_rest(dtype, S, d, device="cpu"):
    """Queries of zeros: a row is the mean of the values it sees, its probabilities are exact (the maximum is 0, each 2^0, the sum
    a whole number), so that nothing but the output's rounding is off by more than some 2^-24."""
    q, _, v, go = inputs(1, S, S, 2, 1, d, dtype, seed=4)
    q = torch.zeros_like(q)
    k = torch.ones(1, S, 1, d, dtype=q.dtype)
    # values next to each other: what rounding takes from their mean is as large as what they differ by
    v = (1.0 + (v.float() * 4).round() * torch.finfo(q.dtype).eps).to(q.dtype)
    on = [t.to(device) for t in (q, k, v, go)]
    out, lse, rest = A.attention_forward(*on[:3], want_lse=True)
    u, e = torch.finfo(q.dtype).eps / 2, 2.0 ** -24
    n = torch.arange(1, S + 1)[:, None, None].double()
    V = v.double()
    mean, size = V.cumsum(1) / n, V.abs().cumsum(1) / n
    # a sum of n terms, a quotient, a product; then rest, itself rounded (or half a step of the subnormal numbers)
    off = (S + 4) * e * size
    left = (mean - out.cpu().double()).abs()
    small = torch.finfo(q.dtype).smallest_normal * u
    b_rest = off + u * (left + off) + small
    assert ((out.cpu().double() + rest.cpu().double() - mean).abs() <= b_rest).all()
    assert rest.abs().max() > 0.2 * u                                     # (there is something to keep)
    # dq = scale * sum of P (dP - delta) over keys of ones.  The formula has 0; P = 1 / n by 2^-lse is off by 8 e, the sum of
    # what P's error multiplies by |dP - delta| at most; dS is rounded to the type; delta is off by b_rest and 2 d roundings
    dq = A.attention_backward(on[3], *on[:3], out, lse, rest)[0].cpu().double()
    g = go.double()
    dP = (g.transpose(1, 2) @ V.transpose(1, 2).transpose(2, 3)).masked_fill(torch.ones(S, S).triu(1).bool(), 0.0)     # [1, 2, S, S]
    delta = (g * mean).sum(-1).transpose(1, 2)[..., None]
    ds = (dP - delta).abs().masked_fill(torch.ones(S, S).triu(1).bool(), 0.0).sum(-1) / n[:, 0, 0]
    b_delta = ((g.abs() * (b_rest + 2 * (d + 2) * e * size)).sum(-1)).transpose(1, 2)
    bound = (ds * (u + (8 + S) * e) + b_delta).transpose(1, 2)[..., None] / math.sqrt(d) * 1.01 + torch.finfo(q.dtype).smallest_normal
    assert (dq.abs() <= bound).all(), (dq.abs() / bound).max()
    for wrong in (None, -rest):                                           # (the bound tells rest from none, and from its opposite)
        dq = A.attention_backward(on[3], *on[:3], out, lse, wrong)[0].cpu().double()
        assert (dq.abs() > bound).any()


@pytest.mark.parametrize("dtype, S, d", [("bf16", 90, 64), ("f16", 70, 64), ("bf16", 40, 128), ("bf16", 35, 13)])
def test_rest(emu_ops, dtype, S, d):
    check_rest(dtype, S, d)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, S, d", [("bf16", 300, 64), ("f16", 300, 96), ("bf16", 200, 128), ("bf16", 200, 13)])
def test_gpu_rest(dtype, S, d):
    check_rest(dtype, S, d, "cuda")


def test_no_copy_into_lds_is_left_behind(emu_ops):
    """What a workgroup has on its way into LDS when it ends would land in the next one's: every copy has been waited for."""
    import ctypes
    left = emu_ops.get_lib().amoe_emu_lds_copies_left
    left.restype = ctypes.c_longlong
    before = left()
    for d in (64, 128):
        for S, T, kw in ((40, 200, dict(starts=torch.tensor([30, 0]))), (3, 70, {}), (70, 40, dict(lengths=torch.tensor([40, 0])))):
            q, k, v, go = inputs(2, S, T, 2, 1, d, "bf16")
            out = A.attention_forward(q, k, v, **kw, want_lse=True)
            A.attention_backward(go, q, k, v, *out, **kw)
            assert left() == before, (d, S, T)


def check_keys_that_no_query_sees(d, T, device="cpu"):
    """Zeros, beside gradients of keys that are seen; the workgroups of the former have nothing to wait for."""
    q, k, v, go = inputs(2, 40, T, 2, 1, d, "bf16")
    starts = torch.tensor([30, 0])
    want, bounds = O.attention(q, k, v, go, starts=starts)
    on, starts = [t.to(device) for t in (q, k, v, go)], starts.to(device)
    out, lse, rest = A.attention_forward(*on[:3], None, starts, want_lse=True)
    grads = A.attention_backward(on[3], *on[:3], out, lse, rest, None, starts)
    compare((out, *grads), want, bounds, d)
    for g in grads[1:]:
        assert g[0, :70].any(-1).all() and not g[0, 70:].any() and g[1, :40].any(-1).all() and not g[1, 40:].any()


@pytest.mark.parametrize("d", [64, 128])
def test_keys_that_no_query_sees(emu_ops, d):
    check_keys_that_no_query_sees(d, 200)


@pytest.mark.gpu
@pytest.mark.parametrize("d, T", [(64, 200), (64, 20000), (128, 5000)])
def test_gpu_keys_that_no_query_sees(d, T):
    check_keys_that_no_query_sees(d, T, "cuda")
