"""Rotary positions into tensors that are there already: what autograd, tracers and other memory see of it."""
import pytest
import torch
from torch.autograd import forward_ad
from torch.utils._python_dispatch import TorchDispatchMode

from analog_moe_amd import attention as A
from analog_moe_amd import rotary as R
from tests.test_emu_kernels import emu_ops  # noqa: F401
from tests.test_rotary import inputs


def test_what_was_saved_and_is_overwritten_is_noticed(emu_ops):
    """A backward pass whose saved tensor has been written to by out= raises, as for any other write in place."""
    r = R.Rotary(16)
    q, k = inputs(1, 4, 2, 1, 16, "f32")
    cache = torch.randn(1, 9, 1, 16, generator=torch.Generator().manual_seed(0))
    x = q.clone().requires_grad_()
    loss = A.attention(x, cache, cache).sum()
    before = cache._version, q._version
    with torch.no_grad():
        r(q, k, out=(q, cache[:, 2:6]))
    assert cache._version > before[0] and q._version > before[1]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():                          # (tensors without versions are written to as well)
        a, b = q.clone(), k.clone()
        want = r(a, b)
        r(a, b, out=(a, b))
        assert torch.equal(a, want[0]) and torch.equal(b, want[1])


def test_watched_calls(emu_ops):
    """With out= as without: forward-mode derivatives and function transforms are refused, modes and traces work."""
    q, k = inputs(1, 4, 1, 1, 16, "f32")
    r = R.Rotary(16)
    want = r(q, k)
    new = lambda: (torch.zeros_like(q), torch.zeros_like(k))          # noqa: E731
    with torch.no_grad(), forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            r(forward_ad.make_dual(q, q), k, out=new())
        out = new()
        r(q, k, out=out)                                              # (nothing here has a tangent)
        assert all(map(torch.equal, out, want))
    with torch.no_grad(), pytest.raises(RuntimeError):
        torch.func.vmap(lambda x: r(x, k, out=new())[0])(q[None])

    class Mode(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))
    out = new()
    with Mode():
        got = r(q, k, out=out)
    assert all(map(torch.equal, out, want)) and all(map(torch.equal, got, want))
    out = new()
    with torch.no_grad():
        traced = torch.jit.trace(lambda x: r(x, k, out=out)[0] + 0, (q,), check_trace=False)
        before = out[0]._version
        assert torch.equal(traced(k), r(k, k)[0]) and out[0]._version > before


def check_compiled(device):
    """A compiled call writes where it is told, in place and into a cache too, and what follows it sees that."""
    q, k = (t.to(device) for t in inputs(2, 3, 2, 1, 64, "bf16"))
    r = R.Rotary(64).to(device)
    cache = torch.zeros(2, 10, 1, 64, dtype=torch.bfloat16, device=device)

    def step(q, k, cache):
        turned, _ = r(q, k, start=4, out=(q, cache[:, 4:7]))
        return turned * 2, cache.sum()
    with torch.no_grad():
        want = r(q, k, start=4)
        torch._dynamo.reset()
        doubled, total = torch.compile(step, fullgraph=True, backend="aot_eager")(q, k, cache)
    assert torch.equal(q, want[0]) and torch.equal(cache[:, 4:7], want[1]) and torch.equal(doubled, want[0] * 2)
    assert not cache[:, :4].any() and not cache[:, 7:].any() and torch.equal(total, cache.sum())


def test_compiled(emu_ops):
    check_compiled("cpu")


@pytest.mark.gpu
def test_gpu_compiled():
    check_compiled("cuda")


def test_outputs_that_overlap_are_refused(emu_ops):
    """out's elements are memory of their own: of each other, of the other output, of both inputs unless they are the input."""
    r = R.Rotary(8)
    q, k = inputs(2, 4, 2, 1, 8, "f32")
    room = torch.randn(2, 6, 3, 8, generator=torch.Generator().manual_seed(1))
    a, b = room[:, 1:5, :2], room[:, 1:5, 2:]                     # packed heads
    flat = torch.zeros(400)
    for bad in (lambda: r(room[:, :4, :2], k, out=(a, k)),                                   # a token further on
                lambda: r(a, k, out=(room[:, 1:5, 1:], torch.empty_like(k))),                # a head further on
                lambda: r(q, b, out=(a, room[:, 1:5, 1:2])),                                 # one in the other
                lambda: r(q, k, out=(torch.empty_like(q), q[:, :, :1])),                     # k's in q
                lambda: r(q, room[:, :4, :1], out=(a, k)),                                   # q's in k, shifted
                lambda: r(k, k, out=(k, torch.empty_like(k))),                               # q is k, and one of them written to
                lambda: r(q, k, out=(q[:, :, :1].expand_as(q), k)),
                lambda: r(q, k, out=(flat.as_strided((2, 4, 2, 8), (64, 8, 8, 1)), k)),      # tokens in heads
                lambda: r(q, k, out=(flat.as_strided((2, 4, 2, 8), (30, 16, 8, 1)), k)),     # sequences in tokens
                lambda: r(q, k, out=(flat.as_strided((2, 4, 2, 8), (60, 15, 7, 1)), k))):    # heads in heads
        keep = [t.clone() for t in (q, k, room, flat)]
        with pytest.raises(ValueError, match="memory"):
            bad()
        assert all(map(torch.equal, (q, k, room, flat), keep))
    # what is not overlapping: in place in packed heads, heads first, tokens that alternate, the next tokens of one buffer
    for B, S, make in ((2, 4, lambda n: n(2, 4, 3, 8)), (2, 4, lambda n: n(2, 3, 4, 8).transpose(1, 2)), (4, 2, lambda n: n(2, 4, 3, 8).transpose(0, 1)),
                       (1, 1, lambda n: n(1, 1, 3, 8))):
        w = make(lambda *s: torch.randn(*s, generator=torch.Generator().manual_seed(2)))
        x, y = w[:, :, :2], w[:, :, 2:]
        want = r(x, y)
        got = r(x, y, out=(x, y))
        assert all(map(torch.equal, got, want)) and torch.equal(w, torch.cat(want, 2))
    w = torch.randn(2, 8, 3, 8, generator=torch.Generator().manual_seed(3))
    even, odd = w[:, ::2], w[:, 1::2]
    want = r(even[:, :, :2], even[:, :, 2:])
    r(even[:, :, :2], even[:, :, 2:], out=(odd[:, :, :2], odd[:, :, 2:]))
    assert torch.equal(odd, torch.cat(want, 2))
    want = r(w[:, :3, :2], w[:, :3, 2:])
    r(w[:, :3, :2], w[:, :3, 2:], out=(w[:, 4:7, :2], w[:, 4:7, 2:]))
    assert torch.equal(w[:, 4:7], torch.cat(want, 2))
    one = torch.randn(1, 1, 2, 8, generator=torch.Generator().manual_seed(4))
    want = r(one, one[:, :, :0])
    r(one, one[:, :, :0], out=(one.as_strided(one.shape, (5, 3, 8, 1)), one[:, :, :0]))      # (strides of single elements)
    assert torch.equal(one, want[0])
    none = r(q[:, :0], k[:, :0], out=(q[:, :0], q[:, :0, :1]))
    assert none[0].shape == (2, 0, 2, 8)
