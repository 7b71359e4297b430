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
