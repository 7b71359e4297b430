"""The decoder's cache under autocast: its type is that of the keys that are written to it, or they are cast."""
import pytest
import torch

from tests.test_decoder_rotary import expert_model, model
from tests.test_emu_kernels import emu_ops  # noqa: F401


def check(m, ids, device):
    """A prompt and single tokens over a cache made inside autocast, outside it, and of another type than the model's; against
    the whole sequences at once.  bf16 everywhere: some ten roundings of 2^-8 in each of two layers that add to one another,
    taken at random signs, stay below 2^-5 of the largest logit."""
    prompt = ids.shape[1] - 3
    with torch.no_grad():
        plain = m.new_cache(ids.shape[0], ids.shape[1])
        assert plain.keys.dtype == torch.float32
        with torch.autocast(device, dtype=torch.bfloat16):
            whole = m(ids)[0]
            low = m.new_cache(ids.shape[0], ids.shape[1])
            assert low.keys.dtype == low.values.dtype == torch.bfloat16
            for cache in (plain, low):
                got = [m(ids[:, :prompt], cache=cache)[0]] + [m(ids[:, s:s + 1], cache=cache)[0] for s in range(prompt, ids.shape[1])]
                got = torch.cat(got, 1)
                assert got.dtype == whole.dtype
                assert (got.float() - whole.float()).abs().max() <= 2.0 ** -5 * whole.float().abs().max()
        # without autocast: the model's own type again, over a cache of either
        whole = m(ids)[0]
        for dtype, tol in ((torch.float32, 2.0 ** -13), (torch.bfloat16, 2.0 ** -5)):
            cache = m.new_cache(ids.shape[0], ids.shape[1])
            cache.keys, cache.values = cache.keys.to(dtype), cache.values.to(dtype)
            got = torch.cat([m(ids[:, :prompt], cache=cache)[0], m(ids[:, prompt:], cache=cache)[0]], 1)
            assert got.dtype == torch.float32 and (got - whole).abs().max() <= tol * whole.abs().max()


def test_cache(emu_ops):
    m = model()
    check(m, torch.randint(0, 31, (2, 9), generator=torch.Generator().manual_seed(1)), "cpu")


@pytest.mark.gpu
def test_gpu_cache():
    """(all experts take part: no choice that a rounding could tip)"""
    m = expert_model(torch.float32, k=4).eval()
    check(m, torch.randint(0, 97, (2, 80), generator=torch.Generator().manual_seed(1)).cuda(), "cuda")
