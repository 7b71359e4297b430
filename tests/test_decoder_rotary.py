"""The decoder with this package's attention and rotary positions: the operators together, as training and serving use them."""
import pytest
import torch
from torch import nn

from analog_moe_amd import decoder as D
from analog_moe_amd.rotary import Rotary
from oracle import attention_oracle as O
from tests.test_emu_kernels import emu_ops  # noqa: F401


class Plain(nn.Module):
    """A feed-forward in place of the expert layer."""

    def __init__(self, d):
        super().__init__()
        self.up, self.down = nn.Linear(d, 2 * d), nn.Linear(2 * d, d)

    def forward(self, x):
        return self.down(torch.relu(self.up(x))), x.new_zeros(())


def model(vocab=31, d=64, layers=2, heads=4, kv_heads=2, dim=16, make=None, **rotary):
    torch.manual_seed(0)
    return D.SigmaMoEDecoder(vocab, d, layers, heads, 64, make or (lambda i: Plain(d)), Rotary(dim, **rotary), kv_heads)


class Formula(torch.autograd.Function):
    """Attention by its formula in 64 bits."""

    @staticmethod
    def forward(ctx, q, k, v, lengths):
        ctx.save_for_backward(q, k, v, lengths)
        return O.attention(q, k, v, lengths=lengths)[0][0].to(q.dtype)

    @staticmethod
    def backward(ctx, go):
        q, k, v, lengths = ctx.saved_tensors
        return (*(g.to(q.dtype) for g in O.attention(q, k, v, go, lengths=lengths)[0][1:]), None)


def by_formula(monkeypatch):
    monkeypatch.setattr(D, "attention", lambda q, k, v, lengths=None, starts=None: Formula.apply(q, k, v, lengths))

    def turn(self, q, k, positions=None):
        R = self.dim
        turns = self.turns.double() / 2.0 ** 64 * 2 * torch.pi
        angle = (torch.arange(q.shape[1]) if positions is None else positions).double()[..., None, None] * turns
        cos, sin = (self.size * angle.cos()).float(), (self.size * angle.sin()).float()

        def one(x):
            a, b = x[..., :R // 2], x[..., R // 2:R]
            return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., R:]), -1)
        return one(q), one(k)
    monkeypatch.setattr(Rotary, "forward", turn)


@pytest.mark.parametrize("lengths", [None, [9, 4]])
def test_training_step(emu_ops, monkeypatch, lengths):
    """Loss and gradients against the same model on formulas.  fp32, two layers of O(1) activations: the operators differ from
    their formulas by some 2^-22 relative, and a layer (a norm, matrices of gain about 1) hands differences on without growing
    them, as it does the rounding of its own sums; 2^-15 of a tensor's largest gradient is a hundred of those."""
    m = model()
    ids = torch.randint(0, 31, (2, 9), generator=torch.Generator().manual_seed(1))
    labels = ids.roll(-1, 1)
    n = None if lengths is None else torch.tensor(lengths)
    if n is not None:
        labels = labels.masked_fill(torch.arange(9) >= n[:, None] - 1, -100)

    def step():
        loss, _ = m(ids, labels, lengths=n)
        return loss.detach(), torch.autograd.grad(loss, list(m.parameters()))
    loss, grads = step()
    with monkeypatch.context() as patch:
        by_formula(patch)
        want, want_grads = step()
    assert abs(loss - want) < 2.0 ** -15 * want
    for a, b in zip(grads, want_grads):
        assert (a - b).abs().max() <= 2.0 ** -15 * b.abs().max()


def stepwise(m, ids, lengths, room, device="cpu"):
    """Logits of a prompt and of the tokens after it, one by one, over a cache.  ids [B, prompt + steps]."""
    prompt = int(lengths.max())
    cache = m.new_cache(ids.shape[0], room)
    cache.keys.fill_(float("nan"))
    cache.values.fill_(float("nan"))
    first = torch.zeros(ids.shape[0], prompt, dtype=torch.int64, device=device)
    for b, n in enumerate(lengths.tolist()):
        first[b, :n] = ids[b, :n]
    out = [m(first, lengths=lengths, cache=cache)[0]]
    rows = torch.arange(ids.shape[0], device=device)
    for s in range(ids.shape[1] - prompt):
        out.append(m(ids[rows, lengths + s][:, None], cache=cache)[0])
    assert cache.held.tolist() == (lengths + ids.shape[1] - prompt).tolist()
    return out


def check_stepwise(m, ids, lengths, tol, device="cpu"):
    """The cached run gives what the whole sequences at once give: same products of the same numbers, summed in another order."""
    with torch.no_grad():
        whole = m(ids)[0]
        got = stepwise(m, ids, lengths, ids.shape[1] + 3, device)
        for b, n in enumerate(lengths.tolist()):
            assert (got[0][b, :n] - whole[b, :n]).abs().max() <= tol
            for s, g in enumerate(got[1:]):
                assert (g[b, 0] - whole[b, n + s]).abs().max() <= tol, (b, s)


def test_cache(emu_ops):
    """fp32, logits of O(1): 2^-15 as above."""
    m = model()
    ids = torch.randint(0, 31, (3, 12), generator=torch.Generator().manual_seed(2))
    check_stepwise(m, ids, torch.tensor([9, 4, 1]), 2.0 ** -15)


def test_lengths_outside_the_ids(emu_ops):
    """A cache never holds less than before nor more than it was given."""
    m = model()
    ids = torch.randint(0, 31, (3, 4), generator=torch.Generator().manual_seed(2))
    with torch.no_grad():
        caches = [m.new_cache(3, 9) for _ in range(2)]
        for cache, lengths in zip(caches, ([7, -2, 3], [4, 0, 3])):
            m(ids, lengths=torch.tensor(lengths, dtype=torch.int32), cache=cache)
            assert cache.held.tolist() == [4, 0, 3] and cache.held.dtype == torch.int64
        assert torch.equal(m(ids[:, :1], cache=caches[0])[0], m(ids[:, :1], cache=caches[1])[0])


def test_refusals(emu_ops):
    m = model()
    ids = torch.zeros(2, 3, dtype=torch.int64)
    old = D.SigmaMoEDecoder(31, 64, 1, 4, 64, lambda i: Plain(64))
    for bad in (lambda: old.new_cache(1, 2), lambda: old(ids, lengths=torch.tensor([1, 2])), lambda: model(dim=32), lambda: model(kv_heads=3),
                lambda: D.SigmaMoEDecoder(31, 64, 1, 4, 64, lambda i: Plain(64), kv_heads=2)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        m(ids, cache=m.new_cache(2, 8))
    with torch.no_grad():
        cache = m.new_cache(2, 5)
        m(ids, cache=cache)
        for bad in (lambda: m(ids, cache=cache), lambda: m(ids[:1], cache=cache)):
            with pytest.raises(ValueError):
                bad()
        m(ids[:, :2], cache=cache)
    assert old(ids)[0].shape == (2, 3, 31) and "blocks.0.attn.rotary.turns" not in m.state_dict()


def expert_model(dtype, k=2, layers=2):
    from analog_moe_amd import config as rpu
    from analog_moe_amd.moe_layer import AnalogSigmaMoELayer

    def make(i):
        r = rpu.TorchInferenceRPUConfig()
        r.pre_post.input_range.enable = True
        return AnalogSigmaMoELayer(r, d_model=128, n_experts=4, expert_size=64, k=k)
    return model(vocab=97, d=128, layers=layers, heads=4, kv_heads=2, dim=32, make=make).cuda().to(dtype)


@pytest.mark.gpu
def test_gpu_cache_with_the_expert_layer():
    """All experts take part (k = 4 of 4: no choice that a rounding could tip)."""
    m = expert_model(torch.float32, k=4).eval()
    ids = torch.randint(0, 97, (3, 200), generator=torch.Generator().manual_seed(2)).cuda()
    check_stepwise(m, ids, torch.tensor([190, 70, 1], device="cuda"), 2.0 ** -13, "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gpu_training_step_captured(dtype):
    """Forward, backward and an optimizer step as a graph: the parameters it leaves are those of eager steps."""
    ids = torch.randint(0, 97, (2, 65), generator=torch.Generator().manual_seed(3)).cuda()
    labels = ids.roll(-1, 1)

    def fresh():
        m = expert_model(dtype)
        return m, torch.optim.SGD(m.parameters(), lr=1e-2)

    def step(m, opt):
        loss, _ = m(ids, labels, reg_weight=0.01)
        loss.backward()
        opt.step()
    eager, opt = fresh()
    for _ in range(4):
        opt.zero_grad(set_to_none=True)
        step(eager, opt)
    m, opt = fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.zero_grad(set_to_none=True)
        step(m, opt)
    torch.cuda.current_stream().wait_stream(side)
    opt.zero_grad(set_to_none=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(m, opt)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
    for (name, a), b in zip(m.named_parameters(), eager.parameters()):
        assert torch.isfinite(a).all() and torch.equal(a, b), name


@pytest.mark.gpu
def test_gpu_single_steps_captured():
    """One token per sequence over a cache as a graph: positions and lengths are device tensors that the replays advance."""
    m = expert_model(torch.bfloat16, k=4).eval()
    ids = torch.randint(0, 97, (2, 40), generator=torch.Generator().manual_seed(4)).cuda()
    with torch.no_grad():
        def filled():
            cache = m.new_cache(2, 64)
            m(ids[:, :30], cache=cache)
            return cache
        cache = filled()
        want = [m(ids[:, 30 + s:31 + s], cache=cache)[0].clone() for s in range(4)]
        cache = filled()
        token = ids[:, 30:31].clone()
        cache.most = 63                                # (the graph's keys reach to the end of the room)
        held, graph = cache.held, torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            logits = m(token, cache=cache)[0]
            held.add_(1)
        for s in range(4):
            token.copy_(ids[:, 30 + s:31 + s])
            graph.replay()
            torch.cuda.synchronize()
            assert (logits - want[s]).abs().max() <= 2.0 ** -5 * want[s].abs().max(), s
