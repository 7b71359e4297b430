"""The decoder with this package's norms, several sequences after one prompt and tokens drawn from the logits: the operators together,
as training and serving use them."""
import pytest
import torch
from torch import nn

from analog_moe_amd import decoder as D
from analog_moe_amd.norm import LayerNorm
from analog_moe_amd.rotary import Rotary
from analog_moe_amd.sampling import sample
from tests.test_decoder_rotary import Plain
from tests.test_emu_kernels import emu_ops  # noqa: F401


def model(norm=LayerNorm, vocab=31, d=64, layers=2, heads=4, kv_heads=2, dim=16, make=None):
    torch.manual_seed(0)
    return D.SigmaMoEDecoder(vocab, d, layers, heads, 64, make or (lambda i: Plain(d)), Rotary(dim), kv_heads, norm)


def same_model(norm):
    m, like = model(norm), model(nn.LayerNorm)
    with torch.no_grad():
        for p in like.parameters():
            p.add_(0.05 * torch.randn(p.shape, generator=torch.Generator().manual_seed(p.numel())))
    m.load_state_dict(like.state_dict())
    return m, like


def check_training_step(device="cpu", lengths=None):
    """Loss and gradients of the model with these norms against nn.LayerNorm's: fp32, two layers of O(1) activations that differ
    by some roundings (2^-22 relative), and 2^-15 of a tensor's largest gradient is a hundred of those."""
    m, like = (x.to(device) for x in same_model(LayerNorm))
    ids = torch.randint(0, 31, (2, 9), generator=torch.Generator().manual_seed(1)).to(device)
    labels = ids.roll(-1, 1)
    got, want = [], []
    for x, out in ((m, got), (like, want)):
        loss, _ = x(ids, labels, lengths=lengths)
        out += [loss.detach(), *torch.autograd.grad(loss, list(x.parameters()))]
    for a, b in zip(got, want):
        assert (a - b).abs().max() <= 2.0 ** -15 * b.abs().max()


def test_training_step(emu_ops):
    check_training_step()


@pytest.mark.gpu
def test_gpu_training_step():
    check_training_step("cuda")


def test_stock_attention_with_these_norms(emu_ops):
    torch.manual_seed(0)
    m = D.SigmaMoEDecoder(31, 64, 2, 4, 64, lambda i: Plain(64), norm=LayerNorm)
    like = D.SigmaMoEDecoder(31, 64, 2, 4, 64, lambda i: Plain(64))
    like.load_state_dict(m.state_dict())
    ids = torch.randint(0, 31, (2, 9), generator=torch.Generator().manual_seed(1))
    with torch.no_grad():
        a, b = m(ids)[0], like(ids)[0]
    assert (a - b).abs().max() <= 2.0 ** -15 * b.abs().max()
    assert [n for n, _ in m.named_parameters()] == [n for n, _ in like.named_parameters()]


def test_norms_of_two_kinds_and_hooks(emu_ops):
    """A norm that is replaced takes the sums back, and what is hooked onto a block runs."""
    m, like = same_model(LayerNorm)
    ids, runs = torch.randint(0, 31, (2, 5), generator=torch.Generator().manual_seed(1)), []
    for blk in m.blocks:
        blk.register_forward_hook(lambda *_: runs.append(1))
    with torch.no_grad():
        want = like(ids)[0]
        for name in (None, "ln_out", "ln_attn"):
            if name is not None:
                owner = m if name == "ln_out" else m.blocks[1]
                setattr(owner, name, getattr(like if name == "ln_out" else like.blocks[1], name))
            assert (m(ids)[0] - want).abs().max() <= 2.0 ** -15 * want.abs().max()
    assert len(runs) == 6


def check_shared(m, ids, prompts, copies, tol, device="cpu"):
    """Prompts [N, S] of the given lengths, then the tokens ids [N * copies, steps] one by one over a cache that shares the prompts:
    the logits of the whole sequences at once.  Then two at once, and the prompts' own cache goes on."""
    N = prompts.shape[0]
    lengths = torch.tensor([prompts.shape[1], prompts.shape[1] - 3][:N], device=device)
    steps = ids.shape[1]
    with torch.no_grad():
        cache = m.new_cache(N, prompts.shape[1] + 2)
        cache.keys.fill_(float("nan"))
        cache.values.fill_(float("nan"))
        m(prompts, lengths=lengths, cache=cache)
        shared = cache.share(copies, steps + 2)
        shared.keys.fill_(float("nan"))
        shared.values.fill_(float("nan"))
        held = cache.held.clone()
        m(prompts[:, :1], cache=cache)                     # (what the prompts' cache gets now is none of the others')
        got = torch.cat([m(ids[:, s:s + 1], cache=shared)[0] for s in range(steps)], 1)
        assert shared.held.tolist() == [steps] * (N * copies) and torch.equal(shared.prefix.held, held)
        pair = m(ids[:, :2], cache=shared)[0]
        for b in range(N * copies):
            n = int(lengths[b // copies])
            whole = m(torch.cat((prompts[b // copies, :n], ids[b], ids[b, :2]))[None])[0][0]
            assert (got[b] - whole[n:n + steps]).abs().max() <= tol * whole.abs().max(), b
            assert (pair[b] - whole[n + steps:]).abs().max() <= tol * whole.abs().max(), b


@pytest.mark.parametrize("norm", [LayerNorm, nn.LayerNorm])
def test_shared_cache(emu_ops, norm):
    g = torch.Generator().manual_seed(2)
    check_shared(model(norm), torch.randint(0, 31, (6, 3), generator=g), torch.randint(0, 31, (2, 9), generator=g), 3, 2.0 ** -15)


def by_hand(m, ids, lengths, steps, copies, generator, **settings):
    """generate over whole sequences, anew for every token."""
    N = ids.shape[0]
    rows = [ids[b // copies, :int(lengths[b // copies])] for b in range(N * copies)]
    out = []
    for s in range(steps):
        u = torch.rand(N * copies, generator=generator, device=ids.device)
        last = torch.stack([m(r[None])[0][0, -1] for r in rows])
        out.append(sample(last, u, **settings))
        rows = [torch.cat((r, t[None])) for r, t in zip(rows, out[-1])]
    return torch.stack(out, 1)


def check_generate(m, ids, steps, device="cpu"):
    """fp32: logits differ from those of whole sequences by some 2^-20, which moves a draw where u comes as close as that to a
    border: not at these seeds, which give the same tokens in both."""
    lengths = torch.tensor([ids.shape[1], ids.shape[1] - 2], device=device)
    with torch.no_grad():
        for copies, how in ((3, dict(temperature=0.8, top_p=0.9)), (1, dict(top_k=5)), (2, dict(temperature=0.0))):
            g = torch.Generator(device).manual_seed(7)
            tokens, logprob = m.generate(ids, steps, copies, lengths, g, want_logprob=True, **how)
            want = by_hand(m, ids, lengths, steps, copies, torch.Generator(device).manual_seed(7), **how)
            assert torch.equal(tokens, want) and torch.isfinite(logprob).all() and (logprob <= 0).all()
    assert torch.equal(tokens[0], tokens[1]) and torch.equal(tokens[2], tokens[3])        # (temperature 0: copies agree)
    assert m.generate(ids, 2, 2, generator=torch.Generator(device).manual_seed(1)).shape == (4, 2)
    assert m.generate(ids, 0).shape == (2, 0)


def test_generate(emu_ops):
    check_generate(model(), torch.randint(0, 31, (2, 6), generator=torch.Generator().manual_seed(5)), 2)


def test_refusals(emu_ops):
    m = model()
    ids = torch.zeros(2, 3, dtype=torch.int64)
    with torch.no_grad():
        cache = m.new_cache(2, 5)
        m(ids, cache=cache)
        shared = cache.share(2, 3)
        for bad in (lambda: shared.share(2, 3), lambda: cache.share(0, 3), lambda: cache.share(1, -1), lambda: m(ids, cache=shared),
                    lambda: m(torch.zeros(4, 4, dtype=torch.int64), cache=shared), lambda: m.generate(ids, -1), lambda: m.generate(ids, 1, 0),
                    lambda: m.generate(ids[:, :0], 1), lambda: m.generate(ids, 1, top_p=2.0)):
            with pytest.raises(ValueError):
                bad()
    with pytest.raises(RuntimeError):
        m(torch.zeros(4, 1, dtype=torch.int64), cache=shared)
    with pytest.raises(ValueError):
        D.SigmaMoEDecoder(31, 64, 1, 4, 64, lambda i: Plain(64), norm=LayerNorm).generate(ids, 1)


# ------------------------------------------------------------------------------ on the GPU
def expert_model(dtype):
    """All experts take part (k = 4 of 4: no choice that a rounding could tip)."""
    from analog_moe_amd import config as rpu
    from analog_moe_amd.moe_layer import AnalogSigmaMoELayer

    def make(i):
        r = rpu.TorchInferenceRPUConfig()
        r.pre_post.input_range.enable = True
        return AnalogSigmaMoELayer(r, d_model=128, n_experts=4, expert_size=64, k=4)
    return model(vocab=97, d=128, heads=4, kv_heads=2, dim=32, make=make).cuda().to(dtype).eval()


@pytest.mark.gpu
def test_gpu_shared_cache():
    g = torch.Generator().manual_seed(2)
    m = expert_model(torch.float32)
    check_shared(m, torch.randint(0, 97, (40, 3), generator=g).cuda(), torch.randint(0, 97, (2, 200), generator=g).cuda(), 20, 2.0 ** -12, "cuda")


@pytest.mark.gpu
def test_gpu_generate():
    m = model(make=lambda i: Plain(64)).cuda()
    check_generate(m, torch.randint(0, 31, (2, 40), generator=torch.Generator().manual_seed(5)).cuda(), 4, "cuda")


@pytest.mark.gpu
def test_gpu_steps_captured():
    """A step of every sequence after a shared prompt, its draw and the next step's token as one graph."""
    m = expert_model(torch.bfloat16)
    ids = torch.randint(0, 97, (2, 40), generator=torch.Generator().manual_seed(4)).cuda()
    u = torch.rand(4, 8, generator=torch.Generator().manual_seed(6)).cuda()
    with torch.no_grad():
        def prompt():
            cache = m.new_cache(2, 40)
            m(ids, cache=cache)
            cache = cache.share(4, 16)
            cache.most = 15                                # (keys to the end of the room, as the graph reads them)
            return cache

        def step(token, number, cache):
            cache.most = 15
            logits, _ = m(token, cache=cache)
            return sample(logits[:, -1], number, temperature=0.9, top_p=0.95)
        cache, token, want = prompt(), ids[:, -1:].repeat_interleave(4, 0), []
        for s in range(4):
            want.append(step(token, u[s], cache))
            token = want[-1][:, None]
        cache, token, number = prompt(), ids[:, -1:].repeat_interleave(4, 0), u[0].clone()
        held, graph = cache.held, torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            drawn = step(token, number, cache)
            token.copy_(drawn[:, None])
            held.add_(1)
        for s in range(4):
            number.copy_(u[s])
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(drawn, want[s]), s


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gpu_training_step_captured(dtype):
    """Forward, backward and an optimizer step as a graph: the parameters it leaves are those of eager steps."""
    ids = torch.randint(0, 97, (2, 65), generator=torch.Generator().manual_seed(3)).cuda()
    labels = ids.roll(-1, 1)

    def fresh():
        m = expert_model(dtype).train()
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
