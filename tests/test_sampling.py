"""The choice of a token against its definition: the kernel's source on the CPU, and the built library on the GPU."""
import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from analog_moe_amd import sampling as S
from oracle import sample_oracle as O
from tests.test_attention import DT, _on_gpu
from tests.test_emu_kernels import emu_ops  # noqa: F401

INF = float("inf")


def test_a_gpu_is_needed():
    with pytest.raises(RuntimeError, match="GPU"):
        S.sample(torch.zeros(2, 8), torch.zeros(2))


def logits(rows, V, dtype, kind="normal", seed=0, layout="own"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, V, generator=g) * 2.5
    if kind == "coarse":                                  # many equal ones
        x = x.round()
    elif kind == "equal":
        x = torch.full((rows, V), 0.375)
    elif kind == "two":                                   # two values, most of them the lower one
        x = torch.where(torch.rand(rows, V, generator=g) < 0.1, 3.0, -1.0)
    elif kind == "zeros":                                 # of both signs
        x = torch.where(torch.rand(rows, V, generator=g) < 0.5, 0.0, -0.0)
    elif kind == "far":
        x = x * 1e4
    elif kind == "near":                                  # differences of some 2^-20 of the values
        x = 1000.0 + x * 1e-3
    elif kind == "huge":
        x = x / x.abs().amax() * torch.finfo(DT[dtype]).max
    if kind == "masked":
        x = x.masked_fill(torch.rand(rows, V, generator=g) < 0.6, -INF)
        x[:, V // 2] = float("nan")
    x = x.to(DT[dtype])
    if layout == "odd":
        x = torch.cat((torch.full((rows, 3), 99.0).to(x), x, torch.full((rows, 4), 99.0).to(x)), 1)[:, 3:3 + V]
    elif layout == "every":
        x = torch.stack((x, x + 5), 1).reshape(2 * rows, V)[::2]
    return x


def numbers(rows, seed=0):
    return torch.rand(rows, generator=torch.Generator().manual_seed(1000 + seed))


def setting(how, name, row, none):
    v = how.get(name, none)
    return float(v[row]) if isinstance(v, torch.Tensor) else v if name == "top_k" else float(np.float32(v))


def check(x, u, device="cpu", **how):
    to = lambda t: t if device == "cpu" else _on_gpu(t)                                   # noqa: E731
    on = {n: to(v) if isinstance(v, torch.Tensor) else v for n, v in how.items()}
    ids, logprob = S.draw(to(x), to(u), want_logprob=True, **on)
    again = S.draw(to(x), to(u), want_logprob=True, **on)
    assert torch.equal(ids, again[0]) and torch.equal(logprob, again[1])
    assert ids.dtype == torch.int64 and logprob.dtype == torch.float32 and ids.shape == logprob.shape == x.shape[:-1]
    V, called = x.shape[-1], 0
    for r, (row, got, lp) in enumerate(zip(x.double().reshape(-1, V).numpy(), ids.cpu().reshape(-1), logprob.cpu().reshape(-1))):
        want = O.draw(row, float(u.reshape(-1)[r]), setting(how, "temperature", r, 1.0), int(setting(how, "top_k", r, 0)),
                      setting(how, "top_p", r, 1.0), setting(how, "min_p", r, 0.0))
        if want is None:
            continue
        called += 1
        assert int(got) in want[0], (r, int(got), want, how)
        log = want[1][want[0].index(int(got))]
        if log == -INF:
            assert lp == -INF
        else:
            # one rounding to fp32; weights and their sum are off by 2^-44 each of the largest, x / temperature by 2^-52 of itself
            assert abs(float(lp) - log) <= 2.0 ** -24 * abs(log) + V * 2.0 ** -44 + 2.0 ** -126, (r, lp, log)
    assert called >= 0.9 * ids.numel()
    return ids


CASES = {
    # rows, V, dtype, kind, layout, settings
    "one": (1, 1, "f32", "normal", "own", {}),
    "two": (7, 2, "bf16", "normal", "own", {}),
    "full_f32": (7, 300, "f32", "normal", "own", {}),
    "full_wide_bf16": (2, 1003, "bf16", "normal", "own", dict(temperature=0.7)),
    "greedy": (7, 77, "f16", "coarse", "odd", dict(temperature=0.0)),
    "k": (7, 500, "f32", "normal", "own", dict(top_k=20)),
    "k_ties": (7, 500, "bf16", "coarse", "odd", dict(top_k=90)),
    "k_one": (6, 41, "f16", "normal", "own", dict(top_k=1)),
    "k_all": (6, 41, "f16", "normal", "own", dict(top_k=41)),
    "p": (7, 611, "bf16", "normal", "own", dict(top_p=0.9)),
    "p_ties": (2, 611, "f16", "coarse", "odd", dict(top_p=0.5)),
    "p_nothing": (6, 50, "f32", "normal", "own", dict(top_p=0.0)),
    "min_p": (6, 400, "f32", "normal", "every", dict(min_p=0.1)),
    "min_one": (6, 400, "f32", "coarse", "own", dict(min_p=1.0)),
    "all": (7, 900, "f32", "normal", "odd", dict(temperature=1.3, top_k=200, top_p=0.8, min_p=0.02)),
    "masked": (6, 333, "bf16", "masked", "own", dict(top_k=50, top_p=0.9)),
    "masked_k": (6, 33, "f32", "masked", "own", dict(top_k=30)),
    "far": (6, 200, "f32", "far", "own", dict(top_p=0.9)),
    "near": (6, 200, "f32", "near", "own", dict(top_p=0.6, temperature=0.001)),
    "huge": (6, 64, "f32", "huge", "own", dict(top_p=0.6, temperature=1e38)),
    "cold": (6, 64, "f32", "normal", "own", dict(top_p=0.6, temperature=1e-30)),
    "coldest": (6, 64, "f32", "normal", "own", dict(top_k=3, temperature=1e-45)),
    "hot": (6, 64, "bf16", "normal", "own", dict(top_p=0.6, temperature=3e38)),
    "zeros": (6, 128, "f32", "zeros", "own", dict(top_k=40)),
    "two_values": (6, 500, "f32", "two", "own", dict(top_k=111, top_p=0.75)),
}


@pytest.mark.parametrize("name", list(CASES))
def test_emulated(emu_ops, name):
    rows, V, dtype, kind, layout, how = CASES[name]
    check(logits(rows, V, dtype, kind, len(name), layout), numbers(rows, len(name)), **how)


def mixed(rows, device="cpu"):
    """Settings of each row's own, among them values that are taken as the nearest allowed."""
    def turn(values, dtype):
        return torch.tensor(values, dtype=dtype)[torch.arange(rows) % len(values)]
    return dict(temperature=turn([1.0, 0.0, 0.5, -1.0, 1.5, INF, float("nan"), 2.0], torch.float32),
                top_k=turn([0, 5, 1, 40, 10 ** 6, -3, 2], torch.int64 if rows % 2 else torch.int32),
                top_p=turn([1.0, 0.9, 0.5, 0.0, 2.0, -1.0, float("nan")], torch.float32),
                min_p=turn([0.0, 0.1, 0.0, 1.0, 0.02, -2.0, 7.0, float("nan"), 0.0], torch.float32))


def allowed(how):
    """What the values of a row's own count as."""
    t, k, p, m = (how[n].clone() for n in ("temperature", "top_k", "top_p", "min_p"))
    return dict(temperature=torch.where(t > 0, t, 0.0), top_k=k.clamp_min(0), top_p=torch.where(p < 1, p.clamp_min(0.0), 1.0),
                min_p=torch.where(m > 0, m.clamp_max(1.0), 0.0))


def check_mixed(rows, V, device="cpu"):
    x, u, how = logits(rows, V, "bf16", seed=5), numbers(rows, 5), mixed(rows)
    to = lambda t: t.to(device)                                                         # noqa: E731
    got = S.draw(to(x), to(u), **{n: to(v) for n, v in how.items()}, want_logprob=True)
    ids = check(x, u, device, **allowed(how))
    assert torch.equal(got[0], ids)


def test_settings_of_each_row(emu_ops):
    check_mixed(21, 120)


def test_cuts_within_many_equal_logits(emu_ops):
    """More equal logits at the cut than are ranked at once: the lower indices are kept."""
    x, u = logits(2, 4500, "f32", "equal"), torch.tensor([0.9999, 0.3])
    ids = S.sample(x, u, top_k=3001)
    assert ids.tolist() == [math.floor(float(v) * 3001) for v in u.double()]
    ids = S.sample(x, u, top_p=0.75)
    assert ids.tolist() == [math.floor(float(v) * 3375) for v in u.double()]
    x = logits(1, 4500, "bf16", "two", 3)
    check(x, torch.tensor([0.97]), top_k=4000)
    check(x, torch.tensor([0.999]), top_p=0.97)


def fill_lists(dtype, device, V=512):
    """What the next call finds in the workgroup's memory: lists full of ranks above all of its own."""
    S.draw(torch.full((1, V), 1e4, dtype=DT[dtype], device=device), torch.zeros(1, device=device), top_k=V - 100, top_p=0.999)


def check_equal(dtype, lengths, device="cpu"):
    """Rows of one value, of lengths that are ranked at once and of a longer one, with numbers missing at either end, and both cuts: what a row is
    padded with is no token, and what an earlier call left is none either."""
    u = torch.tensor([0.25, 0.75, 0.96875])
    for V in lengths:
        for layout in ("own", "odd"):
            x = logits(3, V, dtype, "equal", 0, layout).zero_()
            fill_lists(dtype, device)
            check(x, u, device, top_k=max(1, V * 3 // 4), top_p=0.9)
            if V < 8:
                continue
            x[0, V - 3:] = -INF                                # fewer numbers than top_k
            x[1, 0] = float("nan")
            x[2, 0], x[2, V - 1] = -INF, -INF
            fill_lists(dtype, device)
            check(x, u, device, top_k=V - 1, top_p=0.9)
            if device != "cpu":                                # (the host build takes half a second for each)
                check(x, u, device, top_k=V - 2)


@pytest.mark.parametrize("dtype", list(DT))
def test_rows_of_one_value(emu_ops, dtype):
    check_equal(dtype, (8, 9, 55, 256))


def check_masked_ends(rows, device="cpu", dtypes=tuple(DT), less=(4, 3, 2, 1)):
    """Rows of one value whose last logits are masked, and more of them asked for than there are: all of them are kept."""
    n, *lengths = rows
    for V in lengths:
        for dtype in dtypes:
            x = torch.zeros(n, V, dtype=DT[dtype])
            x[:, V - 3:] = -INF
            u = numbers(n, V)
            for n_less in less:
                check(x, u, device, top_k=V - n_less, top_p=0.9)
                check(x, u, device, top_k=V - n_less)


def test_masked_ends(emu_ops):
    check_masked_ends((1, 5003, 3003), dtypes=("f32", "bf16"), less=(2,))


def check_lowest(device="cpu", temperatures=(1e-30, 1.0, 3e29, 2e31, 1e36, 3e38)):
    """Logits next to the type's lowest value, masks of that value and of another type's among them, and one at minus infinity."""
    lowest, lower = torch.finfo(torch.float32).min, torch.finfo(torch.bfloat16).min
    u = torch.tensor([0.3, 0.9, 0.02, 0.6])
    f32 = torch.empty(4, 70).uniform_(0.0, 1.0, generator=torch.Generator().manual_seed(4)) * -1e37 - 3.3e38
    f32[1] = torch.where(f32[1] < -3.35e38, lowest, lower)
    f32[2, :60], f32[2, 60:] = lowest, -INF
    f32[3, ::2] = -INF
    pair = torch.tensor([[-3.35e38, -3.40e38]]).expand(4, 2)
    for t in temperatures:
        for x in (f32, pair, f32.clamp_min(lower).bfloat16()):
            check(x, u, device, temperature=t)
            check(x, u, device, temperature=t, top_k=max(1, x.shape[1] // 2), top_p=0.9)


def test_lowest_logits(emu_ops):
    check_lowest()


@pytest.mark.gpu
def test_gpu_lowest_logits():
    check_lowest("cuda", (1e-45, 1e-30, 1e-3, 1.0, 1e20, 1e29, 3e29, 6e29, 1e30, 2e31, 1e33, 1e36, 1e37, 1e38, 3e38))


def check_tiny(lengths, device="cpu"):
    """Subnormal temperatures and logits: distances of which the bins tell few apart, or none."""
    g = torch.Generator().manual_seed(3)
    for V in lengths:
        for size, temperature in ((1e-40, 1e-40), (1e-38, 3e-40), (1e-43, 1e-45), (1e-40, 1e-38), (0.0, 1e-42), (2e-37, 1e-38)):
            x = torch.randn(3, V, generator=g) * size
            x[1, V // 2:] = -INF
            fill_lists("f32", device)
            for how in (dict(top_k=V // 3, top_p=0.9), dict(top_k=V - 5, top_p=0.97), dict(top_k=V * 3 // 4), dict(top_p=0.8)):
                check(x, numbers(3, V), device, temperature=temperature, **how)


def test_tiny_temperatures_and_logits(emu_ops):
    check_tiny((300,))


@pytest.mark.gpu
def test_gpu_rows_of_one_value():
    for dtype in DT:
        check_equal(dtype, (1, 7, 8, 9, 55, 63, 65, 256, 300, 511, 512, 600), "cuda")
    check_masked_ends((1, 5003, 3003, 2049, 20003, 50003), "cuda")
    check_masked_ends((300, 5003), "cuda", less=(2, 1))
    check_tiny((40, 300, 700), "cuda")


def check_written_to(lib, V, calls, ks):
    import threading
    import time
    from analog_moe_amd import _abi
    x = torch.zeros(1, V)
    now = [torch.zeros(1, V), torch.full((1, V), -INF), torch.full((1, V), 3.0), logits(1, V, "f32") * 5]
    done = threading.Event()

    def write():
        while not done.is_set():
            for t in now:
                x.copy_(t)
                time.sleep(2e-3)
    writer = threading.Thread(target=write)
    writer.start()
    try:
        for i in range(calls):
            ids, u = torch.full((1,), -7), torch.tensor([(0.999, 0.5, 0.0)[i % 3]])
            k, p = ks[i % len(ks)]
            args = _abi.SAMPLE_ARGS.pack(0, 1, V, x.data_ptr(), V, u.data_ptr(), 0, 0, 0, 0, 0, 0, 1.0, p, 0.0, k, ids.data_ptr(), 0)
            ws = torch.full((lib.amoe_sample_workspace(args) + 8,), 0xf3, dtype=torch.uint8)
            assert lib.amoe_sample(args, ws.data_ptr(), ws.numel(), None) == 0
            assert -1 <= int(ids) < V, i
    finally:
        done.set()
        writer.join()


def test_rows_written_to_meanwhile(emu_ops):
    """Passes over a row that see other logits each time: the token may be any, but it is one of the row, and the call ends."""
    check_written_to(emu_ops.get_lib(), 600, 18, ((300, 0.9), (300, 1.0), (0, 1.0), (0, 0.5)))


PARTED = {
    # rows worked on in parts: as CASES, and more equal logits at a cut than the parts hand on
    "full": (2, 16500, "f32", "normal", "own", {}),
    "greedy": (2, 17001, "bf16", "coarse", "odd", dict(temperature=0.0)),
    "k": (2, 16500, "f32", "normal", "odd", dict(top_k=700)),
    "p": (2, 17003, "bf16", "masked", "odd", dict(top_p=0.9)),
    "both": (2, 20011, "f16", "normal", "own", dict(top_k=900, top_p=0.8, min_p=0.001)),
    "both_equal": (2, 16400, "f32", "equal", "own", dict(top_k=9000, top_p=0.5)),
    "k_two": (1, 16400, "bf16", "two", "odd", dict(top_k=5000)),
    "p_two": (1, 16400, "f32", "two", "own", dict(top_p=0.97)),
    "cold": (2, 16400, "f32", "normal", "own", dict(top_p=0.6, temperature=1e-30)),
}


def check_parted(names, device="cpu"):
    for name in names:
        if name == "rows":                                # settings of each row's own, infinities and rows of nothing
            how = allowed(mixed(5))
            x = logits(5, 16500, "bf16", seed=5)
            x[1, 400], x[1, 16400] = INF, INF
            how["temperature"][1] = 1.0
            x[4] = -INF
            check(x, numbers(5, 5), device, **how)
            continue
        rows, V, dtype, kind, layout, how = PARTED[name]
        check(logits(rows, V, dtype, kind, len(name), layout), numbers(rows, len(name)), device, **how)


@pytest.mark.parametrize("names", [list(PARTED)[:5], list(PARTED)[5:] + ["rows"]])
def test_rows_in_parts(emu_ops, names):
    """On a device of 64 compute units (a process of its own: the library asks once how many there are)."""
    child = ("import sys\nfrom analog_moe_amd import _abi, ops\nfrom tests import test_emu_kernels as t, test_sampling as f\n"
             "ops._LIB, ops._stream, ops._need_gpu = _abi.bind(t.EMU_SO), (lambda x: None), (lambda *a: None)\n"
             "f.check_parted(sys.argv[1:])\nprint('done')\n")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    got = subprocess.run([sys.executable, "-c", child, *names], cwd=root, env={**os.environ, "AMOE_EMU_CUS": "64"}, capture_output=True, text=True)
    assert got.returncode == 0 and got.stdout.endswith("done\n"), got.stderr


def test_masked_ends_and_written_rows_in_parts(emu_ops):
    """Likewise in parts, with a workspace that may hold anything."""
    child = ("from analog_moe_amd import _abi, ops\nfrom tests import test_emu_kernels as t, test_sampling as f\n"
             "ops._LIB, ops._stream, ops._need_gpu = _abi.bind(t.EMU_SO), (lambda x: None), (lambda *a: None)\n"
             "f.check_masked_ends((1, 16403), dtypes=('bf16',), less=(2,))\n"
             "f.check_written_to(ops._LIB, 16403, 6, ((9000, 0.9), (16390, 0.5)))\nprint('done')\n")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    got = subprocess.run([sys.executable, "-c", child], cwd=root, env={**os.environ, "AMOE_EMU_CUS": "64"}, capture_output=True, text=True)
    assert got.returncode == 0 and got.stdout.endswith("done\n"), got.stderr


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(PARTED) + ["rows"])
def test_gpu_rows_in_parts(name):
    check_parted([name], "cuda")


def test_every_token_has_its_share(emu_ops):
    """u from 0 to 1 in equal steps: each token is drawn as often as its weight says, and in the order of the indices."""
    w = torch.tensor([3.0, 0.0, 1.0, 4.0, 0.0, 8.0])
    x = (w.log() / math.log(2)).expand(16, 6) * math.log(2)
    u = (torch.arange(16) + 0.5) / 16
    assert S.sample(x, u).tolist() == [0] * 3 + [2] + [3] * 4 + [5] * 8
    assert S.sample(x, u, top_k=2).tolist() == [3] * 5 + [5] * 11            # 4 and 8 of 12: 16 / 3 = 5.33 draws


def test_numbers_outside_the_interval(emu_ops):
    x = logits(5, 40, "f32")
    x[:, 39] = -INF
    u = torch.tensor([-1.0, 1.0, 7.0, float("nan"), 0.0])
    ids = S.sample(x, u)
    assert ids.tolist() == [0, 38, 38, 0, 0]
    assert torch.equal(S.sample(x, u.double()), ids)
    assert S.sample(x, u, top_k=1).tolist() == x.argmax(-1).tolist()


def test_rows_of_nothing_and_infinities(emu_ops):
    x = torch.tensor([[-INF, float("nan"), -INF, -INF], [-INF, 1.0, -INF, -INF], [0.0, INF, 3.0, INF], [float("nan")] * 4])
    for how in ({}, dict(top_k=2), dict(top_p=0.9), dict(temperature=0.0), dict(top_p=0.9, top_k=1, min_p=0.3)):
        ids, lp = S.sample(x, torch.full((4,), 0.75), **how, want_logprob=True)
        alone = how.get("top_k") == 1 or "temperature" in how
        assert ids.tolist() == [-1, 1, 1 if alone else 3, -1], how
        assert lp.tolist() == [-INF, 0.0, 0.0 if alone else pytest.approx(-math.log(2), rel=1e-6), -INF], how


def test_shapes_and_strides(emu_ops):
    x, u = logits(12, 50, "f32"), numbers(12)
    want = S.sample(x, u, top_k=9)
    assert torch.equal(S.sample(x.reshape(3, 4, 50), u.reshape(3, 4), top_k=9), want.reshape(3, 4))
    assert torch.equal(S.sample(x.t().contiguous().t(), u, top_k=9), want)
    assert S.sample(x[4], u[4], top_k=9).shape == () and S.sample(x[4], u[4], top_k=9) == want[4]
    assert torch.equal(S.sample(x[2].expand(5, 50), u[2].expand(5), top_k=9), want[2].expand(5))
    assert S.sample(torch.empty(0, 7), torch.empty(0)).shape == (0,)
    two = torch.stack((u, u), 1)
    assert torch.equal(S.sample(x, two[:, 0], temperature=torch.ones(12, 2)[:, 0], top_k=9), want)


def test_gradients_and_watchers(emu_ops):
    x, u = logits(3, 40, "f32").requires_grad_(), numbers(3)
    assert not S.sample(x, u).requires_grad
    with pytest.raises(RuntimeError, match="gradient"):
        S.sample(x, u, want_logprob=True)
    with torch.no_grad():
        ids, lp = S.sample(x, u, want_logprob=True)
        traced = torch.jit.trace(lambda t: S.sample(t, u, top_p=0.9), (x,), check_trace=False)
        assert torch.equal(traced(-x), S.sample(-x, u, top_p=0.9))


def test_refusals(emu_ops):
    x, u = logits(3, 40, "f32"), numbers(3)
    for bad in (dict(temperature=-1.0), dict(temperature=INF), dict(temperature=float("nan")), dict(top_k=-1), dict(top_p=1.5), dict(top_p=-0.1),
                dict(top_p=float("nan")), dict(min_p=2.0), dict(min_p=-1.0), dict(temperature=torch.ones(2)), dict(top_p=torch.ones(3, 1)),
                dict(top_k=torch.ones((), dtype=torch.int64))):
        with pytest.raises(ValueError):
            S.sample(x, u, **bad)
    for bad in (dict(temperature=torch.ones(3, dtype=torch.float64)), dict(top_k=torch.ones(3)), dict(top_k=2.5), dict(min_p=torch.ones(3, dtype=torch.float16))):
        with pytest.raises(TypeError):
            S.sample(x, u, **bad)
    for bad in ((x, u[:2]), (x, u[:, None]), (torch.zeros(3, 0), u), (torch.zeros(1, 1 << 20), u[:1]), (torch.tensor(1.0), u[0])):
        with pytest.raises(ValueError):
            S.sample(*bad)
    for bad in ((x.double(), u), (x.long(), u), (x, u.half())):
        with pytest.raises(TypeError):
            S.sample(*bad)


def test_library_refuses(emu_ops):
    from analog_moe_amd import _abi
    lib = emu_ops.get_lib()
    x, u, ids = logits(4, 16, "f32"), numbers(4), torch.zeros(4, dtype=torch.int64)

    def call(**k):
        f = dict(dtype=0, rows=4, V=16, x=x.data_ptr(), ld=16, u=u.data_ptr(), u64=0, t=0, p=0, m=0, k=0, k64=0, t_all=1.0, p_all=1.0,
                 m_all=0.0, k_all=0, ids=ids.data_ptr(), lp=0)
        f.update(k)
        return lib.amoe_sample(_abi.SAMPLE_ARGS.pack(*f.values()), None, 0, None)
    assert call() == 0 and call(rows=0, x=0) == 0
    for k in (dict(dtype=7), dict(rows=-1), dict(V=0), dict(ld=-1), dict(t_all=-1.0), dict(t_all=float("nan")), dict(p_all=1.1),
              dict(p_all=float("nan")), dict(m_all=-0.5), dict(k_all=-1)):
        assert call(**k) == -1, k
    assert call(x=0) == call(u=0) == call(ids=0) == -2
    assert call(x=x.data_ptr() + 2) == call(u=u.data_ptr() + 4, u64=1) == call(ids=ids.data_ptr() + 4) == call(lp=ids.data_ptr() + 2) == -4
    assert call(t=ids.data_ptr() + 1) == call(k=ids.data_ptr() + 4, k64=1) == -4
    assert call(V=1 << 20) == call(rows=1 << 22) == -6
    assert lib.amoe_sample(None, None, 0, None) == -2


@pytest.mark.gpu
def test_gpu_library_refuses_a_small_workspace():
    """(rows in parts: refused on the host, nothing is launched)"""
    from analog_moe_amd import _abi, ops
    lib = ops.get_lib()
    x, u, ids = torch.zeros(2, 50000, device="cuda"), torch.zeros(2, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    args = _abi.SAMPLE_ARGS.pack(0, 2, 50000, x.data_ptr(), 50000, u.data_ptr(), 0, 0, 0, 0, 0, 0, 1.0, 0.9, 0.0, 0, ids.data_ptr(), 0)
    need = lib.amoe_sample_workspace(args)
    ws = torch.empty(need + 8, dtype=torch.uint8, device="cuda")
    assert need > 0 and need % 8 == 0
    assert lib.amoe_sample(args, None, 0, None) == -2
    assert lib.amoe_sample(args, ws.data_ptr(), need - 1, None) == -5
    assert lib.amoe_sample(args, ws.data_ptr() + 4, need, None) == -4


def test_operator_on_meta():
    ids, lp = torch.ops.amoe.sample(torch.empty(3, 5, 16, device="meta"), torch.empty(3, 5, device="meta"), None, None, None, None, 1.0, 0, 1.0, 0.0)
    assert ids.shape == lp.shape == (3, 5) and ids.dtype == torch.int64


# ------------------------------------------------------------------------------ on the GPU
GPU_CASES = dict(CASES, **{
    "many_full": (700, 8000, "f32", "normal", "own", {}),
    "many_p": (700, 3001, "bf16", "normal", "odd", dict(top_p=0.9, temperature=0.8)),
    "many_k": (600, 5003, "f16", "normal", "every", dict(top_k=50)),
    "many_all": (513, 16384, "bf16", "normal", "own", dict(top_k=2000, top_p=0.95, min_p=0.001)),
    "many_long": (300, 32768, "bf16", "normal", "own", dict(top_k=9000, top_p=0.99)),
    "many_equal": (257, 30001, "f16", "equal", "own", dict(top_k=20000, top_p=0.9)),
    "large_f32": (9, 130001, "f32", "normal", "own", dict(top_k=60000, top_p=0.95, temperature=1.2)),
    "large_bf16": (5, 50001, "bf16", "normal", "own", dict(top_p=0.99)),
    "large_masked": (5, 50001, "f16", "masked", "odd", dict(top_p=0.9, min_p=0.01)),
    "large_coarse": (3, 200000, "f32", "coarse", "own", dict(top_k=30001, top_p=0.97)),
    "parted_f32": (30, 130001, "f32", "normal", "own", dict(top_k=60000, top_p=0.95, temperature=1.2)),
    "parted_bf16": (60, 50001, "bf16", "normal", "odd", dict(top_p=0.99)),
    "parted_full": (7, 200003, "bf16", "normal", "odd", dict(min_p=1e-4)),
    "large_equal": (2, 100003, "bf16", "equal", "own", dict(top_k=77777, top_p=0.9)),
    "large_two": (3, 100003, "f32", "two", "own", dict(top_k=90000, top_p=0.9)),
    "large_rows": (100, 50001, "f32", "masked", "own", dict(top_k=5000, top_p=0.95)),
    "largest": (2, (1 << 20) - 1, "f32", "normal", "own", dict(top_p=0.9)),
    "largest_full": (2, (1 << 20) - 1, "bf16", "equal", "own", {}),
})


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(GPU_CASES))
def test_gpu(name):
    rows, V, dtype, kind, layout, how = GPU_CASES[name]
    check(logits(rows, V, dtype, kind, len(name), layout), numbers(rows, len(name)), "cuda", **how)


@pytest.mark.gpu
def test_gpu_settings_of_each_row():
    check_mixed(63, 5000, "cuda")
    check_mixed(1001, 700, "cuda")


@pytest.mark.gpu
def test_gpu_offsets_past_32_bits():
    x = torch.empty(40 * (1 << 26) + 100, dtype=torch.bfloat16, device="cuda").as_strided((40, 100), (1 << 26, 1))
    own = logits(40, 100, "bf16")
    x.copy_(own)
    u = numbers(40).cuda()
    assert torch.equal(S.sample(x, u, top_p=0.9), S.sample(own.cuda(), u, top_p=0.9))


@pytest.mark.gpu
def test_gpu_stream_graph_and_compile():
    """On another stream, captured (every replay draws by the numbers that u holds then) and compiled."""
    x, u = logits(64, 5000, "bf16").cuda(), numbers(64).cuda()
    how = {n: v.cuda() for n, v in allowed(mixed(64)).items()}

    def work():
        return (*S.sample(x, u, **how, want_logprob=True), S.sample(x, u, temperature=0.7))
    want = work()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = work()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    got = torch.compile(work, fullgraph=True, backend="aot_eager")()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = work()
    for step in range(3):
        u.uniform_()
        x.mul_(0.75)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(work(), held)), step
