"""Attention at the sizes that launch the kernels' forms for many workgroups: values against the formula in 64 bits, for a sample
of sequences and key heads."""
import os
import subprocess
import sys

import pytest
import torch

from analog_moe_amd import attention as A
from oracle import attention_oracle as O
from tests import test_attention as base
from tests.test_emu_kernels import HERE, emu_ops  # noqa: F401

# rows: waves over the rows of a workgroup that the launches of 256 CUs take (1, 2, 4); copies: those over the queries for dk and dv
CASES = {
    # B, S, T, H, G, d, dtype, layout, options, rows, copies
    "bf16_64": (16, 515, 515, 8, 4, 64, "bf16", "packed", dict(lengths=[515, 77, 0, 514, 513, 300, 64, 65] * 2), 4, 2),
    "f16_64": (9, 961, 961, 8, 4, 64, "f16", "packed", {}, 4, 2),
    "bf16_64_full": (8, 700, 1000, 16, 8, 64, "bf16", "heads", dict(causal=False, lengths=[1000, 991, 1, 0, 64, 500, 999, 640]), 4, 2),
    "f16_80": (6, 1401, 1401, 8, 4, 80, "f16", "packed", dict(lengths=[1401, 1000, 33, 0, 1400, 700]), 4, 2),
    "bf16_96": (16, 515, 515, 8, 4, 96, "bf16", "own", {}, 4, 2),
    "bf16_128": (4, 1030, 1030, 16, 8, 128, "bf16", "packed", {}, 4, 4),
    "f16_128": (9, 515, 700, 16, 2, 128, "f16", "cache", dict(lengths=[700, 650, 1, 0, 699, 64, 65, 128, 129],
                                                              starts=[185, 140, 0, 0, 184, -400, 300, 100, 0]), 4, 4),
    "f32_64": (9, 515, 515, 16, 8, 64, "f32", "packed", {}, 4, 2),
    "f32_72": (9, 500, 515, 16, 8, 72, "f32", "own", dict(lengths=[515, 3, 0, 400, 64, 65, 66, 500, 514]), 4, 2),
    "f32_128": (9, 500, 500, 16, 8, 128, "f32", "own", {}, 4, 2),
    "bf16_64_two": (4, 515, 515, 8, 4, 64, "bf16", "packed", dict(lengths=[515, 400, 0, 65]), 2, 4),
    "f16_80_two": (4, 577, 600, 8, 2, 80, "f16", "own", {}, 2, 4),
    "bf16_128_two": (2, 1003, 2003, 16, 4, 128, "bf16", "cache", dict(lengths=[2003, 1500], starts=[1000, 497]), 2, 4),
    "f16_128_two": (2, 1003, 2003, 16, 4, 128, "f16", "cache", dict(lengths=[2003, 1500], starts=[1000, 497]), 2, 4),
    "f16_128_one": (2, 300, 3000, 16, 4, 128, "f16", "cache", dict(lengths=[3000, 1999], starts=[2700, 1699]), 1, 4),
    "bf16_45": (9, 515, 515, 16, 8, 45, "bf16", "odd", {}, 4, 2),
}


def expected_forms(B, S, T, H, G, d, cus):
    """What the launch rules say, of operands in whole chunks."""
    rows = 4 if B * H * -(-S // 128) >= 2 * cus else 2 if B * H * -(-S // 64) >= cus else 1
    return rows, 2 if B * G * -(-T // 64) > 2 * cus else 4


def check(sizes, dtype, layout, o, device, pairs):
    B, S, T, H, G, d = sizes
    R = H // G
    o = base.options(o)
    kw = dict(causal=o.get("causal", True), lengths=o.get("lengths"), starts=o.get("starts"))
    q, k, v, go = base.inputs(*sizes, dtype, seed=S, layout=layout)
    to = (lambda t: t) if device == "cpu" else base._on_gpu
    on = [to(t) for t in (q, k, v, go)]
    how = {n: t.to(device) if torch.is_tensor(t) else t for n, t in kw.items()}
    left = A.attention_forward(*on[:3], want_lse=True, **how)
    got = left[0], *A.attention_backward(on[3], *on[:3], *left, **how)
    again = A.attention_forward(*on[:3], **how)[0], *A.attention_backward(on[3], *on[:3], *left, **how)
    assert all(torch.equal(a, b) and torch.isfinite(a).all() for a, b in zip(got, again))
    for b, g in pairs:
        one, heads = slice(b, b + 1), slice(g * R, (g + 1) * R)
        part = {n: t[one] if torch.is_tensor(t) else t for n, t in kw.items()}
        want, bounds = O.attention(q[one, :, heads], k[one, :, g:g + 1], v[one, :, g:g + 1], go[one, :, heads], **part)
        mine = got[0][one, :, heads], got[1][one, :, heads], got[2][one, :, g:g + 1], got[3][one, :, g:g + 1]
        base.compare(mine, want, bounds, (sizes, dtype, b, g))


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(CASES))
def test_gpu(name):
    *sizes, dtype, layout, o, rows, copies = CASES[name]
    B, G, d = sizes[0], sizes[4], sizes[5]
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    if cus == 256:
        form = expected_forms(*sizes, cus)
        if dtype != "f32" and d > 96:
            form = form[0], 4                                             # (two copies' tiles have no room beside v)
        assert layout == "odd" or form == (rows, copies)
    # the first sequences, which have the odd lengths, and the last, whose workgroups come last
    check(sizes, dtype, layout, o, "cuda", sorted({(0, 0), (1, G - 1), (B // 2, G // 2), (B - 1, G - 1)}))


# More than 32 rows that share keys, in parts of the key axis and in one.
FEW = {
    "parts_bf16": (1, 100, 2100, 16, 4, 128, "bf16", "cache", dict(lengths=[2090], starts=[1990])),
    "parts_f16": (1, 250, 4200, 16, 4, 64, "f16", "own", {}),
    "parts_f32": (2, 33, 4100, 4, 1, 64, "f32", "own", dict(lengths=[4100, 77], starts=[4067, 50])),
    "one_bf16": (1, 250, 4000, 16, 4, 128, "bf16", "own", {}),
    "one_f16": (4, 100, 2000, 16, 4, 64, "f16", "cache", {}),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(FEW))
def test_gpu_few_rows(name):
    from analog_moe_amd import ops
    *sizes, dtype, layout, o = FEW[name]
    q, k, v = (torch.empty(sizes[0], n, h, sizes[5], dtype=base.DT[dtype], device="cuda") for n, h in
               ((sizes[1], sizes[3]), (sizes[2], sizes[4]), (sizes[2], sizes[4])))
    need = ops.get_lib().amoe_attention_fwd_workspace(A._Call(q, k, v, None, None, True, None).pack(q, None, None))
    if torch.cuda.get_device_properties(0).multi_processor_count == 256:
        assert (need > 0) == name.startswith("parts")
    check(sizes, dtype, layout, o, "cuda", [(0, 0), (sizes[0] - 1, sizes[4] - 1)])


# On one compute unit the same forms are reached by sizes that the host build can run.
SMALL = {
    "bf16_64": (1, 200, 200, 2, 1, 64, "bf16", "packed", {}),
    "f16_64": (2, 140, 230, 1, 1, 64, "f16", "own", dict(lengths=[230, 100])),
    "bf16_96": (1, 260, 260, 1, 1, 80, "bf16", "own", {}),
    "bf16_128": (1, 300, 300, 1, 1, 128, "bf16", "heads", {}),
    "f16_128": (1, 200, 140, 2, 1, 128, "f16", "own", dict(causal=False)),
    "f32_64": (1, 260, 260, 2, 1, 64, "f32", "own", {}),
    "f32_128": (1, 200, 200, 1, 1, 128, "f32", "own", {}),
}


@pytest.mark.parametrize("name", list(SMALL))
def test_emulated(emu_ops, name):
    """(a process of its own: the library asks once how many compute units there are)"""
    child = ("import sys, torch\nfrom analog_moe_amd import _abi, ops\nfrom tests import test_emu_kernels as t, test_attention_forms as f\n"
             "ops._LIB, ops._stream, ops._need_gpu = _abi.bind(t.EMU_SO), (lambda x: None), (lambda *a: None)\n"
             "*sizes, dtype, layout, o = f.SMALL[sys.argv[1]]\n"
             "f.check(sizes, dtype, layout, o, 'cpu', [(0, 0)])\nprint('done')\n")
    got = subprocess.run([sys.executable, "-c", child, name], cwd=os.path.dirname(HERE), env={**os.environ, "AMOE_EMU_CUS": "1"},
                         capture_output=True, text=True)
    assert got.returncode == 0 and got.stdout.endswith("done\n"), got.stderr
