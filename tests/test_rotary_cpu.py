"""Rotary positions without a GPU: the oracle against its derivative and known angles, the refusals of the Python layer and of
the C ABI, the struct layouts."""

import ctypes
import math
import os
import subprocess

import pytest
import torch

import fa_capi
import flash_attention_interface as fai
from oracle.rotary import frequencies, rotate, tables

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20  # an aligned fake device address


@pytest.mark.parametrize("interleaved", [True, False])
def test_oracle_gradient(interleaved):
    g = torch.Generator().manual_seed(0)
    t = tables(9, 16)
    cos, sin = t["cos"][0], t["sin"][0]
    x = torch.randn(5, 2, 24, generator=g, dtype=torch.float64)
    w = torch.randn(5, 2, 24, generator=g, dtype=torch.float64)
    at = [0, 8, 3, None, 1]
    f = lambda z: float((rotate(z, cos, sin, at, interleaved)[0] * w).sum())  # noqa: E731
    grad = rotate(w, cos, sin, at, interleaved, inverse=True)[0]
    for _ in range(40):
        i = tuple(int(torch.randint(0, n, (1,), generator=g)) for n in x.shape)
        d = torch.zeros_like(x)
        d[i] = 1e-5
        assert abs((f(x + d) - f(x - d)) / 2e-5 - float(grad[i])) < 1e-8
    # A rotation and its inverse: x again.
    once = rotate(x, cos, sin, at, interleaved)[0]
    back = rotate(once, cos, sin, at, interleaved, inverse=True)[0]
    keep = [0, 1, 2, 4]
    assert (back - x)[keep].abs().max() < 1e-12
    assert once[3].abs().max() == 0


def test_frequencies():
    assert frequencies(32)[0] == 1 and abs(float(frequencies(32)[8]) - 0.01) < 1e-15
    assert torch.equal(frequencies(32, factor=4.0), frequencies(32) / 4)
    f = frequencies(64, factor=8.0, original_seqlen=4096, low_turns=1.0, high_turns=32.0)
    turns = 4096 * frequencies(64) / (2 * math.pi)
    assert torch.equal(f[turns >= 32], frequencies(64)[turns >= 32])
    assert torch.equal(f[turns <= 1], frequencies(64)[turns <= 1] / 8)
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and (f[mid] < frequencies(64)[mid]).all() and (f[mid] > frequencies(64)[mid] / 8).all()


def test_arguments():
    f, t = fai.flash_attn_rotary_func, fai.flash_attn_rotary_tables
    q, cos = torch.zeros(1, 4, 2, 64, dtype=torch.float16), torch.zeros(8, 16)
    with pytest.raises(TypeError, match="rotary_cos must be a 2-D"):
        f(q, None, None, cos)
    with pytest.raises(TypeError, match="rotary_sin must be a 2-D"):
        f(q, None, cos, cos[0])
    with pytest.raises(TypeError, match="positions must be a torch.int32"):
        f(q, None, cos, cos, positions=torch.zeros(1, 4))
    with pytest.raises(TypeError, match="cu_seqlens must be a torch.int32"):
        f(q[0], None, cos, cos, cu_seqlens=torch.tensor([0, 4]))
    for bad in (torch.zeros(1), 1.5, None):
        with pytest.raises(TypeError, match="seqlen_offsets must be an int"):
            f(q, None, cos, cos, seqlen_offsets=bad)
    with pytest.raises(RuntimeError, match="no gradient"):
        f(q, None, cos.clone().requires_grad_(), cos)
    with pytest.raises(RuntimeError, match="must be a CUDA"):
        f(q, q, cos, cos)
    for bad in (0, 8, 24, 272, -16):
        with pytest.raises(ValueError, match="rotary_dim"):
            t(4, bad)
    with pytest.raises(ValueError, match="seqlen"):
        t(-1, 32)
    with pytest.raises(TypeError, match="dtype"):
        t(4, 32, dtype=torch.float64)
    for more in (dict(base=0.0), dict(factor=0.0), dict(factor=-2.0), dict(base=math.inf), dict(attention_factor=math.nan)):
        with pytest.raises(ValueError, match="base and factor"):
            t(4, 32, **more)
    for more in (dict(original_seqlen=0), dict(original_seqlen=4096, low_turns=2.0, high_turns=2.0)):
        with pytest.raises(ValueError, match="original_seqlen"):
            t(4, 32, **more)
    with pytest.raises(RuntimeError, match="CUDA"):
        t(4, 32, device="cpu")


def _args():
    a = fa_capi.FaRotaryArgs()
    a.q = a.k = a.q_out = a.k_out = fa_capi.FaTensor(P, 0, 1024, 128)
    a.cos = a.sin = P
    a.cos_stride = a.sin_stride = 64
    a.batch, a.seqlen, a.nheads, a.nheads_k, a.head_dim, a.rotary_dim, a.table_rows = 1, 4, 8, 2, 128, 128, 16
    a.table_dtype = 2
    return a


@pytest.mark.parametrize("field,value,code", [
    ("head_dim", 96, -2), ("dtype", 2, -2), ("table_dtype", 3, -2), ("batch", -1, -1), ("seqlen", -1, -1), ("nheads", -1, -1),
    ("rotary_dim", 0, -1), ("rotary_dim", 24, -1), ("rotary_dim", 144, -1), ("table_rows", 0, -1), ("table_rows", -1, -1),
    ("cos", 0, -1), ("sin", P + 4, -1), ("cos_stride", 60, -1), ("q", fa_capi.FaTensor(P + 8, 0, 1024, 128), -1),
    ("q_out", fa_capi.FaTensor(None, 0, 1024, 128), -1), ("k_out", fa_capi.FaTensor(P, 0, 1020, 128), -1), ("batch", 0, 0),
    ("seqlen", 0, 0),
])
def test_c_arguments(field, value, code):
    lib, a = fa_capi.load(), _args()
    setattr(a, field, value)
    assert lib.fa_rotary(ctypes.byref(a), None) == code
    assert lib.fa_rotary(None, None) == -1


@pytest.mark.parametrize("field,value,code", [
    ("seqlen", -1, -1), ("seqlen", 0, 0), ("rotary_dim", 24, -1), ("rotary_dim", 272, -1), ("dtype", 3, -2), ("base", 0.0, -1),
    ("base", math.nan, -1), ("factor", 0.0, -1), ("original_seqlen", -1.0, -1), ("attention_factor", math.inf, -1),
    ("offset", 1 << 53, -1), ("cos", 0, -1), ("sin", P + 8, -1),
])
def test_c_tables_arguments(field, value, code):
    lib, a = fa_capi.load(), fa_capi.FaRotaryTablesArgs()
    a.cos = a.sin = P
    a.seqlen, a.rotary_dim, a.base, a.factor, a.attention_factor = 4, 32, 10000.0, 1.0, 1.0
    setattr(a, field, value)
    assert lib.fa_rotary_tables(ctypes.byref(a), None) == code


def test_struct_layouts(tmp_path):
    import shutil

    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    structs = {"fa_rotary_tables_args": fa_capi.FaRotaryTablesArgs, "fa_rotary_args": fa_capi.FaRotaryArgs}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "fa_mi355x.h"', "int main(void) {"]
    for cname, st in structs.items():
        lines.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in st._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-I", os.path.join(REPO, "include"), str(src), "-o", str(exe)], check=True)
    for line in filter(None, subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split("\n")):
        cname, field, value = line.split()
        st = structs[cname]
        assert int(value) == (ctypes.sizeof(st) if field == "size" else getattr(st, field).offset), line
