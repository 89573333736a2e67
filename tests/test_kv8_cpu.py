"""A KV cache in 8 bits without a GPU: the oracle's quantiser against torch's own conversions and against brute force, its
attention against torch's softmax, the refusals of the Python layer and of the C ABI, the struct layouts and sizes."""

import ctypes
import math
import os
import subprocess

import pytest
import torch

import fa_capi
import flash_attention_interface as fai
from oracle.kv8 import MOST, Cache, attention, encode, scale_for

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20  # an aligned fake device address


@pytest.mark.parametrize("kind", [torch.float8_e4m3fn, torch.int8])
def test_quantiser(kind):
    g = torch.Generator().manual_seed(0)
    codes = torch.arange(256, dtype=torch.uint8).view(kind).double()
    codes = codes[codes.isfinite() & (codes.abs() <= MOST[kind])].unique()
    for top in (1e-30, 2.0 ** -20, 0.3, 1.0, 440.0, 448.0, 449.0, 127.0, 128.0, 6e4):
        x = (torch.rand(200, generator=g) * 2 - 1).double() * top
        x[0] = top
        s = scale_for(top, kind)
        assert math.log2(s) == round(math.log2(s)) and top <= MOST[kind] * s and (top > MOST[kind] * s / 2 or s == 2.0 ** -126)
        e = encode(x, s, kind)
        near = (codes[None] - (x / s)[:, None]).abs().min(1).values
        assert torch.equal((e - x / s).abs(), near)  # the nearest code (ties: below)
        assert torch.equal(e.float().to(kind).double(), e)
    ties = (codes[1:] + codes[:-1]) / 2
    e = encode(ties, 1.0, kind)
    if kind == torch.int8:
        assert (e % 2 == 0).all()
    else:
        assert torch.equal(e, ties.float().to(kind).double())
    for bad in (math.nan, math.inf):
        assert math.isnan(scale_for(bad, kind))
    assert scale_for(0.0, kind) == 2.0 ** -126


def test_blocks_that_grow():
    c = Cache(torch.zeros(1, 64, 1, 64, dtype=torch.int8), torch.full((1, 2, 1), math.nan))
    c.append(0, 0, torch.full((3, 1, 64), 0.5))
    assert float(c.scales[0, 0, 0]) == 2.0 ** -7 and (c.codes[0, :3] == 64).all()
    c.append(0, 3, torch.full((40, 1, 64), -3.0))  # the first block's scale is raised to 2^-5
    assert float(c.scales[0, 0, 0]) == 2.0 ** -5 and (c.codes[0, :3] == 16).all() and (c.codes[0, 3:43] == -96).all()
    assert float(c.scales[0, 1, 0]) == 2.0 ** -5
    assert torch.equal(c.tokens(0, 43)[:, 0, 0], torch.tensor([0.5] * 3 + [-3.0] * 40, dtype=torch.float64))


@pytest.mark.parametrize("causal,window", [(True, (-1, -1)), (False, (-1, -1)), (True, (3, -1)), (False, (2, 1))])
def test_oracle_attention(causal, window):
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(n, h, 64, generator=g) for n, h in ((5, 4), (9, 2), (9, 2)))
    got = attention(q.half(), k.double(), v.double(), 0.1, causal, window)
    for i in range(4):
        s = q.half()[:, i].double() @ k[:, i // 2].double().T * 0.1
        for a in range(5):
            p = a + 4
            for j in range(9):
                if (causal and j > p) or (window[0] >= 0 and j < p - window[0]) or (not causal and window[1] >= 0 and j > p + window[1]):
                    s[a, j] = -math.inf
        assert (got["out"][0][:, i] - s.softmax(1) @ v[:, i // 2].double()).abs().max() < 1e-12
        assert (got["lse"][0][i] - s.logsumexp(1)).abs().max() < 1e-12
    none = attention(q.half(), k[:3].double(), v[:3].double(), 0.1, True)
    assert none["out"][0][:2].abs().max() == 0 and none["out"][1][:2].max() == 0 and none["lse"][0][:, :2].abs().max() == 0


def _t(*shape, dtype=torch.float16):
    return torch.zeros(*shape, dtype=dtype)


def _i(*v):
    return torch.tensor(v, dtype=torch.int32)


def _caches(tokens=256, block=64, lines=1):
    return (*(_t(lines, tokens, 1, 64, dtype=torch.int8) for _ in "kv"), *(torch.zeros(lines, tokens // block, 1) for _ in "kv"))


def test_attention_arguments():
    f, q, c, new = fai.flash_attn_with_kvcache_q8, _t(1, 1, 2, 64), _caches(), _t(1, 1, 1, 64)
    with pytest.raises(ValueError, match="head_dim 64 or 128"):
        f(_t(1, 1, 2, 96), *c)
    with pytest.raises(ValueError, match="both be provided"):
        f(q, *c, k=new, cache_seqlens=_i(3))
    with pytest.raises(ValueError, match="cache_seqlens is required"):
        f(q, *c, k=new, v=new)
    for bad in (torch.tensor([3]), [3], 2.0):
        with pytest.raises(TypeError, match="cache_seqlens must be a torch.int32"):
            f(q, *c, cache_seqlens=bad)
    with pytest.raises(ValueError, match="cache_seqlens must have batch_size rows"):
        f(q, *c, cache_seqlens=_i(3, 4))
    with pytest.raises(TypeError, match="window_size"):
        f(q, *c, cache_seqlens=_i(3), window_size=(1.0, 2))
    with pytest.raises(TypeError, match="block_table must be a torch.int32"):
        f(q, *c, cache_seqlens=_i(3), block_table=torch.zeros(1, 1))
    with pytest.raises(ValueError, match="block_table must have batch_size rows"):
        f(q, *c, cache_seqlens=_i(3), block_table=_i(0))
    with pytest.raises(NotImplementedError, match="cache_batch_idx"):
        f(q, *c, cache_seqlens=_i(3), block_table=_i(0)[None], cache_batch_idx=_i(0))
    with pytest.raises(ValueError, match="num_splits"):
        f(q, *c, cache_seqlens=_i(3), num_splits=-1)
    for lens in (256, -1, 2 ** 31 - 1):
        with pytest.raises(ValueError, match="capacity"):
            f(q, *c, k=new, v=new, cache_seqlens=_i(lens))
    for row in (-1, 1):
        with pytest.raises(RuntimeError, match="cache_batch_idx"):
            f(q, *c, cache_seqlens=_i(3), cache_batch_idx=_i(row))
    for page in (-1, 1):
        with pytest.raises(RuntimeError, match="block_table entries in use"):
            f(q, *c, k=new, v=new, cache_seqlens=_i(256), block_table=_i(0, page)[None])
    with pytest.raises(RuntimeError, match="must be a CUDA"):  # entries past the length may be anything
        f(q, *c, k=new, v=new, cache_seqlens=_i(255), block_table=_i(0, -1)[None])


def test_append_arguments():
    f, c, new = fai.flash_attn_kvcache_append_q8, _caches(), _t(1, 5, 1, 64)
    with pytest.raises(TypeError, match="cache_seqlens must be a torch.int32"):
        f(new, new, *c, 3)
    with pytest.raises(ValueError, match="cache_seqlens must have batch_size rows"):
        f(new, new, *c, _i(3, 4))
    with pytest.raises(TypeError, match="seqlens_new must be a torch.int32"):
        f(new, new, *c, _i(3), seqlens_new=torch.tensor([3]))
    with pytest.raises(ValueError, match="seqlens_new must have batch_size rows"):
        f(new, new, *c, _i(3), seqlens_new=_i(3, 3))
    with pytest.raises(ValueError, match="seqlens_new must not be larger"):
        f(new, new, *c, _i(3), seqlens_new=_i(6))
    with pytest.raises(ValueError, match="capacity"):
        f(new, new, *c, _i(3), seqlens_new=_i(-1))
    with pytest.raises(ValueError, match="capacity"):
        f(new, new, *c, _i(252))
    with pytest.raises(RuntimeError, match="must be a CUDA"):
        f(new, new, *c, _i(252), seqlens_new=_i(4))


def test_read_arguments():
    f, c = fai.flash_attn_kvcache_read_q8, _caches()
    for bad in (torch.tensor([0, 3]), [0, 3]):
        with pytest.raises(TypeError, match="cu_seqlens_k must be a torch.int32"):
            f(*c, bad, 3)
    with pytest.raises(ValueError, match="batch_size \\+ 1"):
        f(*c, _i(), 3)
    with pytest.raises(TypeError, match="dtype"):
        f(*c, _i(0, 3), 3, dtype=torch.float32)
    with pytest.raises(ValueError, match="total_k"):
        f(*c, _i(0, 3), -1)
    for cu in (_i(0, 4), _i(-1, 2), _i(2, 1)):
        with pytest.raises(ValueError, match="cu_seqlens_k must not decrease"):
            f(*c, cu, 3)
    with pytest.raises(ValueError, match="capacity"):
        f(*c, _i(0, 257), 300)
    with pytest.raises(RuntimeError, match="must be a CUDA"):
        f(*c, _i(0, 256), 300)


def _args(**more):
    a = fa_capi.FaKv8Args()
    c = a.cache
    c.k = c.v = a.q = a.o = a.k_new = a.v_new = fa_capi.FaTensor(P, 1 << 20, 1024, 128)
    c.k_scale = c.v_scale = fa_capi.FaKv8Scales(P, 64, 8, 1)
    c.batch, c.nheads_k, c.head_dim, c.scale_block, c.cache_capacity, c.cache_batch = 2, 8, 128, 64, 4096, 2
    a.cache_seqlens = a.lse = a.ws = P
    a.seqlen_new, a.seqlen_q, a.nheads, a.window_left, a.window_right = 1, 1, 32, -1, -1
    a.softmax_scale, a.ws_bytes = 0.1, 1 << 40
    for name, v in more.items():
        setattr(c if hasattr(c, name) else a, name, v)
    return a


@pytest.mark.parametrize("more,code", [
    (dict(head_dim=96), -2), (dict(kind=2), -2), (dict(dtype=2), -2), (dict(batch=-1), -1), (dict(nheads_k=0), -1),
    (dict(nheads=33), -1), (dict(scale_block=16), -1), (dict(scale_block=96), -1), (dict(cache_capacity=4000), -1),
    (dict(cache_capacity=-64), -1), (dict(block_table=P), -1), (dict(block_table=P, page_block_size=96, num_pages=4), -1),
    (dict(block_table=P, page_block_size=64, num_pages=0), -1),
    (dict(block_table=P, page_block_size=64, num_pages=4, cache_batch_idx=P), -1), (dict(k=fa_capi.FaTensor(P + 8, 0, 1024, 128)), -1),
    (dict(v=fa_capi.FaTensor(P, 0, 1032, 128)), -1), (dict(k=fa_capi.FaTensor(P, 0, 1 << 24, 128)), -1),
    (dict(k_scale=fa_capi.FaKv8Scales(None, 0, 0, 0)), -1), (dict(v_scale=fa_capi.FaKv8Scales(P + 2, 0, 0, 0)), -1),
    (dict(cache_seqlens=0), -1), (dict(seqlen_new=-1), -1), (dict(k_new=fa_capi.FaTensor(P + 2, 0, 1024, 128)), -1),
    (dict(lse=0), -1), (dict(q=fa_capi.FaTensor(None, 0, 0, 0)), -1), (dict(o=fa_capi.FaTensor(P + 8, 0, 0, 0)), -1),
    (dict(window_left=-2), -1), (dict(window_right=-2), -1), (dict(num_splits=-1), -1), (dict(seqlens_new=P), -1),
    (dict(ws=0), -3), (dict(ws=P + 128), -3), (dict(ws_bytes=16), -3), (dict(batch=0), 0),
])
def test_c_arguments(more, code):
    lib = fa_capi.load()
    assert lib.fa_kv8_attention(ctypes.byref(_args(**more)), None) == code
    if code and not set(more) & {"nheads", "lse", "q", "o", "window_left", "window_right", "num_splits", "seqlens_new", "ws", "ws_bytes"}:
        assert lib.fa_kv8_append(ctypes.byref(_args(**more)), None) == code
    for name in ("fa_kv8_attention", "fa_kv8_append", "fa_kv8_read"):
        assert getattr(lib, name)(None, None) == -1


def test_c_read_arguments():
    lib, a = fa_capi.load(), fa_capi.FaKv8ReadArgs()
    a.cache, a.k_out, a.v_out, a.cu_seqlens = _args().cache, _args().q, _args().q, P
    for name, v, code in (("total", -1, -1), ("total", 0, 0)):
        setattr(a, name, v)
        assert lib.fa_kv8_read(ctypes.byref(a), None) == code
    a.total = 5
    for name, v, code in (("dtype", 2, -2), ("cu_seqlens", 0, -1), ("k_out", fa_capi.FaTensor(P + 4, 0, 0, 0), -1)):
        old = getattr(a, name)
        setattr(a, name, v)
        assert lib.fa_kv8_read(ctypes.byref(a), None) == code
        setattr(a, name, old)
    a.cache.scale_block = 48
    assert lib.fa_kv8_read(ctypes.byref(a), None) == -1


def test_workspace():
    lib = fa_capi.load()
    size = lambda **more: lib.fa_kv8_ws_bytes(ctypes.byref(_args(**more)))  # noqa: E731
    assert size(batch=0) == size(seqlen_q=0) == size(nheads_k=0) == 0 and lib.fa_kv8_ws_bytes(None) == 0
    # Whatever the capacity, the pieces of a call without num_splits are about as many as the chip has places.
    assert size(cache_capacity=1 << 30) == size(cache_capacity=1 << 20) < 64 << 20
    assert size(cache_capacity=128) < 4096
    assert size(num_splits=64, cache_capacity=1 << 20) > size(num_splits=2, cache_capacity=1 << 20)


def test_struct_layouts(tmp_path):
    import shutil

    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    structs = {"fa_kv8_scales": fa_capi.FaKv8Scales, "fa_kv8_cache": fa_capi.FaKv8Cache, "fa_kv8_args": fa_capi.FaKv8Args,
               "fa_kv8_read_args": fa_capi.FaKv8ReadArgs}
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
