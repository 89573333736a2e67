"""Host-only checks of differential attention and of the cache's pages (no GPU): the
Python layer's refusals, the C ABI's, its struct layouts and workspace sizes."""

import ctypes
import os

import pytest
import torch

import fa_capi
import flash_attention_interface as fai

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20  # an aligned fake device address


def _t(*shape, dtype=torch.float16):
    return torch.zeros(*shape, dtype=dtype)


def _i(*v):
    return torch.tensor(v, dtype=torch.int32)


def test_diff_arguments():
    f = fai.flash_diff_attn_func
    q, k = _t(1, 4, 2, 64), _t(1, 4, 1, 64)
    with pytest.raises(ValueError, match="head_dim 64 or 128"):
        f(_t(1, 4, 2, 96), _t(1, 4, 1, 96), _t(1, 4, 1, 96), torch.zeros(()))
    with pytest.raises(RuntimeError, match="float16 or bfloat16"):
        f(q.float(), k.float(), k.float(), torch.zeros(()))
    with pytest.raises(TypeError, match="lam must be a torch.float32"):
        f(q, k, k, torch.zeros(2, dtype=torch.float16))
    with pytest.raises(TypeError, match="lam must be a torch.float32"):
        f(q, k, k, 0.5)
    with pytest.raises(RuntimeError, match="must be a CUDA"):
        f(q, k, k, torch.zeros(2))
    with pytest.raises(RuntimeError, match="must be a CUDA"):
        fai.flash_diff_attn_varlen_func(q[0], k[0], k[0], torch.zeros(2), _i(0, 4), _i(0, 4), 4, 4)


def test_diff_kvcache_arguments():
    f = fai.flash_diff_attn_with_kvcache
    q, c, lam = _t(1, 1, 2, 64), _t(1, 256, 1, 64), torch.zeros(2)
    new = _t(1, 1, 1, 64)
    with pytest.raises(ValueError, match="both be provided"):
        f(q, c, c, lam, k=new, cache_seqlens=_i(3))
    with pytest.raises(ValueError, match="cache_seqlens is required"):
        f(q, c, c, lam, k=new, v=new)
    with pytest.raises(TypeError, match="cache_seqlens must be a torch.int32"):
        f(q, c, c, lam, cache_seqlens=torch.tensor([3]))
    with pytest.raises(TypeError, match="cache_seqlens must be an int"):
        f(q, c, c, lam, cache_seqlens=[3])
    with pytest.raises(ValueError, match="cache_seqlens must have batch_size rows"):
        f(q, c, c, lam, cache_seqlens=_i(3, 4))
    with pytest.raises(TypeError, match="block_table must be a torch.int32"):
        f(q, c, c, lam, cache_seqlens=_i(3), block_table=torch.zeros(1, 1))
    with pytest.raises(NotImplementedError, match="cache_batch_idx"):
        f(q, c, c, lam, cache_seqlens=_i(3), block_table=_i(0)[None], cache_batch_idx=_i(0))
    with pytest.raises(ValueError, match="num_splits"):
        f(q, c, c, lam, cache_seqlens=_i(3), num_splits=-1)
    # What is wrong with lengths, rows and pages shows on the host before anything runs.
    for lens in (256, -1, 2 ** 31 - 1):
        with pytest.raises(ValueError, match="capacity"):
            f(q, c, c, lam, k=new, v=new, cache_seqlens=_i(lens))
    for row in (-1, 1):
        with pytest.raises(RuntimeError, match="cache_batch_idx"):
            f(q, c, c, lam, cache_seqlens=_i(3), cache_batch_idx=_i(row))
    for page in (-1, 1):
        with pytest.raises(RuntimeError, match="block_table entries in use"):
            f(q, c, c, lam, k=new, v=new, cache_seqlens=_i(256), block_table=_i(0, page)[None])
    with pytest.raises(RuntimeError, match="device|CUDA"):  # entries past the length may be anything
        f(q, c, c, lam, k=new, v=new, cache_seqlens=_i(255), block_table=_i(0, -1)[None])


def test_page_arguments():
    table, lens, refs = torch.full((2, 3), -1, dtype=torch.int32), _i(0, 0), _i(0, 0, 0, 0)
    c = _t(4, 64, 1, 64)
    for call in (
        lambda t: fai.flash_attn_kvcache_alloc(t, lens, refs, 1, 64),
        lambda t: fai.flash_attn_kvcache_free(t, lens, refs, _i(0)),
        lambda t: fai.flash_attn_kvcache_fork(c, c, t, lens, refs, _i(0), _i(1)),
        lambda t: fai.flash_attn_kvcache_compact(c, c, t, refs),
    ):
        with pytest.raises(TypeError, match="block_table must be a torch.int32"):
            call(table.long())
        with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
            call(table)
    with pytest.raises(TypeError, match="src must be a torch.int32"):
        fai.flash_attn_kvcache_copy_pages(c, c, [0], [1])


@pytest.fixture(scope="module")
def lib():
    return fa_capi.load()


def test_struct_layouts(tmp_path):
    import shutil
    import subprocess

    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    structs = {"fa_diff_lam": fa_capi.FaDiffLam, "fa_diff_dlam": fa_capi.FaDiffLam, "fa_diff_fwd_args": fa_capi.FaDiffFwdArgs,
               "fa_diff_bwd_args": fa_capi.FaDiffBwdArgs, "fa_diff_kvcache_args": fa_capi.FaDiffKvcacheArgs,
               "fa_kvpages_args": fa_capi.FaKvpagesArgs}
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


def _tensor(ptr=P, bs=0, rs=1024, hs=128):
    return fa_capi.FaTensor(ptr, bs, rs, hs)


def _fwd(**more):
    a = fa_capi.FaDiffFwdArgs()
    a.q = a.k = a.v = a.o = _tensor()
    a.lam.ptr = a.lse = P
    a.batch, a.seqlen_q, a.seqlen_k, a.nheads, a.nheads_k, a.head_dim, a.lse_seqlen = 1, 8, 8, 4, 2, 128, 8
    for name, x in more.items():
        setattr(a, name, x)
    return a


@pytest.mark.parametrize("want,change", [
    (-2, {"head_dim": 96}), (-2, {"dtype": 2}), (-1, {"nheads_k": 3}), (-1, {"nheads_k": 0}), (-1, {"lse_seqlen": 4}),
    (-1, {"lse": None}), (-1, {"lam": fa_capi.FaDiffLam()}), (-1, {"q": _tensor(P + 8)}), (-1, {"k": _tensor(rs=1020)}),
    (-1, {"o": _tensor(None)}), (-1, {"o2": _tensor(P + 8)}), (-1, {"cu_seqlens_q": P}), (-1, {"seqlen_q": -1}),
    (-1, {"k": _tensor(rs=1 << 24)}), (-1, {"v": _tensor(rs=-1024)}),
])
def test_forward_refusals(lib, want, change):
    assert lib.fa_diff_fwd(ctypes.byref(_fwd(**change)), None) == want
    assert lib.fa_diff_fwd(None, None) == -1


def _bwd(**more):
    a = fa_capi.FaDiffBwdArgs()
    for n in ("q", "k", "v", "o", "o2", "dout", "dq", "dk", "dv"):
        setattr(a, n, _tensor())
    a.lam.ptr = a.lse = a.dsum = P
    a.batch, a.seqlen_q, a.seqlen_k, a.nheads, a.nheads_k, a.head_dim, a.lse_seqlen = 1, 8, 8, 4, 2, 128, 8
    a.dsum_bytes = fa_capi.load().fa_diff_bwd_ws_bytes(ctypes.byref(a))
    for name, x in more.items():
        setattr(a, name, x)
    return a


@pytest.mark.parametrize("want,change", [
    (-2, {"head_dim": 32}), (-2, {"dtype": -1}), (-1, {"nheads_k": 3}), (-1, {"o2": _tensor(None)}), (-1, {"lse": None}),
    (-1, {"dq": _tensor(P + 2)}), (-3, {"dsum": None}), (-3, {"dsum": P + 4}), (-3, {"dsum_bytes": 16}),
    (-1, {"split_ws": P + 128, "split_ws_bytes": 1 << 30}), (-3, {"batch": 70000}),
])
def test_backward_refusals(lib, want, change):
    assert lib.fa_diff_bwd(ctypes.byref(_bwd(**change)), None) == want
    assert lib.fa_diff_bwd(None, None) == -1


def _kv(**more):
    a = fa_capi.FaDiffKvcacheArgs()
    a.q = a.k_cache = a.v_cache = a.o = _tensor()
    a.lam.ptr = a.lse = a.cache_seqlens = P
    a.batch, a.seqlen_q, a.nheads, a.nheads_k, a.head_dim, a.cache_capacity, a.cache_batch = 2, 1, 4, 2, 128, 100, 2
    for name, x in more.items():
        setattr(a, name, x)
    return a


@pytest.mark.parametrize("want,change", [
    (-2, {"head_dim": 96}), (-2, {"dtype": 7}), (-1, {"nheads_k": 3}), (-1, {"num_splits": -1}), (-1, {"cache_seqlens": None}),
    (-1, {"block_table": P, "page_block_size": 100, "num_pages": 4}), (-1, {"block_table": P, "page_block_size": 64}),
    (-1, {"block_table": P, "page_block_size": 64, "num_pages": 4, "cache_batch_idx": P}),
    (-1, {"seqlen_new": 1}), (-1, {"k_cache": _tensor(P + 8)}), (-1, {"v_cache": _tensor(rs=(1 << 23) + 8)}),
    (-3, {"cache_capacity": 100000}),
    (-3, {"cache_capacity": 100000, "ws": P + 16, "ws_bytes": 1 << 30}),
])
def test_kvcache_refusals(lib, want, change):
    assert lib.fa_diff_kvcache(ctypes.byref(_kv(**change)), None) == want
    assert lib.fa_diff_kvcache(None, None) == -1


def test_workspace_sizes(lib):
    size = lambda **m: lib.fa_diff_kvcache_ws_bytes(ctypes.byref(_kv(**m)))  # noqa: E731
    assert size() == 0  # one piece
    # Two pieces of 2 x 2 heads: 4 counters in 256 bytes, then 2 columns a row (2 rows) of (8 + 4 * 128) bytes each.
    assert size(num_splits=2, cache_capacity=256) == 256 + 4 * 2 * 4 * (8 + 512)
    assert lib.fa_diff_kvcache_ws_bytes(None) == 0 and lib.fa_kvpages_ws_bytes(None) == 0
    b = _bwd()
    # 4 bytes (-D_2) and 32 (the products' operands) a row of 4 heads x 8 queries, 8 a head.
    assert lib.fa_diff_bwd_ws_bytes(ctypes.byref(b)) == 4 * 8 * (4 + 32) + 4 * 8
    assert lib.fa_diff_bwd_split_bytes(ctypes.byref(b)) == 0


def _pages(**more):
    a = fa_capi.FaKvpagesArgs()
    a.k_cache = a.v_cache = _tensor(bs=65536, rs=1024, hs=128)
    a.nheads_k, a.head_bytes, a.page_block_size, a.num_pages = 8, 128, 64, 10
    a.block_table = a.cache_seqlens = a.page_refs = P
    a.block_table_stride, a.rows, a.max_pages = 4, 3, 4
    setattr(a, "from", P)
    a.to, a.n = P, 2
    a.out_table, a.out_refs, a.out_used, a.out_table_stride = 2 * P, 2 * P, 3 * P, 4
    a.ws, a.ws_bytes = P, fa_capi.load().fa_kvpages_ws_bytes(ctypes.byref(a))
    for name, x in more.items():
        setattr(a, name, x)
    return a


@pytest.mark.parametrize("entry,want,change", [
    ("alloc", -1, {"cache_seqlens": None}), ("alloc", -1, {"seqlen_new": -1}), ("alloc", -3, {"ws_bytes": 8}), ("alloc", -1, {"page_block_size": 0}),
    ("alloc", -1, {"page_refs": None}), ("copy", -1, {"from": None}), ("copy", -1, {"to": None}), ("copy", -1, {"head_bytes": 24}),
    ("copy", -1, {"k_cache": _tensor(P + 8)}), ("copy", -1, {"v_cache": _tensor(rs=1000)}), ("copy", -1, {"n": -1}),
    ("fork", -1, {"block_table": None}), ("fork", -1, {"rows": 1 << 19}), ("fork", -3, {"ws": None}), ("free", -1, {"from": None}),
    ("free", -1, {"cache_seqlens": None}), ("compact", -1, {"out_used": None}), ("compact", -1, {"out_table": P}),
    ("compact", -1, {"out_refs": P}), ("compact", -3, {"ws_bytes": 60}),
])
def test_page_refusals(lib, entry, want, change):
    f = getattr(lib, "fa_kvpages_" + entry)
    assert f(ctypes.byref(_pages(**change)), None) == want
    assert f(None, None) == -1
