"""Calls of differential attention with nothing to attend from or over, and with layouts that
need a copy."""

import pytest
import torch

import flash_attention_interface as fai
from oracle.diff import assert_within, diff_attention

pytestmark = pytest.mark.gpu


def _mk(device, *shape, seed=0, dtype=torch.float16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(device)


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("kind", ["layer", "head", "token"])
def test_append_without_queries(device, paged, kind):
    b, h, hk, d, new = 3, 4, 2, 64, 5
    kc, vc = _mk(device, 6, 256, hk, d, seed=1), _mk(device, 6, 256, hk, d, seed=2)
    if not paged:
        kc, vc = kc[:b].contiguous(), vc[:b].contiguous()
    table = torch.tensor([[3], [0], [5]], dtype=torch.int32, device=device) if paged else None
    lens = torch.tensor([0, 250, 17], dtype=torch.int32, device=device)
    k, v = _mk(device, b, new, hk, d, seed=3), _mk(device, b, new, hk, d, seed=4)
    lam = torch.zeros({"layer": (), "head": (h,), "token": (b, 0, h)}[kind], device=device)
    wk, wv = kc.clone(), vc.clone()
    for i, n in enumerate(lens.tolist()):
        page = int(table[i, 0]) if paged else i
        wk[page, n:n + new], wv[page, n:n + new] = k[i], v[i]
    for validate in (True, False):
        fai.flash_attn_kvcache_check()
        for q in (torch.empty(b, 0, h, d, dtype=torch.float16, device=device), _mk(device, b, 2, h, d)[:, :0]):
            gk, gv = kc.clone(), vc.clone()
            out, lse = fai.flash_diff_attn_with_kvcache(q, gk, gv, lam, k, v, cache_seqlens=lens, block_table=table,
                                                        causal=True, return_softmax_lse=True, validate=validate)
            assert out.shape == q.shape and lse.shape == (2, b, h, 0)
            assert torch.equal(gk, wk) and torch.equal(gv, wv)
        fai.flash_attn_kvcache_check()


@pytest.mark.parametrize("sq", [0, 1])
def test_append_without_sequences(device, sq):
    q, k = _mk(device, 0, sq, 4, 64), _mk(device, 0, 1, 2, 64)
    lens = torch.zeros(0, dtype=torch.int32, device=device)
    pool = _mk(device, 3, 256, 2, 64)
    for c, table in ((pool, torch.zeros(0, 2, dtype=torch.int32, device=device)), (pool[:0], None)):
        out, lse = fai.flash_diff_attn_with_kvcache(q, c, c.clone(), torch.zeros(4, device=device), k, k,
                                                    cache_seqlens=lens, block_table=table, return_softmax_lse=True)
        assert out.shape == q.shape and lse.shape == (2, 0, 4, sq)


@pytest.mark.parametrize("max_q,max_k", [(0, 8), (8, 0), (0, 0)])
@pytest.mark.parametrize("kind", ["layer", "head", "token"])
def test_packed_maxima_of_zero(device, max_q, max_k, kind):
    # Sequences are cut to the call's maxima: no row sees a key, and outputs and gradients are 0.
    rows, h, hk, d = 9, 4, 2, 128
    lam = torch.rand({"layer": (), "head": (h,), "token": (rows, h)}[kind]).to(device)
    leaves = [x.requires_grad_() for x in (_mk(device, rows, h, d), _mk(device, rows, hk, d), _mk(device, rows, hk, d), lam)]
    for cu in ([0, 0, 0], [0, 4, 9]):
        cu = torch.tensor(cu, dtype=torch.int32, device=device)
        out = fai.flash_diff_attn_varlen_func(*leaves, cu, cu, max_q, max_k, causal=True)
        assert out.shape == (rows, h, d) and not out.any()
        for x, g in zip(leaves, torch.autograd.grad(out, leaves, torch.ones_like(out))):
            assert g.shape == x.shape and not g.any()


@pytest.mark.parametrize("packed", [False, True])
def test_gradients_of_strided_channels(device, packed):
    # q, k and v whose last dimension is strided are copied; all of them get gradients, lam none.
    b, s, h, d = 2, 50, 2, 64
    base = [_mk(device, b, s, d, h, seed=i).transpose(2, 3) for i in range(3)]
    do, lam = _mk(device, b, s, h, d, seed=5), torch.rand(h).to(device)
    want = diff_attention(*(x.contiguous() for x in base), lam, None, True, do)
    leaves = [x.detach().requires_grad_() for x in base]
    assert all(x.stride(-1) != 1 for x in leaves)
    if packed:
        cu = torch.tensor([0, s, 2 * s], dtype=torch.int32, device=device)
        flat = [x.flatten(0, 1) for x in leaves]
        assert all(x.stride(-1) != 1 for x in flat)
        out = fai.flash_diff_attn_varlen_func(*flat, lam, cu, cu, s, s, causal=True).view(b, s, h, d)
    else:
        out = fai.flash_diff_attn_func(*leaves, lam, causal=True)
    grads = torch.autograd.grad(out, leaves, do)
    for name, x in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        assert_within(name, x, want[name])
