"""Calls of differential attention with nothing to attend from."""

import pytest
import torch

import flash_attention_interface as fai

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
