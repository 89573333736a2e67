"""Attention over a KV cache in 8 bits cut into pieces: with a given number of pieces a row's bits do not depend on the batch,
whichever heads a workgroup takes together."""

import pytest
import torch

import flash_attention_interface as fai
from test_kv8_gpu import Setup, _widen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("splits", [7, 16, 33, 64, 100, 200])
@pytest.mark.parametrize("kind,d,hk,batch,capacity", [
    # Tables so wide that a batch takes two KV heads a workgroup where a sequence alone takes one, pages of a few.
    ("e4m3", 64, 2, 9, 32768), ("int8", 64, 8, 4, 16384), ("e4m3", 128, 2, 9, 262144), ("int8", 128, 4, 4, 262144),
])
def test_a_rows_bits_do_not_depend_on_the_batch(device, kind, d, hk, batch, capacity, splits):
    page = 64
    lens = [13000 - 1500 * i for i in range(4)] + [900] * (batch - 4)
    s = Setup(device, lens, 0, hk, d, kind, 32, "paged", page=page, capacity=13056, held=False)
    for name in ("k", "v"):  # any codes and scales will do
        x = s.normal(*s.kc.shape) * (60 if kind == "e4m3" else 30)
        getattr(s, name + "c").copy_((x.clamp(-440, 440) if kind == "e4m3" else x.clamp(-127, 127).round()).to(s.kind))
        getattr(s, name + "s").copy_(torch.rand(s.ks.shape, generator=s.g) * 0.02 + 0.001)
    _widen(s, capacity - 13056, page)
    for rows in (1, 5, 40):  # (of 2, 10 and 80 rows of a KV head: few, few and many)
        q = s.normal(batch, rows, 2 * hk, d).half().to(device)
        args = dict(causal=True, num_splits=splits, return_softmax_lse=True)
        out, lse = fai.flash_attn_with_kvcache_q8(q, *s.caches, cache_seqlens=s.lens, block_table=s.table, **args)
        for i in range(batch):
            one = fai.flash_attn_with_kvcache_q8(q[i:i + 1], *s.caches, cache_seqlens=s.lens[i:i + 1],
                                                 block_table=s.table[i:i + 1], **args)
            assert torch.equal(out[i:i + 1], one[0]) and torch.equal(lse[i:i + 1], one[1]), (rows, i)
