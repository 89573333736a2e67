"""Attention over a KV cache in 8 bits cut into pieces: with a given number of pieces a row's bits do not depend on the batch,
whichever heads a workgroup takes together."""

import pytest
import torch

import flash_attention_interface as fai
from oracle.kv8 import Cache
from test_kv8_gpu import Setup, _check, _widen

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


@pytest.mark.parametrize("kind,d,heads,hk", [("e4m3", 128, 32, 8), ("int8", 64, 8, 4), ("e4m3", 64, 4, 2)])
def test_split_and_whole_sequences(device, kind, d, heads, hk):
    """Batches of which some sequences are split and others not, in both kernels; more sequences than the plan takes at a time."""
    r = torch.Generator().manual_seed(3)
    for lens in ([5000] + [30] * 20, [0, 4000, 0, 700, 2500, 1], [257, 256, 513, 1800, 129], [100] * 270 + [3500, 60, 0, 3600]):
        s = Setup(device, lens, 0, hk, d, kind, 32, "contiguous", held=False)
        for name in ("k", "v"):
            x = s.normal(*s.kc.shape) * (60 if kind == "e4m3" else 30)
            getattr(s, name + "c").copy_((x.clamp(-440, 440) if kind == "e4m3" else x.clamp(-127, 127).round()).to(s.kind))
            getattr(s, name + "s").copy_(torch.rand(s.ks.shape, generator=s.g) * 0.01 + 0.001)
        look = sorted({int(torch.randint(0, len(lens), (1,), generator=r)) for _ in range(3)} |
                      {i for i, n in enumerate(lens) if n > 1000} | {len(lens) - 1})
        for rows in (1, 4, 40):
            q = s.normal(len(lens), rows, heads, d).half().to(device)
            for splits in (0, 3):
                out, lse = fai.flash_attn_with_kvcache_q8(q, *s.caches, cache_seqlens=s.lens, causal=True, num_splits=splits,
                                                          return_softmax_lse=True)
                _check(_Some(s, look), q[look], out[look], lse[look], [lens[i] for i in look], True, (-1, -1), d ** -0.5)


class _Some:
    """Some sequences of a contiguous cache."""

    def __init__(self, s, rows):
        self.s, self.rows = s, rows

    def oracle(self, name):
        return Cache(getattr(self.s, name + "c")[self.rows], getattr(self.s, name + "s")[self.rows])
