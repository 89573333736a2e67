"""The calls that plan copies of pages by themselves refuse the codes of a KV cache in 8 bits: its scales would stay behind."""

import pytest
import torch

import flash_attention_interface as fai


@pytest.mark.parametrize("kind", [torch.float8_e4m3fn, torch.int8])
def test_fork_and_compact_refuse_codes(kind):
    codes, half = torch.zeros(4, 64, 2, 64, dtype=kind), torch.zeros(4, 64, 2, 64, dtype=torch.float16)
    ints = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    for pools in ((codes, codes), (codes, half), (half, codes)):
        with pytest.raises(NotImplementedError, match="scales of a cache in 8 bits"):
            fai.flash_attn_kvcache_fork(*pools, ints(2, 2), ints(2), ints(4), ints(1), ints(1))
        with pytest.raises(NotImplementedError, match="scales of a cache in 8 bits"):
            fai.flash_attn_kvcache_compact(*pools, ints(2, 2), ints(4))
    # Other pools, and those of plain bytes, get to the next check.
    for pool in (half, codes.view(torch.uint8)):
        with pytest.raises(RuntimeError, match="CUDA"):
            fai.flash_attn_kvcache_fork(pool, pool, ints(2, 2), ints(2), ints(4), ints(1), ints(1))
        with pytest.raises(RuntimeError, match="CUDA"):
            fai.flash_attn_kvcache_compact(pool, pool, ints(2, 2), ints(4))
