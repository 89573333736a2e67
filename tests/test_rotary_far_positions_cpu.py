"""Rotary tables end where angles of 64 bits are no longer right in 32: what is refused, in Python and by the C ABI."""

import ctypes

import pytest

import fa_capi
import flash_attention_interface as fai

MOST = 1 << 26


@pytest.mark.parametrize("seqlen,offset", [(1, MOST + 1), (0, MOST + 1), (2, MOST), (100, MOST - 98), (1, -MOST - 1), (4, 1 << 52)])
def test_refused(seqlen, offset):
    with pytest.raises(ValueError, match="2 \\*\\* 26"):
        fai.flash_attn_rotary_tables(seqlen, 32, offset=offset)
    a = fa_capi.FaRotaryTablesArgs()
    a.cos = a.sin = 1 << 20
    a.seqlen, a.rotary_dim, a.base, a.factor, a.attention_factor, a.offset = seqlen, 32, 10000.0, 1.0, 1.0, offset
    assert fa_capi.load().fa_rotary_tables(ctypes.byref(a), None) == -1


@pytest.mark.parametrize("offset", [MOST, -MOST])
def test_the_last_ones_are_taken(offset):
    with pytest.raises(RuntimeError, match="CUDA"):  # (on the CPU: the next check)
        fai.flash_attn_rotary_tables(1, 32, offset=offset, device="cpu")
    a = fa_capi.FaRotaryTablesArgs()
    a.cos = a.sin = 1 << 20
    a.seqlen, a.rotary_dim, a.base, a.factor, a.attention_factor, a.offset = 0, 32, 10000.0, 1.0, 1.0, offset
    assert fa_capi.load().fa_rotary_tables(ctypes.byref(a), None) == 0
