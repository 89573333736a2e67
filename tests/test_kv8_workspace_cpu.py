"""Workspaces of attention over a KV cache in 8 bits: partial results have places where sequences may be split, and only there."""

import ctypes

import fa_capi
from test_kv8_cpu import _args


def _size(**more):
    return fa_capi.load().fa_kv8_ws_bytes(ctypes.byref(_args(**more)))


def test_calls_whose_sequences_stay_whole():
    # Many rows: a sequence's row tiles fill the chip, and so no sequence is split.  32 bytes a slot.
    for batch, queries, heads in ((64, 2048, 32), (1, 8192, 32), (16, 4096, 64)):
        assert _size(batch=batch, seqlen_q=queries, nheads=heads, cache_capacity=1 << 17) <= 32 * (batch + 2) + 512


def test_partial_results_go_by_the_places_on_the_chip():
    # 4 chunks of 256 queries, 32/8 heads of 128: 64 row tiles of 128 rows a sequence, 8 pieces in all, of which at most 14 are
    # one of several (counts of a split sequence are rounded up), whatever the batch is.
    one = 64 * 128 * (128 * 4 + 8)
    for batch in (4, 64, 256):
        size = _size(batch=batch, seqlen_q=256, cache_capacity=1 << 17)
        assert size <= 14 * one + 32 * (batch + 16) + 4 * 64 * (batch + 14) + 1024
    # One token, 4 rows of 2 heads a workgroup: 4 heads' groups, 128 places at most, twice as many where lengths differ.
    for batch in (4, 64, 1024):
        size = _size(batch=batch, seqlen_q=1, cache_capacity=1 << 17)
        assert size <= 510 * 4 * 8 * (128 * 4 + 8) + 32 * (batch + 256) + 4 * 4 * (batch + 510) + 1024
    # A given number of pieces: every sequence may have as many.
    assert _size(batch=64, num_splits=1) <= 64 * 32 + 512
    assert _size(batch=64, num_splits=4) >= 64 * 4 * 8 * 4 * (128 * 4 + 8)
