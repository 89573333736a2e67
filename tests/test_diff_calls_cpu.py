"""Host-only checks of calls of differential attention that have nothing to do (no GPU)."""

import ctypes

import pytest

import fa_capi

P = 1 << 20  # an aligned fake device address


@pytest.mark.parametrize("want,change", [
    (0, {"batch": 0, "seqlen_new": 3}), (0, {"batch": 0, "seqlen_q": 1}),  # no sequences: nothing has an address
    (0, {"seqlen_q": 0}),                                                    # neither queries nor new tokens
    (-1, {"seqlen_q": 1}), (-1, {"seqlen_new": 2}),                          # no q; no new tokens to append
    (-1, {"batch": 0, "num_splits": -1}), (-2, {"batch": 0, "head_dim": 96}),
])
def test_kvcache_without_queries_or_sequences(want, change):
    a = fa_capi.FaDiffKvcacheArgs()
    a.batch, a.nheads, a.nheads_k, a.head_dim, a.cache_capacity, a.cache_batch = 2, 4, 2, 128, 100, 2
    if change.get("batch") != 0:
        a.k_cache = a.v_cache = fa_capi.FaTensor(P, 0, 1024, 128)
        a.cache_seqlens = P
    for name, x in change.items():
        setattr(a, name, x)
    assert fa_capi.load().fa_diff_kvcache(ctypes.byref(a), None) == want
