"""Host-only checks of calls of differential attention that have nothing to do, and of what
the forward passes on for the backward (no GPU)."""

import ctypes

import pytest
import torch

import fa_capi
import flash_attention_interface as fai

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


@pytest.mark.parametrize("grads", [(1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1), (1, 1, 1, 1), (0, 0, 0, 0)])
@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("packed", [False, True])
def test_what_the_backward_needs_is_kept(monkeypatch, grads, strided, packed):
    """The forward is asked for the second map's output exactly when one of its inputs requires a gradient, whatever
    the layout of the channels, and the backward gets what was kept."""
    asked = []

    class Native:  # stands in for the extension: keeps the calls, returns zeros
        @staticmethod
        def diff_fwd(q, k, v, lam, scale, causal, save):
            assert all(x.stride(-1) == 1 for x in (q, k, v))
            asked.append(save)
            return torch.zeros_like(q), torch.zeros_like(q) if save else None, torch.zeros(2, 1, 2, 3)

        @staticmethod
        def diff_bwd(q, k, v, lam, out, o2, lse, dout, scale, causal, need_dlam):
            assert need_dlam == bool(grads[3])
            return torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), torch.zeros_like(lam)

        @staticmethod
        def diff_varlen_fwd(q, k, v, lam, cu_q, cu_k, max_q, max_k, scale, causal, save):
            return Native.diff_fwd(q, k, v, lam, scale, causal, save)

        @staticmethod
        def diff_varlen_bwd(q, k, v, lam, out, o2, lse, dout, cu_q, cu_k, max_q, max_k, scale, causal, need_dlam):
            return Native.diff_bwd(q, k, v, lam, out, o2, lse, dout, scale, causal, need_dlam)

    monkeypatch.setattr(fai, "flash_attn_gpu", Native)
    shape = (3, 2, 64) if packed else (1, 3, 2, 64)
    mk = lambda: torch.zeros(*shape[:-2], 64, 2).half().transpose(-1, -2) if strided else torch.zeros(shape).half()  # noqa: E731
    inputs = [x.requires_grad_(bool(g)) for x, g in zip((mk(), mk(), mk(), torch.zeros(2)), grads)]
    if packed:
        cu = torch.tensor([0, 3], dtype=torch.int32)
        out = fai.flash_diff_attn_varlen_func(*inputs, cu, cu, 3, 3)
    else:
        out = fai.flash_diff_attn_func(*inputs)
    assert asked == [any(grads)]
    if any(grads):
        out.sum().backward()
        assert all((x.grad is not None) == bool(g) for x, g in zip(inputs, grads))
