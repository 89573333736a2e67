"""Decode of differential attention keeps its probabilities in 32 bits through the product with V, as ordinary
attention over a cache does: its outputs are held to the definition with one rounding to 16 bits, the last one."""

import pytest
import torch

import flash_attention_interface as fai
from oracle.diff import _head, _steps, assert_within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,sq,h,hk,d,splits", [
    ([900, 37], 1, 8, 2, 128, 0),
    ([2000, 1], 2, 4, 4, 64, 5),
    ([300, 700], 4, 16, 1, 64, 1),  # four row tiles
])
def test_one_rounding(device, lens, sq, h, hk, d, splits, dtype):
    g = torch.Generator().manual_seed(12)
    mk = lambda *s: torch.randn(*s, generator=g).to(dtype).to(device)  # noqa: E731
    q, kc, vc = mk(2, sq, h, d), mk(2, 2048, hk, d), mk(2, 2048, hk, d)
    lam = torch.rand(h, generator=g).to(device)
    out = fai.flash_diff_attn_with_kvcache(q, kc, vc, lam, cache_seqlens=torch.tensor(lens, dtype=torch.int32, device=device),
                                           causal=True, num_splits=splits)
    u, t = _steps(dtype)
    for i, n in enumerate(lens):
        for j in range(h):
            k, v = kc[i, :n, j // (h // hk)].double(), vc[i, :n, j // (h // hk)].double()
            # P as the sum of its rounding and the rounding of what that leaves: u^2 of it, or t.
            val, bound = _head(q[i, :, j].double(), k, v, lam[j].double().expand(sq, 1), (d // 2) ** -0.5, True, None, u * u,
                               t)["out"]
            assert_within(f"sequence {i}, head {j}", out[i, :, j], (val, bound + u * (val.abs() + bound) + t))
