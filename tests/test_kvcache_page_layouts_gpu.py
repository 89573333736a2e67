"""Layouts of a paged cache: pools whose pages overlap are refused, interleaved ones are not."""

import pytest
import torch

import flash_attention_interface as fai

pytestmark = pytest.mark.gpu


def test_overlapping_pages_are_refused(device):
    refs = torch.zeros(4, dtype=torch.int32, device=device)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    store = torch.zeros(4 * 8 * 2 * 64, dtype=torch.float16, device=device)
    half = store.as_strided((4, 8, 2, 64), (4 * 2 * 64, 2 * 64, 64, 1))  # each page starts in the middle of the one before
    fine = store.view(4, 8, 2, 64)
    for k, v, name in ((half, fine, "k_cache"), (fine, half, "v_cache")):
        with pytest.raises(RuntimeError, match=f"pages of {name} must not overlap"):
            fai.flash_attn_kvcache_copy_pages(k, v, ints(0), ints(1))
        with pytest.raises(RuntimeError, match=f"pages of {name} must not overlap"):
            fai.flash_attn_kvcache_compact(k, v, torch.full((1, 4), -1, dtype=torch.int32, device=device), refs)
    # Pages whose tokens alternate, and K and V alternating within a token, do not overlap.
    a = torch.arange(4 * 8 * 2 * 2 * 64, device=device).half().view(8, 4, 2, 2, 64).transpose(0, 1)
    k, v = a[:, :, :, 0], a[:, :, :, 1]
    want = a.clone()
    want[1] = want[2]
    fai.flash_attn_kvcache_copy_pages(k, v, ints(2), ints(1))
    assert torch.equal(a, want)
    # Heads that a stride of 0 repeats are one place.
    one = torch.arange(4 * 8 * 64, device=device).half().view(4, 8, 1, 64)
    want = one.clone()
    want[3] = want[0]
    fai.flash_attn_kvcache_copy_pages(one.expand(-1, -1, 2, -1), fine, ints(0), ints(3))
    assert torch.equal(one, want)
