"""Rotary tables at the last positions that they may have, against angles of 64 bits of mantissa (numpy's long double)."""

import numpy as np
import pytest
import torch

import flash_attention_interface as fai

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("more", [{}, dict(base=500000.0, factor=4.0), dict(factor=32.0, original_seqlen=4096, attention_factor=1.35)])
@pytest.mark.parametrize("offset", [2 ** 26 - 300, -(2 ** 26), 2 ** 22 + 1])
def test_far_positions(device, offset, more, dtype):
    if np.finfo(np.longdouble).nmant < 63:
        pytest.skip("long double has no more bits than double")
    n, dim, low, high = 301, 128, 1.0, 32.0
    ld = np.longdouble
    f = ld(more.get("base", 10000.0)) ** (-2 * np.arange(dim // 2, dtype=ld) / dim)
    keep = np.zeros(dim // 2, dtype=ld)
    if "original_seqlen" in more:
        keep = np.clip((more["original_seqlen"] * f / (2 * ld(np.pi)) - low) / ld(high - low), 0, 1)
    f = f * (keep + (1 - keep) / ld(more.get("factor", 1.0)))
    angle = np.outer(np.arange(offset, offset + n, dtype=ld), f)
    size = more.get("attention_factor", 1.0)
    got = fai.flash_attn_rotary_tables(n, dim, offset=offset, dtype=dtype, device=device, **more)
    t = torch.finfo(dtype)
    for x, y in zip(got, (np.cos(angle), np.sin(angle))):
        want = torch.from_numpy((y * ld(size)).astype(np.float64))
        # The angle's 2^-51 of itself (half of a step of fp32 at 2^26), a Taylor sum's 2^-36, one rounding.
        bound = size * (2.0 ** -51 * (2 ** 26) + 2.0 ** -36) + t.eps / 2 * want.abs() + t.smallest_normal * t.eps / 2
        worst = float(((x.double().cpu() - want).abs() - bound).max())
        assert worst <= 0, f"over its bound by {worst:.3g}"
