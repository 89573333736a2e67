"""Attention over a KV cache in 8 bits where its softmax can go wrong: scores far from 0, in the kernels of few and of many
query rows, whole and in pieces, elementwise within the roundings that oracle/kv8.py counts."""

import pytest
import torch

import flash_attention_interface as fai
from test_kv8_gpu import Setup, _check

pytestmark = pytest.mark.gpu

ROWS = [1, 70]  # query rows of a KV head: the kernel of few, and of many


def _put(s, k, v):
    """Write k and v [batch][tokens, heads, dim] into an empty cache."""
    for name, x in (("k", k), ("v", v)):
        o = s.oracle(name)
        for i, t in enumerate(x):
            o.append(i, 0, t.to(torch.bfloat16))
        s.put(name, o)


@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("kind,d", [("e4m3", 64), ("e4m3", 128), ("int8", 64), ("int8", 128)])
@pytest.mark.parametrize("levels", [(-120, -120), (-150, -150), (-92, -90), (-90, -92), (-1000, -1000), (-200, -100), (-60, 40)])
def test_scores_far_from_zero(device, levels, kind, d, rows, splits):
    """Every row of a wave has scores near levels[0] in the first half of its keys and near levels[1] in the second: a common
    offset, which softmax does not see.  Some blocks of V are small, or 0."""
    lens, hk, scale = [256, 700], 2, 1 / 16
    s = Setup(device, lens, 0, hk, d, kind, 32, "contiguous", held=False)
    sign = torch.randint(0, 2, (d,), generator=s.g).float() * 2 - 1
    ks, vs = [], []
    for n in lens:
        size = torch.where(torch.arange(n) < n // 2, *(abs(x) / (4 * d * scale) for x in levels))
        turn = torch.where(torch.arange(n) < n // 2, *(torch.tensor(1.0 if x > 0 else -1.0) for x in levels))
        ks.append((size * turn)[:, None, None] * sign + 0.01 * s.normal(n, hk, d))
        v = s.normal(n, hk, d)
        v[64:96] *= 2.0 ** -20
        v[128:160] = 0
        vs.append(v)
    _put(s, ks, vs)
    q = (4 * sign + 0.01 * s.normal(2, rows, 2 * hk, d)).half().to(device)
    out, lse = fai.flash_attn_with_kvcache_q8(q, *s.caches, cache_seqlens=s.lens, causal=True, softmax_scale=scale,
                                              num_splits=splits, return_softmax_lse=True)
    assert (lse < -50).all() or max(levels) > 0
    _check(s, q, out, lse, lens, True, (-1, -1), scale)


@pytest.mark.parametrize("rows", ROWS)
def test_scores_far_from_zero_behind_a_window(device, rows):
    """The first keys that a row sees lie in the middle of a tile that other rows see from its start."""
    d, lens, scale = 128, [500], 1 / 16
    s = Setup(device, lens, 0, 1, d, "e4m3", 64, "paged", held=False)
    sign = torch.randint(0, 2, (d,), generator=s.g).float() * 2 - 1
    level = torch.linspace(180, 100, 500)
    _put(s, [-(level / (4 * d * scale))[:, None, None] * sign + 0.01 * s.normal(500, 1, d)], [s.normal(500, 1, d)])
    q = (4 * sign + 0.01 * s.normal(1, rows, 3, d)).bfloat16().to(device)
    for window, causal in (((40, -1), True), ((3, 0), False), ((0, -1), True)):
        out, lse = fai.flash_attn_with_kvcache_q8(q, *s.caches, cache_seqlens=s.lens, causal=causal, window_size=window,
                                                  softmax_scale=scale, num_splits=2, return_softmax_lse=True, **s.places)
        _check(s, q, out, lse, lens, causal, window, scale)


@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("kind,d", [("e4m3", 64), ("e4m3", 128), ("int8", 64), ("int8", 128)])
@pytest.mark.parametrize("power", [16, 24, 60])
def test_values_that_a_row_does_not_see(device, power, kind, d, rows, splits):
    """Blocks whose V is 2^power times the others': one that rows before it do not see (causal), one that no row's window
    reaches, and one whose keys have no probability to speak of.  The other rows keep all their bits."""
    n, hk, block = 1000, 2, 32
    for where in ("future", "window", "score"):
        s = Setup(device, [n], 0, hk, d, kind, block, "contiguous", held=False)
        k, v = s.normal(n, hk, d), s.normal(n, hk, d)
        q, window = s.normal(1, rows, 2 * hk, d), (-1, -1)
        if where == "future":  # the last block: rows before it see nothing of the 256 tokens from 768 on, or some of them
            v[992:] *= 2.0 ** power
        elif where == "window":
            v[480:512] *= 2.0 ** power  # (of the 256 tokens from 256 on, which rows do not see)
            window = (300, -1)
        else:
            sign = torch.randint(0, 2, (d,), generator=s.g).float() * 2 - 1
            q, k = q + 2 * sign, k + sign
            k[256:288] -= 40 * sign  # exp(-2 40 d / sqrt d): 2^-900 and less
            v[256:288] *= 2.0 ** power
        _put(s, [k], [v])
        q = q.bfloat16().to(device)
        out, lse = fai.flash_attn_with_kvcache_q8(q, *s.caches, cache_seqlens=s.lens, causal=True, window_size=window,
                                                  num_splits=splits, return_softmax_lse=True)
        _check(s, q, out, lse, [n], True, window, d ** -0.5)
        if where == "future":  # what the rows before it are without it
            s.vc[:, 992:], s.vs[:, 31] = 0, 2.0 ** -126
            few = fai.flash_attn_with_kvcache_q8(q, *s.caches, cache_seqlens=s.lens, causal=True, num_splits=splits)
            before = [r for r in range(rows) if n - rows + r < 992]
            a, b = out[:, before].double(), few[:, before].double()
            # Two roundings to bf16, and what fp16's of P may differ by.
            assert ((a - b).abs() <= 2.0 ** -7 * b.abs() + 2.0 ** -10 * 4).all()


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_values_from_small_to_large(device, kind, rows):
    """V grows 2^4 a block, so that every block is another reference, and shrinks again; scores grow and shrink against it."""
    n, d, hk = 640, 64, 1
    for slope in (0.0, 2.0, -2.0, 6.0, -6.0):
        s = Setup(device, [n], 0, hk, d, kind, 32, "contiguous", held=False)
        step = (torch.arange(n) // 32).float()
        v = s.normal(n, hk, d) * 2.0 ** (40 - 4 * (step - 10).abs())[:, None, None]
        sign = torch.randint(0, 2, (d,), generator=s.g).float() * 2 - 1
        k = (slope * (step - 10).abs() / 64)[:, None, None] * sign + 0.1 * s.normal(n, hk, d)
        _put(s, [k], [v])
        q = (sign + 0.1 * s.normal(1, rows, 2, d)).bfloat16().to(device)
        out, lse = fai.flash_attn_with_kvcache_q8(q, *s.caches, cache_seqlens=s.lens, causal=True, softmax_scale=1.0,
                                                  num_splits=1, return_softmax_lse=True)
        _check(s, q, out, lse, [n], True, (-1, -1), 1.0)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("which", ["k", "v"])
def test_scales_that_are_not_finite(device, which, bad, kind, rows):
    """Rows that see a block with such a scale are NaN, also where all of its scores would be -infinity; no others are."""
    n, d, hk = 300, 128, 2
    for alike in (False, True):
        s = Setup(device, [n, n], 0, hk, d, kind, 32, "contiguous", held=False)
        sign = torch.randint(0, 2, (d,), generator=s.g).float() * 2 - 1
        k = [s.normal(n, hk, d) - (4 * sign if alike else 0) for _ in range(2)]
        _put(s, k, [s.normal(n, hk, d) for _ in range(2)])
        q = (s.normal(2, rows, 4, d) + (4 * sign if alike else 0)).bfloat16().to(device)
        args = dict(cache_seqlens=s.lens, causal=True, window_size=(60, -1), num_splits=1)
        want = fai.flash_attn_with_kvcache_q8(q, *s.caches, **args)
        getattr(s, which + "s")[0, 7, 1] = bad  # keys 224 .. 255 of KV head 1
        getattr(s, which + "s")[1, 2, 0] = bad  # keys 64 .. 95: no window reaches back to them from here
        got = fai.flash_attn_with_kvcache_q8(q, *s.caches, **args)
        assert torch.equal(got[1], want[1])
        for r in range(rows):
            pos = n - rows + r
            assert torch.equal(got[0, r, :2], want[0, r, :2])
            if pos >= 224 and pos - 60 <= 255:
                assert got[0, r, 2:].isnan().all(), r
            else:
                assert torch.equal(got[0, r, 2:], want[0, r, 2:]), r
