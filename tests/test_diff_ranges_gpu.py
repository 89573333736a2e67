"""Differential attention at the ends of its types' ranges: NaN and infinite scores reach
every output that the definition gives them.  Bounds are those of oracle/diff.py."""

import pytest
import torch

import flash_attention_interface as fai
from oracle.diff import _steps, assert_within, diff_attention

pytestmark = pytest.mark.gpu

HALF = {"1": 0, "2": 1}  # the map whose scores a value spoils


def _inputs(device, b, sq, sk, h, hk, d, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    mk = lambda *s: torch.randn(*s, generator=g).to(dtype).to(device)  # noqa: E731
    lam = (torch.rand(h, generator=g) * 0.6 + 0.2).to(device)
    return mk(b, sq, h, d), mk(b, sk, hk, d), mk(b, sk, hk, d), lam


def _check_rows(name, got, want, bad):
    """got NaN throughout where bad (of got's leading sizes), within its bound elsewhere."""
    assert torch.isnan(got[bad]).all(), f"{name}: {int((~torch.isnan(got[bad])).sum())} elements hide a NaN"
    assert_within(name, torch.where(bad[(...,) + (None,) * (got.dim() - bad.dim())], 0.0, got.double()),
                  tuple(torch.where(bad[(...,) + (None,) * (x.dim() - bad.dim())], 0.0, x) for x in want))


# Grids of one and of two wave groups; a key and a query in the middle of a tile, in its first and its last row.
@pytest.mark.parametrize("which", ["k1", "k2", "q1", "q2", "inf1", "inf2"])
@pytest.mark.parametrize("b,sq,sk,h,hk,d,causal,dtype", [
    (1, 70, 90, 4, 2, 64, True, torch.float16),
    (2, 40, 200, 2, 2, 128, False, torch.bfloat16),
    (5, 130, 140, 64, 64, 64, True, torch.bfloat16),
    (5, 33, 70, 64, 64, 128, False, torch.float16),
])
def test_a_nan_reaches_every_row_that_sees_it(device, b, sq, sk, h, hk, d, causal, dtype, which):
    q, k, v, lam = _inputs(device, b, sq, sk, h, hk, d, dtype, 3)
    m = HALF[which[-1]]
    i, c = b - 1, m * (d // 2) + 5
    if which.startswith("inf"):
        q[..., c] = q[..., c].abs() + 0.25  # scores of +infinity: their softmax is NaN
    want = diff_attention(q, k, v, lam, None, causal)
    see = torch.ones(sq, sk, dtype=torch.bool, device=device)
    if causal:
        see = see.tril(sk - sq)
    for at in (0, sk // 2, sk - 1) if which[0] != "q" else (0, sq // 2, sq - 1):
        q1, k1 = q.clone(), k.clone()
        rows = torch.zeros(b, sq, h, dtype=torch.bool, device=device)
        if which[0] == "q":
            q1[i, at, h - 1, c] = float("nan")
            rows[i, at, h - 1] = bool(see[at].any())
        else:
            k1[i, at, hk - 1, c] = float("inf" if which.startswith("inf") else "nan")
            rows[i, :, h - h // hk:] = see[:, at, None]
        out = fai.flash_diff_attn_func(q1, k1, v, lam, causal=causal)
        _check_rows("out", out, want["out"], rows)


@pytest.mark.parametrize("which", ["k1", "k2", "q1", "q2", "inf1", "inf2"])
@pytest.mark.parametrize("lens,sq,h,hk,d,dtype,splits", [
    ([40, 20], 1, 8, 2, 128, torch.float16, 0),       # one piece
    ([700, 1200], 3, 4, 2, 64, torch.bfloat16, 0),    # several, joined
    ([900, 100], 1, 32, 8, 128, torch.bfloat16, 7),
    ([300, 640], 40, 4, 1, 64, torch.float16, 0),     # several row tiles
    ([350, 640], 300, 4, 4, 128, torch.float16, 0),   # the forward kernel
])
def test_a_nan_in_a_cache(device, lens, sq, h, hk, d, dtype, splits, which):
    cap = 1280
    q, kc, vc, lam = _inputs(device, 2, sq, cap, h, hk, d, dtype, 4)
    m = HALF[which[-1]]
    c = m * (d // 2) + 7
    if which.startswith("inf"):
        q[..., c] = q[..., c].abs() + 0.25
    used = torch.tensor(lens, dtype=torch.int32, device=device)

    def want(n, i):
        return diff_attention(q[i:i + 1], kc[i:i + 1, :n], vc[i:i + 1, :n], lam, None, True)

    n = lens[1]
    for at in (0, n // 2, n - sq) if which[0] != "q" else (0, sq - 1):
        q1, k1 = q.clone(), kc.clone()
        rows = torch.zeros(2, sq, h, dtype=torch.bool, device=device)
        if which[0] == "q":
            q1[1, at, h - 1, c] = float("nan")
            rows[1, at, h - 1] = True
        else:
            k1[1, at, hk - 1, c] = float("inf" if which.startswith("inf") else "nan")
            rows[1, :, h - h // hk:] = (torch.arange(sq, device=device) + n - sq >= at)[:, None]
        out, lse = fai.flash_diff_attn_with_kvcache(q1, k1, vc, lam, cache_seqlens=used, causal=True, num_splits=splits,
                                                    return_softmax_lse=True)
        for j in (0, 1):
            w = want(lens[j], j)
            _check_rows("out", out[j:j + 1], w["out"], rows[j:j + 1])
            spoilt = rows[j:j + 1].transpose(1, 2)
            _check_rows("lse", lse[m, j:j + 1], tuple(x[m] for x in w["lse"]), spoilt)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("m", [0, 1])
@pytest.mark.parametrize("sq,d,dtype", [(1, 64, torch.bfloat16), (3, 128, torch.float16), (40, 128, torch.bfloat16)])
def test_a_key_of_one_map_does_not_reach_the_other(device, sq, d, dtype, m, value):
    h, hk, n = 4, 2, 700
    q, kc, vc, lam = _inputs(device, 1, sq, 1024, h, hk, d, dtype, 6)
    want = diff_attention(q, kc[:, :n], vc[:, :n], lam, None, True)["lse"]
    kc[0, 300, :, m * (d // 2) + 1] = value
    used = torch.tensor([n], dtype=torch.int32, device=device)
    _, lse = fai.flash_diff_attn_with_kvcache(q, kc, vc, lam, cache_seqlens=used, causal=True, return_softmax_lse=True)
    assert_within("lse", lse[1 - m], tuple(x[1 - m] for x in want))


# Scores of -infinity are keys that the map does not see.  Each wave group meets whole tiles of them in one map before
# a tile that mixes them with finite ones.
@pytest.mark.parametrize("m", [0, 1])
@pytest.mark.parametrize("lead", [64, 128, None])  # None: all of them
@pytest.mark.parametrize("b,h,d,dtype", [(1, 2, 64, torch.float16), (5, 64, 64, torch.bfloat16), (5, 64, 128, torch.float16)])
def test_scores_of_minus_infinity(device, b, h, d, dtype, lead, m):
    sq, sk = 40, (lead or 64) + 96
    q, k, v, lam = _inputs(device, b, sq, sk, h, h, d, dtype, 5)
    c = m * (d // 2)
    q[..., c] = 1.0
    hidden = torch.zeros(sk, dtype=torch.bool, device=device)
    hidden[:lead] = True
    if lead:
        hidden[[lead + 6, lead + 36, lead + 66, lead + 95]] = True
    low = k.clone()
    low[:, hidden, :, c] = -float("inf")
    out = fai.flash_diff_attn_func(q, low, v, lam)
    # O_1 - lam O_2 from two calls of the definition without a second map, the first map's channels in front.
    none = torch.zeros_like(lam)
    swap = lambda x: torch.cat((x[..., d // 2:], x[..., : d // 2]), -1)  # noqa: E731
    seen = (k[:, ~hidden], v[:, ~hidden])
    sides = [seen if m == 0 else (k, v), seen if m == 1 else (k, v)]
    o1, o2 = (diff_attention(f(q), f(x), y, none, None, False)["out"] for f, (x, y) in zip((lambda x: x, swap), sides))
    u, t = _steps(dtype)
    val = o1[0] - lam.double()[:, None] * o2[0]
    bound = o1[1] + lam.double()[:, None] * o2[1]
    assert_within("out", out, (val, bound + u * (val.abs() + bound) + t))
