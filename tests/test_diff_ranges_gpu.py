"""Differential attention at the ends of its types' ranges: NaN and infinite scores reach
every output that the definition gives them, gradients of any finite size, scales and
scores of any size.

Bounds are those of oracle/diff.py, and exact equality where a power of two scales
everything that is rounded."""

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


# ---------------------------------------------------------------------------
# Gradients.


def _inputs_and_dout(device, b, sq, sk, h, hk, d, dtype, seed):
    do = torch.randn(b, sq, h, d, generator=torch.Generator().manual_seed(seed + 100)).to(dtype).to(device)
    return *_inputs(device, b, sq, sk, h, hk, d, dtype, seed), do


def _grads(q, k, v, lam, do, causal, scale=None):
    leaves = [x.detach().requires_grad_() for x in (q, k, v, lam)]
    return torch.autograd.grad(fai.flash_diff_attn_func(*leaves, softmax_scale=scale, causal=causal), leaves, do)


@pytest.mark.parametrize("power", [23, 60, 100])
@pytest.mark.parametrize("sq,sk,d,causal", [(70, 90, 64, True), (140, 140, 128, True), (40, 200, 128, False)])
def test_gradients_scale_with_dout(device, sq, sk, d, causal, power):
    """bf16: dO times a power of two gives every gradient times that power, bit for bit."""
    q, k, v, lam, do = _inputs_and_dout(device, 1, sq, sk, 4, 2, d, torch.bfloat16, 7)
    one = _grads(q, k, v, lam, do, causal)
    much = _grads(q, k, v, lam, do * 2.0 ** power, causal)
    for name, x, y in zip(("dq", "dk", "dv", "dlam"), one, much):
        assert torch.equal(x * 2.0 ** power, y), f"{name}: off by up to {float((y / 2.0 ** power - x).abs().max())}"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("size", [64.0, 2000.0])
def test_large_dout(device, dtype, size):
    q, k, v, lam, do = _inputs_and_dout(device, 1, 100, 120, 4, 2, 64, dtype, 8)
    do = do * size
    want = diff_attention(q, k, v, lam, None, True, do)
    for name, x in zip(("dq", "dk", "dv", "dlam"), _grads(q, k, v, lam, do, True)):
        assert_within(name, x, want[name])


# |scale| down to where every score is 0 to fp32, and on both sides of 2^-100; a lam of 0 and a negative one.
@pytest.mark.parametrize("scale", [1e-5, 3e-7, -1e-7, 1e-8, 1e-20, -1e-29, 2.0 ** -99, 2.0 ** -101, 1e-36])
@pytest.mark.parametrize("d,dtype", [(64, torch.float16), (128, torch.bfloat16)])
def test_small_scales(device, d, dtype, scale):
    q, k, v, lam, do = _inputs_and_dout(device, 1, 70, 300, 4, 2, d, dtype, 9)
    lam = torch.tensor([0.0, 0.7, -1.5, 1e-40], device=device)
    want = diff_attention(q, k, v, lam, scale, True, do)
    out = fai.flash_diff_attn_func(q, k, v, lam, softmax_scale=scale, causal=True)
    assert_within("out", out, want["out"])
    for name, x in zip(("dq", "dk", "dv", "dlam"), _grads(q, k, v, lam, do, True, scale)):
        assert_within(name, x, want[name])


@pytest.mark.parametrize("dtype,size,scale", [
    (torch.float16, 1500.0, 1e-7),
    (torch.bfloat16, 1e4, 3e-9),
    (torch.bfloat16, 1e10, -2e-21),
])
def test_large_scores_with_a_small_scale(device, dtype, size, scale):
    """Scores near 1 from products that pass 2^24."""
    q, k, v, lam, do = _inputs_and_dout(device, 1, 90, 150, 4, 2, 64, dtype, 10)
    q, k = q * size, k * size
    assert float((q[0, :, 0, :32].float() @ k[0, :, 0, :32].float().T).abs().max()) > 2.0 ** 24
    want = diff_attention(q, k, v, lam, scale, True, do)
    for name, x in zip(("dq", "dk", "dv", "dlam"), _grads(q, k, v, lam, do, True, scale)):
        assert_within(name, x, want[name])


@pytest.mark.parametrize("d,dtype", [(64, torch.float16), (128, torch.bfloat16)])
def test_a_nan_in_the_gradients(device, d, dtype):
    """A value that is NaN makes D NaN in every row that sees it, and with it dK of every key that those rows see, also
    of the keys whose own products are finite."""
    q, k, v, lam, do = _inputs_and_dout(device, 1, 150, 150, 2, 2, d, dtype, 11)
    want = diff_attention(q, k, v, lam, None, True, do)
    v[0, 0, 1, 3] = float("nan")
    dq, dk, dv, dlam = _grads(q, k, v, lam, do, True)
    assert torch.isnan(dk[:, :, 1]).all() and torch.isnan(dq[:, :, 1]).all() and torch.isnan(dlam[1])
    for name, x in (("dq", dq), ("dk", dk), ("dv", dv)):  # the other head is as it was
        assert_within(name, x[:, :, :1], tuple(y[:, :, :1] for y in want[name]))
