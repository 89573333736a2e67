"""The oracle of differential attention (CPU): its values against torch.autograd and
central differences in float64, its bounds against a computation with the roundings
that they count, and closed forms; the page tables' model against its invariants."""

import random

import pytest
import torch

from oracle.diff import Pages, assert_within, diff_attention


def _inputs(b, sq, sk, h, hk, d, kind, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    mk = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
    shape = {"layer": (), "head": (h,), "token": (b, sq, h)}[kind]
    lam = torch.randn(shape, generator=g) * 0.5 + 0.4
    return mk(b, sq, h, d), mk(b, sk, hk, d), mk(b, sk, hk, d), lam, mk(b, sq, h, d)


def _straight(q, k, v, lam, scale, causal):
    """softmax(q1 k1) v - lam softmax(q2 k2) v with torch.softmax, for autograd (no empty rows)."""
    b, sq, h, d = q.shape
    sk, c = k.shape[1], d // 2
    rep = lambda x: x.repeat_interleave(h // k.shape[2], 2).transpose(1, 2)  # noqa: E731
    qh, kh, vh = q.transpose(1, 2), rep(k), rep(v)
    hidden = torch.ones(sq, sk, dtype=torch.bool).triu(sk - sq + 1) if causal else torch.zeros(sq, sk, dtype=torch.bool)
    maps = [torch.softmax((qh[..., m * c:(m + 1) * c] @ kh[..., m * c:(m + 1) * c].transpose(-1, -2) * scale)
                          .masked_fill(hidden, float("-inf")), -1) for m in (0, 1)]
    row = lam.expand(b, sq, h).transpose(1, 2)[..., None]
    return ((maps[0] - row * maps[1]) @ vh).transpose(1, 2)


@pytest.mark.parametrize("kind", ["layer", "head", "token"])
@pytest.mark.parametrize("sq,sk,h,hk,causal", [(5, 7, 4, 2, True), (6, 3, 2, 2, False), (1, 1, 2, 1, True), (4, 4, 3, 1, True)])
def test_values_and_gradients_against_autograd(sq, sk, h, hk, causal, kind):
    q, k, v, lam, do = _inputs(2, sq, sk, h, hk, 8, kind, torch.float16, 3)
    leaves = [x.double().requires_grad_() for x in (q, k, v, lam)]
    out = _straight(*leaves, 0.5, causal)
    grads = torch.autograd.grad(out, leaves, do.double())
    want = diff_attention(q, k, v, lam, 0.5, causal, do)
    for name, x in zip(("out", "dq", "dk", "dv", "dlam"), (out, *grads)):
        torch.testing.assert_close(want[name][0], x.detach(), rtol=1e-12, atol=1e-12)


def test_gradients_against_differences():
    q, k, v, lam, do = _inputs(1, 4, 5, 2, 1, 8, "head", torch.float16, 5)
    want = diff_attention(q, k, v, lam, 0.4, True, do)
    step = 1e-5
    loss = lambda *x: float((_straight(*x, 0.4, True) * do.double()).sum())  # noqa: E731
    base = [x.double() for x in (q, k, v, lam)]
    g = torch.Generator().manual_seed(0)
    for i, name in enumerate(("dq", "dk", "dv", "dlam")):
        for _ in range(4):
            at = tuple(int(torch.randint(n, (1,), generator=g)) for n in base[i].shape)
            hi, lo = [x.clone() for x in base], [x.clone() for x in base]
            hi[i][at] += step
            lo[i][at] -= step
            # Central differences: off by step^2 times a third derivative of order 10, and 1e-16 / step.
            assert abs((loss(*hi) - loss(*lo)) / (2 * step) - float(want[name][0][at])) < 1e-8


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_bounds_hold_for_their_roundings(dtype):
    """fp32 math with P and dS rounded as counted stays within the bounds, and they are not idle: some
    element uses a tenth of its bound."""
    q, k, v, lam, do = _inputs(1, 40, 50, 2, 1, 64, "head", dtype, 7)
    want = diff_attention(q, k, v, lam, None, True, do)
    r = lambda x: x.to(dtype).float()  # noqa: E731
    hidden = torch.ones(40, 50, dtype=torch.bool).triu(11)
    got = {n: torch.zeros(want[n][0].shape) for n in want}
    for h in range(2):
        qf, kf, vf, dof = q[0, :, h].float(), k[0, :, 0].float(), v[0, :, 0].float(), do[0, :, h].float()
        P = []
        for m in (0, 1):
            s = (qf[:, 32 * m:32 * m + 32] @ kf[:, 32 * m:32 * m + 32].T * 32 ** -0.5).masked_fill(hidden, float("-inf"))
            got["lse"][m, 0, h] = torch.logsumexp(s, 1)
            P.append(torch.exp(s - s.amax(1, keepdim=True)))
        O = [r(p) @ vf / p.sum(1, keepdim=True) for p in P]
        P = [p / p.sum(1, keepdim=True) for p in P]
        o = r(O[0] - lam[h] * O[1])
        o2 = r(O[1])
        dp = dof @ vf.T
        d2 = (dof * o2).sum(1, keepdim=True)
        d1 = (dof * o).sum(1, keepdim=True) + lam[h] * d2
        s1, s2 = r(P[0] * (dp - d1)), P[1] * (dp - d2)
        got["out"][0, :, h] = o
        got["dq"][0, :, h] = r(torch.cat((s1 @ kf[:, :32], -lam[h] * (r(s2) @ kf[:, 32:])), 1) * 32 ** -0.5)
        got["dk"][0, :, 0] += torch.cat((s1.T @ qf[:, :32], -(r(lam[h] * s2).T @ qf[:, 32:])), 1) * 32 ** -0.5
        got["dv"][0, :, 0] += r(P[0] - lam[h] * P[1]).T @ dof
        got["dlam"][h] = -(d2 + s2.sum(1, keepdim=True)).sum()
    for name in ("dk", "dv"):
        got[name] = r(got[name])
    for name in want:
        used = assert_within(name, got[name], want[name])
        if name in ("out", "dq", "dk", "dv"):
            assert used > 0.1, (name, used)


def test_closed_forms():
    # One key: o = (1 - lam) v, no gradient of q and k, dlam = -dO . v; no key: zeros.
    q, k, v, lam, do = _inputs(1, 1, 1, 2, 2, 64, "head", torch.float16, 1)
    w = diff_attention(q, k, v, lam, None, True, do)
    torch.testing.assert_close(w["out"][0], (1 - lam.double())[None, None, :, None] * v.double())
    assert w["dq"][0].abs().max() == 0 and w["dk"][0].abs().max() == 0
    torch.testing.assert_close(w["dlam"][0], -(do.double() * v.double()).sum((0, 1, 3)))
    q, k, v, lam, do = _inputs(1, 5, 2, 1, 1, 64, "token", torch.float16, 2)
    w = diff_attention(q, k, v, lam, None, True, do)
    assert w["out"][0][0, :3].abs().max() == 0 and w["lse"][0][:, 0, 0, :3].abs().max() == 0
    assert w["dlam"][0][0, :3].abs().max() == 0 and w["dq"][0][0, :3].abs().max() == 0


def test_pages_model():
    r = random.Random(4)
    m = Pages(40, 4, 8, 10)
    history = [[] for _ in range(8)]
    for _ in range(300):
        op = r.choice(["append", "append", "fork", "free", "compact"])
        live = [i for i in range(8) if m.lens[i]]
        empty = [i for i in range(8) if not m.lens[i] and m.table[i][0] < 0]
        if op == "append" and sum(n == 0 for n in m.refs) > 12:
            row, n = r.randrange(8), r.randrange(1, 6)
            if m.lens[row] + n <= 40:
                m.alloc([n if i == row else 0 for i in range(8)])
                # A page that others share is not written: it is full.
                new = [r.randrange(1000) for _ in range(n)]
                m.append(row, new)
                history[row] += new
        elif op == "fork" and live and empty and 0 in m.refs:
            p, c = r.choice(live), r.choice(empty)
            m.fork([p], [c])
            history[c] = list(history[p])
        elif op == "free":
            row = r.randrange(8)
            m.free([row])
            history[row] = []
        elif op == "compact":
            used = m.compact()
            assert all(n > 0 for n in m.refs[:used]) and not any(m.refs[used:])
        count = [0] * 40
        for row in m.table:
            for p in row:
                if p >= 0:
                    count[p] += 1
        assert count == m.refs
        assert [m.tokens(i) for i in range(8)] == history
