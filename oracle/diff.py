"""Differential attention and cache pages, from their definitions.  Test infrastructure only.

``diff_attention``: one call in float64, forward and closed-form backward
(differentiated by hand; tests/test_diff_oracle.py checks it against
``torch.autograd`` and central differences), with a bound on the error of a
kernel that computes as documented: scores, softmax sums and accumulators in
fp32, P and dS rounded to the tensors' 16-bit type before their products, o and
map 2's output stored in that type and read back for D.

The bounds count roundings.  u = eps / 2 is the relative error of one rounding to
16 bits, t half of the type's smallest step (the absolute error below its normal
range), e = 2^-23 one fp32 operation of a sum that may truncate.  A sum of n
products is off by at most n e times the sum of their magnitudes.  With A the sum
of |q||k| of a score, its exponential is off by c e A + 2^-21 (|s| + |lse| + 1)
relatively (c products, the scaling, the LSE and the exponential itself), and a
normalised P by twice the row's largest such error and n e of its sum.

``Pages``: the tables of a paged cache as Python lists.
"""

import math
from typing import Dict, List, Optional, Tuple

import torch

E = 2.0 ** -23


def _steps(dtype: torch.dtype) -> Tuple[float, float]:
    f = torch.finfo(dtype)
    return f.eps / 2, f.smallest_normal * f.eps / 2


def _head(q, k, v, lam, scale, causal, do, u, t):
    """One head of one sequence in float64: q [sq, d], k, v [sk, d], lam [sq, 1], do [sq, d] or None.
    Returns {name: (value, bound)}; dk and dv are this head's contribution, without the final rounding."""
    sq, d = q.shape
    sk, c = k.shape[0], d // 2
    keep = torch.ones(sq, sk, dtype=torch.bool, device=q.device)
    if causal:
        keep = keep.tril(sk - sq)
    zero = torch.zeros(sq, sk, dtype=q.dtype, device=q.device)
    P, EP, lse, lse_b = [], [], [], []
    for m in (0, 1):
        qm, km = q[:, m * c:(m + 1) * c], k[:, m * c:(m + 1) * c]
        s = (qm @ km.T * scale).masked_fill(~keep, -math.inf)
        top = s.amax(1, keepdim=True) if sk else torch.full((sq, 1), -math.inf, dtype=q.dtype, device=q.device)
        empty = top == -math.inf
        x = torch.exp(s - torch.where(empty, 0.0, top))
        total = x.sum(1, keepdim=True)
        l = torch.where(empty, 0.0, torch.where(empty, 0.0, top) + torch.log(total.clamp_min(1e-300)))
        p = torch.where(empty, zero, x / total.clamp_min(1e-300))
        err = torch.where(keep, c * E * abs(scale) * (qm.abs() @ km.abs().T) +
                          2.0 ** -21 * (s.nan_to_num(neginf=0.0).abs() + l.abs() + 1), zero)
        row = err.amax(1, keepdim=True) if sk else torch.zeros_like(l)
        P.append(p)
        EP.append(2 * row + (sk + 16) * E)
        lse.append(l[:, 0])
        lse_b.append(torch.where(empty, 0.0, row + (sk + 16) * E + 2.0 ** -21 * l.abs())[:, 0])
    o2 = P[1] @ v
    o = P[0] @ v - lam * o2
    A = [p @ v.abs() for p in P]
    V = keep.to(q.dtype) @ v.abs()
    acc = [(u + ep + (sk + 8) * E) * a + t * V for ep, a in zip(EP, A)]  # of O_m before its own rounding
    o_b = acc[0] + lam.abs() * acc[1] + 4 * E * (A[0] + lam.abs() * A[1])
    o_b = o_b + u * (o.abs() + o_b) + t
    o2_b = acc[1] + u * (o2.abs() + acc[1]) + t
    got = {"out": (o, o_b), "lse": (torch.stack(lse), torch.stack(lse_b))}
    if do is None:
        return got
    dp = do @ v.T
    F = d * E * (do.abs() @ v.abs().T)
    D = [(p * dp).sum(1, keepdim=True) for p in P]
    d2_b = (do.abs() * o2_b).sum(1, keepdim=True) + (d + 8) * E * (do.abs() * (o2.abs() + o2_b)).sum(1, keepdim=True)
    d1_b = (do.abs() * o_b).sum(1, keepdim=True) + lam.abs() * d2_b + \
        (d + 8) * E * ((do.abs() * (o.abs() + o_b)).sum(1, keepdim=True) + lam.abs() * D[1].abs())
    dS, dS_b = [], []
    for m, db in ((0, d1_b), (1, d2_b)):
        x = (dp - D[m]).abs()
        dS.append(P[m] * (dp - D[m]))
        b = P[m] * (EP[m] * x + F + db + 4 * E * (dp.abs() + D[0].abs() + D[1].abs()))
        dS_b.append(b + u * (dS[m].abs() + b))
    n = sk + 8
    la = lam.abs()
    dq, dq_b, dk, dk_b = [], [], [], []
    for m, f in ((0, torch.ones_like(lam)), (1, -lam)):
        qm, km = q[:, m * c:(m + 1) * c], k[:, m * c:(m + 1) * c]
        fa = f.abs()
        w = f * (dS[m] @ km) * scale
        b = abs(scale) * fa * ((dS_b[m] + t * keep + n * E * dS[m].abs()) @ km.abs())
        dq.append(w)
        dq_b.append(b + (u + 4 * E) * (w.abs() + b) + t)
        dk.append((f * dS[m]).T @ qm * scale)
        dk_b.append(abs(scale) * ((fa * dS_b[m] + t * keep + (sq + 8) * E * fa * dS[m].abs()).T @ qm.abs()))
    mix = P[0] - lam * P[1]
    mix_b = EP[0] * P[0] + la * EP[1] * P[1] + 4 * E * (P[0] + la * P[1])
    mix_b = mix_b + u * (mix.abs() + mix_b) + t * keep
    x = (dp - D[1]).abs()
    dl_b = (P[1] * ((EP[1] + (sk + 8) * E) * x + F)).sum(1) + (EP[1] * d2_b)[:, 0] + \
        (d + 16) * E * ((do.abs() * A[1]).sum(1) + D[1].abs()[:, 0])
    got.update(dq=(torch.cat(dq, 1), torch.cat(dq_b, 1)), dk=(torch.cat(dk, 1), torch.cat(dk_b, 1)),
               dv=(mix.T @ do, (mix_b + (sq + 8) * E * mix.abs()).T @ do.abs()), dlam=(-D[1][:, 0], dl_b))
    return got


def diff_attention(q, k, v, lam, scale: Optional[float], causal: bool, dout=None) -> Dict[str, Tuple[torch.Tensor, torch.Tensor]]:
    """q [b, sq, h, d], k, v [b, sk, hk, d] in a 16-bit type, lam a scalar, [h] or [b, sq, h].
    Returns {name: (float64 value, bound)} for out, lse [2, b, h, sq] and, with dout, dq, dk, dv, dlam."""
    b, sq, h, d = q.shape
    sk, hk = k.shape[1], k.shape[2]
    scale = (d // 2) ** -0.5 if scale is None else scale
    u, t = _steps(q.dtype)
    f = lambda *s: torch.zeros(s, dtype=torch.float64, device=q.device)  # noqa: E731
    full = lam.double().expand(b, sq, h)
    got = {"out": (f(b, sq, h, d), f(b, sq, h, d)), "lse": (f(2, b, h, sq), f(2, b, h, sq))}
    if dout is not None:
        got.update(dq=(f(b, sq, h, d), f(b, sq, h, d)), dk=(f(b, sk, hk, d), f(b, sk, hk, d)),
                   dv=(f(b, sk, hk, d), f(b, sk, hk, d)))
        rows = (f(b, sq, h), f(b, sq, h))
    for i in range(b):
        for j in range(h):
            g = j // (h // hk)
            r = _head(q[i, :, j].double(), k[i, :, g].double(), v[i, :, g].double(), full[i, :, j, None], scale, causal,
                      None if dout is None else dout[i, :, j].double(), u, t)
            for x in (0, 1):
                got["out"][x][i, :, j] = r["out"][x]
                got["lse"][x][:, i, j] = r["lse"][x]
                if dout is not None:
                    got["dq"][x][i, :, j] = r["dq"][x]
                    got["dk"][x][i, :, g] += r["dk"][x]
                    got["dv"][x][i, :, g] += r["dv"][x]
                    rows[x][i, :, j] = r["dlam"][x]
    if dout is not None:
        for name in ("dk", "dv"):
            val, bound = got[name]
            bound += (u + 4 * E) * (val.abs() + bound) + t
        if lam.dim() == 3:
            got["dlam"] = rows
        else:
            over = (0, 1, 2) if lam.dim() == 0 else (0, 1)
            val, bound = rows[0].sum(over), rows[1].sum(over)
            got["dlam"] = (val, bound + 2.0 ** -23 * val.abs())
    return got


def assert_within(name: str, got: torch.Tensor, want: Tuple[torch.Tensor, torch.Tensor]) -> float:
    """Every element of got within its bound; returns the largest share of a bound that is used."""
    val, bound = want
    assert got.shape == val.shape, (name, got.shape, val.shape)
    if got.numel() == 0:
        return 0.0
    x = got.detach().to(val.device).double()
    assert torch.isfinite(x).all(), f"{name}: non-finite"
    share = ((x - val).abs() / bound.clamp_min(1e-300)).where((x - val).abs() > 0, torch.zeros_like(bound))
    worst = share.max().item()
    assert worst <= 1.0, f"{name}: error {worst:.3g} times its bound at {(share == share.max()).nonzero()[0].tolist()}"
    return worst


class Pages:
    """A paged cache: rows of pages, lengths and reference counts, and the tokens' contents as numbers."""

    def __init__(self, num_pages: int, page: int, rows: int, width: int):
        self.page, self.width = page, width
        self.table: List[List[int]] = [[-1] * width for _ in range(rows)]
        self.lens = [0] * rows
        self.refs = [0] * num_pages
        self.data = [[0] * page for _ in range(num_pages)]

    def take(self) -> int:
        p = self.refs.index(0)
        self.refs[p] = 1
        return p

    def alloc(self, new: List[int]) -> None:
        for r, n in enumerate(new):
            for j in range(self.lens[r] // self.page, -(-(self.lens[r] + n) // self.page) if n else 0):
                if self.table[r][j] < 0:
                    self.table[r][j] = self.take()

    def append(self, r: int, tokens: List[int]) -> None:
        for x in tokens:
            self.data[self.table[r][self.lens[r] // self.page]][self.lens[r] % self.page] = x
            self.lens[r] += 1

    def fork(self, parents: List[int], children: List[int]) -> None:
        for p, c in zip(parents, children):
            for j in range(self.lens[p] // self.page):
                self.table[c][j] = self.table[p][j]
                self.refs[self.table[p][j]] += 1
            self.lens[c] = self.lens[p]
        for p, c in zip(parents, children):
            j, rest = divmod(self.lens[p], self.page)
            if rest:
                self.table[c][j] = x = self.take()
                self.data[x][:rest] = self.data[self.table[p][j]][:rest]

    def free(self, rows: List[int]) -> None:
        for r in rows:
            for p in self.table[r]:
                if p >= 0:
                    self.refs[p] -= 1
            self.table[r], self.lens[r] = [-1] * self.width, 0

    def compact(self) -> int:
        used = sum(n > 0 for n in self.refs)
        free = [p for p in range(used) if self.refs[p] == 0]
        moved = dict(zip((p for p in range(used, len(self.refs)) if self.refs[p]), free))
        for old, new in moved.items():
            self.data[new] = list(self.data[old])
            self.refs[new], self.refs[old] = self.refs[old], 0
        self.table = [[moved.get(p, p) for p in row] for row in self.table]
        return used

    def tokens(self, r: int) -> List[int]:
        return [self.data[self.table[r][i // self.page]][i % self.page] for i in range(self.lens[r])]
