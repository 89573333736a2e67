"""A key-value cache in 8 bits, from its definition, in float64.  Test infrastructure only.

``append`` and ``read`` are exact: scales are powers of two, so that codes and scales have one right value each.
``attention`` gives every output with the error that a kernel may have which computes as documented: scores of exact
products summed in fp32 (e = 2^-23 an operation), scaled, exponentials off by 2^-21 (|s| + |lse| + 1) more, probabilities
times V's scale rounded to fp16 or better (2^-11 relatively; absolutely 2^-30 of the row's largest probability times scale over
the keys that it sees, for each of them), sums in fp32, one rounding of the output (u = eps / 2, t half of the type's smallest
step).  A scale times the largest code is at most twice the largest value of its block, which lies in one of 256 tokens.
"""

import math

import torch

E = 2.0 ** -23
MOST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def scale_for(top: float, kind) -> float:
    """The smallest power of two s >= 2^-126 with top <= most * s; NaN for what is not finite."""
    if not math.isfinite(top):
        return math.nan
    k = -126
    if top > 0:
        k = max(k, math.ceil(math.log2(top / MOST[kind])) - 2)
    while top > MOST[kind] * 2.0 ** k:
        k += 1
    return 2.0 ** k


def encode(x: torch.Tensor, s: float, kind) -> torch.Tensor:
    """x / s rounded to nearest even, as float64 numbers that the codes stand for."""
    v = x.double() / s
    if kind == torch.int8:
        return torch.round(v)
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(v / step) * step


class Cache:
    """codes [lines][tokens][heads][dim] (float64) and scales [lines][blocks][heads] of K or V on the CPU."""

    def __init__(self, codes, scales, index=None, table=None):
        self.kind, self.codes, self.scales = codes.dtype, codes.double().cpu(), scales.double().cpu()
        self.block = codes.shape[1] // scales.shape[1]
        self.index = None if index is None else index.tolist()
        self.table = None if table is None else table.tolist()

    def place(self, b, p):
        if self.table is not None:
            page = self.codes.shape[1]
            return self.table[b][p // page], p % page
        return (b if self.index is None else self.index[b]), p

    def append(self, b, length, x):
        """x [n, heads, dim] behind the first `length` tokens of sequence b."""
        end = length + x.shape[0]
        for start in range(length // self.block * self.block, end, self.block):
            first, stop = max(start, length), min(end, start + self.block)
            if first >= stop:
                continue
            line, row = self.place(b, start)
            for h in range(x.shape[1]):
                new = x[first - length:stop - length, h].double()
                old = float(self.scales[line, row // self.block, h]) if length > start else 2.0 ** -126
                s = scale_for(float(new.abs().max()), self.kind) if bool(new.isfinite().all()) else math.nan
                if math.isnan(s) or math.isnan(old):
                    self.scales[line, row // self.block, h] = math.nan
                    self.codes[line, row + first - start:row + stop - start, h] = 0
                    continue
                s = max(s, old)
                if s != old and length > start:
                    held = slice(row, row + length - start)
                    self.codes[line, held, h] = encode(self.codes[line, held, h] * old, s, self.kind)
                self.codes[line, row + first - start:row + stop - start, h] = encode(new, s, self.kind)
                self.scales[line, row // self.block, h] = s

    def tokens(self, b, n):
        """Values of the first n tokens, [n, heads, dim]."""
        got = []
        for p in range(n):
            line, row = self.place(b, p)
            got.append(self.codes[line, row] * self.scales[line, row // self.block][:, None])
        return torch.stack(got) if got else torch.zeros(0, *self.codes.shape[2:], dtype=torch.float64)


def visible(sq, sk, causal, window):
    p, j = torch.arange(sq)[:, None] + (sk - sq), torch.arange(sk)
    keep = torch.ones(sq, sk, dtype=torch.bool)
    if window[0] >= 0:
        keep &= j >= p - window[0]
    if causal:
        keep &= j <= p
    elif window[1] >= 0:
        keep &= j <= p + window[1]
    return keep


def attention(q, k, v, scale, causal, window=(-1, -1)):
    """q [sq, heads, d] of a 16-bit type, k and v [sk, heads_k, d] in float64: {"out": (value, bound), "lse": ...} with
    out [sq, heads, d] and lse [heads, sq]."""
    sq, h, d = q.shape
    sk, hk = k.shape[:2]
    f = torch.finfo(q.dtype)
    u, t = f.eps / 2, f.smallest_normal * f.eps / 2
    keep = visible(sq, sk, causal, window)
    out, out_b = torch.zeros(sq, h, d, dtype=torch.float64), torch.zeros(sq, h, d, dtype=torch.float64)
    lse, lse_b = torch.zeros(h, sq, dtype=torch.float64), torch.zeros(h, sq, dtype=torch.float64)
    if sk == 0:
        return {"out": (out, out_b), "lse": (lse, lse_b)}
    for i in range(h):
        x, kk, vv = q[:, i].double(), k[:, i // (h // hk)], v[:, i // (h // hk)]
        s = (x @ kk.T * scale).masked_fill(~keep, -math.inf)
        empty = ~keep.any(1)
        top = torch.where(empty, 0.0, s.amax(1))[:, None]
        w = torch.exp(s - top)
        total = w.sum(1, keepdim=True).clamp_min(1e-300)
        p, l = w / total, torch.where(empty[:, None], 0.0, top + torch.log(total))
        err = torch.where(keep, d * E * abs(scale) * (x.abs() @ kk.abs().T) +
                          2.0 ** -21 * (s.nan_to_num(neginf=0.0).abs() + l.abs() + 1), 0.0)
        row = err.amax(1, keepdim=True)
        o = torch.where(keep, p, 0.0) @ torch.where(keep.any(0)[:, None], vv, 0.0)
        a = p @ torch.where(keep.any(0)[:, None], vv.abs(), 0.0)
        size = torch.nn.functional.pad(vv.abs().amax(1), (0, -sk % 256)).view(-1, 256).amax(1).repeat_interleave(256)[:sk]
        floor = 2.0 ** -30 * (torch.where(keep, p, 0.0) * torch.where(keep.any(0), 2 * size, 0.0)).amax(1, keepdim=True)
        acc = (2.0 ** -11 + 2 * row + (2 * sk + 24) * E) * a + floor * keep.sum(1, keepdim=True)
        out[:, i], out_b[:, i] = o, torch.where(empty[:, None], 0.0, acc + u * (o.abs() + acc) + t)
        lse[i], lse_b[i] = l[:, 0], torch.where(empty, 0.0, row[:, 0] + (sk + 16) * E + 2.0 ** -21 * l[:, 0].abs())
    return {"out": (out, out_b), "lse": (lse, lse_b)}
