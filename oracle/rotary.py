"""Rotary positions from their definition, in float64.  Test infrastructure only.

Every value comes with the error that a kernel may have that computes as documented: the
rotation in fp32 (two products and a sum, e = 2^-23 each) from the tables as they are given, rounded
once to the tensors' type (u = eps / 2 relatively, t half of the type's smallest step absolutely);
tables in 64 bits (angles of at most 2^17 turns: 2^-34 absolutely), rounded once.
"""

import math

import torch

E = 2.0 ** -23


def steps(dtype: torch.dtype):
    f = torch.finfo(dtype)
    return f.eps / 2, f.smallest_normal * f.eps / 2


def frequencies(rotary_dim, base=10000.0, factor=1.0, original_seqlen=None, low_turns=1.0, high_turns=32.0):
    got = []
    for j in range(rotary_dim // 2):
        f, keep = base ** (-2 * j / rotary_dim), 0.0
        if original_seqlen:
            keep = min(max((original_seqlen * f / (2 * math.pi) - low_turns) / (high_turns - low_turns), 0.0), 1.0)
        got.append(f * (keep + (1 - keep) / factor))
    return torch.tensor(got, dtype=torch.float64)


def tables(seqlen, rotary_dim, attention_factor=1.0, offset=0, dtype=torch.float32, **more):
    """{name: (value, bound)} of cos and sin."""
    angle = torch.outer(torch.arange(offset, offset + seqlen, dtype=torch.float64), frequencies(rotary_dim, **more))
    u, t = steps(dtype)
    got = {}
    for name, f in (("cos", torch.cos), ("sin", torch.sin)):
        x = f(angle) * attention_factor
        got[name] = (x, u * x.abs() + t + 2.0 ** -34 * abs(attention_factor))
    return got


def rotate(x, cos, sin, positions, interleaved, inverse=False):
    """x [rows, heads, dim], one position a row (None: no sequence covers it): (value, bound), NaN where the tables
    have no such position."""
    half = cos.shape[1]
    y, b = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64)
    u, t = steps(x.dtype)
    for i, p in enumerate(positions):
        if p is None:
            y[i] = 0
            continue
        for j in range(half):
            a, c = (2 * j, 2 * j + 1) if interleaved else (j, j + half)
            if not 0 <= p < cos.shape[0]:
                y[i, :, a] = y[i, :, c] = math.nan
                continue
            co, si = float(cos[p, j]), float(sin[p, j]) * (-1 if inverse else 1)
            x1, x2 = x[i, :, a].double(), x[i, :, c].double()
            y[i, :, a], y[i, :, c] = x1 * co - x2 * si, x2 * co + x1 * si
            for at, m in ((a, (x1 * co).abs() + (x2 * si).abs()), (c, (x2 * co).abs() + (x1 * si).abs())):
                b[i, :, at] = 3 * E * m + u * (y[i, :, at].abs() + 3 * E * m) + t
    return y, b
