"""Ordinary attention over a paged cache whose table names pages that are not there: nothing
outside the pool is read or written, the sequences that do not use such an entry are as
they were, and flash_attn_kvcache_check() says so.

The pool is a slice of a larger tensor of the test's, with pages of NaN on both sides."""

import pytest
import torch

import flash_attention_interface as fai
from oracle.diff import Pages

pytestmark = pytest.mark.gpu

GUARD = 4


def _pool(device, n, page, hk, d, seed):
    whole = torch.full((n + 2 * GUARD, page, hk, d), float("nan"), dtype=torch.float16, device=device)
    pool = whole[GUARD:GUARD + n]
    pool.copy_(torch.randn(pool.shape, generator=torch.Generator().manual_seed(seed)))
    return whole, pool


def _same(a, b):
    return torch.equal(a.view(torch.int16), b.view(torch.int16))  # NaN included


ROUTES = [
    # sequences' lengths, queries, heads, KV heads, channels, splits, options
    ([700, 300, 900], 1, 8, 2, 128, 0, {}),
    ([700, 300, 900], 1, 8, 2, 64, 4, {}),
    ([600] * 40, 1, 32, 8, 64, 8, {}),                                   # more items than workgroups at a time
    ([700, 300, 900], 5, 4, 4, 128, 1, {}),
    ([700, 300, 900], 1, 8, 2, 128, 0, {"window_size": (400, 0), "softcap": 20.0}),
    ([700, 300, 900], 100, 8, 2, 128, 0, {}),                            # the kernel of many rows
    ([700, 300, 900], 100, 8, 2, 64, 3, {"window_size": (300, 0)}),
]


def _call(s, table, validate, **more):
    fai.flash_attn_kvcache_check()
    args = dict(k=s["k"], v=s["v"], cache_seqlens=s["lens"], block_table=table, causal=True, return_softmax_lse=True,
                num_splits=s["splits"], validate=validate, **s["options"])
    args.update(more)
    return fai.flash_attn_with_kvcache(s["q"], s["kp"], s["vp"], **args)


def _setup(device, lens, sq, h, hk, d, splits, options, new=0, page=256, width=5):
    g = torch.Generator().manual_seed(5)
    mk = lambda *s: torch.randn(*s, generator=g).half().to(device)  # noqa: E731
    b = len(lens)
    n = sum(-(-(x + new) // page) for x in lens)
    s = {"q": mk(b, sq, h, d), "k": mk(b, new, hk, d) if new else None, "v": mk(b, new, hk, d) if new else None,
         "lens": torch.tensor(lens, dtype=torch.int32, device=device), "splits": splits, "options": options, "n": n}
    (s["kw"], s["kp"]), (s["vw"], s["vp"]) = _pool(device, n, page, hk, d, 1), _pool(device, n, page, hk, d, 2)
    order = torch.randperm(n, generator=g).tolist()
    table = torch.full((b, width), -1, dtype=torch.int32)
    for i, x in enumerate(lens):
        for j in range(-(-(x + new) // page)):
            table[i, j] = order.pop()
    s["table"] = table.to(device)
    return s


@pytest.mark.parametrize("validate", [False, True])
@pytest.mark.parametrize("lens,sq,h,hk,d,splits,options", ROUTES)
def test_reads_stay_in_the_pool(device, lens, sq, h, hk, d, splits, options, validate):
    s = _setup(device, lens, sq, h, hk, d, splits, options)
    whole = s["kw"].clone(), s["vw"].clone()
    want = _call(s, s["table"], validate)
    fai.flash_attn_kvcache_check()  # entries past the lengths are -1 and are not looked at
    for value in (-1, s["n"], 2 ** 31 - 1, -2 ** 31):
        table, zero = s["table"].clone(), s["table"].clone()
        table[-1, 1], zero[-1, 1] = value, 0
        got = _call(s, table, validate)
        with pytest.raises(RuntimeError, match="block_table entries in use must be pages of the cache"):
            fai.flash_attn_kvcache_check()
        fai.flash_attn_kvcache_check()  # cleared
        read = _call(s, zero, validate)
        for x, y, z in zip(got, read, want):
            assert torch.equal(x, y) and torch.isfinite(x).all()  # page 0 in its place
            assert torch.equal(x[:-1], z[:-1])
    assert _same(s["kw"], whole[0]) and _same(s["vw"], whole[1])


@pytest.mark.parametrize("validate", [False, True])
@pytest.mark.parametrize("lens,sq,h,hk,d,splits,options", ROUTES)
def test_appends_stay_in_the_pool(device, lens, sq, h, hk, d, splits, options, validate):
    new = min(sq, 7)
    s = _setup(device, lens, sq, h, hk, d, splits, options, new=new)
    whole = s["kw"].clone(), s["vw"].clone()
    want = _call(s, s["table"], validate)
    after = s["kw"].clone(), s["vw"].clone()
    last = (lens[-1]) // 256  # the page that takes the last sequence's tokens
    page = int(s["table"][-1, last])
    for x, y in zip(after, whole):
        x[GUARD + page] = y[GUARD + page]
    for value in (-1, s["n"], 2 ** 31 - 1, -2 ** 31):
        s["kw"].copy_(whole[0]), s["vw"].copy_(whole[1])
        table = s["table"].clone()
        table[-1, last] = value
        got = _call(s, table, validate)
        with pytest.raises(RuntimeError, match="block_table entries in use must be pages of the cache"):
            fai.flash_attn_kvcache_check()
        assert _same(s["kw"], after[0]) and _same(s["vw"], after[1])  # the other sequences' tokens, and nothing else
        for x, z in zip(got, want):
            assert torch.isfinite(x).all() and torch.equal(x[:-1], z[:-1])


def test_more_pages_than_a_split_stages(device):
    # 1100 pages in one split: their entries are read from the table tile by tile.
    s = _setup(device, [256, 256, 256], 1, 1, 1, 64, 1, {})
    s["q"], s["lens"] = s["q"][:1], torch.tensor([1100 * 256 - 9], dtype=torch.int32, device=device)
    table = torch.arange(1100, dtype=torch.int32, device=device)[None] % 3
    zero = table.clone()
    for at, value in ((0, -1), (500, 3), (1099, -2 ** 31)):
        table[0, at], zero[0, at] = value, 0
    got = _call(s, table, False)
    with pytest.raises(RuntimeError, match="block_table entries in use"):
        fai.flash_attn_kvcache_check()
    for x, y in zip(got, _call(s, zero, False)):
        assert torch.equal(x, y) and torch.isfinite(x).all()


@pytest.mark.parametrize("diff", [False, True])
def test_a_serving_loop_that_runs_out_of_pages(device, diff):
    """Steps of alloc and attention with validate=False over a pool that is too small: alloc gives nothing, the
    sequences that lack a page are not appended to, and the check says both."""
    n, page, rows, h, hk, d = 3, 256, 2, 4, 2, 64
    (kw, kp), (vw, vp) = _pool(device, n, page, hk, d, 1), _pool(device, n, page, hk, d, 2)
    table = torch.full((rows, 3), -1, dtype=torch.int32, device=device)
    lens = torch.zeros(rows, dtype=torch.int32, device=device)
    refs = torch.zeros(n, dtype=torch.int32, device=device)
    g = torch.Generator().manual_seed(3)
    lam = torch.rand(h, generator=g).to(device)
    model = Pages(n, page, rows, 3)
    fai.flash_attn_kvcache_check()
    for new, enough in ((256, True), (10, False)):
        mk = lambda k: torch.randn(rows, new, k, d, generator=g).half().to(device)  # noqa: E731
        q, k, v = mk(h), mk(hk), mk(hk)
        before = kw.clone(), vw.clone()
        fai.flash_attn_kvcache_alloc(table, lens, refs, new, page, validate=False)
        if diff:
            out = fai.flash_diff_attn_with_kvcache(q, kp, vp, lam, k, v, cache_seqlens=lens, block_table=table, causal=True,
                                                   validate=False)
        else:
            out = fai.flash_attn_with_kvcache(q, kp, vp, k, v, cache_seqlens=lens, block_table=table, causal=True,
                                              validate=False)
        assert torch.isfinite(out).all()
        if enough:
            model.alloc([new] * rows)
            fai.flash_attn_kvcache_check()
            lens += new
        else:
            status = int(fai._KV_STATUS[device.index or 0])
            assert status == 4 | 8  # a page that is none, and fewer pages than needed
            with pytest.raises(RuntimeError, match="block_table entries in use"):
                fai.flash_attn_kvcache_check()
            assert _same(kw, before[0]) and _same(vw, before[1])
        assert table.tolist() == model.table and refs.tolist() == model.refs
    for w in (kw, vw):
        assert torch.isnan(w[:GUARD]).all() and torch.isnan(w[GUARD + n:]).all()


def test_a_checked_call_inside_a_capture(device, monkeypatch):
    """A length that the host knows needs no read, so such a call can be captured with validate=True, also where no
    status word was ever made; the table's entries are bounded without one."""
    s = _setup(device, [700, 300, 900], 1, 4, 2, 64, 2, {})
    table = s["table"].clone()
    table[1, 1] = -1
    call = lambda: fai.flash_attn_with_kvcache(s["q"], s["kp"], s["vp"], cache_seqlens=300, block_table=table,  # noqa: E731
                                               causal=True, num_splits=2)
    want = call()
    with pytest.raises(RuntimeError, match="block_table entries in use"):
        fai.flash_attn_kvcache_check()
    torch.cuda.synchronize()
    monkeypatch.setattr(fai, "_KV_STATUS", {})
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.isfinite(got).all()
        assert torch.equal(call(), want)
