"""Pages of a paged cache on the GPU: alloc, copy, fork, free and compaction against a
model on Python lists (exact), what is wrong with a call, graphs, and a serving loop
that uses them together with differential and ordinary attention."""

import random

import pytest
import torch

import flash_attention_interface as fai
from oracle.diff import Pages, assert_within, diff_attention

pytestmark = pytest.mark.gpu


class Cache:
    """The device's state beside the model's.  A token's K rows hold its number, its V rows the negative."""

    def __init__(self, device, num_pages, page, rows, width, hk=2, d=64, dtype=torch.float16, strided=False):
        self.model = Pages(num_pages, page, rows, width)
        shape = (num_pages, page, hk, d)
        if strided:  # K and V interleaved per page, heads before tokens
            both = torch.zeros(num_pages, 2, hk, page, d, dtype=dtype, device=device).transpose(2, 3)
            self.k, self.v = both[:, 0], both[:, 1]
        else:
            self.k, self.v = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
        self.table = torch.full((rows, width), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(rows, dtype=torch.int32, device=device)
        self.refs = torch.zeros(num_pages, dtype=torch.int32, device=device)
        self.device = device

    def ints(self, v):
        return torch.tensor(v, dtype=torch.int32, device=self.device)

    def alloc(self, new, **more):
        fai.flash_attn_kvcache_alloc(self.table, self.lens, self.refs, self.ints(new) if isinstance(new, list) else new,
                                     self.model.page, **more)

    def fork(self, parents, children, **more):
        fai.flash_attn_kvcache_fork(self.k, self.v, self.table, self.lens, self.refs, self.ints(parents),
                                    self.ints(children), **more)

    def free(self, rows, **more):
        fai.flash_attn_kvcache_free(self.table, self.lens, self.refs, self.ints(rows), **more)

    def append(self, row, tokens):
        m = self.model
        for x in tokens:
            p, at = m.table[row][m.lens[row] // m.page], m.lens[row] % m.page
            self.k[p, at], self.v[p, at] = float(x), -float(x)
            m.append(row, [x])
        self.lens[row] = m.lens[row]

    def check(self):
        m = self.model
        assert self.table.tolist() == m.table
        assert self.lens.tolist() == m.lens
        assert self.refs.tolist() == m.refs
        data = torch.tensor(m.data, dtype=self.k.dtype)
        assert torch.equal(self.k.cpu(), data[:, :, None, None].expand(self.k.shape))
        assert torch.equal(self.v.cpu(), -data[:, :, None, None].expand(self.k.shape))

    def snapshot(self):
        return [x.clone() for x in (self.k, self.v, self.table, self.lens, self.refs)]


@pytest.mark.parametrize("num_pages,page,rows,width,hk,d,dtype,strided,seed", [
    (60, 4, 9, 12, 2, 64, torch.float16, False, 0),
    (60, 4, 9, 12, 3, 64, torch.bfloat16, True, 1),
    (40, 16, 5, 9, 1, 8, torch.float32, False, 2),
    (1300, 1, 30, 50, 1, 16, torch.float16, False, 3),   # more pages than a plan's threads
])
def test_random_calls(device, num_pages, page, rows, width, hk, d, dtype, strided, seed):
    r = random.Random(seed)
    c = Cache(device, num_pages, page, rows, width, hk, d, dtype, strided)
    m = c.model
    for step in range(60):
        live = [i for i in range(rows) if m.lens[i]]
        empty = [i for i in range(rows) if not m.lens[i] and m.table[i][0] < 0]
        op = r.choice(["alloc", "alloc", "fork", "free", "compact", "copy"])
        if op == "alloc":
            new = [r.choice([0, 0, r.randrange(1, 3 * page + 2)]) for _ in range(rows)]
            new = [min(n, width * page - have) for n, have in zip(new, m.lens)]
            need = sum(sum(m.table[i][j] < 0 for j in range(m.lens[i] // page, -(-(m.lens[i] + n) // page) if n else 0))
                       for i, n in enumerate(new))
            if need <= m.refs.count(0):
                c.alloc(new)
                m.alloc(new)
                for i, n in enumerate(new):
                    c.append(i, [r.randrange(1, 200) for _ in range(r.randrange(n + 1))])
        elif op == "fork" and live and empty:
            kids = r.sample(empty, r.randrange(1, len(empty) + 1))
            parents = [r.choice(live) for _ in kids]
            if sum(m.lens[p] % page != 0 for p in parents) <= m.refs.count(0):
                c.fork(parents, kids)
                m.fork(parents, kids)
        elif op == "free":
            which = [r.randrange(rows) for _ in range(r.randrange(1, 4))]  # a row may be named twice, or be empty
            c.free(which)
            m.free(which)
        elif op == "compact":
            before = c.snapshot()
            table, refs, used = fai.flash_attn_kvcache_compact(c.k, c.v, c.table, c.refs)
            assert torch.equal(c.table, before[2]) and torch.equal(c.refs, before[4])  # the old ones stay
            c.table, c.refs = table, refs
            assert used.tolist() == [m.compact()]
        elif op == "copy":
            pages = r.sample(range(num_pages), 2 * r.randrange(1, 5))
            free = [p for p in pages[::2] if m.refs[p] == 0]
            src = pages[1::2][: len(free)]
            fai.flash_attn_kvcache_copy_pages(c.k, c.v, c.ints(src), c.ints(free))
            for a, b in zip(src, free):
                m.data[b] = list(m.data[a])
        c.check()


def test_fork_on_a_page_border_and_of_empty_rows(device):
    c = Cache(device, 12, 4, 6, 4)
    c.alloc([8, 0, 0, 0, 0, 0])
    c.model.alloc([8, 0, 0, 0, 0, 0])
    c.append(0, list(range(1, 9)))
    c.fork([0, 1, 0], [3, 4, 5])  # full pages only; an empty parent; the same parent again
    c.model.fork([0, 1, 0], [3, 4, 5])
    c.check()
    c.alloc(1)  # every row gets a page of its own for the next token
    c.model.alloc([1] * 6)
    c.check()
    c.append(3, [50])
    c.append(5, [60])
    c.check()


def test_whole_pools(device):
    # Every page taken; compaction of a full and of an empty pool; one page.
    c = Cache(device, 8, 4, 2, 8)
    assert fai.flash_attn_kvcache_compact(c.k, c.v, c.table, c.refs)[2].tolist() == [0]
    c.alloc([16, 16])
    c.model.alloc([16, 16])
    c.check()
    table, refs, used = fai.flash_attn_kvcache_compact(c.k, c.v, c.table, c.refs)
    assert torch.equal(table, c.table) and torch.equal(refs, c.refs) and used.tolist() == [8]
    one = Cache(device, 1, 4, 1, 1)
    one.alloc(4)
    one.model.alloc([4])
    one.check()
    one.free([0])
    one.model.free([0])
    one.check()


def test_empty_lists(device):
    c = Cache(device, 8, 4, 2, 3)
    none = c.ints([])
    fai.flash_attn_kvcache_copy_pages(c.k, c.v, none, none)
    c.fork([], [])
    c.free([])
    c.alloc(0)
    c.check()


def _filled(device):
    c = Cache(device, 10, 4, 5, 3)
    c.alloc([6, 3, 0, 0, 0])
    c.model.alloc([6, 3, 0, 0, 0])
    c.append(0, [1, 2, 3, 4, 5, 6])
    c.append(1, [7, 8, 9])
    return c


@pytest.mark.parametrize("name,call,exc,match", [
    ("child taken", lambda c, **m: c.fork([0], [1], **m), ValueError, "out of range, taken or named twice"),
    ("child twice", lambda c, **m: c.fork([0, 1], [2, 2], **m), ValueError, "named twice"),
    ("child is a parent", lambda c, **m: c.fork([0, 2], [2, 3], **m), ValueError, "taken"),
    ("its own child", lambda c, **m: c.fork([2], [2], **m), ValueError, "taken"),
    ("no such parent", lambda c, **m: c.fork([5], [2], **m), ValueError, "out of range"),
    ("negative child", lambda c, **m: c.fork([0], [-1], **m), ValueError, "out of range"),
    ("too many rows at once", lambda c, **m: c.alloc([6, 9, 12, 12, 12], **m), RuntimeError, "fewer free pages"),
    ("past the table", lambda c, **m: c.alloc([7, 0, 0, 0, 0], **m), ValueError, "capacity"),
    ("negative new", lambda c, **m: c.alloc([0, -1, 0, 0, 0], **m), ValueError, "capacity"),
])
def test_wrong_calls_change_nothing(device, name, call, exc, match):
    fai.flash_attn_kvcache_check()
    for validate in (True, False):
        c = _filled(device)
        before = c.snapshot()
        if validate:
            with pytest.raises(exc, match=match):
                call(c)
        else:
            call(c, validate=False)
            with pytest.raises(exc, match=match):
                fai.flash_attn_kvcache_check()
        assert all(torch.equal(a, b) for a, b in zip(before, c.snapshot())), name
    fai.flash_attn_kvcache_check()


def test_fork_without_enough_pages(device):
    c = Cache(device, 3, 4, 5, 3)
    c.alloc([6, 0, 0, 0, 0])
    c.model.alloc([6, 0, 0, 0, 0])
    c.append(0, [1, 2, 3, 4, 5, 6])
    before = c.snapshot()
    with pytest.raises(RuntimeError, match="fewer free pages"):
        c.fork([0, 0], [1, 2])
    assert all(torch.equal(a, b) for a, b in zip(before, c.snapshot()))
    c.fork([0], [1])
    c.model.fork([0], [1])
    c.check()


def test_tables_with_bad_pages(device):
    # Entries that are no pages are neither counted nor followed.
    c = _filled(device)
    c.table[0, 1] = 10
    before = c.snapshot()
    with pytest.raises(RuntimeError, match="block_table"):
        c.fork([0], [2])
    assert all(torch.equal(a, b) for a, b in zip(before, c.snapshot()))
    table, _, _ = fai.flash_attn_kvcache_compact(c.k, c.v, c.table, c.refs)
    assert int(table[0, 1]) == 10
    c.free([0])
    assert c.table[0].tolist() == [-1] * 3 and int(c.refs.sum()) == 2  # the page that only the bad entry replaced


def test_pairs_that_touch_each_other_are_not_copied(device):
    k = torch.arange(6, device=device).half()[:, None, None, None].expand(6, 4, 1, 8).contiguous()
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    for src, dst, want in (
        ((0, 1), (1, 2), [0, 1, 2, 3, 4, 5]),        # 1 is read and written
        ((0, 1, 5), (3, 3, 4), [0, 1, 2, 3, 5, 5]),  # 3 is written twice; the third pair is its own
        ((0, 9), (1, 2), [0, 0, 2, 3, 4, 5]),        # no page 9
        ((0, 1), (2, -1), [0, 1, 0, 3, 4, 5]),
    ):
        a, b = k.clone(), -k
        with pytest.raises(ValueError, match="named twice"):
            fai.flash_attn_kvcache_copy_pages(a, b, ints(*src), ints(*dst))
        assert a[:, 0, 0, 0].tolist() == want and b[:, 0, 0, 0].tolist() == [-x for x in want]
    a, b = k.clone(), -k
    fai.flash_attn_kvcache_copy_pages(a, b, ints(0, 3, 0), ints(1, 3, 2))  # one source twice, a page onto itself
    assert a[:, 0, 0, 0].tolist() == [0, 0, 0, 3, 4, 5]


def test_captured_step(device):
    """Free, fork and alloc in one graph, replayed with other lists, eager work between."""
    fai.flash_attn_kvcache_check()
    c, e = (Cache(device, 30, 4, 8, 6) for _ in range(2))
    lists = [c.ints([4, 5]), c.ints([0, 1]), c.ints([4, 5])]

    def step(x, rows, parents, kids):
        fai.flash_attn_kvcache_free(x.table, x.lens, x.refs, rows, validate=False)
        fai.flash_attn_kvcache_fork(x.k, x.v, x.table, x.lens, x.refs, parents, kids, validate=False)
        fai.flash_attn_kvcache_alloc(x.table, x.lens, x.refs, 1, 4, validate=False)

    for x in (c, e):
        x.alloc([6, 9, 4, 1, 0, 0, 0, 0])
        x.model.alloc([6, 9, 4, 1, 0, 0, 0, 0])
        for i, n in enumerate([6, 9, 4, 1]):
            x.append(i, list(range(1 + i, 1 + i + n)))
    step(e, *lists)  # not captured: what a first call loads
    e.free([4, 5])
    e.table.copy_(c.table), e.refs.copy_(c.refs), e.lens.copy_(c.lens), e.k.copy_(c.k), e.v.copy_(c.v)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(c, *lists)
    # (Alloc gives the rows that are never forked a page, too: the second and third fork, into rows 6 and 7 that hold
    # one, change nothing and are reported.)
    for rows, parents, kids, fine in (([4, 5], [0, 1], [4, 5], True), ([5, 5], [2, 3], [5, 6], False),
                                      ([4, 6], [5, 0], [4, 7], False), ([6, 7], [1, 0], [7, 6], True),
                                      ([6, 4], [7, 7], [6, 4], True)):
        for t, v in zip(lists, (rows, parents, kids)):
            t.copy_(torch.tensor(v, dtype=torch.int32))
        graph.replay()
        step(e, *lists)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(c.snapshot(), e.snapshot()))
        if not fine:
            with pytest.raises(ValueError, match="taken"):
                fai.flash_attn_kvcache_check()
        fai.flash_attn_kvcache_check()


def test_refusals(device):
    c = _filled(device)
    with pytest.raises(RuntimeError, match="k_cache and v_cache must match"):
        fai.flash_attn_kvcache_copy_pages(c.k, c.v[:5], c.ints([0]), c.ints([1]))
    with pytest.raises(RuntimeError, match="contiguous last dimension"):
        x = torch.zeros(4, 4, 2, 7, dtype=torch.float16, device=device)
        fai.flash_attn_kvcache_copy_pages(x, x.clone(), c.ints([0]), c.ints([1]))
    with pytest.raises(RuntimeError, match="same length"):
        c.fork([0, 1], [2])
    with pytest.raises(RuntimeError, match="one entry a page"):
        fai.flash_attn_kvcache_fork(c.k, c.v, c.table, c.lens, c.refs[:5], c.ints([0]), c.ints([2]))
    with pytest.raises(RuntimeError, match="one entry a row"):
        fai.flash_attn_kvcache_free(c.table, c.lens[:2], c.refs, c.ints([0]))
    with pytest.raises(RuntimeError, match="rows of block_table must not overlap"):
        fai.flash_attn_kvcache_free(c.table[:1].expand(c.lens.shape[0], -1), c.lens, c.refs, c.ints([0]))
    with pytest.raises(RuntimeError, match="pages of k_cache must not overlap"):
        fai.flash_attn_kvcache_copy_pages(c.k[:1].expand(4, -1, -1, -1), c.v[:4], c.ints([0]), c.ints([1]))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_serving_loop(device, dtype):
    """Prompts, forks, decode steps, ends and compaction together: every step's output against the definition over
    the row's own token history, and in fp16 ordinary attention on the same cache against itself on a
    contiguous copy of the tokens (whose keys it may split and sum in another order)."""
    h, hk, d, page, rows, width = 4, 2, 64, 256, 6, 4
    g = torch.Generator().manual_seed(5)
    mk = lambda *s: torch.randn(*s, generator=g).to(dtype).to(device)  # noqa: E731
    k_cache, v_cache = mk(24, page, hk, d), mk(24, page, hk, d)
    table = torch.full((rows, width), -1, dtype=torch.int32, device=device)
    lens = torch.zeros(rows, dtype=torch.int32, device=device)
    refs = torch.zeros(24, dtype=torch.int32, device=device)
    lam = torch.rand(h, generator=g).to(device)
    history = [[] for _ in range(rows)]  # (k, v) of each token
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731

    def step(which, n):
        new = [n if i in which else 0 for i in range(rows)]
        fai.flash_attn_kvcache_alloc(table, lens, refs, ints(new), page)
        at = ints(which).long()
        q, k, v = mk(len(which), n, h, d), mk(len(which), n, hk, d), mk(len(which), n, hk, d)
        out = fai.flash_diff_attn_with_kvcache(q, k_cache, v_cache, lam, k, v, cache_seqlens=lens[at],
                                               block_table=table[at], causal=True)
        lens[at] += n
        for i, r in enumerate(which):
            history[r] += [(k[i, t], v[i, t]) for t in range(n)]
            ks, vs = (torch.stack([x[j] for x in history[r]])[None] for j in (0, 1))
            assert_within(f"row {r}", out[i:i + 1], diff_attention(q[i:i + 1], ks, vs, lam, None, True)["out"])
            if dtype == torch.float16 and n == 1:
                a = fai.flash_attn_with_kvcache(q[i:i + 1], k_cache, v_cache, cache_seqlens=lens[r:r + 1],
                                                block_table=table[r:r + 1].clamp_min(0), causal=True)
                b = fai.flash_attn_with_kvcache(q[i:i + 1], ks, vs, causal=True)
                # Two roundings to fp16 (2^-11 each) and twice the fp32 error of 350 keys' scores and sums with
                # |v| < 5: (350 + 16) * 2^-23 * 5 and 2^-21 * 20 * 5.
                worst = float(((a - b).float().abs() - 2.0 ** -10 * a.float().abs()).max())
                assert worst <= 2 * (366 * 2.0 ** -23 * 5 + 2.0 ** -21 * 100), f"ordinary attention, row {r}: {worst}"

    step([0], 300)
    step([1], 256)
    fai.flash_attn_kvcache_fork(k_cache, v_cache, table, lens, refs, ints([0, 0, 1]), ints([2, 3, 4]))
    history[2], history[3], history[4] = list(history[0]), list(history[0]), list(history[1])
    for _ in range(2):
        step([0, 1, 2, 3, 4], 1)
    fai.flash_attn_kvcache_free(table, lens, refs, ints([0, 1]))
    history[0], history[1] = [], []
    step([2, 3, 4], 3)
    table, refs, used = fai.flash_attn_kvcache_compact(k_cache, v_cache, table, refs)
    # Rows 2 and 3 share the old row 0's full page and have one of their own, row 4 has two.
    assert int(used) == int((refs > 0).sum()) == 5 and int(table.max()) == 4
    step([3, 4], 1)
    step([0], 40)
    fai.flash_attn_kvcache_fork(k_cache, v_cache, table, lens, refs, ints([3]), ints([1]))
    history[1] = list(history[3])
    step([0, 1, 2, 3, 4], 1)
    fai.flash_attn_kvcache_free(table, lens, refs, ints(list(range(rows))))
    assert not refs.any() and bool((table == -1).all()) and not lens.any()
