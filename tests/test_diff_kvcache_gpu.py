"""flash_diff_attn_with_kvcache on the GPU: decode steps, drafted tokens and chunks on
contiguous, remapped and paged caches, held to the derived bounds of oracle/diff.py;
what is wrong with a call; graphs."""

import pytest
import torch

import flash_attention_interface as fai
from oracle.diff import assert_within, diff_attention

pytestmark = pytest.mark.gpu


def _setup(device, lens, sq, new, h, hk, d, dtype, layout, kind, page=256, cap=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    b = len(lens)
    cap = cap or -(-(max(lens) + new) // page) * page
    mk = lambda *s: torch.randn(*s, generator=g).to(dtype).to(device)  # noqa: E731
    s = {"q": mk(b, sq, h, d), "k": mk(b, new, hk, d) if new else None, "v": mk(b, new, hk, d) if new else None,
         "lens": torch.tensor(lens, dtype=torch.int32, device=device), "table": None, "index": None}
    shape = {"layer": (), "head": (h,), "token": (b, sq, h)}[kind]
    s["lam"] = torch.rand(shape, generator=g).to(device)
    if layout == "paged":
        need = [-(-(n + new) // page) for n in lens]
        order = torch.randperm(sum(need) + 2, generator=g).int().tolist()
        table = torch.full((b, cap // page), -1, dtype=torch.int32)
        for i, m in enumerate(need):
            for j in range(m):
                table[i, j] = order.pop()
        s["table"] = table.to(device)
        n_pages = sum(need) + 2
        s["kc"], s["vc"] = mk(n_pages, page, hk, d), mk(n_pages, page, hk, d)
    elif layout == "remapped":
        s["index"] = torch.randperm(b + 2, generator=g).int()[:b].to(device)
        s["kc"], s["vc"] = mk(b + 2, cap, hk, d), mk(b + 2, cap, hk, d)
    else:
        s["kc"], s["vc"] = mk(b, cap, hk, d), mk(b, cap, hk, d)
    return s


def _places(s, i, n):
    """Indices of the first n tokens of sequence i in a cache."""
    if s["table"] is not None:
        page = s["kc"].shape[1]
        t = s["table"][i].tolist()
        return [(t[p // page], p % page) for p in range(n)]
    row = i if s["index"] is None else int(s["index"][i])
    return [(row, p) for p in range(n)]


def _rows(cache, places):
    at = torch.tensor(places, device=cache.device).reshape(-1, 2)
    return cache[at[:, 0], at[:, 1]]


def _call(s, **more):
    args = dict(cache_seqlens=s["lens"], cache_batch_idx=s["index"], block_table=s["table"], causal=True,
                return_softmax_lse=True)
    args.update(more)
    return fai.flash_diff_attn_with_kvcache(s["q"], s["kc"], s["vc"], s["lam"], s["k"], s["v"], **args)


def _check(s, causal=True, scale=None, **more):
    new = 0 if s["k"] is None else s["k"].shape[1]
    kc, vc = s["kc"].clone(), s["vc"].clone()
    out, lse = _call(s, causal=causal, softmax_scale=scale, **more)
    for i, n in enumerate(s["lens"].tolist()):
        places = _places(s, i, n + new)
        for c, x in ((kc, s["k"]), (vc, s["v"])):
            for t in range(new):
                c[places[n + t]] = x[i, t]
        lam = s["lam"][i:i + 1] if s["lam"].dim() == 3 else s["lam"]
        want = diff_attention(s["q"][i:i + 1], _rows(kc, places)[None], _rows(vc, places)[None], lam, scale, causal)
        assert_within(f"out {i}", out[i:i + 1], want["out"])
        assert_within(f"lse {i}", lse[:, i:i + 1], want["lse"])
    assert torch.equal(s["kc"], kc) and torch.equal(s["vc"], vc)  # appended, and nothing else touched
    return out


@pytest.mark.parametrize("layout", ["paged", "contiguous", "remapped"])
@pytest.mark.parametrize("lens,sq,new,h,hk,d,dtype,kind", [
    ([0, 1, 63, 700], 1, 1, 8, 2, 128, torch.float16, "head"),
    ([5, 255, 256, 257], 1, 1, 4, 4, 64, torch.bfloat16, "token"),
    ([1500], 1, 1, 32, 8, 128, torch.bfloat16, "layer"),
    ([10, 900], 5, 5, 6, 2, 64, torch.float16, "token"),
    ([33, 400, 1], 17, 17, 4, 1, 128, torch.float16, "head"),   # 68 rows a KV head
    ([0, 300], 130, 130, 4, 4, 64, torch.bfloat16, "token"),
    ([90, 400, 1], 300, 300, 4, 1, 128, torch.float16, "head"),  # 1200 rows a KV head: the forward kernel
    ([0, 290], 400, 310, 4, 4, 64, torch.bfloat16, "token"),
    ([200, 64, 100], 4, 0, 4, 2, 128, torch.float16, "layer"),  # no append
    ([40, 3], 3, 7, 12, 4, 128, torch.bfloat16, "head"),        # more new tokens than queries
])
def test_against_the_definition(device, layout, lens, sq, new, h, hk, d, dtype, kind):
    _check(_setup(device, lens, sq, new, h, hk, d, dtype, layout, kind))


@pytest.mark.parametrize("splits", [1, 2, 7, 100])
def test_split_counts(device, splits):
    _check(_setup(device, [700, 3, 0, 1023], 2, 1, 8, 2, 64, torch.float16, "paged", "head"), num_splits=splits)


def test_fewer_keys_than_queries(device):
    # Causal rows without a key give 0.
    for rows in (8, 40, 300):
        _check(_setup(device, [0, 2], rows, 3, 4, 2, 64, torch.float16, "paged", "token"))


@pytest.mark.parametrize("sq", [1, 40, 300])
def test_no_mask_and_scales(device, sq):
    s = _setup(device, [100, 300], sq, 1, 4, 2, 64, torch.bfloat16, "paged", "head")
    _check(s, causal=False)
    _check(s, causal=True, scale=-0.3)


@pytest.mark.parametrize("page", [64, 128, 320])
def test_page_sizes(device, page):
    for sq in (1, 40, 300):
        _check(_setup(device, [page - 1, page, 3 * page + 5], sq, 1, 4, 2, 128, torch.float16, "paged", "head", page=page))


@pytest.mark.parametrize("layout", ["paged", "contiguous"])
@pytest.mark.parametrize("b,h,hk,d,dtype", [
    (5, 8, 2, 128, torch.float16),    # the longest sequences first
    (70, 3, 3, 64, torch.bfloat16),   # more sequences than a wave has lanes: as they come
    (13, 32, 32, 64, torch.float16),  # more workgroups than the chip has places for
])
def test_chunks_of_many_sequences(device, layout, b, h, hk, d, dtype):
    lens = [(37 * i * i + 11 * i) % 500 for i in range(b)]
    _check(_setup(device, lens, 66, 66, h, hk, d, dtype, layout, "head"))


def test_full_cache(device):
    s = _setup(device, [255, 100], 1, 1, 4, 2, 64, torch.float16, "contiguous", "head", cap=256)
    _check(s)


def test_garbage_past_the_length(device):
    for layout in ("paged", "contiguous"):
        for sq in (1, 40, 300):
            s = _setup(device, [70, 130], sq, 1, 4, 2, 64, torch.float16, layout, "head")
            clean = _call({**s, "kc": s["kc"].clone(), "vc": s["vc"].clone()})
            keep = torch.zeros(s["kc"].shape[:2], dtype=torch.bool, device=device)
            for i, n in enumerate(s["lens"].tolist()):
                for p in _places(s, i, n):
                    keep[p] = True
            for c in (s["kc"], s["vc"]):
                c[~keep] = float("nan")
            got = _call(s)
            assert all(torch.equal(a, b) for a, b in zip(got, clean))


def test_strided_caches(device):
    # K and V in one tensor, and heads before tokens.
    s = _setup(device, [70, 130], 1, 1, 4, 2, 64, torch.float16, "paged", "head")
    both = torch.stack((s["kc"], s["vc"]), 1)
    s["kc"], s["vc"] = both[:, 0], both[:, 1]
    _check(s)
    s["kc"], s["vc"] = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (s["kc"], s["vc"]))
    _check(s)


def test_offsets_past_32_bits(device):
    # A pool of 2.3 G elements for each of K and V, with the sequence's pages at both ends of it.
    n_pages, page, hk, d = 9000, 256, 8, 128
    kc = torch.empty(n_pages, page, hk, d, dtype=torch.float16, device=device)
    vc = torch.empty_like(kc)
    pages = [n_pages - 1, 0, n_pages - 2, 1]
    g = torch.Generator().manual_seed(1)
    for p in pages:
        kc[p] = torch.randn(page, hk, d, generator=g).half().to(device)
        vc[p] = torch.randn(page, hk, d, generator=g).half().to(device)
    for sq in (1, 40, 300):
        mk = lambda h: torch.randn(1, sq, h, d, generator=g).half().to(device)  # noqa: E731
        s = {"q": mk(8), "k": mk(hk), "v": mk(hk), "lam": torch.rand(8, generator=g).to(device), "index": None,
             "lens": torch.tensor([600], dtype=torch.int32, device=device),
             "table": torch.tensor([pages], dtype=torch.int32, device=device), "kc": kc, "vc": vc}
        out, _ = _call(s)
        places = _places(s, 0, 600 + sq)
        want = diff_attention(s["q"], _rows(kc, places)[None], _rows(vc, places)[None], s["lam"], None, True)
        assert_within("out", out, want["out"])
        assert torch.equal(_rows(kc, places[600:]), s["k"][0])


@pytest.mark.parametrize("sq", [1, 40, 300])
def test_bad_sequences_are_reported_and_left_alone(device, sq):
    fai.flash_attn_kvcache_check()
    good = _setup(device, [50, 60, 70], sq, 1, 4, 2, 64, torch.float16, "paged", "head")
    want = _call({**good, "kc": good["kc"].clone(), "vc": good["vc"].clone()})

    def bad(change, exc, match, layout="paged"):
        s = _setup(device, [50, 60, 70], sq, 1, 4, 2, 64, torch.float16, layout, "head")
        change(s)
        kc = s["kc"].clone()
        with pytest.raises(exc, match=match):
            _call(s)
        out, lse = _call(s, validate=False)
        with pytest.raises(exc, match=match):
            fai.flash_attn_kvcache_check()
        fai.flash_attn_kvcache_check()  # cleared
        return s, kc, out, lse

    for value in (-1, 256, 2 ** 31 - 1):
        s, kc, out, lse = bad(lambda s: s["lens"].__setitem__(1, value), ValueError, "capacity")
        assert not out[1].any() and not lse[:, 1].any()
        assert torch.equal(out[0], want[0][0]) and torch.equal(out[2], want[0][2])
        assert torch.equal(s["kc"][int(s["table"][1, 0])], kc[int(s["table"][1, 0])])
    for value in (-1, 10 ** 9):
        s, kc, out, lse = bad(lambda s: s["table"].__setitem__((1, 0), value), RuntimeError, "block_table")
        assert torch.equal(out[0], want[0][0]) and torch.equal(out[2], want[0][2]) and torch.isfinite(out).all()
        assert torch.equal(s["kc"][0][:50], kc[0][:50]) or int(s["table"][0, 0]) == 0
    for value in (-1, 5):
        s, kc, out, lse = bad(lambda s: s["index"].__setitem__(1, value), RuntimeError, "cache_batch_idx", "remapped")
        assert not out[1].any()


def test_captured_decode_step(device):
    """Replays follow new lengths, tables and tokens, with eager work between."""
    fai.flash_attn_kvcache_check()
    s = _setup(device, [300, 20, 511], 1, 1, 8, 2, 128, torch.bfloat16, "paged", "head", cap=768)
    s["table"] = torch.arange(9, dtype=torch.int32, device=device).reshape(3, 3)
    g = torch.Generator().manual_seed(9)
    s["kc"], s["vc"] = (torch.randn(9, 256, 2, 128, generator=g).bfloat16().to(device) for _ in range(2))
    _call({**s, "kc": s["kc"].clone(), "vc": s["vc"].clone()}, validate=False)
    torch.cuda.synchronize()
    graphs = []
    for splits in (0, 3):  # two graphs, with workspaces of their own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, _call(s, validate=False, num_splits=splits), splits))
    for step in range(3):
        s["lens"].copy_(torch.tensor([300 + step, 767 - step, 5 * step], dtype=torch.int32))
        s["table"].copy_(torch.randperm(9, generator=g).int().reshape(3, 3))
        for x in (s["q"], s["k"], s["v"]):
            x.copy_(torch.randn(x.shape, generator=g))
        eager = [_call({**s, "kc": s["kc"].clone(), "vc": s["vc"].clone()}, num_splits=n) for _, _, n in graphs]
        for graph, _, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (_, got, _), want in zip(graphs, eager):
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    fai.flash_attn_kvcache_check()


def test_a_row_does_not_depend_on_the_batch(device):
    s = _setup(device, [700, 30, 520, 90], 1, 1, 8, 2, 64, torch.float16, "paged", "head", cap=1024)
    out, _ = _call({**s, "kc": s["kc"].clone(), "vc": s["vc"].clone()}, num_splits=4)
    one = {**s, **{n: s[n][2:3] for n in ("q", "k", "v", "lens", "table")}}
    assert torch.equal(_call(one, num_splits=4)[0], out[2:3])


def test_refusals(device):
    s = _setup(device, [50, 60], 1, 1, 4, 2, 64, torch.float16, "paged", "head")
    with pytest.raises(RuntimeError, match="divisible by 64"):
        _call({**s, "kc": s["kc"][:, :100], "vc": s["vc"][:, :100]})
    with pytest.raises(RuntimeError, match="contiguous last dimension"):
        _call({**s, "kc": s["kc"].transpose(2, 3).contiguous().transpose(2, 3)})
    with pytest.raises(RuntimeError, match="k_cache must have the dtype"):
        _call({**s, "kc": s["kc"].bfloat16()})
    with pytest.raises(RuntimeError, match="k and v must have shape"):
        _call({**s, "k": s["k"][:, :, :1], "v": s["v"][:, :, :1]})
    with pytest.raises(RuntimeError, match="batch size must match"):
        _call({**s, "table": None, "kc": s["kc"][:1], "vc": s["vc"][:1]})
    with pytest.raises(RuntimeError, match="capacity is insufficient"):  # also without the host's checks
        _call({**s, "kc": s["kc"][:0], "vc": s["vc"][:0]}, validate=False)


@pytest.mark.parametrize("sq", [1, 300])
def test_no_pages_and_no_keys(device, sq):
    # A table of no columns, an empty pool, and sequences of no token: rows without keys are 0.
    s = _setup(device, [0, 0], sq, 0, 4, 2, 64, torch.float16, "paged", "head", cap=256)
    for x in (s, {**s, "table": s["table"][:, :0]}, {**s, "kc": s["kc"][:0], "vc": s["vc"][:0]}):
        for validate in (True, False):
            fai.flash_attn_kvcache_check()
            out, lse = _call(x, validate=validate)
            assert not out.any() and not lse.any()
