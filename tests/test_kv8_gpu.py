"""A KV cache in 8 bits on the GPU: appends and reads bit for bit as the definition says, attention elementwise within the
roundings that oracle/kv8.py counts; layouts, masks, what is wrong with a call, streams and graphs."""

import math

import pytest
import torch

import flash_attention_interface as fai
from oracle.kv8 import Cache, attention

pytestmark = pytest.mark.gpu

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
KINDS = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


class Setup:
    """A cache with garbage everywhere (NaN codes and scales among it) but in the first lens[b] tokens of each sequence."""

    def __init__(self, device, lens, new, hk, d, kind, block, layout, page=256, capacity=None, seed=0, held=True):
        self.g = torch.Generator().manual_seed(seed)
        self.device, self.lens_list, b = device, lens, len(lens)
        page = max(page, block)
        capacity = capacity or max(-(-(max(lens) + new) // page) * page, page)
        self.index = self.table = None
        if layout == "paged":
            need = [-(-(n + new) // page) for n in lens]
            order = torch.randperm(sum(need) + 2, generator=self.g).int().tolist()
            table = torch.full((b, capacity // page), -1, dtype=torch.int32)
            for i, m in enumerate(need):
                for j in range(m):
                    table[i, j] = order.pop()
            self.table, lines, tokens = table.to(device), sum(need) + 2, page
        elif layout == "remapped":
            self.index = torch.randperm(b + 2, generator=self.g).int()[:b].to(device)
            lines, tokens = b + 2, capacity
        else:
            lines, tokens = b, capacity
        self.kind = KINDS[kind]
        for name in ("k", "v"):
            codes = torch.randint(0, 256, (lines, tokens, hk, d), generator=self.g, dtype=torch.uint8).view(self.kind)
            scale = torch.full((lines, tokens // block, hk), math.nan)
            setattr(self, name + "c", codes.to(device))
            setattr(self, name + "s", scale.to(device))
        self.lens = torch.tensor(lens, dtype=torch.int32, device=device)
        if held:  # what the sequences hold: appended by the oracle
            for name in ("k", "v"):
                o = self.oracle(name)
                for i, n in enumerate(lens):
                    o.append(i, 0, self.normal(n, hk, d).to(torch.bfloat16))
                self.put(name, o)

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.g)

    def oracle(self, name):
        return Cache(getattr(self, name + "c"), getattr(self, name + "s"), self.index, self.table)

    def put(self, name, o):
        codes = o.codes.float().to(self.kind)
        # (Garbage e4m3 NaN codes keep being NaN, the others are exact.)
        getattr(self, name + "c").copy_(codes.to(self.device))
        getattr(self, name + "s").copy_(o.scales.float().to(self.device))

    @property
    def caches(self):
        return self.kc, self.vc, self.ks, self.vs

    @property
    def places(self):
        return {"cache_batch_idx": self.index, "block_table": self.table}


def _same(got, want, name):
    got = got.cpu()
    got = got.double()
    assert torch.equal(got.isnan(), want.isnan()), name
    assert torch.equal(got.nan_to_num(), want.nan_to_num()), f"{name}: {(got != want).sum()} of {got.numel()}"


def _check_append(s, news, k, v, dtype):
    for name, x in (("k", k), ("v", v)):
        o = s.oracle(name)
        for i, (n, m) in enumerate(zip(s.lens_list, news)):
            o.append(i, n, x[i, :m].cpu())
        yield name, o


@pytest.mark.parametrize("layout", ["paged", "contiguous", "remapped"])
@pytest.mark.parametrize("kind,dtype", [("e4m3", "fp16"), ("e4m3", "bf16"), ("int8", "fp16"), ("int8", "bf16")])
@pytest.mark.parametrize("d,block,hk", [(64, 32, 3), (128, 64, 2), (128, 256, 1), (64, 128, 8)])
def test_append(device, d, block, hk, kind, dtype, layout):
    for lens, new in (([0, 1, 31, 32, 33], 1), ([0, 63, 200], 2 * block + 5), ([block - 1, 5], 30), ([256, 255], 300)):
        s = Setup(device, lens, new, hk, d, kind, block, layout, seed=new)
        mag = torch.exp2(torch.randint(-3, 4, (len(lens), new, hk, 1), generator=s.g).float())
        k, v = ((s.normal(len(lens), new, hk, d) * mag).to(DTYPES[dtype]).to(device) for _ in range(2))
        want = dict(_check_append(s, [new] * len(lens), k, v, dtype))
        fai.flash_attn_kvcache_append_q8(k, v, *s.caches, s.lens, **s.places)
        for name, o in want.items():
            _same(getattr(s, name + "c"), o.codes, f"codes of {name}, {lens}, {new}")
            _same(getattr(s, name + "s"), o.scales, f"scales of {name}, {lens}, {new}")


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_append_token_by_token(device, kind):
    """A block that grows one token at a time, whose scale is raised now and then."""
    s = Setup(device, [0, 3], 70, 2, 64, kind, 32, "paged")
    for step in range(70):
        k, v = ((s.normal(2, 1, 2, 64) * 2.0 ** (step % 7 - 3 + step // 20)).half().to(device) for _ in range(2))
        want = dict(_check_append(s, [1, 1], k, v, "fp16"))
        fai.flash_attn_kvcache_append_q8(k, v, *s.caches, s.lens, **s.places)
        for name, o in want.items():
            _same(getattr(s, name + "c"), o.codes, f"codes of {name}, step {step}")
            _same(getattr(s, name + "s"), o.scales, f"scales of {name}, step {step}")
        s.lens_list = [n + 1 for n in s.lens_list]
        s.lens += 1


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_append_of_a_padded_batch(device, kind):
    s = Setup(device, [0, 40, 7, 100], 130, 2, 128, kind, 64, "paged")
    news = [130, 0, 1, 64]
    k, v = (s.normal(4, 130, 2, 128).half() for _ in range(2))
    for x in (k, v):
        for i, n in enumerate(news):
            x[i, n:] = math.nan  # not looked at
    k, v = k.to(device), v.to(device)
    want = dict(_check_append(s, news, k, v, "fp16"))
    fai.flash_attn_kvcache_append_q8(k, v, *s.caches, s.lens, seqlens_new=torch.tensor(news, dtype=torch.int32, device=device),
                                     **s.places)
    for name, o in want.items():
        _same(getattr(s, name + "c"), o.codes, f"codes of {name}")
        _same(getattr(s, name + "s"), o.scales, f"scales of {name}")


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_append_of_extreme_values(device, dtype, kind):
    f = torch.finfo(DTYPES[dtype])
    tiny = f.smallest_normal * f.eps
    tops = [0.0, tiny, 3 * tiny, f.smallest_normal, f.max, f.max / 3, 448.0, 448.0 * (1 + f.eps), 127.0, 127.0 * (1 + f.eps),
            224.0, 63.5, 1.0, 2.0 ** -9 * 448, 1.75, 1.984375]
    s = Setup(device, [0] * len(tops) + [20] * len(tops), 40, 1, 64, kind, 32, "contiguous")
    x = torch.rand(2 * len(tops), 40, 1, 64, generator=s.g) * 2 - 1
    for i, t in enumerate(tops + tops):
        x[i] *= t
        x[i, ::7, 0, 3] = t
        x[i, 1::7, 0, 5] = -t
    x = x.to(DTYPES[dtype]).to(device)
    want = dict(_check_append(s, [40] * len(x), x, -x, dtype))
    fai.flash_attn_kvcache_append_q8(x, -x, *s.caches, s.lens)
    for name, o in want.items():
        _same(getattr(s, name + "c"), o.codes, f"codes of {name}")
        _same(getattr(s, name + "s"), o.scales, f"scales of {name}")


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_append_of_what_is_not_finite(device, bad, kind):
    s = Setup(device, [0, 10, 33], 40, 2, 64, kind, 32, "contiguous")
    k, v = (s.normal(3, 40, 2, 64).bfloat16() for _ in range(2))
    k[0, 35, 1, 7] = k[1, 0, 0, 0] = v[2, 39, 1, 63] = bad
    k, v = k.to(device), v.to(device)
    want = dict(_check_append(s, [40] * 3, k, v, "bf16"))
    fai.flash_attn_kvcache_append_q8(k, v, *s.caches, s.lens)
    for name, o in want.items():
        _same(getattr(s, name + "c"), o.codes, f"codes of {name}")
        _same(getattr(s, name + "s"), o.scales, f"scales of {name}")
    # Whoever sees such a key gets NaN, the others do not: queries before it, the other heads, the other sequences.
    q = s.normal(3, 40, 2, 64).bfloat16().to(device)
    lens = s.lens + 40
    out = fai.flash_attn_with_kvcache_q8(q, *s.caches, cache_seqlens=lens, causal=True).isnan().all(-1).cpu()
    any_ = fai.flash_attn_with_kvcache_q8(q, *s.caches, cache_seqlens=lens, causal=True).isnan().any(-1).cpu()
    assert torch.equal(out, any_)
    expect = torch.zeros(3, 40, 2, dtype=torch.bool)
    expect[0, 32:, 1] = True   # the block of tokens 32..39
    expect[1, :, 0] = True     # the block of tokens 0..31: every query sees some of it
    expect[2, 31:, 1] = True   # the block of tokens 64..72
    assert torch.equal(out, expect)
    # A block that starts anew forgets.
    fai.flash_attn_kvcache_append_q8(k.nan_to_num(0, 0, 0), v.nan_to_num(0, 0, 0), *s.caches, torch.zeros_like(s.lens))
    assert s.ks[:, 0].isfinite().all() and s.vs[:, 0].isfinite().all()


@pytest.mark.parametrize("layout", ["paged", "contiguous", "remapped"])
@pytest.mark.parametrize("kind,dtype", [("e4m3", "fp16"), ("int8", "bf16")])
@pytest.mark.parametrize("d,block,hk", [(64, 32, 3), (128, 64, 8), (128, 256, 1)])
def test_read(device, d, block, hk, kind, dtype, layout):
    lens = [1, 300, 0, 64, 77]
    s = Setup(device, lens, 0, hk, d, kind, block, layout)
    take, before, behind = [1, 299, 0, 64, 30], 3, 5
    cu = [before]
    for n in take:
        cu.append(cu[-1] + n)
    got = fai.flash_attn_kvcache_read_q8(*s.caches, torch.tensor(cu, dtype=torch.int32, device=device), cu[-1] + behind,
                                         dtype=DTYPES[dtype], **s.places)
    for name, y in zip("kv", got):
        assert y.shape == (cu[-1] + behind, hk, d) and y.dtype == DTYPES[dtype]
        o, want = s.oracle(name), torch.zeros(y.shape, dtype=torch.float64)
        for i, n in enumerate(take):
            want[cu[i]:cu[i + 1]] = o.tokens(i, n)
        assert torch.equal(y.cpu(), want.to(DTYPES[dtype])), name


CASES = [
    # lens, new, queries, heads, heads_k
    ([0, 5, 255], 1, 1, 4, 4), ([700, 1, 64], 1, 1, 8, 2), ([1500], 1, 1, 32, 8), ([31, 290, 0, 513], 3, 3, 6, 2),
    ([100, 640], 20, 20, 8, 1), ([0, 0], 40, 40, 4, 4), ([33, 900], 0, 5, 4, 2), ([0, 3], 0, 4, 4, 2), ([260], 150, 150, 6, 3),
    ([1000, 90], 70, 130, 4, 1),
]


def _check(s, q, out, lse, lens, causal, window, scale):
    k, v = s.oracle("k"), s.oracle("v")
    out, lse = out.double().cpu(), lse.double().cpu()
    for i, n in enumerate(lens):
        want = attention(q[i].cpu(), k.tokens(i, n), v.tokens(i, n), scale, causal, window)
        for name, got in (("out", out[i]), ("lse", lse[i])):
            y, bound = want[name]
            assert torch.isfinite(got).all(), (name, i)
            worst = float(((got - y).abs() - bound).max())
            assert worst <= 0, f"{name} of sequence {i}: over its bound by {worst:.3g}"


@pytest.mark.parametrize("layout", ["paged", "contiguous", "remapped"])
@pytest.mark.parametrize("kind,dtype", [("e4m3", "fp16"), ("e4m3", "bf16"), ("int8", "fp16"), ("int8", "bf16")])
@pytest.mark.parametrize("d,block", [(64, 32), (128, 64), (128, 256)])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention(device, case, d, block, kind, dtype, layout):
    lens, new, sq, h, hk = CASES[case]
    s = Setup(device, lens, new, hk, d, kind, block, layout, seed=case)
    mk = lambda *shape: s.normal(*shape).to(DTYPES[dtype]).to(device)  # noqa: E731
    q = mk(len(lens), sq, h, d)
    k, v = (mk(len(lens), new, hk, d), mk(len(lens), new, hk, d)) if new else (None, None)
    want = dict(_check_append(s, [new] * len(lens), k, v, dtype)) if new else {}
    total = [n + new for n in lens]
    for i, (causal, window, splits, scale) in enumerate((
            (True, (-1, -1), 0, None), (False, (-1, -1), 3, 0.2), (True, (70, -1), 0, -0.1), (False, (40, 9), 2, None))):
        if i > 0 and (layout, case % 3) not in (("paged", i % 3), ("contiguous", (i + 1) % 3)):
            continue
        args = dict(k=k, v=v, cache_seqlens=s.lens) if i == 0 else dict(cache_seqlens=s.lens + new)
        out, lse = fai.flash_attn_with_kvcache_q8(q, *s.caches, causal=causal, window_size=window, num_splits=splits,
                                                  softmax_scale=scale, return_softmax_lse=True, **args, **s.places)
        if i == 0:
            for name, o in want.items():
                _same(getattr(s, name + "c"), o.codes, f"codes of {name}")
                _same(getattr(s, name + "s"), o.scales, f"scales of {name}")
        _check(s, q, out, lse, total, causal, window, d ** -0.5 if scale is None else scale)


def test_many_sequences(device):
    """More sequences than the plan takes at a time, empty ones among them, and more pieces than a join's weights."""
    g = torch.Generator().manual_seed(1)
    lens = torch.randint(0, 90, (600,), generator=g).tolist()
    lens[5:9] = [0] * 4
    s = Setup(device, lens, 0, 1, 64, "e4m3", 32, "contiguous", capacity=96)
    q = s.normal(600, 1, 2, 64).half().to(device)
    out, lse = fai.flash_attn_with_kvcache_q8(q, *s.caches, cache_seqlens=s.lens, return_softmax_lse=True)
    _check(s, q, out, lse, lens, False, (-1, -1), 0.125)
    s = Setup(device, [9000], 0, 1, 64, "int8", 128, "contiguous", capacity=9088)
    q = s.normal(1, 2, 3, 64).half().to(device)
    for splits in (0, 71, 1):
        out, lse = fai.flash_attn_with_kvcache_q8(q, *s.caches, cache_seqlens=s.lens, causal=True, num_splits=splits,
                                                  return_softmax_lse=True)
        _check(s, q, out, lse, [9000], True, (-1, -1), 0.125)


def test_any_scales(device):
    """Scales that are no powers of two, 0 and far apart, as another quantiser may write them."""
    for kind in ("e4m3", "int8"):
        s = Setup(device, [300, 97], 0, 2, 64, kind, 32, "contiguous")
        for name in ("ks", "vs"):
            x = getattr(s, name)
            x.copy_(torch.rand(x.shape, generator=s.g) * (0.02 if kind == "e4m3" else 0.05))
        s.vs[0, 1] = 0
        s.vs[0, 2] = 2.0 ** -40
        s.ks[0, 3] = 0
        q = s.normal(2, 3, 4, 64).half().to(device)
        out, lse = fai.flash_attn_with_kvcache_q8(q, *s.caches, cache_seqlens=s.lens, causal=True, return_softmax_lse=True)
        _check(s, q, out, lse, [300, 97], True, (-1, -1), 0.125)
        # New tokens into such a block: the scale stays where it suffices, else becomes a power of two.
        s.ks[:, 9], s.ks[1, 3] = 0.3, 0.3
        k = (s.normal(2, 20, 2, 64)).half().to(device)
        want = dict(_check_append(s, [20, 20], k, k, "fp16"))
        fai.flash_attn_kvcache_append_q8(k, k, *s.caches, s.lens)
        assert 0.3 in [round(float(x), 6) for x in s.ks[:, 9].flatten()]
        _same(s.kc, want["k"].codes, "codes")
        _same(s.ks, want["k"].scales.float().double(), "scales")


def test_strided_caches_and_tensors(device):
    """Heads before tokens, a cache inside a larger tensor, scales that are slices, misaligned and strided q, k and v."""
    lens, new, h, hk, d = [40, 300], 3, 4, 2, 64
    s = Setup(device, lens, new, hk, d, "e4m3", 64, "paged", page=64)
    t = Setup(device, lens, new, hk, d, "e4m3", 64, "paged", page=64)
    q, k, v = (s.normal(2, new, n, d).half().to(device) for n in (h, hk, hk))
    want = fai.flash_attn_with_kvcache_q8(q, *s.caches, k, v, cache_seqlens=s.lens, causal=True, **s.places)
    both = torch.zeros(2, *t.kc.transpose(1, 2).shape, dtype=torch.uint8, device=device).view(t.kind)
    both[0], both[1] = t.kc.transpose(1, 2), t.vc.transpose(1, 2)
    scale = torch.zeros(*t.ks.shape, 3, device=device)
    scale[..., 0], scale[..., 2] = t.ks, t.vs
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device=device)[1:].view(q.shape)
    odd.copy_(q)
    kv = torch.stack((k, v), 2)
    wide = torch.zeros(2, 2 * t.table.shape[1], dtype=torch.int32, device=device)
    wide[:, ::2] = t.table
    out = fai.flash_attn_with_kvcache_q8(
        odd, both[0].transpose(1, 2), both[1].transpose(1, 2), scale[..., 0], scale[..., 2], kv[:, :, 0],
        v.transpose(1, 3).contiguous().transpose(1, 3), cache_seqlens=t.lens, causal=True, block_table=wide[:, ::2])
    assert torch.equal(out, want)
    got, ref = both[0].transpose(1, 2).float(), s.kc.float()
    assert torch.equal(got.nan_to_num(7e3), ref.nan_to_num(7e3)) and torch.equal(scale[..., 2].nan_to_num(-1), s.vs.nan_to_num(-1))


def test_append_alone_and_no_sequences(device):
    s, t = (Setup(device, [5, 64], 4, 2, 64, "int8", 32, "contiguous") for _ in range(2))
    k, v = (s.normal(2, 4, 2, 64).half().to(device) for _ in range(2))
    out = fai.flash_attn_with_kvcache_q8(k[:, :0].repeat(1, 1, 2, 1), *s.caches, k, v, cache_seqlens=s.lens)
    assert out.shape == (2, 0, 4, 64)
    fai.flash_attn_kvcache_append_q8(k, v, *t.caches, t.lens)
    for x, y in zip(s.caches, t.caches):
        assert torch.equal(x.float().nan_to_num(-1), y.float().nan_to_num(-1))
    none = torch.zeros(0, dtype=torch.int32, device=device)
    out = fai.flash_attn_with_kvcache_q8(k[:0].repeat(1, 1, 2, 1), *(x[:0] for x in s.caches), k[:0], v[:0], cache_seqlens=none)
    assert out.shape == (0, 4, 4, 64)
    fai.flash_attn_kvcache_append_q8(k[:0], v[:0], *(x[:0] for x in s.caches), none)
    fai.flash_attn_kvcache_append_q8(k[:, :0], v[:, :0], *s.caches, s.lens)
    got = fai.flash_attn_kvcache_read_q8(*s.caches, torch.zeros(3, dtype=torch.int32, device=device), 0)
    assert got[0].shape == (0, 2, 64)


def test_default_length(device):
    s = Setup(device, [64, 64], 0, 2, 64, "e4m3", 32, "contiguous", capacity=64)
    q = s.normal(2, 1, 2, 64).half().to(device)
    want = fai.flash_attn_with_kvcache_q8(q, *s.caches, cache_seqlens=s.lens)
    assert torch.equal(fai.flash_attn_with_kvcache_q8(q, *s.caches), want)
    assert torch.equal(fai.flash_attn_with_kvcache_q8(q, *s.caches, cache_seqlens=64), want)


def test_refusals(device):
    s = Setup(device, [5, 64], 4, 2, 64, "int8", 32, "contiguous")
    q, k = s.normal(2, 4, 4, 64).half().to(device), s.normal(2, 4, 2, 64).half().to(device)
    f = fai.flash_attn_with_kvcache_q8
    kc, vc, ks, vs = s.caches
    for caches, args, more, match in (
        ((kc.float(), vc, ks, vs), (), {}, "float8_e4m3fn or int8"),
        ((kc, vc.view(torch.float8_e4m3fn), ks, vs), (), {}, "must match"),
        ((kc, vc, ks.half(), vs), (), {}, "float32"),
        ((kc, vc, ks[:, :3], vs), (), {}, "must match"),
        ((kc, vc, ks[:, :3], vs[:, :3]), (), {}, "multiple of its scales"),
        ((kc, vc, ks.repeat(1, 2, 1), vs.repeat(1, 2, 1)), (), {}, "32, 64, 128 or 256"),
        ((kc, vc, ks[..., :1], vs), (), {}, "shape"),
        ((kc[..., :48], vc[..., :48], ks, vs), (), {}, "head_dim"),
        ((kc[:, :, :, 1:], vc, ks, vs), (), {}, "contiguous last dimension"),
        ((kc, vc, ks, vs), (k, k.bfloat16()), {}, "one dtype"),
        ((kc, vc, ks, vs), (k.bfloat16(), k.bfloat16()), {}, "dtype of q"),
        ((kc, vc, ks, vs), (k[:, :, :1], k[:, :, :1]), {}, "shape"),
        ((kc[:1].expand(2, -1, -1, -1), vc, ks, vs), (k, k), {}, "overlap"),
        ((kc, vc, ks[:1].expand(2, -1, -1), vs), (k, k), {}, "overlap"),
        ((kc[:1], vc[:1], ks[:1], vs[:1]), (), {}, "batch size"),
        ((kc.cpu(), vc, ks, vs), (), {}, "CUDA"),
    ):
        with pytest.raises(RuntimeError, match=match):
            f(q, *caches, *args, cache_seqlens=s.lens, **more)
    with pytest.raises(RuntimeError, match="divisible"):
        f(q[:, :, :3], *s.caches, cache_seqlens=s.lens)
    with pytest.raises(RuntimeError, match="float16 or bfloat16"):
        f(q.float(), *s.caches, cache_seqlens=s.lens)
    # One value of a scale for all blocks may be read, but not written.
    f(q, kc, vc, ks[:, :1].expand(-1, ks.shape[1], -1), vs, cache_seqlens=s.lens)


def test_device_checks(device):
    """validate=False: what is wrong is left alone and reported; the other sequences are served."""
    fai.flash_attn_kvcache_check()
    s = Setup(device, [5, 64, 20], 4, 2, 64, "e4m3", 32, "remapped", capacity=96)
    before = [x.clone() for x in s.caches]
    q, k, v = (s.normal(3, 4, n, 64).half().to(device) for n in (4, 2, 2))
    good = fai.flash_attn_with_kvcache_q8(q[:1], *s.caches, k[:1], v[:1], cache_seqlens=s.lens[:1], causal=True,
                                          cache_batch_idx=s.index[:1])
    after = [x.clone() for x in s.caches]
    for x, y in zip(s.caches, before):
        x.copy_(y)
    lens, index = s.lens.clone(), s.index.clone()
    lens[1], index[2] = 93, 5
    out, lse = fai.flash_attn_with_kvcache_q8(q, *s.caches, k, v, cache_seqlens=lens, causal=True, cache_batch_idx=index,
                                              validate=False, return_softmax_lse=True)
    assert torch.equal(out[:1], good) and out[1:].abs().max() == 0 and lse[1:].abs().max() == 0
    for x, y in zip(s.caches, after):
        assert torch.equal(x.float().nan_to_num(-1), y.float().nan_to_num(-1))
    with pytest.raises(ValueError, match="capacity"):
        fai.flash_attn_kvcache_check()
    for bad in (-1, 2 ** 31 - 1, 93):
        lens = s.lens.clone()
        lens[0] = bad
        fai.flash_attn_kvcache_append_q8(k, v, *s.caches, lens, cache_batch_idx=s.index, validate=False)
        with pytest.raises(ValueError, match="capacity"):
            fai.flash_attn_kvcache_check()
    new = torch.tensor([4, 5, -1], dtype=torch.int32, device=device)
    fai.flash_attn_kvcache_append_q8(k, v, *s.caches, s.lens, s.index, seqlens_new=new, validate=False)
    with pytest.raises(ValueError, match="capacity"):
        fai.flash_attn_kvcache_check()
    index = s.index.clone()
    index[0] = -1
    fai.flash_attn_kvcache_append_q8(k, v, *s.caches, s.lens, index, validate=False)
    with pytest.raises(RuntimeError, match="cache_batch_idx"):
        fai.flash_attn_kvcache_check()
    # Reads: a sequence that is longer than the capacity is 0, the others are there.
    cu = torch.tensor([0, 5, 105, 125], dtype=torch.int32, device=device)
    got = fai.flash_attn_kvcache_read_q8(*s.caches, cu, 125, s.index, validate=False)[0]
    assert got[5:105].abs().max() == 0 and got[:5].abs().max() > 0 and got[105:].abs().max() > 0
    with pytest.raises(ValueError, match="capacity"):
        fai.flash_attn_kvcache_check()
    # Starts that run backwards, or past what there is.
    for cu in ([5, 3, 9, 2], [0, 500, 20, 125], [-7, 2 ** 31 - 1, 0, 4], [200, 300, 400, 500]):
        fai.flash_attn_kvcache_read_q8(*s.caches, torch.tensor(cu, dtype=torch.int32, device=device), 125, s.index, validate=False)
        try:
            fai.flash_attn_kvcache_check()
        except ValueError:
            pass


def test_bad_pages(device):
    fai.flash_attn_kvcache_check()
    s = Setup(device, [70, 130], 4, 2, 64, "int8", 32, "paged", page=64)
    q, k, v = (s.normal(2, 4, n, 64).half().to(device) for n in (4, 2, 2))
    for bad in (-1, 10 ** 6):
        table = s.table.clone()
        table[1, 2] = bad
        before = [x.clone() for x in s.caches]
        with pytest.raises(RuntimeError, match="block_table"):
            fai.flash_attn_with_kvcache_q8(q, *s.caches, k, v, cache_seqlens=s.lens, block_table=table)
        out = fai.flash_attn_with_kvcache_q8(q, *s.caches, k, v, cache_seqlens=s.lens, block_table=table, validate=False)
        with pytest.raises(RuntimeError, match="block_table"):
            fai.flash_attn_kvcache_check()
        for x, y in zip(before, s.caches):  # the bad sequence wrote nothing
            page = int(s.table[0, 1])
            keep = [i for i in range(x.shape[0]) if i != page]
            assert torch.equal(x[keep].float().nan_to_num(-1), y[keep].float().nan_to_num(-1))
        again = fai.flash_attn_with_kvcache_q8(q[:1], *s.caches, cache_seqlens=s.lens[:1] + 4, block_table=s.table[:1])
        assert torch.equal(out[:1], again)
        cu = torch.tensor([0, 74, 74 + 134], dtype=torch.int32, device=device)
        fai.flash_attn_kvcache_read_q8(*s.caches, cu, 208, block_table=table, validate=False)
        with pytest.raises(RuntimeError, match="block_table"):
            fai.flash_attn_kvcache_check()


@pytest.mark.parametrize("queries", [1, 150])
def test_streams_and_graphs(device, queries):
    fai.flash_attn_kvcache_check()
    s = Setup(device, [300, 5, 130], 2 * queries + 8, 2, 64, "e4m3", 32, "paged", page=64)
    q, k, v = (s.normal(3, queries, n, 64).bfloat16().to(device) for n in (8, 2, 2))

    def step():
        out = fai.flash_attn_with_kvcache_q8(q, *s.caches, k, v, cache_seqlens=s.lens, causal=True, validate=False, **s.places)
        cu = torch.tensor([0, 5, 8, 20], dtype=torch.int32).to(device) if not torch.cuda.is_current_stream_capturing() else step.cu
        step.cu = cu
        return (out, *fai.flash_attn_kvcache_read_q8(*s.caches, cu, 20, validate=False, **s.places))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(want, got):
        assert torch.equal(x, y)
    graphs = []
    for _ in range(2):  # two graphs with workspaces of their own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, step()))
    for i in range(4):
        q.copy_(s.normal(*q.shape))
        s.lens.copy_(torch.tensor([300 - i, 5 + i, 130], dtype=torch.int32))
        outs = []
        for graph, out in graphs:
            graph.replay()
            torch.cuda.synchronize()
            outs.append([x.clone() for x in out])
        want = step()
        for out in outs:
            for x, y in zip(want, out):
                assert torch.equal(x, y)
    fai.flash_attn_kvcache_check()


def test_repeats_bit_for_bit(device):
    s = Setup(device, [3000, 100, 1], 0, 4, 128, "e4m3", 64, "paged")
    for sq in (1, 60):
        q = s.normal(3, sq, 16, 128).half().to(device)
        first = fai.flash_attn_with_kvcache_q8(q, *s.caches, cache_seqlens=s.lens, **s.places)
        for _ in range(5):
            assert torch.equal(first, fai.flash_attn_with_kvcache_q8(q, *s.caches, cache_seqlens=s.lens, **s.places))
    q = s.normal(3, 2, 16, 128).half().to(device)
    whole = fai.flash_attn_with_kvcache_q8(q, *s.caches, cache_seqlens=s.lens, num_splits=4, **s.places)
    for i in range(3):  # with a number of pieces, a row does not depend on the batch
        one = fai.flash_attn_with_kvcache_q8(q[i:i + 1], *s.caches, cache_seqlens=s.lens[i:i + 1], num_splits=4,
                                             block_table=s.table[i:i + 1])
        assert torch.equal(whole[i:i + 1], one)


@pytest.mark.parametrize("kind,dtype", [("e4m3", "fp16"), ("int8", "bf16")])
def test_as_it_is_used(device, kind, dtype):
    """A prompt in two pieces and ten tokens, rotated, written and attended over, against attention over the same values:
    what is read back, through the packed forward kernel (fp16) or the definition."""
    d, h, hk, prompt = 128, 8, 2, [150, 61]
    s = Setup(device, [0, 0], 320, hk, d, kind, 64, "paged", held=False)
    cos, sin = fai.flash_attn_rotary_tables(512, 64, factor=4.0, original_seqlen=128, device=device)
    mk = lambda n, heads: s.normal(2, n, heads, d).to(DTYPES[dtype]).to(device)  # noqa: E731
    lens = torch.zeros(2, dtype=torch.int32, device=device)
    q, k, v = mk(150, h), mk(150, hk), mk(150, hk)
    q, k = fai.flash_attn_rotary_func(q, k, cos, sin, seqlen_offsets=lens)
    new = torch.tensor(prompt, dtype=torch.int32, device=device)
    fai.flash_attn_kvcache_append_q8(k, v, *s.caches, lens, seqlens_new=new, **s.places)
    lens = lens + new
    for n in [40] + [1] * 10:
        q, k, v = mk(n, h), mk(n, hk), mk(n, hk)
        q, k = fai.flash_attn_rotary_func(q, k, cos, sin, seqlen_offsets=lens)
        out, lse = fai.flash_attn_with_kvcache_q8(q, *s.caches, k, v, cache_seqlens=lens, causal=True, return_softmax_lse=True,
                                                  **s.places)
        lens = lens + n
        _check(s, q, out, lse, lens.tolist(), True, (-1, -1), d ** -0.5)
    cu = torch.tensor([0, *lens.cumsum(0).tolist()], dtype=torch.int32, device=device)
    k, v = fai.flash_attn_kvcache_read_q8(*s.caches, cu, int(cu[-1]), dtype=DTYPES[dtype], **s.places)
    if dtype == "fp16":  # the last step again, over the values in 16 bits
        cu_q = torch.tensor([0, 1, 2], dtype=torch.int32, device=device)
        ref = fai.flash_attn_varlen_func(q.reshape(2, h, d), k, v, cu_q, cu, 1, int(lens.max()), causal=True)
        assert (ref.float() - out.reshape(2, h, d).float()).abs().max() <= 2.0 ** -9 * v.float().abs().max()
    # How far 8 bits are from the values: 2^-4 of each (e4m3), half a step of the largest of its block (int8).
    exact = {name: s.oracle(name) for name in "kv"}
    assert torch.equal(k[: int(lens[0])].cpu().double(), exact["k"].tokens(0, int(lens[0])))
    assert torch.equal(v[int(lens[0]):].cpu().double(), exact["v"].tokens(1, int(lens[1])))


def _widen(s, tokens, page):
    """The same cache behind a table of a larger capacity, whose further entries are no pages."""
    more = torch.full((s.table.shape[0], tokens // page), -1, dtype=torch.int32, device=s.device)
    s.table = torch.cat((s.table, more), 1)


@pytest.mark.parametrize("splits", [1, 3, 200])
@pytest.mark.parametrize("kind,dtype", [("e4m3", "bf16"), ("int8", "fp16"), ("e4m3", "fp16"), ("int8", "bf16")])
@pytest.mark.parametrize("d,block,page", [(64, 32, 32), (128, 32, 96), (128, 64, 64), (64, 256, 256)])
def test_attention_of_many_rows(device, d, block, page, kind, dtype, splits):
    """At least 64 rows a KV head and a given number of pieces: the kernel of many rows, whatever the size; heads that the
    eight XCDs do not share evenly, and more queries than keys."""
    for i, (lens, sq, h, hk, causal, window) in enumerate((
            ([0, 95, 900], 64, 3, 3, True, (-1, -1)), ([33, 20], 130, 4, 2, True, (-1, -1)), ([600, 31], 70, 6, 1, True, (200, -1)),
            ([400, 1], 65, 4, 4, False, (50, 20)), ([257], 129, 2, 2, False, (-1, 0)), ([1200], 40, 8, 1, False, (-1, -1)))):
        s = Setup(device, lens, 0, hk, d, kind, block, "paged", page=page, seed=i)
        q = s.normal(len(lens), sq, h, d).to(DTYPES[dtype]).to(device)
        out, lse = fai.flash_attn_with_kvcache_q8(q, *s.caches, cache_seqlens=s.lens, causal=causal, window_size=window,
                                                  num_splits=splits, return_softmax_lse=True, **s.places)
        _check(s, q, out, lse, lens, causal, window, d ** -0.5)


@pytest.mark.parametrize("d,kind", [(64, "e4m3"), (128, "int8")])
def test_long_pieces(device, d, kind):
    """Pieces longer than a table of places holds, with and without a window, in both kernels."""
    s = Setup(device, [17000, 8200], 0, 1, d, kind, 64, "paged", page=64)
    for sq, splits in ((4, 1), (70, 1), (70, 2), (4, 60), (70, 60)):
        q = s.normal(2, sq, 2, d).bfloat16().to(device)
        for window in ((-1, -1), (9000, -1)):
            out, lse = fai.flash_attn_with_kvcache_q8(q, *s.caches, cache_seqlens=s.lens, causal=True, window_size=window,
                                                      num_splits=splits, return_softmax_lse=True, **s.places)
            _check(s, q, out, lse, [17000, 8200], True, window, d ** -0.5)


@pytest.mark.parametrize("d,hk,capacity", [(128, 4, 0), (128, 4, 200 << 10), (128, 3, 400 << 10), (64, 4, 200 << 10),
                                           (64, 4, 800 << 10), (64, 6, 800 << 10), (64, 3, 800 << 10)])
def test_heads_of_a_workgroup(device, d, hk, capacity):
    """Few rows over capacities where a workgroup takes one, two or four KV heads."""
    lens, page = [700, 0, 77, 2000], 64
    s = Setup(device, lens, 0, hk, d, "e4m3", 64, "paged", page=page)
    for sq in (1, 3, 9):
        q = s.normal(4, sq, 4 * hk, d).bfloat16().to(device)
        args = dict(cache_seqlens=s.lens, causal=True, num_splits=0, return_softmax_lse=True)
        want = fai.flash_attn_with_kvcache_q8(q, *s.caches, block_table=s.table, **args)
        _check(s, q, *want, lens, True, (-1, -1), d ** -0.5)
        if capacity:
            table = s.table
            _widen(s, capacity, page)
            got = fai.flash_attn_with_kvcache_q8(q, *s.caches, block_table=s.table, **args)
            _check(s, q, *got, lens, True, (-1, -1), d ** -0.5)
            s.table = table


def test_many_rows_by_the_work(device):
    """The same call on both sides of the amount of work where the kernel of many rows takes over."""
    lens, page = [3000, 400, 1100], 64
    s = Setup(device, lens, 0, 4, 128, "e4m3", 64, "paged", page=page)
    table = s.table
    for sq, h in ((8, 16), (33, 4), (100, 8)):
        q = s.normal(3, sq, h, 128).half().to(device)
        for wide in (0, 1 << 20):
            s.table = table
            if wide:
                _widen(s, wide, page)
            out, lse = fai.flash_attn_with_kvcache_q8(q, *s.caches, cache_seqlens=s.lens, causal=True, return_softmax_lse=True,
                                                      **s.places)
            _check(s, q, out, lse, lens, True, (-1, -1), 128 ** -0.5)


@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("kind,dtype", [("e4m3", "fp16"), ("e4m3", "bf16"), ("int8", "fp16"), ("int8", "bf16")])
def test_any_scales_of_few_and_many_rows(device, kind, dtype, rows):
    """Scales of another quantiser, 0, far apart; a softmax_scale of either sign and 0; scores that grow along the keys."""
    lens, d = [700, 97], 64
    for i, (scale, growth) in enumerate(((0.125, 1), (-0.3, 1), (0.0, 1), (0.5, 40), (-0.5, 40))):
        s = Setup(device, lens, 0, 2, d, kind, 32, "contiguous", seed=i)
        for name in ("ks", "vs"):
            x = getattr(s, name)
            x.copy_(torch.rand(x.shape, generator=s.g) * (0.02 if kind == "e4m3" else 0.05))
        s.vs[0, 1] = 0
        s.vs[0, 2] = 2.0 ** -40
        s.vs[0, 5] *= 300
        s.ks[0, 3] = 0
        s.ks *= torch.linspace(1 / growth, growth ** 0.5, s.ks.shape[1], device=device)[None, :, None]
        q = s.normal(2, rows, 4, d).to(DTYPES[dtype]).to(device)
        out, lse = fai.flash_attn_with_kvcache_q8(q, *s.caches, cache_seqlens=s.lens, causal=True, softmax_scale=scale,
                                                  num_splits=i % 2 + 1, return_softmax_lse=True)
        _check(s, q, out, lse, lens, True, (-1, -1), scale)


@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_not_a_number_and_infinity(device, kind, rows):
    """A block that is not finite makes those rows NaN that see it, and no others."""
    lens, d, block = [300, 300], 128, 32
    for bad in ("k", "v"):
        s = Setup(device, lens, 0, 2, d, kind, block, "contiguous")
        q = s.normal(2, rows, 4, d).bfloat16().to(device)
        args = dict(cache_seqlens=s.lens, causal=True, window_size=(60, -1), num_splits=1)
        want = fai.flash_attn_with_kvcache_q8(q, *s.caches, **args)
        getattr(s, bad + "s")[0, 7, 1] = math.nan  # keys 224 .. 255 of KV head 1
        getattr(s, bad + "s")[1, 2, 0] = math.nan  # keys 64 .. 95: no window reaches back to them from here
        got = fai.flash_attn_with_kvcache_q8(q, *s.caches, **args)
        assert torch.equal(got[1], want[1])
        for r in range(rows):
            pos = 300 - rows + r
            hit = pos >= 224 and pos - 60 <= 255
            assert torch.equal(got[0, r, :2], want[0, r, :2])
            assert got[0, r, 2:].isnan().all() if hit else torch.equal(got[0, r, 2:], want[0, r, 2:])


def test_offsets_past_32_bits(device):
    """The last pages of a pool of 4.6 GB of codes each for K and V, against the same pages in a small one."""
    page, hk, d, pages = 64, 8, 128, 70000
    small = Setup(device, [150, 64], 0, hk, d, "e4m3", 64, "paged", page=page, capacity=320)
    big = [torch.empty(pages, *x.shape[1:], dtype=x.dtype, device=device) for x in small.caches]
    n = small.kc.shape[0]
    for x, y in zip(big, small.caches):
        x[-n:] = y
    far = torch.where(small.table >= 0, small.table + pages - n, small.table)
    table = small.table
    q = small.normal(2, 70, 16, d).bfloat16().to(device)
    cu = torch.tensor([0, 150, 214], dtype=torch.int32, device=device)
    for splits, rows in ((0, 1), (1, 70), (0, 70)):
        args = dict(cache_seqlens=small.lens, causal=True, num_splits=splits)
        want = fai.flash_attn_with_kvcache_q8(q[:, :rows], *small.caches, block_table=table, **args)
        assert torch.equal(fai.flash_attn_with_kvcache_q8(q[:, :rows], *big, block_table=far, **args), want)
    for x, y in zip(fai.flash_attn_kvcache_read_q8(*big, cu, 214, block_table=far),
                    fai.flash_attn_kvcache_read_q8(*small.caches, cu, 214, block_table=table)):
        assert torch.equal(x, y)
    k = small.normal(2, 10, hk, d).bfloat16().to(device)
    lens = small.lens - 10
    fai.flash_attn_kvcache_append_q8(k, k, *small.caches, lens, block_table=table)
    fai.flash_attn_kvcache_append_q8(k, k, *big, lens, block_table=far)
    for x, y in zip(big, small.caches):
        assert torch.equal(x[-n:].float().nan_to_num(-1), y.float().nan_to_num(-1))


def test_copied_pages(device):
    """copy_pages moves codes and, as pools of their own, scales: attention over the copies is attention over the originals."""
    s = Setup(device, [150, 64], 0, 4, 64, "e4m3", 32, "paged", page=64)
    pages = s.kc.shape[0]
    pools = [torch.cat((x, torch.zeros_like(x))) for x in s.caches]
    src = torch.arange(pages, dtype=torch.int32, device=device)
    fai.flash_attn_kvcache_copy_pages(pools[0], pools[1], src, src + pages)
    fai.flash_attn_kvcache_copy_pages(*(x.view(2 * pages, 1, 1, -1) for x in pools[2:]), src, src + pages)
    q = s.normal(2, 3, 8, 64).half().to(device)
    want = fai.flash_attn_with_kvcache_q8(q, *s.caches, cache_seqlens=s.lens, causal=True, **s.places)
    table = torch.where(s.table >= 0, s.table + pages, s.table)
    assert torch.equal(fai.flash_attn_with_kvcache_q8(q, *pools, cache_seqlens=s.lens, causal=True, block_table=table), want)


def test_c_entry_points(device):
    """The plain C calls: what they refuse before anything is launched, and workspace sizes of calls that have none."""
    import ctypes

    import fa_capi

    lib = fa_capi.load()
    a = fa_capi.FaKv8Args()
    assert lib.fa_kv8_attention(None, None) < 0 and lib.fa_kv8_append(None, None) < 0 and lib.fa_kv8_read(None, None) < 0
    for head_dim in (0, 48, 512, -64):
        a.cache.batch, a.cache.nheads_k, a.nheads, a.seqlen_q, a.cache.head_dim = 2, 2, 4, 1, head_dim
        assert lib.fa_kv8_ws_bytes(ctypes.byref(a)) == 0
        assert lib.fa_kv8_attention(ctypes.byref(a), None) < 0
    a.cache.head_dim, a.cache.cache_capacity, a.cache.nheads_k = 64, 256, 8
    assert lib.fa_kv8_ws_bytes(ctypes.byref(a)) == 0  # more KV heads than heads
    a.cache.nheads_k = 2
    assert lib.fa_kv8_ws_bytes(ctypes.byref(a)) > 0
    assert lib.fa_kv8_attention(ctypes.byref(a), None) < 0  # (no tensors)


def test_the_largest_capacity(device):
    """2^30 tokens behind a table; one page more is refused."""
    page = 1 << 10
    s = Setup(device, [3000, 1], 0, 2, 64, "e4m3", 32, "paged", page=page)
    q = s.normal(2, 1, 4, 64).half().to(device)
    table = s.table
    for cols, rows in ((1 << 20, 1), (1 << 20, 70)):
        s.table = table
        _widen(s, cols * page - table.shape[1] * page, page)
        q = s.normal(2, rows, 4, 64).half().to(device)
        out, lse = fai.flash_attn_with_kvcache_q8(q, *s.caches, cache_seqlens=s.lens, causal=True, return_softmax_lse=True,
                                                  validate=False, **s.places)
        _check(s, q, out, lse, [3000, 1], True, (-1, -1), 0.125)
    fai.flash_attn_kvcache_check()
    _widen(s, page, page)
    with pytest.raises(RuntimeError):
        fai.flash_attn_with_kvcache_q8(q, *s.caches, cache_seqlens=s.lens, validate=False, **s.places)
