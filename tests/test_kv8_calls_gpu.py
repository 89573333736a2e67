"""Calls on a KV cache in 8 bits that its documents allow: rows and pages that several sequences of a call read, appends and
reads that are captured and replayed, and calls on two streams at once."""

import pytest
import torch

import flash_attention_interface as fai
from test_kv8_gpu import Setup, _check_append, _same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 70])
def test_rows_and_pages_that_sequences_share(device, rows):
    """The same cache row, or pages, for several sequences of a call that appends nothing, to different lengths."""
    s = Setup(device, [300, 200], 0, 2, 64, "e4m3", 32, "contiguous")
    index = torch.tensor([1, 0, 1, 0, 0], dtype=torch.int32, device=device)
    lens = torch.tensor([200, 300, 7, 0, 129], dtype=torch.int32, device=device)
    q = s.normal(5, rows, 4, 64).half().to(device)
    out = fai.flash_attn_with_kvcache_q8(q, *s.caches, cache_seqlens=lens, cache_batch_idx=index, causal=True, num_splits=2)
    for i in range(5):
        one = fai.flash_attn_with_kvcache_q8(q[i:i + 1], *s.caches, cache_seqlens=lens[i:i + 1], cache_batch_idx=index[i:i + 1],
                                             causal=True, num_splits=2)
        assert torch.equal(out[i:i + 1], one)
    p = Setup(device, [300, 200], 0, 2, 64, "int8", 32, "paged", page=64)
    table = p.table[[1, 0, 0]].clone()
    table[2, 2:] = -1
    lens = torch.tensor([200, 300, 128], dtype=torch.int32, device=device)
    out = fai.flash_attn_with_kvcache_q8(q[:3], *p.caches, cache_seqlens=lens, block_table=table, causal=True, num_splits=2)
    for i in range(3):
        one = fai.flash_attn_with_kvcache_q8(q[i:i + 1], *p.caches, cache_seqlens=lens[i:i + 1], block_table=table[i:i + 1],
                                             causal=True, num_splits=2)
        assert torch.equal(out[i:i + 1], one)
    cu = torch.tensor([0, 200, 500, 628], dtype=torch.int32, device=device)
    k, v = fai.flash_attn_kvcache_read_q8(*p.caches, cu, 628, block_table=table)
    assert torch.equal(k[500:], k[200:328]) and torch.equal(v[500:], v[200:328])


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_captured_appends_and_reads(device, kind):
    """A padded append and a read in one graph, replayed while lengths, new tokens and their magnitudes change, so that scales
    grow and blocks fill and begin between the replays."""
    fai.flash_attn_kvcache_check()
    s = Setup(device, [0, 20, 63], 140, 2, 64, kind, 32, "paged", page=64)
    k, v = (torch.zeros(3, 40, 2, 64, dtype=torch.bfloat16, device=device) for _ in "kv")
    new = torch.zeros(3, dtype=torch.int32, device=device)
    cu = torch.zeros(4, dtype=torch.int32, device=device)

    def step():
        fai.flash_attn_kvcache_append_q8(k, v, *s.caches, s.lens, seqlens_new=new, validate=False, **s.places)
        return fai.flash_attn_kvcache_read_q8(*s.caches, cu, 500, dtype=torch.bfloat16, validate=False, **s.places)

    step()  # (of no tokens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i, news in enumerate(([40, 0, 1], [1, 12, 0], [25, 40, 40], [0, 3, 5])):
        x, y = (s.normal(3, 40, 2, 64) * 2.0 ** (2 * i) for _ in "kv")
        k.copy_(x)
        v.copy_(y)
        new.copy_(torch.tensor(news, dtype=torch.int32))
        s.lens.copy_(torch.tensor(s.lens_list, dtype=torch.int32))
        after = [n + m for n, m in zip(s.lens_list, news)]
        cu.copy_(torch.tensor([0, after[0], sum(after[:2]), sum(after)], dtype=torch.int32))
        want = dict(_check_append(s, news, k, v, "bf16"))
        graph.replay()
        torch.cuda.synchronize()
        s.lens_list = after
        for j, (name, o) in enumerate(want.items()):
            _same(getattr(s, name + "c"), o.codes, f"codes of {name}, replay {i}")
            _same(getattr(s, name + "s"), o.scales, f"scales of {name}, replay {i}")
            values = torch.cat([o.tokens(b, n) for b, n in enumerate(after)]).to(torch.bfloat16)
            assert torch.equal(out[j][:len(values)].cpu(), values) and out[j][len(values):].abs().max() == 0
    fai.flash_attn_kvcache_check()


def test_two_streams_at_once(device):
    """Calls of both kernels over one cache, split into pieces, on two streams without order between them."""
    s = Setup(device, [3000, 100, 1700], 0, 4, 128, "e4m3", 64, "paged")
    few, many = (s.normal(3, n, 16, 128).bfloat16().to(device) for n in (1, 60))
    call = lambda q: fai.flash_attn_with_kvcache_q8(q, *s.caches, cache_seqlens=s.lens, causal=True, num_splits=n,  # noqa: E731
                                                    validate=False, **s.places)
    for n in (0, 5):
        want = [call(few), call(many)]
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for x in streams:
            x.wait_stream(torch.cuda.current_stream())
        got = [[], []]
        for i in range(12):
            with torch.cuda.stream(streams[i % 2]):
                got[i % 2].append((i // 2 % 2, call((few, many)[i // 2 % 2])))
        torch.cuda.synchronize()
        for side in got:
            for which, x in side:
                assert torch.equal(x, want[which])


def test_captured_tables(device):
    graph = torch.cuda.CUDAGraph()
    want = fai.flash_attn_rotary_tables(300, 64, factor=4.0, original_seqlen=128, device=device)
    with torch.cuda.graph(graph):
        got = fai.flash_attn_rotary_tables(300, 64, factor=4.0, original_seqlen=128, device=device)
    for _ in range(3):
        for x in got:
            x.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
