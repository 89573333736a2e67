"""Rotary positions on the GPU: tables and rotation against the definition in 64 bits, elementwise, within the roundings that
oracle/rotary.py counts; gradients, layouts, positions, streams and graphs."""

import pytest
import torch

import flash_attention_interface as fai
from oracle.rotary import rotate, tables

pytestmark = pytest.mark.gpu

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _close(got, want, bound, name):
    got = got.detach().double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), name
    worst = ((got - want).abs() - bound).nan_to_num(nan=-1.0).max()
    assert float(worst) <= 0, f"{name}: over its bound by {float(worst):.3g}"


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("seqlen,rotary,more", [
    (1, 16, {}), (77, 48, dict(base=500000.0)), (513, 128, dict(factor=4.0, attention_factor=1.2)),
    (300, 64, dict(factor=32.0, original_seqlen=4096, attention_factor=1.35, offset=131000 - 300)),
    (9, 256, dict(offset=1 << 17)), (5, 32, dict(offset=-3)),
])
def test_tables(device, dtype, seqlen, rotary, more):
    got = dict(zip(("cos", "sin"), fai.flash_attn_rotary_tables(seqlen, rotary, dtype=DTYPES[dtype], device=device, **more)))
    want = tables(seqlen, rotary, dtype=DTYPES[dtype], **more)
    for name in got:
        assert got[name].shape == (seqlen, rotary // 2) and got[name].dtype == DTYPES[dtype]
        _close(got[name], *want[name], name)


def test_tables_of_no_rows(device):
    cos, sin = fai.flash_attn_rotary_tables(0, 32, device=device)
    assert cos.shape == sin.shape == (0, 16)


def _tables(g, rows, rotary, dtype, device):
    # Any numbers will do: the rotation takes what the tables hold.
    return [torch.randn(rows, rotary // 2, generator=g).to(dtype).to(device) for _ in range(2)]


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("dtype,table", [("fp16", "fp32"), ("bf16", "bf16"), ("bf16", "fp32"), ("fp16", "fp16"), ("fp16", "bf16")])
@pytest.mark.parametrize("dim,rotary", [(64, 64), (64, 16), (128, 128), (128, 48), (128, 64), (128, 112)])
def test_dense(device, dim, rotary, dtype, table, interleaved):
    g = torch.Generator().manual_seed(dim + rotary)
    for batch, seqlen, heads, heads_k in ((1, 1, 1, 1), (2, 7, 6, 2), (1, 5, 40, 8), (3, 3, 5, 0)):
        mk = lambda n: torch.randn(batch, seqlen, n, dim, generator=g).to(DTYPES[dtype])  # noqa: E731
        q, k = mk(heads), mk(heads_k) if heads_k else None
        dq, dk = mk(heads), mk(heads_k) if heads_k else None
        cos, sin = _tables(g, seqlen + 4, rotary, DTYPES[table], "cpu")
        qd = q.to(device).requires_grad_()
        kd = k.to(device).requires_grad_() if heads_k else None
        got = fai.flash_attn_rotary_func(qd, kd, cos.to(device), sin.to(device), rotary_interleaved=interleaved, seqlen_offsets=4)
        outs = got if heads_k else (got,)
        grads = torch.autograd.grad(outs, (qd, kd) if heads_k else (qd,), [t.to(device) for t in (dq, dk) if t is not None])
        at = list(range(4, 4 + seqlen)) * batch
        for name, x, d, y, dx in zip("qk", (q, k), (dq, dk), outs, grads):
            assert y.shape == x.shape and y.dtype == x.dtype
            for what, a, b, inverse in ((name, x, y, False), ("d" + name, d, dx, True)):
                want, bound = rotate(a.flatten(0, 1), cos, sin, at, interleaved, inverse)
                _close(b.flatten(0, 1), want, bound, f"{what} {batch, seqlen, heads, heads_k}")
                if rotary < dim:  # the channels that are left keep their bits
                    assert torch.equal(b[..., rotary:].cpu(), a[..., rotary:])


@pytest.mark.parametrize("lengths,before,behind", [([1], 0, 0), ([3, 0, 5], 2, 4), ([0, 0, 1, 0], 0, 1), ([2] * 130 + [0] * 70 + [1], 0, 3)])
def test_packed(device, lengths, before, behind):
    g = torch.Generator().manual_seed(len(lengths))
    cu, at = [before], [None] * before
    offsets = torch.randint(0, 6, (len(lengths),), generator=g, dtype=torch.int32)
    for n, o in zip(lengths, offsets.tolist()):
        cu.append(cu[-1] + n)
        at += range(o, o + n)
    at += [None] * behind
    q, k = (torch.randn(len(at), h, 64, generator=g).to(torch.bfloat16) for h in (4, 2))
    cos, sin = _tables(g, 12, 32, torch.float32, "cpu")
    qd, kd = (t.to(device).requires_grad_() for t in (q, k))
    cu = torch.tensor(cu, dtype=torch.int32, device=device)
    out = fai.flash_attn_rotary_func(qd, kd, cos.to(device), sin.to(device), False, cu_seqlens=cu, seqlen_offsets=offsets.to(device))
    grads = torch.autograd.grad(out, (qd, kd), (out[0].detach(), out[1].detach()))
    for name, x, y, d in zip("qk", (q, k), out, grads):
        _close(y, *rotate(x, cos, sin, at, False), name)
        _close(d, *rotate(y.detach().cpu(), cos, sin, at, False, inverse=True), "d" + name)
    # The same places, named one by one; rows of no sequence are at 0 there.
    positions = torch.tensor([p or 0 for p in at], dtype=torch.int32, device=device)
    again = fai.flash_attn_rotary_func(qd, kd, cos.to(device), sin.to(device), False, cu_seqlens=cu, positions=positions)
    for y, z in zip(out, again):
        assert torch.equal(y, z)


def test_positions_and_ends_of_the_tables(device):
    g = torch.Generator().manual_seed(5)
    q = torch.randn(2, 4, 3, 64, generator=g).to(torch.float16)
    cos, sin = _tables(g, 10, 32, torch.float32, "cpu")
    at = [[9, 0, 10, -1], [3, 3, 2 ** 31 - 1, -(2 ** 31)]]
    got = fai.flash_attn_rotary_func(q.to(device), None, cos.to(device), sin.to(device),
                                     positions=torch.tensor(at, dtype=torch.int32, device=device))
    _close(got.flatten(0, 1), *rotate(q.flatten(0, 1), cos, sin, at[0] + at[1], True), "q")
    # Every second column of a wider tensor of positions, and offsets that pass 32 bits with the row.
    wide = torch.tensor(at, dtype=torch.int32, device=device).repeat_interleave(2, 1)[:, ::2]
    again = fai.flash_attn_rotary_func(q.to(device), None, cos.to(device), sin.to(device), positions=wide)
    assert torch.equal(got.view(torch.int16), again.view(torch.int16))
    for offset in (2 ** 31 - 2, -(2 ** 31), torch.full((2,), 2 ** 31 - 2, dtype=torch.int32, device=device)):
        far = fai.flash_attn_rotary_func(q.to(device), None, cos.to(device), sin.to(device), seqlen_offsets=offset)
        assert far[..., :32].isnan().all() and torch.equal(far[..., 32:].cpu(), q[..., 32:])


def test_strides_and_expanded_gradients(device):
    g = torch.Generator().manual_seed(6)
    qkv = torch.randn(2, 6, 3, 4, 128, generator=g).to(torch.bfloat16).to(device)
    cos, sin = _tables(g, 6, 128, torch.float32, device)
    want = fai.flash_attn_rotary_func(*(qkv[:, :, i].contiguous() for i in (0, 1)), cos, sin)
    wide = torch.zeros(6, 72, device=device)
    wide[:, 3:67] = cos
    odd = torch.empty(2 * 6 * 4 * 128 + 1, dtype=torch.bfloat16, device=device)[1:].view(2, 6, 4, 128)
    odd.copy_(qkv[:, :, 1])
    for q, k, c in ((qkv[:, :, 0], qkv[:, :, 1], cos), (qkv[:, :, 0].transpose(1, 2).contiguous().transpose(1, 2), odd, cos),
                    (qkv[:, :, 0].transpose(1, 3).contiguous().transpose(1, 3), odd, wide[:, 3:67])):
        for y, z in zip(want, fai.flash_attn_rotary_func(q, k, c, sin)):
            assert torch.equal(y, z)
    q, k = (qkv[:, :, i].detach().requires_grad_() for i in (0, 1))
    out = fai.flash_attn_rotary_func(q, k, cos, sin)
    one = torch.ones((), dtype=torch.bfloat16, device=device).expand(out[0].shape)
    dq, dk = torch.autograd.grad(out, (q, k), (one, one))
    full = fai.flash_attn_rotary_func(one.contiguous(), one.contiguous(), cos, -sin)
    assert torch.equal(dq, full[0]) and torch.equal(dk, full[1])
    # One of the two alone gets a gradient.
    for i in (0, 1):
        out = fai.flash_attn_rotary_func(q, k, cos, sin)
        d = torch.autograd.grad(out[i], (q, k)[i], one)[0]
        assert torch.equal(d, full[i])
    # A head shared by all, broadcast: its gradient is the heads' sum.
    shared = torch.randn(2, 6, 1, 128, generator=g).to(torch.bfloat16).to(device).requires_grad_()
    out = fai.flash_attn_rotary_func(shared.expand(2, 6, 4, 128), None, cos, sin)
    d = torch.autograd.grad(out, shared, one)[0]
    assert d.shape == shared.shape
    assert torch.equal(d, (full[0].float().sum(2, keepdim=True)).to(torch.bfloat16)) or \
        (d.float() - full[0].float().sum(2, keepdim=True)).abs().max() <= 2.0 ** -7 * full[0].float().abs().sum(2).max()


def test_empty(device):
    cos, sin = _tables(torch.Generator().manual_seed(0), 4, 32, torch.float32, device)
    for shape in ((0, 4, 2, 64), (2, 0, 2, 64), (2, 4, 0, 64)):
        q = torch.zeros(shape, dtype=torch.float16, device=device)
        out = fai.flash_attn_rotary_func(q, q, cos, sin)
        assert out[0].shape == out[1].shape == shape
    q, k = torch.zeros(2, 4, 0, 64, dtype=torch.float16, device=device), torch.ones(2, 4, 1, 64, dtype=torch.float16, device=device)
    assert torch.equal(fai.flash_attn_rotary_func(q, k, cos, sin)[1], fai.flash_attn_rotary_func(k, None, cos, sin))


def test_refusals(device):
    g = torch.Generator().manual_seed(0)
    cos, sin = _tables(g, 4, 32, torch.float32, device)
    q = torch.zeros(1, 4, 2, 64, dtype=torch.float16, device=device)
    f = fai.flash_attn_rotary_func
    for args, more, match in (
        ((q.float(), None, cos, sin), {}, "float16 or bfloat16"),
        ((q, q.bfloat16(), cos, sin), {}, "dtype of q"),
        ((q, q[:, :3], cos, sin), {}, "shape of q"),
        ((q[0], None, cos, sin), {}, "rank-4"),
        ((q, None, cos, sin), dict(cu_seqlens=torch.zeros(2, dtype=torch.int32, device=device)), "rank-3"),
        ((q, None, cos, sin[:3]), {}, "must match"),
        ((q, None, cos.double(), sin.double()), {}, "float32, float16 or bfloat16"),
        ((q, None, cos[:, :4], sin[:, :4]), {}, "rotary_dim"),
        ((q, None, torch.zeros(4, 48, device=device), torch.zeros(4, 48, device=device)), {}, "rotary_dim"),
        ((q, None, cos[:0], sin[:0]), {}, "must have a row"),
        ((q, None, cos.cpu(), sin.cpu()), {}, "device of q"),
        ((q[..., :32], None, cos, sin), {}, "head_dim"),
        ((q, None, cos, sin), dict(positions=torch.zeros(1, 3, dtype=torch.int32, device=device)), "leading shape"),
        ((q, None, cos, sin), dict(positions=torch.zeros(1, 4, dtype=torch.int32, device=device), seqlen_offsets=1), "exclude"),
        ((q, None, cos, sin), dict(seqlen_offsets=torch.zeros(2, dtype=torch.int32, device=device)), "batch_size"),
        ((q, None, cos, sin), dict(seqlen_offsets=1 << 40), "32 bits"),
    ):
        with pytest.raises(RuntimeError, match=match):
            f(*args, **more)


def test_streams_and_graphs(device):
    g = torch.Generator().manual_seed(8)
    cos, sin = _tables(g, 40, 64, torch.float32, device)
    q, k, d = (torch.randn(2, 33, h, 64, generator=g).to(torch.float16).to(device) for h in (4, 2, 4))
    q.requires_grad_()
    offsets = torch.tensor([0, 5], dtype=torch.int32, device=device)

    def step():
        a, b = fai.flash_attn_rotary_func(q, k, cos, sin, seqlen_offsets=offsets)
        return a, b, torch.autograd.grad(a, q, d)[0]

    want = [t.detach().clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(want, got):
        assert torch.equal(x, y)
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        with torch.no_grad():
            q.copy_(torch.randn(q.shape, generator=g).to(q.dtype))
        offsets.copy_(torch.tensor([i, 7 - i], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(step(), out):
            assert torch.equal(x, y)


def test_same_as_the_caches_rotation(device):
    """q and k rotated here and then attended over equal flash_attn_with_kvcache's own rotation, within the rounding
    of the cache's k and of q to fp16 (both round once)."""
    g = torch.Generator().manual_seed(9)
    mk = lambda *s: torch.randn(*s, generator=g).to(torch.float16).to(device)  # noqa: E731
    q, k, v, kc, vc = mk(2, 3, 4, 64), mk(2, 3, 2, 64), mk(2, 3, 2, 64), mk(2, 64, 2, 64), mk(2, 64, 2, 64)
    lens = torch.tensor([5, 40], dtype=torch.int32, device=device)
    for interleaved in (True, False):
        cos, sin = fai.flash_attn_rotary_tables(64, 32, dtype=torch.float16, device=device)
        kc2, vc2 = kc.clone(), vc.clone()
        fai.flash_attn_with_kvcache(q, kc, vc, k, v, cos, sin, cache_seqlens=lens, causal=True, rotary_interleaved=interleaved)
        q2, k2 = fai.flash_attn_rotary_func(q, k, cos, sin, interleaved, seqlen_offsets=lens)
        fai.flash_attn_with_kvcache(q2, kc2, vc2, k2, v, cache_seqlens=lens, causal=True)
        assert (kc.float() - kc2.float()).abs().max() <= 2.0 ** -10 * kc.float().abs().max()
        assert torch.equal(vc, vc2)
