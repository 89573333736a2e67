"""Differential attention on the GPU: forward, gradients, packed batches, layouts, streams and graphs.

Every value is held to the elementwise error bound that oracle/diff.py derives from
the roundings of a kernel that computes as documented."""

import pytest
import torch

import flash_attention_interface as fai
from helpers import cu_from_lengths
from oracle.diff import assert_within, diff_attention

pytestmark = pytest.mark.gpu


def _inputs(device, b, sq, sk, h, hk, d, kind, dtype, seed, scale_q=1.0):
    g = torch.Generator().manual_seed(seed)
    mk = lambda *s: torch.randn(*s, generator=g).to(dtype).to(device)  # noqa: E731
    shape = {"layer": (), "head": (h,), "token": (b, sq, h)}[kind]
    lam = (torch.randn(shape, generator=g) * 0.5 + 0.4).to(device)
    return mk(b, sq, h, d) * scale_q, mk(b, sk, hk, d), mk(b, sk, hk, d), lam, mk(b, sq, h, d)


def _check(q, k, v, lam, do, causal, scale=None, names=("out", "dq", "dk", "dv", "dlam")):
    leaves = [x.detach().requires_grad_() for x in (q, k, v, lam)]
    out = fai.flash_diff_attn_func(*leaves, softmax_scale=scale, causal=causal)
    grads = torch.autograd.grad(out, leaves, do)
    want = diff_attention(q, k, v, lam, scale, causal, do)
    got = dict(zip(("out", "dq", "dk", "dv", "dlam"), (out, *grads)))
    for name in names:
        assert got[name].dtype == (torch.float32 if name == "dlam" else q.dtype)
        assert_within(name, got[name], want[name])
    with torch.no_grad():
        plain = fai.flash_diff_attn_func(q, k, v, lam, softmax_scale=scale, causal=causal)
    assert torch.equal(plain, out)  # keeping what the backward needs changes nothing
    return got


# Sizes around the 32-row tiles, 64-key blocks, 128-row and 128-key workgroups, from one token on; queries without
# keys; groups that pack into a workgroup (1, 2, 4, 8) and that do not (3); grids below and above the CU count (one
# and two wave groups); shared and unshared dK/dV items.
CASES = [
    (1, 1, 1, 1, 1, 64, True, "layer", torch.float16),
    (2, 1, 1, 4, 2, 128, False, "token", torch.bfloat16),
    (1, 1, 70, 8, 2, 64, True, "token", torch.float16),
    (2, 31, 33, 2, 2, 128, True, "head", torch.bfloat16),
    (1, 64, 64, 4, 4, 128, False, "layer", torch.float16),
    (1, 64, 64, 3, 1, 64, True, "head", torch.bfloat16),
    (2, 65, 63, 6, 2, 64, True, "token", torch.float16),
    (1, 127, 129, 8, 1, 128, True, "head", torch.float16),
    (1, 130, 5, 4, 2, 128, True, "token", torch.bfloat16),
    (1, 5, 300, 4, 4, 128, False, "layer", torch.bfloat16),
    (2, 257, 257, 4, 1, 64, True, "layer", torch.float16),
    (1, 200, 320, 2, 1, 128, True, "token", torch.float16),
    (1, 520, 520, 8, 2, 128, True, "head", torch.bfloat16),
    (4, 140, 140, 32, 8, 64, True, "head", torch.float16),
    (3, 300, 130, 32, 32, 64, False, "layer", torch.bfloat16),
    (9, 33, 40, 32, 32, 128, True, "head", torch.float16),
]


@pytest.mark.parametrize("b,sq,sk,h,hk,d,causal,kind,dtype", CASES)
def test_forward_and_gradients(device, b, sq, sk, h, hk, d, causal, kind, dtype):
    _check(*_inputs(device, b, sq, sk, h, hk, d, kind, dtype, 11), causal)


# More workgroups than the chip has places for, with and without a mask, so that every one of them has whole rows,
# ragged ones and a row of its own (one group of waves); and causal grids between one and two workgroups on a CU.
@pytest.mark.parametrize("b,sq,sk,h,hk,d,causal,dtype", [
    (13, 150, 170, 32, 32, 128, True, torch.float16),
    (13, 129, 129, 32, 32, 64, True, torch.bfloat16),
    (9, 150, 97, 32, 32, 128, False, torch.bfloat16),
    (10, 200, 200, 32, 16, 64, True, torch.float16),
    (5, 129, 260, 32, 32, 128, True, torch.bfloat16),
])
def test_grids_that_fill_the_chip(device, b, sq, sk, h, hk, d, causal, dtype):
    _check(*_inputs(device, b, sq, sk, h, hk, d, "head", dtype, 23), causal)


@pytest.mark.parametrize("scale", [-0.2, 0.0, 2.0])
def test_scales(device, scale):
    _check(*_inputs(device, 1, 100, 140, 4, 2, 64, "token", torch.float16, 5), True, scale)


@pytest.mark.parametrize("value", [0.0, 1.0, -3.5])
def test_lam_values(device, value):
    q, k, v, lam, do = _inputs(device, 2, 90, 90, 4, 2, 128, "head", torch.bfloat16, 6)
    _check(q, k, v, torch.full_like(lam, value), do, True)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_rising_and_large_scores(device, dtype):
    # Keys that grow along the sequence raise every row's maximum in every block; rows are dominated by few keys.
    q, k, v, lam, do = _inputs(device, 1, 256, 256, 2, 2, 128, "layer", dtype, 8, scale_q=3.0)
    k = (k * torch.linspace(0.1, 3.0, 256, device=device)[None, :, None, None]).to(dtype)
    _check(q, k, v, lam, do, False)
    q = q.abs()
    k = (torch.linspace(0.0, 2.0, 256, device=device)[None, :, None, None] * k.abs()).to(dtype)
    _check(q, k, v, lam, do, True, names=("out", "dv", "dlam"))


@pytest.mark.parametrize("jump", [9.0, 10.5, 25.0, 300.0, -60.0])
@pytest.mark.parametrize("d,dtype", [(64, torch.float16), (128, torch.bfloat16)])
def test_scores_that_jump(device, d, dtype, jump):
    # Keys from 130 on score `jump` above the ones before, in one map for even queries and in both for odd ones: short
    # of what the forward kernel's maximum lets pass (2^15, 10.4), past it, far past it, and below.
    q, k, v, lam, do = _inputs(device, 2, 200, 260, 4, 2, d, "head", dtype, 17)
    scale = (d // 2) ** -0.5
    for half in (0, d // 2):
        q[..., half] = 8.0
        k[..., half] = 0.0
        k[:, 130:, :, half] = jump / (8.0 * scale)
    q[:, ::2, :, d // 2] = 0.0
    for causal in (False, True):
        _check(q, k, v, lam, do, causal)


def test_a_dlam_that_many_rows_share(device):
    # 2 x 1024 rows x 8 heads: the terms' signs vary and the sum is small, so a common leaning of the terms shows
    # (they were once 3e-8 low each).  Bound: 16384 terms of at most 4e-7 each that do not lean add up to
    # 128 * 4e-7 = 5e-5 at most in the root of the sum of squares; leaning they were 5e-4.
    q, k, v, lam, do = _inputs(device, 2, 1024, 1024, 8, 8, 128, "token", torch.float16, 3)
    shared = torch.tensor(0.6, device=device).requires_grad_()
    each = torch.full_like(lam, 0.6).requires_grad_()
    a = torch.autograd.grad(fai.flash_diff_attn_func(q, k, v, shared), shared, do)[0]
    rows = torch.autograd.grad(fai.flash_diff_attn_func(q, k, v, each), each, do)[0]
    assert abs(float(rows.double().sum()) - float(a)) <= 2.0 ** -23 * abs(float(a)) + 1e-9
    want = sum(float(diff_attention(q[i:i + 1, :, j:j + 1], k[i:i + 1, :, j:j + 1], v[i:i + 1, :, j:j + 1],
                                    torch.tensor(0.6, device=device), None, False, do[i:i + 1, :, j:j + 1])["dlam"][0])
               for i in range(2) for j in range(8))
    assert abs(float(a) - want) <= 5e-5


def test_layouts(device):
    # Slices of a packed tensor, [b, h, s, d] tensors transposed, a shifted base, strided heads, and a lam and a dO
    # that are expanded.
    g = torch.Generator().manual_seed(2)
    b, s, h, d = 2, 70, 4, 64
    packed = torch.randn(b, s, 3, h, d, generator=g).half().to(device)
    q, k, v = packed.unbind(2)
    lam = torch.rand(h, generator=g).to(device).expand(b, s, h)
    do = torch.randn(b, h, s, d, generator=g).half().to(device).transpose(1, 2)
    _check(q, k, v, lam, do, True)
    qt, kt, vt = (torch.randn(b, h, s, d, generator=g).half().to(device).transpose(1, 2) for _ in range(3))
    _check(qt, kt, vt, torch.rand(h, s, b, generator=g).to(device).permute(2, 1, 0), do, False)
    base = torch.randn(b * s * h * d + 1, generator=g).half().to(device)[1:].view(b, s, h, d)  # not 16-byte aligned
    _check(base, kt, vt, lam, do, True)
    wide = torch.randn(b, s, 2 * h, d + 8, generator=g).half().to(device)[:, :, ::2, :d]
    _check(wide, kt, vt, lam, do, True)
    leaves = [x.detach().requires_grad_() for x in (q, k, v, lam[0, 0])]
    fai.flash_diff_attn_func(*leaves, causal=True).sum().backward()
    want = diff_attention(q, k, v, lam[0, 0], None, True, torch.ones_like(q))
    for name, x in zip(("dq", "dk", "dv", "dlam"), leaves):
        assert_within(name, x.grad, want[name])


def test_rows_far_apart(device):
    # Rows 2^23 + 64 elements apart, past the tiles' 32-bit offsets, are copied; 2^23 apart they are read in place.
    q, k, v, lam, do = _inputs(device, 1, 70, 70, 2, 2, 64, "head", torch.float16, 10)
    want = _check(q, k, v, lam, do, True)
    for far in ((1 << 23) + 64, 1 << 23):
        pool = torch.zeros(70 * far, dtype=torch.float16, device=device)
        x = pool.as_strided(q.shape, (0, far, 64, 1))
        for i in range(3):
            x.copy_((q, k, v)[i])
            leaves = [y.detach().requires_grad_() for y in (q, k, v)]
            leaves[i] = x.detach().requires_grad_()
            out = fai.flash_diff_attn_func(*leaves, lam, causal=True)
            assert torch.equal(out, want["out"])
            for name, y in zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, do)):
                assert torch.equal(y, want[name])
        x.copy_(do)
        leaves = [y.detach().requires_grad_() for y in (q, k, v)]
        out = fai.flash_diff_attn_func(*leaves, lam, causal=True)
        for name, y in zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, x)):
            assert torch.equal(y, want[name])


def test_broadcast_lam_gets_its_summed_gradient(device):
    q, k, v, _, do = _inputs(device, 2, 40, 40, 4, 2, 64, "layer", torch.float16, 9)
    lam = torch.tensor([0.3, 0.5, 0.7, 0.9], device=device).requires_grad_()
    out = fai.flash_diff_attn_func(q, k, v, lam.expand(2, 40, 4))
    want = diff_attention(q, k, v, lam.detach(), None, False, do)
    assert_within("dlam", torch.autograd.grad(out, lam, do)[0], want["dlam"])


def test_a_batch_past_the_grids_second_dimension(device):
    # 65536 sequences and more, a lam for each row, the last sequences checked.
    b = 65540
    q, k, v, lam, do = _inputs(device, b, 2, 3, 1, 1, 64, "token", torch.float16, 29)
    leaves = [x.requires_grad_() for x in (q, k, v, lam)]
    out = fai.flash_diff_attn_func(*leaves, causal=True)
    grads = torch.autograd.grad(out, leaves, do)
    tail = slice(b - 8, b)
    want = diff_attention(q[tail], k[tail], v[tail], lam[tail], None, True, do[tail])
    for name, x in zip(("out", "dq", "dk", "dv", "dlam"), (out, *grads)):
        assert_within(name, x[tail], want[name])


def test_no_rows_and_no_keys(device):
    for b, sq, sk in ((0, 4, 4), (2, 0, 4), (2, 4, 0)):
        q, k, v, lam, do = _inputs(device, b, sq, sk, 2, 1, 64, "head", torch.float16, 1)
        leaves = [x.requires_grad_() for x in (q, k, v, lam)]
        out = fai.flash_diff_attn_func(*leaves, causal=True)
        assert out.shape == q.shape and not out.any()
        for x, gx in zip(leaves, torch.autograd.grad(out, leaves, do)):
            assert gx.shape == x.shape and not gx.any()


def test_hidden_keys_reach_nothing(device):
    # Infinities and NaN behind the last sequence and in other sequences' rows of a packed batch stay there.
    lens = [5, 0, 70, 1]
    cu = cu_from_lengths(lens)
    g = torch.Generator().manual_seed(3)
    total, h, d = int(cu[-1]) + 40, 2, 64
    mk = lambda: torch.randn(total, h, d, generator=g).half().to(device)  # noqa: E731
    q, k, v, do = mk(), mk(), mk(), mk()
    clean = [x.clone() for x in (q, k, v, do)]
    for x in (q, k, v, do):
        x[int(cu[-1]):] = float("nan")
        x[int(cu[-1]) + 3] = float("inf")
    lam = torch.rand(total, h, generator=g).to(device)

    def grads(q, k, v, do):
        leaves = [x.detach().requires_grad_() for x in (q, k, v, lam)]
        out = fai.flash_diff_attn_varlen_func(*leaves, cu.to(device), cu.to(device), 70, 70, causal=True)
        return [out, *torch.autograd.grad(out, leaves, do)]

    for a, b in zip(grads(q, k, v, do), grads(*clean)):
        assert torch.equal(a, b) and not a[int(cu[-1]):].any()


@pytest.mark.parametrize("h,hk,d,causal,kind,dtype", [
    (4, 2, 64, True, "token", torch.float16),
    (8, 2, 128, True, "head", torch.bfloat16),
    (3, 1, 128, False, "layer", torch.float16),
])
def test_varlen(device, h, hk, d, causal, kind, dtype):
    """Sequences of no, one and many tokens, with gaps before, between (a maximum below a length) and behind them."""
    lens_q, lens_k = [1, 64, 0, 200, 33, 7], [1, 64, 5, 130, 190, 0]
    shift = 3
    cu_q, cu_k = cu_from_lengths(lens_q) + shift, cu_from_lengths(lens_k) + shift
    g = torch.Generator().manual_seed(7)
    tq, tk = int(cu_q[-1]) + 4, int(cu_k[-1]) + 4
    mk = lambda *s: torch.randn(*s, generator=g).to(dtype).to(device)  # noqa: E731
    q, k, v, do = mk(tq, h, d), mk(tk, hk, d), mk(tk, hk, d), mk(tq, h, d)
    shape = {"layer": (), "head": (h,), "token": (tq, h)}[kind]
    lam = torch.rand(shape, generator=g).to(device)
    leaves = [x.requires_grad_() for x in (q, k, v, lam)]
    out = fai.flash_diff_attn_varlen_func(*leaves, cu_q.to(device), cu_k.to(device), 200, 190, causal=causal)
    got = dict(zip(("out", "dq", "dk", "dv", "dlam"), (out, *torch.autograd.grad(out, leaves, do))))
    sums = None
    seen_q, seen_k = torch.zeros(tq, dtype=torch.bool), torch.zeros(tk, dtype=torch.bool)
    for i in range(len(lens_q)):
        a, b = slice(int(cu_q[i]), int(cu_q[i + 1])), slice(int(cu_k[i]), int(cu_k[i + 1]))
        seen_q[a], seen_k[b] = True, True
        want = diff_attention(q[a][None].detach(), k[b][None].detach(), v[b][None].detach(),
                              lam.detach()[a][None] if kind == "token" else lam.detach(), None, causal, do[a][None])
        for name, at in (("out", a), ("dq", a), ("dk", b), ("dv", b)):
            assert_within(f"{name} {i}", got[name][at][None], want[name])
        if kind == "token":
            assert_within(f"dlam {i}", got["dlam"][a][None], want["dlam"])
        else:
            sums = want["dlam"] if sums is None else (sums[0] + want["dlam"][0], sums[1] + want["dlam"][1])
    if kind != "token":
        assert_within("dlam", got["dlam"], sums)
    for name, seen in (("out", seen_q), ("dq", seen_q), ("dk", seen_k), ("dv", seen_k)):
        assert not got[name][~seen].any(), name
    if kind == "token":
        assert not got["dlam"][~seen_q].any()


def test_varlen_rows_past_the_maximum_are_zero(device):
    g = torch.Generator().manual_seed(1)
    mk = lambda: torch.randn(60, 2, 64, generator=g).half().to(device)  # noqa: E731
    q, k, v, do = mk(), mk(), mk(), mk()
    lam = torch.rand(60, 2, generator=g).to(device)
    cu = torch.tensor([0, 60], dtype=torch.int32, device=device)
    leaves = [x.requires_grad_() for x in (q, k, v, lam)]
    out = fai.flash_diff_attn_varlen_func(*leaves, cu, cu, 40, 60)
    dq, _, _, dlam = torch.autograd.grad(out, leaves, do)
    assert out[:40].any() and not out[40:].any() and not dq[40:].any() and not dlam[40:].any()


def test_repeats_are_the_same_bits(device):
    q, k, v, lam, do = _inputs(device, 1, 700, 700, 8, 2, 128, "layer", torch.bfloat16, 4)
    leaves = [x.requires_grad_() for x in (q, k, v, lam)]
    runs = []
    for _ in range(3):
        out = fai.flash_diff_attn_func(*leaves, causal=True)
        runs.append([out, *torch.autograd.grad(out, leaves, do)])
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_another_stream(device):
    q, k, v, lam, do = _inputs(device, 2, 300, 300, 8, 2, 64, "head", torch.float16, 12)
    leaves = [x.requires_grad_() for x in (q, k, v, lam)]
    want = fai.flash_diff_attn_func(*leaves, causal=True)
    grads = torch.autograd.grad(want, leaves, do)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = fai.flash_diff_attn_func(*leaves, causal=True)
        again = torch.autograd.grad(out, leaves, do)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(again, grads))


@pytest.mark.parametrize("kind", ["layer", "head", "token"])
def test_captured_training_step(device, kind):
    """Forward and backward in one graph, replayed on new inputs with eager work between."""
    import flash_attn_turing as ext

    q, k, v, lam, do = _inputs(device, 1, 200, 200, 8, 2, 64, kind, torch.float16, 21)

    def step():
        out, o2, lse = ext.diff_fwd(q, k, v, lam, 0.2, True, True)
        return [out, *ext.diff_bwd(q, k, v, lam, out, o2, lse, do, 0.2, True, True)]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (22, 23, 24):
        for x, y in zip((q, k, v, lam, do), _inputs(device, 1, 200, 200, 8, 2, 64, kind, torch.float16, seed)):
            x.copy_(y)
        graph.replay()
        got = [x.clone() for x in captured]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_captured_autograd_step(device):
    """The public function's forward and backward in one graph, with an eager step of the same leaves before (its graph
    gone), eager work between the replays and an eager step after."""
    g = torch.Generator().manual_seed(31)
    q, k, v, lam, do = _inputs(device, 2, 150, 150, 8, 2, 64, "head", torch.bfloat16, 31)
    leaves = [x.requires_grad_() for x in (q, k, v, lam)]

    def step():
        out = fai.flash_diff_attn_func(*leaves, causal=True)
        return [out.detach(), *torch.autograd.grad(out, leaves, do)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for turn in range(3):
        with torch.no_grad():
            for x in (*leaves, do):
                x.copy_(torch.randn(x.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        for a, b in zip(captured, eager):
            assert torch.equal(a, b), turn


def test_two_at_once(device):
    """Steps on two streams at once, eager and as two graphs, give the bits that each gives alone (small grids, whose
    key blocks several workgroups share through workspaces)."""
    sets = [_inputs(device, 1, 400, 400, 8, 2, 128, kind, torch.bfloat16, seed) for kind, seed in (("layer", 41), ("token", 42))]

    def step(q, k, v, lam, do):
        leaves = [x.detach().requires_grad_() for x in (q, k, v, lam)]
        out = fai.flash_diff_attn_func(*leaves, causal=True)
        return [out.detach(), *torch.autograd.grad(out, leaves, do)]

    alone = [step(*x) for x in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(*sets[i]))
    torch.cuda.synchronize()
    graphs, captured = [], []
    for i, s in enumerate(streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            captured.append(step(*sets[i]))
        graphs.append(g)
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            for one in (*got[i], captured[i]):
                for a, b in zip(one, alone[i]):
                    assert torch.equal(a, b)


def test_refusals(device):
    q, k, v, lam, _ = _inputs(device, 2, 8, 8, 4, 2, 64, "head", torch.float16, 1)
    f = fai.flash_diff_attn_func
    with pytest.raises(RuntimeError, match="k must have the dtype of q"):
        f(q, k.bfloat16(), v, lam)
    with pytest.raises(RuntimeError, match="k and v must have the same shape"):
        f(q, k, v[:, :4], lam)
    with pytest.raises(RuntimeError, match="num_heads_q must be divisible"):
        f(q[:, :, :3], k, v, lam[:3])
    with pytest.raises(RuntimeError, match="lam must be a scalar tensor"):
        f(q, k, v, lam[:3])
    with pytest.raises(RuntimeError, match="lam must be a scalar tensor"):
        f(q, k, v, lam.expand(8, 4))
    with pytest.raises(RuntimeError, match="lam must be on the device"):
        f(q, k, v, lam.cpu())
    with pytest.raises(RuntimeError, match="k must be on the device"):
        f(q, k.cpu(), v.cpu(), lam)
    cu = torch.tensor([0, 8], dtype=torch.int32, device=device)
    g = fai.flash_diff_attn_varlen_func
    with pytest.raises(RuntimeError, match="cu_seqlens_q must be on the device"):
        g(q[0], k[0], v[0], lam, cu.cpu(), cu, 8, 8)
    with pytest.raises(RuntimeError, match="batch_size \\+ 1"):
        g(q[0], k[0], v[0], lam, cu, torch.cat((cu, cu[-1:])), 8, 8)
    with pytest.raises(RuntimeError, match="int32"):
        g(q[0], k[0], v[0], lam, cu.long(), cu, 8, 8)
