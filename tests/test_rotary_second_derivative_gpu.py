"""Rotary positions inside a gradient that is differentiated again (a gradient penalty): the rotation is linear, its
gradient the rotation back, and so is that one's."""

import pytest
import torch

import flash_attention_interface as fai
from oracle.rotary import rotate

pytestmark = pytest.mark.gpu


def _make(device, dtype, packed, dim=64, rotary=32):
    g = torch.Generator().manual_seed(4)
    lead, at = ((9,), [0, 1, 2, 3, 0, 1, 2, 3, 4]) if packed else ((2, 5), [3, 4, 5, 6, 7] * 2)
    mk = lambda h: torch.randn(*lead, h, dim, generator=g).to(dtype)  # noqa: E731
    cos, sin = (torch.randn(8, rotary // 2, generator=g) for _ in range(2))
    more = dict(cu_seqlens=torch.tensor([0, 4, 9], dtype=torch.int32, device=device)) if packed else dict(seqlen_offsets=3)
    return mk(4), mk(2), mk(4), mk(2), cos, sin, at, more


def _within(got, want, bound):
    assert float(((got.double().cpu() - want).abs() - bound).max()) <= 0


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_gradients_of_gradients(device, dtype, packed, interleaved):
    q, k, u, w, cos, sin, at, more = _make(device, dtype, packed)
    qd, kd = (x.to(device).requires_grad_() for x in (q, k))
    ud, wd = (x.to(device).requires_grad_() for x in (u, w))  # gradients of the outputs
    out = fai.flash_attn_rotary_func(qd, kd, cos.to(device), sin.to(device), interleaved, **more)
    grads = torch.autograd.grad(out, (qd, kd), (ud, wd), create_graph=True)
    for name, x, y in (("dq", u, grads[0]), ("dk", w, grads[1])):
        assert y.requires_grad, name
        _within(y.detach().flatten(0, -3), *rotate(x.flatten(0, -3), cos, sin, at, interleaved, inverse=True))
    # d <dq, a> / d u: a rotated forward; the same of k, and of either alone.
    again = torch.autograd.grad(grads, (ud, wd), (qd.detach(), kd.detach()), retain_graph=True, create_graph=True)
    for x, y in ((q, again[0]), (k, again[1])):
        _within(y.detach().flatten(0, -3), *rotate(x.flatten(0, -3), cos, sin, at, interleaved))
    for i, x in ((0, q), (1, k)):
        one = torch.autograd.grad(grads[i], (ud, wd)[i], x.to(device), retain_graph=True)[0]
        assert torch.equal(one, again[i])


def test_a_gradient_penalty(device):
    """The gradient of |d loss / d q|^2 where the loss is not linear in what is rotated, against differences in 64 bits."""
    q, _, _, _, cos, sin, at, more = _make(device, torch.float16, False)
    q = q / 4

    def penalty(x, rot):
        y = rot(x)
        g = torch.autograd.grad((y ** 3).sum(), x, create_graph=True)[0]
        return (g ** 2).sum()

    def rot64(x):
        half = cos.shape[1]
        c, s = (t[torch.tensor(at).view(2, 5)][:, :, None].double() for t in (cos, sin))
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        return torch.cat((torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2), x[..., 2 * half:]), -1)

    x = q.double().requires_grad_()
    want = torch.autograd.grad(penalty(x, rot64), x)[0]
    xd = q.to(device).requires_grad_()
    got = torch.autograd.grad(
        penalty(xd, lambda t: fai.flash_attn_rotary_func(t, None, cos.to(device), sin.to(device), True, **more)), xd)[0]
    # Eight roundings to fp16 on the way (2^-11 each: y, its powers, the products with g, three rotations), of two terms that
    # may each be twice what remains: 8 * 2 * 2 * 2^-11 = 2^-6.
    size = want.abs().max()
    assert (got.double().cpu() - want).abs().max() <= 2.0 ** -6 * size
    i = (1, 2, 3, 5)  # and the 64-bit gradient against a difference
    e = torch.zeros_like(x)
    e[i] = 1e-4
    with torch.enable_grad():
        up, down = (float(penalty((q.double() + z * e).requires_grad_(), rot64)) for z in (1, -1))
    assert abs((up - down) / 2e-4 - float(want[i])) <= 1e-4 * float(size)


def test_no_graph_is_made_without_create_graph(device):
    q, k, u, w, cos, sin, at, more = _make(device, torch.float16, False)
    qd, kd = (x.to(device).requires_grad_() for x in (q, k))
    out = fai.flash_attn_rotary_func(qd, kd, cos.to(device), sin.to(device), **more)
    dq, dk = torch.autograd.grad(out, (qd, kd), (u.to(device), w.to(device)))
    assert not dq.requires_grad and not dk.requires_grad
