"""Rotary positions (casmtr_rotary_fwd) against complex multiplication in 64 bits.

Tolerance: half a step of the output's type, and per component 2^-20 gain (|a| + |b|): the angle's remainder is rounded to fp32 (2^-25
turns = 1.9e-7 rad), sine and cosine are good to 2 steps of fp32, and three roundings follow -- below 6e-7 together."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
half = lambda t: torch.finfo(t).eps / 2
sub = lambda t: torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def _pairs(x, n, layout):
    x = x.double()[..., :2 * n]
    return (x[..., :n], x[..., n:]) if layout == "half" else (x[..., 0::2], x[..., 1::2])


def _check(x, y, pos, freq, layout, gain, sign=1):
    n, T = freq.numel(), x.shape[0]
    axis = torch.arange(n, device="cuda") * (pos.dim()) // n if pos.dim() == 2 else torch.zeros(n, dtype=torch.long, device="cuda")
    t = sign * (pos.double().view(T, -1)[:, axis] * freq)[:, None]
    (a, b), (u, v) = _pairs(x, n, layout), _pairs(y, n, layout)
    tol = 2.0 ** -20 * gain * (a.abs() + b.abs()) + sub(x.dtype)
    for got, ref in ((u, gain * (a * t.cos() - b * t.sin())), (v, gain * (b * t.cos() + a * t.sin()))):
        assert ((got - ref).abs() <= tol + half(x.dtype) * ref.abs()).all()
    assert torch.equal(x[..., 2 * n:], y[..., 2 * n:])


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("T,Hq,Hk,D,rot", [(1, 1, 1, 2, 2), (1, 32, 8, 128, 128), (7, 5, 1, 40, 40), (300, 4, 4, 64, 32), (2500, 2, 1, 96, 24), (33, 3, 3, 31, 14),
                                           (5, 2, 2, 50, 36), (9000, 1, 1, 16, 16), (4, 1, 2, 2048, 2048)])
def test_against_64_bits(T, Hq, Hk, D, rot, layout, dt):
    from casmtr_amd import ops
    g = torch.Generator().manual_seed(T + D)
    q, k = torch.randn(T, Hq, D, generator=g).to(dt).cuda(), torch.randn(T, Hk, D, generator=g).to(dt).cuda()
    freq, _ = ops.rotary_freqs(rot)
    for far, gain in ((50, 1.0), (4_000_000, 1.25)):
        pos = torch.randint(-far, far, (T,), generator=g).cuda()
        oq, ok = ops.rotary(q, k, pos, freq, layout, gain)
        _check(q, oq, pos, freq, layout, gain), _check(k, ok, pos, freq, layout, gain)
        o32 = ops.rotary(q, k, pos.int(), freq, layout, gain)
        assert torch.equal(o32[0], oq) and torch.equal(o32[1], ok)
        only, none = ops.rotary(q, None, pos, freq, layout, gain, inverse=True)
        assert none is None
        _check(q, only, pos, freq, layout, gain, sign=-1)
    if rot % 4 == 0:
        pos = torch.randint(0, 300, (T, 2), generator=g).cuda()
        f2, _ = ops.rotary_freqs(rot, axes=2)
        oq, ok = ops.rotary(q, k, pos, f2, layout)
        _check(q, oq, pos, f2, layout, 1.0), _check(k, ok, pos, f2, layout, 1.0)


@pytest.mark.parametrize("dt", TYPES)
def test_views(dt):
    """column ranges of a fused projection, a stride of zero, a view that starts at an odd element"""
    from casmtr_amd import ops
    qkv = torch.randn(70, 12 * 24 + 1, device="cuda").to(dt)[:, 1:].unflatten(1, (12, 24))
    freq, _ = ops.rotary_freqs(20)
    pos = torch.arange(70, device="cuda")
    a = ops.rotary(qkv[:, :8], qkv[:, 8:10], pos, freq)
    b = ops.rotary(qkv[:, :8].contiguous(), qkv[:, 8:10].contiguous(), pos, freq)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    one = qkv[:1, :8].expand(70, 8, 24)
    assert torch.equal(ops.rotary(one, None, pos, freq)[0], ops.rotary(one.contiguous(), None, pos, freq)[0])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_gradient(layout):
    """against the formula (the transpose of the turn) and against differences, which are exact for a linear map up to rounding"""
    from casmtr_amd import ops
    from casmtr_amd.functions.rotary import rotary_op
    q, k = torch.randn(40, 4, 48, device="cuda", requires_grad=True), torch.randn(40, 2, 48, device="cuda", requires_grad=True)
    freq, _ = ops.rotary_freqs(32)
    pos = torch.randint(0, 1000, (40,), device="cuda")
    oq, ok = rotary_op(q, k, pos, freq, layout, 1.1)
    gq, gk = torch.randn_like(oq), torch.randn_like(ok)
    dq, dk = torch.autograd.grad((oq, ok), (q, k), (gq, gk))
    _check(gq, dq, pos, freq, layout, 1.1, sign=-1), _check(gk, dk, pos, freq, layout, 1.1, sign=-1)
    v = torch.randn_like(q)
    up, down = ops.rotary(q.detach() + v, None, pos, freq, layout, 1.1)[0], ops.rotary(q.detach() - v, None, pos, freq, layout, 1.1)[0]
    diff = ((up - down).double() / 2 * gq.double()).sum()
    got = (dq.double() * v.double()).sum()
    assert abs(diff - got) <= 2.0 ** -19 * 1.1 * 2 * (gq.abs().double().sum() * (v.abs().max() + q.abs().max()))
    only = rotary_op(q, None, pos, freq, layout, 1.1)[0]
    assert torch.equal(torch.autograd.grad(only, q, gq)[0], dq)


def test_empty_and_refusals():
    from casmtr_amd import ops
    freq, _ = ops.rotary_freqs(16)
    q, pos = torch.randn(6, 2, 16, device="cuda"), torch.arange(6, device="cuda")
    assert ops.rotary(q[:0], q[:0], pos[:0], freq)[0].shape == (0, 2, 16)
    for bad in (lambda: ops.rotary(q, q, pos, freq, "pairs"), lambda: ops.rotary(q, q[:5], pos, freq), lambda: ops.rotary(q, q.half(), pos, freq),
                lambda: ops.rotary(q, q, pos[:5], freq), lambda: ops.rotary(q, q, pos.float(), freq), lambda: ops.rotary(q, q, pos, freq.float()),
                lambda: ops.rotary(q, q, pos, torch.cat([freq, freq])), lambda: ops.rotary(q, q, pos.cpu(), freq), lambda: ops.rotary(q.cpu(), None, pos, freq),
                lambda: ops.rotary(q, q, torch.stack([pos, pos], 1), freq[:3]), lambda: ops.rotary(q[0], None, pos, freq),
                lambda: ops.rotary(q.transpose(1, 2), None, pos, freq), lambda: ops.rotary(q, q, pos, freq[:0])):
        with pytest.raises(RuntimeError):
            bad()
