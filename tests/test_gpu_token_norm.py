"""RMS norm with residual / 8-bit output and its gradient (casmtr_rms_norm_fwd / _bwd) against the formulas in 64 bits.

Tolerances.  u = 2^-24 is half a step of fp32, half(T) half a step of the output's type.  The sum of squares adds at most 8 * 4 + 6 + 16 terms in a
row (a thread's columns, the wave, the waves): relative error <= 54 u, halved by the square root; division, square root and the two
products add 4 roundings: 32 u.  Outputs below the normal range are off by half a subnormal step.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]
half = lambda t: torch.finfo(t).eps / 2
sub = lambda t: torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2   # half a subnormal step
TOP = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0, torch.int8: 127.0}
SHAPES = [(1, 1), (3, 7), (5, 8), (2, 64), (9, 127), (7, 512), (4, 513), (3, 1000), (5, 1024), (2, 1025), (3, 2048), (2, 4095), (2, 5000), (3, 8192), (2, 8200), (2, 16384), (1030, 96)]


def _data(R, C, dt, seed=0, residual=True):
    g = torch.Generator().manual_seed(seed)
    x, r, w = torch.randn(R, C, generator=g), 3 * torch.randn(R, C, generator=g), 1 + 0.3 * torch.randn(C, generator=g)
    return x.to(dt).cuda(), r.to(dt).cuda() if residual else None, w.to(dt).cuda()


def _stream(x, r):
    return x if r is None else (x.float() + r.float()).to(x.dtype)


def _ref(h, w, eps):
    h = h.double()
    return h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps) * w.double()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("R,C", SHAPES)
def test_forward(R, C, dt):
    from casmtr_amd import ops
    for residual in (False, True):
        x, r, w = _data(R, C, dt, R + C, residual)
        y, h = ops.rms_norm(x, w, 1e-5, residual=r)
        ref = _ref(_stream(x, r), w, 1e-5)
        assert (h is None) == (r is None) and (r is None or torch.equal(h, _stream(x, r)))
        assert ((y.double() - ref).abs() <= ref.abs() * (half(dt) + 32 * U) + sub(dt)).all()
        y32, _ = ops.rms_norm(x, w.float(), 1e-5, residual=r)   # an fp32 weight with the same values: the same result
        assert torch.equal(y32, y)


@pytest.mark.parametrize("dt", TYPES)
def test_views(dt):
    """rows of a wider matrix, starting at any element"""
    from casmtr_amd import ops
    wide = torch.randn(33, 777, device="cuda").to(dt)
    for at, C in ((0, 700), (1, 701), (3, 512), (5, 60)):
        x, r = wide[:, at:at + C], wide[:, 777 - C:]
        w = torch.randn(C + 1, device="cuda").to(dt)[1:]
        y, h = ops.rms_norm(x, w, residual=r)
        yc, hc = ops.rms_norm(x.contiguous(), w.clone(), residual=r.contiguous())
        assert torch.equal(y, yc) and torch.equal(h, hc)
    x3 = wide[:32, :700].view(4, 8, 700)
    assert torch.equal(ops.rms_norm(x3, w.new_ones(700))[0].view(32, 700), ops.rms_norm(wide[:32, :700], w.new_ones(700))[0])


@pytest.mark.parametrize("q8", list(TOP))
@pytest.mark.parametrize("group", [None, 128])
@pytest.mark.parametrize("R,C", [(1, 128), (5, 384), (4, 1024), (3, 2176), (2, 8192), (2, 16384), (3, 1000), (2, 77)])
def test_quant(R, C, group, q8):
    """|q scale - y| is at most half a step of the 8-bit type: 2^-4 (e4m3), 2^-3 (e5m2) of the value, half of the subnormal step 2^-9 / 2^-16
    (int8: of the step 1) of the scale; y itself is off by 32 u, the scale's and the quotient's roundings add 3 u."""
    from casmtr_amd import ops
    if group and C % group:
        pytest.skip("blocks of 128 columns")
    for dt in TYPES:
        x, r, w = _data(R, C, dt, C)
        x[0] = 0
        if R > 1:
            r[0] = 0   # a row of zeros
        q, scale, h = ops.rms_norm_quant(x, w, 1e-5, residual=r, dtype=q8, group=group)
        ref = _ref(_stream(x, r), w, 1e-5).view(R, -1, group or C)
        want = (ref.abs().amax(-1, keepdim=True) / TOP[q8]).clamp(min=2.0 ** -126)
        s = scale.double().view_as(want)
        assert torch.equal(h, _stream(x, r)) and ((s - want).abs() <= want * 40 * U).all()
        rel, floor = {torch.float8_e4m3fn: (2.0 ** -4, 2.0 ** -10), torch.float8_e5m2: (2.0 ** -3, 2.0 ** -17), torch.int8: (0.0, 0.5)}[q8]
        err = (q.float().double().view_as(ref) * s - ref).abs()
        assert (err <= torch.maximum(rel * ref.abs(), floor * s) * (1 + 2.0 ** -10) + ref.abs() * 40 * U).all()


def test_not_finite():
    """infinities and NaN stay in their row (and reach its scale); the other rows are what they are without them"""
    from casmtr_amd import ops
    x, _, w = _data(4, 640, torch.bfloat16, residual=False)
    clean = ops.rms_norm(x, w)[0]
    x[1, 5], x[2, 600] = math.inf, math.nan
    y = ops.rms_norm(x, w)[0]
    assert torch.equal(y[[0, 3]], clean[[0, 3]]) and y[2].isnan().all() and y[1, 5].isnan() and (y[1, :5] == 0).all()
    q, s, _ = ops.rms_norm_quant(x, w)
    assert s[[0, 3]].isfinite().all() and s[1:3].isnan().all()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("R,C", SHAPES)
def test_backward(R, C, dt):
    """dx sums C signed products: |error of mean(g n)| <= 64 u mean|g n|; dw adds a part's rows (R / 512 or one), 32 lanes of parts / 32 each and
    the lanes: (R / 512 + 100) u of the sum of the magnitudes.  n carries rstd's 32 u."""
    from casmtr_amd import ops
    x, r, w = _data(R, C, dt, R * C)
    dy, dh = torch.randn(R, C, device="cuda").to(dt), torch.randn(R, C, device="cuda").to(dt)
    for tail in (None, dh):
        y, h, rstd = ops.rms_norm(x, w, 1e-5, residual=r, want_rstd=True)
        dx, dw = ops.rms_norm_bwd(dy, h, w, rstd, dh=tail)
        rs = 1 / torch.sqrt(h.double().square().mean(-1, keepdim=True) + 1e-5)
        n, g = h.double() * rs, dy.double() * w.double()
        c = (g * n).mean(-1, keepdim=True)
        ref = (g - n * c) * rs + (0 if tail is None else tail.double())
        mag = (g.abs() + 2 * n.abs() * (g * n).abs().mean(-1, keepdim=True)) * rs
        assert ((dx.double() - ref).abs() <= half(dt) * ref.abs() + 140 * U * mag + 2 * U * ref.abs() + sub(dt)).all()
        terms = dy.double() * n
        assert ((dw.double() - terms.sum(0)).abs() <= half(dt) * terms.sum(0).abs() + (R / 512 + 140) * U * terms.abs().sum(0) + sub(dt)).all()
        again = ops.rms_norm_bwd(dy, h, w, rstd, dh=tail)
        assert torch.equal(again[0], dx) and torch.equal(again[1], dw)


def test_gradient_against_differences():
    """directional derivatives of sum(dy y + dh h) from central differences in 64 bits; the kernel's fp32 gradients are within 140 u of the
    magnitudes that they sum"""
    from casmtr_amd.functions.rms_norm import rms_norm_op
    x, r, w = (t.requires_grad_() for t in _data(6, 300, torch.float32, 5))
    dy, dh = torch.randn(6, 300, device="cuda"), torch.randn(6, 300, device="cuda")
    y, h = rms_norm_op(x, w, 1e-5, r)
    grads = torch.autograd.grad((y, h), (x, w, r), (dy, dh))
    dirs = [torch.randn_like(t).double() for t in (x, w, r)]

    def loss(e):
        xx, ww, rr = (t.detach().double() + e * d for t, d in zip((x, w, r), dirs))
        return (dy.double() * _ref(xx + rr, ww, 1e-5) + dh.double() * (xx + rr)).sum()

    diff = (loss(1e-5) - loss(-1e-5)) / 2e-5
    got = sum((g.double() * d).sum() for g, d in zip(grads, dirs))
    mag = sum((g.double() * d).abs().sum() for g, d in zip(grads, dirs))
    assert abs(got - diff) <= 2e-5 * mag


def test_function_paths():
    from casmtr_amd import ops
    from casmtr_amd.functions.rms_norm import rms_norm_op
    x, r, w = (t.requires_grad_() for t in _data(5, 96, torch.float32))
    y, h = rms_norm_op(x, w, 1e-6, r)
    dh = torch.randn_like(h)
    gx, gr = torch.autograd.grad(h, (x, r), dh)                          # the stream alone
    assert torch.equal(gx, dh) and torch.equal(gr, dh)
    y, h = rms_norm_op(x, w, 1e-6, r)
    y.sum().backward()                                                    # the norm alone; y.sum()'s gradient is a broadcast view
    n = h.detach()
    dx, dw = ops.rms_norm_bwd(torch.ones_like(n), n, w.detach(), ops.rms_norm(n, w.detach(), 1e-6, want_rstd=True)[2])
    assert torch.equal(x.grad, dx) and torch.equal(r.grad, dx) and torch.equal(w.grad, dw)
    assert x.grad.data_ptr() != r.grad.data_ptr()


def test_no_rows():
    from casmtr_amd import ops
    w = torch.ones(16, device="cuda")
    x = torch.empty(0, 16, device="cuda")
    y, h, rstd = ops.rms_norm(x, w, residual=x, want_rstd=True)
    assert y.shape == h.shape == (0, 16) and rstd.shape == (0,)
    dx, dw = ops.rms_norm_bwd(x, x, w, rstd)
    assert dx.shape == (0, 16) and (dw == 0).all()
    assert ops.rms_norm_quant(x, w)[1].shape == (0,)


def test_refusals():
    from casmtr_amd import ops
    x, r, w = _data(4, 256, torch.bfloat16)
    for bad in (lambda: ops.rms_norm(x.double(), w), lambda: ops.rms_norm(x, w.half()), lambda: ops.rms_norm(x, w[:255]), lambda: ops.rms_norm(x.t(), w),
                lambda: ops.rms_norm(x, w, residual=r.float()), lambda: ops.rms_norm(x, w, residual=r[:3]), lambda: ops.rms_norm(x[:, :0], w[:0]),
                lambda: ops.rms_norm(x.view(2, 2, 256).transpose(0, 1), w), lambda: ops.rms_norm(x.cpu(), w), lambda: ops.rms_norm(x, w.cpu()),
                lambda: ops.rms_norm_quant(x, w, dtype=torch.uint8), lambda: ops.rms_norm_quant(x, w, group=64),
                lambda: ops.rms_norm_quant(x[:, :200], w[:200], group=128), lambda: ops.rms_norm(x.new_zeros(1, 16385), w.new_zeros(16385)),
                lambda: ops.rms_norm_bwd(x, x, w, torch.ones(3, device="cuda")), lambda: ops.rms_norm_bwd(x[:3], x, w, torch.ones(4, device="cuda"))):
        with pytest.raises(RuntimeError):
            bad()
