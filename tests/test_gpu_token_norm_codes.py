"""The 8-bit codes of the norm are round(y / scale) to the last one: y is made exact (rows of +-1 and eps = 0 give rstd = 1, y = +-weight), the
weights lie on and next to the borders between two codes, and scales are 3, 5, 7, ... times a power of two, whose reciprocals are not."""
import pytest
import torch

pytestmark = pytest.mark.gpu
TOP = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0, torch.int8: 127.0}


def _borders(q8):
    if q8 == torch.int8:
        return torch.arange(127) + 0.5
    codes = torch.arange(128, dtype=torch.uint8).view(q8).float()
    codes = codes[codes.isfinite()].sort().values
    return (codes[1:] + codes[:-1]) / 2


@pytest.mark.parametrize("q8", list(TOP))
@pytest.mark.parametrize("group", [None, 128])
@pytest.mark.parametrize("C", [1024, 8192])
def test_codes(C, group, q8):
    from casmtr_amd import ops
    b = _borders(q8)
    for odd in (1, 3, 5, 7, 11, 13, 41, 79, 127):
        s = odd * 2.0 ** -7
        y = torch.cat([b, b, b])[:C - 1] * s                        # exact: at most 8 + 7 bits
        y[len(b):2 * len(b)] = torch.nextafter(y[len(b):2 * len(b)], torch.tensor(0.0))
        y[2 * len(b):] = torch.nextafter(y[2 * len(b):], torch.tensor(1e9))
        y = y.repeat(-(-C // len(y)))[:C]
        y = y[torch.randperm(C, generator=torch.Generator().manual_seed(odd))].clamp(max=TOP[q8] * s)
        y[::128] = TOP[q8] * s                                      # every block's and the row's largest
        sign = torch.where(torch.arange(C) % 3 == 0, -1.0, 1.0)
        q, scale, _ = ops.rms_norm_quant(sign.expand(3, C).contiguous().cuda(), y.cuda(), 0.0, dtype=q8, group=group)
        assert (scale == s).all()
        want = (sign * y / s).clamp(-TOP[q8], TOP[q8])              # one correctly rounded division
        want = want.round() if q8 == torch.int8 else want.to(q8).float()
        assert torch.equal(q.float().cpu(), want.expand(3, C))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("R,C", [(3, 64), (2, 1000), (3, 4096), (2, 16384)])
@pytest.mark.parametrize("size", [1e20, 1e30, 1e38])
def test_rows_whose_squares_pass_fp32(size, R, C, dt):
    """The norm of large rows: their squares do not fit fp32, the result does.  rstd may be subnormal (a row of 1e38: 1e-38 and less, of steps of
    2^-149): 2^-22 of itself, beside the 32 u that the sums, the root and the products are off by.  Ordinary rows beside them keep their bits."""
    from casmtr_amd import ops
    u = 2.0 ** -24
    g = torch.Generator().manual_seed(C)
    x = torch.rand(R, C, generator=g) * 2.0 + 0.5
    x = torch.where(torch.rand(R, C, generator=g) < 0.5, -x, x).to(dt).cuda()
    w = (1 + 0.3 * torch.randn(C, generator=g)).cuda()
    big = x.clone()
    big[0] = (x[0].double() * size).to(dt)
    y, _, rstd = ops.rms_norm(big, w, 1e-5, want_rstd=True)
    h = big[0].double()
    ref = h / (h.square().mean() + 1e-5).sqrt() * w.double()
    assert ((y[0].double() - ref).abs() <= (torch.finfo(dt).eps / 2 + 32 * u + 2.0 ** -21) * ref.abs()).all()
    assert torch.equal(y[1:], ops.rms_norm(x, w, 1e-5)[0][1:])
    dy = torch.randn(R, C, generator=g).to(dt).cuda()
    dx, dw = ops.rms_norm_bwd(dy, big, w, rstd)
    n = big.double() / (big.double().square().mean(1, keepdim=True) + 1e-5).sqrt()
    terms = dy.double() * n
    assert ((dw.double() - terms.sum(0)).abs() <= (140 * u + 2.0 ** -21) * terms.abs().sum(0) + u * terms.sum(0).abs()).all()
    assert (dx[0].double().abs() * size <= 40.0).all() and dx.isfinite().all()
