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
