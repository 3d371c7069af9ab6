"""CPU: further calls of the packed-token C entries that come back as a code, before a launch."""
import math


def test_scales_that_pass_fp32_in_bits_and_missing_pointers():
    from casmtr_amd import _lib
    l, bad, p = _lib.lib(), _lib.ERR_UNSUPPORTED, 4096   # p: never read
    attn = lambda scale: l.casmtr_packed_attn_fwd(p, p, p, p, None, p, p, p, None, 8, 8, 1, 4, 2, 64, 256, 64, 128, 64, 128, 64, scale, 0, 2, None)
    # scores are held in bits: scale log2(e) has to be a number too
    assert attn(3e38) == bad and attn(2.4e38) == bad and attn(math.inf) == bad
    bwd = lambda scale=0.1, lse=p: l.casmtr_packed_attn_bwd(p, p, p, p, p, lse, p, p, p, p, p, p, None, 8, 8, 1, 4, 2, 64, 256, 64, 128, 64, 128, 64, scale, 0, 2, None)
    assert bwd(scale=3e38) == bad and bwd(lse=None) == bad
    norm = lambda rstd=p, ws=p: l.casmtr_rms_norm_bwd(p, None, p, p, rstd, p, p, ws, 4, 64, 64, 64, 64, 2, 2, None)
    assert norm(rstd=None) == bad and norm(ws=None) == bad
