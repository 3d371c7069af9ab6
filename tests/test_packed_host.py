"""CPU: what the packed-token operators refuse before anything reaches a GPU, and the frequency tables."""
import math

import pytest
import torch


def test_operators_reject_host_tensors():
    from casmtr_amd import ops
    x, w = torch.zeros(4, 32), torch.ones(32)
    q = torch.zeros(4, 2, 32)
    for call in (lambda: ops.rms_norm(x, w), lambda: ops.rms_norm_quant(x, w), lambda: ops.rms_norm_bwd(x, x, w, torch.ones(4)),
                 lambda: ops.rotary(q, q, torch.arange(4), torch.ones(8, dtype=torch.float64)),
                 lambda: ops.packed_attn(q, q, q, torch.tensor([0, 4], dtype=torch.int32))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_c_entries_refuse_sizes():
    """every refusal comes back as a code, before a launch"""
    from casmtr_amd import _lib
    l = _lib.lib()
    bad = _lib.ERR_UNSUPPORTED
    p = 4096   # never read
    norm = lambda rows=4, C=64, dtype=2, w=2, quant=0, group=0, scale=p, res=None, h=None: l.casmtr_rms_norm_fwd(
        p, res, p, p, h, None, scale, rows, C, C, C, 1e-6, dtype, w, quant, group, None)
    assert norm(rows=0) == 0
    assert norm(rows=-1) == bad and norm(C=0) == bad and norm(C=16385) == bad and norm(dtype=3, w=3) == bad and norm(w=1) == bad and norm(quant=4) == bad
    assert norm(quant=1, scale=None) == bad and norm(quant=1, group=64) == bad and norm(quant=1, group=128) == bad and norm(group=128, C=128) == bad
    assert norm(res=p) == bad and norm(rows=1 << 31) == bad
    assert l.casmtr_rms_norm_bwd(p, None, p, p, p, p, p, p, 0, 64, 64, 64, 64, 2, 2, None) == bad
    assert l.casmtr_rms_norm_bwd(p, None, p, p, p, p, p, p, 4, 16385, 64, 64, 64, 2, 2, None) == bad
    assert l.casmtr_rms_norm_bwd_ws_floats(0, 64) == 0 and l.casmtr_rms_norm_bwd_ws_floats(3, 4096) == 3 * 4096
    rot = lambda T=4, Hq=2, Hk=2, D=64, n=32, axes=1, layout=0, dtype=2: l.casmtr_rotary_fwd(p, p, p, p, p, p, T, Hq, Hk, D, n, axes, 0, layout, 1.0, 0, Hq * D, D,
                                                                                       Hk * D, D, dtype, None)
    assert rot(T=0) == 0 and rot(Hq=0, Hk=0) == 0
    assert rot(n=33) == bad and rot(n=0) == bad and rot(axes=3) == bad and rot(axes=2, n=31) == bad and rot(layout=2) == bad and rot(dtype=7) == bad
    assert rot(D=4096, n=1025) == bad and rot(Hq=1 << 20, D=64) == bad and rot(T=-1) == bad
    attn = lambda Tq=8, Tk=8, n=1, H=4, Hk=2, D=64, scale=0.1, dtype=2, ws=p: l.casmtr_packed_attn_fwd(p, p, p, p, None, ws, p, p, None, Tq, Tk, n, H, Hk, D, H * D, D,
                                                                                                   Hk * D, D, Hk * D, D, scale, 0, dtype, None)
    assert attn(Tq=0) == 0
    assert attn(Tq=-1) == bad and attn(Tk=-1) == bad and attn(n=-1) == bad and attn(H=3) == bad and attn(Hk=0) == bad and attn(D=129) == bad and attn(D=0) == bad
    assert attn(scale=0.0) == bad and attn(scale=-1.0) == bad and attn(scale=math.nan) == bad and attn(scale=math.inf) == bad and attn(dtype=3) == bad
    assert attn(Tq=1 << 31) == bad and attn(Tk=1 << 31) == bad
    assert l.casmtr_packed_attn_ws_floats(1, 1 << 20, 1, 8, 8, 128) > 0 and attn(Tq=1, Tk=1 << 20, ws=None) == bad   # split keys need the workspace
    bwd = lambda Tq=8, Tk=8, n=1, H=4, Hk=2, D=64, scale=0.1, dtype=2: l.casmtr_packed_attn_bwd(*(p,) * 12, None, Tq, Tk, n, H, Hk, D, H * D, D, Hk * D, D, Hk * D, D,
                                                                                        scale, 0, dtype, None)
    assert bwd(Tq=0, Tk=0) == 0
    assert bwd(Tq=-1) == bad and bwd(Tk=-1) == bad and bwd(n=-1) == bad and bwd(H=3) == bad and bwd(D=129) == bad and bwd(scale=0.0) == bad and bwd(dtype=3) == bad


def test_rotary_freqs():
    from casmtr_amd import ops
    f, gain = ops.rotary_freqs(8, device="cpu")
    assert f.dtype == torch.float64 and gain == 1.0
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-15)
    f2, _ = ops.rotary_freqs(8, axes=2, device="cpu")
    assert torch.allclose(f2, torch.tensor([1.0, 0.01, 1.0, 0.01], dtype=torch.float64), rtol=1e-15)
    f4, gain = ops.rotary_freqs(8, factor=4.0, device="cpu")
    assert torch.equal(f4, f / 4) and gain == 1.0
    fy, gain = ops.rotary_freqs(128, factor=8.0, trained=4096, device="cpu")
    f, _ = ops.rotary_freqs(128, device="cpu")
    turns = 4096 * f / (2 * math.pi)
    assert gain == pytest.approx(0.1 * math.log(8) + 1)
    assert torch.equal(fy[turns >= 32], f[turns >= 32]) and torch.equal(fy[turns <= 1], f[turns <= 1] / 8)
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and ((fy < f) & (fy > f / 8))[mid].all() and (fy[1:] < fy[:-1]).all()
    assert ops.rotary_freqs(128, factor=1.0, trained=4096, device="cpu")[1] == 1.0
    for bad in (dict(dim=7), dict(dim=0), dict(dim=6, axes=2), dict(dim=8, axes=3), dict(dim=8, factor=0.5), dict(dim=8, base=0), dict(dim=8, trained=0)):
        with pytest.raises(RuntimeError):
            ops.rotary_freqs(device="cpu", **bad)
