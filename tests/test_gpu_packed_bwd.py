"""Backward paths that the grid of test_gpu_packed_attn.py does not reach: keys enough that no rows are split (dk and dv stored directly),
strided operands in 16 bits, rows enough for the norm's largest number of parts.  References and bounds are those of test_gpu_packed_attn.py."""
import pytest
import torch

from test_gpu_packed_attn import TYPES, U, check, cu, half, make, reference, reference_grads, sub

pytestmark = pytest.mark.gpu


def _parts(lens, H, Hk, D, Tk):
    """parts of the rows, from the workspace's size: Tq H floats for delta, and 2 parts Tk Hk D + 3 where there are several"""
    from casmtr_amd import _lib
    Tq = sum(a for a, _ in lens) + 3
    rest = _lib.lib().casmtr_packed_attn_bwd_ws_floats(Tq, Tk, len(lens), H, Hk, D) - Tq * H
    return max(1, rest // (2 * Tk * Hk * D))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("H,Hk,D", [(8, 8, 32), (16, 8, 64), (8, 8, 128), (8, 8, 40), (16, 16, 5)])
def test_rows_in_one_part(H, Hk, D, dt):
    from casmtr_amd import ops
    lens = ([(7, 7), (25, 25), (1, 1), (3, 40), (33, 5), (0, 9), (4, 0), (2, 64)] * 17)[:130] + [(300, 300), (129, 257)]
    q, k, v, cq, ck = make(lens, H, Hk, D, dt, seed=D)
    assert _parts(lens, H, Hk, D, k.shape[0]) == 1
    g = torch.randn(q.shape, generator=torch.Generator().manual_seed(3)).to(dt).cuda()
    for causal in (False, True):
        out, lse = ops.packed_attn(q, k, v, cq, ck, causal=causal, want_lse=True)
        ref = reference(q, k, v, lens, causal, D ** -0.5)
        check(out, lse, ref)
        got = ops.packed_attn_bwd(g, q, k, v, out, lse, cq, ck, causal=causal)
        for x, (want, tol) in zip(got, reference_grads(g, q, k, v, lens, causal, D ** -0.5, ref[1])):
            assert x.dtype == dt and ((x.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("H,Hk,D", [(8, 2, 128), (8, 2, 64), (6, 3, 32), (5, 1, 40), (2, 2, 128), (3, 3, 7)])
@pytest.mark.parametrize("causal", [False, True])
def test_views(causal, H, Hk, D, dt):
    """column ranges of a fused projection that starts at an aligned and at an odd element, head-major tensors, keys shared by a stride of zero:
    the same bits as contiguous operands"""
    from casmtr_amd import ops
    lens = [(170, 170), (3, 3), (64, 64), (0, 0), (129, 129)]
    T, c = 366, cu([a for a, _ in lens])
    for at in (0, 1):
        N = H + 2 * Hk
        qkv = torch.randn(T, N * D + 8 * at, device="cuda").to(dt)[:, at:at + N * D].unflatten(1, (N, D))
        q, k, v = qkv.split([H, Hk, Hk], 1)
        g = torch.randn(T, H, D, device="cuda").to(dt)

        def grads(q, k, v):
            out, lse = ops.packed_attn(q, k, v, c, causal=causal, want_lse=True)
            return (out, *ops.packed_attn_bwd(g, q, k, v, out, lse, c, causal=causal))

        want = grads(q.contiguous(), k.contiguous(), v.contiguous())
        hm = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)
        for views in ((q, k, v), (hm(q), hm(k), hm(v)), (q, hm(k), v.contiguous())):
            assert all(torch.equal(a, b) for a, b in zip(grads(*views), want))
        one = lambda t: t[:, :1].expand(T, H, D)
        wide = grads(q, one(k), one(v))
        assert all(torch.equal(a, b) for a, b in zip(wide, grads(q, one(k).contiguous(), one(v).contiguous())))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("R,C", [(4100, 96), (20001, 64), (9000, 1000), (1300, 1100), (2500, 5000), (1030, 9000)])
def test_norm_gradient_of_many_rows(R, C, dt):
    """Rows beyond the norm's largest number of parts (1024 workgroups of one row, of four for up to 1024 columns), so that a part adds several.  A
    column of dw adds the rows of a part, every 32nd part, and the 32 lanes: that many roundings u of the magnitudes' sum, 2 u for each term's products,
    and n carries rstd's 32 u."""
    from casmtr_amd import ops
    r = torch.Generator().manual_seed(R)
    x, dy, dh = (torch.randn(R, C, generator=r).to(dt).cuda() for _ in range(3))
    w = (1 + 0.3 * torch.randn(C, generator=r)).to(dt).cuda()
    per = 4 if C <= 1024 else 1
    parts = min(-(-R // per), 1024) * per
    assert parts < R
    y, _, rstd = ops.rms_norm(x, w, 1e-5, want_rstd=True)
    dx, dw = ops.rms_norm_bwd(dy, x, w, rstd, dh=dh)
    rs = 1 / torch.sqrt(x.double().square().mean(-1, keepdim=True) + 1e-5)
    n, g = x.double() * rs, dy.double() * w.double()
    ref = (g - n * (g * n).mean(-1, keepdim=True)) * rs + dh.double()
    mag = (g.abs() + 2 * n.abs() * (g * n).abs().mean(-1, keepdim=True)) * rs
    assert ((dx.double() - ref).abs() <= half(dt) * ref.abs() + 140 * U * mag + 2 * U * ref.abs() + sub(dt)).all()
    terms = dy.double() * n
    adds = -(-R // parts) + -(-parts // 32) + 32
    want = terms.sum(0)
    assert ((dw.double() - want).abs() <= half(dt) * want.abs() + (adds + 36) * U * terms.abs().sum(0) + sub(dt)).all()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("H,Hk,D", [(8, 2, 128), (6, 2, 32), (4, 4, 64)])
def test_prompts_beside_single_tokens(H, Hk, D, dt):
    """a serving batch in one call: a whole prompt, parts of prompts behind what their caches hold, single tokens over long and short caches"""
    from casmtr_amd import ops
    cap, lens = 3000, [(1, 2999), (700, 700), (1, 5), (300, 2500), (1, 3000), (0, 90), (1, 1), (17, 1400), (1, 0)]
    q, k, v, cq, _ = make([(a, cap) for a, _ in lens], H, Hk, D, dt, tail=0)
    for s, (_, n) in enumerate(lens):
        k[s * cap + n:(s + 1) * cap], v[s * cap + n:(s + 1) * cap] = float("nan"), float("inf")
    ln = torch.tensor([n for _, n in lens], dtype=torch.int32).cuda()
    for causal in (False, True):
        out, lse = ops.packed_attn(q, k, v, cq, cu([cap] * len(lens)), len_k=ln, causal=causal, want_lse=True)
        check(out, lse, reference(q, k, v, lens, causal, D ** -0.5, starts=[s * cap for s in range(len(lens))]))
