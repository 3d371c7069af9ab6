"""Packed attention at the edges of its numbers: shares of the keys whose weight underflows, probabilities and score gradients below fp16's
normal range, fp32 magnitudes next to the largest."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def cu(lens):
    t = torch.zeros(len(lens) + 1, dtype=torch.int32)
    t[1:] = torch.tensor(lens).cumsum(0)
    return t.cuda()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("H,Hk,D", [(8, 2, 128), (4, 4, 32), (4, 2, 64)])
@pytest.mark.parametrize("rows,keys", [(1, 4096), (5, 700), (1, 300), (40, 3000), (300, 3000), (5, 100)])
@pytest.mark.parametrize("at", [2, -1])
def test_visible_infinities_in_shares_of_no_weight(at, rows, keys, H, Hk, D, dt):
    """One key's score lies 400 above all others, so whatever part of the keys it is not in weighs exp(-400) = 0 beside it.  An infinity or NaN
    at a visible key of such a part reaches the row all the same (0 * inf), however the keys are split, and no other row or column."""
    from casmtr_amd import ops
    g = torch.Generator().manual_seed(keys)
    q, k, v = (0.1 * torch.randn(n, h, D, generator=g) for n, h in ((2 * rows, H), (2 * keys, Hk), (2 * keys, Hk)))
    q[..., 0], k[..., 0] = 20.0, 0.0
    top = -1 if at == 2 else 2           # of each sequence
    for s in (0, 1):
        k[s * keys + top % keys, :, 0] = 20.0
    q, k, v = (t.to(dt).cuda() for t in (q, k, v))
    cq, ck = cu([rows] * 2), cu([keys] * 2)
    clean, lse = ops.packed_attn(q, k, v, cq, ck, scale=1.0, want_lse=True)
    assert clean.isfinite().all() and (lse >= 390).all()
    cols = torch.arange(D, device="cuda") != 5
    for bad in (math.nan, math.inf):
        v2 = v.clone()
        v2[at % keys, :, 5] = bad        # the first sequence alone
        out, l2 = ops.packed_attn(q, k, v2, cq, ck, scale=1.0, want_lse=True)
        assert not out[:rows, :, 5].isfinite().any()
        assert torch.equal(out[:rows][..., cols], clean[:rows][..., cols]) and torch.equal(out[rows:], clean[rows:]) and torch.equal(l2, lse)
    k2 = k.clone()
    k2[at % keys, :, 3] = math.nan       # a score that is not a number
    out, l2 = ops.packed_attn(q, k2, v, cq, ck, scale=1.0, want_lse=True)
    assert out[:rows].isnan().all() and l2[:rows].isnan().all()
    assert torch.equal(out[rows:], clean[rows:]) and torch.equal(l2[rows:], lse[rows:])


# ---- fp16: what lies below its normal range.  u = 2^-24.  A probability is rounded at 2^7 (forward) and 2^12 (dv) times its value: half a step of fp16 of
# itself (2^-11), and below the normal range half a subnormal step, 2^-25, of that: 2^-32 of the row's sum, 2^-37.  A ds is rounded at a power of two that brings
# the largest so far of its row (dq) or key (dk) to 2^8 at least: 2^-11 of itself or 2^-33 of that largest one.  The other terms are those of
# test_gpu_packed_attn.py: a score is off by es = (D + 8) u scale sum |q k| + 4 u |s|, a probability by 2 es + (nk + 36) u + 4 u |lse| of itself.
U = 2.0 ** -24
H16 = 2.0 ** -11


def _grads16(q, k, v, g, scale, causal, o):
    """one head, [n, D] each, o the forward pass' result in fp16 -> (out, tol), (dq, tol), (dk, tol), (dv, tol) in 64 bits"""
    q, k, v, g, o16 = (t.double() for t in (q, k, v, g, o))
    (a, D), b = q.shape, k.shape[0]
    s = q @ k.t() * scale
    if causal:
        s = s.masked_fill(torch.ones(a, b, dtype=torch.bool, device="cuda").triu(b - a + 1), -math.inf)
    es = ((D + 8) * U * scale * (q.abs() @ k.abs().t()) + 4 * U * s.abs().nan_to_num(posinf=0.0)).amax(1, keepdim=True)
    lse, p = torch.logsumexp(s, 1, keepdim=True), torch.softmax(s, 1)
    out, ep = p @ v, 2 * es + (b + 36) * U + 4 * U * lse.abs()
    otol = (H16 + ep) * (p @ v.abs()) + b * 2.0 ** -32 * v.abs().amax(0) + H16 * out.abs() + 2.0 ** -25
    dp, delta = g @ v.t(), (g * out).sum(1, keepdim=True)
    edelta = (g.abs() * ((o16 - out).abs() + (D + 8) * U * out.abs())).sum(1, keepdim=True)   # the kernel takes the rounded output's
    ds = p * (dp - delta)
    eds = p * (ep * (dp - delta).abs() + (D + 8) * U * (g.abs() @ v.abs().t()) + edelta) + H16 * ds.abs()
    low = 2.0 ** -33 * (ds.abs() + eds).amax(1, keepdim=True)
    dq, tq = ds @ k * scale, scale * ((eds + low + (b + 32) * U * ds.abs()) @ k.abs())
    low = 2.0 ** -33 * (ds.abs() + eds).amax(0, keepdim=True)
    dk, tk = ds.t() @ q * scale, scale * ((eds + low + (a + 32) * U * ds.abs()).t() @ q.abs())
    dv, tv = p.t() @ g, (p * (ep + H16 + (a + 32) * U) + 2.0 ** -37).t() @ g.abs()
    fin = lambda x, t: (x, t + H16 * x.abs() + 2.0 ** -25)
    return (out, otol), fin(dq, tq), fin(dk, tk), fin(dv, tv)


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("rows,keys,causal", [(64, 4096, False), (33, 16384, False), (1500, 1500, True), (2, 9000, True)])
@pytest.mark.parametrize("size,spread", [(1e-4, 1.0), (1e-3, 1.0), (100.0, 4.0), (6e4, 0.0)])
def test_fp16_gradients_of_any_size(size, spread, rows, keys, causal, D):
    """Gradients far below and above 1 (a mean over many tokens, a scaled loss), over keys that weigh 1 / nk and less: every ds and many
    probabilities lie below fp16's normal range while the results lie in it."""
    from casmtr_amd import ops
    r = torch.Generator().manual_seed(rows + D)
    q, k, v, g = (torch.randn(n, 2, D, generator=r) for n in (rows, keys, keys, rows))
    g = g / g.abs().amax()
    q, k, v, g = (t.half().cuda() for t in (q * spread / 16, k * 16, v, g * size))
    cq, ck = cu([rows]), cu([keys])
    out, lse = ops.packed_attn(q, k, v, cq, ck, causal=causal, want_lse=True)
    got = (out, *ops.packed_attn_bwd(g, q, k, v, out, lse, cq, ck, causal=causal))
    for h in (0, 1):
        want = _grads16(q[:, h], k[:, h], v[:, h], g[:, h], D ** -0.5, causal, out[:, h])
        for name, x, (ref, tol) in zip(("out", "dq", "dk", "dv"), got, want):
            err = (x[:, h].double() - ref).abs()
            over = err > tol
            big = ref.abs() + tol > 65504.0          # (past the type's range: infinite)
            assert not (over & ~big).any(), f"{name}: {(err / tol)[~big].max().item():.2f} of the tolerance"


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("rows,keys", [(1, 65536), (40, 20000), (200, 8192), (3, 200)])
def test_fp16_many_small_probabilities(rows, keys, D):
    """one key takes nearly all the weight and has a value of 0; the others weigh 2^-17 to 2^-25 of it each and make up the result together"""
    from casmtr_amd import ops
    for bits in (17.0, 21.5, 24.75):
        q, k = torch.zeros(rows, 1, D), torch.zeros(keys, 1, D)
        q[..., 0], k[1:, :, 0] = 1.0, -bits * math.log(2)
        v = torch.rand(keys, 1, D, generator=torch.Generator().manual_seed(D)) + 0.5
        v[0] = 0
        q, k, v = (t.half().cuda() for t in (q, k, v))
        for top in (0, keys - 1):
            k[[0, top]], v[[0, top]] = k[[top, 0]], v[[top, 0]]
            out = ops.packed_attn(q, k, v, cu([rows]), cu([keys]), scale=1.0)
            p = torch.softmax(q[:, 0].double() @ k[:, 0].double().t(), 1)
            ref = p @ v[:, 0].double()
            es = ((D + 8) * U * (q[:, 0].abs().double() @ k[:, 0].abs().double().t()) * 2).amax()
            tol = (2 * H16 + 2 * es + (keys + 32) * U) * ref + keys * 2.0 ** -32 * 1.5 + 2.0 ** -25
            assert ((out[:, 0].double() - ref).abs() <= tol).all(), ((out[:, 0].double() - ref).abs() / tol).max().item()


@pytest.mark.parametrize("H,Hk,D", [(4, 2, 32), (2, 1, 64), (2, 2, 128)])
@pytest.mark.parametrize("rows,keys", [(1, 300), (9, 100), (150, 300), (700, 90)])
@pytest.mark.parametrize("causal", [False, True])
def test_largest_fp32_magnitudes(causal, rows, keys, H, Hk, D):
    """The largest finite fp32 numbers are numbers on every path: keys of that magnitude meet zeros or numbers small enough, values of it weigh
    nothing (their key's score is far below the others') or 2^-20.  Bounds as in test_gpu_packed_attn.py; scores are exact here but for (D + 8) u of what they add."""
    from casmtr_amd import ops
    top = torch.finfo(torch.float32).max
    r = torch.Generator().manual_seed(rows)
    q, k, v, g = (torch.randn(n, h, D, generator=r).cuda() for n, h in ((rows, H), (keys, Hk), (keys, Hk), (rows, H)))
    cq, ck = cu([rows]), cu([keys])
    q[..., 0], k[..., 0] = 0.0, 0.0
    q[..., 1], k[..., 1] = 2.0 ** -126, 0.0
    g[..., 2] = 0.0
    for s in (1.0, -1.0):
        k2, v2 = k.clone(), v.clone()
        k2[1, :, 0], k2[3, :, 1] = s * top, -s * top    # meets 0; meets 2^-126: +-4 in the score
        v2[5, :, 2] = s * top * 2.0 ** -20              # (weighs at most 1: well inside)
        v2[6, :, 2], k2[6] = s * top, 0.0
        k2[6, :, 3], q[..., 3] = -4000.0, 1.0           # weight exp(-4000 scale): nothing
        o, lse = ops.packed_attn(q, k2, v2, cq, ck, causal=causal, scale=1.0, want_lse=True)
        dq, dk, dv = ops.packed_attn_bwd(g, q, k2, v2, o, lse, cq, ck, causal=causal, scale=1.0)
        assert o.isfinite().all() and dk.isfinite().all() and dv.isfinite().all()
        for h in range(H):
            m = h // (H // Hk)
            Q, K, V, G = q[:, h].double(), k2[:, m].double(), v2[:, m].double(), g[:, h].double()
            sc = Q @ K.t()
            if causal:
                sc = sc.masked_fill(torch.ones(rows, keys, dtype=torch.bool, device="cuda").triu(keys - rows + 1), -math.inf)
            es = ((D + 8) * U * (Q.abs() @ K.abs().t()) + 4 * U * sc.abs()).masked_fill(sc == -math.inf, 0).masked_fill(sc < -3000, 0).amax(1, keepdim=True)
            p = torch.softmax(sc, 1).nan_to_num(0.0)
            lost = torch.where(p < 2.0 ** -125, p, 0.0)     # (the exponential gives 0 below the smallest normal number, 2^-126: such a p may go as a whole)
            tol = (2 * es + (keys + 34) * U) * (p @ V.abs()) + lost @ V.abs() + 2.0 ** -149
            assert ((o[:, h].double() - p @ V).abs() <= tol).all()
            # dq: the 64-bit gradient within its bound, but where that passes fp32's range: |ds| above 1 times a key of the largest magnitude
            dp, O = G @ V.t(), p @ V
            delta = (G * O).sum(1, keepdim=True)
            ds = p * (dp - delta)
            ep = 2 * es + (keys + 36) * U + 4 * U * lse[:, h].double().abs().nan_to_num(posinf=0.0)[:, None]
            eds = lost * (dp - delta).abs() + p * (ep * (dp - delta).abs() + (D + 8) * U * (G.abs() @ V.abs().t()) + (G.abs() * (tol + (D + 8) * U * O.abs())).sum(1, keepdim=True))
            ref, tq = ds @ K, (eds + (keys + 32) * U * ds.abs()) @ K.abs()
            fits = ref.abs() + tq + U * ref.abs() <= top
            assert fits.double().mean() > 0.9 and ((dq[:, h].double() - ref).abs() <= tq + U * ref.abs())[fits].all()
