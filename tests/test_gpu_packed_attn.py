"""Packed attention (casmtr_packed_attn_fwd / _bwd) against the formulas in 64 bits, sequence by sequence.

Tolerances.  u = 2^-24, half(T) half a step of the element type.  A score sums D products in fp32: off by at most
ds = (D + 8) u scale sum_d |q_d k_d| + 4 u |s|.  A probability is off by 2 ds relative to its row's sum, is rounded to the values' type
(half(T); fp32: not at all), and products and sum add up to nk terms in fp32: (nk + 32) u.  So
  |o - ref| <= (half16 + 2 ds + (nk + 32) u) sum_j p_j |v_j| + half(T) |ref| + half a subnormal step,
  |lse - ref| <= ds + (nk + 32) u + 4 u |lse|.
Backward: p is recomputed from the scores and lse, off by ep = 2 ds + (nk + 32) u + 4 u |lse| + 4 u relative to itself; do . v is off by (D + 8) u sum |do v|;
delta = do . o by the output's tolerance, sum |do| tol(o), and (D + 8) u sum |do o|.  So ds is off by
  eds = p (ep |do . v - delta| + (D + 8) u sum |do v| + edelta) + half16 |ds| + half a subnormal step,
and the products add n terms: (n + 32) u of the summed magnitudes.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.bfloat16, torch.float16, torch.float32]
half = lambda t: torch.finfo(t).eps / 2
sub = lambda t: torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2
step16 = lambda t: 0.0 if t == torch.float32 else half(t)

# (rows, keys) of the sequences
LENS = {
    "one token": [(1, 1)],
    "single tokens": [(1, 700), (1, 1), (1, 33), (1, 2100), (1, 64)],
    "prompts": [(130, 130), (1, 1), (257, 257), (64, 64), (33, 33)],
    "empty ones": [(0, 0), (5, 0), (0, 7), (40, 40), (0, 0)],
    "more rows than keys": [(200, 70), (90, 89), (3, 1)],
    "more keys than rows": [(3, 500), (65, 129), (2, 2)],
    "long": [(1100, 1100)],
    "many": [(7, 7), (25, 25), (1, 1)] * 30,
}
HEADS = [(1, 1, 64), (8, 2, 128), (6, 2, 32), (5, 1, 40), (4, 4, 16), (2, 1, 96), (3, 3, 33), (16, 1, 128), (2, 2, 1)]


def cu(lens):
    t = torch.zeros(len(lens) + 1, dtype=torch.int32)
    t[1:] = torch.tensor(lens).cumsum(0)
    return t.cuda()


def make(lens, H, Hk, D, dt, seed=0, tail=3):
    """packed operands with `tail` rows behind the last sequence"""
    g = torch.Generator().manual_seed(seed)
    nq, nk = sum(a for a, _ in lens) + tail, sum(b for _, b in lens) + tail
    q, k, v = (torch.randn(n, h, D, generator=g).to(dt).cuda() for n, h in ((nq, H), (nk, Hk), (nk, Hk)))
    return q, k, v, cu([a for a, _ in lens]), cu([b for _, b in lens])


def seen(a, b, causal):
    i, j = torch.arange(a, device="cuda")[:, None], torch.arange(b, device="cuda")
    return (j <= i + b - a) if causal else torch.ones(a, b, dtype=torch.bool, device="cuda")


def reference(q, k, v, lens, causal, scale, starts=None):
    """-> out, lse and their tolerances, in 64 bits; starts: first key of each sequence"""
    H, Hk, D = q.shape[1], k.shape[1], q.shape[2]
    out, tol = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse, ltol = (torch.full(q.shape[:2], x, dtype=torch.float64, device="cuda") for x in (-math.inf, 0.0))
    q0 = k0 = 0
    for s, (a, b) in enumerate(lens):
        at = k0 if starts is None else starts[s]
        if a and b:
            vis = seen(a, b, causal)
            for h in range(H):
                qq, kk, vv = q[q0:q0 + a, h].double(), k[at:at + b, h // (H // Hk)].double(), v[at:at + b, h // (H // Hk)].double()
                sc = (qq @ kk.t() * scale).masked_fill(~vis, -math.inf)
                ds = ((D + 8) * U * scale * (qq.abs() @ kk.abs().t()) + 4 * U * sc.abs()).masked_fill(~vis, 0).amax(1, keepdim=True)
                p = torch.softmax(sc, 1).masked_fill(~vis.any(1, keepdim=True), 0)
                out[q0:q0 + a, h] = p @ vv
                n = (b + 32) * U
                tol[q0:q0 + a, h] = (step16(q.dtype) + 2 * ds + n) * (p @ vv.abs())
                lse[q0:q0 + a, h] = torch.logsumexp(sc, 1)
                ltol[q0:q0 + a, h] = ds[:, 0] + n + 4 * U * lse[q0:q0 + a, h].abs().nan_to_num(posinf=0.0)
        q0, k0 = q0 + a, k0 + b
    return out, tol + half(q.dtype) * out.abs() + sub(q.dtype), lse, ltol


def reference_grads(g, q, k, v, lens, causal, scale, otol):
    """-> (dq, tol), (dk, tol), (dv, tol)"""
    H, Hk, D = q.shape[1], k.shape[1], q.shape[2]
    z = lambda t: torch.zeros(t.shape, dtype=torch.float64, device="cuda")
    dq, dk, dv, tq, tk, tv = z(q), z(k), z(v), z(q), z(k), z(v)
    r, low = step16(q.dtype), (0.0 if q.dtype == torch.float32 else sub(q.dtype))
    q0 = k0 = 0
    for a, b in lens:
        if a and b:
            vis = seen(a, b, causal)
            any_ = vis.any(1, keepdim=True)
            for h in range(H):
                m = h // (H // Hk)
                qq, gg, kk, vv = q[q0:q0 + a, h].double(), g[q0:q0 + a, h].double(), k[k0:k0 + b, m].double(), v[k0:k0 + b, m].double()
                sc = (qq @ kk.t() * scale).masked_fill(~vis, -math.inf)
                err = ((D + 8) * U * scale * (qq.abs() @ kk.abs().t()) + 4 * U * sc.abs()).masked_fill(~vis, 0).amax(1, keepdim=True)
                lse = torch.logsumexp(sc, 1, keepdim=True).masked_fill(~any_, 0)
                p = torch.softmax(sc, 1).masked_fill(~any_, 0)
                o, dp = p @ vv, gg @ vv.t()
                ds = p * (dp - (gg * o).sum(1, keepdim=True))
                ep = 2 * err + (b + 36) * U + 4 * U * lse.abs()
                edelta = (gg.abs() * (otol[q0:q0 + a, h] + (D + 8) * U * o.abs())).sum(1, keepdim=True)
                eds = (p * (ep * (dp - (gg * o).sum(1, keepdim=True)).abs() + (D + 8) * U * (gg.abs() @ vv.abs().t()) + edelta) + r * ds.abs() + low) * vis
                epp = (p * (ep + r) + low) * vis
                dq[q0:q0 + a, h] = ds @ kk * scale
                tq[q0:q0 + a, h] = scale * ((eds + (b + 32) * U * ds.abs()) @ kk.abs())
                n = a * (H // Hk) + 32
                dk[k0:k0 + b, m] += ds.t() @ qq * scale
                tk[k0:k0 + b, m] += scale * ((eds + n * U * ds.abs()).t() @ qq.abs())
                dv[k0:k0 + b, m] += p.t() @ gg
                tv[k0:k0 + b, m] += (epp + n * U * p).t() @ gg.abs()
        q0, k0 = q0 + a, k0 + b
    fin = lambda x, t: (x, t + half(q.dtype) * x.abs() + sub(q.dtype))
    return fin(dq, tq), fin(dk, tk), fin(dv, tv)


def check(got, lse, ref):
    out, tol, rl, ltol = ref
    assert ((got.double() - out).abs() <= tol).all()
    none = rl == -math.inf
    assert torch.equal(lse == -math.inf, none) and (got[none] == 0).all()
    assert ((lse.double() - rl).abs()[~none] <= ltol[~none]).all()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("H,Hk,D", HEADS)
@pytest.mark.parametrize("name", list(LENS))
def test_forward(name, H, Hk, D, dt):
    from casmtr_amd import ops
    lens = LENS[name]
    q, k, v, cq, ck = make(lens, H, Hk, D, dt)
    for causal in (False, True):
        for scale in (None, 0.3):
            out, lse = ops.packed_attn(q, k, v, cq, ck, causal=causal, scale=scale, want_lse=True)
            check(out, lse, reference(q, k, v, lens, causal, scale or D ** -0.5))
            assert torch.equal(ops.packed_attn(q, k, v, cq, ck, causal=causal, scale=scale), out)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("H,Hk,D", HEADS)
@pytest.mark.parametrize("name", list(LENS))
def test_backward(name, H, Hk, D, dt):
    from casmtr_amd import ops
    lens = LENS[name]
    q, k, v, cq, ck = make(lens, H, Hk, D, dt, seed=1)
    g = torch.randn(q.shape, generator=torch.Generator().manual_seed(2)).to(dt).cuda()
    for causal in (False, True):
        out, lse = ops.packed_attn(q, k, v, cq, ck, causal=causal, want_lse=True)
        got = ops.packed_attn_bwd(g, q, k, v, out, lse, cq, ck, causal=causal)
        otol = reference(q, k, v, lens, causal, D ** -0.5)[1]
        for x, (ref, tol) in zip(got, reference_grads(g, q, k, v, lens, causal, D ** -0.5, otol)):
            assert x.dtype == dt and ((x.double() - ref).abs() <= tol).all()
        again = ops.packed_attn_bwd(g, q, k, v, out, lse, cq, ck, causal=causal)
        assert all(torch.equal(x, y) for x, y in zip(got, again))


def test_backward_cache_and_views():
    """shares that are not in use get zero gradients whatever they hold; operands are views, the gradient of a sum is a broadcast view"""
    from casmtr_amd import ops
    from casmtr_amd.functions.packed_attention import packed_attention_op
    used, cap, rows = [40, 0, 7, 64], 64, 5
    q, k, v, cq, _ = make([(rows, cap)] * 4, 4, 2, 32, torch.float32, tail=0)
    ck, ln = cu([cap] * 4), torch.tensor(used, dtype=torch.int32).cuda()
    packed = torch.cat([torch.arange(s * cap, s * cap + n) for s, n in enumerate(used)]).cuda()
    want = [t.clone().requires_grad_() for t in (q, k[packed], v[packed])]
    packed_attention_op(*want, cq, cu(used), None, True).sum().backward()
    for s, n in enumerate(used):
        k[s * cap + n:(s + 1) * cap], v[s * cap + n:(s + 1) * cap] = math.nan, math.inf
    hm = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1).requires_grad_()
    got = [hm(q), hm(k), hm(v)]
    packed_attention_op(*got, cq, ck, ln, True).sum().backward()
    assert torch.equal(got[0].grad, want[0].grad)
    rest = torch.ones(4 * cap, dtype=torch.bool, device="cuda")
    rest[packed] = False
    for a, b in zip(got[1:], want[1:]):
        assert torch.equal(a.grad[packed], b.grad) and (a.grad[rest] == 0).all()


def test_gradient_against_differences():
    """central differences of sum(g o) in 64 bits along random directions; the kernel's gradients are held to the formula's tolerances"""
    from casmtr_amd.functions.packed_attention import packed_attention_op
    lens = [(30, 44), (17, 17)]
    q, k, v, cq, ck = make(lens, 4, 2, 24, torch.float32, tail=0)
    g = torch.randn_like(q)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(packed_attention_op(*leaves, cq, ck, None, True, 0.25), leaves, g)
    dirs = [torch.randn_like(t).double() for t in leaves]

    def loss(e):
        x = [t.detach().double() + e * d for t, d in zip(leaves, dirs)]
        return (g.double() * reference(*x, lens, True, 0.25)[0]).sum()

    diff = (loss(1e-4) - loss(-1e-4)) / 2e-4      # the third derivative's share is 1e-8 of the scale
    got = sum((a.double() * d).sum() for a, d in zip(grads, dirs))
    mag = sum((a.double() * d).abs().sum() for a, d in zip(grads, dirs))
    assert abs(got - diff) <= 1e-5 * mag


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("H,Hk,D", [(4, 2, 64), (3, 1, 128), (2, 2, 32)])
def test_hidden_infinities_backward(H, Hk, D, dt):
    """a key's infinities stay away from the gradients of rows that do not see it, a row's from those of keys that it does not see"""
    from casmtr_amd import ops
    lens = [(150, 150), (90, 90)]
    q, k, v, cq, ck = make(lens, H, Hk, D, dt)
    g = torch.randn(q.shape, device="cuda").to(dt)

    def grads(q, k, v, g):
        out, lse = ops.packed_attn(q, k, v, cq, ck, causal=True, want_lse=True)
        return ops.packed_attn_bwd(g, q, k, v, out, lse, cq, ck, causal=True)

    clean = grads(q, k, v, g)
    for bad in (math.nan, math.inf):
        k2, v2 = k.clone(), v.clone()
        k2[100, :, 3], v2[100, :, 5] = bad, bad
        dq, _, _ = grads(q, k2, v2, g)
        assert torch.equal(dq[:100], clean[0][:100]) and torch.equal(dq[150:], clean[0][150:])
        q2, g2 = q.clone(), g.clone()
        q2[60, :, 3], g2[60, :, 5] = bad, bad
        _, dk, dv = grads(q2, k, v, g2)
        assert torch.equal(dk[61:], clean[1][61:]) and torch.equal(dv[61:], clean[2][61:])


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("H,Hk,D", [(8, 2, 128), (4, 4, 32), (12, 4, 64), (5, 1, 80)])
@pytest.mark.parametrize("rows", [1, 2, 5])
def test_cache(rows, H, Hk, D, dt):
    """rows per sequence against caches of fixed shares; what is not in use is NaN"""
    from casmtr_amd import ops
    cap, used = 1500, [1500, 1, 0, 7, 800, 64, 65, 1499]
    lens = [(rows, n) for n in used]
    q, k, v, cq, _ = make([(rows, cap)] * len(used), H, Hk, D, dt, tail=0)
    for s, n in enumerate(used):
        k[s * cap + n:(s + 1) * cap], v[s * cap + n:(s + 1) * cap] = math.nan, math.inf
    ck, ln = cu([cap] * len(used)), torch.tensor(used, dtype=torch.int32).cuda()
    for causal in (False, True):
        out, lse = ops.packed_attn(q, k, v, cq, ck, len_k=ln, causal=causal, want_lse=True)
        check(out, lse, reference(q, k, v, lens, causal, D ** -0.5, starts=[s * cap for s in range(len(used))]))


@pytest.mark.parametrize("dt", TYPES)
def test_views(dt):
    """column ranges of a fused projection, head-major tensors, a view that starts at an odd element, keys shared by a stride of zero"""
    from casmtr_amd import ops
    lens = [(70, 70), (3, 3), (140, 140)]
    T = 213
    c = cu([a for a, _ in lens])
    for at in (0, 1):
        qkv = torch.randn(T, 12 * 48 + at, device="cuda").to(dt)[:, at:].unflatten(1, (12, 48))
        q, k, v = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]
        want = ops.packed_attn(q.contiguous(), k.contiguous(), v.contiguous(), c, causal=True)
        assert torch.equal(ops.packed_attn(q, k, v, c, causal=True), want)
        hm = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)
        assert torch.equal(ops.packed_attn(hm(q), hm(k), hm(v), c, causal=True), want)
        one = lambda t: t[:, :1].expand(T, 4, 48)
        assert torch.equal(ops.packed_attn(q, one(k), one(v), c), ops.packed_attn(q, k[:, :1], v[:, :1], c))


@pytest.mark.parametrize("dt", TYPES)
def test_large_scores(dt):
    """scores that grow along the keys by far more than an exponential holds: the running maximum has to follow"""
    from casmtr_amd import ops
    lens = [(40, 600), (300, 300)]
    q, k, v, cq, ck = make(lens, 2, 1, 64, dt)
    k *= torch.linspace(0.01, 30, k.shape[0], device="cuda").view(-1, 1, 1).to(dt)
    for causal in (False, True):
        out, lse = ops.packed_attn(q, k, v, cq, ck, causal=causal, scale=1.0, want_lse=True)
        check(out, lse, reference(q, k, v, lens, causal, 1.0))
    kn = -k.abs()   # only very low scores: nothing may underflow to an empty row
    qn = q.abs()
    out, lse = ops.packed_attn(qn, kn, v, cq, ck, scale=1.0, want_lse=True)
    check(out, lse, reference(qn, kn, v, lens, False, 1.0))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("H,Hk,D", [(4, 2, 64), (3, 1, 128), (2, 2, 32)])
def test_hidden_infinities(H, Hk, D, dt):
    """infinities and NaN in keys and values that a row does not see change nothing for it; rows that see them get them"""
    from casmtr_amd import ops
    lens = [(150, 150), (90, 90)]
    q, k, v, cq, ck = make(lens, H, Hk, D, dt)
    clean = ops.packed_attn(q, k, v, cq, ck, causal=True)
    for bad in (math.nan, math.inf, -math.inf):
        k2, v2 = k.clone(), v.clone()
        v2[100, :, D // 2] = bad
        k2[150 + 70, :, 1] = bad
        k2[240:], v2[240:] = bad, bad   # rows of no sequence
        out = ops.packed_attn(q, k2, v2, cq, ck, causal=True)
        keep = torch.ones(q.shape[0], dtype=torch.bool, device="cuda")
        keep[100:150], keep[220:240] = False, False
        assert torch.equal(out[keep], clean[keep])
        assert not out[100:150, :, D // 2].isfinite().any()
        cols = torch.arange(D, device="cuda") != D // 2
        assert torch.equal(out[100:150][..., cols], clean[100:150][..., cols])
        if math.isnan(bad):
            assert out[220:240].isnan().all()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("H,Hk,D", [(4, 2, 64), (3, 1, 128), (2, 2, 32)])
def test_key_of_no_weight(H, Hk, D, dt):
    """a key whose scores are -inf weighs nothing: the outputs are those without it, its own gradients are 0 (row counts beside the tiles')"""
    from casmtr_amd import ops
    for lens in ([(70, 50)], [(33, 90), (5, 21)]):
        q, k, v, cq, ck = make(lens, H, Hk, D, dt, tail=0)
        q[..., 0] = q[..., 0].abs() + 0.1
        g = torch.randn(q.shape, device="cuda").to(dt)
        k2 = k.clone()
        k2[20, :, 0] = -math.inf
        out, lse = ops.packed_attn(q, k2, v, cq, ck, want_lse=True)
        _, dk, dv = ops.packed_attn_bwd(g, q, k2, v, out, lse, cq, ck)
        less = [(lens[0][0], lens[0][1] - 1)] + lens[1:]
        keep = torch.arange(k.shape[0], device="cuda") != 20
        check(out, lse, reference(q, k[keep], v[keep], less, False, D ** -0.5))
        assert (dk[20] == 0).all() and (dv[20] == 0).all()
        otol = reference(q, k[keep], v[keep], less, False, D ** -0.5)[1]
        _, (rk, tk), (rv, tv) = reference_grads(g, q, k[keep], v[keep], less, False, D ** -0.5, otol)
        assert ((dk[keep].double() - rk).abs() <= tk).all() and ((dv[keep].double() - rv).abs() <= tv).all()


def test_wrong_lengths_stay_inside():
    """arrays that claim more than there is: nothing outside the tensors is read or written (what the rows hold is not defined)"""
    from casmtr_amd import ops
    q, k, v, cq, ck = make([(50, 50), (60, 60)], 2, 1, 64, torch.bfloat16, tail=0)
    for c in ([0, 900, 2000], [0, -5, 110], [-9, 50, 2 ** 31 - 1], [110, 50, 0]):
        t = torch.tensor(c, dtype=torch.int32).cuda()
        assert ops.packed_attn(q, k, v, t, t, len_k=torch.tensor([2 ** 31 - 1, -3], dtype=torch.int32).cuda()).shape == q.shape


def test_uncovered_rows():
    from casmtr_amd import ops
    q, k, v, _, _ = make([(200, 200)], 2, 2, 32, torch.float32, tail=0)
    c = torch.tensor([13, 100, 150], dtype=torch.int32).cuda()   # 13 rows before the first, 50 behind the last sequence
    out, lse = ops.packed_attn(q, k, v, c, want_lse=True)
    ref = ops.packed_attn(q[13:150].clone(), k[13:150].clone(), v[13:150].clone(), cu([87, 50]))
    assert torch.equal(out[13:150], ref) and (out[:13] == 0).all() and (out[150:] == 0).all() and (lse[:13] == -math.inf).all()


def test_no_sequences_and_no_rows():
    from casmtr_amd import ops
    q = torch.randn(5, 2, 32, device="cuda")
    z = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert (ops.packed_attn(q, q, q, z) == 0).all()
    assert ops.packed_attn(q[:0], q, q, cu([0]), cu([5])).shape == (0, 2, 32)
    out, lse = ops.packed_attn(q, q[:0], q[:0], cu([5]), cu([0]), want_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()


def test_refusals():
    from casmtr_amd import ops
    q, k, v, cq, ck = make([(9, 9)], 4, 2, 64, torch.bfloat16, tail=0)
    for bad in (lambda: ops.packed_attn(q.cpu(), k, v, cq), lambda: ops.packed_attn(q, k.float(), v, cq), lambda: ops.packed_attn(q, k, v[:8], cq),
                lambda: ops.packed_attn(q[:, :3], k, v, cq), lambda: ops.packed_attn(q, k, v, cq.long()), lambda: ops.packed_attn(q, k, v, cq.cpu()),
                lambda: ops.packed_attn(q[:8], k, v, cq), lambda: ops.packed_attn(q, k, v, cq, ck[:1]), lambda: ops.packed_attn(q, k, v, cq[:0], ck[:0]),
                lambda: ops.packed_attn(q, k, v, cq, ck, len_k=ck), lambda: ops.packed_attn(q, k, v, cq, scale=0.0), lambda: ops.packed_attn(q, k, v, cq, scale=-1.0),
                lambda: ops.packed_attn(q, k, v, cq, scale=math.nan), lambda: ops.packed_attn(q, k, v, cq, scale=math.inf),
                lambda: ops.packed_attn(q.double(), k.double(), v.double(), cq), lambda: ops.packed_attn(q[..., ::2], k[..., ::2], v[..., ::2], cq),
                lambda: ops.packed_attn(q, k[..., :32], v[..., :32], cq), lambda: ops.packed_attn(*(torch.zeros(9, 2, 136, device="cuda"),) * 3, cq),
                lambda: ops.packed_attn(q[0], k[0], v[0], cq), lambda: ops.packed_attn(q, k[:, :0], v[:, :0], cq), lambda: ops.packed_attn(q, k, v, cq.view(1, 2))):
        with pytest.raises(RuntimeError):
            bad()
    out, lse = ops.packed_attn(q, k, v, cq, want_lse=True)
    for bad in (lambda: ops.packed_attn_bwd(out[:8], q, k, v, out, lse, cq), lambda: ops.packed_attn_bwd(out.float(), q, k, v, out, lse, cq),
                lambda: ops.packed_attn_bwd(out, q, k, v, out, lse[:, :2], cq), lambda: ops.packed_attn_bwd(out, q, k, v, out, lse.half(), cq),
                lambda: ops.packed_attn_bwd(out[:1].expand(9, 4, 64), q, k, v, out, lse, cq), lambda: ops.packed_attn_bwd(out, q, k, v, out.cpu(), lse, cq)):
        with pytest.raises(RuntimeError):
            bad()
