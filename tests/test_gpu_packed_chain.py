"""The packed-token operators as they are used together: a pre-norm attention block on packed sequences, prompts against single tokens over a
cache, the backbone's global attention; on other streams, in captured graphs, beyond 32-bit offsets."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def cu(lens):
    t = torch.zeros(len(lens) + 1, dtype=torch.int32)
    t[1:] = torch.tensor(lens).cumsum(0)
    return t.cuda()


class Block:
    """h = x + residual; q, k, v = projection(norm(h)); attention of the turned q and k"""

    def __init__(self, C, H, Hk, D, dt, seed=0):
        from casmtr_amd import ops
        g = torch.Generator().manual_seed(seed)
        self.H, self.Hk, self.D = H, Hk, D
        self.w = (1 + 0.1 * torch.randn(C, generator=g)).to(dt).cuda()
        self.p = (torch.randn((H + 2 * Hk) * D, C, generator=g) / C ** 0.5).to(dt).cuda()
        self.freq, self.gain = ops.rotary_freqs(D, factor=4.0, trained=256)

    def heads(self, qkv):
        q, k, v = qkv.view(-1, self.H + 2 * self.Hk, self.D).split([self.H, self.Hk, self.Hk], 1)
        return q, k, v

    def serve(self, x, res, pos):
        from casmtr_amd import ops
        y, h = ops.rms_norm(x, self.w, residual=res)
        q, k, v = self.heads(y @ self.p.t())
        return (*ops.rotary(q, k, pos, self.freq, gain=self.gain), v, h)


def positions(lens):
    return torch.cat([torch.arange(n) for n in lens]).cuda()


def test_training_step_against_64_bits():
    """Every stage is off by at most about 1e-5 of its magnitude in fp32 (sums of C, D and nk terms of 2^-24 each); scores of magnitude below 10
    amplify that by 20 at most, and so do the gradients: 1e-3 of the result's norm holds them all, by a factor of several."""
    from casmtr_amd.functions.packed_attention import packed_attention_op
    from casmtr_amd.functions.rms_norm import rms_norm_op
    from casmtr_amd.functions.rotary import rotary_op
    lens, C = [70, 1, 129, 33], 96
    b = Block(C, 6, 2, 32, torch.float32)
    x, r = torch.randn(sum(lens), C, device="cuda"), torch.randn(sum(lens), C, device="cuda")
    g, gh = torch.randn(sum(lens), 6, 32, device="cuda"), torch.randn_like(x)
    pos, c = positions(lens), cu(lens)
    leaves = [t.clone().requires_grad_() for t in (x, r, b.w, b.p)]
    y, h = rms_norm_op(leaves[0], leaves[2], 1e-6, leaves[1])
    q, k, v = b.heads(y @ leaves[3].t())
    q, k = rotary_op(q, k, pos, b.freq, "half", b.gain)
    o = packed_attention_op(q, k, v, c, None, None, True)
    got = [o, *torch.autograd.grad((o, h), leaves, (g, gh))]

    ref = [t.double().requires_grad_() for t in (x, r, b.w, b.p)]
    h64 = ref[0] + ref[1]
    y64 = h64 / (h64.square().mean(-1, keepdim=True) + 1e-6).sqrt() * ref[2]
    q, k, v = b.heads(y64 @ ref[3].t())
    t = (pos.double()[:, None] * b.freq)[:, None]

    def turn(a):
        u, w = a[..., :16], a[..., 16:]
        return b.gain * torch.cat([u * t.cos() - w * t.sin(), w * t.cos() + u * t.sin()], -1)

    q, k, outs, at = turn(q), turn(k), [], 0
    for n in lens:
        s = torch.einsum("ihd,jhd->hij", q[at:at + n], k[at:at + n].repeat_interleave(3, 1)) / 32 ** 0.5
        s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), -math.inf)
        outs.append(torch.einsum("hij,jhd->ihd", s.softmax(-1), v[at:at + n].repeat_interleave(3, 1)))
        at += n
    o64 = torch.cat(outs)
    want = [o64, *torch.autograd.grad((o64, h64), ref, (g.double(), gh.double()))]
    for a, w in zip(got, want):
        assert (a.double() - w).norm() <= 1e-3 * w.norm()


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_prompt_then_single_tokens(dt):
    """the prompt's rows one by one, as single tokens against a growing cache, give what the whole prompt gave: the same sums in another order, each
    within 2 (nk + D) 2^-24 and half a step of the type of 64 bits, for values of magnitude below 4"""
    from casmtr_amd import ops
    lens, C, cap = [37, 5, 90], 64, 96
    b = Block(C, 4, 2, 32, dt)
    x, r = torch.randn(sum(lens), C, device="cuda").to(dt), torch.randn(sum(lens), C, device="cuda").to(dt)
    q, k, v, _ = b.serve(x, r, positions(lens))
    whole = ops.packed_attn(q, k, v, cu(lens), causal=True)
    kc, vc = (torch.full((3 * cap, 2, 32), math.nan, device="cuda", dtype=dt) for _ in range(2))
    ends = torch.tensor(lens).cumsum(0).tolist()
    step = 3 * (2 * (cap + 32) * 2.0 ** -24 + torch.finfo(dt).eps) * 4
    for i in range(max(lens)):
        live = [s for s, n in enumerate(lens) if i < n]
        rows = torch.tensor([ends[s] - lens[s] + i for s in live], device="cuda")
        for s, row in zip(live, rows.tolist()):
            kc[s * cap + i], vc[s * cap + i] = k[row], v[row]
        used = torch.tensor([min(i + 1, n) for n in lens], dtype=torch.int32).cuda()
        qs = q.new_zeros(3, 4, 32)
        qs[live] = q[rows]
        out = ops.packed_attn(qs, kc, vc, cu([1] * 3), cu([cap] * 3), len_k=used, causal=True)
        assert ((out[live].double() - whole[rows].double()).abs() <= step).all()


def test_global_attention_of_the_backbone(monkeypatch):
    """the backbone's reduced global attention through packed_attn against its library path: fp32 sums of 36 keys and 32 columns in another order"""
    from casmtr_amd.model.casmtr4c import _ReducedAttention
    torch.manual_seed(0)
    m = _ReducedAttention(128, 4, 8, True).eval().cuda()
    x = torch.randn(2, 48 * 48, 128, device="cuda")
    with torch.no_grad():
        want = m(x, 48, 48)
        monkeypatch.setenv("CASMTR_GLOBAL_ATTN", "packed")
        got = m(x, 48, 48)
    assert not torch.equal(got, torch.zeros_like(got)) and (got - want).abs().max() <= 1e-4 * want.abs().max()
    x.requires_grad_()
    m(x, 48, 48).sum().backward()   # with autograd on: the library path, whatever is selected
    assert x.grad is not None


def _serve_step(b, x, r, pos, kc, vc, ck, used, cq):
    from casmtr_amd import ops
    q, k, v, h = b.serve(x, r, pos)
    o = ops.packed_attn(q, kc, vc, cq, ck, len_k=used, causal=True)
    q8, s8, _ = ops.rms_norm_quant(h, b.w, residual=x, group=None)
    return o, h, q8.float(), s8


def test_captured_serving_step():
    """norm, rotary, split single-token attention and 8-bit norm in one captured graph, replayed with new contents and eager work in between"""
    from casmtr_amd import ops
    n, cap, C = 3, 2048, 256
    b = Block(C, 8, 2, 64, torch.bfloat16)
    mk = lambda *s: torch.randn(*s, device="cuda").to(torch.bfloat16)
    x, r, kc, vc = mk(n, C), mk(n, C), mk(n * cap, 2, 64), mk(n * cap, 2, 64)
    pos, used = torch.tensor([5, 900, 2000], device="cuda"), torch.tensor([6, 901, 2001], dtype=torch.int32, device="cuda")
    cq, ck = cu([1] * n), cu([cap] * n)
    assert ops._lib.lib().casmtr_packed_attn_ws_floats(n, n * cap, n, 8, 2, 64) > 0   # the keys are split
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _serve_step(b, x, r, pos, kc, vc, ck, used, cq)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):   # two graphs over the same operands, each with workspaces of its own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = _serve_step(b, x, r, pos, kc, vc, ck, used, cq)
        graphs.append((g, outs))
    for turn in range(4):
        x.copy_(mk(n, C)), kc.copy_(mk(n * cap, 2, 64))
        used.copy_(torch.tensor([1 + turn, 700 * turn, 2048 - turn], dtype=torch.int32))
        for g, _ in graphs:
            g.replay()
        want = _serve_step(b, x, r, pos, kc, vc, ck, used, cq)
        torch.cuda.synchronize()
        for _, outs in graphs:
            assert all(torch.equal(a, w) for a, w in zip(outs, want))


def test_captured_backward():
    """the gradients' kernels (split rows, partial sums) in a captured graph"""
    from casmtr_amd import ops
    lens = [300, 41]
    q, k, v, g = (torch.randn(341, h, 64, device="cuda").to(torch.float16) for h in (4, 2, 2, 4))
    x, w = torch.randn(341, 128, device="cuda"), torch.randn(128, device="cuda")
    c = cu(lens)

    def step():
        o, lse = ops.packed_attn(q, k, v, c, causal=True, want_lse=True)
        y, _, rstd = ops.rms_norm(x, w, want_rstd=True)
        return (o, *ops.packed_attn_bwd(g, q, k, v, o, lse, c, causal=True), *ops.rms_norm_bwd(y, x, w, rstd))

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for _ in range(3):
        q.normal_(), x.normal_()
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_side_streams():
    """operands made and used on a stream that is not the default one, two streams at once"""
    from casmtr_amd import ops
    cap = 4096
    c1, ck = cu([1, 1]), cu([cap, cap])
    used = torch.tensor([cap, 77], dtype=torch.int32).cuda()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for i, st in enumerate(streams):
        with torch.cuda.stream(st):
            gen = torch.Generator(device="cuda").manual_seed(i)
            q, k, v = (torch.randn(n, h, 128, device="cuda", generator=gen).to(torch.bfloat16) for n, h in ((2, 8), (2 * cap, 2), (2 * cap, 2)))
            outs = [ops.packed_attn(q * (1 + j), k, v, c1, ck, len_k=used) for j in range(5)]
            got.append((q, k, v, outs))
    torch.cuda.synchronize()
    for q, k, v, outs in got:
        for j, o in enumerate(outs):
            assert torch.equal(o, ops.packed_attn(q * (1 + j), k, v, c1, ck, len_k=used))


def test_offsets_beyond_32_bits():
    """a cache of more than 2^31 elements (and 2^32 bytes): the last sequences read their own keys, prompts and single tokens"""
    from casmtr_amd import ops
    cap, n = 360000, 3
    k = torch.empty(n * cap, 16, 128, device="cuda", dtype=torch.bfloat16).normal_()
    assert k.numel() > 2 ** 31
    used = torch.tensor([10, 3000, 777], dtype=torch.int32).cuda()
    at = [s * cap + torch.arange(u) for s, u in enumerate(used.tolist())]
    few = k[torch.cat(at).cuda()]
    for rows in (1, 40):
        q = torch.randn(n * rows, 16, 128, device="cuda").to(torch.bfloat16)
        got = ops.packed_attn(q, k, k, cu([rows] * n), cu([cap] * n), len_k=used)
        want = ops.packed_attn(q, few, few, cu([rows] * n), cu(used.tolist()))
        # (the keys may be split otherwise: sums in another order, both within (nk + D) 2^-24 of 64 bits, then rounded)
        assert ((got.double() - want.double()).abs() <= 4 * 2.0 ** -8).all() and (got.double() - want.double()).norm() <= 2.0 ** -8 * want.double().norm()
    del k


@pytest.mark.skipif("torch.cuda.device_count() < 2")
def test_other_device():
    from casmtr_amd import ops
    q = torch.randn(9, 2, 32, device="cuda:1")
    c = torch.tensor([0, 9], dtype=torch.int32, device="cuda:1")
    assert torch.equal(ops.packed_attn(q, q, q, c).cpu(), ops.packed_attn(q.to("cuda:0"), q.to("cuda:0"), q.to("cuda:0"), c.to("cuda:0")).cpu())
