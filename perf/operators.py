"""Workloads of the packed-token operators: attention over packed sequences (`ops.packed_attn`), rotary positions
(`ops.rotary`) and the root-mean-square norm with residual and 8-bit output (`ops.rms_norm`).

`listed()` / `draw()` give the cases, `prepare()` what a program holds before the call, `run()` one pass -- in elementary torch
operations, or, where `own` is true, through this package's operators -- `work()` the bytes and operations the pass cannot do
without, and `exact()` the result from the definitions in 64 bits.

Fields of a case:
  attention  `dtype`, `heads`, `kv_heads`, `dim`; `seqs` sequences, the longest of `longest` keys, the others' lengths spread below it by
             `mix` (0: all alike); `q_len` query rows per sequence (0: as many as keys); `causal`; `cap` > 0: the keys lie in a cache of
             `cap` rows per sequence of which the first ones are valid; `fused`: q, k, v are column ranges of one projection's output
  rotary     `tokens`, `heads`, `kv_heads`, `dim`, `rot` leading columns that rotate, `layout`, `axes` (1: a position, 2: row and
             column), `far` the largest position, `scaled` the factor of a long-context table (1: none)
  norm       `rows`, `width`, `dtype`, `residual`, `quant` ("" or an 8-bit type), `group` columns per scale (0: the whole row)
`op` ending in "_train": the pass goes forward and back and returns the gradients too.
"""
import math
import random

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_F8 = {"e4m3": (torch.float8_e4m3fn, 448.0), "e5m2": (torch.float8_e5m2, 57344.0)}
_TINY = 2.0 ** -126


def _attn(name, dtype, heads, kv_heads, dim, seqs, longest, mix, q_len=0, causal=False, cap=0, fused=False, train=False):
    c = dict(op="attn_train" if train else "attn", dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, seqs=seqs, longest=longest, mix=mix,
             q_len=q_len, causal=causal, cap=cap, fused=fused)
    return dict(c, name=name) if name else c


def _rot(name, dtype, tokens, heads, kv_heads, dim, rot, layout, axes, far, scaled, train=False):
    c = dict(op="rotary_train" if train else "rotary", dtype=dtype, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, rot=rot, layout=layout,
             axes=axes, far=far, scaled=scaled)
    return dict(c, name=name) if name else c


def _norm(name, dtype, rows, width, residual, quant="", group=0, train=False):
    c = dict(op="norm_train" if train else "norm", dtype=dtype, rows=rows, width=width, residual=residual, quant=quant, group=group)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one generated token for each of a few short conversations: nothing but latency
        _attn("attn single tokens", "bf16", 32, 8, 128, 8, 1000, 3, q_len=1, cap=1024),
        # one generated token each against long caches: a read of the caches
        _attn("attn single tokens, long", "bf16", 32, 8, 128, 16, 32768, 5, q_len=1, cap=32768),
        # a batch of prompts of different lengths, packed, straight out of the fused projection
        _attn("attn prompts packed", "bf16", 32, 8, 128, 12, 4095, 7, causal=True, fused=True),
        # one long prompt
        _attn("attn long prompt", "fp16", 32, 8, 128, 1, 16384, 0, causal=True),
        # the backbone's reduced global attention: the 208 x 208 tokens of an 832 x 832 image at 1/4 against 26 x 26 keys, batch of 8
        _attn("attn image tokens", "fp32", 4, 4, 32, 8, 676, 0, q_len=43264),
        # training on packed documents
        _attn("attn train packed", "bf16", 16, 4, 64, 6, 4096, 11, causal=True, train=True),
        # training on the 60 x 80 coarse tokens of two 480 x 640 images
        _attn("attn train image tokens", "fp32", 8, 8, 32, 2, 4800, 0, train=True),
        # one generated token for each of a few conversations, deep into their contexts
        _rot("rotary single tokens", "bf16", 8, 32, 8, 128, 128, "half", 1, 1000000, 8.0),
        # a training step's rotation of half of each head, forward and back
        _rot("rotary train", "bf16", 16384, 32, 8, 128, 64, "interleaved", 1, 16384, 1.0, train=True),
        # one token each for a few conversations, into an 8-bit product
        _norm("norm single tokens e4m3", "bf16", 8, 4096, True, "e4m3"),
        # a long prompt's rows into an 8-bit product with scales for blocks of 128
        _norm("norm prompt e4m3", "bf16", 16384, 8192, True, "e4m3", 128),
        # a training step's norm with the residual stream, forward and back
        _norm("norm train", "bf16", 8192, 4096, True, train=True),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["single", "prompt", "image", "train", "rotary", "rotary_train", "norm", "norm_train"])
    dt = rng.choice(["bf16", "fp16", "bf16", "fp32"])
    if kind in ("single", "prompt", "image", "train"):
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 3, 4, 5, 8])
        dim = rng.choice([16, 32, 40, 64, 80, 96, 128, 128])
        mix = rng.randint(1, 1 << 20)
        if kind == "single":
            longest = _spread(rng, 16, 32768)
            return _attn("", dt, heads, kv, dim, _spread(rng, 1, max(1, min(64, 262144 // longest))), longest, mix, q_len=rng.choice([1, 1, 1, 2, 5]),
                         causal=rng.random() < 0.5, cap=longest + rng.randint(0, 100))
        if kind == "image":
            return _attn("", dt, heads, kv, dim, rng.randint(1, 4), _spread(rng, 20, 1500), mix, q_len=_spread(rng, 100, 12000))
        longest = _spread(rng, 20, 4096)
        seqs = _spread(rng, 1, max(1, min(64, 65536 // longest, (1 << 32) // (heads * longest * longest))))
        return _attn("", dt, heads, kv, dim, seqs, longest, mix, causal=rng.random() < 0.75, fused=rng.random() < 0.5, train=kind == "train")
    if kind in ("rotary", "rotary_train"):
        dim = rng.choice([32, 64, 96, 128])
        kv = rng.choice([1, 2, 4, 8])
        rot = rng.choice([dim, dim, dim // 2, dim // 4])
        return _rot("", dt, _spread(rng, 1, 16384), kv * rng.choice([1, 2, 4]), kv, dim, rot, rng.choice(["half", "interleaved"]), rng.choice([1, 1, 2]),
                    _spread(rng, 100, 4000000), rng.choice([1.0, 4.0, 16.0]), train=kind == "rotary_train")
    rows = _spread(rng, 1, 16384)
    width = min(_spread(rng, 32, 16384), (1 << 26) // rows)
    if kind == "norm_train":
        return _norm("", dt, rows, width, rng.random() < 0.7, train=True)
    quant = rng.choice(["", "e4m3", "e5m2", "e4m3"])
    group = rng.choice([0, 128]) if quant else 0
    return _norm("", dt, rows, -(-width // 128) * 128 if group else width, rng.random() < 0.7, quant, group)


# ------------------------------------------------------------------------------------------------------------ inputs
def _lens(case):
    r = random.Random(case["mix"])
    rest = [case["longest"] if case["mix"] == 0 else max(1, int(case["longest"] * r.random() ** 1.5)) for _ in range(case["seqs"] - 1)]
    at = r.randint(0, case["seqs"] - 1)
    lk = rest[:at] + [case["longest"]] + rest[at:]
    lq = [case["q_len"]] * case["seqs"] if case["q_len"] else list(lk)
    return lq, lk


def _rand(g, dt, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dt)


def _cu(lens):
    t = [0]
    for n in lens:
        t.append(t[-1] + n)
    return torch.tensor(t, dtype=torch.int32, device="cuda")


def _freqs(case):
    """inverse frequencies in 64 bits; a long-context table divides the slow ones by the factor and blends in between"""
    n = case["rot"] // 2 // case["axes"]
    f = 10000.0 ** (-torch.arange(n, dtype=torch.float64) / n)
    turns = 4096.0 * f / (2 * math.pi)
    keep = ((turns - 1.0) / 31.0).clamp(0.0, 1.0)
    f = f * keep + f / case["scaled"] * (1.0 - keep)
    return torch.cat([f] * case["axes"]).cuda(), (0.1 * math.log(case["scaled"]) + 1.0)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    op, dt = case["op"], _DT[case["dtype"]]
    train = op.endswith("_train")
    s = dict(case=case, train=train)
    if op.startswith("attn"):
        lq, lk = _lens(case)
        H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
        s.update(cu_q=_cu(lq), max_q=max(lq), max_k=max(lk), len_k=None, scale=D ** -0.5)
        if case["cap"]:
            s["cu_k"] = _cu([case["cap"]] * case["seqs"])
            s["len_k"] = torch.tensor(lk, dtype=torch.int32, device="cuda")
            tk = case["cap"] * case["seqs"]
        else:
            s["cu_k"], tk = _cu(lk), sum(lk)
        if case["fused"] and not case["q_len"] and not case["cap"]:
            qkv = _rand(g, dt, tk, H + 2 * Hk, D)
            s["q"], s["k"], s["v"] = qkv[:, :H], qkv[:, H:H + Hk], qkv[:, H + Hk:]
        else:
            s["q"], s["k"], s["v"] = _rand(g, dt, sum(lq), H, D), _rand(g, dt, tk, Hk, D), _rand(g, dt, tk, Hk, D)
        if train:
            s["dout"] = _rand(g, dt, sum(lq), H, D)
            for n in "qkv":
                s[n] = s[n].detach().requires_grad_()
    elif op.startswith("rotary"):
        T, D = case["tokens"], case["dim"]
        s["q"], s["k"] = _rand(g, dt, T, case["heads"], D), _rand(g, dt, T, case["kv_heads"], D)
        p = torch.randint(0, case["far"] + 1, (T, 2) if case["axes"] == 2 else (T,), generator=g, device="cuda")
        s["positions"] = p.to(torch.int32)
        s["inv_freq"], s["gain"] = _freqs(case)
        if train:
            s["dq"], s["dk"] = _rand(g, dt, T, case["heads"], D), _rand(g, dt, T, case["kv_heads"], D)
            s["q"].requires_grad_(), s["k"].requires_grad_()
    else:
        R, C = case["rows"], case["width"]
        s["x"] = _rand(g, dt, R, C)
        s["w"] = (1.0 + 0.1 * torch.randn(C, generator=g, device="cuda")).to(dt)
        s["res"] = _rand(g, dt, R, C).mul_(2.0) if case["residual"] else None
        if train:
            s["dy"] = _rand(g, dt, R, C)
            s["dh"] = _rand(g, dt, R, C) if case["residual"] else None
            s["x"].requires_grad_(), s["w"].requires_grad_()
            if case["residual"]:
                s["res"].requires_grad_()
    return s


# ------------------------------------------------------------------------------------------------------------ attention
def _place(cu, total):
    """sequence and place in it of every packed row"""
    t = torch.arange(total, device=cu.device)
    seq = torch.searchsorted(cu[1:].long(), t, right=True).clamp_(max=cu.numel() - 2)
    return seq, t - cu[seq].long()


def _padded(x, cu, longest):
    """packed [T, H, D] -> [B, longest, H, D] in 32 bits; rows past a sequence's end hold some other row"""
    at = (cu[:-1, None].long() + torch.arange(longest, device=cu.device)).clamp_(max=x.shape[0] - 1)
    return x.detach()[at].float()


def _attn_plain(s):
    c = s["case"]
    B, H, Hk, D, G = c["seqs"], c["heads"], c["kv_heads"], c["dim"], c["heads"] // c["kv_heads"]
    Lq, Lk = s["max_q"], s["max_k"]
    nq = (s["cu_q"][1:] - s["cu_q"][:-1]).long()
    nk = s["len_k"].long() if s["len_k"] is not None else (s["cu_k"][1:] - s["cu_k"][:-1]).long()
    group = lambda x: x.view(B, Lq, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * Lq, D)
    each = lambda x: x.permute(0, 2, 1, 3).contiguous()
    q, k, v = group(_padded(s["q"], s["cu_q"], Lq)), each(_padded(s["k"], s["cu_k"], Lk)), each(_padded(s["v"], s["cu_k"], Lk))
    i, j = torch.arange(Lq, device=q.device)[:, None], torch.arange(Lk, device=q.device)
    see = (i < nq[:, None, None]) & (j < nk[:, None, None])
    if c["causal"]:
        see = see & (j <= i + (nk - nq)[:, None, None])
    p = ((q * s["scale"]) @ k.transpose(-1, -2)).view(B, Hk, G, Lq, Lk)
    p.masked_fill_(~see[:, None, None], -math.inf)
    m = p.amax(-1, keepdim=True)
    p.sub_(torch.where(m == -math.inf, torch.zeros_like(m), m)).exp_()
    p.div_(p.sum(-1, keepdim=True).clamp_(min=1e-37))
    p = p.view(B, Hk, G * Lq, Lk)
    o = p @ v
    seq, at = _place(s["cu_q"], s["q"].shape[0])
    back = lambda x: x.view(B, Hk, G, Lq, D).permute(0, 3, 1, 2, 4).reshape(B, Lq, H, D)[seq, at].to(s["q"].dtype)
    if not s["train"]:
        return back(o)
    do = group(_padded(s["dout"], s["cu_q"], Lq))
    do = torch.where((torch.arange(Lq, device=q.device) < nq[:, None]).view(B, 1, 1, Lq).expand(B, Hk, G, Lq).reshape(B, Hk, G * Lq, 1), do, torch.zeros_like(do))
    dv = p.transpose(-1, -2) @ do
    ds = do @ v.transpose(-1, -2)
    ds.sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(s["scale"])
    dq, dk = ds @ k, ds.transpose(-1, -2) @ q
    seq, at = _place(s["cu_k"], s["k"].shape[0])
    kback = lambda x: x.permute(0, 2, 1, 3)[seq, at].to(s["q"].dtype)
    return [back(o), back(dq), kback(dk), kback(dv)]


def _attn_own(s):
    if s["train"]:
        from casmtr_amd.functions.packed_attention import packed_attention_op
        o = packed_attention_op(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], s["len_k"], s["case"]["causal"], s["scale"])
        return [o, *torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["dout"])]
    from casmtr_amd import ops
    return ops.packed_attn(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], len_k=s["len_k"], causal=s["case"]["causal"], scale=s["scale"])


# ------------------------------------------------------------------------------------------------------------ rotary positions
def _turn(x, cos, sin, layout):
    n = cos.shape[-1]
    y = x.detach().float()
    r, tail = y[..., :2 * n], y[..., 2 * n:]
    a, b = (r[..., :n], r[..., n:]) if layout == "half" else (r[..., 0::2], r[..., 1::2])
    u, w = a * cos - b * sin, b * cos + a * sin
    r = torch.cat([u, w], -1) if layout == "half" else torch.stack([u, w], -1).flatten(-2)
    return torch.cat([r, tail], -1).to(x.dtype)


def _rotary_plain(s):
    c, p = s["case"], s["positions"].double()
    n = s["inv_freq"].numel()
    p = p.repeat_interleave(n // 2, dim=1) if c["axes"] == 2 else p[:, None]
    a = p * s["inv_freq"]
    cos, sin = (a.cos() * s["gain"]).float()[:, None], (a.sin() * s["gain"]).float()[:, None]
    y = [_turn(s["q"], cos, sin, c["layout"]), _turn(s["k"], cos, sin, c["layout"])]
    if s["train"]:
        y += [_turn(s["dq"], cos, -sin, c["layout"]), _turn(s["dk"], cos, -sin, c["layout"])]
    return y


def _rotary_own(s):
    if s["train"]:
        from casmtr_amd.functions.rotary import rotary_op
        q, k = rotary_op(s["q"], s["k"], s["positions"], s["inv_freq"], s["case"]["layout"], s["gain"])
        return [q, k, *torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))]
    from casmtr_amd import ops
    return list(ops.rotary(s["q"], s["k"], s["positions"], s["inv_freq"], layout=s["case"]["layout"], gain=s["gain"]))


# ------------------------------------------------------------------------------------------------------------ norm
def _norm_plain(s):
    c, dt = s["case"], s["x"].dtype
    h = s["x"].detach().float()
    if c["residual"]:
        h = (h + s["res"].detach().float()).to(dt).float()
    w = s["w"].detach().float()
    r = torch.rsqrt((h * h).mean(-1, keepdim=True) + 1e-6)
    n = h * r
    y = n * w
    hs = [h.to(dt)] if c["residual"] else []
    if s["train"]:
        dy = s["dy"].float()
        g = dy * w
        dx = (g - n * (g * n).mean(-1, keepdim=True)) * r
        dw = (dy * n).sum(0).to(dt)
        if c["residual"]:
            dx = (dx + s["dh"].float()).to(dt)
            return [y.to(dt), *hs, dx, dw, dx]
        return [y.to(dt), dx.to(dt), dw]
    if not c["quant"]:
        return [y.to(dt), *hs]
    t, top = _F8[c["quant"]]
    y = y.view(c["rows"], -1, c["group"] or c["width"])
    scale = (y.abs().amax(-1, keepdim=True) / top).clamp_(min=_TINY)
    return [(y / scale).clamp_(-top, top).to(t).view(c["rows"], -1), scale[..., 0], *hs]


def _norm_own(s):
    c = s["case"]
    if s["train"]:
        from casmtr_amd.functions.rms_norm import rms_norm_op
        if c["residual"]:
            y, h = rms_norm_op(s["x"], s["w"], 1e-6, s["res"])
            dx, dw, dr = torch.autograd.grad((y, h), (s["x"], s["w"], s["res"]), (s["dy"], s["dh"]))
            return [y, h, dx, dw, dr]
        y = rms_norm_op(s["x"], s["w"], 1e-6)
        return [y, *torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])]
    from casmtr_amd import ops
    if c["quant"]:
        q, scale, h = ops.rms_norm_quant(s["x"], s["w"], 1e-6, residual=s["res"], dtype=_F8[c["quant"]][0], group=c["group"] or None)
        return [t for t in (q, scale.view(c["rows"], -1), h) if t is not None]
    return [t for t in ops.rms_norm(s["x"], s["w"], 1e-6, residual=s["res"]) if t is not None]


def run(state):
    op = state["case"]["op"]
    if op.startswith("attn"):
        return _attn_own(state) if own else _attn_plain(state)
    if op.startswith("rotary"):
        return _rotary_own(state) if own else _rotary_plain(state)
    return _norm_own(state) if own else _norm_plain(state)


# ------------------------------------------------------------------------------------------------------------ work
def _pairs(case):
    """(query, key) pairs that see each other, of one head"""
    n = 0
    for a, b in zip(*_lens(case)):
        if not case["causal"]:
            n += a * b
        else:   # row i sees the keys up to i + b - a
            first = max(0, a - b)
            n += (a - first) * b - (a - first) * (a - first - 1) // 2
    return n


def work(case):
    e = _DT[case["dtype"]].itemsize
    if case["op"].startswith("attn"):
        lq, lk = _lens(case)
        q, kv = sum(lq) * case["heads"] * case["dim"] * e, sum(lk) * case["kv_heads"] * case["dim"] * e
        train = case["op"] == "attn_train"
        return {"bytes": (4 * q + 4 * kv) if train else (2 * q + 2 * kv), "flops": (14 if train else 4) * _pairs(case) * case["heads"] * case["dim"]}
    if case["op"].startswith("rotary"):
        x = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"] * e
        passes = 2 if case["op"] == "rotary_train" else 1
        return {"bytes": passes * 2 * x + 4 * case["tokens"] * case["axes"], "flops": passes * 3 * x // e * case["rot"] // case["dim"]}
    n = case["rows"] * case["width"]
    r = int(case["residual"])
    if case["op"] == "norm_train":
        return {"bytes": (4 + 3 * r) * n * e + 2 * case["width"] * e, "flops": 14 * n}
    out = n + 4 * case["rows"] * (case["width"] // case["group"] if case["group"] else 1) if case["quant"] else n * e
    return {"bytes": (1 + 2 * r) * n * e + out + case["width"] * e, "flops": 6 * n}


# ------------------------------------------------------------------------------------------------------------ 64 bits
def _attn_exact(case, s):
    """sequence by sequence and head by head from o_i = sum_j softmax_j(scale q_i . k_j) v_j"""
    H, Hk, G = case["heads"], case["kv_heads"], case["heads"] // case["kv_heads"]
    lq, lk = _lens(case)
    q, k, v = (s[n].detach() for n in "qkv")
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    train = case["op"] == "attn_train"
    if train:
        dq, dk, dv = (torch.zeros(t.shape, dtype=torch.float64, device=q.device) for t in (q, k, v))
    q0 = k0 = 0
    for a, b in zip(lq, lk):
        hidden = None
        if case["causal"]:
            hidden = torch.ones(a, b, dtype=torch.bool, device=q.device).triu_(b - a + 1)
        for h in range(H):
            qh, kh, vh = q[q0:q0 + a, h].double(), k[k0:k0 + b, h // G].double(), v[k0:k0 + b, h // G].double()
            x = qh @ kh.t()
            x *= s["scale"]
            if hidden is not None:
                x.masked_fill_(hidden, -math.inf)
            p = torch.softmax(x, -1)
            if a > b and case["causal"]:
                p[:a - b] = 0.0
            del x
            out[q0:q0 + a, h] = p @ vh
            if train:
                g = s["dout"][q0:q0 + a, h].double()
                dv[k0:k0 + b, h // G] += p.t() @ g
                ds = p * (g @ vh.t() - (g * out[q0:q0 + a, h]).sum(1, keepdim=True)) * s["scale"]
                dq[q0:q0 + a, h] = ds @ kh
                dk[k0:k0 + b, h // G] += ds.t() @ qh
        q0, k0 = q0 + a, k0 + (case["cap"] or b)
    return [out, dq, dk, dv] if train else out


def _rotary_exact(case, s):
    n = s["inv_freq"].numel()
    axis = torch.arange(n, device="cuda") * case["axes"] // n
    pos = s["positions"].double().view(case["tokens"], case["axes"])
    z = torch.polar(torch.full((case["tokens"], n), s["gain"], dtype=torch.float64, device="cuda"), pos[:, axis] * s["inv_freq"])[:, None]

    def turned(x, z):
        x = x.detach().double()
        r = x[..., :2 * n]
        pair = r.unflatten(-1, (2, n)).transpose(-1, -2) if case["layout"] == "half" else r.unflatten(-1, (n, 2))
        w = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * z)
        return torch.cat([(w.transpose(-1, -2) if case["layout"] == "half" else w).flatten(-2), x[..., 2 * n:]], -1)

    y = [turned(s["q"], z), turned(s["k"], z)]
    return y + [turned(s["dq"], z.conj()), turned(s["dk"], z.conj())] if case["op"] == "rotary_train" else y


def _norm_exact(case, s):
    h = s["x"].detach().double()
    if case["residual"]:
        h = (h + s["res"].detach().double()).to(s["x"].dtype).double()   # the norm is of the stream as it is handed on, in its own type
    w = s["w"].detach().double()
    norm = torch.sqrt(h.square().sum(1, keepdim=True) / case["width"] + 1e-6)
    y = h / norm * w
    hs = [h] if case["residual"] else []
    if case["op"] == "norm_train":
        dy = s["dy"].double()
        # d(h_i / norm)/dh_j = (delta_ij - h_i h_j / (width norm^2)) / norm
        dx = (dy * w - h * ((dy * w * h).sum(1, keepdim=True) / (case["width"] * norm * norm))) / norm
        dw = (dy * h / norm).sum(0)
        if case["residual"]:
            dx = dx + s["dh"].double()
            return [y, *hs, dx, dw, dx]
        return [y, dx, dw]
    if not case["quant"]:
        return [y, *hs]
    top = _F8[case["quant"]][1]
    y = y.view(case["rows"], -1, case["group"] or case["width"])
    scale = (y.abs().amax(-1, keepdim=True) / top).clamp(min=_TINY)
    return [(y / scale).view(case["rows"], -1), scale[..., 0], *hs]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"].startswith("attn"):
        return _attn_exact(case, s)
    return _rotary_exact(case, s) if case["op"].startswith("rotary") else _norm_exact(case, s)
