"""CPU: what the packed-token autograd functions hand to their gradients' kernels where saved tensors come back through hooks (offloading,
compression): the operands as they ARE then, not as the forward pass had them.  The library calls are replaced by a recorder."""
import pytest
import torch

from casmtr_amd import _lib, ops


class Recorder:
    """stands for the library: no kernel runs, every call is kept"""

    def __init__(self):
        self.calls = {}

    def __getattr__(self, name):
        def call(*args):
            self.calls[name] = args
            return 4096 if name.endswith("ws_floats") else 0
        return call


@pytest.fixture
def stub(monkeypatch):
    rec = Recorder()
    monkeypatch.setattr(_lib, "lib", lambda: rec)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops, "_on", lambda device: ops._SAME_DEVICE)
    monkeypatch.setattr(torch.Tensor, "is_cuda", True, raising=False)
    return rec


def _qkv(T=10, H=4, Hk=2, D=16):
    qkv = torch.randn(T, H + 2 * Hk, D).bfloat16().requires_grad_()
    return qkv, (qkv[:, :H], qkv[:, H:H + Hk], qkv[:, H + Hk:]), torch.tensor([0, T], dtype=torch.int32)


def _hooked(change):
    """-> the context, and what the hook gave back by address"""
    given = {}

    def unpack(t):
        t = change(t)
        given[t.data_ptr()] = t
        return t

    return torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(memory_format=torch.contiguous_format), unpack), given


def _attention_strides(rec, given):
    a = rec.calls["casmtr_packed_attn_bwd"]
    st = a[19:25]
    for i, (ptr, at) in enumerate(((a[1], 0), (a[2], 2), (a[3], 4))):
        t = given[ptr]
        assert tuple(st[at:at + 2]) == t.stride()[:2], f"operand {i}: strides {st[at:at + 2]} of a tensor with {t.stride()}"


def test_attention_strides_follow_the_saved_tensors(stub):
    from casmtr_amd.functions.packed_attention import packed_attention_op
    _, (q, k, v), c = _qkv()
    ctx, given = _hooked(lambda t: t)
    with ctx:
        o = packed_attention_op(q, k, v, c, None, None, True)
    o.sum().backward()
    _attention_strides(stub, given)
    # copies that are laid out head by head
    _, (q, k, v), c = _qkv()
    ctx, given = _hooked(lambda t: t.transpose(0, 1).contiguous().transpose(0, 1) if t.dim() == 3 and t.shape[1] == 2 else t)
    with ctx:
        o = packed_attention_op(q, k, v, c, None, None, True)
    o.sum().backward()
    _attention_strides(stub, given)


@pytest.mark.parametrize("change", [lambda t: t.float() if t.dim() == 3 and t.shape[1] == 2 else t,                       # another type: k and v
                                    lambda t: t.long() if t.dtype == torch.int32 else t,                                   # the bounds
                                    lambda t: t.half() if t.dtype == torch.float32 else t,                                 # lse
                                    lambda t: t[:-1] if t.dim() == 3 else t])                                              # fewer rows
def test_attention_refuses_changed_tensors(stub, change):
    from casmtr_amd.functions.packed_attention import packed_attention_op
    _, (q, k, v), c = _qkv()
    ctx, _ = _hooked(change)
    with ctx:
        o = packed_attention_op(q, k, v, c, None, None, True)
    with pytest.raises(RuntimeError):
        o.sum().backward()
    assert "casmtr_packed_attn_bwd" not in stub.calls


@pytest.mark.parametrize("change", [lambda t: t.float() if t.dtype == torch.bfloat16 and t.dim() == 2 else t, lambda t: t[:-1] if t.dim() == 2 else t,
                                    lambda t: t.half() if t.dtype == torch.float32 else t])
def test_norm_refuses_changed_tensors(stub, change):
    from casmtr_amd.functions.rms_norm import rms_norm_op
    x, w = torch.randn(6, 32).bfloat16().requires_grad_(), torch.ones(32).bfloat16().requires_grad_()
    ctx, _ = _hooked(change)
    with ctx:
        y = rms_norm_op(x, w)
    with pytest.raises(RuntimeError):
        y.sum().backward()
    assert "casmtr_rms_norm_bwd" not in stub.calls


def test_norm_strides_follow_the_saved_tensors(stub):
    from casmtr_amd.functions.rms_norm import rms_norm_op
    wide = torch.randn(6, 50).requires_grad_()
    w = torch.ones(32).requires_grad_()
    ctx, given = _hooked(lambda t: t)
    with ctx:
        y = rms_norm_op(wide[:, 3:35], w)
    y.sum().backward()
    a = stub.calls["casmtr_rms_norm_bwd"]
    assert a[12] == given[a[2]].stride(0) == 32


def test_rotary_refuses_changed_tensors(stub):
    from casmtr_amd.functions.rotary import rotary_op
    q = torch.randn(6, 2, 16, requires_grad=True)
    ctx, _ = _hooked(lambda t: t.float())
    with ctx:
        oq, _ = rotary_op(q, None, torch.arange(6), ops.rotary_freqs(16, device="cpu")[0])
    stub.calls.clear()
    with pytest.raises(RuntimeError):
        oq.sum().backward()
    assert "casmtr_rotary_fwd" not in stub.calls
