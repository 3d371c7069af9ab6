"""The packed-token autograd functions under saved-tensor hooks: the same gradients, bit for bit, whatever layout the saved copies have."""
import pytest
import torch

pytestmark = pytest.mark.gpu

HOOKS = {
    "contiguous copies": lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(memory_format=torch.contiguous_format), lambda t: t),
    "on the host": lambda: torch.autograd.graph.save_on_cpu(),
    "head-major copies": lambda: torch.autograd.graph.saved_tensors_hooks(
        lambda t: t.detach().transpose(0, 1).contiguous() if t.dim() == 3 and t.shape[1] == 2 else t.detach(),
        lambda t: t.transpose(0, 1) if t.dim() == 3 and t.shape[0] == 2 else t),
}


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("H,Hk,D", [(8, 2, 128), (4, 2, 64), (6, 2, 40)])
@pytest.mark.parametrize("hook", list(HOOKS))
def test_attention_of_a_fused_projection(hook, H, Hk, D, dt):
    from casmtr_amd.functions.packed_attention import packed_attention_op
    T = 301
    qkv = torch.randn(T, H + 2 * Hk, D, device="cuda").to(dt).requires_grad_()
    c = torch.tensor([0, 90, 91, 301], dtype=torch.int32, device="cuda")
    g = torch.randn(T, H, D, device="cuda").to(dt)

    def gradient():
        return torch.autograd.grad(packed_attention_op(*qkv.split([H, Hk, Hk], 1), c, None, None, True), qkv, g)[0]

    want = gradient()
    with HOOKS[hook]():
        got = gradient()
    assert torch.equal(got, want) and want.abs().sum() > 0


@pytest.mark.parametrize("hook", ["contiguous copies", "on the host"])
def test_norm_and_rotary(hook):
    from casmtr_amd import ops
    from casmtr_amd.functions.rms_norm import rms_norm_op
    from casmtr_amd.functions.rotary import rotary_op
    wide = torch.randn(77, 300, device="cuda").bfloat16().requires_grad_()
    w = torch.randn(256, device="cuda").bfloat16().requires_grad_()
    freq, _ = ops.rotary_freqs(32)
    pos = torch.arange(77, device="cuda")

    def gradients():
        y = rms_norm_op(wide[:, 5:261], w)
        q, k = rotary_op(*y.view(77, 8, 32).split([6, 2], 1), pos, freq)
        return torch.autograd.grad((q.float().square().sum() + k.float().sum()), (wide, w))

    want = gradients()
    with HOOKS[hook]():
        got = gradients()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
