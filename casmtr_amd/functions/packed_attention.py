"""autograd.Function of the attention over packed sequences (ops.packed_attn / ops.packed_attn_bwd)."""
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from .. import ops


class PackedAttention(Function):
    """q [Tq,H,D], k, v [Tk,Hk,D], cu_q, cu_k (None: cu_q), len_k (None), causal, scale (None: D ** -0.5) -> [Tq,H,D]; arguments as in
    ops.packed_attn.  The scores are recomputed in the backward pass; what is kept of the forward pass is its output and one number per row."""

    @staticmethod
    def forward(ctx, q, k, v, cu_q, cu_k=None, len_k=None, causal=False, scale=None):
        out, lse = ops.packed_attn(q, k, v, cu_q, cu_k, len_k, causal, scale, want_lse=True)
        ctx.save_for_backward(q, k, v, out, lse, cu_q, cu_k, len_k)
        ctx.args = causal, scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        q, k, v, out, lse, cu_q, cu_k, len_k = ctx.saved_tensors
        # everything about the operands is taken from the tensors as they are NOW: hooks (offloading, compression) may give back other strides
        dq, dk, dv = ops.packed_attn_bwd(grad.contiguous(), q, k, v, out, lse, cu_q, cu_k, len_k, *ctx.args)
        return dq, dk, dv, None, None, None, None, None


packed_attention_op = PackedAttention.apply
