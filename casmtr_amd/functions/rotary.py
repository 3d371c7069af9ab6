"""autograd.Function of the rotary positions (ops.rotary): the gradient is the turn by the opposite angle."""
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from .. import ops


class Rotary(Function):
    """q [T,Hq,D], k [T,Hk,D] or None, positions [T] or [T,2], inv_freq fp64 [n], layout, gain -> q', k'"""

    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, layout="half", gain=1.0):
        ctx.save_for_backward(positions, inv_freq)
        ctx.layout, ctx.gain = layout, gain
        return ops.rotary(q, k, positions, inv_freq, layout, gain)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        positions, inv_freq = ctx.saved_tensors
        dq, dk = ops.rotary(dq.contiguous(), None if dk is None else dk.contiguous(), positions, inv_freq, ctx.layout, ctx.gain, inverse=True)
        return dq, dk, None, None, None, None


rotary_op = Rotary.apply
