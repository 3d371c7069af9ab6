"""autograd.Function of the RMS norm with the residual's addition (ops.rms_norm / ops.rms_norm_bwd)."""
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from .. import ops


class RMSNorm(Function):
    """x [..., C], weight [C], eps, residual like x or None -> y, with a residual (y, h = x + residual).  The gradient of h (the stream that the
    next block adds to) is folded into the norm's own gradient."""

    @staticmethod
    def forward(ctx, x, weight, eps=1e-6, residual=None):
        y, h, rstd = ops.rms_norm(x, weight, eps, residual, want_rstd=True)
        ctx.has_residual = residual is not None
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(h if ctx.has_residual else x, weight, rstd)
        return (y, h) if ctx.has_residual else y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh=None):
        h, weight, rstd = ctx.saved_tensors
        if dy is None:   # only the stream was used
            return dh, None, None, dh
        rows = lambda g: None if g is None else g.contiguous()
        dx, dw = ops.rms_norm_bwd(rows(dy), h, weight, rstd, rows(dh))   # (checked again: hooks on saved tensors may give back others)
        return dx, dw, None, dx if ctx.has_residual else None


rms_norm_op = RMSNorm.apply
