"""Layer norm of Gaussian features, with the residual sum before it: what stands between the attention layers that make the
features.  No counterpart in the reference, whose features arrive finished; the kernels live in libg2v_hip.so and are reached
through ``_C`` on the caller's current stream.
"""
import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _C
from .attention import _differentiated

__all__ = ["layer_norm", "PyLayerNorm"]


class _LayerNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, eps):
        y, total, stats = _C.layer_norm_forward(x, weight, bias, residual, eps, True)
        ctx.save_for_backward(x if residual is None else total, weight, stats)
        ctx.bias_dtype = None if bias is None else bias.dtype
        ctx.set_materialize_grads(False)
        return y if residual is None else (y, total)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y, grad_sum=None):
        x, weight, stats = ctx.saved_tensors
        need = ctx.needs_input_grad
        if grad_y is None:    # the sum alone was used
            return grad_sum if need[0] else None, None, None, grad_sum if need[3] else None, None
        dx, dw, db = _C.layer_norm_backward(grad_y, x, weight, stats, grad_sum, (need[1], need[2]), ctx.bias_dtype)
        return dx if need[0] else None, dw, db, dx if need[3] else None, None


def layer_norm(x, weight=None, bias=None, *, residual=None, eps=1e-5):
    """Layer norm over the last dimension of x (..., C), float32 or bfloat16, C at most 8192, in one pass.

    (x - mean) (variance + eps)^-1/2 weight + bias, with weight and bias (C,) float32 or bfloat16 (both of one type, whatever x's), None for
    ones and zeros.  With ``residual`` (x's shape and type) the sum x + residual, rounded to x's type, is normed and returned too:
    (y, x + residual), the residual stream of a stack of layers.  Any strides (rows of unit stride are read in place); y and the sum
    are contiguous and of x's type.  Sums are float32 and the variance is that of the differences to the mean.

    Gradients flow to x, residual, weight and bias, the weights' summed over the rows in float32 and in a fixed order.
    Gradients of gradients and forward-mode derivatives are refused."""
    if _differentiated(x, weight, bias, residual):
        return _LayerNormFunction.apply(x, weight, bias, residual, eps)
    y, total, _ = _C.layer_norm_forward(x, weight, bias, residual, eps)
    return y if residual is None else (y, total)


class PyLayerNorm(nn.Module):
    """layer_norm with a weight and a bias; parameters and their names are those of torch.nn.LayerNorm(embed_dim)."""

    def __init__(self, embed_dim, eps=1e-5, *, bias=True, device="cuda", dtype=torch.float32):
        super().__init__()
        self.embed_dim, self.eps = embed_dim, eps
        self.weight = nn.Parameter(torch.ones(embed_dim, device=device, dtype=dtype))
        self.bias = nn.Parameter(torch.zeros(embed_dim, device=device, dtype=dtype)) if bias else None

    def forward(self, x, residual=None):
        """The norm of x (..., embed_dim), or (norm, sum) of x + residual."""
        return layer_norm(x, self.weight, self.bias, residual=residual, eps=self.eps)
