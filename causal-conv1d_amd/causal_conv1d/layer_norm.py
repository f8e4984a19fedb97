"""The layer norm with the residual's addition: `layer_norm_fn` (differentiable).

    h = x + residual                 summed in float32, rounded once to residual's dtype
    y = (h - mean(h)) * rsqrt(mean((h - mean(h))^2) + eps) * weight + bias

As with the root-mean-square norm, the norm is taken of h as it is stored.  x and residual are (..., dim); residual and weight
are each of x's dtype or float32, bias of weight's.  There is no host path.  `layer_norm_ref` states the operator in plain PyTorch.
"""
import torch
from torch.compiler import is_compiling

import causal_conv1d_cuda as _ext              # loading it registers the ops

_fwd = torch.ops.DaoAILab._layer_norm_fwd_cpp
_bwd = torch.ops.DaoAILab._layer_norm_bwd_cpp


class LayerNormFn(torch.autograd.Function):
    """Saves what was normalised (h, or x without a residual), each row's mean and factor, and the weight."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, eps):
        y, h, stats = _fwd(x, weight, bias, residual, eps, True)
        ctx.x_dtype = x.dtype
        ctx.save_for_backward(x if residual is None else h, stats, weight)
        ctx.set_materialize_grads(False)
        return y if residual is None else (y, h)

    @staticmethod
    def backward(ctx, dy, dh=None):
        h, stats, weight = ctx.saved_tensors
        needs_residual = ctx.needs_input_grad[3]
        if dy is None:                                   # only the sum was used
            if dh is None:
                return (None,) * 5
            dy = torch.zeros(h.shape, dtype=ctx.x_dtype, device=h.device)
        dx, dresidual, dweight, dbias = _bwd(h, stats, weight, dy, dh, ctx.needs_input_grad[2])
        if not needs_residual:
            dresidual = None
        elif dx.dtype == h.dtype:
            dresidual = dx
        return (dx if ctx.needs_input_grad[0] else None, dweight if ctx.needs_input_grad[1] else None,
                dbias if ctx.needs_input_grad[2] else None, dresidual, None)


def layer_norm_fn(x, weight, bias=None, residual=None, eps=1e-5):
    """y, or (y, h) with a residual; y has x's dtype, h = x + residual has residual's."""
    if not is_compiling():
        res = _ext._layer_norm_call(x, weight, bias, residual, eps)
        if res is not NotImplemented:
            return res
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual)):
        return LayerNormFn.apply(x, weight, bias, residual, eps)
    y, h, _ = _fwd(x, weight, bias, residual, eps, False)
    return y if residual is None else (y, h)


def layer_norm_ref(x, weight, bias=None, residual=None, eps=1e-5):
    """The operator in plain PyTorch on any device, in float32 (float64 for float64 tensors)."""
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    h = x if residual is None else (x.to(wide) + residual.to(wide)).to(residual.dtype)
    f = h.to(wide)
    f = f - f.mean(-1, keepdim=True)
    y = f * torch.rsqrt(f.square().mean(-1, keepdim=True) + eps) * weight.to(wide)
    y = (y if bias is None else y + bias.to(wide)).to(x.dtype)
    return y if residual is None else (y, h)
