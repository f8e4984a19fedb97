"""The root-mean-square norm with the residual's addition: `rms_norm_fn` (differentiable), its inference form with an
output in 8 bits `rms_norm_quant_fn`, and such rows read back, `dequantize_rows`.

    h = x + residual                 summed in float32, rounded once to residual's dtype
    y = h * rsqrt(mean(h^2) + eps) * weight

The norm is taken of h as it is stored, so that the gradients, which read h again, are those of what the forward
computed.  x and residual are (..., dim); residual and weight are each of x's dtype or float32.  There is no host path.
`rms_norm_ref` states the operator in plain PyTorch.
"""
import torch
from torch.compiler import is_compiling

import causal_conv1d_cuda as _ext              # loading it registers the ops

_fwd = torch.ops.DaoAILab._rms_norm_fwd_cpp
_bwd = torch.ops.DaoAILab._rms_norm_bwd_cpp
_quant = torch.ops.DaoAILab._rms_norm_quant_cpp
_dequantize = torch.ops.DaoAILab._dequantize_rows_cpp


class RMSNormFn(torch.autograd.Function):
    """Saves what was normalised (h, or x without a residual) and the weight."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, h = _fwd(x, weight, residual, eps)
        ctx.eps, ctx.x_dtype = eps, x.dtype
        ctx.save_for_backward(x if residual is None else h, weight)
        ctx.set_materialize_grads(False)
        return y if residual is None else (y, h)

    @staticmethod
    def backward(ctx, dy, dh=None):
        h, weight = ctx.saved_tensors
        needs_residual = ctx.needs_input_grad[2]
        if dy is None:                                   # only the sum was used
            if dh is None:
                return None, None, None, None
            dy = torch.zeros(h.shape, dtype=ctx.x_dtype, device=h.device)
        dx, dresidual, dweight = _bwd(h, weight, dy, dh, ctx.eps)
        if not needs_residual:
            dresidual = None
        elif dx.dtype == h.dtype:
            dresidual = dx
        return dx if ctx.needs_input_grad[0] else None, dweight if ctx.needs_input_grad[1] else None, dresidual, None


def rms_norm_fn(x, weight, residual=None, eps=1e-5):
    """y, or (y, h) with a residual; y has x's dtype, h = x + residual has residual's."""
    if not is_compiling():
        res = _ext._rms_norm_call(x, weight, residual, eps)
        if res is not NotImplemented:
            return res
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (residual is not None and residual.requires_grad)):
        return RMSNormFn.apply(x, weight, residual, eps)
    y, h = _fwd(x, weight, residual, eps)
    return y if residual is None else (y, h)


def rms_norm_quant_fn(x, weight, residual=None, eps=1e-5):
    """(y8, scales), or (y8, scales, h) with a residual: y8 (..., dim) float8_e4m3fn, scales (...) float32 with
    y8 the code next to y / scales[..., None] and scales = max|y| / 448 of each row.  No backward."""
    if not is_compiling():
        res = _ext._rms_norm_quant_call(x, weight, residual, eps)
        if res is not NotImplemented:
            return res
    y8, scales, h = _quant(x, weight, residual, eps)
    return (y8, scales) if residual is None else (y8, scales, h)


def dequantize_rows(y8, scales, dtype=torch.bfloat16):
    """y8 (..., dim) float8_e4m3fn times scales (...), as `dtype`.  No backward."""
    if not is_compiling():
        res = _ext._dequantize_rows_call(y8, scales, dtype)
        if res is not NotImplemented:
            return res
    return _dequantize(y8, scales, dtype)


def rms_norm_ref(x, weight, residual=None, eps=1e-5):
    """The operator in plain PyTorch on any device, in float32 (float64 for float64 tensors)."""
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    h = x if residual is None else (x.to(wide) + residual.to(wide)).to(residual.dtype)
    f = h.to(wide)
    y = (f * torch.rsqrt(f.square().mean(-1, keepdim=True) + eps) * weight.to(wide)).to(x.dtype)
    return y if residual is None else (y, h)
