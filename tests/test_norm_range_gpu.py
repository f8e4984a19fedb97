"""Gradients of rms_norm_fn over rows of any size that float32 holds the squares of.  Tolerances are those of test_rms_norm_gpu.py."""
import pytest
import torch

from test_rms_norm_gpu import close


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [40, 1500, 20000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("power", [-47, -30, 0, 30, 42, 50])
def test_gradients_of_large_and_small_rows(pkg, gpu_device, dim, dtype, power):
    """Rows of 2^power: the gradient is as many times smaller, and nothing on the way to it may be no normal number (the root's third
    power was none from 2^42 on, and infinite below 2^-42)."""
    r = torch.Generator().manual_seed(dim)
    x = (torch.randn(5, dim, generator=r) * 2.0 ** power).to(dtype).to(gpu_device).requires_grad_()
    w = (torch.rand(dim, generator=r) + 0.5).to(gpu_device).requires_grad_()
    dy = torch.randn(5, dim, generator=r).to(dtype).to(gpu_device)
    dx, dw = torch.autograd.grad(pkg.rms_norm_fn(x, w, eps=0.0), [x, w], dy)
    h, wdy = x.detach().double(), w.detach().double() * dy.double()
    inv = h.square().mean(-1, keepdim=True).rsqrt()
    want = inv * wdy - h * inv ** 3 * (h * wdy).mean(-1, keepdim=True)
    size = (inv * wdy).abs() + (h * inv ** 3).abs() * (h * wdy).abs().mean(-1, keepdim=True)
    close(dx, want, dtype, dim, size)
    terms = dy.double() * h * inv
    close(dw, terms.sum(0), torch.float32, dim + 512 * 5, terms.abs().sum(0))
