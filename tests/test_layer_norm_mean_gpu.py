"""Layer norm of rows whose mean is far larger than their spread: the mean's own rounding must not be taken for spread.

With c the mean's size, a sum of up to 2^15 numbers in trees leaves it off by up to 64 2^-24 c.  The differences h - mean are exact where h is within a factor of 2 of
the mean; their own mean, 64 2^-24 of that offset wrong, is taken off: 2^-36 c is left of it, and 64 2^-24 of the differences' size."""
import pytest
import torch

from causal_conv1d.layer_norm import layer_norm_ref
from test_layer_norm_gpu import make, run

BF16, FP32 = torch.bfloat16, torch.float32
pytestmark = pytest.mark.gpu
N_EFF = 64 * 2.0 ** -24


@pytest.mark.parametrize("dim", [7, 300, 700, 1001, 2560, 5120, 9000, 17000])
@pytest.mark.parametrize("value", [37.3, 10001.0, -100003.0])
def test_constant_rows(pkg, gpu_device, dim, value):
    """No spread: y is the bias, and nothing comes back to x along it."""
    eps = 1e-5
    s = make(gpu_device, 4, dim, FP32, None, FP32)
    s["x"] = torch.full_like(s["x"], value)
    got = run(pkg, s, eps)
    left = 2.0 ** -36 * abs(s["x"][0, 0].item()) * eps ** -0.5       # of a normalised value
    assert ((got["y"] - s["bias"]).abs() <= left * s["weight"].abs() + 2.0 ** -24 * s["bias"].abs()).all()
    assert (got["dweight"].abs() <= left * s["dy"].abs().sum(0)).all()


@pytest.mark.parametrize("dim", [300, 1001, 2560, 17000])
@pytest.mark.parametrize("offset", [1000.0, 1e5])
@pytest.mark.parametrize("residual", [None, FP32])
def test_spread_far_below_the_mean(pkg, gpu_device, dim, offset, residual):
    """As near to 64 bits as rows without an offset are."""
    s = make(gpu_device, 9, dim, FP32, residual, FP32, offset=offset)
    got = run(pkg, s)
    h = (s["x"] if residual is None else got["h"]).double().requires_grad_()
    w, b = s["weight"].double().requires_grad_(), s["bias"].double().requires_grad_()
    y = layer_norm_ref(h, w, b)
    dh, dw, db = torch.autograd.grad(y, [h, w, b], s["dy"].double())
    r = 1 / (h.detach().var(-1, unbiased=False, keepdim=True) + 1e-5).sqrt()
    unit = ((h.detach() - h.detach().mean(-1, keepdim=True)) * r).abs()
    wdy, rel = w.detach().abs() * s["dy"].double().abs(), N_EFF + 2.0 ** -36 * offset * r
    mean = wdy.mean(-1, keepdim=True)
    assert ((got["y"] - y.detach()).abs() <= rel * (1 + unit) * w.detach().abs() + N_EFF * b.detach().abs() + 2.0 ** -24 * y.detach().abs()).all()
    bound = rel * r * (wdy + mean + (1 + unit) * (wdy * (1 + unit)).mean(-1, keepdim=True))
    want = dh
    if residual is not None:
        want, bound = dh + s["dh"].double(), bound + N_EFF * s["dh"].double().abs()
    assert ((got["dx"] - want).abs() <= bound + 2.0 ** -24 * want.abs()).all()
    assert ((got["dweight"] - dw).abs() <= (s["dy"].double().abs() * (1 + unit) * (rel + 80 * 2.0 ** -24)).sum(0)).all()


@pytest.mark.parametrize("dim", [64, 700, 2560, 17000])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_no_number_stays_none(pkg, gpu_device, dim, bad):
    """A row with a NaN or an infinity has no mean: all of it is NaN, forward and backward, and no other row is."""
    s = make(gpu_device, 5, dim, FP32, None, FP32)
    clean = run(pkg, s)
    s["x"][2, dim // 2] = bad
    got = run(pkg, s)
    for n in ("y", "dx"):
        assert got[n][2].isnan().all(), n
        assert torch.equal(got[n][[0, 1, 3, 4]], clean[n][[0, 1, 3, 4]]), n


@pytest.mark.parametrize("dim", [700, 17000])
def test_numbers_whose_sums_overflow(pkg, gpu_device, dim):
    """Rows past float32's range have no spread in float32 either: no finite wrong ones come out of it but zeros (and the bias)."""
    s = make(gpu_device, 3, dim, FP32, None, FP32, bias=False)
    for size in (1e25, 3e38):
        s["x"] = torch.where(torch.arange(dim, device=gpu_device) % 2 == 0, size, 0.5 * size).expand(3, -1).contiguous()
        y = pkg.layer_norm_fn(s["x"], s["weight"])
        assert ((y == 0) | y.isnan()).all()
