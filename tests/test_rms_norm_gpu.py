"""rms_norm_fn, rms_norm_quant_fn and dequantize_rows against the formulas in 64 bits.

Tolerances.  An output is rounded once to its type (half a unit in the last place: 2^-8 of its value for bfloat16, 2^-11
for float16, 2^-24 for float32).  The root and the sums are formed in float32: a sum over n terms in partial sums of at most
8 + n/512 terms a lane and a tree over the lanes is off by less than (16 + n/512) 2^-24 of the sum of its terms'
magnitudes; four times that covers the handful of multiplications behind it.  dweight adds `rows` terms in the same way."""
import pytest
import torch

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
HALF_ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
EPS = 1e-6

# one element, below and at a vector, a wavefront's reach and one over, odd, workgroups of both sizes, rows read twice
DIMS = [1, 7, 8, 64, 511, 513, 1001, 1024, 2049, 4100, 8200, 16384, 16391]


def close(got, want, dtype, terms, magnitude=None):
    """`magnitude`: the largest sum of magnitudes behind a value, where sums cancel (default: the values' own)."""
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape
    room = want.abs() if magnitude is None else torch.maximum(want.abs(), magnitude.double().cpu())
    tol = HALF_ULP[dtype] * want.abs() * 1.01 + 4 * (16 + terms / 512) * 2.0 ** -24 * room + (6e-8 if dtype == torch.float16 else 0)
    bad = (got - want).abs() > tol
    assert not bad.any(), "%d of %d, worst %.3e against %.3e" % (bad.sum(), bad.numel(), ((got - want).abs() / tol).max(), 1)


def inputs(rows, dim, dtype, rdtype, wdtype, dev, seed=0):
    g = torch.Generator().manual_seed(seed + dim)
    x = torch.randn(rows, dim, generator=g).to(dtype).to(dev)
    r = None if rdtype is None else (2 * torch.randn(rows, dim, generator=g)).to(rdtype).to(dev)
    w = (torch.rand(dim, generator=g) + 0.5).to(wdtype).to(dev)
    return x, r, w


def formula(x, r, w):
    h = x if r is None else (x.float() + r.float()).to(r.dtype)
    h64 = h.double()
    inv = (h64.square().mean(-1, keepdim=True) + EPS).rsqrt()
    return h, h64, inv, h64 * inv * w.double()


@pytest.mark.gpu
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("dtype,rdtype,wdtype", [
    (torch.float32, torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16, torch.bfloat16),
    (torch.bfloat16, torch.float32, torch.float32), (torch.float16, torch.float16, torch.float32),
    (torch.float16, torch.float32, torch.float16), (torch.bfloat16, None, torch.float32), (torch.float32, None, torch.float32)])
def test_forward_and_backward(pkg, gpu_device, dim, dtype, rdtype, wdtype):
    rows = 37 if dim < 4000 else 5
    x, r, w = inputs(rows, dim, dtype, rdtype, wdtype, gpu_device)
    for t in (x, r, w):
        if t is not None:
            t.requires_grad_()
    res = pkg.rms_norm_fn(x, w, residual=r, eps=EPS)
    y, h = res if r is not None else (res, None)
    hs, h64, inv, want = formula(x.detach(), None if r is None else r.detach(), w.detach())
    assert y.dtype == dtype and (h is None or (h.dtype == rdtype and torch.equal(h, hs)))
    close(y, want, dtype, dim)
    g = torch.Generator().manual_seed(9)
    dy = torch.randn(rows, dim, generator=g).to(dtype).to(gpu_device)
    dh = None if r is None else torch.randn(rows, dim, generator=g).to(rdtype).to(gpu_device)
    grads = torch.autograd.grad([y] if r is None else [y, h], [x, w] if r is None else [x, w, r], [dy] if r is None else [dy, dh])
    wdy = w.detach().double() * dy.double()
    mean = (h64 * wdy).mean(-1, keepdim=True)
    dx = inv * wdy - h64 * inv ** 3 * mean + (0 if dh is None else dh.double())
    size = (inv * wdy).abs() + (h64 * inv ** 3).abs() * (h64 * wdy).abs().mean(-1, keepdim=True) + (0 if dh is None else dh.double().abs())
    close(grads[0], dx, dtype, dim, size)
    if r is not None:
        close(grads[2], dx, rdtype, dim, size)
    terms = dy.double() * h64 * inv
    close(grads[1], terms.sum(0), wdtype, dim + 512 * rows, terms.abs().sum(0))


@pytest.mark.gpu
def test_gradients_against_differences(pkg, gpu_device):
    """The backward against differences of the forward itself, in float32: central differences of step s are off by
    the third derivative's share, s^2 / 6, and by the forward's rounding, 2^-24 sqrt(n) / s: 1e-3 covers both at s = 0.02."""
    x, r, w = inputs(3, 40, torch.float32, torch.float32, torch.float32, gpu_device, 5)
    dy = torch.randn(3, 40, generator=torch.Generator().manual_seed(1)).to(gpu_device)
    dh = torch.randn(3, 40, generator=torch.Generator().manual_seed(2)).to(gpu_device)

    def loss(x, r, w):
        y, h = pkg.rms_norm_fn(x, w, residual=r, eps=EPS)
        return float((y.double() * dy.double()).sum() + (h.double() * dh.double()).sum())

    for t in (x, r, w):
        t.requires_grad_()
    y, h = pkg.rms_norm_fn(x, w, residual=r, eps=EPS)
    grads = torch.autograd.grad([y, h], [x, r, w], [dy, dh])
    for i, grad in enumerate(grads):
        for seed in range(3):
            d = torch.randn(grad.shape, generator=torch.Generator().manual_seed(seed)).to(gpu_device)
            d /= d.norm()
            up, down = ([t.detach() + (s * d if j == i else 0) for j, t in enumerate((x, r, w))] for s in (0.02, -0.02))
            slope = (loss(*up) - loss(*down)) / 0.04
            assert abs(slope - float((grad.double() * d.double()).sum())) < 1e-3 * max(1.0, float(grad.norm()))


@pytest.mark.gpu
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("dtype,rdtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                          (torch.bfloat16, torch.float32), (torch.float16, None)])
def test_output_in_8_bits(pkg, gpu_device, dim, dtype, rdtype):
    rows = 37 if dim < 4000 else 5
    x, r, w = inputs(rows, dim, dtype, rdtype, dtype, gpu_device)
    x[1] = 0
    if r is not None:
        r[1] = 0
    res = pkg.rms_norm_quant_fn(x, w, residual=r, eps=EPS)
    y8, scales = res[0], res[1]
    hs, _, _, want = formula(x, r, w)
    if r is not None:
        assert torch.equal(res[2], hs)
    assert y8.dtype == torch.float8_e4m3fn and scales.dtype == torch.float32 and scales.shape == (rows,)
    most = want.abs().amax(-1) / 448
    close(scales, most, torch.float32, dim)
    assert scales[1] == 0 and not y8[1].float().any()
    # Half a step of e4m3: 2^-4 of the value, 2^-10 of the scale below its smallest normal number; the rest is float32's.
    tol = want.abs() * (2.0 ** -4 + 1e-5) + most[:, None] * (2.0 ** -10 + 1e-5)
    assert ((y8.double() * scales.double()[:, None] - want).abs() <= tol).all()
    assert (y8.float().abs().amax(-1)[scales > 0] == 448).all()
    for out in DTYPES:
        back = pkg.dequantize_rows(y8, scales, out)
        assert torch.equal(back, (y8.float() * scales[:, None]).to(out))


@pytest.mark.gpu
def test_layouts(pkg, gpu_device):
    """Rows of a wider buffer, rows that start off the vector grid, leading dimensions, strided rows, no rows at all."""
    wide = torch.randn(6, 5, 300, device=gpu_device).to(torch.bfloat16)
    w = torch.rand(203, device=gpu_device)
    x = wide[..., 3:206]
    want = pkg.rms_norm_fn(x.contiguous(), w, eps=EPS)
    assert torch.equal(pkg.rms_norm_fn(x, w, eps=EPS), want)
    assert torch.equal(pkg.rms_norm_fn(x.transpose(0, 1), w, eps=EPS), want.transpose(0, 1))
    strided = torch.randn(203, 7, device=gpu_device).t()
    assert torch.equal(pkg.rms_norm_fn(strided, w), pkg.rms_norm_fn(strided.contiguous(), w))
    assert pkg.rms_norm_fn(x[:0], w).shape == (0, 5, 203)
    y8, scales = pkg.rms_norm_quant_fn(x[:0], w)
    assert y8.shape == (0, 5, 203) and scales.shape == (0, 5) and pkg.dequantize_rows(y8, scales).shape == (0, 5, 203)
    xg, wg = x[:0].clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(pkg.rms_norm_fn(xg, wg).sum(), [xg, wg])
    assert dx.shape == xg.shape and not dw.any()


@pytest.mark.gpu
def test_unused_outputs_and_single_gradients(pkg, gpu_device):
    x, r, w = inputs(9, 130, torch.bfloat16, torch.float32, torch.float32, gpu_device)
    for t in (x, r, w):
        t.requires_grad_()
    y, h = pkg.rms_norm_fn(x, w, residual=r, eps=EPS)
    gx, gr = torch.autograd.grad(h.sum(), [x, r], retain_graph=True)     # only the sum: ones
    assert torch.equal(gx, torch.ones_like(x)) and torch.equal(gr, torch.ones_like(r))
    only_y = torch.autograd.grad(y.float().sum(), [x, r, w], retain_graph=True)
    both = torch.autograd.grad([y, h], [x, r, w], [torch.ones_like(y), torch.zeros_like(h)])
    assert all(torch.equal(a, b) for a, b in zip(only_y, both))


@pytest.mark.gpu
def test_values_that_are_not_finite_stay_in_their_rows(pkg, gpu_device):
    x, r, w = inputs(8, 700, torch.bfloat16, torch.bfloat16, torch.float32, gpu_device)
    good, _ = pkg.rms_norm_fn(x, w, residual=r, eps=EPS)
    good8, good_s, _ = pkg.rms_norm_quant_fn(x, w, residual=r, eps=EPS)
    x[2, 5], x[4, 600] = float("nan"), float("inf")
    y, _ = pkg.rms_norm_fn(x, w, residual=r, eps=EPS)
    y8, s, _ = pkg.rms_norm_quant_fn(x, w, residual=r, eps=EPS)
    rest = [0, 1, 3, 5, 6, 7]
    assert torch.equal(y[rest], good[rest]) and torch.equal(s[rest], good_s[rest]) and torch.equal(y8[rest].float(), good8[rest].float())
    assert y[2].isnan().all() and s[2].isnan() and y[4, 600].isnan() and not y[4, :600].any()


@pytest.mark.gpu
def test_same_bits_every_time_and_on_another_stream(pkg, gpu_device):
    x, r, w = inputs(3000, 1000, torch.bfloat16, torch.float32, torch.float32, gpu_device)
    for t in (x, r, w):
        t.requires_grad_()

    def step():
        y, h = pkg.rms_norm_fn(x, w, residual=r, eps=EPS)
        return [y, h] + list(torch.autograd.grad([y, h], [x, r, w], [torch.ones_like(y), h.detach()]))

    first = step()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        second = step()
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(first, second))


@pytest.mark.gpu
def test_refusals(pkg, gpu_device):
    x, w = torch.zeros(4, 16, device=gpu_device, dtype=torch.bfloat16), torch.ones(16, device=gpu_device)
    with pytest.raises(RuntimeError, match="must have shape"):
        pkg.rms_norm_fn(x, w[:8])
    with pytest.raises(RuntimeError, match="residual must have the shape"):
        pkg.rms_norm_fn(x, w, residual=x[:2])
    with pytest.raises(RuntimeError, match="residual must have the dtype"):
        pkg.rms_norm_fn(x, w, residual=x.half())
    with pytest.raises(RuntimeError, match="weight must have the dtype"):
        pkg.rms_norm_fn(x, w.half())
    with pytest.raises(RuntimeError, match="GPU"):
        pkg.rms_norm_fn(x, w.cpu())
    with pytest.raises(RuntimeError, match="float32, float16 or bfloat16"):
        pkg.rms_norm_fn(x.double(), w.double())
    with pytest.raises(RuntimeError, match="e4m3"):
        pkg.dequantize_rows(x, w[:4])
    y8, scales = pkg.rms_norm_quant_fn(x, w)
    with pytest.raises(RuntimeError, match="scales must have the shape"):
        pkg.dequantize_rows(y8, scales[:2])
