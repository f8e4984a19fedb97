"""Layer norm with the residual's addition against its statement in 64 bits.

Tolerances, n the row's length: a sum of n terms in fp32 is off by at most n 2^-24 of the sum of magnitudes.  The mean is off by n 2^-24 mean|h|,
which each difference h - mean then has, and beside it the spread s: an error of n 2^-24 mean|h| / s of a normalised value.  y and dx are products of a few such
factors; each result is rounded once, eps / 2 of itself.  The sums here are made in trees of at most 16384 / 512 terms a lane: with n_eff = 64 in place of n
the bound holds with room and still sees a wrong term."""
import pytest
import torch

from causal_conv1d.layer_norm import layer_norm_ref

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
pytestmark = pytest.mark.gpu


def make(dev, rows, dim, dtype, res, w, bias=True, offset=0.0, seed=0):
    r = torch.Generator(device=dev).manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, generator=r, device=dev)
    s = {"x": rand(rows, dim).add_(offset).to(dtype), "weight": rand(dim).to(w), "bias": rand(dim).to(w) if bias else None,
         "residual": None if res is None else rand(rows, dim).mul_(2).to(res)}
    s["dy"], s["dh"] = rand(rows, dim).to(dtype), None if res is None else rand(rows, dim).to(res)
    return s


def run(pkg, s, eps=1e-5):
    leaves = {n: s[n].detach().requires_grad_() for n in ("x", "weight", "bias", "residual") if s[n] is not None}
    got = pkg.layer_norm_fn(leaves["x"], leaves["weight"], leaves.get("bias"), residual=leaves.get("residual"), eps=eps)
    y, h = got if s["residual"] is not None else (got, None)
    outs = [y] + ([h] if h is not None else [])
    grads = torch.autograd.grad(outs, list(leaves.values()), [s["dy"], s["dh"]][:len(outs)])
    res = {"y": y.detach(), **{"d" + n: d for n, d in zip(leaves, grads)}}
    if h is not None:
        res["h"] = h.detach()
    return res


def check(got, s, eps=1e-5):
    x, res = s["x"], s["residual"]
    h = x if res is None else (x.float() + res.float()).to(res.dtype)
    if res is not None:
        assert torch.equal(got["h"], h)
    hd = h.double().requires_grad_()
    w, b = s["weight"].double().requires_grad_(), None if s["bias"] is None else s["bias"].double().requires_grad_()
    y = layer_norm_ref(hd, w, b, eps=eps)
    leaves = [hd, w] + ([] if b is None else [b])
    grads = torch.autograd.grad(y, leaves, s["dy"].double())
    dh = grads[0] + (0 if s["dh"] is None else s["dh"].double())
    n_eff = 64 * 2.0 ** -24
    hv = h.double()
    spread = (hv.var(-1, unbiased=False, keepdim=True) + eps).sqrt()
    rel = n_eff * (1 + hv.abs().mean(-1, keepdim=True) / spread)       # of a normalised value of size one
    unit = ((hv - hv.mean(-1, keepdim=True)) / spread).abs()
    wd, dy = s["weight"].double().abs(), s["dy"].double().abs()
    wdy = (wd * dy).mean(-1, keepdim=True)
    bounds = {"y": rel * (1 + unit) * wd + (0 if b is None else n_eff * s["bias"].double().abs()),
              "dx": rel / spread * (wd * dy + wdy + (1 + unit) * (wd * dy * (1 + unit)).mean(-1, keepdim=True)) + (0 if s["dh"] is None else n_eff * s["dh"].double().abs()),
              "dweight": (dy * (1 + unit) * (rel + (x.shape[0] + 64) * 2.0 ** -24)).sum(0), "dbias": (dy * (x.shape[0] + 64) * 2.0 ** -24).sum(0)}
    bounds["dresidual"] = bounds["dx"]
    want = {"y": y.detach(), "dx": dh, "dresidual": dh, "dweight": grads[1], "dbias": grads[-1]}
    for name, t in got.items():
        if name == "h":
            continue
        bound = bounds[name] + torch.finfo(t.dtype).eps / 2 * 1.01 * want[name].abs() + 2 * torch.finfo(t.dtype).tiny
        off = (t.double() - want[name]).abs()
        assert t.isfinite().all() and (off <= bound).all(), (name, (off / bound).max().item())


@pytest.mark.parametrize("types", [(FP32, FP32, FP32), (BF16, FP32, FP32), (BF16, BF16, BF16), (BF16, None, FP32), (FP16, FP16, FP16), (FP16, FP32, FP16), (FP16, None, FP32), (FP32, None, FP32)])
@pytest.mark.parametrize("shape", [(1, 1), (5, 7), (3, 64), (67, 500), (9, 513), (33, 1000), (6, 1025), (40, 2560), (3, 5120), (2, 9000), (2, 16384), (3, 16385), (2, 20001)])
def test_shapes_and_types(pkg, gpu_device, types, shape):
    """Every workgroup shape, whole vectors and cut ones, rows beyond the registers."""
    s = make(gpu_device, *shape, *types, seed=shape[1])
    check(run(pkg, s), s)


@pytest.mark.parametrize("rows", [2, 4099, 16384])
@pytest.mark.parametrize("bias", [True, False])
def test_many_rows(pkg, gpu_device, rows, bias):
    s = make(gpu_device, rows, 520, BF16, FP32, FP32, bias=bias)
    check(run(pkg, s), s)


@pytest.mark.parametrize("dim", [500, 2560, 17000])
def test_mean_large_beside_the_spread(pkg, gpu_device, dim):
    """A thousand times the spread: the square of the mean would swallow it."""
    s = make(gpu_device, 9, dim, FP32, None, FP32, offset=1000.0)
    check(run(pkg, s), s)


def test_constant_rows_and_eps(pkg, gpu_device):
    """No spread: y is the bias, whatever the row's value is, since the mean of equal numbers of 2^k columns is exact."""
    for value in (0.0, 3.0, -1e4):
        s = make(gpu_device, 4, 512, FP32, None, FP32)
        s["x"] = torch.full_like(s["x"], value)
        got = run(pkg, s)
        assert torch.equal(got["y"], s["bias"].expand(4, -1))
        assert got["dx"].isfinite().all()
    s = make(gpu_device, 4, 512, FP32, None, FP32)
    check(run(pkg, s, eps=0.5), s, eps=0.5)


def test_large_and_small_rows(pkg, gpu_device):
    s = make(gpu_device, 6, 700, FP32, None, FP32)
    s["x"] = s["x"] * torch.tensor([1e15, 1e-3, 1e8, 1.0, 1e-8, 1e-15], device=gpu_device)[:, None]
    check(run(pkg, s), s)


def test_layouts_streams_and_bits(pkg, gpu_device):
    """Rows that start anywhere, leading dimensions, another stream, the same bits again."""
    base = make(gpu_device, 30, 100, BF16, BF16, BF16)
    want = run(pkg, base)
    wide = {n: torch.zeros(30, 107, dtype=BF16, device=gpu_device) for n in ("x", "residual", "dy", "dh")}
    off = dict(base)
    for n, t in wide.items():
        t[:, 3:103] = base[n]
        off[n] = t[:, 3:103]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(pkg, off)
    torch.cuda.current_stream().wait_stream(side)
    cube = {n: t.view(5, 6, 100) if t.dim() == 2 else t for n, t in base.items()}
    third = run(pkg, cube)
    for n, t in want.items():
        assert torch.equal(t, got[n]), n
        assert torch.equal(t, third[n].view(t.shape)), n


def test_partial_gradients(pkg, gpu_device):
    """Only some inputs require a gradient, only the sum is used, and nothing at all."""
    s = make(gpu_device, 8, 96, FP32, FP32, FP32)
    full = run(pkg, s)
    x = s["x"].clone().requires_grad_()
    y, h = pkg.layer_norm_fn(x, s["weight"], s["bias"], residual=s["residual"])
    dx, = torch.autograd.grad([y, h], [x], [s["dy"], s["dh"]])
    assert torch.equal(dx, full["dx"])
    y, h = pkg.layer_norm_fn(x, s["weight"], None, residual=s["residual"])
    dx, = torch.autograd.grad([h], [x], [s["dh"]])
    assert torch.equal(dx, s["dh"])
    with torch.no_grad():
        y2 = pkg.layer_norm_fn(s["x"], s["weight"], s["bias"], residual=s["residual"])[0]
    assert torch.equal(y2, full["y"])


def test_no_rows_and_no_columns(pkg, gpu_device):
    w = torch.ones(16, device=gpu_device, requires_grad=True)
    b = torch.zeros(16, device=gpu_device, requires_grad=True)
    x = torch.zeros(0, 16, device=gpu_device, requires_grad=True)
    dx, dw, db = torch.autograd.grad(pkg.layer_norm_fn(x, w, b), [x, w, b], torch.zeros(0, 16, device=gpu_device))
    assert dx.shape == (0, 16) and torch.equal(dw, torch.zeros_like(dw)) and torch.equal(db, torch.zeros_like(db))
    assert pkg.layer_norm_fn(torch.zeros(3, 0, device=gpu_device), torch.zeros(0, device=gpu_device)).shape == (3, 0)


def test_against_differences(pkg, gpu_device):
    """Central differences in random directions, h = 1e-2: the third derivative's share, h^2, and rounding, 2^-24 sqrt(n) / h, are both below 2e-3."""
    s = make(gpu_device, 5, 60, FP32, FP32, FP32)
    got = run(pkg, s)
    r = torch.Generator(device=gpu_device).manual_seed(1)
    for n in ("x", "residual", "weight", "bias"):
        d = torch.randn(s[n].shape, generator=r, device=gpu_device)

        def loss(t):
            y, h = pkg.layer_norm_fn(*(t[m] for m in ("x", "weight", "bias")), residual=t["residual"])
            return ((y * s["dy"]).double().sum() + (h * s["dh"]).double().sum()).item()
        found = (loss(dict(s, **{n: s[n] + 1e-2 * d})) - loss(dict(s, **{n: s[n] - 1e-2 * d}))) / 2e-2
        each = got["d" + n].double() * d.double()
        assert abs(found - each.sum().item()) <= 1e-2 * each.norm().item(), n
