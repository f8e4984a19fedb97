"""The 8-bit codes of rms_norm_quant_fn one by one: y / scales[row], a float32 quotient rounded to nearest, to the nearest e4m3, ties to even.

Where y is known to the bit (rows of one magnitude, a power of two, have a root that is a power of two; y is the weight, with
a sign) the codes are compared for equality, at the ties between two codes and next to them above all.  Elsewhere y is known to within
float32's rounding of its sums, and a code has to be one that some y inside that has."""
import pytest
import torch

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
F8 = torch.float8_e4m3fn


def codes_of(q):
    return q.to(F8).view(torch.uint8)


def ties():
    """The numbers half way between two neighbouring codes, exact in 5 bits, and the codes themselves."""
    codes = torch.arange(0x7f, dtype=torch.uint8).view(F8).float()           # 0 .. 448
    return torch.cat([(codes[1:] + codes[:-1]) / 2, codes])


def weights(dim, dtype, most, seed):
    """`dim` numbers of `dtype` up to `most`: ties of rows whose largest is `most`, their neighbours in the type, others at random."""
    r = torch.Generator().manual_seed(seed)
    most = torch.tensor(most).to(dtype)
    scale = most.float() * torch.tensor(1 / 448)
    t = ties()
    w = (t[torch.randint(len(t), (dim,), generator=r)] * scale).to(dtype)
    bits = w.view(torch.int32 if dtype == torch.float32 else torch.int16)
    near = torch.randint(-2, 3, (dim,), generator=r).to(bits.dtype)
    w = torch.where((bits > 8), (bits + near), bits).view(dtype)
    some = torch.rand(dim, generator=r) < 0.3
    w = torch.where(some, (torch.rand(dim, generator=r) * most.float()).to(dtype), w).clamp(max=most)
    w[torch.randint(dim, (1,), generator=r)] = most
    return w


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 1024, 4096, 16384, 32768])
@pytest.mark.parametrize("dtype,wdtype", [(torch.float32, torch.float32), (torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16),
                                          (torch.bfloat16, torch.float32), (torch.float16, torch.float32)])
def test_codes_are_quotients(pkg, gpu_device, dim, dtype, wdtype):
    rows = 8
    size = 2.0 ** torch.arange(-4, 4)
    sign = torch.where(torch.rand(rows, dim, generator=torch.Generator().manual_seed(dim)) < 0.5, -1.0, 1.0)
    x = (size[:, None] * sign).to(dtype).to(gpu_device)
    for seed, most in enumerate([448.0, 7.0, 1.0, 1.9, 2.3, 0.05, 3.0 / 7, 447.0, 100.1, 1e-3, 6e-5, 1e4]):
        w = weights(dim, wdtype, most, seed + dim)
        y8, scales = (t.cpu() for t in pkg.rms_norm_quant_fn(x, w.to(gpu_device), eps=0.0))
        y = sign * w.float()
        assert torch.equal(pkg.rms_norm_fn(x, w.to(gpu_device), eps=0.0).cpu(), y.to(dtype))            # y is what it is taken for
        assert ((scales.double() * 448 / y.abs().amax(-1).double() - 1).abs() <= 2.0 ** -23).all()
        want = codes_of(y / scales[:, None])
        wrong = y8.view(torch.uint8) != want
        assert not wrong.any(), "largest %g: %d of %d codes, the first of y %r over %r" % (
            most, wrong.sum(), wrong.numel(), y[wrong][0].item(), scales[wrong.any(-1)][0].item())


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [1, 7, 64, 130, 513, 1001, 2049, 8200, 16391])
@pytest.mark.parametrize("dtype,rdtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
                                          (torch.float16, None)])
def test_codes_of_rows_at_random(pkg, gpu_device, dim, dtype, rdtype):
    """y is off by less than 4 (16 + dim / 512) 2^-24 of itself (its root by a tree of sums over at most that many terms a lane, four
    times that for the multiplications behind it), and so is the quotient, which is rounded once more."""
    rows = 300 if dim < 4000 else 20
    r = torch.Generator().manual_seed(dim)
    x = torch.randn(rows, dim, generator=r).to(dtype).to(gpu_device)
    res = None if rdtype is None else (2 * torch.randn(rows, dim, generator=r)).to(rdtype).to(gpu_device)
    w = (torch.rand(dim, generator=r) + 0.5).to(gpu_device)
    y8, scales = pkg.rms_norm_quant_fn(x, w.to(dtype), residual=res, eps=1e-6)[:2]
    h = (x if res is None else (x.float() + res.float()).to(rdtype)).double()
    y = (h * (h.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w.to(dtype).double()).cpu()
    q = (y / scales.double().cpu()[:, None]).abs()
    room = (4 * (16 + dim / 512) + 1) * 2.0 ** -24
    low, high = codes_of((q * (1 - room)).float()), codes_of((q * (1 + room)).clamp(max=448.0).float())
    got = y8.cpu().view(torch.uint8) & 0x7f
    assert ((got >= low) & (got <= high)).all()
    assert torch.equal(torch.signbit(y8.cpu().float())[got > 0], torch.signbit(y)[got > 0])
