"""The example block runs the operators together: decoding continues a prefill as the whole sequence does, its gradients are those of the
same block on plain operators, and padding leaves the caches alone."""
import importlib.util
import os

import pytest
import torch
import torch.nn.functional as F

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "causal-conv1d_amd", "examples", "delta_block.py")


@pytest.fixture(scope="module")
def example(pkg):
    spec = importlib.util.spec_from_file_location("delta_block", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def block_of(example, seed=0):
    torch.manual_seed(seed)
    return example.DeltaBlock(96, 2, 4, dim_k=32, dim_v=48, dtype=torch.float32)


def plain(block, x, stream):
    """The block on plain PyTorch operators, in the parameters' type."""
    from causal_conv1d.gated_delta_rule import gated_delta_rule_ref
    from causal_conv1d.rms_norm import rms_norm_ref
    y, stream = rms_norm_ref(x, block.norm, residual=stream, eps=block.eps)
    mixed, z, a, b = F.linear(y, block.w_in).split(block.parts, -1)
    mixed = F.conv1d(F.pad(mixed.transpose(1, 2), (block.width - 1, 0)), block.conv_weight[:, None], block.conv_bias, groups=block.channels)
    q, k, v = block._heads(F.silu(mixed).transpose(1, 2))
    g, beta = -block.a_log.exp() * F.softplus(a + block.dt), torch.sigmoid(b)
    o = gated_delta_rule_ref(q, k, v, g, beta, qk_l2norm=True)
    o = rms_norm_ref(o, block.head_norm, eps=block.eps)
    return F.linear(o.flatten(-2) * F.silu(z), block.w_out), stream


@pytest.mark.gpu
def test_gradients_of_the_block(example, gpu_device):
    """In float32 against 64 bits: each of some twenty operators in a row adds its own rounding, of sums of up to a few hundred terms,
    2^-24 sqrt(n) of the largest value each at most: 2e-4 of the largest value of each tensor leaves room for all of them."""
    block = block_of(example)
    x, stream = torch.randn(2, 70, 96, device=gpu_device, requires_grad=True), torch.randn(2, 70, 96, device=gpu_device, requires_grad=True)
    leaves = [x, stream] + list(block.parameters())
    out = block(x, stream)
    seeds = [torch.randn_like(t) for t in out]
    got = list(out) + list(torch.autograd.grad(out, leaves, seeds))
    wide = block_of(example).double()
    xd, sd = x.detach().cpu().double().to(gpu_device).requires_grad_(), stream.detach().double().requires_grad_()
    out = plain(wide, xd, sd)
    want = list(out) + list(torch.autograd.grad(out, [xd, sd] + list(wide.parameters()), [t.double() for t in seeds]))
    for i, (a, b) in enumerate(zip(got, want)):
        assert (a.double() - b).abs().max() <= 2e-4 * b.abs().max(), i


@pytest.mark.gpu
def test_decoding_continues_a_prefill(example, gpu_device):
    """The same sums in another order: 1e-4 of the largest value, as above; in 8 bits a value of the first norm is off by 2^-4 of
    itself at most, and the outputs, which are sums of many, by less than that of the largest."""
    block = block_of(example, 1)
    x, stream = torch.randn(3, 75, 96, device=gpu_device), torch.randn(3, 75, 96, device=gpu_device)
    with torch.no_grad():
        whole, whole_stream = block(x, stream)
        for in_8_bits, tol in ((False, 1e-4), (True, 2.0 ** -4)):
            cache = example.Cache(block, 6)
            slots = torch.tensor([4, 0, 2], device=gpu_device)
            block(x[:, :70], stream[:, :70], cache=cache, slots=slots)
            before = cache.conv.clone(), cache.state.clone()
            padded = torch.tensor([4, -1, 0, 2], dtype=torch.int32, device=gpu_device)
            for t in range(70, 75):
                xs, ss = (torch.cat([a[:1, t], torch.zeros(1, 96, device=gpu_device), a[1:, t]]) for a in (x, stream))
                out, new = block.step(xs, ss, cache, padded, in_8_bits=in_8_bits)
                assert (out[[0, 2, 3]] - whole[:, t]).abs().max() <= tol * whole.abs().max()
                assert torch.equal(new[[0, 2, 3]], whole_stream[:, t])
            for a, b in zip((cache.conv, cache.state), before):
                assert torch.equal(a[[1, 3, 5]], b[[1, 3, 5]])
                assert not torch.equal(a[[0, 2, 4]], b[[0, 2, 4]])


@pytest.mark.gpu
def test_compiled_block(example, gpu_device):
    """Traced whole by torch.compile (aot_eager: no generated code): the same kernels, the same bits."""
    block = block_of(example, 2)
    x, stream = torch.randn(1, 66, 96, device=gpu_device), torch.randn(1, 66, 96, device=gpu_device)
    with torch.no_grad():
        want = block(x, stream)
        got = torch.compile(block, backend="aot_eager", fullgraph=True)(x, stream)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_compiled_training(example, gpu_device):
    """The same with gradients, which torch.compile takes through the Python functions' graph: the same kernels, the same bits (plain
    operators around them may be traced into other ones, so float32's rounding of those is allowed: 2^-20 of the largest value)."""
    block = block_of(example, 3)
    x, stream = (torch.randn(1, 66, 96, device=gpu_device, requires_grad=True) for _ in range(2))
    leaves = [x, stream] + list(block.parameters())
    want = block(x, stream)
    seeds = [torch.randn_like(t) for t in want]
    want = list(want) + list(torch.autograd.grad(want, leaves, seeds))
    got = torch.compile(block, backend="aot_eager", fullgraph=True)(x, stream)
    got = list(got) + list(torch.autograd.grad(got, leaves, seeds))
    for a, b in zip(got, want):
        assert (a - b).abs().max() <= 2.0 ** -20 * b.abs().max()
