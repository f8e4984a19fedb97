"""The gated delta rule at the edges of what it takes.  Tolerances are those of test_gated_delta_rule_gpu.py and
test_gated_delta_rule_bwd_gpu.py."""
import pytest
import torch

from test_gated_delta_rule_gpu import make


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim_k", [5, 64])
def test_no_value_heads(pkg, gpu_device, dtype, dim_k):
    """Nothing depends on q and k then: zeros, whatever the memory of the gradients held before."""
    q, k = (torch.randn(2, 70, 3, dim_k, device=gpu_device, dtype=dtype).requires_grad_() for _ in range(2))
    v = torch.randn(2, 70, 0, 16, device=gpu_device, dtype=dtype).requires_grad_()
    g = torch.zeros(2, 70, 0, device=gpu_device)
    out, final = pkg.gated_delta_rule_fn(q, k, v, g, g, return_final_states=True)
    assert out.shape == v.shape and final.shape == (2, 0, dim_k, 16)
    used = [torch.full_like(q, float("nan")) for _ in range(8)]              # what the allocator hands out next
    torch.cuda.synchronize()
    del used
    dq, dk, dv = torch.autograd.grad([out, final], [q, k, v], [torch.ones_like(out), torch.ones_like(final)])
    assert dv.shape == v.shape and torch.equal(dq, torch.zeros_like(q)) and torch.equal(dk, torch.zeros_like(k))


@pytest.mark.gpu
def test_one_token_of_any_stride(pkg, gpu_device):
    """A training step over one token whose stride along the tokens is far beyond what a chunk's rows may have: the same bits."""
    q, k, v, g, beta, _ = make(3, 1, 1, 2, 32, 16, torch.bfloat16, gpu_device, l2norm=True)
    far = v.contiguous().as_strided(v.shape, (v[0].numel(), 1 << 30, 16, 1))
    dout = torch.randn(v.shape, device=gpu_device).bfloat16()
    results = []
    for x, d in ((v.contiguous(), dout), (far, dout.as_strided(dout.shape, far.stride()))):
        leaves = [t.detach().requires_grad_() for t in (q, k, x, g, beta)]
        out = pkg.gated_delta_rule_fn(*leaves, qk_l2norm=True)
        results.append([out, *torch.autograd.grad(out, leaves, d)])
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("seqlen", [1, 70])
def test_gates_at_the_ends_of_the_exponential(pkg, gpu_device, seqlen):
    """exp(g) by itself: a state of ones, read by a query of one row, nothing learned.  Two units in the last place where it is a normal number of 32
    bits, 2^-126 at most below that; above the largest number nothing finite comes out."""
    for g0 in (0.0, -1e-3, 3.7, -20.3, -87.0, 88.0, 88.7, -88.0, -95.0, -103.5, -104.5, -1e30, float("-inf")):
        q, k = torch.zeros(1, seqlen, 1, 8, device=gpu_device), torch.zeros(1, seqlen, 1, 8, device=gpu_device)
        q[..., 0] = 1
        v, beta, g = torch.zeros(1, seqlen, 1, 8, device=gpu_device), torch.zeros(1, seqlen, 1, device=gpu_device), torch.zeros(1, seqlen, 1, device=gpu_device)
        g[:, 0] = g0
        out, final = pkg.gated_delta_rule_fn(q, k, v, g, beta, scale=1.0, initial_states=torch.ones(1, 1, 8, 8, device=gpu_device), return_final_states=True)
        want = g[0, 0, 0].double().exp()
        # (by chunks the state is read as the sum of three numbers of 16 bits, exact for a power of two)
        assert ((out.double() - want).abs() <= 2 * 2.0 ** -23 * want + 2.0 ** -126).all() and ((final.double() - want).abs() <= 2 * 2.0 ** -23 * want + 2.0 ** -126).all(), g0
    for g0 in (89.0, 100.0, float("inf"), float("nan")):
        g[:, 0] = g0
        out, final = pkg.gated_delta_rule_fn(q, k, v, g, beta, scale=1.0, initial_states=torch.ones(1, 1, 8, 8, device=gpu_device), return_final_states=True)
        assert not torch.isfinite(out).any() and not torch.isfinite(final).any(), g0
