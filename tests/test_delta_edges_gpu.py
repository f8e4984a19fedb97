"""The gated delta rule at the edges of what it takes.  Tolerances are those of test_gated_delta_rule_gpu.py and
test_gated_delta_rule_bwd_gpu.py."""
import pytest
import torch

from test_gated_delta_rule_bwd_gpu import check as check_gradients
from test_gated_delta_rule_gpu import close, make, recurrence


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


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,group,dim_k,dim_v", [
    (torch.float32, 2, 128, 32), (torch.float32, 2, 250, 24), (torch.bfloat16, 2, 256, 40), (torch.float16, 3, 224, 16),       # dq and dk leave one after the other
    (torch.float32, 2, 96, 64), (torch.bfloat16, 2, 192, 64),                                                               # at once, their largest
    (torch.bfloat16, 1, 192, 128), (torch.float16, 1, 160, 64), (torch.float32, 1, 176, 32), (torch.bfloat16, 2, 136, 72)])    # six steps of dim_k, whole vectors
@pytest.mark.parametrize("l2norm", [False, True])
def test_gradients_of_wide_heads(pkg, gpu_device, dtype, group, dim_k, dim_v, l2norm):
    check_gradients(pkg, gpu_device, 1, 100, 2, group, dim_k, dim_v, dtype, l2norm, True)


@pytest.mark.gpu
@pytest.mark.parametrize("sequences", [65, 130])
def test_many_packed_sequences_by_chunks(pkg, gpu_device, sequences):
    """More than 64: a chunk's sequence is found in two steps."""
    lengths = [(37 * i) % 90 + 20 for i in range(sequences)]
    q, k, v, g, beta, s0 = make(1, sum(lengths), 1, 1, 32, 16, torch.bfloat16, gpu_device, sequences=sequences, l2norm=True)
    cu = torch.tensor([0] + lengths).cumsum(0).to(torch.int32).to(gpu_device)
    out, final = pkg.gated_delta_rule_fn(q, k, v, g, beta, initial_states=s0, return_final_states=True, cu_seqlens=cu, qk_l2norm=True)
    for i, (lo, hi) in enumerate(zip(cu.tolist()[:-1], cu.tolist()[1:])):
        want, want_final = recurrence(*(t[:, lo:hi] for t in (q, k, v, g, beta)), s0[i:i + 1], True)
        close(out[:, lo:hi], want, torch.bfloat16, 32, "out of sequence %d" % i)
        close(final[i:i + 1], want_final, torch.float32, 32, "final of sequence %d" % i)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("seqlen", [5, 130])
def test_range_of_values(pkg, gpu_device, dtype, seqlen):
    """v and the states times a power of two: outputs, states and the gradients of q exactly as many times as large, or, where the third terms
    of numbers fall below the smallest normal one (2^-126 against 2^-100, at most half of it each), off by 2^-24 and a few sums of that."""
    q, k, v, g, beta, s0 = make(1, seqlen, 2, 1, 64, 64, dtype, gpu_device, l2norm=True)

    def run(power):
        leaves = [q.detach().requires_grad_(), (v.float() * 2.0 ** power).to(dtype).requires_grad_()]
        out, final = pkg.gated_delta_rule_fn(leaves[0], k, leaves[1], g, beta, initial_states=s0 * 2.0 ** power, return_final_states=True, qk_l2norm=True)
        dq, _ = torch.autograd.grad([out, final], leaves, [torch.ones_like(out), torch.ones_like(final)])
        return [t.detach().double() * 2.0 ** -power for t in (out, final, dq)]
    base = run(0)
    for power in (-80, 60, 110):
        assert all(torch.equal(a, b) for a, b in zip(run(power), base)), power
    # (a value of 16 bits may also come out one rounding beside the other)
    for a, b, t in zip(run(-100), base, (dtype, torch.float32, dtype)):
        assert (a - b).norm() <= (64 ** 0.5 * 2.0 ** -24 + (0 if t == torch.float32 else 2.0 ** -8)) * b.norm()
