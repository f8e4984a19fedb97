"""What the mixer's operators have to hold beside their formulas: offsets past 32 bits, launches cut into slices, other streams,
values that are not finite, rows too small to be divided by, torch.library's checks and torch.compile.

Tolerances are those of test_gated_delta_rule_gpu.py and test_rms_norm_gpu.py; where two calls do the same work
their bits are compared."""
import pytest
import torch

from test_gated_delta_rule_gpu import close as close_delta
from test_gated_delta_rule_gpu import make, recurrence

BEYOND = 1 << 31


@pytest.mark.gpu
def test_states_beyond_32_bits(pkg, gpu_device):
    """The last of 2^31 elements' worth of states, by its index."""
    heads, dim = 2, 128
    slots = BEYOND // (heads * dim * dim) + 3
    state = torch.empty(slots, heads, dim, dim, device=gpu_device)
    q, k, v, g, beta, s0 = make(3, 1, 1, heads, dim, dim, torch.bfloat16, gpu_device, l2norm=True)
    index = torch.tensor([slots - 1, 0, slots - 2], dtype=torch.int32, device=gpu_device)
    state[index.long()] = s0
    out = pkg.gated_delta_rule_update(q, k, v, g, beta, state, state_indices=index, qk_l2norm=True)
    want, want_state = recurrence(q, k, v, g, beta, s0, True)
    close_delta(out, want, torch.bfloat16, dim, "out")
    close_delta(state[index.long()], want_state, torch.float32, dim, "state")


@pytest.mark.gpu
@pytest.mark.parametrize("seqlen", [4, 70])
def test_batch_entries_beyond_32_bits(pkg, gpu_device, seqlen):
    q, k, v, g, beta, _ = make(2, seqlen, 1, 2, 32, 16, torch.bfloat16, gpu_device, l2norm=True)
    base = torch.empty(BEYOND + v[0].numel() + 8, dtype=torch.bfloat16, device=gpu_device)
    far = base.as_strided(v.shape, (BEYOND + 8, 2 * 16, 16, 1))
    far.copy_(v)
    out = pkg.gated_delta_rule_fn(q, k, far, g, beta, qk_l2norm=True)
    assert torch.equal(out, pkg.gated_delta_rule_fn(q, k, v.contiguous(), g, beta, qk_l2norm=True))


@pytest.mark.gpu
def test_tokens_far_apart(pkg, gpu_device):
    """Tokens 2^25 bytes apart: further than 64 of them can be reached with 32 bits, so that the forward goes by tokens; a little nearer
    it goes by chunks.  Both are right; gradients are refused at the larger distance."""
    seqlen = 66
    q, k, v, g, beta, _ = make(1, seqlen, 1, 1, 16, 16, torch.bfloat16, gpu_device, l2norm=True)
    want, _ = recurrence(q, k, v, g, beta, None, True)
    base = torch.empty(seqlen << 24, dtype=torch.bfloat16, device=gpu_device)
    for stride in (1 << 24, (1 << 24) - 8):
        far = base.as_strided(v.shape, (0, stride, 16, 1))
        far.copy_(v)
        close_delta(pkg.gated_delta_rule_fn(q, k, far, g, beta, qk_l2norm=True), want, torch.bfloat16, 16, "stride %d" % stride)
        if stride == 1 << 24:
            with pytest.raises(RuntimeError, match="too large"):
                pkg.gated_delta_rule_fn(q, k, far.requires_grad_(), g, beta, qk_l2norm=True)


@pytest.mark.gpu
def test_rows_beyond_32_bits(pkg, gpu_device):
    base = torch.empty(BEYOND + 4096, dtype=torch.bfloat16, device=gpu_device)
    x = base.as_strided((2, 1001), (BEYOND + 9, 1))
    x.copy_(torch.randn(2, 1001, generator=torch.Generator().manual_seed(0)))
    w = torch.rand(1001, device=gpu_device)
    assert torch.equal(pkg.rms_norm_fn(x, w), pkg.rms_norm_fn(x.contiguous(), w))
    y8, scales = pkg.rms_norm_quant_fn(x, w)
    z8, zs = pkg.rms_norm_quant_fn(x.contiguous(), w)
    assert torch.equal(y8.view(torch.uint8), z8.view(torch.uint8)) and torch.equal(scales, zs)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [100, 1500, 9000, 20000])
def test_launches_in_slices(pkg, gpu_device, cc1d_lib, dim):
    """More rows than one launch may have, shown with a small limit: the same bits."""
    rows = 150
    r = torch.Generator().manual_seed(1)
    x, h = (torch.randn(rows, dim, generator=r).bfloat16().to(gpu_device) for _ in range(2))
    w = torch.rand(dim, generator=r).bfloat16().to(gpu_device)

    def all_of_it():
        y, s = pkg.rms_norm_fn(x, w, residual=h)
        y8, scales, s8 = pkg.rms_norm_quant_fn(x, w, residual=h)
        return y, s, y8.view(torch.uint8), scales, s8, pkg.dequantize_rows(y8, scales)
    want = all_of_it()
    try:
        assert cc1d_lib.cc1d_set_tunable(b"launch_limit_shift", 18) == 0       # 2^13 threads
        got = all_of_it()
    finally:
        cc1d_lib.cc1d_set_tunable(b"launch_limit_shift", 0)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("seqlen", [1, 130])
def test_another_stream(pkg, gpu_device, seqlen):
    args = make(2, seqlen, 2, 2, 64, 48, torch.bfloat16, gpu_device, l2norm=True)
    q, k, v, g, beta, s0 = (t.detach().clone().requires_grad_() for t in args)

    def both():
        out, final = pkg.gated_delta_rule_fn(q, k, v, g, beta, initial_states=s0, return_final_states=True, qk_l2norm=True)
        return (out, final) + torch.autograd.grad([out, final], [q, k, v, g, beta, s0], [torch.ones_like(out), torch.ones_like(final)])
    want = both()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_no_sequence(pkg, gpu_device):
    """Tokens without a sequence are refused (nobody would write their zeros); without tokens there is nothing to do."""
    q, k, v, g, beta, _ = make(1, 70, 1, 2, 32, 16, torch.bfloat16, gpu_device)
    cu = torch.zeros(1, dtype=torch.int32, device=gpu_device)
    for leaf in (v, v.detach().clone().requires_grad_()):
        with pytest.raises(RuntimeError, match="names no sequence"):
            pkg.gated_delta_rule_fn(q, k, leaf, g, beta, cu_seqlens=cu)
    out, final = pkg.gated_delta_rule_fn(q[:, :0], k[:, :0], v[:, :0], g[:, :0], beta[:, :0], return_final_states=True, cu_seqlens=cu)
    assert out.shape == (1, 0, 2, 16) and final.shape == (0, 2, 32, 16)


@pytest.mark.gpu
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_values_that_are_not_finite_stay_where_they_belong(pkg, gpu_device, value):
    """In one sequence's token of one head: the chunks in front of it, the other heads and the other sequences do not notice, packed or
    not, and neither do their gradients; tokens of no sequence may hold anything."""
    lengths = [100, 130, 64]
    cu = torch.tensor([3] + [3 + sum(lengths[:i + 1]) for i in range(3)], dtype=torch.int32, device=gpu_device)
    total = int(cu[-1]) + 5
    q, k, v, g, beta, _ = make(1, total, 2, 1, 32, 32, torch.bfloat16, gpu_device, l2norm=True)
    at = 3 + 100 + 70                                    # the second sequence's second chunk

    def run(v, k):
        leaves = [t.detach().clone().requires_grad_() for t in (q, k, v, g, beta)]
        out, final = pkg.gated_delta_rule_fn(*leaves, return_final_states=True, cu_seqlens=cu, qk_l2norm=True)
        return [out, *torch.autograd.grad(out, leaves, torch.ones_like(out)), final]
    clean = run(v, k)
    bad_v, bad_k = v.clone(), k.clone()
    bad_v[0, at, 1] = value
    for t in (bad_v, bad_k):
        t[0, :3] = value
        t[0, total - 5:] = value
    dirty = run(bad_v, bad_k)
    assert not torch.isfinite(dirty[0][0, at, 1]).any()
    for a, b in zip(dirty[:-1], clean[:-1]):             # per token
        assert torch.equal(a[:, :, 0], b[:, :, 0])       # the other head
        assert torch.equal(a[:, :103], b[:, :103]) and torch.equal(a[:, 233:], b[:, 233:])         # the other sequences
    assert torch.equal(dirty[0][:, :103 + 64], clean[0][:, :103 + 64])     # the chunk in front
    assert torch.equal(dirty[-1][[0, 2]], clean[-1][[0, 2]]) and torch.equal(dirty[-1][1, 0], clean[-1][1, 0])


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [40, 1500, 20000])
def test_rows_of_tiny_values_in_8_bits(pkg, gpu_device, dim):
    """Rows whose 448 / max|y| is no finite float32, or hardly one.  A weight that is a power of two scales a row exactly: the same 8 bits,
    and the same scale times that power, to half of float32's last unit, 2^-150, where it is not a normal number."""
    x = torch.randn(4, dim, generator=torch.Generator().manual_seed(2)).to(gpu_device)
    want, one = pkg.rms_norm_quant_fn(x, torch.ones(dim, device=gpu_device))
    for k in (99, 110, 122):
        y8, scales = pkg.rms_norm_quant_fn(x, torch.full((dim,), 2.0 ** -k, device=gpu_device))
        assert torch.equal(y8.view(torch.uint8), want.view(torch.uint8))
        assert ((scales.double() - one.double() * 2.0 ** -k).abs() <= 2.0 ** -150).all()


@pytest.mark.gpu
def test_torch_library(pkg, gpu_device):
    ops = torch.ops.DaoAILab
    checks = ("test_schema", "test_faketensor")
    q, k, v, g, beta, s0 = make(1, 70, 1, 2, 32, 16, torch.bfloat16, gpu_device, l2norm=True)
    final = torch.empty_like(s0)
    torch.library.opcheck(ops._gated_delta_rule_fwd_cpp, (q, k, v, g, beta, s0, None, final, 0.2, True), test_utils=checks)
    torch.library.opcheck(ops._gated_delta_rule_fwd_cpp, (q, k, v, g, beta, None, None, None, 0.2, True), test_utils=checks)
    torch.library.opcheck(ops._gated_delta_rule_update_cpp, (q, k, v, g, beta, s0, None, 0.2, True), test_utils=checks)
    x, w = torch.randn(3, 40, device=gpu_device).bfloat16(), torch.rand(40, device=gpu_device)
    torch.library.opcheck(ops._rms_norm_fwd_cpp, (x, w, x.float(), 1e-5), test_utils=checks)
    torch.library.opcheck(ops._rms_norm_bwd_cpp, (x, w, x, None, 1e-5), test_utils=checks)
    torch.library.opcheck(ops._rms_norm_quant_cpp, (x, w, None, 1e-5), test_utils=checks)
    y8, scales = pkg.rms_norm_quant_fn(x, w)
    torch.library.opcheck(ops._dequantize_rows_cpp, (y8, scales, torch.float16), test_utils=checks[1:])    # (the first multiplies its inputs)


@pytest.mark.gpu
def test_python_and_native_graphs_agree(pkg, gpu_device):
    """The graph recorded by the extension and the one of the Python functions, which functorch and torch.compile get."""
    from causal_conv1d.gated_delta_rule import GatedDeltaRuleFn
    from causal_conv1d.rms_norm import RMSNormFn
    leaves = [t.detach().clone().requires_grad_() for t in make(2, 90, 2, 2, 32, 48, torch.float16, gpu_device, l2norm=True)]
    q, k, v, g, beta, s0 = leaves
    native = pkg.gated_delta_rule_fn(q, k, v, g, beta, scale=0.5, initial_states=s0, return_final_states=True, qk_l2norm=True)
    python = GatedDeltaRuleFn.apply(q, k, v, g, beta, 0.5, s0, True, None, True)
    x, w, h = leaves[2].flatten(2), torch.rand(4 * 48, device=gpu_device, requires_grad=True), torch.randn(2, 90, 4 * 48, device=gpu_device, requires_grad=True)
    native += pkg.rms_norm_fn(x, w, residual=h)
    python += RMSNormFn.apply(x, w, h, 1e-5)
    seeds = [torch.randn_like(t) for t in python]
    for a, b in zip(native, python):
        assert torch.equal(a, b)
    for a, b in zip(torch.autograd.grad(native, leaves + [w, h], seeds), torch.autograd.grad(python, leaves + [w, h], seeds)):
        assert torch.equal(a, b)
