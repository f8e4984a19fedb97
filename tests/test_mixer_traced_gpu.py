"""The ops of the gated delta rule's training call against their shapes on fake tensors, and the decode step in a compiled function."""
import pytest
import torch

from test_gated_delta_rule_gpu import make

CHECKS = ("test_schema", "test_faketensor")


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [None, [70], [100, 0, 29], [1] * 9, [0, 0]])
@pytest.mark.parametrize("states", [False, True])
def test_forward_that_saves_and_backward(pkg, gpu_device, lengths, states):
    ops = torch.ops.DaoAILab
    total = 70 if lengths is None else sum(lengths)
    q, k, v, g, beta, s0 = make(2 if lengths is None else 1, total, 1, 2, 32, 16, torch.bfloat16, gpu_device, l2norm=True, sequences=lengths and len(lengths))
    cu = None if lengths is None else torch.tensor([0] + lengths).cumsum(0).to(torch.int32).to(gpu_device)
    s0 = s0 if states else None
    final = None if s0 is None else torch.empty_like(s0)
    args = (q, k, v, g, beta, s0, cu)
    # (what tokens that are not there left in `saved` is anybody's: its shape is compared, its bytes are not)
    torch.library.opcheck(ops._gated_delta_rule_fwd_save_cpp, args + (final, 0.2, True), test_utils=CHECKS[1:])
    out, saved = ops._gated_delta_rule_fwd_save_cpp(*args, final, 0.2, True)
    dout = torch.randn(out.shape, device=gpu_device).bfloat16()
    torch.library.opcheck(ops._gated_delta_rule_bwd_cpp, args + (saved, dout, None if s0 is None else torch.randn_like(s0), 0.2, True, states), test_utils=CHECKS)


@pytest.mark.gpu
def test_compiled_decode_step(pkg, gpu_device):
    """Traced whole by torch.compile (aot_eager): the same bits, in the output and in the state."""
    q, k, v, g, beta, s0 = make(3, 1, 1, 2, 32, 16, torch.bfloat16, gpu_device, l2norm=True)
    index = torch.tensor([2, -1, 0], dtype=torch.int32, device=gpu_device)

    def step(q, k, v, g, beta, state):
        return pkg.gated_delta_rule_update(q * 2, k, v, g, beta, state, state_indices=index, qk_l2norm=True) + 1
    a, b = s0.clone(), s0.clone()
    compiled = torch.compile(step, backend="aot_eager", fullgraph=True)
    for _ in range(2):
        assert torch.equal(step(q, k, v, g, beta, a), compiled(q, k, v, g, beta, b)) and torch.equal(a, b)
