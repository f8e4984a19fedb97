"""Linear attention whose states lie by borders between segments, or by segments where there are states in front or behind: no result comes out of memory that
the call has not written, and no two states share a place."""
import pytest
import torch

import linear_cases as cases

BF16, FP32 = torch.bfloat16, torch.float32
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("states,dfinal", [(False, False), (False, True), (True, False), (True, True)])
@pytest.mark.parametrize("cu", [None, [0, 1300], [0, 0, 255, 256, 513, 770, 1026, 1026, 1300], [0, 3, 700, 701, 1299, 1300], [0, 256, 512, 1024, 1300], list(range(0, 1301, 100))])
def test_states_by_borders(pkg, gpu_device, dtype, states, dfinal, cu):
    """Borders on and beside the 256 tokens that name them; against 64 bits, and the same bits whatever the memory held."""
    s = cases.inputs(gpu_device, 1 if cu else 2, 1300, 1, 2, 32, 48, dtype, states=states, sequences=len(cu) - 1 if cu else 0, seed=3)
    got = cases.run(pkg, s, cu, dfinal=dfinal)
    cases.check(got, s, cu, dfinal=dfinal)
    del got["final"]
    torch.cuda.empty_cache()
    for fill in (float("nan"), 0.0):
        before = [torch.full((1 << 24,), fill, device=gpu_device), torch.full((1 << 18,), fill, device=gpu_device)]
        del before
        again = cases.run(pkg, s, cu, dfinal=dfinal)
        for n, t in got.items():
            assert torch.equal(t, again[n]), n


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("states", [True, False])
def test_each_by_its_own_length_by_borders(pkg, gpu_device, dtype, states):
    """Without gradients: long sequences among many short ones."""
    cu = [0] + list(range(5, 305, 5)) + [561, 1300, 1303, 1304, 1900]
    s = cases.inputs(gpu_device, 1, 1900, 1, 2, 32, 48, dtype, states=states, sequences=len(cu) - 1, seed=4)
    got = cases.run(pkg, s, cu, grads=False)
    cases.check(got, s, cu, grads=False)
    torch.cuda.empty_cache()
    before = torch.full((1 << 24,), float("nan"), device=gpu_device)
    del before
    at = torch.tensor(cu, dtype=torch.int32, device=gpu_device)
    assert torch.equal(pkg.linear_attention_fn(s["q"], s["k"], s["v"], s["g"], beta=s["beta"], initial_states=s["states"], cu_seqlens=at), got["out"])
