"""Linear attention whose gates grow and fall, up to 32 together over any run of at most 256 tokens: every weight exp(G_i - G_j) that they make counts, whatever
lies between its two tokens.  One that two factors lift by e^64 out of less than e^-87 may be missing, e^-23 beside the token's own: less than the bound, which is
as in linear_cases.py."""
import pytest
import torch

import linear_cases as cases

BF16, FP32 = torch.bfloat16, torch.float32
pytestmark = pytest.mark.gpu


def gates(kind, seqlen, dev):
    g = torch.zeros(1, seqlen, 2, device=dev)
    if kind == "rise, then fall":                        # over a block's 64 tokens, and at once behind them: e^-9 is left
        g[:, 64:128], g[:, 128] = 31 / 64, -40.0
    elif kind == "fall, then rise":
        g[:, 70], g[:, 130:194] = -35.0, 31 / 64
    elif kind == "two rises":                            # with a fall between that only both make up for
        g[:, 40:60], g[:, 70], g[:, 100:120] = 31 / 20, -60.0, 31 / 20
    elif kind == "within 32":                            # and at their borders
        g[:, 33], g[:, 40], g[:, 94], g[:, 95], g[:, 97] = -95.0, 31.0, -31.0, 31.0, -85.0
    else:                                                # one head only, and a second segment
        g[:, 10:20, 1], g[:, 250:260, 1], g[:, 290, 1] = -9.0, 3.1, -30.0
    return g


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("dims", [(32, 32), (128, 64), (64, 128), (128, 128), (160, 48)])
@pytest.mark.parametrize("kind", ["rise, then fall", "fall, then rise", "two rises", "within 32", "over segments"])
def test_gates_that_grow(pkg, gpu_device, dtype, dims, kind):
    s = cases.inputs(gpu_device, 1, 320, 1, 2, *dims, dtype, states=False, seed=dims[0])
    s["g"] = gates(kind, 320, gpu_device)
    total = s["g"].double().cumsum(1)
    assert max((total[:, min(t + 1, 319):t + 257] - total[:, t:t + 1]).max().item() for t in range(320)) < 32
    cases.check(cases.run(pkg, s, dfinal=False), s, dfinal=False)
