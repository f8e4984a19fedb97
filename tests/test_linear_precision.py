"""How many bits the gradients of beta and of the gates keep, which are fp32 whatever q, k and v are: errors over all elements together, against 64 bits.

dbeta[j] is the sum over i of E_ij (dout_i.v_j) (q_i.k_j), E_ij = exp(G_i - G_j).  With 2^-25.3 for the mean square of a rounding to 24 bits, E is a product of
two or three exponentials (2^-23.9 each with the last rounding of its own, 2^-23 at worst) and meets three more products: 2^-23.1.  Sums: 2^-24.3 for
dout.v, four steps of 32 columns; 2^-23.8 for the rows times z, eight steps of 32 tokens; 2^-24.3 for the products inside a lane.  Together 2^-22.7; twice
that is the bound.

dg is a running sum, over 256 tokens at most, of what token t reads less what it wrote, without its own share in either: dg[t] - dg[t+1], each side
with the error above.  Closed at both ends of a segment, the running sum of n independent errors is off by sqrt(n / 6) of one, and no token's by more than
those in front of it make.  Where gates are strong
a token's own share is nearly all of q.dq and of k.dk, and nothing of dg.

States and their gradients: a segment's decay is one exponential for all elements, 2^-22.4 off at worst.  With two segments' and the sums above 2^-21.1."""
import pytest
import torch

import linear_cases as cases

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
DBETA, STATES = 2.0 ** -21.7, 2.0 ** -21.1


def bound_of_dg(want):
    return DBETA * (256 / 6) ** 0.5 * (torch.diff(want, dim=1).norm() / want.norm()).item()


def off(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


def forgetting_gates(*shape, generator, dev="cpu"):
    """Nearly nothing forgotten, but for one token of every 32, which forgets all: what decides E among the others is a difference of sums near -40."""
    g = -0.05 * torch.rand(*shape, generator=generator, device=dev)
    g[:, 3::32] = -35 - 10 * torch.rand(g[:, 3::32].shape, generator=generator, device=dev)
    return g


def modelled(arguments, terms, n=64, dim=128):
    """dbeta of 64 tokens with E as a product of two exponentials inside 32 tokens and the weighted products in `terms` bfloat16, all else in 64 bits."""
    r = torch.Generator().manual_seed(1)
    q, k, v, dout = (torch.randn(n, dim, generator=r).bfloat16().double() for _ in range(4))
    total = forgetting_gates(1, n, generator=r)[0].double().cumsum(0)
    want, got = torch.zeros(n, dtype=torch.float64), torch.zeros(n, dtype=torch.float64)
    for lo in range(0, n, 32):
        s = slice(lo, lo + 32)
        since = total[s] - (total[lo - 1] if lo else 0.0)
        w, a = (dout[s] @ v[s].T).tril(), q[s] @ k[s].T
        exact = w * (since[:, None] - since[None, :]).tril().exp()
        arg = since.to(arguments).double()
        p = w * (arg.exp()[:, None] * (-arg).exp()[None, :])
        kept = torch.zeros_like(p)
        for _ in range(terms):
            kept += (p - kept).bfloat16().double()
        want[s], got[s] = (exact * a).sum(0), (kept * a).sum(0)
    return off(got, want)


def test_the_bound_sees_what_it_is_for():
    """Arguments rounded to 24 bits, or two terms where three belong, are beyond it; what the kernels mean to do is inside."""
    assert modelled(torch.float64, 3) < DBETA
    assert modelled(torch.float32, 3) > 2 * DBETA and modelled(torch.float64, 2) > 2 * DBETA


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("dims", [(64, 64), (128, 64), (64, 128), (128, 128), (160, 96)])
@pytest.mark.parametrize("heads", [(2, 2), (1, 3)])
def test_weights_gradient_behind_strong_gates(pkg, gpu_device, dtype, dims, heads):
    s = cases.inputs(gpu_device, 1, 320, *heads, *dims, dtype, states=False, seed=dims[0])
    s["g"] = forgetting_gates(1, 320, heads[1], generator=torch.Generator(device=gpu_device).manual_seed(2), dev=gpu_device)
    s["beta"] = s["beta"].float()
    got, want = cases.run(pkg, s, dfinal=False), cases.reference(s, dfinal=False)
    assert off(got["dbeta"], want["dbeta"]) <= DBETA, off(got["dbeta"], want["dbeta"])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("dims", [(64, 64), (128, 64), (64, 128), (128, 128), (160, 96), (96, 192)])
@pytest.mark.parametrize("rate", [0.02, 0.3, 1.6, 5.0])
def test_gates_gradient(pkg, gpu_device, dtype, dims, rate):
    s = cases.inputs(gpu_device, 1, 320, 1, 2, *dims, dtype, seed=dims[0])
    s["g"] = -rate * (0.9 + 0.2 * torch.rand(1, 320, 2, generator=torch.Generator(device=gpu_device).manual_seed(3), device=gpu_device))
    s["beta"] = s["beta"].float()
    got, want = cases.run(pkg, s), cases.reference(s)
    assert off(got["dg"], want["dg"]) <= bound_of_dg(want["dg"]), (off(got["dg"], want["dg"]), bound_of_dg(want["dg"]))
    assert off(got["dbeta"], want["dbeta"]) <= DBETA, off(got["dbeta"], want["dbeta"])
    assert off(got["final"], want["final"]) <= STATES and off(got["dstates"], want["dstates"]) <= STATES, (off(got["final"], want["final"]), off(got["dstates"], want["dstates"]))


@pytest.mark.gpu
@pytest.mark.parametrize("dims", [(32, 32), (72, 72)])
def test_gates_gradient_of_many_heads(pkg, gpu_device, dims):
    """Several value heads a workgroup, several workgroups a key head."""
    s = cases.inputs(gpu_device, 4, 200, 1, 80, *dims, BF16, states=False)
    s["g"], s["beta"] = s["g"] * 40, s["beta"].float()
    got, want = cases.run(pkg, s, dfinal=False), cases.reference(s, dfinal=False)
    assert off(got["dg"], want["dg"]) <= bound_of_dg(want["dg"])
    assert off(got["dbeta"], want["dbeta"]) <= DBETA
    cases.check(got, s, dfinal=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("dims", [(64, 64), (128, 128), (160, 96)])
def test_gates_gradient_in_front_of_larger_ones(pkg, gpu_device, dtype, dims):
    """Strong gates with small gradients, and behind them, in the same segment, weak ones with gradients some thousand times as large.  (Behind larger ones
    the running sum keeps their error.)"""
    s = cases.inputs(gpu_device, 1, 320, 1, 2, *dims, dtype, states=False, seed=dims[0])
    s["g"][:, :128] = s["g"][:, :128] - 6.0
    s["beta"] = s["beta"].float()
    got, want = cases.run(pkg, s, dfinal=False)["dg"][:, :128], cases.reference(s, dfinal=False)["dg"][:, :128]
    assert off(got, want) <= bound_of_dg(want), (off(got, want), bound_of_dg(want))
