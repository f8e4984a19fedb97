"""Gradients of gated_delta_rule_fn against automatic differentiation of the recurrence in 64 bits, and against differences.

Tolerances, of the 2-norm of a gradient's error against the gradient's.  All sums are carried to float32's precision, 2^-24 of a
term each; the longest chain of additions behind a value is that of dg, 64 tokens of dim_k + dim_v + 64 terms, and errors
that are independent of each other grow with the root of their number: sqrt(64 (dim_k + dim_v + 64)) 2^-24, about 8e-6 at
128 x 128.  What is stored in 16 bits is rounded once more, by at most half a unit in the last place."""
import pytest
import torch

from test_gated_delta_rule_gpu import DTYPES, HALF_ULP, make

NAMES = ["q", "k", "v", "g", "beta", "states"]


def gradients64(args, dout, dfinal, l2norm, scale=None):
    from causal_conv1d.gated_delta_rule import gated_delta_rule_ref
    wide = [None if t is None else t.detach().double().requires_grad_() for t in args]
    out, final = gated_delta_rule_ref(*wide[:5], scale=scale, initial_states=wide[5], return_final_states=True, qk_l2norm=l2norm)
    loss = (out * dout.double()).sum() + (0 if dfinal is None else (final * dfinal.double()).sum())
    some = [t for t in wide if t is not None]
    return [torch.zeros_like(t) if d is None else d for t, d in zip(some, torch.autograd.grad(loss, some, allow_unused=True))]


def gradients(pkg, args, dout, dfinal, l2norm, scale=None, cu=None):
    some = [None if t is None else t.detach().requires_grad_() for t in args]
    res = pkg.gated_delta_rule_fn(*some[:5], scale=scale, initial_states=some[5], return_final_states=dfinal is not None, cu_seqlens=cu, qk_l2norm=l2norm)
    outs, given = ([res], [dout]) if dfinal is None else (list(res), [dout, dfinal])
    return torch.autograd.grad(outs, [t for t in some if t is not None], given)


def near(got, want, dim_k, dim_v, what):
    assert got.shape == want.shape, what
    if want.numel() == 0:
        return
    limit = (64.0 * (dim_k + dim_v + 64)) ** 0.5 * 2.0 ** -24 + (HALF_ULP[got.dtype] if got.dtype != torch.float32 else 0)
    # fp16 cannot hold less than 2^-25 of its own, which adds up over a tensor of small gradients.
    floor = 2.0 ** -25 * want.numel() ** 0.5 if got.dtype == torch.float16 else 1e-30
    off = (got.double() - want).norm().item()
    assert off <= limit * want.norm().item() + floor, "%s: %.3e of %.3e" % (what, off / max(want.norm().item(), 1e-300), limit)


def check(pkg, dev, batch, seqlen, heads, group, dim_k, dim_v, dtype, l2norm, states, seed=0, **types):
    q, k, v, g, beta, s0 = make(batch, seqlen, heads, group, dim_k, dim_v, dtype, dev, seed=seed, l2norm=l2norm, **types)
    r = torch.Generator().manual_seed(seed + 77)
    dout = torch.randn(v.shape, generator=r).to(dtype).to(dev)
    dfinal = torch.randn(s0.shape, generator=r).to(dev) if states else None
    args = [q, k, v, g, beta, s0 if states else None]
    got, want = gradients(pkg, args, dout, dfinal, l2norm), gradients64(args, dout, dfinal, l2norm)
    assert len(got) == len(want)
    for name, a, b, t in zip(NAMES, got, want, args):
        assert a.dtype == t.dtype
        near(a, b, dim_k, dim_v, "d" + name)


@pytest.mark.gpu
@pytest.mark.parametrize("seqlen", [1, 2, 17, 63, 64, 65, 128, 200])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("states", [False, True])
def test_lengths(pkg, gpu_device, seqlen, dtype, states):
    check(pkg, gpu_device, 2, seqlen, 2, 2, 64, 48, dtype, True, states)


@pytest.mark.gpu
@pytest.mark.parametrize("dim_k,dim_v", [(1, 1), (3, 5), (16, 16), (24, 40), (32, 33), (48, 80), (65, 64), (100, 7), (128, 128), (128, 256), (130, 66),
                                         (250, 100), (256, 256), (64, 512)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_head_sizes(pkg, gpu_device, dim_k, dim_v, dtype):
    check(pkg, gpu_device, 1, 100, 2, 1, dim_k, dim_v, dtype, False, True)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,group", [(1, 1), (3, 1), (2, 3), (1, 8)])
@pytest.mark.parametrize("l2norm", [False, True])
def test_shared_heads(pkg, gpu_device, heads, group, l2norm):
    check(pkg, gpu_device, 2, 90, heads, group, 32, 48, torch.float32, l2norm, True)
    check(pkg, gpu_device, 2, 90, heads, group, 32, 48, torch.bfloat16, l2norm, True, g_dtype=torch.float16, b_dtype=torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [[0, 1, 64, 65, 0, 130, 7], [300], [1] * 9])
@pytest.mark.parametrize("states", [False, True])
def test_packed_sequences(pkg, gpu_device, lengths, states):
    total = sum(lengths)
    q, k, v, g, beta, s0 = make(1, total, 2, 2, 40, 24, torch.bfloat16, gpu_device, sequences=len(lengths))
    cu = torch.tensor([0] + lengths).cumsum(0).to(torch.int32).to(gpu_device)
    r = torch.Generator().manual_seed(5)
    dout = torch.randn(v.shape, generator=r).bfloat16().to(gpu_device)
    dfinal = torch.randn(s0.shape, generator=r).to(gpu_device) if states else None
    args = [q, k, v, g, beta, s0 if states else None]
    got = gradients(pkg, args, dout, dfinal, True, cu=cu)
    want = [torch.zeros(t.shape, dtype=torch.float64, device=gpu_device) for t in args if t is not None]
    for i, (lo, hi) in enumerate(zip(cu.tolist()[:-1], cu.tolist()[1:])):
        if lo == hi:
            if states:
                want[5][i] = dfinal[i]
            continue
        part = [t[:, lo:hi] for t in args[:5]] + [s0[i:i + 1] if states else None]
        for j, d in enumerate(gradients64(part, dout[:, lo:hi], None if dfinal is None else dfinal[i:i + 1], True)):
            if j < 5:
                want[j][:, lo:hi] = d
            else:
                want[5][i:i + 1] = d
    for name, a, b in zip(NAMES, got, want):
        near(a, b, 40, 24, "d" + name)


@pytest.mark.gpu
def test_tokens_of_no_sequence_have_no_gradient(pkg, gpu_device):
    q, k, v, g, beta, _ = make(1, 200, 1, 2, 32, 32, torch.bfloat16, gpu_device)
    cu = torch.tensor([70, 150], dtype=torch.int32, device=gpu_device)
    got = gradients(pkg, [q, k, v, g, beta, None], torch.ones_like(v), None, True, cu=cu)
    want = gradients64([t[:, 70:150] for t in (q, k, v, g, beta)] + [None], torch.ones_like(v[:, 70:150]), None, True)
    for name, a, b in zip(NAMES, got, want):
        assert not a[:, :70].any() and not a[:, 150:].any(), name
        near(a[:, 70:150], b, 32, 32, name)


@pytest.mark.gpu
def test_gates_that_forget_everything_or_learn_nothing(pkg, gpu_device):
    q, k, v, g, beta, s0 = make(1, 140, 1, 2, 32, 32, torch.float32, gpu_device)
    g[:, 2, 0], g[:, 4, 1], g[:, 70], g[:, 90, 1] = float("-inf"), torch.finfo(torch.float32).min, float("-inf"), -90.0
    beta[:, 3], beta[:, 100] = 0, 0
    dout, dfinal = torch.randn_like(v), torch.randn_like(s0)
    args = [q, k, v, g, beta, s0]
    # In 64 bits too, exp(-inf) (-inf's gradient is 0 times something finite) is taken at a gate whose exponential is 0.
    want = gradients64([q, k, v, g.clamp_min(-1000.), beta, s0], dout, dfinal, False)
    for name, a, b in zip(NAMES, gradients(pkg, args, dout, dfinal, False), want):
        near(a, b, 32, 32, "d" + name)


@pytest.mark.gpu
def test_against_differences(pkg, gpu_device):
    """Central differences of the forward in float32, step 0.02 along random directions: off by the third derivative's share,
    about s^2 of the gradient, and by the forward's rounding over the step, sqrt(n) 2^-24 / s: 2e-3 of the gradient covers both."""
    q, k, v, g, beta, s0 = (t.contiguous() for t in make(1, 70, 1, 2, 24, 20, torch.float32, gpu_device))
    r = torch.Generator().manual_seed(3)
    dout, dfinal = torch.randn(v.shape, generator=r).to(gpu_device), torch.randn(s0.shape, generator=r).to(gpu_device)
    args = [q, k, v, g, beta, s0]
    grads = gradients(pkg, args, dout, dfinal, True)

    def loss(a):
        out, final = pkg.gated_delta_rule_fn(*a[:5], initial_states=a[5], return_final_states=True, qk_l2norm=True)
        return float((out.double() * dout.double()).sum() + (final.double() * dfinal.double()).sum())

    for i, grad in enumerate(grads):
        for seed in range(2):
            d = torch.randn(grad.shape, generator=torch.Generator().manual_seed(seed)).to(gpu_device)
            d /= d.norm()
            up, down = ([t + s * d if j == i else t for j, t in enumerate(args)] for s in (0.02, -0.02))
            slope = (loss(up) - loss(down)) / 0.04
            assert abs(slope - float((grad.double() * d.double()).sum())) < 2e-3 * float(grad.norm()), NAMES[i]


@pytest.mark.gpu
def test_gradients_through_broadcast_and_strided_inputs(pkg, gpu_device):
    """Gates shared by all heads (expanded), q, k and v cut from one buffer, dout expanded: autograd adds up what belongs together."""
    buf = torch.randn(2, 80, 3 * 64, device=gpu_device).requires_grad_()
    gate = (-torch.rand(2, 80, 1, device=gpu_device)).requires_grad_()

    def heads(b, wide):
        b = b.to(wide)
        q, k, v = (t.unflatten(-1, (2, 32)) for t in b.split(64, -1))
        return torch.nn.functional.normalize(q, dim=-1), torch.nn.functional.normalize(k, dim=-1), v

    out = pkg.gated_delta_rule_fn(*heads(buf, torch.float32), gate.expand(2, 80, 2), torch.sigmoid(gate).expand(2, 80, 2))
    got = torch.autograd.grad(out.sum(), [buf, gate])
    from causal_conv1d.gated_delta_rule import gated_delta_rule_ref
    b64, g64 = buf.detach().double().requires_grad_(), gate.detach().double().requires_grad_()
    ref = gated_delta_rule_ref(*heads(b64, torch.float64), g64.expand(2, 80, 2), torch.sigmoid(g64).expand(2, 80, 2))
    for a, b in zip(got, torch.autograd.grad(ref.sum(), [b64, g64])):
        near(a, b, 32, 32, "gradient")


@pytest.mark.gpu
def test_unused_outputs(pkg, gpu_device):
    q, k, v, g, beta, s0 = make(1, 70, 1, 1, 32, 32, torch.bfloat16, gpu_device)
    args = [t.detach().requires_grad_() for t in (q, k, v, g, beta, s0)]
    out, final = pkg.gated_delta_rule_fn(*args[:5], initial_states=args[5], return_final_states=True)
    only_final = torch.autograd.grad(final.sum(), args, retain_graph=True)
    both = torch.autograd.grad([out, final], args, [torch.zeros_like(out), torch.ones_like(final)], retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(only_final, both))
    only_out = torch.autograd.grad(out.float().sum(), args)
    plain = torch.autograd.grad(pkg.gated_delta_rule_fn(*args[:5], initial_states=args[5]).float().sum(), args)
    assert all(torch.equal(a, b) for a, b in zip(only_out, plain))


@pytest.mark.gpu
def test_same_bits_every_time(pkg, gpu_device):
    q, k, v, g, beta, s0 = make(2, 500, 2, 2, 64, 64, torch.bfloat16, gpu_device)
    dout, dfinal = torch.randn_like(v), torch.randn_like(s0)
    runs = [gradients(pkg, [q, k, v, g, beta, s0], dout, dfinal, True) for _ in range(3)]
    assert all(torch.equal(a, b) for run in runs[1:] for a, b in zip(runs[0], run))


@pytest.mark.gpu
def test_empty(pkg, gpu_device):
    for batch, seqlen in ((0, 10), (2, 0)):
        q, k, v, g, beta, s0 = make(batch, seqlen, 1, 2, 16, 16, torch.bfloat16, gpu_device)
        dfinal = torch.randn_like(s0)
        got = gradients(pkg, [q, k, v, g, beta, s0], torch.zeros_like(v), dfinal, False)
        assert all(a.shape == t.shape for a, t in zip(got, (q, k, v, g, beta, s0))) and torch.equal(got[5], dfinal)


@pytest.mark.gpu
def test_refusals(pkg, gpu_device):
    q, k, v, g, beta, s0 = (t.requires_grad_() for t in make(1, 70, 1, 1, 32, 32, torch.bfloat16, gpu_device))
    with pytest.raises(RuntimeError, match="where gradients are recorded"):
        pkg.gated_delta_rule_fn(q, k, v, g, beta, return_final_states=True, final_states_out=torch.empty_like(s0))
