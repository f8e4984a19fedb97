"""Linear attention with a decay for each head against its statement in 64 bits (linear_cases.py)."""
import pytest
import torch

import linear_cases as cases

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("seqlen", [1, 2, 15, 16, 63, 64, 65, 100, 129, 256, 257, 520])
def test_lengths(pkg, gpu_device, dtype, seqlen):
    """From one token on: token by token below 16, one segment, several, ends inside a block."""
    s = cases.inputs(gpu_device, 2, seqlen, 2, 4, 32, 48, dtype, seed=seqlen)
    cases.check(cases.run(pkg, s, grads=False), s, grads=False)
    cases.check(cases.run(pkg, s), s)


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("dims", [(1, 1), (3, 5), (16, 33), (31, 64), (48, 80), (64, 128), (96, 130), (128, 64), (130, 128), (192, 17), (256, 256), (64, 512), (256, 511)])
def test_head_sizes(pkg, gpu_device, dtype, dims):
    """Every number of 32-column steps, halves and tiles of columns; odd sizes are read by elements."""
    s = cases.inputs(gpu_device, 1, 330, 1, 2, *dims, dtype, seed=dims[0])
    cases.check(cases.run(pkg, s), s)


@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("heads", [(1, 1), (1, 7), (3, 3), (2, 10), (1, 80)])
@pytest.mark.parametrize("beta,states,decay", [(False, False, "token"), (True, False, "head"), (False, True, "head")])
def test_heads_and_options(pkg, gpu_device, dtype, heads, beta, states, decay):
    s = cases.inputs(gpu_device, 2, 300, *heads, 32, 32, dtype, decay=decay, beta=beta, states=states, seed=heads[1])
    cases.check(cases.run(pkg, s), s)
    cases.check(cases.run(pkg, s, dfinal=False), s, dfinal=False)


def test_shares_of_a_key_head(pkg, gpu_device):
    """Long enough that one workgroup takes several value heads, and several workgroups a key head: 16 x 4 x 4 x 80 value heads' blocks."""
    s = cases.inputs(gpu_device, 4, 1024, 1, 80, 16, 16, BF16, states=False)
    cases.check(cases.run(pkg, s, dfinal=False), s, dfinal=False)


@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("cu", [[0, 400], [0, 0, 1, 65, 65, 400, 400], [0, 256, 400], [0, 100, 200, 300, 400], [0, 399, 400], [7, 300, 350], [0, 3]])
@pytest.mark.parametrize("heads", [(2, 2), (1, 3)])
def test_packed_sequences(pkg, gpu_device, dtype, cu, heads):
    """Empty ones, single tokens, ends on and beside segments, tokens in front of the first and behind the last: those give zeros."""
    s = cases.inputs(gpu_device, 1, 400, *heads, 32, 64, dtype, sequences=len(cu) - 1, seed=len(cu))
    cases.check(cases.run(pkg, s, cu), s, cu)
    cases.check(cases.run(pkg, s, cu, grads=False, cu_dtype=torch.int64), s, cu, grads=False)


def test_many_short_sequences(pkg, gpu_device):
    cu = list(range(0, 601, 6))
    s = cases.inputs(gpu_device, 1, 600, 1, 2, 32, 32, BF16, sequences=100)
    cases.check(cases.run(pkg, s, cu), s, cu)
    cases.check(cases.run(pkg, s, cu, grads=False), s, cu, grads=False)


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_layouts(pkg, gpu_device, dtype):
    """Rows off the 16-byte and the pair grid, heads in front of tokens, gates with strides, a scale."""
    def check(s):
        cases.check(cases.run(pkg, s, scale=0.3), s, scale=0.3)
    base = cases.inputs(gpu_device, 2, 150, 2, 4, 32, 32, dtype)
    off = dict(base)
    for n in ("q", "k", "v"):
        wide = torch.zeros(*base[n].shape[:3], 37, dtype=dtype, device=gpu_device)
        wide[..., 1:33] = base[n]
        off[n] = wide[..., 1:33]
    check(off)
    turned = {n: t.transpose(1, 2).contiguous().transpose(1, 2) if n in ("q", "k", "v", "dout") else t for n, t in base.items()}
    check(turned)
    turned["g"], turned["beta"] = (base[n].transpose(1, 2).contiguous().transpose(1, 2) for n in ("g", "beta"))
    turned["states"], turned["dfinal"] = (base[n].transpose(0, 1).contiguous().transpose(0, 1) for n in ("states", "dfinal"))
    check(turned)
    check(dict(base, q=base["q"][:, :1].expand(-1, 150, -1, -1), g=base["g"].to(dtype), beta=base["beta"].half()))


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_strong_and_no_decay(pkg, gpu_device, dtype):
    """Gates from nothing forgotten to everything forgotten, in one sequence; and gates that grow."""
    s = cases.inputs(gpu_device, 1, 400, 1, 3, 32, 32, dtype)
    g = torch.zeros(1, 400, 3, device=gpu_device)
    g[:, ::7, 1] = -50.0
    g[:, 100, 1], g[:, 300:, 1] = -1e4, -1.0
    g[..., 2] = 0.05
    s["g"] = g
    cases.check(cases.run(pkg, s), s)


def test_minus_infinity_forgets(pkg, gpu_device):
    """exp(-inf) = 0: what stands in front of such a gate has no weight, and no gradient."""
    s = cases.inputs(gpu_device, 1, 200, 1, 2, 32, 32, FP32)
    s["g"][:, 70] = -float("inf")
    got = cases.run(pkg, s)
    tail = {n: t[:, 70:] if n in ("q", "k", "v", "g", "beta", "dout") else t for n, t in s.items()}
    tail["states"] = torch.zeros_like(s["states"])
    tail["g"] = tail["g"].clone()
    tail["g"][:, 0] = 0.0
    want = cases.run(pkg, tail)
    for n in ("out", "dq", "dk", "dv", "dbeta"):
        assert (got[n][:, 70:] - want[n]).abs().max() <= 2e-5 * want[n].abs().max(), n
    head = {n: t[:, :70] if n in ("q", "k", "v", "g", "beta", "dout") else t for n, t in s.items()}
    want = cases.run(pkg, head, dfinal=False)
    for n in ("out", "dq", "dk", "dv", "dbeta", "dstates"):
        t = got[n] if n == "dstates" else got[n][:, :70]
        assert (t - want[n]).abs().max() <= 2e-5 * want[n].abs().max(), n
    assert got["dg"].isfinite().all()


def test_first_gate_without_states(pkg, gpu_device):
    """Nothing stands in front of a sequence's first token: its gate's gradient is 0, not a rounding."""
    s = cases.inputs(gpu_device, 2, 300, 1, 2, 32, 32, BF16, states=False)
    assert torch.equal(cases.run(pkg, s)["dg"][:, 0], torch.zeros(2, 2, device=gpu_device))


def test_nan_stays_where_it_belongs(pkg, gpu_device):
    """From the start of its 64 tokens on, in its own head and sequence."""
    s = cases.inputs(gpu_device, 2, 400, 2, 2, 32, 32, BF16, slices=False)
    clean = cases.run(pkg, s, grads=False)
    s["v"][0, 150, 1, 3] = float("nan")
    got = cases.run(pkg, s, grads=False)
    assert torch.equal(got["out"][1], clean["out"][1]) and torch.equal(got["out"][0, :, 0], clean["out"][0, :, 0])
    assert torch.equal(got["out"][0, :128, 1], clean["out"][0, :128, 1])
    assert got["out"][0, 150:, 1, 3].isnan().all() and got["final"][0, 1, :, 3].isnan().all()
    assert torch.equal(got["final"][1], clean["final"][1]) and torch.equal(got["final"][0, 0], clean["final"][0, 0])


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("dims", [(1, 1), (33, 31), (64, 32), (128, 64), (256, 100)])
def test_update(pkg, gpu_device, dtype, dims):
    """Slots, padding, one token and a few, with and without beta: the state in place, other slots as they were."""
    for tokens, beta, decay in ((1, True, "token"), (1, False, "head"), (3, True, "token")):
        s = cases.inputs(gpu_device, 5, tokens, 2, 4, *dims, dtype, beta=beta, decay=decay, seed=tokens)
        state = torch.randn(9, 4, *dims, device=gpu_device)
        at = torch.tensor([4, -1, 0, 8, 9], dtype=torch.int32, device=gpu_device)
        live = [0, 2, 3]
        part = {n: t[live] if n in ("q", "k", "v", "beta", "dout") and t is not None else t for n, t in s.items()}
        part["g"] = s["g"] if decay == "head" else s["g"][live]
        part["states"] = state[[4, 0, 8]]
        now = state.clone()
        flat = tokens == 1
        one = (lambda t: None if t is None else t[:, 0]) if flat else (lambda t: t)
        out = pkg.linear_attention_update(one(s["q"]), one(s["k"]), one(s["v"]), s["g"] if decay == "head" else one(s["g"]), now,
                                          beta=one(s["beta"]), state_indices=at)
        out = out[:, None] if flat else out
        cases.check({"out": out[live], "final": now[[4, 0, 8]]}, part, grads=False)
        assert torch.equal(out[[1, 4]], torch.zeros_like(out[[1, 4]]))
        assert torch.equal(now[[1, 2, 3, 5, 6, 7]], state[[1, 2, 3, 5, 6, 7]])


def test_update_continues_a_prefill(pkg, gpu_device):
    s = cases.inputs(gpu_device, 2, 300, 1, 4, 64, 64, FP32, states=False)
    whole = cases.run(pkg, s, grads=False)
    head = {n: t[:, :290] if n in ("q", "k", "v", "g", "beta", "dout") else t for n, t in s.items()}
    state = cases.run(pkg, head, grads=False)["final"]
    for t in range(290, 300):
        out = pkg.linear_attention_update(*(s[n][:, t] for n in ("q", "k", "v", "g")), state, beta=s["beta"][:, t])
        # two sums of some 600 terms each, 2^-24 of their magnitudes; these are a few times the largest value
        assert (out - whole["out"][:, t]).abs().max() <= 600 * 2.0 ** -24 * 8 * whole["out"].abs().max()
    assert (state - whole["final"]).abs().max() <= 600 * 2.0 ** -24 * 8 * whole["final"].abs().max()


def test_states_in_place_and_truncated_sequences(pkg, gpu_device):
    """final_states_out may be the initial states; two halves are the whole."""
    s = cases.inputs(gpu_device, 1, 700, 1, 2, 32, 32, FP32)
    keep = s["states"].clone()
    whole = cases.run(pkg, s, grads=False)
    for cut in (5, 300):
        state = keep.clone()
        outs = []
        for lo, hi in ((0, cut), (cut, 700)):
            out, same = pkg.linear_attention_fn(*(s[n][:, lo:hi] for n in ("q", "k", "v", "g", "beta")), initial_states=state, return_final_states=True, final_states_out=state)
            assert same is state
            outs.append(out)
        part = {"out": torch.cat(outs, 1), "final": state}
        cases.check(part, dict(s, states=keep), grads=False)
        assert torch.equal(whole["final"].isfinite(), state.isfinite())


def test_same_bits_again_and_on_another_stream(pkg, gpu_device):
    s = cases.inputs(gpu_device, 2, 600, 1, 8, 64, 64, BF16)
    first = cases.run(pkg, s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = cases.run(pkg, s)
    torch.cuda.current_stream().wait_stream(side)
    third = cases.run(pkg, s)
    for n, t in first.items():
        assert torch.equal(t, second[n]) and torch.equal(t, third[n]), n


def test_gradients_against_differences(pkg, gpu_device):
    """fp32, central differences in a random direction: third derivatives' share (h^2) and the sums' rounding over 2 h, both below 1e-3 of the
    magnitude for these sizes."""
    s = cases.inputs(gpu_device, 1, 140, 1, 2, 16, 16, FP32)
    grads = cases.run(pkg, s)
    r = torch.Generator(device=gpu_device).manual_seed(5)
    for n in cases.NAMES:
        d = torch.randn(s[n].shape, generator=r, device=gpu_device)
        h = 2e-3

        def loss(sign):
            got = cases.run(pkg, dict(s, **{n: s[n] + sign * h * d}), grads=False)
            return ((got["out"] * s["dout"]).double().sum() + (got["final"] * s["dfinal"]).double().sum()).item()
        found, want = (loss(1) - loss(-1)) / (2 * h), (grads["d" + n].double() * d.double()).sum().item()
        size = (grads["d" + n].double() * d.double()).norm().item()
        assert abs(found - want) <= 2e-2 * size, (n, found, want)


def test_empty_calls(pkg, gpu_device):
    def zeros(*shape):
        return torch.zeros(*shape, device=gpu_device)
    for b, l, hv in ((0, 5, 2), (2, 0, 2), (2, 5, 0)):
        q, v, g, st = zeros(b, l, 1, 8).requires_grad_(), zeros(b, l, hv, 4).requires_grad_(), zeros(b, l, hv), torch.randn(b, hv, 8, 4, device=gpu_device).requires_grad_()
        out, final = pkg.linear_attention_fn(q, q, v, g, initial_states=st, return_final_states=True)
        assert out.shape == v.shape and (l > 0 or torch.equal(final, st))
        dq, dst = torch.autograd.grad([out, final], [q, st], [zeros(b, l, hv, 4), torch.ones_like(final)])
        assert torch.equal(dq, torch.zeros_like(dq)) and (l > 0 or torch.equal(dst, torch.ones_like(dst)))
    cu = torch.tensor([0, 0, 0], dtype=torch.int32, device=gpu_device)
    st = torch.randn(2, 1, 8, 4, device=gpu_device)
    out, final = pkg.linear_attention_fn(zeros(1, 0, 1, 8), zeros(1, 0, 1, 8), zeros(1, 0, 1, 4), zeros(1, 0, 1), initial_states=st, return_final_states=True, cu_seqlens=cu)
    assert torch.equal(final, st)
