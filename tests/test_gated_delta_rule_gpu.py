"""gated_delta_rule_fn and gated_delta_rule_update against the recurrence in 64 bits, token by token.

Tolerances.  out is rounded once to its type.  Everything else is carried to float32's precision: a value is formed from a few
sums of dim_k or 64 terms, each addition off by at most 2^-24 of a partial sum, and partial sums are at most a few times
the largest value of the result; 4 (dim_k + 64) 2^-24 of that largest value covers it, since errors decay with the
state that carries them (|k| <= 1 and beta < 1 let no direction of the state grow)."""
import pytest
import torch

HALF_ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def make(batch, seqlen, heads, group, dim_k, dim_v, dtype, dev, seed=0, l2norm=False, g_dtype=torch.float32, b_dtype=None, sequences=None):
    """Inputs as a mixer has them: q, k, v column slices of one buffer."""
    r = torch.Generator().manual_seed(seed + 1000 * seqlen + dim_k)
    hv = heads * group
    mixed = torch.randn(batch, seqlen, 2 * heads * dim_k + hv * dim_v, generator=r)
    if not l2norm:
        qk = mixed[..., :2 * heads * dim_k].unflatten(-1, (2 * heads, dim_k))
        qk /= qk.norm(dim=-1, keepdim=True).clamp_min(1e-3) * 1.01
    mixed = mixed.to(dtype).to(dev)
    q = mixed[..., :heads * dim_k].unflatten(-1, (heads, dim_k))
    k = mixed[..., heads * dim_k:2 * heads * dim_k].unflatten(-1, (heads, dim_k))
    v = mixed[..., 2 * heads * dim_k:].unflatten(-1, (hv, dim_v))
    g = (-0.5 * torch.rand(batch, seqlen, hv, generator=r) ** 3).to(g_dtype).to(dev)
    beta = torch.sigmoid(torch.randn(batch, seqlen, hv, generator=r)).to(b_dtype or dtype).to(dev)
    s0 = torch.randn(sequences or batch, hv, dim_k, dim_v, generator=r).to(dev)
    return q, k, v, g, beta, s0


def recurrence(q, k, v, g, beta, s0, l2norm=False, scale=None):
    from causal_conv1d.gated_delta_rule import gated_delta_rule_ref
    args = [t.double() for t in (q, k, v, g, beta)]
    return gated_delta_rule_ref(*args, scale=scale, initial_states=None if s0 is None else s0.double(), return_final_states=True, qk_l2norm=l2norm)


def close(got, want, dtype, dim_k, what=""):
    got, want = got.detach().double(), want.detach().double()
    assert got.shape == want.shape, what
    if want.numel() == 0:
        return
    tol = 1.01 * HALF_ULP[dtype] * want.abs() + 4 * (dim_k + 64) * 2.0 ** -24 * want.abs().max() + (6e-8 if dtype == torch.float16 else 0)
    worst = ((got - want).abs() / tol).max().item() if torch.isfinite(got).all() else float("inf")
    assert worst <= 1, "%s: %.3f of the tolerance" % (what, worst)


LENGTHS = [1, 2, 15, 16, 17, 63, 64, 65, 128, 200, 513]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("seqlen", LENGTHS)
@pytest.mark.parametrize("l2norm", [False, True])
def test_forward_lengths(pkg, gpu_device, dtype, seqlen, l2norm):
    q, k, v, g, beta, s0 = make(2, seqlen, 2, 2, 64, 64, dtype, gpu_device, l2norm=l2norm)
    out, final = pkg.gated_delta_rule_fn(q, k, v, g, beta, initial_states=s0, return_final_states=True, qk_l2norm=l2norm)
    want, want_final = recurrence(q, k, v, g, beta, s0, l2norm)
    assert out.dtype == dtype and final.dtype == torch.float32
    close(out, want, dtype, 64, "out")
    close(final, want_final, torch.float32, 64, "final")


@pytest.mark.gpu
@pytest.mark.parametrize("dim_k,dim_v", [(1, 1), (3, 5), (16, 16), (24, 40), (32, 33), (48, 80), (64, 128), (65, 64), (100, 7), (128, 128), (128, 256),
                                         (130, 66), (160, 144), (192, 192), (250, 100), (256, 512)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_forward_head_sizes(pkg, gpu_device, dim_k, dim_v, dtype):
    q, k, v, g, beta, s0 = make(1, 150, 2, 1, dim_k, dim_v, dtype, gpu_device)
    out, final = pkg.gated_delta_rule_fn(q, k, v, g, beta, initial_states=s0, return_final_states=True)
    want, want_final = recurrence(q, k, v, g, beta, s0)
    close(out, want, dtype, dim_k, "out")
    close(final, want_final, torch.float32, dim_k, "final")


@pytest.mark.gpu
@pytest.mark.parametrize("g_dtype,b_dtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.float16), (torch.float16, torch.bfloat16)])
@pytest.mark.parametrize("heads,group", [(1, 1), (3, 1), (2, 3), (1, 8)])
def test_forward_gate_types_and_shared_heads(pkg, gpu_device, g_dtype, b_dtype, heads, group):
    q, k, v, g, beta, _ = make(2, 90, heads, group, 32, 48, torch.bfloat16, gpu_device, g_dtype=g_dtype, b_dtype=b_dtype)
    out, final = pkg.gated_delta_rule_fn(q, k, v, g, beta, scale=0.3, return_final_states=True)
    want, want_final = recurrence(q, k, v, g, beta, None, scale=0.3)
    close(out, want, torch.bfloat16, 32, "out")
    close(final, want_final, torch.float32, 32, "final")


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [[0, 1, 64, 65, 0, 130, 7], [300], [1] * 20, [0, 0], [63, 64, 65, 0]])
@pytest.mark.parametrize("index_dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("with_states", [False, True])
def test_packed_sequences(pkg, gpu_device, lengths, index_dtype, with_states):
    total = sum(lengths)
    q, k, v, g, beta, s0 = make(1, total, 2, 2, 40, 24, torch.bfloat16, gpu_device, sequences=len(lengths))
    s0 = s0 if with_states else None
    cu = torch.tensor([0] + lengths, dtype=index_dtype).cumsum(0).to(index_dtype).to(gpu_device)
    out, final = pkg.gated_delta_rule_fn(q, k, v, g, beta, initial_states=s0, return_final_states=True, cu_seqlens=cu, qk_l2norm=True)
    assert final.shape == (len(lengths), 4, 40, 24)
    for i, (lo, hi) in enumerate(zip(cu.tolist()[:-1], cu.tolist()[1:])):
        first = None if s0 is None else s0[i:i + 1]
        if lo == hi:
            assert torch.equal(final[i], torch.zeros_like(final[i]) if s0 is None else s0[i])
            continue
        want, want_final = recurrence(*(t[:, lo:hi] for t in (q, k, v, g, beta)), first, True)
        close(out[:, lo:hi], want, torch.bfloat16, 40, "out of sequence %d" % i)
        close(final[i:i + 1], want_final, torch.float32, 40, "final of sequence %d" % i)


@pytest.mark.gpu
def test_tokens_of_no_sequence_give_zeros(pkg, gpu_device):
    q, k, v, g, beta, _ = make(1, 300, 1, 2, 32, 32, torch.bfloat16, gpu_device)
    cu = torch.tensor([40, 120, 250], dtype=torch.int32, device=gpu_device)
    out, final = pkg.gated_delta_rule_fn(q, k, v, g, beta, return_final_states=True, cu_seqlens=cu)
    want, want_final = recurrence(*(t[:, 120:250] for t in (q, k, v, g, beta)), None)
    close(out[:, 120:250], want, torch.bfloat16, 32)
    close(final[1:], want_final, torch.float32, 32)
    assert not out[:, :40].any() and not out[:, 250:].any()


@pytest.mark.gpu
def test_entries_outside_the_tokens_are_clamped(pkg, gpu_device):
    q, k, v, g, beta, _ = make(1, 100, 1, 1, 32, 32, torch.bfloat16, gpu_device)
    inside, outside = (torch.tensor(c, dtype=torch.int32, device=gpu_device) for c in ([0, 60, 100], [-5, 60, 400]))
    a = pkg.gated_delta_rule_fn(q, k, v, g, beta, return_final_states=True, cu_seqlens=inside)
    b = pkg.gated_delta_rule_fn(q, k, v, g, beta, return_final_states=True, cu_seqlens=outside)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.gpu
@pytest.mark.parametrize("seqlen", [5, 100])
def test_gates_that_forget_everything_or_learn_nothing(pkg, gpu_device, seqlen):
    q, k, v, g, beta, s0 = make(1, seqlen, 1, 2, 32, 32, torch.float32, gpu_device)
    g[:, 2, 0], g[:, 4, 1] = float("-inf"), torch.finfo(torch.float32).min
    beta[:, 3] = 0
    if seqlen > 70:
        g[:, 70, :], g[:, 71, 0], g[:, 90, 1] = float("-inf"), float("-inf"), -90.0
    out, final = pkg.gated_delta_rule_fn(q, k, v, g, beta, initial_states=s0, return_final_states=True)
    want, want_final = recurrence(q, k, v, g, beta, s0)
    close(out, want, torch.float32, 32)
    close(final, want_final, torch.float32, 32)


@pytest.mark.gpu
def test_strong_gates_keep_their_precision(pkg, gpu_device):
    """Decay of e^-8 a token: the sum over a chunk is 512, whose float32 spacing is 6e-5, but neighbours' differences are not
    to lose anything by that."""
    q, k, v, g, beta, s0 = make(1, 192, 1, 1, 64, 64, torch.float32, gpu_device)
    g.mul_(0).sub_(8 * torch.rand(g.shape, generator=torch.Generator().manual_seed(3)).to(gpu_device))
    out, final = pkg.gated_delta_rule_fn(q, k, v, g, beta, initial_states=s0, return_final_states=True)
    want, want_final = recurrence(q, k, v, g, beta, s0)
    close(out, want, torch.float32, 64)
    close(final, want_final, torch.float32, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("seqlen", [3, 130])
def test_layouts(pkg, gpu_device, seqlen):
    """Heads in front of tokens, rows off the vector grid, a last dimension that is not contiguous, states of other strides, the
    final states written over the initial ones."""
    q, k, v, g, beta, s0 = (t.contiguous() for t in make(2, seqlen, 2, 1, 48, 56, torch.bfloat16, gpu_device))
    want, final = pkg.gated_delta_rule_fn(q, k, v, g, beta, initial_states=s0, return_final_states=True)

    def heads_first(t):
        return t.transpose(1, 2).contiguous().transpose(1, 2)

    def shifted(t):
        wide = torch.zeros(*t.shape[:-1], t.shape[-1] + 5, dtype=t.dtype, device=t.device)
        wide[..., 3:3 + t.shape[-1]] = t
        return wide[..., 3:3 + t.shape[-1]]

    def last_strided(t):
        return t.transpose(-1, -2).contiguous().transpose(-1, -2)

    for f in (heads_first, shifted, last_strided):
        got, end = pkg.gated_delta_rule_fn(f(q), f(k), f(v), f(g), f(beta), initial_states=f(s0), return_final_states=True)
        assert torch.equal(got, want) and torch.equal(end, final), f
    into = shifted(s0)
    got, end = pkg.gated_delta_rule_fn(q, k, v, g, beta, initial_states=into, return_final_states=True, final_states_out=into)
    assert end is into and torch.equal(got, want) and torch.equal(into, final)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("seqlen", [0, 1, 3])
@pytest.mark.parametrize("dim_k,dim_v", [(128, 128), (64, 33), (7, 20), (256, 96)])
def test_update(pkg, gpu_device, dtype, seqlen, dim_k, dim_v):
    """seqlen 0 stands for tensors without a seqlen axis."""
    n = max(seqlen, 1)
    q, k, v, g, beta, s0 = make(5, n, 2, 2, dim_k, dim_v, dtype, gpu_device, l2norm=True)
    pool = torch.randn(9, 4, dim_k, dim_v, device=gpu_device)
    at = torch.tensor([7, -1, 0, 3, 8], dtype=torch.int32, device=gpu_device)
    live = [0, 2, 3, 4]
    pool[at[live].long()] = s0[live]
    before = pool.clone()
    args = [t[:, 0] if seqlen == 0 else t for t in (q, k, v, g, beta)]
    out = pkg.gated_delta_rule_update(*args, pool, state_indices=at, qk_l2norm=True)
    assert out.shape == args[2].shape and out.dtype == dtype
    want, want_state = recurrence(q, k, v, g, beta, s0, True)
    full = out.unsqueeze(1) if seqlen == 0 else out
    close(full[live], want[live], dtype, dim_k, "out")
    assert not full[1].any()
    close(pool[at[live].long()], want_state[live], torch.float32, dim_k, "state")
    untouched = [i for i in range(9) if i not in at.tolist()]
    assert torch.equal(pool[untouched], before[untouched])
    direct = s0.clone()
    again = pkg.gated_delta_rule_update(*args, direct, qk_l2norm=True)
    assert torch.equal((again.unsqueeze(1) if seqlen == 0 else again)[live], full[live]) and torch.equal(direct[live], pool[at[live].long()])


@pytest.mark.gpu
def test_update_continues_a_prefill(pkg, gpu_device):
    q, k, v, g, beta, _ = make(2, 140, 2, 2, 64, 64, torch.float32, gpu_device)
    whole, last = pkg.gated_delta_rule_fn(q, k, v, g, beta, return_final_states=True)
    head, state = pkg.gated_delta_rule_fn(*(t[:, :133] for t in (q, k, v, g, beta)), return_final_states=True)
    tail = torch.cat([pkg.gated_delta_rule_update(*(t[:, i] for t in (q, k, v, g, beta)), state).unsqueeze(1) for i in range(133, 140)], 1)
    close(torch.cat([head, tail], 1), whole, torch.float32, 64)
    close(state, last, torch.float32, 64)


@pytest.mark.gpu
def test_update_refuses_slots_that_do_not_exist(pkg, gpu_device):
    """An index past the last slot is padding, like a negative one."""
    q, k, v, g, beta, s0 = make(2, 1, 1, 1, 32, 32, torch.bfloat16, gpu_device)
    before = s0.clone()
    out = pkg.gated_delta_rule_update(q, k, v, g, beta, s0, state_indices=torch.tensor([2, -7], dtype=torch.int32, device=gpu_device))
    assert not out.any() and torch.equal(s0, before)


@pytest.mark.gpu
def test_empty(pkg, gpu_device):
    for batch, seqlen in ((0, 10), (2, 0), (0, 0)):
        q, k, v, g, beta, s0 = make(batch, seqlen, 1, 2, 16, 16, torch.bfloat16, gpu_device)
        out, final = pkg.gated_delta_rule_fn(q, k, v, g, beta, initial_states=s0, return_final_states=True)
        assert out.shape == (batch, seqlen, 2, 16) and torch.equal(final, s0)
        out, final = pkg.gated_delta_rule_fn(q, k, v, g, beta, return_final_states=True)
        assert not final.any()


@pytest.mark.gpu
def test_refusals(pkg, gpu_device):
    q, k, v, g, beta, s0 = make(2, 8, 2, 2, 16, 16, torch.bfloat16, gpu_device)
    fn = pkg.gated_delta_rule_fn
    with pytest.raises(RuntimeError, match="same dtype"):
        fn(q, k.float(), v, g, beta)
    with pytest.raises(RuntimeError, match="must have shape"):
        fn(q, k[:, :4], v, g, beta)
    with pytest.raises(RuntimeError, match="must have shape"):
        fn(q, k, v, g[..., :2], beta)
    with pytest.raises(RuntimeError, match="multiple of the number of key heads"):
        fn(q, k, v[:, :, :3], g[..., :3], beta[..., :3])
    with pytest.raises(RuntimeError, match="must be float32"):
        fn(q, k, v, g, beta, initial_states=s0.bfloat16())
    with pytest.raises(RuntimeError, match="batch of 1"):
        fn(q, k, v, g, beta, cu_seqlens=torch.tensor([0, 8], dtype=torch.int32, device=gpu_device))
    with pytest.raises(RuntimeError, match="int32 or int64"):
        fn(q[:1], k[:1], v[:1], g[:1], beta[:1], cu_seqlens=torch.tensor([0., 8.], device=gpu_device))
    with pytest.raises(RuntimeError, match="GPU"):
        fn(q, k.cpu(), v, g, beta)
    big = torch.zeros(1, 2, 1, 257, dtype=torch.bfloat16, device=gpu_device)
    with pytest.raises(RuntimeError, match="dim_k <= 256"):
        fn(big, big, v[:1, :2, :1], g[:1, :2, :1], beta[:1, :2, :1])
    with pytest.raises(RuntimeError, match="int32"):
        pkg.gated_delta_rule_update(q, k, v, g, beta, s0, state_indices=torch.zeros(2, dtype=torch.int64, device=gpu_device))
    with pytest.raises(RuntimeError, match="must have shape"):
        pkg.gated_delta_rule_update(q, k, v, g, beta, s0[:1])
