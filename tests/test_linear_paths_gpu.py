"""Linear attention's ways of a call (by tokens, by segments, each sequence by its own length), far and large memory, refusals, traced calls,
and the operators together.  Tolerances are those of linear_cases.py where nothing else is said."""
import pytest
import torch

import linear_cases as cases

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
pytestmark = pytest.mark.gpu

RAGGED = {
    "one_long": [1] * 40 + [300] + [1] * 40,
    "edges": [255, 256, 257, 1, 0, 511, 512, 513] + [2] * 300,
    "long_ends": [600] + [0, 1, 3] * 40 + [400],
    "empty_ones": [0] * 100 + [600] + [0] * 70,
    "neighbours": [256, 256, 257, 258, 300] + [1] * 150,
    "none_long": [20] * 3 + [10] * 60,
    "many": [1] * 4500 + [320] + [0] * 30 + [270],
}


@pytest.mark.parametrize("name", list(RAGGED))
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("front,behind", [(0, 0), (5, 70)])
def test_each_by_its_own_length(pkg, gpu_device, name, dtype, front, behind):
    """Packed sequences that are short on average with long ones among them; states in place; tokens of no sequence give zeros."""
    lengths = RAGGED[name]
    total = front + sum(lengths) + behind
    s = cases.inputs(gpu_device, 1, total, 1, 2, 40, 24, dtype, sequences=len(lengths), seed=len(name))
    cu = torch.tensor([front] + lengths).cumsum(0).to(torch.int32 if front else torch.int64).to(gpu_device)
    state = s["states"].clone()
    out, final = pkg.linear_attention_fn(s["q"], s["k"], s["v"], s["g"], beta=s["beta"], initial_states=state, return_final_states=True, final_states_out=state, cu_seqlens=cu)
    assert final is state and not out[:, :front].any() and not out[:, total - behind:].any()
    edges = cu.tolist()
    by_length = {}
    for i, n in enumerate(lengths):
        by_length.setdefault(n, []).append(i)
    for n, which in by_length.items():                   # sequences of a length as one batch
        if n == 0:
            assert torch.equal(final[which], s["states"][which])
            continue
        part = {m: torch.cat([s[m][:, edges[i]:edges[i] + n] for i in which]) for m in ("q", "k", "v", "g", "beta", "dout")}
        part["states"] = s["states"][which]
        cases.check({"out": torch.cat([out[:, edges[i]:edges[i] + n] for i in which]), "final": final[which]}, part, grads=False)


@pytest.mark.parametrize("dtype,batch,v_heads,seqlen", [(FP32, 4, 128, 40), (FP32, 2, 256, 120), (BF16, 8, 128, 49), (BF16, 8, 128, 50)])
def test_many_heads(pkg, gpu_device, dtype, batch, v_heads, seqlen):
    """States that fill the card, by tokens and by segments."""
    s = cases.inputs(gpu_device, batch, seqlen, 2, v_heads, 128, 128, dtype)
    cases.check(cases.run(pkg, s, grads=False), s, grads=False)


@pytest.mark.parametrize("seqlen", [1, 15, 16, 21, 22, 23, 31, 32])
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_the_same_with_and_without_gradients(pkg, gpu_device, dtype, seqlen):
    """A training call goes by segments at any length, an inference call by tokens below some: both within their bounds of the statement."""
    s = cases.inputs(gpu_device, 2, seqlen, 1, 2, 64, 64, dtype)
    for grads in (False, True):
        cases.check(cases.run(pkg, s, grads=grads), s, grads=grads)


@pytest.mark.parametrize("name", ["q", "k", "v"])
def test_tokens_far_apart(pkg, gpu_device, name):
    """2^23 bytes between tokens: by tokens, to the same bounds; where gradients are recorded the call is refused."""
    s = cases.inputs(gpu_device, 1, 40, 1, 2, 32, 16, BF16, slices=False)
    t = s[name]
    far = torch.zeros((t.shape[1] - 1) * (1 << 22) + t[0, 0].numel(), device=gpu_device, dtype=BF16).as_strided(t.shape, (1 << 30, 1 << 22, t.shape[3], 1))
    far.copy_(t)
    s[name] = far
    cases.check(cases.run(pkg, s, grads=False), s, grads=False)
    with pytest.raises(RuntimeError):
        cases.run(pkg, s, grads=True)


def test_offsets_past_32_bits(pkg, gpu_device):
    """Batch entries and heads more than 2^31 elements apart, and a decode step on slots behind 2^32 bytes: the same bits as close together."""
    s = cases.inputs(gpu_device, 2, 270, 1, 2, 32, 64, BF16, slices=False)
    whole = cases.run(pkg, s)
    far = {}
    for name, axis in (("q", 0), ("k", 0), ("v", 2)):
        t = s[name]
        stride = list(t.stride())
        stride[axis] = (1 << 31) + 64
        room = torch.empty(sum((n - 1) * st for n, st in zip(t.shape, stride)) + 1, device=gpu_device, dtype=BF16)
        far[name] = room.as_strided(t.shape, stride)
        far[name].copy_(t)
    moved = cases.run(pkg, dict(s, **far))
    for n in whole:
        assert torch.equal(whole[n], moved[n]), n
    del far, moved, room
    states = torch.zeros(1100, 16, 256, 256, device=gpu_device)              # 4.6e9 bytes
    d = cases.inputs(gpu_device, 2, 1, 16, 16, 256, 256, BF16)
    states[[1099, 3]] = d["states"]
    close = d["states"].clone()
    at = torch.tensor([1099, 3], dtype=torch.int32, device=gpu_device)
    one = lambda n: d[n][:, 0]  # noqa: E731
    a = pkg.linear_attention_update(one("q"), one("k"), one("v"), one("g"), states, beta=one("beta"), state_indices=at)
    b = pkg.linear_attention_update(one("q"), one("k"), one("v"), one("g"), close, beta=one("beta"))
    assert torch.equal(a, b) and torch.equal(states[[1099, 3]], close) and not states[4].any() and not states[1098].any()


def test_large_output_of_one_call(pkg, gpu_device):
    """More than 2^31 elements of v and out: the last rows are those of a call on the last rows, with the state in front of them."""
    b, l, h, d = 1, 66000, 256, 128
    q, k = (torch.randn(b, l, 1, 16, device=gpu_device).bfloat16() for _ in range(2))
    v = torch.randn(b, 1000, h, d, device=gpu_device).bfloat16().repeat(1, 66, 1, 1)
    g = torch.full((h,), -0.05, device=gpu_device)
    assert v.numel() > 1 << 31
    out, final = pkg.linear_attention_fn(q, k, v, g, return_final_states=True)
    cut = 65536                                          # a whole number of segments: the same sums
    front, state = pkg.linear_attention_fn(q[:, :cut], k[:, :cut], v[:, :cut], g, return_final_states=True)
    rest, last = pkg.linear_attention_fn(q[:, cut:], k[:, cut:], v[:, cut:], g, initial_states=state, return_final_states=True)
    assert torch.equal(out[:, :cut], front) and torch.equal(out[:, cut:], rest) and torch.equal(final, last)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_two_calls_at_once(pkg, gpu_device, dtype):
    """Two training calls on two streams that wait for nothing of each other: the bits of each alone."""
    cases_ = [cases.inputs(gpu_device, 1, 700, 1, 8, 64, 64, dtype, seed=i) for i in range(2)]
    alone = [cases.run(pkg, s) for s in cases_]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        both = []
        for s, stream in zip(cases_, streams):
            with torch.cuda.stream(stream):
                both.append(cases.run(pkg, s))
        torch.cuda.synchronize()
        for a, b in zip(alone, both):
            for n in a:
                assert torch.equal(a[n], b[n]), n


def test_capture_is_refused(pkg, gpu_device):
    """As the other operators do: an error, and the stream works afterwards."""
    s = cases.inputs(gpu_device, 1, 64, 1, 2, 32, 32, BF16)
    x, w = torch.randn(4, 64, device=gpu_device), torch.ones(64, device=gpu_device)
    calls = (lambda: pkg.linear_attention_fn(s["q"], s["k"], s["v"], s["g"]),
             lambda: pkg.linear_attention_update(s["q"][:, 0], s["k"][:, 0], s["v"][:, 0], s["g"][:, 0], s["states"]), lambda: pkg.layer_norm_fn(x, w, w, residual=x))
    for call in calls:
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        refused = []
        with torch.cuda.graph(graph):
            x + 1
            try:
                call()
            except RuntimeError as e:
                refused.append(str(e))
        assert len(refused) == 1 and "captur" in refused[0]
        call()
        torch.cuda.synchronize()


def test_refusals(pkg, gpu_device):
    """Arguments that do not belong together, each an error before a launch."""
    s = cases.inputs(gpu_device, 2, 30, 2, 4, 16, 24, BF16)
    q, k, v, g, beta, st = (s[n] for n in ("q", "k", "v", "g", "beta", "states"))
    cu = torch.tensor([0, 30], dtype=torch.int32, device=gpu_device)
    fn, step = pkg.linear_attention_fn, pkg.linear_attention_update
    one = [t[:, 0] for t in (q, k, v, g)]
    wide = torch.zeros(2, 4, 16, 48, device=gpu_device)[..., ::2]
    index = torch.zeros(2, dtype=torch.int32, device=gpu_device)
    for call in (lambda: fn(q, k.float(), v, g), lambda: fn(q, k, v.half(), g), lambda: fn(q, k[:, :, :1], v, g), lambda: fn(q, k, v[:, :, :3], g[:, :, :3]),
                 lambda: fn(q, k, v, g[:, :29]), lambda: fn(q, k, v, g[0, 0, :3]), lambda: fn(q, k, v, g, beta=beta[:, :, :2]), lambda: fn(q, k, v, g.double()),
                 lambda: fn(q, k, v, g, beta=beta.double()), lambda: fn(q[0], k[0], v[0], g[0]), lambda: fn(q, k, v, g, initial_states=st[:1]),
                 lambda: fn(q, k, v, g, initial_states=st.bfloat16()), lambda: fn(q.cpu(), k, v, g), lambda: fn(q, k, v, g.cpu()),
                 lambda: fn(q, k, v, g, initial_states=st.cpu()), lambda: fn(q, k, v, g, return_final_states=True, final_states_out=st[:1]),
                 lambda: fn(q, k, v, g, return_final_states=True, final_states_out=wide), lambda: fn(q, k, v, g, cu_seqlens=cu), lambda: fn(q[:1], k[:1], v[:1], g[:1], cu_seqlens=cu.float()),
                 lambda: fn(q[:1], k[:1], v[:1], g[:1], cu_seqlens=cu[:1]), lambda: fn(q[:1], k[:1], v[:1], g[:1], initial_states=st, cu_seqlens=cu),
                 lambda: fn(torch.zeros(1, 5, 1, 257, device=gpu_device), torch.zeros(1, 5, 1, 257, device=gpu_device), torch.zeros(1, 5, 1, 8, device=gpu_device), g[:1, :5, :1]),
                 lambda: fn(q, k, torch.zeros(2, 30, 4, 513, device=gpu_device, dtype=BF16), g),
                 lambda: step(*one, st[:1]), lambda: step(*one, st.half()), lambda: step(*one, wide), lambda: step(*one, st, state_indices=index.long()),
                 lambda: step(*one, st, state_indices=index[:1]), lambda: step(*one, st[:, :3]), lambda: step(*one, st, beta=beta[:, 0, :2]), lambda: step(*one[:3], g, st),
                 lambda: step(*one, st.cpu()), lambda: step(one[0], one[1].float(), *one[2:], st)):
        with pytest.raises((RuntimeError, ValueError, NotImplementedError, TypeError, IndexError)):
            call()
    wide.copy_(st)                                       # (states that are read may lie anyhow)
    assert torch.equal(fn(q, k, v, g, initial_states=wide), fn(q, k, v, g, initial_states=st))
    x, w = torch.zeros(3, 16, device=gpu_device, dtype=BF16), torch.ones(16, device=gpu_device)
    ln = pkg.layer_norm_fn
    for call in (lambda: ln(x, w[:8]), lambda: ln(x, w.half()), lambda: ln(x, w, w[:8]), lambda: ln(x, w, w.bfloat16()), lambda: ln(x, w, residual=x[:2]),
                 lambda: ln(x, w, residual=x.half()), lambda: ln(x.double(), w), lambda: ln(x, w.cpu()), lambda: ln(x, w, w.cpu()), lambda: ln(x, w, residual=x.cpu())):
        with pytest.raises((RuntimeError, ValueError, NotImplementedError)):
            call()
    torch.cuda.synchronize()


CHECKS = ("test_schema", "test_faketensor")


@pytest.mark.parametrize("lengths", [None, [70], [100, 0, 29], [1] * 9, [0, 0]])
@pytest.mark.parametrize("states", [False, True])
@pytest.mark.parametrize("beta", [False, True])
def test_ops_on_fake_tensors(pkg, gpu_device, lengths, states, beta):
    ops = torch.ops.DaoAILab
    total = 70 if lengths is None else sum(lengths)
    s = cases.inputs(gpu_device, 2 if lengths is None else 1, total, 1, 2, 32, 16, BF16, sequences=lengths and len(lengths), states=states, beta=beta)
    cu = None if lengths is None else torch.tensor([0] + lengths).cumsum(0).to(torch.int32).to(gpu_device)
    final = None if s["states"] is None else torch.empty_like(s["states"])
    args = (s["q"], s["k"], s["v"], s["g"], s["beta"], s["states"], cu)
    # (what tokens that are not there left in `saved` is anybody's: its shape is compared, its bytes are not)
    torch.library.opcheck(ops._linear_attention_fwd_save_cpp, args + (final, 0.2), test_utils=CHECKS[1:])
    torch.library.opcheck(ops._linear_attention_fwd_cpp, args + (final, 0.2), test_utils=CHECKS)
    out, saved = ops._linear_attention_fwd_save_cpp(*args, final, 0.2)
    torch.library.opcheck(ops._linear_attention_bwd_cpp, args + (saved, s["dout"], None if final is None else s["dfinal"], 0.2, states), test_utils=CHECKS)


def test_layer_norm_ops_on_fake_tensors(pkg, gpu_device):
    ops = torch.ops.DaoAILab
    x, w, r = torch.randn(5, 70, device=gpu_device).bfloat16(), torch.randn(70, device=gpu_device), torch.randn(5, 70, device=gpu_device)
    for b, res in ((w, r), (None, None), (None, r)):
        torch.library.opcheck(ops._layer_norm_fwd_cpp, (x, w, b, res, 1e-5, True), test_utils=CHECKS)
        y, h, stats = ops._layer_norm_fwd_cpp(x, w, b, res, 1e-5, True)
        torch.library.opcheck(ops._layer_norm_bwd_cpp, (x if res is None else h, stats, w, torch.ones_like(y), None if res is None else r, b is not None), test_utils=CHECKS)


def test_compiled_functions(pkg, gpu_device):
    """Traced whole by torch.compile (aot_eager): the same bits, with gradients and in a decode step."""
    s = cases.inputs(gpu_device, 2, 300, 1, 2, 32, 16, BF16)
    w = torch.randn(32, device=gpu_device)

    def train(q, k, v, g, beta, states, w):
        out, final = pkg.linear_attention_fn(q * 2, k, v, g, beta=beta, initial_states=states, return_final_states=True)
        y, h = pkg.layer_norm_fn(out.flatten(2), w, w, residual=v.flatten(2))
        return y.float().square().sum() + h.float().sum() + final.square().sum()
    results = []
    for f in (train, torch.compile(train, backend="aot_eager", fullgraph=True)):
        leaves = [s[n].detach().clone().requires_grad_() for n in ("q", "k", "v", "g", "beta", "states")] + [w.clone().requires_grad_()]
        loss = f(*leaves)
        results.append([loss, *torch.autograd.grad(loss, leaves)])
    for a, b in zip(*results):
        assert torch.equal(a, b)

    def step(q, k, v, g, state):
        return pkg.linear_attention_update(q * 2, k, v, g, state) + 1
    a, b = s["states"].clone(), s["states"].clone()
    compiled = torch.compile(step, backend="aot_eager", fullgraph=True)
    args = [s[n][:, 0].contiguous() for n in ("q", "k", "v", "g")]
    for _ in range(2):
        assert torch.equal(step(*args, a), compiled(*args, b)) and torch.equal(a, b)


# ---- together ----------------------------------------------------------------------------------

HEADS, DIM_K, DIM_V = 4, 32, 64
WIDTH = HEADS * DIM_V + 2 * DIM_K


def parameters(dev, dim, seed=0):
    r = torch.Generator(device=dev).manual_seed(seed)

    def rand(*shape, by=1.0):
        return torch.randn(*shape, generator=r, device=dev) * by
    return {"norm_w": 1 + rand(dim, by=0.1), "norm_b": rand(dim, by=0.1), "in": rand(WIDTH + 8, dim, by=dim ** -0.5), "conv_w": rand(WIDTH, 4, by=0.5), "conv_b": rand(WIDTH, by=0.1),
            "rate": -torch.rand(HEADS, generator=r, device=dev) - 0.1, "out": rand(dim, HEADS * DIM_V, by=0.05)}


def state_space_block(pkg, p, x, residual, conv_state=None, state=None, plain=False):
    """Norm with the residual, projection, short convolution, linear attention with a decay dt A: a state-space mixer.  One token a sequence where the states are given."""
    from causal_conv1d.layer_norm import layer_norm_ref
    from causal_conv1d.linear_attention import linear_attention_ref
    norm = layer_norm_ref if plain else pkg.layer_norm_fn
    y, h = norm(x, p["norm_w"], p["norm_b"], residual=residual)
    z = y @ p["in"].t()
    dt = torch.nn.functional.softplus(z[..., WIDTH:WIDTH + HEADS])         # (the rows stay a multiple of 8 long, as the convolution wants them)
    g = dt * p["rate"]
    if state is not None:
        z = pkg.causal_conv1d_update(z[..., :WIDTH].contiguous(), conv_state, p["conv_w"], p["conv_b"], "silu")
    else:
        z = z[..., :WIDTH]
        if plain:
            wide = torch.nn.functional.conv1d(z.transpose(1, 2), p["conv_w"][:, None], p["conv_b"], padding=3, groups=WIDTH)[..., :z.shape[1]]
            z = torch.nn.functional.silu(wide).transpose(1, 2)
        else:
            z = pkg.causal_conv1d_fn(z.transpose(1, 2), p["conv_w"], p["conv_b"], activation="silu").transpose(1, 2)
    v = z[..., :HEADS * DIM_V].unflatten(-1, (HEADS, DIM_V))
    k, q = (z[..., HEADS * DIM_V + i * DIM_K:][..., :DIM_K].unflatten(-1, (1, DIM_K)) for i in range(2))
    if state is not None:
        return pkg.linear_attention_update(q, k, v, g, state, beta=dt, scale=1.0).flatten(-2) @ p["out"].t(), h
    if plain:
        out, final = linear_attention_ref(q, k, v, g, dt, scale=1.0, return_final_states=True)
    else:
        out, final = pkg.linear_attention_fn(q, k, v, g, beta=dt, scale=1.0, return_final_states=True)
    return out.flatten(-2) @ p["out"].t(), h, final


def test_together_in_training_and_in_a_decode_loop(pkg, gpu_device):
    """A prompt, then tokens one by one, against the whole sequence at once; and the gradients of all parameters against the plain forms in 64 bits."""
    dim, total, prompt = 96, 290, 270
    p = parameters(gpu_device, dim)
    r = torch.Generator(device=gpu_device).manual_seed(5)
    x, residual = (torch.randn(2, total, dim, generator=r, device=gpu_device) for _ in range(2))
    leaves = {n: t.clone().requires_grad_() for n, t in p.items()}
    weights = torch.randn(2, total, dim, generator=r, device=gpu_device)

    def loss(q, plain, wide):
        out, h, final = state_space_block(pkg, q, wide(x), wide(residual), plain=plain)
        return (out * wide(weights)).sum() + (h * wide(weights)).sum() * 0.1 + final.square().sum() * 0.01, out, final
    value, out, final = loss(leaves, False, lambda t: t)
    grads = torch.autograd.grad(value, list(leaves.values()))
    exact = {n: t.double().requires_grad_() for n, t in p.items()}
    value64, out64, final64 = loss(exact, True, lambda t: t.double())
    grads64 = torch.autograd.grad(value64, list(exact.values()))
    # Chains of sums in fp32, 96, 4, 256 and a few hundred terms long: 1000 2^-24 of a tensor's largest value, and 290 x 2 rows of such errors, which are
    # independent, add up in a parameter's gradient to sqrt(580) of one row's beside a sum that itself grows so.
    for got, want in [(out, out64), (final, final64)] + list(zip(grads, grads64)):
        assert (got.double() - want).abs().max() <= 1000 * 2.0 ** -24 * 4 * want.abs().max()

    with torch.no_grad():
        head, _, state = state_space_block(pkg, p, x[:, :prompt], residual[:, :prompt])
        y, _ = pkg.layer_norm_fn(x[:, :prompt], p["norm_w"], p["norm_b"], residual=residual[:, :prompt])
        conv_state = (y @ p["in"].t())[..., :WIDTH].transpose(1, 2)[..., -4:].contiguous()
        tails = []
        for t in range(prompt, total):
            o, h = state_space_block(pkg, p, x[:, t], residual[:, t], conv_state, state)
            assert torch.equal(h, x[:, t] + residual[:, t])
            tails.append(o)
        both = torch.cat([head, torch.stack(tails, 1)], 1)
    assert (both - out).abs().max() <= 1000 * 2.0 ** -24 * 4 * out.abs().max()
    assert (state - final).abs().max() <= 1000 * 2.0 ** -24 * 4 * final.abs().max()


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("cu", [None, [3, 200, 200, 280, 340]])
def test_rows_that_are_no_whole_vectors(pkg, gpu_device, dtype, cu):
    """Each tensor on its own at an odd address, with an odd stride or with a column more, in both directions: the bits of aligned copies; and what
    surrounds them is left alone."""
    s = cases.inputs(gpu_device, 1 if cu else 2, 340, 1, 2, 32, 64, dtype, sequences=len(cu) - 1 if cu else 0, slices=False)
    want = cases.run(pkg, s, cu)

    def moved(t, how):
        shape = list(t.shape)
        if how == "address":
            room = torch.full((t.numel() + 1,), 7.0, device=gpu_device, dtype=t.dtype)
            view = room[1:].view(shape)
        elif how == "stride":
            room = torch.full((shape[0], shape[1], shape[2] * shape[3] + 3), 7.0, device=gpu_device, dtype=t.dtype)
            view = room[..., :-3].unflatten(-1, shape[2:])
        else:
            room = torch.full(shape[:3] + [shape[3] + 1], 7.0, device=gpu_device, dtype=t.dtype)
            view = room[..., :-1]
        view.copy_(t)
        return room, view
    for how in ("address", "stride", "column"):
        for names in (["q"], ["k"], ["v"], ["dout"], ["q", "k", "v", "dout"]):
            rooms = {n: moved(s[n], how) for n in names}
            before = {n: r[0].clone() for n, r in rooms.items()}
            got = cases.run(pkg, dict(s, **{n: r[1] for n, r in rooms.items()}), cu)
            for n in want:
                assert torch.equal(got[n], want[n]), (how, names, n)
            for n in names:
                assert torch.equal(rooms[n][0], before[n])


@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("dims", [(100, 100), (41, 32), (154, 80), (128, 63), (130, 260), (7, 250)])
def test_odd_sizes_of_many_segments(pkg, gpu_device, dtype, dims):
    """More than one segment, shared key heads, states: each size's rows end inside a vector."""
    s = cases.inputs(gpu_device, 2, 530, 1, 3, *dims, dtype, slices=False)
    cases.check(cases.run(pkg, s), s)


@pytest.mark.parametrize("seed", [1, 2, 3])
def test_gradient_of_a_constant_decay(pkg, gpu_device, seed):
    """Its sum over many tokens, where the error of a segment's S0.dS0 stands in every one of its tokens.  Elements of S0 and dS0 are off by some 2^-23 of
    their size each, independently: S0.dS0 by 2^-23 |S0| |dS0| / sqrt(elements), here four times that, for 256 tokens, and over the segments as they come.
    An offset that all elements share, of 2^-24 as much, would be past it where states have a mean."""
    from causal_conv1d.linear_attention import linear_attention_ref
    b, l, h, d = 2, 1000, 8, 128
    s = cases.inputs(gpu_device, b, l, h, h, d, d, BF16, decay="head", beta=False, seed=seed, slices=False)
    s["g"] = -0.7 * 0.45 ** torch.arange(h, device=gpu_device, dtype=torch.float32)
    got = cases.run(pkg, s)["dg"].double()
    w = {n: s[n].detach().double().requires_grad_() for n in ("q", "k", "v", "g", "states")}
    state, outs, states = w["states"], [], []
    for t in range(0, l, 256):
        state.retain_grad()
        states.append(state)
        e = min(l, t + 256)
        out, state = linear_attention_ref(w["q"][:, t:e], w["k"][:, t:e], w["v"][:, t:e], w["g"].expand(b, e - t, h), initial_states=state, return_final_states=True)
        outs.append(out)
    ((torch.cat(outs, 1) * s["dout"].double()).sum() + (state * s["dfinal"].double()).sum()).backward()
    bound = sum((x.norm(dim=(2, 3)) * x.grad.norm(dim=(2, 3))).sum(0) for x in states) * 256 * 4 * 2.0 ** -23 / d
    off = (got - w["g"].grad).abs()
    # and what the tokens between add: q.dq and k.dk off by 2^-24 |q| |dq| / sqrt(d) each, twice that, added up over up to 256 tokens and summed over these
    between = 4 * 2.0 ** -24 / d ** 0.5 * 256 / 3 ** 0.5 * (w["q"].grad.norm(dim=-1) * w["q"].norm(dim=-1)).square().sum((0, 1)).sqrt()
    assert (off <= bound + between + 2.0 ** -23 * w["g"].grad.abs()).all(), (off / (bound + between)).tolist()
