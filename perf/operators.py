"""The operators of the blocks around the convolution, as their speed and results are measured: the gated delta rule
(a forward without gradients, a training step, a decode step) and the root-mean-square norm with the residual's addition
(a training step, and the inference form with an output in 8 bits).

A case is a dict of plain values.  Its "op" is one of
  prefill  the gated delta rule over whole prompts, without gradients: `gated_delta_rule_fn`;
  train    its forward and backward through autograd;
  decode   one token (or a few) of every running sequence, states updated in place: `gated_delta_rule_update`;
  norm     `rms_norm_fn` with its backward through autograd;
  norm8    `rms_norm_quant_fn`, and its rows read back by `dequantize_rows`.
q, k and v are column slices of one buffer (batch, seqlen, channels), as a channel-last convolution leaves them.
With `own` false everything is computed in elementary torch operations in 32 bits.
"""
import math
import os
import sys

import torch

own = False

_TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_CHUNK = 64
_EPS = 1e-6
_F8_MAX = 448.0


def _package():
    at = os.path.join(os.getcwd(), "causal-conv1d_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import causal_conv1d
    return causal_conv1d


def _delta(name, op, **values):
    base = {"name": name, "op": op, "batch": 1, "seqlen": 1, "heads": 16, "v_heads": 32, "dim_k": 128, "dim_v": 128,
            "dtype": "bf16", "l2norm": True}
    return dict(base, **values)


def _norm(name, op, **values):
    return dict({"name": name, "op": op, "dtype": "bf16", "res_dtype": "bf16", "w_dtype": "bf16"}, **values)


def listed():
    return [
        # One chunk of a chunked prefill of a single request: states in, states out, two value heads to a key head.
        _delta("prefill_chunk", "prefill", seqlen=512, sequences=0, states=True),
        # Prompts of twelve requests packed into one row, ragged, and the states their decode starts from.
        _delta("prefill_packed", "prefill", seqlen=4096, sequences=12, states=False),
        # One long document through a layer with few heads: the sequence is long, the heads do not fill the card.
        _delta("prefill_long", "prefill", seqlen=16384, sequences=0, heads=16, v_heads=16, states=False, dtype="fp16"),
        # A training step of one layer at full batch.
        _delta("train_layer", "train", batch=4, seqlen=2048, heads=16, v_heads=16, states=False),
        # A training step with shared key heads, truncated backpropagation (states in, their gradient out), a length that
        # is no whole number of chunks.
        _delta("train_shared_heads", "train", batch=2, seqlen=1000, heads=4, v_heads=8, states=True),
        # A small model at full precision, head sizes that are no powers of two.
        _delta("train_small_fp32", "train", batch=2, seqlen=197, heads=3, v_heads=3, dim_k=48, dim_v=80, states=True,
               dtype="fp32", l2norm=False),
        # One request generating text: latency.
        _delta("decode_one_request", "decode", batch=1, slots=0),
        # A server with continuous batching: states in slots, a quarter of the batch is padding.
        _delta("decode_slots", "decode", batch=128, slots=256),
        # The norm in front of a mixer in training: residual stream in 32 bits.
        _norm("norm_train", "norm", rows=16384, dim=2560, res_dtype="fp32", w_dtype="fp32"),
        # A small model's rows, neither a power of two nor whole vectors.
        _norm("norm_train_odd", "norm", rows=777, dim=1001, dtype="fp32", res_dtype="fp32", w_dtype="fp32"),
        # The norm in front of an 8-bit projection in a decode step.
        _norm("norm8_decode", "norm8", rows=64, dim=5120),
        # The same in a prefill.
        _norm("norm8_prefill", "norm8", rows=8192, dim=5120),
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _head_size(rng):
    n = _spread(rng, 16, 256)
    return n if rng.random() < 0.2 else max(16, n // 16 * 16)


def draw(rng):
    limit = {}
    for c in listed():
        w = work(c)
        limit[c["op"]] = max(limit.get(c["op"], 0.0), w["bytes"] / 5e12 + w["flops"] / 1e14)
    while True:
        op = rng.choice(["prefill", "prefill", "train", "train", "decode", "decode", "norm", "norm8"])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        if op in ("norm", "norm8"):
            c = {"op": op, "rows": _spread(rng, 1, 16384), "dim": _spread(rng, 64, 8192), "dtype": dtype,
                 "res_dtype": rng.choice([dtype, "fp32"]), "w_dtype": rng.choice([dtype, "fp32"])}
            if rng.random() < 0.6:
                c["dim"] = max(64, c["dim"] // 64 * 64)
        else:
            heads = _spread(rng, 1, 32)
            c = {"op": op, "heads": heads, "v_heads": heads * rng.choice([1, 1, 2, 3]), "dim_k": _head_size(rng),
                 "dim_v": _head_size(rng), "dtype": dtype, "l2norm": rng.random() < 0.5}
            if op == "decode":
                c.update(batch=_spread(rng, 1, 256), seqlen=rng.choice([1, 1, 1, 2, 4]))
                c["slots"] = rng.choice([0, c["batch"] + rng.randint(1, 64)])
            else:
                c.update(batch=_spread(rng, 1, 16), seqlen=_spread(rng, 1, 16384), states=rng.random() < 0.5)
            if op == "prefill":
                c["sequences"] = rng.choice([0, _spread(rng, 1, 32)])
                if c["sequences"]:
                    c["batch"] = 1
        w = work(c)
        sizes = [v for v in c.values() if isinstance(v, int)] + [c.get("heads", 0) * c.get("dim_k", 0), c.get("v_heads", 0) * c.get("dim_v", 0)]
        if w["bytes"] / 5e12 + w["flops"] / 1e14 <= limit[op] and 3072 not in sizes:
            return c


def work(case):
    """What a pass cannot do without: inputs read once, outputs written once, the recurrence's own operations."""
    eb = {"fp32": 4, "fp16": 2, "bf16": 2}
    e = eb[case["dtype"]]
    if case["op"] in ("norm", "norm8"):
        n, r = case["rows"] * case["dim"], eb[case["res_dtype"]]
        if case["op"] == "norm":       # x, residual -> h, y; dy, dh, h -> dx, dresidual
            return {"bytes": float(n * (e + r + r + e) + n * (e + r + r + e + r)), "flops": float(n * 16)}
        # x, residual -> h, y8, scales; y8, scales -> y
        return {"bytes": float(n * (e + r + r + 1) + n * (1 + e)), "flops": float(n * 8)}
    tokens, h, hv, dk, dv = case["batch"] * case["seqlen"], case["heads"], case["v_heads"], case["dim_k"], case["dim_v"]
    qkv = tokens * (2 * h * dk + hv * dv) * e
    o, gates = tokens * hv * dv * e, tokens * hv * (4 + e)
    flops = tokens * hv * dk * dv * 7.0
    if case["op"] == "decode":
        # three quarters of a batch with slots are live
        live = max(1, case["batch"] - case["batch"] // 4 if case["slots"] else case["batch"])
        return {"bytes": float(qkv + o + gates + 8 * live * hv * dk * dv), "flops": flops * live / case["batch"]}
    state = max(case["batch"], case.get("sequences", 0)) * hv * dk * dv * 4
    if case["op"] == "prefill":
        return {"bytes": float(qkv + o + gates + state * (2 if case["states"] else 1)), "flops": flops}
    return {"bytes": float(3 * qkv + 2 * o + 3 * gates + state * (5 if case["states"] else 2)), "flops": 3 * flops}


def _lengths(case, gen):
    """Ragged lengths that add up to the case's tokens; a sequence may be empty or a single token."""
    n, total = case["sequences"], case["seqlen"]
    share = torch.rand(n, generator=gen).add_(0.02).square_()
    cuts = (share.cumsum(0) / share.sum() * total).round().to(torch.int64)
    cuts[-1] = total
    return torch.diff(cuts, prepend=torch.zeros(1, dtype=torch.int64)).tolist()


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    host = torch.Generator().manual_seed(int(seed))
    t = _TYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device=dev)

    if case["op"] in ("norm", "norm8"):
        rows, dim = case["rows"], case["dim"]
        r = _TYPES[case["res_dtype"]]
        s = {"case": case, "x": randn(rows, dim).to(t), "residual": randn(rows, dim).mul_(2).to(r),
             "weight": rand(dim).mul_(0.5).add_(0.75).to(_TYPES[case["w_dtype"]])}
        if case["op"] == "norm":
            for name in ("x", "residual", "weight"):
                s[name].requires_grad_()
            s["dy"], s["dh"] = randn(rows, dim).to(t), randn(rows, dim).to(r)
        return s

    b, l, h, hv, dk, dv = (case[n] for n in ("batch", "seqlen", "heads", "v_heads", "dim_k", "dim_v"))
    mixed = torch.nn.functional.silu(randn(b, l, 2 * h * dk + hv * dv))      # what the convolution's activation leaves
    if not case["l2norm"]:                                                   # keys and queries of unit length
        qk = mixed[..., :2 * h * dk].unflatten(-1, (2 * h, dk))
        qk /= qk.norm(dim=-1, keepdim=True) + 1e-3
    mixed = mixed.to(t)
    s = {"case": case,
         "q": mixed[..., :h * dk].unflatten(-1, (h, dk)),
         "k": mixed[..., h * dk:2 * h * dk].unflatten(-1, (h, dk)),
         "v": mixed[..., 2 * h * dk:].unflatten(-1, (hv, dv)),
         # decay rates 1 .. 16 a head, time steps of about 0.001 .. 0.1 that the token shifts
         "g": -(1 + 15 * rand(hv)) * torch.nn.functional.softplus(randn(b, l, hv) + torch.log(torch.expm1(0.001 * 100 ** rand(hv)))),
         "beta": torch.sigmoid(randn(b, l, hv)).to(t)}
    if case["op"] == "decode":
        slots = case["slots"]
        s["state"] = randn(slots or b, hv, dk, dv).mul_(0.3)
        s["indices"] = s["live"] = None
        if slots:
            at = torch.randperm(slots, generator=host)[:b].to(torch.int32)
            idle = torch.randperm(b, generator=host)[:b // 4]
            at[idle] = -1
            s["indices"] = at.to(dev)
            s["live"] = torch.nonzero(at >= 0).flatten().to(dev)             # a scheduler knows which entries are padding
        return s
    n = case.get("sequences", 0) or b
    s["states"] = randn(n, hv, dk, dv).mul_(0.3) if case["states"] else None
    s["cu_seqlens"] = s["place"] = None
    if case.get("sequences", 0):
        lengths = _lengths(case, host)
        s["cu_seqlens"] = torch.tensor([0] + lengths, dtype=torch.int32).cumsum(0).to(torch.int32).to(dev)
        # The plan of the plain form: the rows of a padded batch that the packed tokens take.
        longest = max(lengths)
        s["longest"] = longest
        s["place"] = torch.cat([torch.arange(m) + i * longest for i, m in enumerate(lengths)]).to(dev)
    if case["op"] == "train":
        for name in ("q", "k", "v", "g", "beta"):
            s[name] = s[name].detach().requires_grad_()
        if s["states"] is not None:
            s["states"].requires_grad_()
        s["dout"] = randn(b, l, hv, dv).to(t)
        s["dfinal"] = randn(n, hv, dk, dv) if case["states"] else None
    return s


# ---- plain forms -----------------------------------------------------------------------------------------------------

def _unit(t, wanted):
    t = t.float()
    return t * torch.rsqrt(t.square().sum(-1, keepdim=True) + _EPS) if wanted else t


def _unit_lower_inverse(a):
    """(I + a)^-1 of strictly lower triangular a (..., c, c), c a power of two: from blocks of one entry, whose inverse is 1,
    to twice the size each time, [[X, 0], [B, Y]]^-1 = [[X^-1, 0], [-Y^-1 B X^-1, Y^-1]]."""
    c = a.shape[-1]
    inv, size = a.new_ones(*a.shape[:-2], c, 1, 1), 1
    while size < c:
        n = c // (2 * size)
        below = a.unflatten(-2, (n, 2, size)).unflatten(-1, (n, 2, size))[..., 1, :, :, 0, :].diagonal(0, -4, -2).movedim(-1, -3)
        x, y = inv.unflatten(-3, (n, 2)).unbind(-3)
        low = -torch.matmul(torch.matmul(y, below), x)
        inv = torch.cat([torch.cat([x, torch.zeros_like(x)], -1), torch.cat([low, y], -1)], -2)
        size *= 2
    return inv[..., 0, :, :]


def _plain_chunks(q, k, v, g, beta, state, l2norm):
    """(batch, seqlen, ...) -> out (batch, seqlen, v_heads, dim_v) and the last state, both in 32 bits.  Chunks of 64 tokens
    as matrix products; what one chunk hands to the next is the only loop, since it is a recurrence."""
    b, l, hv, dv = v.shape
    dk, group = q.shape[-1], hv // q.shape[2]
    scale = dk ** -0.5
    c = min(_CHUNK, 1 << (l - 1).bit_length())
    n = -(-l // c)
    pad = n * c - l

    def cut(t):          # (batch, seqlen, heads, ...) -> (batch, heads, chunks, c, ...)
        t = torch.nn.functional.pad(t.float(), (0, 0) * (t.dim() - 2) + (0, pad)) if pad else t.float()
        return t.unflatten(1, (n, c)).movedim(3, 1)

    q, k = (cut(_unit(t, l2norm).repeat_interleave(group, 2)) for t in (q, k))
    v, g, beta = cut(v), cut(g), cut(beta)
    total = g.cumsum(-1)
    lower = torch.ones(c, c, dtype=torch.bool, device=v.device).tril()
    decay = torch.exp((total[..., :, None] - total[..., None, :]).masked_fill(~lower, -math.inf))
    keys = k.transpose(-1, -2)
    mix = (torch.matmul(k, keys) * decay * beta[..., None]).tril(-1)
    solved = torch.matmul(_unit_lower_inverse(mix), torch.cat([v * beta[..., None], k * (beta * total.exp())[..., None]], -1))
    fresh, seen = solved[..., :dv], solved[..., dv:]
    reads = torch.matmul(q, keys) * decay
    q = q * total.exp()[..., None]
    carry = (k * (total[..., -1:] - total).exp()[..., None]).transpose(-1, -2)
    last = total[..., -1].exp()[..., None, None]
    if state is None:
        state = v.new_zeros(b, hv, dk, dv)
    outs = []
    for i in range(n):
        u = fresh[:, :, i] - torch.matmul(seen[:, :, i], state)
        outs.append(torch.matmul(q[:, :, i], state) + torch.matmul(reads[:, :, i], u))
        state = state * last[:, :, i] + torch.matmul(carry[:, :, i], u)
    out = torch.stack(outs, 2).movedim(1, 3).flatten(1, 2)[:, :l]
    return out * scale, state


def _plain_delta(s):
    case = s["case"]
    q, k, v, g, beta = (s[n] for n in ("q", "k", "v", "g", "beta"))
    if s["place"] is None:
        out, state = _plain_chunks(q, k, v, g, beta, s["states"], case["l2norm"])
    else:
        n, longest = case["sequences"], s["longest"]

        def padded(t):   # tokens that are not there: no gate, no key, nothing learned
            full = t.new_zeros(n * longest, *t.shape[2:])
            full[s["place"]] = t[0]
            return full.unflatten(0, (n, longest))

        out, state = _plain_chunks(*(padded(t) for t in (q, k, v, g, beta)), s["states"], case["l2norm"])
        out = out.flatten(0, 1)[s["place"]].unsqueeze(0)
    return out.to(v.dtype), state


def _plain_decode(s):
    case, state, live = s["case"], s["state"], s["live"]
    group = case["v_heads"] // case["heads"]
    rows = [s[n] if live is None else s[n][live] for n in ("q", "k", "v", "g", "beta")]
    at = None if live is None else s["indices"][live].long()
    now = state if at is None else state[at]
    q, k = (_unit(t, case["l2norm"]).repeat_interleave(group, 2) for t in rows[:2])
    v, g, beta = (t.float() for t in rows[2:])
    outs = []
    for i in range(case["seqlen"]):
        now = now * g[:, i].exp()[..., None, None]
        u = (v[:, i] - torch.matmul(k[:, i, :, None], now).squeeze(2)) * beta[:, i, :, None]
        now = now + k[:, i, :, :, None] * u[:, :, None]
        outs.append(torch.matmul(q[:, i, :, None], now).squeeze(2))
    out = (torch.stack(outs, 1) * case["dim_k"] ** -0.5).to(s["v"].dtype)
    if at is None:
        state.copy_(now)
        return out
    state[at] = now
    return out.new_zeros(case["batch"], *out.shape[1:]).index_copy_(0, live, out)


def _plain_norm(x, residual, weight):
    h = (x.float() + residual.float()).to(residual.dtype)
    wide = h.float()
    return h, wide * torch.rsqrt(wide.square().mean(-1, keepdim=True) + _EPS) * weight.float()


def _grads(outs, wanted, given):
    return list(torch.autograd.grad(outs, wanted, given))


def run(s):
    case = s["case"]
    op = case["op"]
    if op == "norm":
        if own:
            y, h = _package().rms_norm_fn(s["x"], s["weight"], residual=s["residual"], eps=_EPS)
        else:
            h, y = _plain_norm(s["x"], s["residual"], s["weight"])
            y = y.to(s["x"].dtype)
        return {"y": y, "h": h, "grads": _grads([y, h], [s["x"], s["residual"], s["weight"]], [s["dy"], s["dh"]])}
    if op == "norm8":
        if own:
            pkg = _package()
            y8, scales, h = pkg.rms_norm_quant_fn(s["x"], s["weight"], residual=s["residual"], eps=_EPS)
            return {"y": pkg.dequantize_rows(y8, scales, s["x"].dtype), "scales": scales, "h": h}
        h, y = _plain_norm(s["x"], s["residual"], s["weight"])
        scales = y.abs().amax(-1) / _F8_MAX
        y8 = (y / scales[:, None]).clamp(-_F8_MAX, _F8_MAX).to(torch.float8_e4m3fn)
        return {"y": (y8.float() * scales[:, None]).to(s["x"].dtype), "scales": scales, "h": h}
    if op == "decode":
        if own:
            out = _package().gated_delta_rule_update(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"],
                                                     state_indices=s["indices"], qk_l2norm=case["l2norm"])
        else:
            out = _plain_decode(s)
        return {"out": out, "state": s["state"]}
    if own:
        out, final = _package().gated_delta_rule_fn(s["q"], s["k"], s["v"], s["g"], s["beta"], initial_states=s["states"],
                                                    return_final_states=True, cu_seqlens=s["cu_seqlens"],
                                                    qk_l2norm=case["l2norm"])
    else:
        out, final = _plain_delta(s)
    if op == "prefill":
        return {"out": out, "final": final}
    wanted = [s[n] for n in ("q", "k", "v", "g", "beta")]
    if s["states"] is None:
        return {"out": out, "final": final.detach(), "grads": _grads([out], wanted, [s["dout"]])}
    return {"out": out, "final": final.detach(), "grads": _grads([out, final], wanted + [s["states"]], [s["dout"], s["dfinal"]])}


# ---- 64 bits, token by token -----------------------------------------------------------------------------------------

def _exact_norm(case, s):
    h = (s["x"].detach().float() + s["residual"].detach().float()).to(s["residual"].dtype).double()
    w = s["weight"].detach().double()
    r = (h.pow(2).sum(-1, keepdim=True) / case["dim"] + _EPS).pow(-0.5)
    y = h * r * w
    if case["op"] == "norm8":
        # The rows read back carry the rounding to 8 bits; the scales and the sum have values in 64 bits.
        return {"y": None, "scales": y.abs().amax(-1) / _F8_MAX, "h": h}
    dy = s["dy"].double()
    wdy = w * dy
    dh = r * wdy - h * r.pow(3) * ((h * wdy).sum(-1, keepdim=True) / case["dim"]) + s["dh"].double()
    return {"y": y, "h": h, "grads": [dh, dh, (dy * h * r).sum(0)]}


def _tokens64(q, k, v, g, beta, state, scale, dout=None, dstate=None):
    """The recurrence over (batch, seqlen, v_heads, ...) in 64 bits, one token after the other, and with dout its adjoint."""
    outs, states, fresh, missed = [], [], [], []
    keep = dout is not None
    for t in range(q.shape[1]):
        if keep:
            states.append(state)
        state = state * torch.exp(g[:, t])[..., None, None]
        miss = v[:, t] - (state * k[:, t, :, :, None]).sum(2)
        u = beta[:, t, :, None] * miss
        state = state + k[:, t, :, :, None] * u[:, :, None, :]
        outs.append(scale * (state * q[:, t, :, :, None]).sum(2))
        if keep:
            fresh.append(u)
            missed.append(miss)
    if not keep:
        return torch.stack(outs, 1), state
    dq, dk, dv, dg, db = (torch.empty_like(x) for x in (q, k, v, g, beta))
    d = torch.zeros_like(state) if dstate is None else dstate
    for t in range(q.shape[1] - 1, -1, -1):
        a = torch.exp(g[:, t])[..., None, None]
        before = states[t] * a
        do = scale * dout[:, t]
        after = before + k[:, t, :, :, None] * fresh[t][:, :, None, :]
        dq[:, t] = (after * do[:, :, None, :]).sum(-1)
        d = d + q[:, t, :, :, None] * do[:, :, None, :]
        du = (d * k[:, t, :, :, None]).sum(2)
        db[:, t] = (du * missed[t]).sum(-1)
        dv[:, t] = beta[:, t, :, None] * du
        dk[:, t] = (d * fresh[t][:, :, None, :]).sum(-1) - (before * dv[:, t, :, None, :]).sum(-1)
        d = d - k[:, t, :, :, None] * dv[:, t, :, None, :]
        dg[:, t] = (d * before).sum((-1, -2))
        d = d * a
    return torch.stack(outs, 1), state, dq, dk, dv, dg, db, d


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("norm", "norm8"):
        return _exact_norm(case, s)
    heads, group = case["heads"], case["v_heads"] // case["heads"]
    # One launch or so an operation and token: above this it takes longer than it is worth.
    if case["seqlen"] > 20000 or (case["op"] == "train" and case["batch"] * case["seqlen"] * case["v_heads"] * case["dim_k"] * case["dim_v"] > 4e9):
        return None
    scale = 1 / math.sqrt(case["dim_k"])
    raw = [s[n].detach().double() for n in ("q", "k")]
    inv = [(x.pow(2).sum(-1, keepdim=True) + _EPS).pow(-0.5) if case["l2norm"] else torch.ones_like(x[..., :1]) for x in raw]
    q, k = ((x * r).repeat_interleave(group, dim=2) for x, r in zip(raw, inv))
    v, g, beta = (s[n].detach().double() for n in ("v", "g", "beta"))
    if case["op"] == "decode":
        state = s["state"].double()
        out = torch.zeros_like(v)
        at = torch.arange(case["batch"], device=v.device) if s["indices"] is None else s["indices"].long()
        live = torch.nonzero(at >= 0).flatten()
        out[live], state[at[live]] = _tokens64(*(x[live] for x in (q, k, v, g, beta)), state[at[live]], scale)
        return {"out": out, "state": state}
    n = case.get("sequences", 0) or case["batch"]
    first = torch.zeros(n, case["v_heads"], case["dim_k"], case["dim_v"], dtype=torch.float64, device=v.device) if s["states"] is None else s["states"].detach().double()
    if s["cu_seqlens"] is not None:
        out, final = torch.empty_like(v), first.clone()
        cu = s["cu_seqlens"].tolist()
        for i, (lo, hi) in enumerate(zip(cu[:-1], cu[1:])):
            if hi > lo:
                out[:, lo:hi], final[i:i + 1] = _tokens64(*(x[:, lo:hi] for x in (q, k, v, g, beta)), first[i:i + 1], scale)
        return {"out": out, "final": final}
    if case["op"] == "prefill":
        out, final = _tokens64(q, k, v, g, beta, first, scale)
        return {"out": out, "final": final}
    dfinal = None if s["dfinal"] is None else s["dfinal"].double()
    out, final, dq, dk, dv, dg, db, dfirst = _tokens64(q, k, v, g, beta, first, scale, s["dout"].double(), dfinal)
    grads = []
    for d, x, r in zip((dq, dk), raw, inv):
        d = d.unflatten(2, (heads, group)).sum(3)
        grads.append(r * d - x * r.pow(3) * (x * d).sum(-1, keepdim=True) if case["l2norm"] else d)
    grads += [dv, dg, db] + ([dfirst] if s["states"] is not None else [])
    return {"out": out, "final": final, "grads": grads}
