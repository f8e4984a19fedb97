"""Inputs of linear attention, its results in 64 bits, and how far a kernel may be from them.

A sum of n terms in fp32, in any order, is off by at most n 2^-24 of the sum of the terms' magnitudes, and so is a chain of such sums
with n their lengths together.  The sum of magnitudes is the operator itself on the inputs' magnitudes: every term is then positive, in the
gradients of q, k, v, beta and the states as well.  n: dim_k or dim_v products, 256 tokens of a segment, the segments, and 64 for the
exponentials (2^-22 each), the factors and the products' own 2^-25.  Factors of two bfloat16 terms (the state and the weighted products, where they
make out and dv of 16 bits) are off by 2^-17 each: 2^-16 of the magnitudes.  And each result is rounded once, by eps / 2."""
import torch

from causal_conv1d.linear_attention import linear_attention_ref

NAMES = ("q", "k", "v", "g", "beta", "states")


def inputs(dev, batch, seqlen, heads, v_heads, dim_k, dim_v, dtype=torch.float32, decay="token", beta=True, states=True, sequences=0, seed=0,
           slices=True):
    r = torch.Generator(device=dev).manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, generator=r, device=dev)
    v0, k0 = v_heads * dim_v, v_heads * dim_v + heads * dim_k
    mixed = rand(batch, seqlen, k0 + heads * dim_k).to(dtype)
    s = {"v": mixed[..., :v0].unflatten(-1, (v_heads, dim_v)), "k": mixed[..., v0:k0].unflatten(-1, (heads, dim_k)), "q": mixed[..., k0:].unflatten(-1, (heads, dim_k))}
    if not slices:
        s = {n: t.contiguous() for n, t in s.items()}
    s["g"] = -torch.rand(*((v_heads,) if decay == "head" else (batch, seqlen, v_heads)), generator=r, device=dev) * 0.1
    s["beta"] = torch.rand(batch, seqlen, v_heads, generator=r, device=dev).to(dtype) if beta else None
    s["states"] = rand(sequences or batch, v_heads, dim_k, dim_v) if states else None
    s["dout"], s["dfinal"] = rand(batch, seqlen, v_heads, dim_v).to(dtype), rand(sequences or batch, v_heads, dim_k, dim_v)
    return s


def reference(s, cu=None, scale=None, magnitudes=False, grads=True, dfinal=True):
    """{"out", "final", and the gradients by name} in 64 bits; of the inputs' magnitudes (g as it is) if asked for."""
    def wide(n):
        t = s.get(n)
        if t is None:
            return None
        t = t.detach().double()
        t = t.abs() if magnitudes and n != "g" else t
        return t.requires_grad_() if grads and n in NAMES else t
    w = {n: wide(n) for n in NAMES + ("dout", "dfinal")}
    scale = abs(scale) if magnitudes and scale is not None else scale
    g = w["g"].expand(w["v"].shape[:3])
    if cu is None:
        out, final = linear_attention_ref(w["q"], w["k"], w["v"], g, w["beta"], scale, w["states"], True)
    else:
        outs, finals = [w["v"][:, :cu[0]] * 0], []
        for i, (lo, hi) in enumerate(zip(cu[:-1], cu[1:])):
            part = lambda t: None if t is None else t[:, lo:hi]  # noqa: E731
            o, f = linear_attention_ref(part(w["q"]), part(w["k"]), part(w["v"]), part(g), part(w["beta"]), scale,
                                        None if w["states"] is None else w["states"][i:i + 1], True)
            outs.append(o if hi > lo else w["v"][:, lo:hi])
            finals.append(f)
        out, final = torch.cat(outs + [w["v"][:, cu[-1]:] * 0], 1), torch.cat(finals)
    res = {"out": out.detach(), "final": final.detach()}
    if grads:
        names = [n for n in NAMES if w[n] is not None]
        given = [w["dout"]] + ([w["dfinal"]] if dfinal else [])
        found = torch.autograd.grad([out, final][:len(given)], [w[n] for n in names], given, allow_unused=True)
        res.update({"d" + n: torch.zeros_like(w[n]) if d is None else d for n, d in zip(names, found)})
    return res


def gate_magnitudes(s, most, cu=None):
    """What dg is a difference of: S0.dS0 at a segment's start, and q.dq and k.dk of the tokens in front, each segment for itself."""
    b, l, hv, _ = s["v"].shape
    group = hv // s["q"].shape[2]
    qd, kd = (s[n].double().abs().repeat_interleave(group, 2) for n in ("q", "k"))
    # dq and dk of a shared head are the sums over its value heads: more than each one's own
    each = (qd * most["dq"].repeat_interleave(group, 2)).sum(-1) + (kd * most["dk"].repeat_interleave(group, 2)).sum(-1)
    total = torch.zeros_like(each)
    start = most["dg"] if most["dg"].dim() == 3 else None
    for lo, hi in zip([0] + list(cu), list(cu) + [l]) if cu is not None else [(0, l)]:
        for t in range(lo, hi, 256):
            e = min(hi, t + 256)
            total[:, t:e] = each[:, t:e].cumsum(1) + (each[:, t:t + 1] if start is None else start[:, t:t + 1])
    return total


def check(got, s, cu=None, scale=None, grads=True, dfinal=True):
    """Every tensor of `got` element by element."""
    want, most = (reference(s, cu, scale, m, grads, dfinal) for m in (False, True))
    if grads:
        most["dg"] = gate_magnitudes(s, most, cu)
    l, dk, dv = s["v"].shape[1], s["k"].shape[-1], s["v"].shape[-1]
    group = s["v"].shape[2] // s["q"].shape[2]
    n = max(dk, dv) + 256 + l // 256 + 64 + (group if grads else 0)
    for name, t in got.items():
        w, m = want[name], most[name]
        if name == "dg":
            n_g = n + 256
            if w.dim() == 1:                             # summed over all tokens
                m, n_g = m.sum((0, 1)), n_g + m[..., 0].numel()
            bound = n_g * 2.0 ** -24 * m
        else:
            bound = n * 2.0 ** -24 * m
            if name in ("out", "dv") and t.dtype != torch.float32:
                bound = bound + 2.0 ** -16 * m
        bound = bound + torch.finfo(t.dtype).eps / 2 * w.abs() * 1.01 + torch.finfo(t.dtype).tiny * 2
        assert t.shape == w.shape, name
        assert torch.isfinite(t).all(), name
        off = (t.double() - w).abs()
        assert (off <= bound).all(), (name, (off / bound).max().item(), off.max().item())


def run(pkg, s, cu=None, scale=None, grads=True, dfinal=True, cu_dtype=torch.int32):
    """The public function on these inputs, as `check` takes it."""
    leaves = {n: s[n].detach().requires_grad_(grads) for n in NAMES if s.get(n) is not None}
    at = None if cu is None else torch.tensor(cu, dtype=cu_dtype, device=s["v"].device)
    out, final = pkg.linear_attention_fn(leaves["q"], leaves["k"], leaves["v"], leaves["g"], beta=leaves.get("beta"), scale=scale,
                                         initial_states=leaves.get("states"), return_final_states=True, cu_seqlens=at)
    res = {"out": out.detach(), "final": final.detach()}
    if grads:
        given = [s["dout"]] + ([s["dfinal"]] if dfinal else [])
        found = torch.autograd.grad([out, final][:len(given)], list(leaves.values()), given)
        res.update({"d" + n: d for n, d in zip(leaves, found)})
    return res
