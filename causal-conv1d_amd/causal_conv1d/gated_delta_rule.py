"""The gated delta rule, the recurrence that reads the causal convolution's output in a linear-attention mixer:
`gated_delta_rule_fn` over whole sequences and `gated_delta_rule_update` for the steps of a decode loop.  Per sequence
and value head, with a state S (dim_k, dim_v) in float32:

    D = exp(g[t]) S
    u = beta[t] (v[t] - D^T k[t])
    S = D + k[t] u^T
    out[t] = scale S^T q[t]

q, k (batch, seqlen, heads, dim_k), v (batch, seqlen, v_heads, dim_v), all of one dtype; g (the logarithm of the decay,
-inf forgets everything) and beta (batch, seqlen, v_heads) of any of the three dtypes.  v_heads is a multiple of heads:
value head h reads q and k of head h // (v_heads // heads).  Any strides with the last dimension contiguous are taken as they
are, so q, k and v may be column slices of the channel-last convolution's output:

    x = causal_conv1d_fn(x, weight, bias, activation="silu").transpose(1, 2)        # (batch, seqlen, channels)
    q, k, v = (t.unflatten(-1, (-1, d)) for t, d in zip(x.split(...), (dim_k, dim_k, dim_v)))

Whole sequences are worked through in chunks of 64 tokens: a NaN or an infinity reaches its own head's outputs from the start of its chunk on,
where the recurrence alone would give it to the tokens behind it only.  Other heads, sequences and earlier chunks do not see it.

There is no host path.  `gated_delta_rule_ref` states the operator in plain PyTorch.
"""
import torch
from torch.compiler import is_compiling

import causal_conv1d_cuda as _ext              # loading it registers the ops

_fwd = torch.ops.DaoAILab._gated_delta_rule_fwd_cpp
_fwd_save = torch.ops.DaoAILab._gated_delta_rule_fwd_save_cpp
_bwd = torch.ops.DaoAILab._gated_delta_rule_bwd_cpp
_update = torch.ops.DaoAILab._gated_delta_rule_update_cpp


def _new_states(q, v, cu_seqlens):
    n = q.shape[0] if cu_seqlens is None else cu_seqlens.shape[0] - 1
    return torch.empty(n, v.shape[2], q.shape[-1], v.shape[-1], dtype=torch.float32, device=v.device)


class GatedDeltaRuleFn(torch.autograd.Function):
    """Saves the inputs and, in float32, the state in front of every 64 tokens and what they added to it: for 128 x 128 heads 1.5 KB
    a token and value head, beside the 1 KB of its q, k, v and out in 16 bits.  Computing them again took a third of the backward's time."""

    @staticmethod
    def forward(ctx, q, k, v, g, beta, scale, initial_states, return_final_states, cu_seqlens, qk_l2norm):
        final = _new_states(q, v, cu_seqlens) if return_final_states else None
        out, saved = _fwd_save(q, k, v, g, beta, initial_states, cu_seqlens, final, scale, qk_l2norm)
        ctx.save_for_backward(q, k, v, g, beta, initial_states, cu_seqlens, saved)
        ctx.scale, ctx.qk_l2norm = scale, qk_l2norm
        ctx.set_materialize_grads(False)
        return (out, final) if return_final_states else out

    @staticmethod
    def backward(ctx, dout, dfinal=None):
        q, k, v, g, beta, initial_states, cu_seqlens, saved = ctx.saved_tensors
        if dout is None and dfinal is None:
            return (None,) * 10
        if dout is None:                                 # only the states were used
            dout = torch.zeros_like(v)
        wants_states = initial_states is not None and ctx.needs_input_grad[6]
        dq, dk, dv, dg, dbeta, dinitial = _bwd(q, k, v, g, beta, initial_states, cu_seqlens, saved, dout, dfinal, ctx.scale,
                                               ctx.qk_l2norm, wants_states)
        return dq, dk, dv, dg, dbeta, None, dinitial if wants_states else None, None, None, None


def gated_delta_rule_fn(q, k, v, g, beta, scale=None, initial_states=None, return_final_states=False,
                        final_states_out=None, cu_seqlens=None, qk_l2norm=False):
    """out (batch, seqlen, v_heads, dim_v) of v's dtype, or (out, final_states).

    scale: 1 / sqrt(dim_k) if None.  qk_l2norm: q and k are divided by their length, sqrt(sum of squares + 1e-6).
    initial_states (sequences, v_heads, dim_k, dim_v) float32, zeros if None; final_states like it, written to
    final_states_out if given (which may be initial_states itself; without gradients only, and with return_final_states only).
    cu_seqlens (sequences + 1,) int32 or int64, ascending from 0 to seqlen, with a batch of 1: sequence n is tokens
    cu_seqlens[n] .. cu_seqlens[n+1]-1; a sequence may be empty."""
    if not is_compiling():
        res = _ext._gated_delta_rule_call(q, k, v, g, beta, scale, initial_states, return_final_states, final_states_out,
                                          cu_seqlens, qk_l2norm)
        if res is not NotImplemented:
            return res
    if scale is None:
        scale = q.shape[-1] ** -0.5
    if cu_seqlens is not None:
        cu_seqlens = cu_seqlens.contiguous()
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, g, beta, initial_states)):
        if return_final_states and final_states_out is not None:
            raise RuntimeError("final_states_out cannot be given where gradients are recorded")
        return GatedDeltaRuleFn.apply(q, k, v, g, beta, float(scale), initial_states, return_final_states, cu_seqlens, qk_l2norm)
    if not return_final_states:
        final_states_out = None
    elif final_states_out is None:
        final_states_out = _new_states(q, v, cu_seqlens)
    out = _fwd(q, k, v, g, beta, initial_states, cu_seqlens, final_states_out, float(scale), qk_l2norm)
    return (out, final_states_out) if return_final_states else out


def gated_delta_rule_update(q, k, v, g, beta, state, scale=None, state_indices=None, qk_l2norm=False):
    """The step of a decode loop: out like v, and the states advanced in place.  No backward: out
    belongs to no graph, and a state that requires a gradient is refused where gradients are recorded.

    q, k (batch, heads, dim_k), v (batch, v_heads, dim_v), g, beta (batch, v_heads); or all of them with a seqlen axis
    behind the batch, for a few tokens at once.  state (slots, v_heads, dim_k, dim_v) float32.
    state_indices (batch,) int32: entry b uses state[state_indices[b]]; a negative index gives zeros and leaves
    every state alone.  No slot may be named twice."""
    if not is_compiling():
        res = _ext._gated_delta_rule_update_call(q, k, v, g, beta, state, state_indices, scale, qk_l2norm)
        if res is not NotImplemented:
            return res
    if scale is None:
        scale = q.shape[-1] ** -0.5
    return _update(q, k, v, g, beta, state, state_indices, float(scale), qk_l2norm)


def gated_delta_rule_ref(q, k, v, g, beta, scale=None, initial_states=None, return_final_states=False, qk_l2norm=False):
    """The recurrence in plain PyTorch on any device, token by token, in float32 (float64 for float64 tensors);
    differentiable.  Sequences of one length; no cu_seqlens."""
    wide = torch.float64 if q.dtype == torch.float64 else torch.float32
    group = v.shape[2] // q.shape[2]
    q, k, vw, g, beta = (t.to(wide) for t in (q, k, v, g, beta))
    if qk_l2norm:
        q, k = (t * torch.rsqrt(t.square().sum(-1, keepdim=True) + 1e-6) for t in (q, k))
    q, k = (t.repeat_interleave(group, dim=2) for t in (q, k))
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    s = q.new_zeros(v.shape[0], v.shape[2], q.shape[-1], v.shape[-1]) if initial_states is None else initial_states.to(wide)
    outs = []
    for t in range(v.shape[1]):
        s = s * g[:, t].exp()[..., None, None]
        u = beta[:, t, :, None] * (vw[:, t] - (s * k[:, t, :, :, None]).sum(-2))
        s = s + k[:, t, :, :, None] * u[:, :, None, :]
        outs.append(scale * (s * q[:, t, :, :, None]).sum(-2))
    out = (torch.stack(outs, 1) if outs else vw).to(v.dtype)
    return (out, s) if return_final_states else out
