"""Linear attention with a decay for each head: `linear_attention_fn` over whole sequences and `linear_attention_update` for the
steps of a decode loop.  Per sequence and value head, with a state S (dim_k, dim_v) in float32:

    S = exp(g[t]) S + beta[t] k[t] v[t]^T
    out[t] = scale S^T q[t]

q, k (batch, seqlen, heads, dim_k), v (batch, seqlen, v_heads, dim_v), all of one dtype; g, the logarithm of the decay (-inf forgets
everything), (batch, seqlen, v_heads), or (v_heads,) for one that is the same at every token; beta (batch, seqlen, v_heads), a token's
weight, or None for 1.  g and beta are of any of the three dtypes.  v_heads is a multiple of heads: value head h reads q and k of head
h // (v_heads // heads).  Any strides with the last dimension contiguous are taken as they are, so q, k and v may be column slices
of the channel-last convolution's output.  A state-space block with a step size dt and rates A is v = x, k = B, q = C, g = dt A, beta = dt, scale = 1.

Gates below -200 count as -200, which leaves nothing of a float32 state.  They may be positive, as long as they add up to less than 32 (a state grows by
less than 2^46) over any run of at most 256 tokens: beyond that, what falls far and is brought back may be lost.  Whole sequences are worked through in blocks of 64 tokens: a NaN or an infinity reaches its own head's outputs from the start of
its block on.  Other heads, sequences and earlier blocks do not see it.

There is no host path.  `linear_attention_ref` states the operator in plain PyTorch.
"""
import torch
from torch.compiler import is_compiling

import causal_conv1d_cuda as _ext              # loading it registers the ops

_fwd = torch.ops.DaoAILab._linear_attention_fwd_cpp
_fwd_save = torch.ops.DaoAILab._linear_attention_fwd_save_cpp
_bwd = torch.ops.DaoAILab._linear_attention_bwd_cpp
_update = torch.ops.DaoAILab._linear_attention_update_cpp


def _new_states(q, v, cu_seqlens):
    n = q.shape[0] if cu_seqlens is None else cu_seqlens.shape[0] - 1
    return torch.empty(n, v.shape[2], q.shape[-1], v.shape[-1], dtype=torch.float32, device=v.device)


class LinearAttentionFn(torch.autograd.Function):
    """Saves the inputs and the states between segments of 256 tokens (with initial states that in front of the first too), 6 bytes an element."""

    @staticmethod
    def forward(ctx, q, k, v, g, beta, scale, initial_states, return_final_states, cu_seqlens):
        final = _new_states(q, v, cu_seqlens) if return_final_states else None
        out, saved = _fwd_save(q, k, v, g, beta, initial_states, cu_seqlens, final, scale)
        ctx.save_for_backward(q, k, v, g, beta, initial_states, cu_seqlens, saved)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return (out, final) if return_final_states else out

    @staticmethod
    def backward(ctx, dout, dfinal=None):
        q, k, v, g, beta, initial_states, cu_seqlens, saved = ctx.saved_tensors
        if dout is None and dfinal is None:
            return (None,) * 9
        if dout is None:                                 # only the states were used
            dout = torch.zeros_like(v)
        wants_states = initial_states is not None and ctx.needs_input_grad[6]
        dq, dk, dv, dg, dbeta, dinitial = _bwd(q, k, v, g, beta, initial_states, cu_seqlens, saved, dout, dfinal, ctx.scale, wants_states)
        return dq, dk, dv, dg, None if beta is None else dbeta, None, dinitial if wants_states else None, None, None


def linear_attention_fn(q, k, v, g, beta=None, scale=None, initial_states=None, return_final_states=False,
                        final_states_out=None, cu_seqlens=None):
    """out (batch, seqlen, v_heads, dim_v) of v's dtype, or (out, final_states).

    scale: 1 / sqrt(dim_k) if None.  initial_states (sequences, v_heads, dim_k, dim_v) float32, zeros if None; final_states like it,
    written to final_states_out if given (which may be initial_states itself; without gradients only, and with return_final_states only).
    cu_seqlens (sequences + 1,) int32 or int64, ascending from 0 to seqlen, with a batch of 1: sequence n is tokens
    cu_seqlens[n] .. cu_seqlens[n+1]-1; a sequence may be empty."""
    if not is_compiling():
        res = _ext._linear_attention_call(q, k, v, g, beta, scale, initial_states, return_final_states, final_states_out, cu_seqlens)
        if res is not NotImplemented:
            return res
    if scale is None:
        scale = q.shape[-1] ** -0.5
    if g.dim() == 1:
        g = g.expand(v.shape[:3])
    if cu_seqlens is not None:
        cu_seqlens = cu_seqlens.contiguous()
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, g, beta, initial_states)):
        if return_final_states and final_states_out is not None:
            raise RuntimeError("final_states_out cannot be given where gradients are recorded")
        return LinearAttentionFn.apply(q, k, v, g, beta, float(scale), initial_states, return_final_states, cu_seqlens)
    if not return_final_states:
        final_states_out = None
    elif final_states_out is None:
        final_states_out = _new_states(q, v, cu_seqlens)
    out = _fwd(q, k, v, g, beta, initial_states, cu_seqlens, final_states_out, float(scale))
    return (out, final_states_out) if return_final_states else out


def linear_attention_update(q, k, v, g, state, beta=None, scale=None, state_indices=None):
    """The step of a decode loop: out like v, and the states advanced in place.  No backward: out
    belongs to no graph, and a state that requires a gradient is refused where gradients are recorded.

    q, k (batch, heads, dim_k), v (batch, v_heads, dim_v), g (batch, v_heads) or (v_heads,), beta (batch, v_heads) or None; or all of
    them with a seqlen axis behind the batch, for a few tokens at once.  state (slots, v_heads, dim_k, dim_v) float32.
    state_indices (batch,) int32: entry b uses state[state_indices[b]]; a negative index, or one that is not below the number of slots,
    gives zeros and leaves every state alone.  No slot may be named twice."""
    if not is_compiling():
        res = _ext._linear_attention_update_call(q, k, v, g, state, beta, state_indices, scale)
        if res is not NotImplemented:
            return res
    if scale is None:
        scale = q.shape[-1] ** -0.5
    if g.dim() == 1:
        g = g.expand(v.shape[:-1])
    return _update(q, k, v, g, state, beta, state_indices, float(scale))


def linear_attention_ref(q, k, v, g, beta=None, scale=None, initial_states=None, return_final_states=False):
    """The recurrence in plain PyTorch on any device, token by token, in float32 (float64 for float64 tensors);
    differentiable.  Sequences of one length; no cu_seqlens."""
    wide = torch.float64 if q.dtype == torch.float64 else torch.float32
    group = v.shape[2] // q.shape[2]
    g = g.to(wide).expand(v.shape[:3])
    q, k = (t.to(wide).repeat_interleave(group, dim=2) for t in (q, k))
    vw = v.to(wide) if beta is None else v.to(wide) * beta.to(wide)[..., None]
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    s = q.new_zeros(v.shape[0], v.shape[2], q.shape[-1], v.shape[-1]) if initial_states is None else initial_states.to(wide)
    outs = []
    for t in range(v.shape[1]):
        s = s * g[:, t].exp()[..., None, None] + k[:, t, :, :, None] * vw[:, t, :, None, :]
        outs.append(scale * (s * q[:, t, :, :, None]).sum(-2))
    out = (torch.stack(outs, 1) if outs else vw).to(v.dtype)
    return (out, s) if return_final_states else out
