"""A linear-attention block from this package's operators, trained, prefilled and decoded:

    y, stream = rms_norm_fn(x, weight, residual=stream)
    q | k | v | z | a | b = y W_in                                 z gates the output, a and b the state
    q | k | v = causal_conv1d_fn(q | k | v, activation="silu")      read in place by the next line, as column slices
    o = gated_delta_rule_fn(q, k, v, g = -exp(A) softplus(a + dt), beta = sigmoid(b))
    x = (rms_norm_fn(o) * silu(z)) W_out

`DeltaBlock.forward` runs whole sequences (with gradients, or as a prefill that fills a cache), `DeltaBlock.step` one
token of each entry of a batch whose states lie in slots.  In a step the norm in front of the projection leaves 8 bits a
value if asked to (rms_norm_quant_fn), which is what a cache or a link between devices would carry.

    python delta_block.py [--dim 512] [--heads 4] [--v-heads 8] [--steps 20]
"""
import argparse
import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
from causal_conv1d import (causal_conv1d_fn, causal_conv1d_update, dequantize_rows, gated_delta_rule_fn, gated_delta_rule_update,  # noqa: E402
                           rms_norm_fn, rms_norm_quant_fn)


class Cache:
    """What a decode step reads: the convolution's last inputs and the rule's states, one slot a request."""

    def __init__(self, block, slots):
        w = block.conv_weight
        # rows of channels, as the channel-last convolution takes them
        self.conv = torch.zeros(slots, block.width - 1, block.channels, dtype=w.dtype, device=w.device).transpose(1, 2)
        self.state = torch.zeros(slots, block.v_heads, block.dim_k, block.dim_v, device=w.device)


class DeltaBlock(torch.nn.Module):
    def __init__(self, dim, heads, v_heads, dim_k=128, dim_v=128, width=4, eps=1e-6, device="cuda", dtype=torch.bfloat16):
        super().__init__()
        self.heads, self.v_heads, self.dim_k, self.dim_v, self.width, self.eps = heads, v_heads, dim_k, dim_v, width, eps
        self.channels = 2 * heads * dim_k + v_heads * dim_v
        parts = (self.channels, v_heads * dim_v, v_heads, v_heads)
        self.parts = parts

        def rand(*shape, scale=1.0, dtype=dtype):
            return torch.nn.Parameter((scale * torch.randn(*shape, device=device)).to(dtype))
        self.norm = torch.nn.Parameter(torch.ones(dim, device=device))
        self.w_in = rand(sum(parts), dim, scale=dim ** -0.5)
        self.conv_weight = rand(self.channels, width, scale=0.5)
        self.conv_bias = rand(self.channels, scale=0.1)
        self.a_log = torch.nn.Parameter(torch.linspace(0.0, 2.0, v_heads, device=device))
        self.dt = torch.nn.Parameter(torch.full((v_heads,), -4.0, device=device))
        self.head_norm = torch.nn.Parameter(torch.ones(dim_v, device=device))
        self.w_out = rand(dim, v_heads * dim_v, scale=(v_heads * dim_v) ** -0.5)

    def _gates(self, a, b):
        return -self.a_log.exp() * F.softplus(a.float() + self.dt), torch.sigmoid(b)

    def _heads(self, mixed):
        """q, k, v as views of the convolution's output (..., channels)."""
        k0, v0 = self.heads * self.dim_k, 2 * self.heads * self.dim_k
        return (mixed[..., :k0].unflatten(-1, (self.heads, self.dim_k)), mixed[..., k0:v0].unflatten(-1, (self.heads, self.dim_k)),
                mixed[..., v0:].unflatten(-1, (self.v_heads, self.dim_v)))

    def _out(self, o, z):
        return F.linear(rms_norm_fn(o, self.head_norm, eps=self.eps).flatten(-2) * F.silu(z), self.w_out)

    def forward(self, x, stream, cache=None, slots=None):
        """x (batch, seqlen, dim) and the residual stream like it, in float32 -> the block's x and the new stream.  With a cache
        the states behind the last token go to its rows `slots` (batch,)."""
        y, stream = rms_norm_fn(x, self.norm, residual=stream, eps=self.eps)
        mixed, z, a, b = F.linear(y, self.w_in).split(self.parts, -1)
        mixed = mixed.transpose(1, 2)                    # (batch, channels, seqlen), channels contiguous
        if cache is None:
            mixed = causal_conv1d_fn(mixed, self.conv_weight, self.conv_bias, activation="silu")
        else:
            mixed, last = causal_conv1d_fn(mixed, self.conv_weight, self.conv_bias, return_final_states=True, activation="silu")
            cache.conv[slots] = last
        q, k, v = self._heads(mixed.transpose(1, 2))
        g, beta = self._gates(a, b)
        if cache is None:
            o = gated_delta_rule_fn(q, k, v, g, beta, qk_l2norm=True)
        else:
            o, cache.state[slots] = gated_delta_rule_fn(q, k, v, g, beta, return_final_states=True, qk_l2norm=True)
        return self._out(o, z), stream

    @torch.no_grad()
    def step(self, x, stream, cache, slots, in_8_bits=False):
        """x and stream (batch, dim), one token of each entry; slots (batch,) int32, negative for entries that are padding."""
        if in_8_bits:
            y8, scales, stream = rms_norm_quant_fn(x, self.norm, residual=stream, eps=self.eps)
            y = dequantize_rows(y8, scales, x.dtype)
        else:
            y, stream = rms_norm_fn(x, self.norm, residual=stream, eps=self.eps)
        mixed, z, a, b = F.linear(y, self.w_in).split(self.parts, -1)
        mixed = causal_conv1d_update(mixed, cache.conv, self.conv_weight, self.conv_bias, activation="silu", conv_state_indices=slots)
        q, k, v = self._heads(mixed)
        g, beta = self._gates(a, b)
        o = gated_delta_rule_update(q, k, v, g, beta, cache.state, state_indices=slots, qk_l2norm=True)
        return self._out(o, z), stream


def main():
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--dim", type=int, default=512)
    p.add_argument("--heads", type=int, default=4)
    p.add_argument("--v-heads", type=int, default=8)
    p.add_argument("--steps", type=int, default=20)
    a = p.parse_args()
    torch.manual_seed(0)
    blocks = torch.nn.ModuleList(DeltaBlock(a.dim, a.heads, a.v_heads) for _ in range(2))

    def run(x, **more):
        stream = torch.zeros(x.shape, device=x.device)
        for i, block in enumerate(blocks):
            x, stream = block(x, stream, **{k: v[i] for k, v in more.items()})
        return x.float() + stream

    # Training: recall the token of four places before.
    data = torch.randn(4, 512, a.dim, device="cuda").bfloat16()
    target = F.pad(data, (0, 0, 4, 0))[:, :-4].float()
    optimizer = torch.optim.AdamW(blocks.parameters(), lr=3e-3)
    for step in range(a.steps):
        loss = F.mse_loss(run(data), target)
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        if step % 5 == 0 or step == a.steps - 1:
            print("step %3d  loss %.4f" % (step, loss.item()), flush=True)

    # Serving: prefill two prompts into slots 3 and 1, then decode on, beside what whole sequences give.
    caches = [Cache(block, 5) for block in blocks]
    slots = torch.tensor([3, 1], device="cuda")
    with torch.no_grad():
        whole = run(data[:2, :80])
        run(data[:2, :70], cache=caches, slots=[slots] * 2)
        worst = 0.0
        for t in range(70, 80):
            x, stream = data[:2, t], torch.zeros(2, a.dim, device="cuda")
            for block, cache in zip(blocks, caches):
                x, stream = block.step(x, stream, cache, slots.int())
            worst = max(worst, (x.float() + stream - whole[:, t]).abs().max().item())
    print("decoding after a prefill differs from the whole sequence by %.3g of %.3g" % (worst, whole.abs().max().item()))


if __name__ == "__main__":
    main()
