"""Causal depthwise conv1d for AMD MI355X (gfx950): same Python surface as
Dao-AILab/causal-conv1d 1.6.1 (causal_conv1d/__init__.py:1-3 of the reference)."""
__version__ = "1.6.1"

from causal_conv1d.causal_conv1d_interface import causal_conv1d_fn, causal_conv1d_update
from causal_conv1d.causal_conv1d_varlen import causal_conv1d_fwd_varlen_states, causal_conv1d_varlen_states
from causal_conv1d.gated_delta_rule import gated_delta_rule_fn, gated_delta_rule_update
from causal_conv1d.layer_norm import layer_norm_fn
from causal_conv1d.linear_attention import linear_attention_fn, linear_attention_update
from causal_conv1d.rms_norm import dequantize_rows, rms_norm_fn, rms_norm_quant_fn

__all__ = ["causal_conv1d_fn", "causal_conv1d_update", "causal_conv1d_varlen_states",
           "causal_conv1d_fwd_varlen_states", "gated_delta_rule_fn", "gated_delta_rule_update", "rms_norm_fn",
           "rms_norm_quant_fn", "dequantize_rows", "linear_attention_fn", "linear_attention_update", "layer_norm_fn"]
