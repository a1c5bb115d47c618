"""Low-level ops: Philox RNG restatement, sync-free quantise/pack helpers, and
the attention operators of the models."""

from .attention import AttentionMask, attention, attention_mask
from .philox import philox4x32_10, uniforms_for_elements
from .quant import pack_codes, quantize_codes, quantize_pack, unpack_dequant
from .rotary import qk_norm_rotary, rotary_frequencies

__all__ = [
    "philox4x32_10", "uniforms_for_elements", "pack_codes", "quantize_codes", "quantize_pack", "unpack_dequant",
    "AttentionMask", "attention", "attention_mask", "qk_norm_rotary", "rotary_frequencies",
]
