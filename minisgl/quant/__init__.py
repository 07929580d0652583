"""Quantisation formats: MXFP4 routed experts, 4-bit group-scaled dense weights, MXFP8 rows, 4-bit KV cache rows."""

from .int4 import Int4Weight, dequantize_int4, int4_codes, int4_weight, quantize_int4
from .kv4 import dequantize_kv4, kv4_block_bytes, pack_kv4, quantize_kv4_reference, unpack_kv4
from .mx8 import dequantize_mx8_rows, quantize_mx8_rows_reference
from .mxfp4 import (MxfpExperts, block_scales, dequantize_mx8, dequantize_mxfp4, moe_experts_mx_reference,
                    quantize_mx8_reference, quantize_mxfp4, quantize_mxfp4_reference, scale_block_offsets)

__all__ = ["MxfpExperts", "quantize_mxfp4", "quantize_mxfp4_reference", "dequantize_mxfp4", "block_scales", "scale_block_offsets",
           "quantize_mx8_reference", "dequantize_mx8", "moe_experts_mx_reference", "Int4Weight", "int4_weight",
           "int4_codes", "quantize_int4", "dequantize_int4", "quantize_mx8_rows_reference", "dequantize_mx8_rows",
           "quantize_kv4_reference", "dequantize_kv4", "pack_kv4", "unpack_kv4", "kv4_block_bytes"]
