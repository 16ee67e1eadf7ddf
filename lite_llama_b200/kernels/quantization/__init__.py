"""Quantised GEMMs with the reference's signatures (reference: lite_llama/kernels/quantization/__init__.py:13-17), and the
products of microscaled 4-bit operands, which it has not."""

from .mxfp4 import (MXFP4, fused_moe_mxfp4, mxfp4_dequantize, mxfp4_gate_up, mxfp4_matmul, mxfp4_pack, mxfp4_quantize, mxfp4_quantize_weight,
                    skip_rmsnorm_mxfp4)
from .w4a16 import PackedW4, interleave_gate_up, w4a16_matmul, w4a16_matmul_packed, w4a16_pack
from .w8a16 import w8a16_matmul
from .w8a8 import quantize_activations_int8, smoothquant_matmul, smoothquant_matmul_prequant

__all__ = ["w8a16_matmul", "w4a16_matmul", "smoothquant_matmul", "smoothquant_matmul_prequant", "quantize_activations_int8", "w4a16_pack", "w4a16_matmul_packed", "PackedW4", "interleave_gate_up",
           "MXFP4", "mxfp4_dequantize", "mxfp4_gate_up", "mxfp4_matmul", "mxfp4_pack", "mxfp4_quantize", "mxfp4_quantize_weight", "skip_rmsnorm_mxfp4", "fused_moe_mxfp4"]
