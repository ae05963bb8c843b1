"""spark_kernels for B200 (sm_100a): the quantized-weight GEMM path of the reference library --
w4gemm (int4 W4A16), fp8gemm (e4m3) and fp4gemm (NVFP4 / MXFP4) with their quantizers and
packers -- behind the reference's op names, and the operators of a decode step between those GEMMs (a paged KV cache
in 4 bits with the attention over it, the residual norm). Hand-written CUDA in libspark_b200.so, reached
through its C ABI; torch is used for device memory and streams only."""

from . import _C, formats, kv4, ops, quant
from .kv4 import KV4Cache, kv4_append, kv4_attention, kv4_read
from .ops import (W4_GROUP, W4GateUpWeight, W4Weight, add_rmsnorm, w4gemm_swiglu, fp4_quantize, fp4gemm, fp8_quantize, fp8_quantize_block128, fp8gemm,
                  fp8gemm_block128, grouped_gemm_fp8, grouped_gemm_swiglu_fp8, num_variants, w4_quantize, w4_repack, w4gemm)
from .quant import FORMATS, FP4Linear, FP8Linear, Int4Linear, MXFP8Linear, make_linear

__all__ = ["_C", "ops", "quant", "formats", "kv4", "KV4Cache", "kv4_append", "kv4_attention", "kv4_read", "add_rmsnorm", "W4_GROUP", "W4Weight", "num_variants", "w4_quantize", "w4_repack",
           "w4gemm", "W4GateUpWeight", "w4gemm_swiglu", "fp8gemm", "fp8_quantize", "fp4gemm", "fp4_quantize", "fp8_quantize_block128",
           "fp8gemm_block128", "grouped_gemm_fp8", "grouped_gemm_swiglu_fp8", "FORMATS", "Int4Linear", "FP8Linear", "MXFP8Linear", "FP4Linear", "make_linear"]
