"""MI355X (gfx950) fused tANS FP8 decode: drop-in for the reference's
``rans_vectoradd`` package (rans_vectoradd/__init__.py:1-18)."""
from rans_vectoradd._C import (
    fp8_gemm_fused_tans,
    fp8_gemm_raw,
    fp8_memcpy,
    fp8_vecadd_fused_tans,
    fp8_vecadd_raw,
    gpu_tans_decode,
)
from rans_vectoradd.attention import (
    KvCache,
    rotary,
    rotary_append,
    rotary_frequencies,
    tree_attention,
)
from rans_vectoradd.layer import fp8_linear, fp8_quantize_rows, fp8_rmsnorm
from rans_vectoradd.data import QWEN3_14B_FP8_EXP, random_fp8_bytes
from . import tans_codec

__all__ = [
    "KvCache",
    "QWEN3_14B_FP8_EXP",
    "fp8_gemm_fused_tans",
    "fp8_gemm_raw",
    "fp8_linear",
    "fp8_memcpy",
    "fp8_quantize_rows",
    "fp8_rmsnorm",
    "fp8_vecadd_fused_tans",
    "fp8_vecadd_raw",
    "gpu_tans_decode",
    "random_fp8_bytes",
    "rotary",
    "rotary_append",
    "rotary_frequencies",
    "tans_codec",
    "tree_attention",
]
