"""Beside the other products of this package: 4-bit weights with group scales."""
from flydsl_amd.kernels.gemm.w4a16_gemm import compile_w4a16_gemm  # noqa: F401
