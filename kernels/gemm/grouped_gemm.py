"""Beside the other products of this package: rows grouped by expert, ragged sizes."""
from flydsl_amd.kernels.gemm.grouped_gemm import compile_grouped_gemm  # noqa: F401
