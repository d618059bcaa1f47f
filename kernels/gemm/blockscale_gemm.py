"""Beside the other products of this package: e4m3 with an fp32 scale for every block of 128, dense and grouped by expert."""
from flydsl_amd.kernels.gemm.blockscale_gemm import compile_blockscale_gemm, compile_grouped_blockscale_gemm  # noqa: F401
