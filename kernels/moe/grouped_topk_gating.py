"""Beside the softmax gating of this package: sigmoid or softmax scores, a bias, groups of experts."""
from flydsl_amd.kernels.moe.grouped_topk_gating import build_grouped_topk_gating_module  # noqa: F401

__all__ = ["build_grouped_topk_gating_module"]
