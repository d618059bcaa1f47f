"""Router gating with a bias for balance and groups of experts, beside ``build_topk_gating_softmax_module``: sigmoid or softmax scores, the best groups, the best experts of these.

    launch = build_grouped_topk_gating_module(256, 8, "f32", scores="sigmoid", groups=8, topk_groups=4, group_score="top2", renormalize=True, scale=2.5)
    launch(gating, bias, topk_weights, topk_indices, num_tokens, stream=stream)

``gating`` ``[tokens, num_experts]`` f32 / f16 / bf16 logits, ``bias`` ``[num_experts]`` fp32 or ``None``, ``topk_weights`` ``[tokens, topk]`` fp32 and ``topk_indices`` ``[tokens, topk]`` int32, in the
order found (best first).

``s`` is the sigmoid of the logits, or their softmax over the experts; ``c = s + bias`` is what is compared, without a bias the logits themselves, which order like ``s``.  The experts lie in ``groups``
runs of ``num_experts / groups``; a group is worth the sum of its two best ``s + bias`` (``group_score="top2"``) or its best ``c`` (``"max"``), the ``topk_groups`` best groups are kept, and of their experts the ``topk`` best.  The weights are ``s`` of these, without the
bias; with ``renormalize`` divided by ``max(their sum, 1e-20)``; then times ``scale``.  Scores, comparisons and weights are in 64 bits, the weights rounded once, and of equal ones the lower index comes first.

A logit of -inf masks its expert, a logit of NaN or a ``c`` that is NaN too: such an expert, or one of a group that is not kept, is taken only when nothing else is left, the lowest index first
and with weight 0, so a token always has ``topk`` different experts.
"""

from __future__ import annotations

import ctypes

import torch

from ... import _lib

_DTYPES = {"f32": (0, torch.float32, _lib.TYPE_FP32), "bf16": (1, torch.bfloat16, _lib.TYPE_BF16), "f16": (2, torch.float16, _lib.TYPE_FP16)}
_SCORES = {"sigmoid": 0, "softmax": 1}
_GROUP_SCORES = {"max": 0, "top2": 1}


class GroupedTopkGating:
    """Launcher returned by :func:`build_grouped_topk_gating_module`.  Holds no tensor references."""

    def __init__(self, num_experts, topk, dtype_str, scores, groups, topk_groups, group_score, renormalize, scale):
        self.num_experts, self.topk, self.dtype_str = num_experts, topk, dtype_str
        a = _lib.MoeGroupedGatingArgs()
        a.experts, a.topk, a.dtype, a.scores, a.groups, a.topk_groups = num_experts, topk, _DTYPES[dtype_str][0], _SCORES[scores], groups, topk_groups
        a.group_score, a.renormalize, a.scale = _GROUP_SCORES[group_score], int(renormalize), scale
        self._bytes = bytes(a)
        self._lib = _lib.lib()
        self._plans = {}  # (argument struct without its addresses, operands) by the number of tokens

    def _args(self, tokens):
        if not 0 <= tokens < 1 << 24:
            raise ValueError(f"num_tokens={tokens} outside [0, 2^24)")
        a = _lib.MoeGroupedGatingArgs.from_buffer_copy(self._bytes)
        a.tokens = tokens
        return a

    def _plan(self, tokens):
        f, e, k = _lib.MoeGroupedGatingArgs, self.num_experts, self.topk
        dt = _DTYPES[self.dtype_str]
        size = dt[1].itemsize
        ops = _lib.operands((f.gating, size, dt[2], size * tokens * e), (f.bias, 4, _lib.TYPE_FP32 + _lib.OPTIONAL, 4 * e), (f.weights, 4, _lib.TYPE_FP32, 4 * tokens * k),
                            (f.indices, 4, _lib.TYPE_INT32, 4 * tokens * k))
        return (bytes(self._args(tokens)),), ops

    def __call__(self, gating, bias, topk_weights, topk_indices, num_tokens, stream=None):
        """Launch on ``stream`` (``None``: the current stream of the device of ``gating``)."""
        if stream is not None and type(num_tokens) is int and type(gating) is torch.Tensor and gating.is_cuda and _lib.is_current(gating.get_device()):
            plan = self._plans.get(num_tokens)
            if plan is None:
                if len(self._plans) >= 256:
                    self._plans.clear()
                plan = self._plans[num_tokens] = self._plan(num_tokens)
            rc = _lib._native.launch(_lib.address("psg_moe_grouped_topk_gating"), plan[0], plan[1], stream, gating, bias, topk_weights, topk_indices)
            if rc != _lib._native.DECLINED:
                if rc:
                    _lib.check(rc, "psg_moe_grouped_topk_gating")
                return
        tokens = int(num_tokens)
        a = self._args(tokens)
        dev = None
        for name, field, t, least, dtype in (("gating", "gating", gating, tokens * self.num_experts, _DTYPES[self.dtype_str][1]), ("bias", "bias", bias, self.num_experts, torch.float32),
                                             ("topk_weights", "weights", topk_weights, tokens * self.topk, torch.float32), ("topk_indices", "indices", topk_indices, tokens * self.topk, torch.int32)):
            if t is None and name == "bias":
                continue
            if not isinstance(t, torch.Tensor):
                raise ValueError(f"{name} must be a device (cuda) tensor, got {type(t).__name__}")
            dev = dev or t.device
            _lib.check_operand(name, t, min_elems=least, elem_sizes=(dtype.itemsize,), device=dev)
            if t.dtype != dtype:
                raise ValueError(f"{name} is {t.dtype}, this launcher needs {dtype}")
            setattr(a, field, t.data_ptr())
        rc = _lib.launch_on(dev, self._lib.psg_moe_grouped_topk_gating, ctypes.byref(a), _lib.stream_on(stream, dev))
        if rc:
            _lib.check(rc, "psg_moe_grouped_topk_gating")


def build_grouped_topk_gating_module(num_experts: int, topk: int, dtype_str: str = "f32", *, scores: str = "sigmoid", groups: int = 1, topk_groups: int = 1, group_score: str = "top2",
                                     renormalize: bool = True, scale: float = 1.0):
    """Build the launcher; see the module for its call.  Up to 1024 experts, a multiple of ``groups``; up to 64 groups; ``topk`` up to 32 and to the experts of ``topk_groups`` groups."""
    if dtype_str not in _DTYPES:
        raise ValueError(f"dtype_str must be 'f32', 'f16' or 'bf16', got {dtype_str!r}")
    if scores not in _SCORES:
        raise ValueError(f"scores must be 'sigmoid' or 'softmax', got {scores!r}")
    if group_score not in _GROUP_SCORES:
        raise ValueError(f"group_score must be 'top2' or 'max', got {group_score!r}")
    num_experts, topk, groups, topk_groups, scale = int(num_experts), int(topk), int(groups), int(topk_groups), float(scale)
    if not 1 <= num_experts <= 1024:
        raise ValueError(f"num_experts={num_experts} is not supported: this kernel holds at most 1024 experts")
    if not 1 <= groups <= 64 or num_experts % groups:
        raise ValueError(f"groups={groups} must divide num_experts={num_experts} and be at most 64")
    if not 1 <= topk_groups <= groups:
        raise ValueError(f"topk_groups={topk_groups} must lie in [1, groups={groups}]")
    size = num_experts // groups
    if not 1 <= topk <= min(32, size * topk_groups):
        raise ValueError(f"topk={topk} must lie in [1, min(32, {size * topk_groups} experts of {topk_groups} groups)]")
    if group_score == "top2" and topk_groups < groups and size < 2:
        raise ValueError("group_score='top2' needs groups of at least two experts")
    if not abs(scale) <= torch.finfo(torch.float32).max:
        raise ValueError(f"scale must be a finite number of fp32, got {scale}")
    return GroupedTopkGating(num_experts, topk, dtype_str, scores, groups, topk_groups, group_score, bool(renormalize), scale)
