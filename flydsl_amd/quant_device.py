"""On-device activation quantisers (HIP kernels behind the C ABI): the same bytes as the host helpers in
``flydsl_amd.quant`` (and therefore as the reference's ``pertoken_quant`` tests/utils.py:29-73 and
``per_1x32_f4_quant`` + ``shuffle_scale_w4`` tests/kernels/utils/gemm_common_utils.py:675-704, 645-672), produced
without leaving the GPU.  torch is used for the output allocations only."""

from __future__ import annotations

import contextlib
import ctypes

import torch

from . import _lib
from .quant import fp4x2, fp8_e8m0

_OUT_CODE = {torch.int8: 0, torch.float8_e4m3fn: 1}
_X_DTYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _x_code(x):
    if x.dtype not in _X_DTYPE:
        raise TypeError(f"input dtype {x.dtype} is not supported (fp32 / bf16 / fp16)")
    if not x.is_cuda or x.dim() != 2 or not x.is_contiguous():
        raise ValueError("x must be a contiguous 2-D device tensor")
    return _X_DTYPE[x.dtype]


def _check_out(x, *outs):
    index = x.get_device()
    for t in outs:
        if not t.is_cuda or t.get_device() != index or not t.is_contiguous():
            raise ValueError("out tensors must be contiguous and on the same device as x")


def pertoken_quant(x: torch.Tensor, quant_dtype=torch.int8, stream=None, out=None):
    """Per-row symmetric quantisation on the device.  Returns ``(y [M,K] quant_dtype, scale [M,1] fp32)``.
    ``out=(y, scale)`` reuses caller-owned outputs (1-byte ``[M,K]`` and fp32 ``[M]`` / ``[M,1]``): no allocation, so the
    call can be recorded into a HIP graph."""
    if type(out) in (tuple, list) and len(out) == 2 and stream is not None and isinstance(quant_dtype, torch.dtype) and quant_dtype in _OUT_CODE:
        y, scale = out
        rc = _lib._native.quant_pertoken(_lib.address("psg_quant_pertoken"), x, y, scale, _OUT_CODE[quant_dtype], stream)
        if rc != _lib._native.DECLINED:
            if rc:
                _lib.check(rc, "psg_quant_pertoken")
            return y if y.dtype == quant_dtype else y.view(quant_dtype), scale if scale.dim() == 2 and scale.shape[1] == 1 else scale.view(-1, 1)
    code = _x_code(x)
    if quant_dtype == torch.int8:
        out_code = 0
    elif quant_dtype == torch.float8_e4m3fn:
        out_code = 1
    else:
        raise ValueError(f"quant_dtype must be torch.int8 or torch.float8_e4m3fn, got {quant_dtype}")
    m, k = x.shape
    if out is None:
        y = torch.empty((m, k), dtype=torch.uint8, device=x.device)
        scale = torch.empty((m, 1), dtype=torch.float32, device=x.device)
    else:
        y, scale = out
        _check_out(x, y, scale)
        if y.numel() != m * k or y.element_size() != 1 or scale.numel() != m or scale.dtype != torch.float32:
            raise ValueError("out must be (1-byte [M,K], fp32 [M]) tensors")
    rc = _lib.lib().psg_quant_pertoken(x.data_ptr(), code, y.data_ptr(), scale.data_ptr(), m, k, out_code, _lib.stream_handle(stream))
    if rc:
        _lib.check(rc, "psg_quant_pertoken")
    return y if y.dtype == quant_dtype else y.view(quant_dtype), scale if scale.shape == (m, 1) else scale.view(m, 1)


def per_1x32_f4_quant(x: torch.Tensor, shuffle: bool = True, stream=None, out=None):
    """OCP-MX fp4 quantisation on the device.  Returns ``(packed [M,K/2], scales)`` where ``scales`` are e8m0 bytes over
    ``ceil(M/32)*32`` rows x ``K/32``: in the GEMM's shuffled layout when ``shuffle`` (default), row-major otherwise.
    Finite inputs only: a NaN / Inf in a block does not give the reference's 0xFF scale byte (the block maximum drops
    NaN)."""
    if type(out) in (tuple, list) and len(out) == 2 and stream is not None and type(shuffle) in (bool, int):
        packed, scales = out
        rc = _lib._native.quant_mxfp4(_lib.address("psg_quant_mxfp4"), x, packed, scales, 1 if shuffle else 0, stream)
        if rc != _lib._native.DECLINED:
            if rc:
                _lib.check(rc, "psg_quant_mxfp4")
            return packed if packed.dtype == fp4x2 else packed.view(fp4x2), scales if scales.dtype == fp8_e8m0 else scales.view(fp8_e8m0)
    code = _x_code(x)
    m, k = x.shape
    r = (m + 31) // 32 * 32
    if out is None:
        packed = torch.empty((m, k // 2), dtype=torch.uint8, device=x.device)
        scales = torch.empty((r, k // 32), dtype=torch.uint8, device=x.device)
    else:  # caller-owned outputs: no allocation, graph-capturable
        _check_out(x, *out)
        packed, scales = out
        if packed.element_size() != 1 or scales.element_size() != 1:  # counted in bytes, whatever the element type
            packed, scales = packed.view(torch.uint8), scales.view(torch.uint8)
        if packed.numel() != m * (k // 2) or scales.numel() != r * (k // 32):
            raise ValueError("out must be (packed [M,K/2], scales [ceil(M/32)*32, K/32]) byte tensors")
    rc = _lib.lib().psg_quant_mxfp4(x.data_ptr(), code, packed.data_ptr(), scales.data_ptr(), m, k, 1 if shuffle else 0,
                                    _lib.stream_handle(stream))
    if rc:
        _lib.check(rc, "psg_quant_mxfp4")
    return packed if packed.dtype == fp4x2 else packed.view(fp4x2), scales if scales.dtype == fp8_e8m0 else scales.view(fp8_e8m0)


_TENSORS = (torch.Tensor, torch.nn.Parameter)
_norm_plans = {}  # what shapes and types alone decide about a call of rmsnorm_quant, by them


def _norm_row_stride(name, t, x):
    """Elements from a row of ``t`` to the next; ``t`` has the shape, type and device of ``x`` and dense rows."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.shape != x.shape or t.dtype != x.dtype or t.device != x.device:
        raise ValueError(f"{name} must be a {tuple(x.shape)} {x.dtype} tensor on {x.device}, got {tuple(t.shape)} {t.dtype} on {t.device}")
    if (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        raise ValueError(f"{name} must have dense rows that do not overlap (strides {tuple(t.stride())})")
    return t.stride(0) if t.shape[0] > 1 else 0


def _allocating_for(stream, device):
    """Outputs of a launch on ``stream`` come from that stream's memory: a block of the current stream's may still be in use by what is queued there."""
    handle = _lib.stream_on(stream, device)
    if handle == torch.cuda.current_stream(device).cuda_stream:
        return contextlib.nullcontext()
    return torch.cuda.stream(torch.cuda.ExternalStream(handle, device=device) if handle else torch.cuda.default_stream(device))


def _norm_args(x, weight, eps, quant_dtype):
    """The argument struct of a call, without its addresses and strides."""
    if quant_dtype is not None and quant_dtype not in _OUT_CODE:
        raise ValueError(f"quant_dtype must be torch.int8, torch.float8_e4m3fn or None, got {quant_dtype}")
    if not isinstance(x, torch.Tensor) or x.dtype not in _X_DTYPE:
        raise TypeError(f"x must be a tensor of fp32, bf16 or fp16, got {getattr(x, 'dtype', type(x).__name__)}")
    if not x.is_cuda or x.dim() != 2 or x.shape[1] < 1:
        raise ValueError("x must be a 2-D device tensor with at least one column")
    if x.shape[0] >= 1 << 31 or x.shape[1] > 1 << 24:
        raise ValueError(f"x may have up to 2^31 - 1 rows of up to 2^24 elements, got {tuple(x.shape)}")
    if not isinstance(weight, torch.Tensor) or weight.dtype not in (x.dtype, torch.float32) or weight.numel() != x.shape[1]:
        raise ValueError(f"weight must hold {x.shape[1]} elements of {x.dtype} or fp32")
    eps = float(eps)
    if not 0.0 <= eps < float("inf"):
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    a = _lib.RmsnormArgs()
    a.rows, a.dim = x.shape
    a.x_dtype, a.weight_dtype = _X_DTYPE[x.dtype], _X_DTYPE[weight.dtype]
    a.out_dtype = -1 if quant_dtype is None else _OUT_CODE[quant_dtype]
    a.eps = eps
    return a


def _norm_plan(x, weight, eps, quant_dtype):
    a = _norm_args(x, weight, eps, quant_dtype)
    f, any_, rows, dim, eb = _lib.RmsnormArgs, _lib.TYPE_ANY, a.rows, a.dim, x.element_size()
    typed = {torch.float32: _lib.TYPE_FP32, torch.bfloat16: _lib.TYPE_BF16, torch.float16: _lib.TYPE_FP16}
    xt, size, optional, exact = typed[x.dtype] + _lib.ROWS, rows << 32 | dim, _lib.OPTIONAL, _lib.EXACT
    ops = _lib.operands((f.x, eb, xt, size), (f.weight, weight.element_size(), typed[weight.dtype] + exact, dim * weight.element_size()), (f.residual, eb, xt + optional, size),
                        (f.residual_out, eb, xt + optional, size), (f.normed, eb, xt + optional, size), (f.q, 1, any_ + exact, rows * dim), (f.scale, 4, _lib.TYPE_FP32 + exact, 4 * rows))
    return (bytes(a),), ops


def rmsnorm_quant(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: torch.Tensor | None = None, quant_dtype=torch.float8_e4m3fn,
                  residual_out: torch.Tensor | None = None, normed: torch.Tensor | None = None, stream=None, out=None):
    """Residual addition, root-mean-square norm and per-row quantisation in one launch: what a decoder layer has in front of its quantised
    products.

    ``h = x + residual``, rounded to the type of ``x`` and written to ``residual_out`` (``None``: to ``residual`` itself); ``h = x`` without a residual.
    ``y = h * weight / sqrt(mean(h^2) + eps)`` in fp32, written to ``normed`` in the type of ``x`` where one is given (what a router or an unquantised layer reads).
    Returns ``(q [rows, dim] quant_dtype, scale [rows, 1] fp32)`` by the rules of :func:`pertoken_quant` (``scale`` 1 for a row of zeros, NaN as 0, infinities as the largest
    value, int8 towards zero), but from ``y`` before it is rounded; with ``quant_dtype=None`` the norm alone, and ``normed`` (allocated if it is ``None``) is returned.

    ``x``, ``residual``, ``residual_out`` and ``normed`` are ``[rows, dim]`` of one type (fp32 / bf16 / fp16), each with dense rows any distance apart (a slice of the
    columns of a wider tensor will do); ``weight`` ``[dim]`` has that type or fp32.  ``residual_out`` may be ``residual`` or ``x``, ``normed`` may be ``x``, but not both the same.  ``rows`` may be
    0, and ``dim`` anything up to 2^24.  ``out=(q, scale)`` reuses caller-owned outputs (1-byte ``[rows, dim]`` and fp32 ``[rows]`` / ``[rows, 1]``): no allocation, so
    the call can be recorded into a HIP graph.  ``stream=None`` is the current stream of the device of ``x``; without ``out`` the outputs are allocated for that stream, as torch
    allocates what is made with it as the current one."""
    # a call with its outputs, on the current device, goes on in native code, which looks at the operands (eps a number: a tensor would be found by its identity, whatever it holds now)
    if stream is not None and type(out) is tuple and len(out) == 2 and type(x) is torch.Tensor and type(weight) in _TENSORS and quant_dtype is not None and (residual is not None or residual_out is None) and isinstance(eps, (float, int)):
        q, scale = out
        h = residual if residual_out is None else residual_out
        if type(q) is type(scale) is torch.Tensor and x.is_cuda and _lib.is_current(x.get_device()):
            key = (x.shape, x.dtype, weight.dtype, eps, quant_dtype)
            plan = _norm_plans.get(key)
            if plan is None:
                a = _norm_plan(x, weight, eps, quant_dtype)
                if len(_norm_plans) >= 256:
                    _norm_plans.clear()
                plan = _norm_plans[key] = a
            rc = _lib._native.launch(_lib.address("psg_rmsnorm_quant"), plan[0], plan[1], stream, x, weight, residual, h, normed, q, scale)
            if rc != _lib._native.DECLINED:
                if rc:
                    _lib.check(rc, "psg_rmsnorm_quant")
                return q.view(quant_dtype) if q.dtype is not quant_dtype else q, scale if scale.dim() == 2 and scale.shape[1] == 1 else scale.view(-1, 1)
    a = _norm_args(x, weight, eps, quant_dtype)
    rows, dim = x.shape
    if weight.device != x.device or not weight.is_contiguous():
        raise ValueError("weight must be contiguous and on the device of x")
    a.x_stride = _norm_row_stride("x", x, x)
    a.x, a.weight = x.data_ptr(), weight.data_ptr()
    if residual is not None:
        h = residual if residual_out is None else residual_out
        a.residual_stride, a.residual_out_stride = _norm_row_stride("residual", residual, x), _norm_row_stride("residual_out", h, x)
        a.residual, a.residual_out = residual.data_ptr(), h.data_ptr()
    elif residual_out is not None:
        raise ValueError("residual_out is given without a residual")
    q = scale = None
    if quant_dtype is None:
        if out is not None:
            raise ValueError("out is given with quant_dtype=None: the result is normed")
        if normed is None:
            with _allocating_for(stream, x.device):
                normed = torch.empty((rows, dim), dtype=x.dtype, device=x.device)
    elif out is None:
        with _allocating_for(stream, x.device):
            q, scale = torch.empty((rows, dim), dtype=quant_dtype, device=x.device), torch.empty((rows, 1), dtype=torch.float32, device=x.device)
    else:
        q, scale = out
        _check_out(x, q, scale)
        if q.numel() != x.numel() or q.element_size() != 1 or scale.numel() != rows or scale.dtype != torch.float32:
            raise ValueError("out must be (1-byte [rows, dim], fp32 [rows] or [rows, 1]) tensors")
    if normed is not None:
        a.normed_stride = _norm_row_stride("normed", normed, x)
        a.normed = normed.data_ptr()
    if q is not None:
        a.q, a.scale = q.data_ptr(), scale.data_ptr()
    rc = _lib.launch_on(x.device, _lib.lib().psg_rmsnorm_quant, ctypes.byref(a), _lib.stream_on(stream, x.device))
    if rc:
        _lib.check(rc, "psg_rmsnorm_quant")
    if q is None:
        return normed
    return q if q.dtype == quant_dtype else q.view(quant_dtype), scale if scale.shape == (rows, 1) else scale.view(rows, 1)
