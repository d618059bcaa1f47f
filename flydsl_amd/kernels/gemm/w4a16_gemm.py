"""Products of a few rows of 16-bit activations with 4-bit weights, one scale (and a zero point or none) per group along K.

    fn = compile_w4a16_gemm(N=..., K=..., group_size=128, in_dtype="bf16", zero_points=False, epilogue="none")
    fn(C, A, W, scales, zeros, bias, M, stream)

``C[m, n] = sum_k A[m, k] * scales[n, k / group] * (code[n, k] - zero[n, k / group])`` with the epilogues of :func:`compile_preshuffle_gemm`; sums in fp32.  ``A [M, K]``, ``C [M, N]``,
``scales`` and ``bias [N]`` have the type ``in_dtype`` (bf16 / fp16).  ``W``, ``scales`` and ``zeros`` are in the order of ``flydsl_amd.layout.shuffle_weight_w4a16``,
``shuffle_group_scales`` and ``shuffle_group_zeros``, laid out once (``flydsl_amd.quant.pergroup_w4_quant`` makes the codes); without zero points a code counts from 8 and
``zeros`` is ``None``.

Infinities and NaN of ``A`` go where the sum of ``A * (scale * (code - zero))`` in fp32 has them, rows beside them are as without; such values are taken one at a time, so a batch full of
them is slow.

It is made for decode: the weights are read once for every 32 rows, or for every 16 where ``N`` and ``K`` are large (more than 96 columns a compute unit on rows too long for one pass).
"""

from __future__ import annotations

import ctypes
import functools

import torch

from ... import _lib

_TYPES = {"bf16": (torch.bfloat16, _lib.TYPE_BF16), "fp16": (torch.float16, _lib.TYPE_FP16)}


class W4A16Gemm:
    """Launcher returned by :func:`compile_w4a16_gemm`.  Holds no tensor references."""

    def __init__(self, N, K, group_size, in_dtype, zero_points, epilogue):
        self.N, self.K, self.group_size = N, K, group_size
        self.in_dtype, self.zero_points, self.epilogue = in_dtype, zero_points, epilogue
        self.dtype, self._type = _TYPES[in_dtype]
        self._has_bias = epilogue != "none"
        self._lib = _lib.lib()
        self._plans = {}  # (argument struct without its addresses, operands) by M
        scales = N * (K // group_size)
        # least elements and sizes of the weight's tensors
        self._sizes = {"W": N * ((K + 127) // 128) * 64, "scales": scales, "zeros": scales // 2 if zero_points else 0, "bias": N if self._has_bias else 0}

    def _args(self, M):
        if M < 1 or M > 65536:
            raise ValueError(f"M={M} outside [1, 65536]")
        a = _lib.W4A16Args()
        a.M, a.N, a.K, a.group = M, self.N, self.K, self.group_size
        a.dtype, a.epilogue = _lib.OUT_DTYPE[self.in_dtype], _lib.EPILOGUE[self.epilogue]
        return a

    def _plan(self, M):
        f, s, t, byte = _lib.W4A16Args, self._sizes, self._type, _lib.TYPE_ANY
        ops = [(f.c, 2, t, 2 * M * self.N), (f.a, 2, t, 2 * M * self.K), (f.w, 1, byte, s["W"]), (f.scales, 2, t, 2 * s["scales"])]
        if self.zero_points:
            ops.append((f.zeros, 1, byte, s["zeros"]))
        if self._has_bias:
            ops.append((f.bias, 2, t, 2 * self.N))
        return (bytes(self._args(M)),), _lib.operands(*ops)

    def __call__(self, C, A, W, scales, zeros, bias, M, stream=None):
        """Launch on ``stream`` (``None``: the current stream of the device of ``C``).  ``zeros`` is only read with zero points, ``bias`` only with an epilogue."""
        if stream is not None and type(M) is int and type(C) is torch.Tensor and C.is_cuda and _lib.is_current(C.get_device()):
            plan = self._plans.get(M)
            if plan is None:
                if len(self._plans) >= 256:
                    self._plans.clear()
                plan = self._plans[M] = self._plan(M)
            more = (zeros, bias) if self.zero_points and self._has_bias else (zeros,) if self.zero_points else (bias,) if self._has_bias else ()
            rc = _lib._native.launch(_lib.address("psg_gemm_w4a16"), plan[0], plan[1], stream, C, A, W, scales, *more)
            if rc != _lib._native.DECLINED:
                if rc:
                    _lib.check(rc, "psg_gemm_w4a16")
                return
        M = int(M)
        a = self._args(M)
        named = {"C": (C, M * self.N, 2), "A": (A, M * self.K, 2), "W": (W, self._sizes["W"], 1), "scales": (scales, self._sizes["scales"], 2)}
        if self.zero_points:
            named["zeros"] = (zeros, self._sizes["zeros"], 1)
        if self._has_bias:
            named["bias"] = (bias, self.N, 2)
        dev = None
        for name, (t, least, size) in named.items():
            if not isinstance(t, torch.Tensor):
                raise ValueError(f"{name} must be a device (cuda) tensor, got {type(t).__name__}")
            dev = dev or t.device
            _lib.check_operand(name, t, min_elems=least, elem_sizes=(size,), device=dev)
            if size == 2 and t.dtype != self.dtype:
                raise ValueError(f"{name} is {t.dtype}, this launcher was built for {self.dtype}")
            setattr(a, name.lower(), t.data_ptr())
        rc = _lib.launch_on(dev, self._lib.psg_gemm_w4a16, ctypes.byref(a), _lib.stream_on(stream, dev))
        if rc:
            _lib.check(rc, "psg_gemm_w4a16")


def compile_w4a16_gemm(*, N: int, K: int, group_size: int = 128, in_dtype: str = "bf16", zero_points: bool = False, epilogue: str = "none"):
    """Build the launcher; see the module for its call.  ``group_size`` 32, 64 or 128, ``K`` a multiple of it, ``N`` of 16; ``epilogue`` as in
    :func:`compile_preshuffle_gemm`."""
    if in_dtype not in _TYPES:
        raise ValueError(f"in_dtype must be bf16/fp16, got {in_dtype!r}")
    if epilogue not in _lib.EPILOGUE:
        raise ValueError(f"epilogue must be none/bias/bias_relu/bias_silu/bias_gelu, got {epilogue!r}")
    if group_size not in (32, 64, 128):
        raise ValueError(f"group_size must be 32, 64 or 128, got {group_size!r}")
    N, K = int(N), int(K)
    if N < 16 or N % 16:
        raise ValueError(f"N must be a positive multiple of 16, got {N}")
    if K < group_size or K % group_size:
        raise ValueError(f"K must be a positive multiple of group_size={group_size}, got {K}")
    return _cached_launcher(N, K, int(group_size), in_dtype, bool(zero_points), epilogue)


@functools.lru_cache(maxsize=256)
def _cached_launcher(N, K, group_size, in_dtype, zero_points, epilogue):
    return W4A16Gemm(N, K, group_size, in_dtype, zero_points, epilogue)
