"""Products of rows grouped by expert with the experts' own weights, the groups' sizes ragged and known on the device only.

    fn = compile_grouped_gemm(N=..., K=..., groups=..., in_dtype="fp8", out_dtype="bf16")
    fn(C, A, B, scale_a, scale_b, offsets, M, stream)

``C[r] = A[r] @ B[e].T`` (times ``scale_a[r] * scale_b[e]`` for 8-bit operands) for ``offsets[e] <= r < offsets[e + 1]``: ``A [M, K]`` and ``C [M, N]`` row-major, sorted by group, without
padding; ``B`` ``[groups, N, K]``, every weight in the order of ``flydsl_amd.layout.shuffle_weight``; ``scale_a [M]``, ``scale_b [groups, N]`` fp32; ``offsets [groups + 1]`` int32 on the
device, not decreasing.  Nothing is read on the host, so the call can be recorded into a HIP graph and replayed with other sizes.  Groups may be empty; rows of ``C``
outside of ``[offsets[0], offsets[groups])`` are left as they are.  ``M`` bounds the rows, and decides with ``groups`` which tiles are taken: it should be near the rows that
there are.

The MoE stages (``compile_moe_gemm1`` / ``compile_moe_gemm2``) fuse the gather of the tokens, the gated activation and the routing weights into such a product, over
blocks padded by the sorter; this is the plain one, also in 16 bits: experts of another form, adapters per request, the rows of a sorted batch as they lie.
"""

from __future__ import annotations

import ctypes
import functools
import threading

import torch

from ... import _lib

_IN = {"fp8": (1, torch.float8_e4m3fn), "int8": (1, torch.int8), "fp16": (2, torch.float16), "bf16": (2, torch.bfloat16)}
_OUT = {"bf16": (torch.bfloat16, _lib.TYPE_BF16), "fp16": (torch.float16, _lib.TYPE_FP16)}


class _Forced(threading.local):
    tile_rows = 0  # rows of a tile; 0: the library's choice (another for tests)


class GroupedGemm:
    """Launcher returned by :func:`compile_grouped_gemm`.  Holds no tensor references."""

    def __init__(self, N, K, groups, in_dtype, out_dtype):
        self.N, self.K, self.groups, self.in_dtype, self.out_dtype = N, K, groups, in_dtype, out_dtype
        self._eb, self._scaled = _IN[in_dtype][0], _IN[in_dtype][0] == 1
        self._lib = _lib.lib()
        self._plans = {}  # (argument struct without its addresses, operands) by M
        self._forced = _Forced()  # (one launcher serves all callers of its sizes: what a thread forces is its own)

    @property
    def tile_rows(self):
        return self._forced.tile_rows

    @tile_rows.setter
    def tile_rows(self, rows):
        self._forced.tile_rows = rows

    def _args(self, M):
        if M < 1 or M > 1 << 22:
            raise ValueError(f"M={M} outside [1, 2^22]")
        a = _lib.GroupedArgs()
        a.M, a.N, a.K, a.groups = M, self.N, self.K, self.groups
        a.in_dtype, a.out_dtype, a.tile_rows = _lib.IN_DTYPE[self.in_dtype], _lib.OUT_DTYPE[self.out_dtype], self.tile_rows
        return a

    def _plan(self, M):
        f, any_ = _lib.GroupedArgs, _lib.TYPE_ANY
        typed = any_ if self._scaled else {"bf16": _lib.TYPE_BF16, "fp16": _lib.TYPE_FP16}[self.in_dtype]
        ops = [(f.c, 2, _OUT[self.out_dtype][1], 2 * M * self.N), (f.a, self._eb, typed, self._eb * M * self.K), (f.w, self._eb, typed, self._eb * self.groups * self.N * self.K),
               (f.offsets, 4, _lib.TYPE_INT32, 4 * (self.groups + 1))]
        if self._scaled:
            ops += [(f.scale_a, 4, _lib.TYPE_FP32, 4 * M), (f.scale_b, 4, _lib.TYPE_FP32, 4 * self.groups * self.N)]
        return (bytes(self._args(M)),), _lib.operands(*ops)

    def __call__(self, C, A, B, scale_a, scale_b, offsets, M, stream=None):
        """Launch on ``stream`` (``None``: the current stream of the device of ``C``).  ``scale_a`` and ``scale_b`` are only read for 8-bit operands."""
        if stream is not None and type(M) is int and type(C) is torch.Tensor and C.is_cuda and _lib.is_current(C.get_device()):
            key = (M, self._forced.tile_rows)
            plan = self._plans.get(key)
            if plan is None:
                if len(self._plans) >= 256:
                    self._plans.clear()
                plan = self._plans[key] = self._plan(M)
            more = (scale_a, scale_b) if self._scaled else ()
            rc = _lib._native.launch(_lib.address("psg_gemm_grouped"), plan[0], plan[1], stream, C, A, B, offsets, *more)
            if rc != _lib._native.DECLINED:
                if rc:
                    _lib.check(rc, "psg_gemm_grouped")
                return
        M = int(M)
        a = self._args(M)
        named = [("C", "c", C, M * self.N, 2, _OUT[self.out_dtype][0]), ("A", "a", A, M * self.K, self._eb, None if self._scaled else _IN[self.in_dtype][1]),
                 ("B", "w", B, self.groups * self.N * self.K, self._eb, None if self._scaled else _IN[self.in_dtype][1]), ("offsets", "offsets", offsets, self.groups + 1, 4, torch.int32)]
        if self._scaled:
            named += [("scale_a", "scale_a", scale_a, M, 4, torch.float32), ("scale_b", "scale_b", scale_b, self.groups * self.N, 4, torch.float32)]
        dev = None
        for name, field, t, least, size, dtype in named:
            if not isinstance(t, torch.Tensor):
                raise ValueError(f"{name} must be a device (cuda) tensor, got {type(t).__name__}")
            dev = dev or t.device
            _lib.check_operand(name, t, min_elems=least, elem_sizes=(size,), device=dev)
            if dtype is not None and t.dtype != dtype:
                raise ValueError(f"{name} is {t.dtype}, this launcher needs {dtype}")
            setattr(a, field, t.data_ptr())
        rc = _lib.launch_on(dev, self._lib.psg_gemm_grouped, ctypes.byref(a), _lib.stream_on(stream, dev))
        if rc:
            _lib.check(rc, "psg_gemm_grouped")


def compile_grouped_gemm(*, N: int, K: int, groups: int, in_dtype: str = "fp8", out_dtype: str = "bf16"):
    """Build the launcher; see the module for its call.  ``in_dtype`` fp8 / int8 / fp16 / bf16, ``out_dtype`` bf16 / fp16, ``N % 16 == 0``, ``K`` bytes of a row a multiple of 64, up to
    4096 groups."""
    if in_dtype not in _IN:
        raise ValueError(f"in_dtype must be fp8/int8/fp16/bf16, got {in_dtype!r}")
    if out_dtype not in _OUT:
        raise ValueError(f"out_dtype must be bf16/fp16, got {out_dtype!r}")
    N, K, groups = int(N), int(K), int(groups)
    if N < 16 or N % 16:
        raise ValueError(f"N must be a positive multiple of 16 (preshuffled B layout), got {N}")
    if K < 1 or K * _IN[in_dtype][0] % 64:
        raise ValueError(f"K*elem_bytes must be a positive multiple of 64 (preshuffled B layout), got K={K}")
    if not 1 <= groups <= 4096:
        raise ValueError(f"groups={groups} outside [1, 4096]")
    return _cached_launcher(N, K, groups, in_dtype, out_dtype)


@functools.lru_cache(maxsize=256)
def _cached_launcher(N, K, groups, in_dtype, out_dtype):
    return GroupedGemm(N, K, groups, in_dtype, out_dtype)
