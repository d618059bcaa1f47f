"""The grouped products without a GPU: what is refused."""

import ctypes

import pytest
import torch

from flydsl_amd import _lib
from kernels.gemm.grouped_gemm import compile_grouped_gemm

SHAPE, DTYPE, NULL, ALIGN = -2, -3, -1, -6


@pytest.mark.parametrize("change", [dict(in_dtype="fp4"), dict(out_dtype="fp32"), dict(N=24), dict(N=0), dict(K=0), dict(K=96), dict(K=48, in_dtype="bf16"), dict(groups=0), dict(groups=4097)])
def test_builder_refuses(change):
    with pytest.raises(ValueError):
        compile_grouped_gemm(**{**dict(N=64, K=128, groups=4), **change})


def test_builder_caches():
    assert compile_grouped_gemm(N=64, K=128, groups=4) is compile_grouped_gemm(N=64, K=128, groups=4, in_dtype="fp8", out_dtype="bf16")


def _args(**change):
    a = _lib.GroupedArgs()
    a.c = a.a = a.w = a.scale_a = a.scale_b = a.offsets = 0x1000
    a.M, a.N, a.K, a.groups, a.in_dtype = 10, 64, 128, 4, 1
    for k, v in change.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,code", [
    (dict(c=0), NULL), (dict(a=0), NULL), (dict(w=0), NULL), (dict(offsets=0), NULL), (dict(scale_a=0), NULL), (dict(scale_b=0, in_dtype=0), NULL), (dict(in_dtype=6), DTYPE), (dict(in_dtype=-1), DTYPE),
    (dict(out_dtype=2), DTYPE), (dict(M=0), SHAPE), (dict(M=(1 << 22) + 1), SHAPE), (dict(groups=0), SHAPE), (dict(groups=4097), SHAPE), (dict(N=40), SHAPE), (dict(K=96), SHAPE),
    (dict(K=0), SHAPE), (dict(N=1 << 18, K=1 << 14), SHAPE), (dict(N=1 << 24, K=64), SHAPE), (dict(N=16, K=1 << 25), SHAPE), (dict(tile_rows=48), SHAPE), (dict(M=1 << 22, N=1 << 20, tile_rows=16), SHAPE),
    (dict(M=1 << 22, N=1 << 12, tile_rows=16), SHAPE),  # 2^24 workgroups and more
    (dict(a=0x1008), ALIGN), (dict(w=0x1008), ALIGN), (dict(c=0x1008), ALIGN), (dict(scale_b=0x1008), ALIGN), (dict(scale_a=0x1002), ALIGN), (dict(offsets=0x1002), ALIGN),
])
def test_c_entry_refuses(change, code):
    handle = _lib.lib()
    assert handle.psg_gemm_grouped(ctypes.byref(_args(**change)), None) == code
    assert handle.psg_last_error()
    assert handle.psg_gemm_grouped(None, None) == NULL


def test_host_tensors_are_refused():
    fn = compile_grouped_gemm(N=64, K=128, groups=4, in_dtype="int8")
    z = lambda *s, dt=torch.int8: torch.zeros(*s, dtype=dt)
    good = z(10, 64, dt=torch.bfloat16), z(10, 128), z(4, 64, 128), z(10, dt=torch.float32), z(4, 64, dt=torch.float32), z(5, dt=torch.int32)
    for stream in (None, 7):
        with pytest.raises(ValueError, match="device"):
            fn(*good, 10, stream)
        with pytest.raises(ValueError, match="device"):
            fn(None, *good[1:], 10, stream)
        with pytest.raises(ValueError, match="outside"):
            fn(*good, 0, stream)


def test_tile_rows_are_those_of_the_thread_that_set_them():
    """The launcher is one for all callers of its sizes; what a thread forces is its own, also in the plans that are kept."""
    import threading

    fn = compile_grouped_gemm(N=64, K=192, groups=4)
    fn.tile_rows = 32
    try:
        seen = []

        def other():
            seen.append(fn.tile_rows)
            seen.append(fn._args(10).tile_rows)
            fn.tile_rows = 64
            seen.append(fn._args(10).tile_rows)

        t = threading.Thread(target=other)
        t.start()
        t.join()
        assert seen == [0, 0, 64] and fn.tile_rows == 32 and fn._args(10).tile_rows == 32
    finally:
        fn.tile_rows = 0
    assert fn._args(10).tile_rows == 0
