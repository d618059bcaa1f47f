"""The 4-bit weights with group scales without a GPU: layout, quantiser, refusals."""

import ctypes

import pytest
import torch

from flydsl_amd import _lib, layout, quant
from kernels.gemm.w4a16_gemm import compile_w4a16_gemm

SHAPE, DTYPE, NULL, ALIGN = -2, -3, -1, -6


@pytest.mark.parametrize("n,k", [(16, 32), (48, 128), (32, 416)])
def test_layout_is_the_documented_map(n, k):
    g = torch.Generator().manual_seed(n + k)
    codes = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8)
    flat = layout.shuffle_weight_w4a16(codes).view(-1)
    blocks = (k + 127) // 128
    assert flat.numel() == n * blocks * 64
    seen = torch.zeros(flat.numel() * 2, dtype=torch.bool)
    for row in range(n):
        for e in range(k):
            j, gr, i = e % 128 // 32, e % 32 // 8, e % 8
            bit = 2 * i if i % 2 == 0 else 16 + 2 * (i - 1)
            byte = ((row // 16) * blocks + e // 128) * 1024 + gr * 256 + (row % 16) * 16 + j * 4 + bit // 8
            assert (int(flat[byte]) >> (bit % 8)) & 15 == int(codes[row, e])
            seen[byte * 2 + (bit % 8) // 4] = True
    nibbles = torch.stack([flat & 15, flat >> 4], -1).view(-1)
    assert (nibbles[~seen] == 0).all()  # what pads a row to whole blocks


def test_scales_and_zeros_layout():
    s = torch.arange(32 * 3).view(32, 3)
    v = layout.shuffle_group_scales(s)
    z = torch.randint(0, 16, (32, 3), dtype=torch.uint8)
    p = layout.shuffle_group_zeros(z)
    for row in range(32):
        for g in range(3):
            assert v[row // 16, g, row % 16] == s[row, g]
            assert (int(p[row // 16, g, row % 16 // 2]) >> (4 * (row & 1))) & 15 == int(z[row, g])


@pytest.mark.parametrize("zero_points", [False, True])
@pytest.mark.parametrize("group", [32, 128])
def test_quantiser(group, zero_points):
    w = torch.randn(32, 256, generator=torch.Generator().manual_seed(1))
    w[3, :group] = 0
    w[4, :group] = w[4, :group].abs() + 1  # 0 lies outside of what the group has
    codes, scale, zero = quant.pergroup_w4_quant(w, group, zero_points)
    assert codes.dtype == torch.uint8 and codes.max() <= 15 and scale.shape == (32, 256 // group) and scale.dtype == torch.bfloat16
    assert (zero is None) == (not zero_points)
    z = torch.full_like(scale, 8, dtype=torch.float32) if zero is None else zero.float()
    back = (codes.view(32, -1, group).float() - z.unsqueeze(-1)) * scale.float().unsqueeze(-1)
    # half a step, and at an end of the codes another half (symmetric: 7.5 steps on codes up to 7; zero points: the range's ends are rounded) and what the scale's rounding
    # takes off 15 steps (2^-8 each)
    off = (back.view(32, 256) - w).abs().view(32, -1, group) / scale.float().unsqueeze(-1)
    assert (off <= 1.0 + 16 * 2.0**-8).all() and (off <= 0.5 + 1e-6).float().mean() > 0.9
    assert (back.view(32, 256)[3, :group] == 0).all()
    with pytest.raises(ValueError, match="multiple of group_size"):
        quant.pergroup_w4_quant(w[:, :100], group)


def test_layout_refusals():
    z = lambda *s, dt=torch.uint8: torch.zeros(*s, dtype=dt)
    for bad in (z(8, 32), z(16, 48), z(16, 32, dt=torch.int8), z(16, 32) + 16):
        with pytest.raises(ValueError):
            layout.shuffle_weight_w4a16(bad)
    with pytest.raises(ValueError):
        layout.shuffle_group_scales(z(8, 2))
    for bad in (z(16, 2) + 16, z(16, 2, dt=torch.int32)):
        with pytest.raises(ValueError):
            layout.shuffle_group_zeros(bad)


@pytest.mark.parametrize("change", [dict(in_dtype="fp8"), dict(epilogue="tanh"), dict(group_size=16), dict(group_size=96), dict(N=24), dict(N=0), dict(K=64), dict(K=192), dict(K=0)])
def test_builder_refuses(change):
    with pytest.raises(ValueError):
        compile_w4a16_gemm(**{**dict(N=64, K=256, group_size=128), **change})


def test_builder_caches():
    assert compile_w4a16_gemm(N=64, K=256) is compile_w4a16_gemm(N=64, K=256, group_size=128)


def _args(**change):
    a = _lib.W4A16Args()
    a.c = a.a = a.w = a.scales = 0x1000
    a.M, a.N, a.K, a.group = 1, 64, 256, 128
    for k, v in change.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,code", [
    (dict(c=0), NULL), (dict(a=0), NULL), (dict(w=0), NULL), (dict(scales=0), NULL), (dict(epilogue=1), NULL), (dict(dtype=2), DTYPE), (dict(epilogue=5), NULL), (dict(epilogue=5, bias=0x1000), DTYPE),
    (dict(M=0), SHAPE), (dict(M=65537), SHAPE), (dict(N=8), SHAPE), (dict(N=72), SHAPE), (dict(K=192), SHAPE), (dict(K=0), SHAPE), (dict(group=16), SHAPE), (dict(N=1 << 20, K=1 << 13), SHAPE),
    (dict(M=65536, K=1 << 16), SHAPE), (dict(a=0x1008), ALIGN), (dict(w=0x1008), ALIGN), (dict(c=0x1004), ALIGN), (dict(scales=0x1004), ALIGN), (dict(zeros=0x1001), ALIGN),
    (dict(epilogue=1, bias=0x1002), ALIGN),
])
def test_c_entry_refuses(change, code):
    handle = _lib.lib()
    assert handle.psg_gemm_w4a16(ctypes.byref(_args(**change)), None) == code
    assert handle.psg_last_error()
    assert handle.psg_gemm_w4a16(None, None) == NULL


def test_host_tensors_are_refused():
    fn = compile_w4a16_gemm(N=64, K=256, zero_points=True, epilogue="bias")
    b = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="device"):
        fn(b(1, 64), b(1, 256), torch.zeros(64, 128, dtype=torch.uint8), b(4, 2, 16), torch.zeros(4, 2, 8, dtype=torch.uint8), b(64), 1, 7)
    with pytest.raises(ValueError, match="device"):
        fn(None, b(1, 256), None, None, None, None, 1)
    with pytest.raises(ValueError, match="outside"):
        fn(None, None, None, None, None, None, 0)


@pytest.mark.parametrize("zero_points", [False, True])
def test_quantiser_refuses_scales_that_are_none(zero_points):
    """A group whose scale is beyond the type of the scales would stand for NaN."""
    w = torch.ones(16, 128)
    w[5, 7] = -8e5  # over 7.5 steps; with zero points the next row, over 15: beyond 65504
    w[6, 7] = 8e5 if zero_points else 0.0
    w[6, 8] = -8e5 if zero_points else 0.0
    with pytest.raises(ValueError, match="float16"):
        quant.pergroup_w4_quant(w, 64, zero_points, torch.float16)
    codes, scale, zero = quant.pergroup_w4_quant(w, 64, zero_points, torch.bfloat16)
    assert torch.isfinite(scale).all()
    w[1, 1] = float("inf")
    with pytest.raises(ValueError, match="finite"):
        quant.pergroup_w4_quant(w, 64, zero_points)
