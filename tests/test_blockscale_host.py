"""The block-scaled products, their quantiser and the routing by groups without a GPU: host quantisers, and what is refused."""

import ctypes

import pytest
import torch

from flydsl_amd import _lib, quant, quant_device
from kernels.gemm.blockscale_gemm import compile_blockscale_gemm, compile_grouped_blockscale_gemm
from kernels.moe.grouped_topk_gating import build_grouped_topk_gating_module

SHAPE, DTYPE, NULL, ALIGN = -2, -3, -1, -6


# ---- host quantisers ----


@pytest.mark.parametrize("m,k", [(1, 1), (3, 127), (5, 128), (2, 129), (7, 1000)])
def test_rows_by_their_definition(m, k):
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(k)) * 7
    x[0, :1] = 0
    if k > 300:
        x[1, 128:256] = 0
        x[2, 5], x[2, 200], x[2, 201] = float("nan"), float("inf"), float("-inf")
    q, s = quant.per_1x128_f8_quant(x)
    assert q.shape == (m, k) and q.dtype == torch.float8_e4m3fn and s.shape == (-(-k // 128), m) and s.dtype == torch.float32
    for r in range(m):
        for b in range(s.shape[0]):
            v = x[r, 128 * b : 128 * b + 128].clone()
            v[v.isnan()] = 0
            v = v.clamp(-448, 448) if v.isinf().any() else v
            want = v.abs().max() / 448
            assert s[b, r] == (want if want > 0 else 1)
            assert torch.equal(q[r, 128 * b : 128 * b + 128].float(), (v / s[b, r]).to(torch.float8_e4m3fn).float())


@pytest.mark.parametrize("shape", [(16, 64), (3, 128, 128), (2, 144, 320), (272, 192)])
def test_weights_by_their_definition(shape):
    w = torch.randn(*shape, generator=torch.Generator().manual_seed(shape[-1]))
    w.view(-1, *shape[-2:])[0, :16, :64] *= 100
    q, s = quant.per_128x128_f8_quant(w)
    n, k = shape[-2:]
    assert q.shape == w.shape and s.shape == (*shape[:-2], -(-n // 128), -(-k // 128))
    q, s, w = q.float().view(-1, n, k), s.view(-1, *s.shape[-2:]), w.view(-1, n, k)
    for e in range(w.shape[0]):
        for i in range(s.shape[1]):
            for j in range(s.shape[2]):
                at = slice(128 * i, 128 * i + 128), slice(128 * j, 128 * j + 128)
                assert s[e, i, j] == w[e][at].abs().max() / 448
                assert torch.equal(q[e][at], (w[e][at] / s[e, i, j]).to(torch.float8_e4m3fn).float())
    zero, one = quant.per_128x128_f8_quant(torch.zeros(16, 64))
    assert (zero.float() == 0).all() and (one == 1).all()
    with pytest.raises(ValueError, match="finite"):
        quant.per_128x128_f8_quant(torch.full((16, 64), float("nan")))


# ---- products ----


@pytest.mark.parametrize("change", [dict(out_dtype="fp32"), dict(N=24), dict(N=0), dict(K=0), dict(K=96), dict(K=-64)])
def test_product_builders_refuse(change):
    with pytest.raises(ValueError):
        compile_blockscale_gemm(**{**dict(N=64, K=128), **change})
    with pytest.raises(ValueError):
        compile_grouped_blockscale_gemm(**{**dict(N=64, K=128, groups=4), **change})


def test_product_builders():
    for groups in (0, 4097):
        with pytest.raises(ValueError):
            compile_grouped_blockscale_gemm(N=64, K=128, groups=groups)
    assert compile_blockscale_gemm(N=64, K=128) is compile_blockscale_gemm(N=64, K=128, out_dtype="bf16")
    assert compile_grouped_blockscale_gemm(N=64, K=128, groups=1) is not compile_blockscale_gemm(N=64, K=128)


def _product(**change):
    a = _lib.BlockscaleArgs()
    a.c = a.a = a.w = a.scale_a = a.scale_b = a.offsets = 0x1000
    a.M, a.N, a.K, a.groups = 10, 64, 128, 4
    for k, v in change.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,code", [
    (dict(c=0), NULL), (dict(a=0), NULL), (dict(w=0), NULL), (dict(scale_a=0), NULL), (dict(scale_b=0), NULL), (dict(offsets=0), NULL), (dict(out_dtype=2), DTYPE), (dict(out_dtype=-1), DTYPE),
    (dict(M=0), SHAPE), (dict(M=(1 << 22) + 1), SHAPE), (dict(groups=0), SHAPE), (dict(groups=4097), SHAPE), (dict(groups=0, offsets=0), SHAPE), (dict(N=40), SHAPE), (dict(N=0), SHAPE), (dict(K=96), SHAPE),
    (dict(K=0), SHAPE), (dict(N=1 << 18, K=1 << 14), SHAPE), (dict(N=1 << 24, K=64), SHAPE), (dict(N=16, K=1 << 25), SHAPE), (dict(tile_rows=48), SHAPE), (dict(tile_rows=1), SHAPE), (dict(slice_columns=16), SHAPE), (dict(tile_rows=16, slice_columns=64), SHAPE), (dict(tile_rows=128, slice_columns=64), SHAPE), (dict(tile_rows=64, slice_columns=128), SHAPE), (dict(tile_rows=128, slice_columns=256), SHAPE), (dict(tile_rows=1, slice_columns=16), SHAPE), (dict(scale_a_stride=9), SHAPE),
    (dict(scale_a_stride=-1), SHAPE), (dict(K=1 << 15, M=1 << 22), SHAPE), (dict(scale_a_stride=1 << 31), SHAPE), (dict(K=256, scale_a_stride=1 << 29), SHAPE), (dict(M=1 << 22, N=1 << 12, tile_rows=16), SHAPE), (dict(M=1 << 22, N=1 << 16, K=64, groups=4096), SHAPE),
    (dict(a=0x1008), ALIGN), (dict(w=0x1008), ALIGN), (dict(c=0x1008), ALIGN), (dict(scale_b=0x1002), ALIGN), (dict(scale_a=0x1002), ALIGN), (dict(offsets=0x1002), ALIGN),
])
def test_product_entry_refuses(change, code):
    handle = _lib.lib()
    assert handle.psg_gemm_blockscale(ctypes.byref(_product(**change)), None) == code
    assert handle.psg_last_error()
    assert handle.psg_gemm_blockscale(None, None) == NULL


def test_products_of_host_tensors_are_refused():
    z = lambda *s, dt=torch.int8: torch.zeros(*s, dtype=dt)
    fn, grouped = compile_blockscale_gemm(N=64, K=128), compile_grouped_blockscale_gemm(N=64, K=128, groups=4)
    good = z(10, 64, dt=torch.bfloat16), z(10, 128), z(64, 128), z(1, 10, dt=torch.float32), z(1, 1, dt=torch.float32)
    for stream in (None, 7):
        for call in (lambda *a: fn(*a, stream), lambda *a: grouped(*a[:-1], z(5, dt=torch.int32), a[-1], stream)):
            with pytest.raises(ValueError, match="device"):
                call(*good, 10)
            with pytest.raises(ValueError, match="device"):
                call(None, *good[1:], 10)
            with pytest.raises(ValueError, match="outside"):
                call(*good, 0)
    with pytest.raises(TypeError):
        fn(*good)  # no M
    with pytest.raises(TypeError):
        grouped(*good, 10)  # no offsets


def test_tiles_are_those_of_the_thread_that_set_them():
    import threading

    fn, seen = compile_blockscale_gemm(N=64, K=192), []
    fn.tile = (32, 64)
    try:
        t = threading.Thread(target=lambda: seen.append((fn._args(10).tile_rows, fn._args(10).slice_columns)))
        t.start()
        t.join()
        assert seen == [(0, 0)] and (fn._args(10).tile_rows, fn._args(10).slice_columns) == (32, 64)
    finally:
        fn.tile = (0, 0)


# ---- quantiser ----


def _quant(**change):
    a = _lib.QuantBlockArgs()
    a.x = a.q = a.scale = 0x1000
    a.rows, a.dim = 4, 128
    for k, v in change.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,code", [
    (dict(x=0), NULL), (dict(q=0), NULL), (dict(scale=0), NULL), (dict(x_dtype=3), DTYPE), (dict(x_dtype=-1), DTYPE), (dict(rows=-1), SHAPE), (dict(rows=1 << 31), SHAPE), (dict(dim=0), SHAPE),
    (dict(dim=(1 << 24) + 1), SHAPE), (dict(gated=2), SHAPE), (dict(gated=-1), SHAPE), (dict(x_stride=127), SHAPE), (dict(x_stride=255, gated=1), SHAPE), (dict(x_stride=1 << 41), SHAPE), (dict(scale_stride=3), SHAPE),
    (dict(scale_stride=1 << 41), SHAPE), (dict(x=0x1002), ALIGN), (dict(x=0x1001, x_dtype=1), ALIGN), (dict(scale=0x1002), ALIGN),
])
def test_quantiser_entry_refuses(change, code):
    handle = _lib.lib()
    assert handle.psg_quant_block(ctypes.byref(_quant(**change)), None) == code
    assert handle.psg_last_error()
    assert handle.psg_quant_block(None, None) == NULL


def test_quantiser_without_rows_launches_nothing():
    assert _lib.lib().psg_quant_block(ctypes.byref(_quant(rows=0, x=0, q=0, scale=0)), None) == 0


def test_quantiser_refuses_host_tensors():
    with pytest.raises(ValueError, match="device"):
        quant_device.per_1x128_f8_quant(torch.zeros(4, 128))
    with pytest.raises(TypeError):
        quant_device.per_1x128_f8_quant(torch.zeros(4, 128, dtype=torch.int32))


# ---- routing ----


@pytest.mark.parametrize("change", [
    dict(dtype_str="f64"), dict(scores="relu"), dict(group_score="mean"), dict(num_experts=0), dict(num_experts=1025), dict(groups=0), dict(groups=3), dict(groups=128, num_experts=256), dict(topk_groups=0),
    dict(topk_groups=9), dict(topk=0), dict(topk=33, topk_groups=8), dict(topk=17, topk_groups=2), dict(groups=64, topk_groups=4, topk=4), dict(scale=float("inf")), dict(scale=float("nan")), dict(scale=1e39),
])
def test_routing_builder_refuses(change):
    with pytest.raises(ValueError):
        build_grouped_topk_gating_module(**{**dict(num_experts=64, topk=4, groups=8, topk_groups=4), **change})


def test_routing_builder():
    build_grouped_topk_gating_module(64, 4, groups=64, topk_groups=4, group_score="max")
    build_grouped_topk_gating_module(64, 4, groups=64, topk_groups=64)
    build_grouped_topk_gating_module(1, 1)
    fn = build_grouped_topk_gating_module(64, 4)
    good = torch.zeros(3, 64), None, torch.zeros(3, 4), torch.zeros(3, 4, dtype=torch.int32)
    for stream in (None, 7):
        with pytest.raises(ValueError, match="device"):
            fn(*good, 3, stream=stream)
        with pytest.raises(ValueError, match="outside"):
            fn(*good, -1, stream=stream)


def _route(**change):
    a = _lib.MoeGroupedGatingArgs()
    a.gating = a.bias = a.weights = a.indices = 0x1000
    a.tokens, a.experts, a.topk, a.groups, a.topk_groups, a.group_score, a.scale = 5, 64, 4, 8, 4, 1, 1.0
    for k, v in change.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,code", [
    (dict(gating=0), NULL), (dict(weights=0), NULL), (dict(indices=0), NULL), (dict(dtype=3), DTYPE), (dict(scores=2), DTYPE), (dict(group_score=2), DTYPE), (dict(tokens=-1), SHAPE), (dict(tokens=1 << 24), SHAPE),
    (dict(experts=0), SHAPE), (dict(experts=1032), SHAPE), (dict(groups=0), SHAPE), (dict(groups=7), SHAPE), (dict(groups=128, experts=128), SHAPE), (dict(topk_groups=0), SHAPE), (dict(topk_groups=9), SHAPE),
    (dict(topk=0), SHAPE), (dict(topk=33), SHAPE), (dict(topk=9, topk_groups=1), SHAPE), (dict(groups=64), SHAPE), (dict(scale=float("nan")), SHAPE), (dict(scale=float("inf")), SHAPE), (dict(gating=0x1002), ALIGN),
    (dict(bias=0x1002), ALIGN), (dict(weights=0x1002), ALIGN), (dict(indices=0x1002), ALIGN),
])
def test_routing_entry_refuses(change, code):
    handle = _lib.lib()
    assert handle.psg_moe_grouped_topk_gating(ctypes.byref(_route(**change)), None) == code
    assert handle.psg_last_error()
    assert handle.psg_moe_grouped_topk_gating(None, None) == NULL


def test_routing_without_tokens_launches_nothing():
    assert _lib.lib().psg_moe_grouped_topk_gating(ctypes.byref(_route(tokens=0, gating=0, weights=0, indices=0)), None) == 0
