"""What the norm with quantised rows refuses, without a GPU: nothing is launched."""

import ctypes

import pytest
import torch

from flydsl_amd import _lib, quant_device

BAD = -2, -3, -1, -6  # PSG_E_SHAPE, PSG_E_DTYPE, PSG_E_NULL, PSG_E_ALIGN
SHAPE, DTYPE, NULL, ALIGN = BAD


def _args(**change):
    a = _lib.RmsnormArgs()
    a.x = a.weight = a.q = a.scale = 0x1000
    a.rows, a.dim, a.x_dtype, a.weight_dtype, a.out_dtype, a.eps = 3, 64, 1, 1, 1, 1e-6
    for k, v in change.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,code", [
    (dict(x=0), NULL), (dict(weight=0), NULL), (dict(q=0), NULL), (dict(scale=0), NULL), (dict(residual=0x1000), NULL), (dict(out_dtype=-1), NULL),
    (dict(x_dtype=3), DTYPE), (dict(x_dtype=-1), DTYPE), (dict(weight_dtype=2), DTYPE), (dict(out_dtype=2), DTYPE),
    (dict(rows=-1), SHAPE), (dict(rows=1 << 31), SHAPE), (dict(dim=0), SHAPE), (dict(dim=(1 << 24) + 1), SHAPE), (dict(eps=-1e-6), SHAPE), (dict(eps=float("nan")), SHAPE),
    (dict(eps=float("inf")), SHAPE), (dict(x_stride=63), SHAPE), (dict(normed_stride=-64), SHAPE), (dict(residual_out_stride=(1 << 40) + 1), SHAPE),
    (dict(x=0x1001), ALIGN), (dict(weight=0x1001), ALIGN), (dict(scale=0x1002), ALIGN), (dict(normed=0x1001), ALIGN), (dict(weight=0x1002, weight_dtype=0), ALIGN),
])
def test_c_entry_refuses(change, code):
    handle = _lib.lib()
    assert handle.psg_rmsnorm_quant(ctypes.byref(_args(**change)), None) == code
    assert handle.psg_last_error()


def test_c_entry_takes_no_rows_and_no_arguments():
    handle = _lib.lib()
    assert handle.psg_rmsnorm_quant(ctypes.byref(_args(rows=0, x=0, q=0, scale=0)), None) == 0
    assert handle.psg_rmsnorm_quant(None, None) == NULL


def test_host_tensors_and_wrong_arguments_are_refused():
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.ones(64, dtype=torch.bfloat16)
    out = torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4)
    for more in (dict(), dict(out=out, stream=7), dict(residual=x, out=out, stream=7)):
        with pytest.raises(ValueError, match="device tensor"):
            quant_device.rmsnorm_quant(x, w, **more)
    with pytest.raises(ValueError, match="quant_dtype"):
        quant_device.rmsnorm_quant(x, w, quant_dtype=torch.float16)
    with pytest.raises(TypeError, match="fp32, bf16 or fp16"):
        quant_device.rmsnorm_quant(x.double(), w)
    with pytest.raises(TypeError, match="fp32, bf16 or fp16"):
        quant_device.rmsnorm_quant(None, w, out=out, stream=7)


def test_both_16_bit_outputs_in_one_place_are_refused():
    handle = _lib.lib()
    for change in (dict(residual=0x2000, residual_out=0x1000, normed=0x1000), dict(residual=0x2000, residual_out=0x2000, normed=0x2000), dict(residual=0x2000, residual_out=0x3000, normed=0x3000, out_dtype=-1)):
        assert handle.psg_rmsnorm_quant(ctypes.byref(_args(**change)), None) == SHAPE
        assert b"lost" in handle.psg_last_error()
