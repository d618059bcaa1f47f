"""GPU tests of the quantiser with a scale for every 128 columns.

Without the gate the bytes are the host quantiser's: the same fp32 quotients, rounded the same way.  Gated, against the definition in 64 bits; u = 2^-24: z = exp(-|g|) is off by 3 u (the
exponential instruction two, its correction one), 1 + z by 2.5 u at most, its reciprocal by 1.5 u more, sigmoid's product, g's and the other half's by u each: y by 10.5 u together, the scale by
one more, the quotient by those and one of its own.
"""

import pytest
import torch

from flydsl_amd import quant, quant_device

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn
U = 2.0**-24
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _x(rows, cols, dt, seed, std=3.0):
    return (std * torch.randn(rows, cols, generator=torch.Generator().manual_seed(seed))).to(dt)


def _bytes(t):
    return t.view(torch.uint8)


def _check_plain(x, q, s):
    want_q, want_s = quant.per_1x128_f8_quant(x.cpu())
    assert q.shape == want_q.shape and q.dtype == FP8 and s.shape == want_s.shape
    assert torch.equal(s.cpu(), want_s)
    assert torch.equal(_bytes(q.cpu()), _bytes(want_q))


def _check_gated(x, q, s):
    dim = x.shape[1] // 2
    g, v = x.double().cpu().split(dim, 1)
    y = g / (1 + torch.exp(-g)) * v
    b = torch.nn.functional.pad(y, (0, -dim % 128)).view(y.shape[0], -1, 128)
    want = b.abs().amax(-1) / 448
    want[want == 0] = 1
    assert ((s.double().cpu().t() - want).abs() <= 11.5 * U * want).all()
    v = (b / want.unsqueeze(-1)).view(y.shape[0], -1)[:, :dim]
    assert ((q.double().cpu() - v).abs() <= torch.clamp(2.0**-4 * v.abs(), min=2.0**-10) * (1 + 2.0**-4) + 24 * U * v.abs()).all()


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("dim", [1, 7, 8, 9, 120, 127, 128, 129, 136, 511, 512, 513, 520, 640, 1021, 2056, 7168])
@pytest.mark.parametrize("rows", [1, 3, 17])
def test_rows_are_the_host_quantisers(rows, dim, dt):
    x = _x(rows, dim, dt, dim)
    if dim > 300:
        x[0, 128:256] = 0
    print(f"quant {rows}x{dim} {dt}", flush=True)
    _check_plain(x, *quant_device.per_1x128_f8_quant(x.cuda()))
    x = _x(rows, 2 * dim, dt, dim + 1)
    _check_gated(x, *quant_device.per_1x128_f8_quant(x.cuda(), gated=True))


@pytest.mark.parametrize("rows,dim,gated", [(16384, 512, False), (5003, 2056, False), (9000, 1000, True), (4111, 2050, True), (70000, 129, False)])
def test_many_rows(rows, dim, gated):
    """Grids of many workgroups, and their end."""
    x = _x(rows, dim * (2 if gated else 1), torch.bfloat16, rows)
    print(f"quant {rows}x{dim} gated={gated}", flush=True)
    q, s = quant_device.per_1x128_f8_quant(x.cuda(), gated=gated)
    (_check_gated if gated else _check_plain)(x, q, s)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows,dim,off", [(5, 200, 1), (19, 512, 3), (3, 1025, 8), (40, 7, 5), (2500, 512, 1)])
def test_strided_rows_and_outputs(rows, dim, off, gated, dt):
    """x a slice of a wider tensor at any element, scales into the first columns of a wider one; what lies around the outputs stays as it is."""
    cols = dim * (2 if gated else 1)
    wide = _x(rows, cols + off + 9, dt, rows).cuda()
    x = wide[:, off : off + cols]
    blocks = -(-dim // 128)
    q = torch.full((rows * dim + 64,), 0x55, dtype=torch.uint8, device="cuda")
    scale = torch.full((blocks + 1, rows + 6), -3.0, device="cuda")
    print(f"quant strided {rows}x{dim}+{off} gated={gated} {dt}", flush=True)
    for stream in (None, torch.cuda.current_stream()):
        out = q[32 : 32 + rows * dim].view(rows, dim), scale[:blocks, 2 : 2 + rows]
        got, s = quant_device.per_1x128_f8_quant(x, gated, stream, out)
        assert got.data_ptr() == out[0].data_ptr() and got.dtype == FP8 and s.data_ptr() == out[1].data_ptr()
        (_check_gated if gated else _check_plain)(x, got, s)
        assert (q[:32] == 0x55).all() and (q[32 + rows * dim :] == 0x55).all()
        assert (scale[:, :2] == -3).all() and (scale[:, 2 + rows :] == -3).all() and (scale[blocks] == -3).all()
        q[32 : 32 + rows * dim] = 0x55
        scale[:blocks, 2 : 2 + rows] = -3


@pytest.mark.parametrize("dt", DTYPES)
def test_special_values(dt):
    x = _x(8, 640, dt, 1)
    inf = float("inf")
    x[0, 3], x[1, 130], x[2, 5], x[2, 6] = float("nan"), inf, -inf, inf
    x[3, :128] = float("nan")
    x[4, :] = inf
    x[5, 128:256] = 0
    x[5, 130] = -0.0
    x[6, 639] = torch.finfo(dt).max
    x[7, :128] = torch.finfo(dt).tiny
    _check_plain(x, *quant_device.per_1x128_f8_quant(x.cuda()))


def test_scales_of_a_few_bits():
    """Blocks whose scale is near or below the smallest number: 1 where it is rounded to 0, and no code beyond the largest."""
    x = torch.zeros(6, 128)
    for i, e in enumerate((-126, -135, -140, -141, -142, -149)):
        x[i] = torch.linspace(-1, 1, 128) * 2.0**e
    q, s = quant_device.per_1x128_f8_quant(x.cuda())
    _check_plain(x, q, s)
    assert (q.float().abs() <= 448).all()
    big = torch.full((2, 128), 3e38)
    big[1, 7] = -1.0
    _check_plain(big, *quant_device.per_1x128_f8_quant(big.cuda()))


def test_gated_special_values():
    inf, nan = float("inf"), float("nan")
    g = torch.tensor([1.0, inf, -inf, nan, 2.0, -200.0, 200.0, -100.0, 0.0, -0.0, inf, 1.0])
    u = torch.tensor([2.0, 3.0, 5.0, 1.0, nan, 7.0, -7.0, inf, inf, 1.0, 0.0, -inf])
    # silu(inf) = inf, silu(-inf) = -inf * 0 = NaN, as the formula has it; silu(-100) * inf = -inf, 0 * inf and inf * 0 NaN
    y = torch.tensor([2 / (1 + torch.e**-1), 448.0, 0.0, 0.0, 0.0, 0.0, -1400.0, -448.0, 0.0, 0.0, 0.0, -448.0])
    x = torch.cat([g, u]).unsqueeze(0)
    q, s = quant_device.per_1x128_f8_quant(x.cuda(), gated=True)
    assert (s.cpu() - 1400 / 448).abs() < 1e-6
    want = (y / (1400 / 448)).to(FP8).float()
    assert torch.equal(q.cpu().float(), want.unsqueeze(0))


def test_gate_far_below_zero():
    """exp(g) below the normal range, the other half as far above 1."""
    g, u = torch.linspace(-80, -100, 128), torch.full((128,), 2.0**110)
    q, s = quant_device.per_1x128_f8_quant(torch.cat([g, u]).unsqueeze(0).cuda(), gated=True)
    y = g.double() * torch.exp(g.double()) * 2.0**110
    want = y.abs().max() / 448
    assert (s.double().cpu() - want).abs() <= 11.5 * U * want
    # (silu itself is a subnormal number for g below -82, off by half of 2^-149)
    slack = 2.0**-149 * 2.0**110 / want
    v = y / want
    assert ((q.double().cpu() - v).abs() <= torch.clamp(2.0**-4 * v.abs(), min=2.0**-10) * (1 + 2.0**-4) + 24 * U * v.abs() + slack).all()


def test_no_rows_and_refusals():
    q, s = quant_device.per_1x128_f8_quant(torch.empty(0, 300, dtype=torch.bfloat16, device="cuda"))
    assert q.shape == (0, 300) and s.shape == (3, 0)
    x = torch.zeros(4, 256, dtype=torch.bfloat16, device="cuda")
    f = quant_device.per_1x128_f8_quant
    out = lambda q=(4, 256), s=(2, 4), qd=torch.uint8, sd=torch.float32, dev="cuda": (torch.zeros(q, dtype=qd, device=dev), torch.zeros(s, dtype=sd, device=dev))
    for stream in (None, torch.cuda.current_stream()):
        for bad in (out(q=(4, 255)), out(s=(4, 2)), out(s=(1, 4)), out(qd=torch.int16), out(sd=torch.float16), out(dev="cpu"), (out()[0].t().contiguous().t(), out()[1]), (out()[0], out(s=(4, 2))[1].t())):
            with pytest.raises(ValueError):
                f(x, stream=stream, out=bad)
        with pytest.raises(TypeError):
            f(x, stream=stream, out=(None, None))
        with pytest.raises(ValueError, match="dense rows"):
            f(x.t(), stream=stream, out=out(q=(256, 4), s=(1, 256)))
        with pytest.raises(ValueError, match="dense rows"):
            f(x[:1].expand(4, 256), stream=stream, out=out())
        with pytest.raises(ValueError, match="even"):
            f(x[:, :255], True, stream=stream, out=out())
        with pytest.raises(ValueError):
            f(x[0], stream=stream, out=out())


def test_replayed():
    x = _x(33, 1000, torch.bfloat16, 2).cuda()
    out = torch.empty(33, 1000, dtype=FP8, device="cuda"), torch.empty(8, 33, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        quant_device.per_1x128_f8_quant(x, stream=side, out=out)
    for k in range(3):
        x.copy_(_x(33, 1000, torch.bfloat16, 10 + k))
        graph.replay()
        torch.cuda.synchronize()
        _check_plain(x, *out)


@pytest.mark.parametrize("gated", [False, True])
def test_rows_past_four_gib(gated):
    """q of more than 2^32 bytes, x of two and four times as many, in more than one launch: rows at the front, about the borders and at the end."""
    m, dim = 4200007, 1032
    x = _x(65521, dim * (2 if gated else 1), torch.bfloat16, 4).cuda().repeat(-(-m // 65521), 1)[:m]
    print(f"quant {m}x{dim} gated={gated}", flush=True)
    q, s = quant_device.per_1x128_f8_quant(x, gated=gated)
    torch.cuda.synchronize()
    rows = torch.tensor([r for at in (0, 2**31 // dim, 2**32 // dim, 2**32 // x.shape[1] // 2, 4 * ((1 << 23) // 3), m) for r in range(max(at - 9, 0), min(at + 9, m))], device="cuda")
    (_check_gated if gated else _check_plain)(x[rows], q.view(torch.uint8)[rows].view(FP8), s[:, rows])
