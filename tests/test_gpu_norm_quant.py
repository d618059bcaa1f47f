"""GPU tests of the norm with quantised rows against its definition in 64 bits.

Tolerances, in units of u = 2^-24 (half a step of fp32): all squares are positive, so their sum is off by at most as many u as a chain of additions is long.  A thread adds at
most dim / 64 squares one after the other (one wavefront a row; fewer with more threads), then come 6 exchanges and up to 16 partial sums; the mean, the root, the reciprocal and
two products add at most 8.  The root halves what was before it.  So y and the scale are within (dim / 64 + 40) u relatively, and every output within that and its own rounding.
"""

import numpy
import pytest
import torch

from flydsl_amd import quant_device

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn
QMAX = {FP8: 448.0, torch.int8: 127.0}
STEP = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}  # half a step, relative


def _inputs(rows, dim, dt, residual, seed, wt=None):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, dim, generator=g) * (1 + 30 * (torch.rand(dim, generator=g) < 0.01))).to(dt)
    w = (1 + 0.3 * torch.randn(dim, generator=g)).to(wt or dt)
    r = (3 * torch.randn(rows, dim, generator=g)).to(dt) if residual else None
    return x.cuda(), w.cuda(), None if r is None else r.cuda()


def _exact(x, w, r, eps, qd):
    h = x if r is None else (x.float() + r.float()).to(x.dtype)
    d = h.double()
    y = d * w.double() / (d.square().mean(-1, keepdim=True) + eps).sqrt()
    s = y.abs().amax(-1, keepdim=True) / QMAX[qd] if qd is not None else None
    if s is not None:
        s = torch.where(s == 0, torch.ones_like(s), s)
    return h, y, s


def _check(x, w, r, eps, qd, q, scale, h_out, normed):
    h, y, s = _exact(x, w, r, eps, qd)
    tol = (x.shape[1] / 64 + 40) * 2.0**-24
    if r is not None:
        assert torch.equal(h_out, h)
    if normed is not None:
        # (below the normal range a rounding is off by half a smallest step)
        tiny = torch.finfo(x.dtype).tiny * 2 * STEP[x.dtype]
        assert ((normed.double() - y).abs() <= (STEP[x.dtype] * (1 + tol) + tol) * y.abs() + tiny).all()
    if qd is None:
        return
    assert scale.shape == (x.shape[0], 1) and scale.dtype == torch.float32
    assert ((scale.double() - s).abs() <= tol * s).all()
    want = y / s
    off = (q.to(torch.float64) - want).abs()
    assert (q.to(torch.float64).abs().amax(-1) == torch.where(y.abs().amax(-1) == 0, 0.0, QMAX[qd])).all()  # the maximum of a row is the largest value
    slack = 4 * 2.0**-24 * want.abs()  # the norm cancels in y / s: a product with the weight, one with the largest value, the quotient
    if qd == FP8:
        assert (off <= torch.clamp(2.0**-4 * (want.abs() + slack), min=2.0**-10) + slack).all()
    else:  # towards zero
        assert (off < 1 + slack).all() and (q.double().abs() <= want.abs() + slack).all()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,dim", [(1, 1), (3, 7), (1, 64), (2, 2051), (67, 4096), (2100, 512), (2049, 1543), (5, 8192), (3, 8200), (2, 33003), (1, 70000)])
def test_against_the_definition(rows, dim, dt):
    for residual, qd in ((True, FP8), (False, torch.int8)):
        x, w, r = _inputs(rows, dim, dt, residual, seed=rows * 7 + dim)
        keep = None if r is None else r.clone()
        normed = torch.empty_like(x)
        q, s = quant_device.rmsnorm_quant(x, w, 1e-5, residual=r, quant_dtype=qd, normed=normed)
        _check(x, w, keep, 1e-5, qd, q, s, r, normed)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_weight_in_fp32_and_norm_alone(dt):
    x, w, r = _inputs(33, 1000, dt, True, seed=4, wt=torch.float32)
    h = torch.empty_like(x)
    y = quant_device.rmsnorm_quant(x, w, 1e-6, residual=r, residual_out=h, quant_dtype=None)
    _check(x, w, r, 1e-6, None, None, None, h, y)
    q, s = quant_device.rmsnorm_quant(x, w, 1e-6, quant_dtype=torch.int8)
    _check(x, w, None, 1e-6, torch.int8, q, s, None, None)


@pytest.mark.parametrize("qd", [FP8, torch.int8])
@pytest.mark.parametrize("dim", [5, 256, 2056, 9000, 40008])
def test_special_rows_as_the_quantiser_has_them(dim, qd):
    """Rows of zeros, NaN and infinities, tiny and huge ones, against the quantiser on the fp32 rows that the norm wrote: the same bytes, and in the ordinary rows, whose
    values are divided before their rounding here, at most one step beside it."""
    x, w, _ = _inputs(40, dim, torch.float32, False, seed=dim)
    x[1] = 0
    x[2, dim // 2] = float("nan")
    x[3, dim - 1] = float("inf")
    x[4] *= 1e-30
    x[5] *= 1e15
    x[6, 0] = -float("inf")
    w[dim // 3] = 0
    normed = torch.empty_like(x)
    for eps in (1e-6, 0.0):
        q, s = quant_device.rmsnorm_quant(x, w, eps, quant_dtype=qd, normed=normed)
        pad = torch.nn.functional.pad(normed, (0, -dim % 8))  # (the quantiser wants multiples of 8; zeros change nothing)
        q2, s2 = quant_device.pertoken_quant(pad, quant_dtype=qd)
        assert torch.equal(s, s2)
        q2 = q2[:, :dim]
        odd = [1, 2, 3, 4, 6]
        assert torch.equal(q.view(torch.uint8)[odd], q2.view(torch.uint8)[odd])
        a, b = q.float(), q2.float()
        assert ((a - b).abs() <= torch.clamp(2.0**-3 * b.abs(), min=2.0**-9) if qd == FP8 else (a - b).abs() <= 1).all()
    bad = torch.ones(dim, device="cuda")
    bad[0] = float("inf")  # an infinite weight: that column saturates, the others stay
    q, s = quant_device.rmsnorm_quant(x, bad, 1e-6, quant_dtype=qd, normed=normed)
    q2, s2 = quant_device.pertoken_quant(torch.nn.functional.pad(normed, (0, -dim % 8)), quant_dtype=qd)
    assert torch.equal(s, s2) and torch.equal(q.view(torch.uint8), q2.view(torch.uint8)[:, :dim])
    assert (q[:3, 0].float() == 0).sum() == 2 and q[0, 0].float().abs() == QMAX[qd]


def test_slices_of_wider_tensors_and_rows_in_place():
    rows, dim = 50, 1027
    x, w, r = _inputs(rows, dim, torch.bfloat16, True, seed=1)
    wide = {k: torch.full((rows, dim + 29), 7.0, dtype=torch.bfloat16, device="cuda") for k in ("x", "r", "h", "n")}
    wide["x"][:, 3 : 3 + dim], wide["r"][:, 11 : 11 + dim] = x, r
    v = {k: t[:, o : o + dim] for (k, t), o in zip(wide.items(), (3, 11, 5, 0))}
    q, s = quant_device.rmsnorm_quant(v["x"], w, residual=v["r"], residual_out=v["h"], normed=v["n"])
    _check(x, w, r, 1e-6, FP8, q, s, v["h"], v["n"])
    assert torch.equal(v["x"], x) and torch.equal(v["r"], r)
    for k, o in zip(wide, (3, 11, 5, 0)):  # nothing beside the slices
        assert (wide[k][:, :o] == 7).all() and (wide[k][:, o + dim :] == 7).all()
    # the sum in place of the residual or of x, the norm in place of x: also where a row is longer than what the registers hold
    for d in (dim, 41000):
        x, w, r = _inputs(4, d, torch.float16, True, seed=2)
        a, b = x.clone(), r.clone()
        q, s = quant_device.rmsnorm_quant(a, w, residual=b, normed=a)
        _check(x, w, r, 1e-6, FP8, q, s, b, a)
        a = x.clone()
        q, s = quant_device.rmsnorm_quant(a, w, residual=r, residual_out=a)
        _check(x, w, r, 1e-6, FP8, q, s, a, None)
        a = x.clone()
        q, s = quant_device.rmsnorm_quant(a, w, normed=a)
        _check(x, w, None, 1e-6, FP8, q, s, None, a)


def test_rows_far_apart():
    """Offsets of rows beyond 32 bits."""
    far = torch.empty(3 * 1_300_000_000, dtype=torch.bfloat16, device="cuda").as_strided((3, 264), (1_300_000_000, 1))
    x, w, _ = _inputs(3, 264, torch.bfloat16, False, seed=3)
    far.copy_(x)
    normed = torch.empty_like(x)
    q, s = quant_device.rmsnorm_quant(far, w, normed=normed)
    _check(x, w, None, 1e-6, FP8, q, s, None, normed)


def test_no_rows_and_reused_outputs():
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    q, s = quant_device.rmsnorm_quant(torch.empty(0, 64, dtype=torch.bfloat16, device="cuda"), w)
    assert q.shape == (0, 64) and s.shape == (0, 1)
    x, w, _ = _inputs(9, 64, torch.bfloat16, False, seed=5)
    out = torch.empty(9, 64, dtype=torch.uint8, device="cuda"), torch.empty(9, device="cuda")
    q, s = quant_device.rmsnorm_quant(x, w, stream=torch.cuda.current_stream(), out=out)
    assert q.data_ptr() == out[0].data_ptr() and s.data_ptr() == out[1].data_ptr() and q.dtype == FP8
    _check(x, w, None, 1e-6, FP8, q, s, None, None)
    q, s = quant_device.rmsnorm_quant(x, torch.nn.Parameter(w), stream=torch.cuda.current_stream(), out=out)  # a module's weight
    _check(x, w, None, 1e-6, FP8, q, s, None, None)


def test_graph_replays_and_another_stream():
    x, w, r = _inputs(20, 4096, torch.bfloat16, True, seed=6)
    out = torch.empty(20, 4096, dtype=FP8, device="cuda"), torch.empty(20, 1, device="cuda")
    h = torch.empty_like(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        quant_device.rmsnorm_quant(x, w, residual=r, residual_out=h, stream=side, out=out)
    for k in range(3):
        x.copy_(torch.roll(x, 1, 0) * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        _check(x, w, r, 1e-6, FP8, out[0], out[1], h, None)
        again = quant_device.rmsnorm_quant(x, w, residual=r, residual_out=torch.empty_like(x))  # eager work between the replays
        assert torch.equal(again[0].view(torch.uint8), out[0].view(torch.uint8)) and torch.equal(again[1], out[1])


def test_refusals():
    x, w, r = _inputs(4, 64, torch.bfloat16, True, seed=7)
    out = torch.empty(4, 64, dtype=torch.uint8, device="cuda"), torch.empty(4, device="cuda")
    f = quant_device.rmsnorm_quant
    for stream in (None, torch.cuda.current_stream()):
        with pytest.raises(ValueError, match="residual must be"):
            f(x, w, residual=r[:3], out=out, stream=stream)
        with pytest.raises(ValueError, match="residual must be"):
            f(x, w, residual=r.half(), out=out, stream=stream)
        with pytest.raises(ValueError, match="normed must be"):
            f(x, w, normed=torch.empty(4, 65, dtype=torch.bfloat16, device="cuda"), out=out, stream=stream)
        with pytest.raises(ValueError, match="out must be"):
            f(x, w, out=(out[0][:3], out[1]), stream=stream)
        with pytest.raises(ValueError, match="out must be"):
            f(x, w, out=(out[0], out[1][:3]), stream=stream)
        with pytest.raises(ValueError, match="weight must"):
            f(x, w[:32], out=out, stream=stream)
        with pytest.raises(ValueError, match="weight must"):
            f(x, w.half(), out=out, stream=stream)
        with pytest.raises(ValueError, match="without a residual"):
            f(x, w, residual_out=r, out=out, stream=stream)
    with pytest.raises(ValueError, match="dense rows"):
        f(x.t().contiguous().t(), w)
    with pytest.raises(ValueError, match="dense rows"):
        f(x[:1].expand(4, 64), w)
    with pytest.raises(ValueError, match="eps"):
        f(x, w, -1.0)
    with pytest.raises(ValueError, match="quant_dtype=None"):
        f(x, w, quant_dtype=None, out=out)


@pytest.mark.parametrize("qd", [torch.int8, FP8])
def test_scale_near_the_smallest_number(qd):
    """Rows whose scale has two or three bits: it is off by up to u / 2 (u = 2^-149), the outputs stay within the largest value all the same.  y is off by 2 u (a product rounded to u / 2, times
    at most 1.25, and rounded again); an output held back at the largest value by as much times u / 2; then the output's own step."""
    g = torch.Generator().manual_seed(11)
    x, w = torch.randn(64, 256, generator=g), torch.full((256,), 2.0**-140)
    assert w[0] > 0
    y = x.double() * w.double() / x.double().square().mean(-1, keepdim=True).sqrt()
    assert (x.square().mean(-1).sqrt() - 1).abs().max() < 0.25
    q, s = quant_device.rmsnorm_quant(x.cuda(), w.cuda(), 0.0, quant_dtype=qd)
    q, s = q.cpu().double(), s.cpu().double()
    u = 2.0**-149
    assert ((s - y.abs().amax(-1, keepdim=True) / QMAX[qd]).abs() <= u).all()
    assert (q.abs() <= QMAX[qd]).all()
    step = s if qd == torch.int8 else torch.maximum(y.abs() / 16, s * 2.0**-10)
    assert ((q * s - y).abs() <= 1.1 * step + (QMAX[qd] / 2 + 3) * u).all()


def test_more_rows_than_a_launch_holds():
    rows, at = (1 << 22) + 5, slice((1 << 22) - 3, None)  # 512 threads a row at most
    x = torch.randn(rows, 8, dtype=torch.bfloat16, device="cuda")
    r = torch.randn(rows, 8, dtype=torch.bfloat16, device="cuda")
    w = torch.rand(8, device="cuda") + 0.5
    q, s = torch.zeros(rows, 8, dtype=torch.int8, device="cuda"), torch.full((rows, 1), -1.0, device="cuda")
    x0, r0, h0, n0 = x[at].clone(), r[at].clone(), torch.empty(8, 8, dtype=x.dtype, device="cuda"), torch.empty(8, 8, dtype=x.dtype, device="cuda")
    print(f"norm rows={rows} dim=8", flush=True)
    quant_device.rmsnorm_quant(x, w, residual=r, normed=x, quant_dtype=torch.int8, out=(q, s))
    q0, s0 = quant_device.rmsnorm_quant(x0, w, residual=r0, residual_out=h0, normed=n0, quant_dtype=torch.int8)
    assert torch.equal(q[at], q0) and torch.equal(s[at], s0) and torch.equal(r[at], h0) and torch.equal(x[at], n0)
    _check(x0, w, r0, 1e-6, torch.int8, q0, s0, h0, n0)
    assert (s > 0).all() and (torch.maximum(q.amax(-1), -q.amin(-1)) == 127).all()


def test_sizes_refused():
    out = torch.empty(4, 8, dtype=torch.uint8, device="cuda"), torch.empty(4, device="cuda")
    one = torch.ones(1, 1, dtype=torch.bfloat16, device="cuda")
    for stream in (None, torch.cuda.current_stream()):
        with pytest.raises(ValueError, match="2\\^31"):
            quant_device.rmsnorm_quant(one.expand(1 << 31, 1), one[0], out=out, stream=stream)
        with pytest.raises(ValueError, match="2\\^31"):
            quant_device.rmsnorm_quant(one.expand(1, (1 << 24) + 1), one.expand(1, (1 << 24) + 1), out=out, stream=stream)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("vecs", [1, 64, 65, 256, 513, 4100])
def test_every_end_of_a_row(vecs, dt):
    """Ends of one to seven elements, the residual in place, in launches of few and of many rows; what stands between the rows stays as it is."""
    for end in range(1, 8):
        dim = vecs * 8 + end
        for rows in (3, 2300) if dim < 2048 else (3,):
            x, w, r = _inputs(rows, dim, dt, True, seed=dim)
            wide = torch.full((rows, dim + 11), -5.0, dtype=dt, device="cuda")
            h = wide[:, :dim]
            h.copy_(r)
            y = torch.full_like(wide, -6.0)
            out = torch.empty(rows, dim, dtype=torch.uint8, device="cuda"), torch.empty(rows, 1, device="cuda")
            q, s = quant_device.rmsnorm_quant(x, w, 1e-6, residual=h, normed=y[:, :dim], out=out, stream=torch.cuda.current_stream())
            _check(x, w, r, 1e-6, FP8, q, s, h, y[:, :dim])
            assert (wide[:, dim:] == -5).all() and (y[:, dim:] == -6).all()


def test_scale_that_is_rounded_to_zero():
    """A row whose values are below the smallest scale has scale 1, and codes of what the values are then, none, however far from zero h is: 2^-142 / 448 is below half of the smallest
    number, 2^-149.  2^-142 / 127 = 2^-148.99 is rounded to it, and 2^-142 / 2^-149 = 128 is held at 127."""
    h = torch.full((3, 8), 2.0**62, device="cuda")
    h[:, 1::2] *= -1
    h[1] = 0
    w = torch.full((8,), 2.0**-142, device="cuda")
    for qd in (FP8, torch.int8):
        normed = torch.empty_like(h)
        q, s = quant_device.rmsnorm_quant(h, w, quant_dtype=qd, normed=normed)
        assert torch.equal(normed, h * 2.0**-62 * w)
        if qd == FP8:
            assert (s == 1).all() and (q.float() == 0).all()
        else:
            assert s.view(-1).tolist() == [2.0**-149, 1.0, 2.0**-149] and torch.equal(q.float(), h * (127 * 2.0**-62))


def _far(rows, dim, dt, residual, seed, exponents):
    x, w, r = _inputs(rows, dim, dt, residual, seed)
    by = torch.tensor([2.0**e for e in exponents], dtype=torch.float64, device="cuda").unsqueeze(1)
    return (x.double() * by).to(dt), w, None if r is None else (r.double() * by).to(dt)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim", [1, 7, 256, 4096, 5003, 9000, 12296, 40008, 40011])
def test_rows_whose_squares_leave_the_range(dim, dt):
    """h from 2^-120 to 2^118 beside ordinary rows: the squares, or their sum, are beyond fp32, the norm is not.  (With an eps, rows far below its root are h w / sqrt(eps), exact as far
    as the products are normal numbers.)"""
    for eps, exponents in ((0.0, (0, 59, 64, 90, 118, -50, -60, -64, -90, -120, 0, 30)), (1e-6, (0, 59, 64, 90, 118, -20, -50, -60, -70, 1, 0, 30))):
        for residual, qd in ((True, FP8), (False, torch.int8)):
            x, w, r = _far(12, dim, dt, residual, dim, exponents)
            keep, normed = None if r is None else r.clone(), torch.empty_like(x)
            q, s = quant_device.rmsnorm_quant(x, w, eps, residual=r, quant_dtype=qd, normed=normed)
            _check(x, w, keep, eps, qd, q, s, r, normed)


@pytest.mark.parametrize("dim", [2048, 41003])
def test_rows_whose_squares_leave_the_range_in_place(dim):
    exponents = (64, 0, -70, 110)
    for residual in (False, True):
        x, w, r = _far(4, dim, torch.bfloat16, residual, 3, exponents)
        a = x.clone()
        q, s = quant_device.rmsnorm_quant(a, w, 0.0, residual=None if r is None else r.clone(), normed=a)
        _check(x, w, None if r is None else r, 0.0, FP8, q, s, (x.float() + r.float()).to(x.dtype) if residual else None, a)
    a = x.clone()
    q, s = quant_device.rmsnorm_quant(a, w, 0.0, residual=r, residual_out=a)
    _check(x, w, r, 0.0, FP8, q, s, a, None)


def test_products_with_the_weight_that_leave_the_range():
    """h and y are numbers of fp32, h w is beyond the largest or below the smallest."""
    x, _, _ = _inputs(6, 300, torch.float32, False, 5)
    for e, f in ((55, 80), (30, 100), (-45, -60)):
        h, w = x * 2.0**e, (torch.rand(300, generator=torch.Generator().manual_seed(1)) + 0.5).cuda() * 2.0**f
        normed = torch.empty_like(h)
        q, s = quant_device.rmsnorm_quant(h, w, 0.0, normed=normed)
        _check(h, w, None, 0.0, FP8, q, s, None, normed)
    # a scale below 2^-80: y is divided, with two roundings of y, three of the scale and one of the quotient
    h, w = x * 2.0**-45, torch.full((300,), 2.0**-105, device="cuda")
    q, s = quant_device.rmsnorm_quant(h, w, 0.0)
    _, y, want = _exact(h, w, None, 0.0, FP8)
    assert ((s.double() - want).abs() <= (300 / 64 + 40) * 2.0**-24 * want).all()
    slack = 6 * 2.0**-24 * (y / want).abs()
    assert ((q.double() - y / want).abs() <= torch.clamp(2.0**-4 * ((y / want).abs() + slack), min=2.0**-10) + slack).all()


def test_eps_that_is_no_python_number():
    """A tensor or an array is read at every call."""
    x, w, _ = _inputs(3, 256, torch.bfloat16, False, 6)
    out = torch.empty(3, 256, dtype=FP8, device="cuda"), torch.empty(3, 1, device="cuda")
    for eps in (torch.tensor(1e-6), numpy.array(1e-6)):
        for value in (1e-6, 4.0):
            eps[...] = value
            q, s = quant_device.rmsnorm_quant(x, w, eps, stream=torch.cuda.current_stream(), out=out)
            _check(x, w, None, value, FP8, q, s, None, None)


def test_outputs_are_allocated_for_the_stream_of_the_launch():
    x, w, _ = _inputs(2048, 2048, torch.bfloat16, False, 8)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    made = {0: torch.cuda.default_stream().cuda_stream, side: side.cuda_stream, side.cuda_stream: side.cuda_stream, None: torch.cuda.current_stream().cuda_stream}
    for stream, handle in made.items():
        q, s = quant_device.rmsnorm_quant(x, w, stream=stream)
        y = quant_device.rmsnorm_quant(x, w, quant_dtype=None, stream=stream)
        torch.cuda.synchronize()
        _check(x, w, None, 1e-6, FP8, q, s, None, y)
        segments = torch.cuda.memory_snapshot()
        for t in (q, s, y):
            at = [g["stream"] for g in segments if g["address"] <= t.data_ptr() < g["address"] + g["total_size"]]
            assert at == [handle]


@pytest.mark.parametrize("dt,wt", [(torch.float32, None), (torch.bfloat16, None), (torch.bfloat16, torch.float32), (torch.float16, None), (torch.float16, torch.float32)])
@pytest.mark.parametrize("rows,dim", [(3, 12296), (2, 16384), (1100, 4099), (1030, 9001), (3, 16392), (2, 20001), (2, 32768), (4, 9001), (3, 12281)])
def test_long_rows_of_every_build(rows, dim, dt, wt):
    """Four vectors a thread on up to 512 threads (4097 elements and more, by rows and ends), on 576 to 1024, and two on up to 768 with a row's end."""
    for residual, qd in ((True, FP8), (False, torch.int8)):
        x, w, r = _inputs(rows, dim, dt, residual, seed=dim, wt=wt)
        wide = torch.full((rows, dim + 3), 7.0, dtype=dt, device="cuda")  # (rows off 16 bytes, and something behind them)
        v = wide[:, :dim]
        v.copy_(x)
        keep, out = None if r is None else r.clone(), (torch.empty(rows, dim, dtype=qd, device="cuda"), torch.empty(rows, 1, device="cuda"))
        print(f"norm rows={rows} dim={dim} {dt} {wt}", flush=True)
        q, s = quant_device.rmsnorm_quant(v, w, 1e-6, residual=r, quant_dtype=qd, normed=v, stream=torch.cuda.current_stream(), out=out)
        _check(x, w, keep, 1e-6, qd, q, s, r, v)
        assert (wide[:, dim:] == 7).all()


@pytest.mark.parametrize("dim", [515, 40011])
def test_residual_that_is_x(dim):
    x, w, _ = _inputs(5, dim, torch.bfloat16, False, seed=9)
    a, normed = x.clone(), torch.empty_like(x)
    q, s = quant_device.rmsnorm_quant(a, w, residual=a, normed=normed)
    _check(x, w, x, 1e-6, FP8, q, s, a, normed)
