"""GPU tests of the block-scaled products, dense and by group, against their definition in 64 bits.

Exact inputs: operands are whole numbers up to 4, scales powers of two from 2^-3 on, so every partial sum is a multiple of 2^-6 below 16 K, exact in fp32 (K < 2^14) whatever its order, and the output is
the definition rounded once.  Random inputs: 128 additions inside a block, the product of the scales, and an addition for every block, off by 2^-23 of the magnitudes' sum each at most, then the
rounding to 16 bits.
"""

import pytest
import torch

from flydsl_amd import layout, quant
from kernels.gemm.blockscale_gemm import compile_blockscale_gemm, compile_grouped_blockscale_gemm

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
HALF = {"bf16": 2.0**-8, "fp16": 2.0**-11}
GUARD = -77.0
AUTO, STREAM = (0, 0), (1, 0)
WHOLE = [(16, 0), (32, 0), (64, 0), (128, 0), (128, 128)]  # rows of a tile (and 128 columns in place of 256), K in one piece
SLICED = [(16, 16), (16, 32), (32, 32), (32, 64), (64, 64)]  # rows and columns of a tile, K in slices


def _operands(rows, n, k, groups, seed, exact=True):
    g = torch.Generator().manual_seed(seed)
    kb, nb = -(-k // 128), -(-n // 128)
    if exact:
        a, w = (torch.randint(-4, 5, s, generator=g).float().to(FP8) for s in ((rows, k), (groups, n, k)))
        return a, w, torch.exp2(-torch.randint(0, 4, (kb, rows), generator=g).float()), torch.exp2(-torch.randint(0, 4, (groups, nb, kb), generator=g).float())
    a, sa = quant.per_1x128_f8_quant(torch.randn(rows, k, generator=g))
    w, sb = quant.per_128x128_f8_quant(0.05 * torch.randn(groups, n, k, generator=g))
    return a, w, sa, sb


def _shuffled(w):
    return layout.shuffle_weight(w.view(torch.int8)).view(FP8).contiguous()


def _product(a, w, sa, sb):
    """One group's rows: values and the sum of their terms' magnitudes."""
    n, k = w.shape
    wide = lambda s, times, size: s.double().repeat_interleave(128, times)[..., :size]
    av = a.double() * wide(sa.t(), 1, k)
    wv = w.double() * sb.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    return av @ wv.t(), av.abs() @ wv.abs().t()


def _want(a, w, sa, sb, offsets):
    rows, vals, mags = [], [], []
    for e in range(len(offsets) - 1):
        r = slice(offsets[e], offsets[e + 1])
        if r.stop > r.start:
            v, m = _product(a[r], w[e], sa[:, r], sb[e])
            vals.append(v)
            mags.append(m)
            rows += range(r.start, r.stop)
    n = w.shape[1]
    return rows, torch.cat(vals or [torch.empty(0, n, dtype=torch.float64)]), torch.cat(mags or [torch.empty(0, n, dtype=torch.float64)])


def _run(a, w, sa, sb, offsets, out, tile=AUTO, strided=False, same=True):
    """offsets None: the dense product of the one weight."""
    groups, n, k = w.shape
    m = a.shape[0]
    fn = compile_blockscale_gemm(N=n, K=k, out_dtype=out) if offsets is None else compile_grouped_blockscale_gemm(N=n, K=k, groups=groups, out_dtype=out)
    c = torch.full((m + 3, n), GUARD, dtype=DT[out], device="cuda")
    scales = sa.cuda()
    if strided:
        wide = torch.full((sa.shape[0], m + 5), 3e30, device="cuda")
        wide[:, 1 : 1 + m] = scales
        scales = wide[:, 1 : 1 + m]
    rest = (m,) if offsets is None else (torch.tensor(offsets, dtype=torch.int32).cuda(), m)
    args = a.cuda(), _shuffled(w).cuda(), scales, sb.cuda(), *rest
    print(f"blockscale M={m} N={n} K={k} groups={groups if offsets is not None else '-'} {out} tile {tile} strided {strided}", flush=True)
    fn.tile = tile
    try:
        fn(c, *args, torch.cuda.current_stream())
        again = torch.full_like(c, GUARD)
        fn(again, *args)
        torch.cuda.synchronize()
    finally:
        fn.tile = AUTO
    assert not same or torch.equal(c.view(torch.int16), again.view(torch.int16))
    return c.cpu()


def _check_exact(c, a, w, sa, sb, offsets, out):
    rows, vals, _ = _want(a, w, sa, sb, offsets or [0, a.shape[0]])
    assert torch.equal(c[rows], vals.float().to(DT[out]))
    rest = torch.ones(c.shape[0], dtype=torch.bool)
    rest[rows] = False
    assert (c[rest] == GUARD).all()


def _check_random(c, a, w, sa, sb, offsets, out):
    rows, vals, mags = _want(a, w, sa, sb, offsets or [0, a.shape[0]])
    k = a.shape[1]
    assert ((c[rows].double() - vals).abs() <= HALF[out] * vals.abs() + (128 + -(-k // 128) + 2) * 2.0**-23 * (1 + HALF[out]) * mags + 2.0**-25).all()


@pytest.mark.parametrize("tile", [AUTO, STREAM] + WHOLE + SLICED)
@pytest.mark.parametrize("m,n,k", [(1, 16, 64), (1, 272, 192), (5, 128, 128), (17, 400, 576), (33, 256, 1088), (64, 144, 2048), (129, 528, 320), (300, 640, 1152), (257, 272, 64), (16, 16, 8192)])
def test_dense_exact(m, n, k, tile):
    a, w, sa, sb = _operands(m, n, k, 1, m + n + k)
    for out in ("bf16", "fp16"):
        _check_exact(_run(a, w, sa, sb, None, out, tile), a, w, sa, sb, None, out)


@pytest.mark.parametrize("tile", [AUTO, STREAM] + WHOLE + SLICED)
def test_scales_of_a_wider_tensor(tile):
    a, w, sa, sb = _operands(150, 272, 448, 1, 3)
    _check_exact(_run(a, w, sa, sb, None, "bf16", tile, strided=True), a, w, sa, sb, None, "bf16")


@pytest.mark.parametrize("tile", [(128, 0), (128, 128)])
@pytest.mark.parametrize("steps", range(1, 15))
def test_every_length_of_the_large_tile(steps, tile):
    """1 to 14 steps of K, with half a step at the end and without: the loop's builds with and without checks, and its ends."""
    for k in (steps * 128 - 64, steps * 128):
        a, w, sa, sb = _operands(140, 288, k, 1, k)
        _check_exact(_run(a, w, sa, sb, None, "bf16", tile), a, w, sa, sb, None, "bf16")


@pytest.mark.parametrize("tile", SLICED)
@pytest.mark.parametrize("steps", [1, 2, 7, 8, 9, 15, 16, 17, 23, 24, 25, 31, 32, 33, 40, 41, 48, 49, 57])
def test_every_length_of_the_slices(steps, tile):
    """Up to eight steps a slice, with some slices a step shorter: the loop, its ends, and slices without a step."""
    for k in (steps * 128 - 64, steps * 128):
        a, w, sa, sb = _operands(70, 144, k, 1, k)
        _check_exact(_run(a, w, sa, sb, None, "bf16", tile), a, w, sa, sb, None, "bf16")


SIZES = {
    "one group": [40],
    "one row each": [1] * 9,
    "empty ones": [0, 0, 5, 0, 17, 1, 0, 33, 0],
    "ragged": [3, 130, 64, 16, 15, 17, 128, 129, 2, 0, 250],
    "many": [(7 * i) % 23 if i % 5 else 0 for i in range(150)],
    "nothing": [0, 0, 0],
}


def _offsets(sizes, first=0):
    o = [first]
    for s in sizes:
        o.append(o[-1] + s)
    return o


@pytest.mark.parametrize("out", ["bf16", "fp16"])
@pytest.mark.parametrize("tile", [AUTO] + WHOLE + SLICED)
@pytest.mark.parametrize("sizes", SIZES)
def test_groups_exact(sizes, tile, out):
    s = SIZES[sizes]
    n, k = 272, 320  # half a step at the end, columns that end inside every tile and block
    offsets = _offsets(s, first=2)
    a, w, sa, sb = _operands(offsets[-1] + 5, n, k, len(s), len(s))
    _check_exact(_run(a, w, sa, sb, offsets, out, tile, strided=tile == AUTO), a, w, sa, sb, offsets, out)


@pytest.mark.parametrize("n,k", [(16, 64), (1040, 4096), (512, 1600)])
@pytest.mark.parametrize("sizes", [[1], [20, 0, 31], [300, 1, 700]])
def test_groups_widths_and_lengths(sizes, n, k):
    offsets = _offsets(sizes)
    a, w, sa, sb = _operands(offsets[-1], n, k, len(sizes), n + k)
    _check_exact(_run(a, w, sa, sb, offsets, "bf16"), a, w, sa, sb, offsets, "bf16")


@pytest.mark.parametrize("out", ["bf16", "fp16"])
def test_random_values_and_the_same_bits_on_every_tile(out):
    offsets = _offsets(SIZES["ragged"])
    a, w, sa, sb = _operands(offsets[-1], 400, 1088, len(offsets) - 1, 3, exact=False)
    for tiles in WHOLE, SLICED:
        first = None
        for tile in tiles:
            c = _run(a, w, sa, sb, offsets, out, tile)
            _check_random(c, a, w, sa, sb, offsets, out)
            first = c if first is None else first
            assert torch.equal(c.view(torch.int16), first.view(torch.int16))


@pytest.mark.parametrize("m,n,k", [(1, 6144, 4096), (16, 2048, 7168), (100, 1536, 2240), (333, 2832, 2240), (700, 1024, 5120)])
def test_dense_random(m, n, k):
    a, w, sa, sb = _operands(m, n, k, 1, m, exact=False)
    _check_random(_run(a, w, sa, sb, None, "bf16"), a, w, sa, sb, None, "bf16")


def test_a_group_alone_is_the_dense_product():
    a, w, sa, sb = _operands(300, 512, 1024, 1, 9, exact=False)
    for tile in WHOLE + SLICED:
        assert torch.equal(_run(a, w, sa, sb, [0, 300], "bf16", tile).view(torch.int16), _run(a, w, sa, sb, None, "bf16", tile).view(torch.int16))


def test_scales_of_one_are_the_plain_product():
    """Against the fp8 product of the same operands with one scale a row: the same values where both are exact."""
    from kernels.gemm.preshuffle_gemm import compile_preshuffle_gemm

    a, w, sa, sb = _operands(200, 512, 1024, 1, 4)
    c = _run(a, w, torch.ones_like(sa), torch.ones_like(sb), None, "bf16")
    dense = torch.empty(200, 512, dtype=torch.bfloat16, device="cuda")
    compile_preshuffle_gemm(N=512, K=1024, tile_m=128, tile_n=256, tile_k=128, in_dtype="fp8")(
        dense, a.cuda(), _shuffled(w[0]).cuda(), torch.ones(200, device="cuda"), torch.ones(512, device="cuda"), torch.empty(0, dtype=torch.bfloat16, device="cuda"), 200, 512, torch.cuda.current_stream())
    assert torch.equal(c[:200], dense.cpu())


@pytest.mark.parametrize("tile", [AUTO, STREAM] + WHOLE + SLICED)
def test_special_values_stay_in_their_rows_and_columns(tile):
    a, w, sa, sb = _operands(70, 288, 640, 1, 8)
    clean = _run(a, w, sa, sb, None, "bf16", tile)[:70]
    a2, w2, sa2, sb2 = a.clone(), w.clone(), sa.clone(), sb.clone()
    a2.view(torch.uint8)[3, 200] = 0x7F  # NaN
    w2.view(torch.uint8)[0, 17, 5] = 0xFF
    sa2[1, 9], sa2[4, 33] = float("inf"), float("nan")
    sb2[0, 2, 0] = float("nan")
    c = _run(a2, w2, sa2, sb2, None, "bf16", tile)[:70]
    bad = torch.zeros(70, 288, dtype=torch.bool)
    bad[[3, 33]] = True
    bad[:, 17] = True
    bad[:, 256:] = True
    assert c[bad].isnan().all()
    free = ~bad
    free[9] = False
    assert torch.equal(c[free], clean[free])
    assert not c[9, ~bad[9]].isfinite().any()  # an infinite scale times a block's sum, or times its zero


def test_offsets_that_go_back_or_leave_the_rows():
    """They move nothing out of the operands: rows that one group alone has, in front of those that go back, are its product, and the guard rows stay.  (Rows 10 to 33 are of two groups each here: which
    of the two is not said.)"""
    a, w, sa, sb = _operands(60, 272, 192, 5, 1)
    c = _run(a, w, sa, sb, [-5, 20, 33, 10, 60, 1 << 30], "bf16", same=False)
    rows, vals, _ = _want(a, w, sa, sb, [0, 20, 33, 33, 33, 33])
    assert rows[:10] == list(range(10)) and torch.equal(c[:10], vals[:10].float().to(torch.bfloat16))
    assert (c[60:] == GUARD).all()


def test_last_tiles_at_the_end_of_the_arrays():
    """Operands that end where their allocation's used part ends: rows and scales behind the last are not needed."""
    for m, n, k in ((129, 272, 192), (130, 16, 64), (7, 400, 704)):
        a, w, sa, sb = _operands(m, n, k, 2, m)
        offsets = [0, m // 2, m]
        for tile in WHOLE + SLICED:
            _check_exact(_run(a, w, sa, sb, offsets, "bf16", tile), a, w, sa, sb, offsets, "bf16")


def test_replayed_with_other_sizes():
    groups, n, k, m = 6, 272, 320, 200
    a, w, sa, sb = _operands(m, n, k, groups, 5)
    fn = compile_grouped_blockscale_gemm(N=n, K=k, groups=groups)
    c = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    off = torch.zeros(groups + 1, dtype=torch.int32, device="cuda")
    da, dw, dsa, dsb = a.cuda(), _shuffled(w).cuda(), sa.cuda(), sb.cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        fn(c, da, dw, dsa, dsb, off, m, side)
    for sizes in ([0, 3, 150, 1, 40, 6], [200, 0, 0, 0, 0, 0], [33, 33, 33, 33, 33, 33]):
        o = _offsets(sizes)
        off.copy_(torch.tensor(o, dtype=torch.int32))
        c.fill_(GUARD)
        graph.replay()
        torch.cuda.synchronize()
        _check_exact(c.cpu(), a, w, sa, sb, o, "bf16")


def test_other_streams():
    a, w, sa, sb = _operands(90, 272, 1024, 1, 6)
    args = a.cuda(), _shuffled(w).cuda(), sa.cuda(), sb.cuda(), 90
    fn = compile_blockscale_gemm(N=272, K=1024)
    torch.cuda.synchronize()
    outs = [torch.empty(90, 272, dtype=torch.bfloat16, device="cuda") for _ in range(4)]
    streams = [torch.cuda.Stream() for _ in outs]
    torch.cuda.synchronize()
    for _ in range(3):
        for c, s in zip(outs, streams):
            fn(c, *args, s)
    torch.cuda.synchronize()
    for c in outs:
        _check_exact(c.cpu(), a, w, sa, sb, None, "bf16")


def test_refusals():
    fn = compile_blockscale_gemm(N=144, K=192)
    e = lambda *s, dt=FP8, dev="cuda": torch.zeros(*s, dtype=dt, device=dev)
    f32 = torch.float32
    good = [e(10, 144, dt=torch.bfloat16), e(10, 192), e(144, 192), e(2, 10, dt=f32), e(2, 2, dt=f32)]
    for stream in (None, torch.cuda.current_stream()):
        fn(*good, 10, stream)
        for at, bad in ((0, e(9, 144, dt=torch.bfloat16)), (0, e(10, 144, dt=torch.float16)), (0, e(10, 144, dt=f32)), (1, e(9, 192)), (1, e(10, 192, dt=torch.bfloat16)), (1, e(10, 192, dev="cpu")), (1, e(192, 10).t()),
                        (2, e(143, 192)), (3, e(10, 2, dt=f32)), (3, e(1, 10, dt=f32)), (3, e(2, 9, dt=f32)), (3, e(2, 11, dt=f32)), (3, e(10, 2, dt=f32).t()), (3, e(2, 10, dt=torch.float16)), (3, e(20, dt=f32)),
                        (3, e(1, 10, dt=f32).expand(2, 10)), (3, e(2, 10, dt=f32, dev="cpu")), (3, None), (4, e(3, dt=f32)), (4, e(2, 2, dt=torch.float16)), (4, None)):
            args = list(good)
            args[at] = bad
            with pytest.raises(ValueError):
                fn(*args, 10, stream)
        with pytest.raises(ValueError):
            fn(*good, (1 << 22) + 1, stream)
        with pytest.raises(ValueError, match="aligned"):
            fn(good[0], e(10 * 192 + 8)[8:].view(10, 192), *good[2:], 10, stream)
    grouped = compile_grouped_blockscale_gemm(N=144, K=192, groups=2)
    good[2], good[4] = e(2, 144, 192), e(2, 2, 2, dt=f32)
    for stream in (None, torch.cuda.current_stream()):
        grouped(*good, e(3, dt=torch.int32), 10, stream)
        for off in (e(2, dt=torch.int32), e(3, dt=torch.int64), e(3, dt=torch.int32, dev="cpu"), None):
            with pytest.raises(ValueError):
                grouped(*good, off, 10, stream)


@pytest.mark.parametrize("n,k,tile", [(16, 1088, AUTO), (16, 1088, STREAM), (16, 1088, (16, 0)), (16, 1088, (128, 0)), (16, 1088, (128, 128)), (16, 1088, (64, 64)), (528, 64, AUTO), (528, 64, STREAM), (528, 64, (64, 64))])
def test_rows_past_four_gib(n, k, tile):
    """A (k = 1088) or C (n = 528) of more than 2^32 bytes: rows at the front, about the border and at the end."""
    m = 4190003
    block, w, _, sb = _operands(65521, n, k, 1, 11)
    a = block.cuda().view(torch.uint8).repeat(-(-m // 65521), 1)[:m].view(FP8)
    sa = torch.exp2(-torch.randint(0, 4, (-(-k // 128), m), device="cuda", generator=torch.Generator("cuda").manual_seed(1)).float())
    c = torch.full((m + 1, n), GUARD, dtype=torch.bfloat16, device="cuda")
    fn = compile_blockscale_gemm(N=n, K=k)
    print(f"blockscale M={m} N={n} K={k} tile {tile}", flush=True)
    fn.tile = tile
    try:
        fn(c, a, _shuffled(w).cuda(), sa, sb.cuda(), m, torch.cuda.current_stream())
        torch.cuda.synchronize()
    finally:
        fn.tile = AUTO
    border = 2**32 // (k if n == 16 else 2 * n)
    rows = torch.tensor([r for at in (0, border // 2, border, m) for r in range(max(at - 70, 0), min(at + 70, m))], device="cuda")
    want, _ = _product(a.view(torch.uint8)[rows].view(FP8).cpu(), w[0], sa[:, rows].cpu(), sb[0])
    assert torch.equal(c[rows].cpu(), want.float().bfloat16())
    assert (c[m] == GUARD).all()


@pytest.mark.parametrize("tile", [AUTO, (32, 0), (128, 0), (128, 128), (16, 16)])
def test_weights_past_four_gib(tile):
    """37 groups' weights of 5 GB: rows of the first, of those about the border and of the last."""
    groups, n, k = 37, 16400, 8128
    sizes = [3 if e in (0, 31, 32, 36) else 0 for e in range(groups)]
    offsets, m = _offsets(sizes), sum(sizes)
    a, _, sa, _ = _operands(m, 16, k, 1, 21)
    codes = torch.arange(-4, 5).float().to(FP8).view(torch.int8).cuda()
    laid, plain = torch.empty(groups, n, k, dtype=torch.int8, device="cuda"), {}
    for e in range(groups):
        w = codes[torch.randint(0, 9, (n, k), device="cuda", generator=torch.Generator("cuda").manual_seed(e))]
        laid[e] = layout.shuffle_weight(w.unsqueeze(0))[0]
        if sizes[e]:
            plain[e] = w.view(FP8)
    sb = torch.exp2(-torch.randint(0, 4, (groups, -(-n // 128), -(-k // 128)), generator=torch.Generator().manual_seed(1)).float())
    fn = compile_grouped_blockscale_gemm(N=n, K=k, groups=groups)
    c = torch.full((m + 1, n), GUARD, dtype=torch.bfloat16, device="cuda")
    print(f"blockscale {groups} x {n} x {k} tile {tile}", flush=True)
    fn.tile = tile
    try:
        fn(c, a.cuda(), laid.view(FP8), sa.cuda(), sb.cuda(), torch.tensor(offsets, dtype=torch.int32).cuda(), m, torch.cuda.current_stream())
        torch.cuda.synchronize()
    finally:
        fn.tile = AUTO
    for e, w in plain.items():
        r = slice(offsets[e], offsets[e + 1])
        want, _ = _product(a[r].cuda(), w, sa[:, r].cuda(), sb[e].cuda())
        assert torch.equal(c[r], want.float().bfloat16()), e
    assert (c[m] == GUARD).all()
