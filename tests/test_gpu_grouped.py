"""GPU tests of the grouped products against their definition in 64 bits.

Exact inputs: operands are whole numbers up to 4 (8 in int8) and scales powers of two, so every partial sum is exact in fp32 (K * 16 < 2^24) whatever its order, and the output is the
definition rounded once.  Random inputs: K additions, off by 2^-23 of the magnitudes' sum each at most, then the rounding to 16 bits.
"""

import pytest
import torch

from flydsl_amd import layout
from kernels.gemm.grouped_gemm import compile_grouped_gemm

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp8": torch.float8_e4m3fn, "int8": torch.int8}
HALF = {"bf16": 2.0**-8, "fp16": 2.0**-11}
GUARD = -77.0


def _operands(rows, n, k, groups, dtype, seed, exact=True):
    g = torch.Generator().manual_seed(seed)
    top = 8 if dtype == "int8" else 4
    if exact or dtype == "int8":
        a, w = (torch.randint(-top, top + 1, s, generator=g).to(torch.float32).to(DT[dtype]) for s in ((rows, k), (groups, n, k)))
    else:
        a, w = (torch.randn(*s, generator=g).to(DT[dtype]) for s in ((rows, k), (groups, n, k)))
    if dtype not in ("fp8", "int8"):
        return a, w, None, None
    if exact:
        return a, w, torch.exp2(-torch.randint(0, 4, (rows,), generator=g).float()), torch.exp2(-torch.randint(0, 4, (groups, n), generator=g).float())
    return a, w, 0.01 + torch.rand(rows, generator=g), 0.01 + torch.rand(groups, n, generator=g)


def _shuffled(w):
    return layout.shuffle_weight(w.view(torch.int8) if w.element_size() == 1 else w).view(w.dtype).contiguous()


def _want(a, w, sa, sb, offsets, out):
    """Definition in 64 bits: (rows that are written, their values, the sum of their terms' magnitudes)."""
    rows, vals, mags = [], [], []
    for e in range(len(offsets) - 1):
        r = slice(offsets[e], offsets[e + 1])
        if r.stop > r.start:
            s = 1.0 if sa is None else sa[r, None].double() * sb[e].double()
            vals.append((a[r].double() @ w[e].double().t()) * s)
            mags.append((a[r].double().abs() @ w[e].double().abs().t()) * s)
            rows += range(r.start, r.stop)
    n = w.shape[1]
    return rows, torch.cat(vals or [torch.empty(0, n, dtype=torch.float64)]), torch.cat(mags or [torch.empty(0, n, dtype=torch.float64)])


def _run(a, w, sa, sb, offsets, dtype, out, tile_rows=0, m=None):
    groups, n, k = w.shape
    fn = compile_grouped_gemm(N=n, K=k, groups=groups, in_dtype=dtype, out_dtype=out)
    m = a.shape[0] if m is None else m
    c = torch.full((a.shape[0] + 3, n), GUARD, dtype=DT[out], device="cuda")
    args = a.cuda(), _shuffled(w).cuda(), None if sa is None else sa.cuda(), None if sb is None else sb.cuda(), torch.tensor(offsets, dtype=torch.int32).cuda(), m
    print(f"grouped M={m} N={n} K={k} groups={groups} {dtype} tile {tile_rows}", flush=True)
    fn.tile_rows = tile_rows
    try:
        fn(c, *args, torch.cuda.current_stream())
        again = torch.full_like(c, GUARD)
        fn(again, *args)
        torch.cuda.synchronize()
    finally:
        fn.tile_rows = 0
    assert torch.equal(c.view(torch.int16), again.view(torch.int16))
    return c.cpu()


def _check_exact(c, a, w, sa, sb, offsets, out):
    rows, vals, _ = _want(a, w, sa, sb, offsets, out)
    assert torch.equal(c[rows], vals.float().to(DT[out]))
    rest = torch.ones(c.shape[0], dtype=torch.bool)
    rest[rows] = False
    assert (c[rest] == GUARD).all()


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


@pytest.mark.parametrize("dtype,out", [("fp8", "bf16"), ("int8", "fp16"), ("bf16", "bf16"), ("fp16", "fp16"), ("bf16", "fp16")])
@pytest.mark.parametrize("tile_rows", [0, 16, 32, 64, 128])
@pytest.mark.parametrize("sizes", SIZES)
def test_exact_sums(sizes, tile_rows, dtype, out):
    s = SIZES[sizes]
    n, k = (272, 192) if dtype in ("fp8", "int8") else (336, 96)  # a half step at the end, columns that end inside every tile
    offsets = _offsets(s, first=2)
    a, w, sa, sb = _operands(offsets[-1] + 5, n, k, len(s), dtype, len(s))
    _check_exact(_run(a, w, sa, sb, offsets, dtype, out, tile_rows), a, w, sa, sb, offsets, out)


@pytest.mark.parametrize("dtype,n,k", [("fp8", 16, 64), ("fp8", 1040, 4096), ("int8", 512, 1600), ("bf16", 16, 32), ("bf16", 528, 1056), ("fp16", 2048, 544)])
@pytest.mark.parametrize("sizes", [[1], [20, 0, 31], [300, 1, 700]])
def test_widths_and_lengths(sizes, dtype, n, k):
    offsets = _offsets(sizes)
    a, w, sa, sb = _operands(offsets[-1], n, k, len(sizes), dtype, n + k)
    _check_exact(_run(a, w, sa, sb, offsets, dtype, "bf16"), a, w, sa, sb, offsets, "bf16")


@pytest.mark.parametrize("dtype", ["fp8", "int8", "bf16", "fp16"])
def test_random_values_and_the_same_bits_on_every_tile(dtype):
    offsets = _offsets(SIZES["ragged"])
    n, k, out = 400, 1088, "fp16" if dtype == "fp16" else "bf16"
    a, w, sa, sb = _operands(offsets[-1], n, k, len(offsets) - 1, dtype, 3, exact=False)
    if dtype == "fp16":
        w = w / 64  # inside fp16's range
    rows, vals, mags = _want(a, w, sa, sb, offsets, out)
    first = None
    for tile_rows in (16, 32, 64, 128):
        c = _run(a, w, sa, sb, offsets, dtype, out, tile_rows)
        assert ((c[rows].double() - vals).abs() <= HALF[out] * vals.abs() + (k + 3) * 2.0**-23 * (1 + HALF[out]) * mags + 2.0**-25).all()
        first = c if first is None else first
        assert torch.equal(c.view(torch.int16), first.view(torch.int16))


def test_same_bits_as_the_dense_product():
    """A group alone is the dense product of the same rows."""
    from kernels.gemm.preshuffle_gemm import compile_preshuffle_gemm

    rows, n, k = 300, 512, 1024
    a, w, sa, sb = _operands(rows, n, k, 1, "fp8", 9, exact=False)
    c = _run(a, w, sa, sb, [0, rows], "fp8", "bf16")
    dense = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda")
    fn = compile_preshuffle_gemm(N=n, K=k, tile_m=128, tile_n=256, tile_k=128, in_dtype="fp8")
    fn.launch_forced(dense, a.cuda(), _shuffled(w[0]).cuda(), sa.cuda(), sb[0].cuda(), None, rows, n, force_path=1, tile=(128, 256))
    assert torch.equal(c[:rows].view(torch.int16), dense.cpu().view(torch.int16))


@pytest.mark.parametrize("tile_rows", [16, 32, 64, 128])
def test_offsets_that_leave_the_rows(tile_rows):
    """Offsets before 0, past M and going back: nothing outside of C is written, and groups with sound offsets in front of the first bad one are right."""
    n, k, rows = 272, 128, 90
    a, w, sa, sb = _operands(rows, n, k, 4, "fp8", 4)
    for offsets, sound in [([-5, 20, 60, 400, 1000], [0, 20, 60, 90, 90]), ([90, 90, 90, 90, 90], [90] * 5), ([0, 30, 10, 10, 5], None), ([-(2**31), 2**31 - 1, 2**31 - 1, 0, 0], None),
                           ([0, 90, 0, 90, 0], None), ([0, 90, -1, 90, 90], None)]:
        c = _run(a, w, sa, sb, offsets, "fp8", "bf16", tile_rows) if sound else None
        if sound:
            _check_exact(c, a, w, sa, sb, sound, "bf16")
            continue
        fn = compile_grouped_gemm(N=n, K=k, groups=4)
        fn.tile_rows = tile_rows
        c = torch.full((rows + 150, n), GUARD, dtype=torch.bfloat16, device="cuda")
        try:
            fn(c, a.cuda(), _shuffled(w).cuda(), sa.cuda(), sb.cuda(), torch.tensor(offsets, dtype=torch.int32).cuda(), rows)
            torch.cuda.synchronize()
        finally:
            fn.tile_rows = 0
        assert (c[rows:] == GUARD).all()


def test_rows_that_are_not_finite_stay_by_themselves():
    offsets = _offsets([5, 40, 3])
    a, w, sa, sb = _operands(48, 64, 128, 3, "bf16", 6)
    clean = _run(a, w, sa, sb, offsets, "bf16", "bf16")
    a[4, 3], a[6, 0] = float("nan"), float("inf")
    w[2, 5, 9] = float("nan")
    c = _run(a, w, sa, sb, offsets, "bf16", "bf16")
    keep = torch.ones(48, 64, dtype=torch.bool)
    keep[4], keep[6], keep[45:, 5] = False, False, False
    assert torch.isnan(c[4]).all() and not torch.isfinite(c[6]).any() and torch.isnan(c[45:48, 5]).all()
    assert torch.equal(c[:48][keep], clean[:48][keep])


def test_graph_replays_with_other_sizes():
    n, k, groups, rows = 512, 256, 6, 200
    a, w, sa, sb = _operands(rows, n, k, groups, "int8", 2)
    fn = compile_grouped_gemm(N=n, K=k, groups=groups, in_dtype="int8")
    dev = [t.cuda() for t in (a, _shuffled(w), sa, sb)]
    offsets = torch.zeros(groups + 1, dtype=torch.int32, device="cuda")
    c = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        fn(c, *dev, offsets, rows, side)
    for sizes in ([10, 0, 90, 1, 50, 49], [200, 0, 0, 0, 0, 0], [0, 0, 0, 0, 0, 3], [33] * 6):
        o = _offsets(sizes)
        offsets.copy_(torch.tensor(o, dtype=torch.int32))
        c.fill_(GUARD)
        graph.replay()
        eager = torch.full_like(c, GUARD)
        fn(eager, *dev, offsets, rows)
        torch.cuda.synchronize()
        assert torch.equal(c, eager)
        _check_exact(c.cpu(), a, w, sa, sb, o, "bf16")


def test_rows_and_weights_beyond_32_bits():
    """C and A past 2^32 bytes, and a weight that begins past 2^32 bytes."""
    n, k, rows = 8192, 2048, 300_000  # C 4.9 GB
    fn = compile_grouped_gemm(N=n, K=k, groups=3, in_dtype="bf16", out_dtype="bf16")
    a = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(3, n, k, dtype=torch.bfloat16, device="cuda")
    a[-7:, 5], a[3, 5] = 3.0, 2.0
    w[2, :, 5], w[0, :, 5] = 0.5, 4.0
    c = torch.full((rows, n), GUARD, dtype=torch.bfloat16, device="cuda")
    offsets = torch.tensor([0, 10, 10, rows], dtype=torch.int32, device="cuda")
    laid = torch.stack([layout.shuffle_weight(x) for x in w])
    fn(c, a, laid, None, None, offsets, rows)
    torch.cuda.synchronize()
    assert (c[3] == 8).all() and (c[-7:] == 1.5).all() and (c[4:-7] == 0).all()
    big = torch.zeros(34, n, 16384, dtype=torch.int8, device="cuda")  # 4.6 GB
    big[33, :, 7] = 3
    x = torch.zeros(5, 16384, dtype=torch.int8, device="cuda")
    x[:, 7] = 2
    laid = torch.zeros_like(big)
    laid[33] = layout.shuffle_weight(big[33])
    fn = compile_grouped_gemm(N=n, K=16384, groups=34, in_dtype="int8")
    c = torch.zeros(5, n, dtype=torch.bfloat16, device="cuda")
    fn(c, x, laid, torch.ones(5, device="cuda"), torch.ones(34, n, device="cuda"), torch.tensor([0] * 34 + [5], dtype=torch.int32, device="cuda"), 5)
    torch.cuda.synchronize()
    assert (c == 6).all()


def test_refusals():
    fn = compile_grouped_gemm(N=64, K=128, groups=2, in_dtype="fp8")
    b = lambda *s, dt=torch.float32: torch.zeros(*s, dtype=dt, device="cuda")
    good = dict(C=b(4, 64, dt=torch.bfloat16), A=b(4, 128, dt=DT["fp8"]), B=b(2, 64, 128, dt=DT["fp8"]), scale_a=b(4), scale_b=b(2, 64), offsets=b(3, dt=torch.int32))
    for stream in (None, torch.cuda.current_stream()):
        fn(*good.values(), 4, stream)
        for name, bad in [("C", b(3, 64, dt=torch.bfloat16)), ("A", b(4, 127, dt=DT["fp8"])), ("B", b(1, 64, 128, dt=DT["fp8"])), ("scale_a", b(3)), ("scale_b", b(64)), ("offsets", b(2, dt=torch.int32)),
                          ("offsets", b(3, dt=torch.int64)), ("C", b(4, 64, dt=torch.float16)), ("scale_a", None), ("A", b(4, 256, dt=DT["fp8"])[:, ::2]), ("offsets", b(3))]:
            with pytest.raises(ValueError, match=name):
                fn(*{**good, name: bad}.values(), 4, stream)
        with pytest.raises(ValueError, match="outside"):
            fn(*good.values(), 0, stream)


def _exact_on_the_device(rows, n, k, groups, dtype, out, sizes, tile_rows):
    """Whole numbers as in _operands, made and compared on the device; rows behind the last group stay as they were."""
    g = torch.Generator(device="cuda").manual_seed(rows + n)
    top = 8 if dtype == "int8" else 4
    a, w = (torch.randint(-top, top + 1, s, generator=g, device="cuda", dtype=torch.int8).to(DT[dtype]) for s in ((rows, k), (groups, n, k)))
    sa = sb = None
    if dtype in ("fp8", "int8"):
        sa, sb = (torch.exp2(-torch.randint(0, 4, s, generator=g, device="cuda").float()) for s in ((rows,), (groups, n)))
    offsets = _offsets(sizes)
    c = torch.full((rows, n), GUARD, dtype=DT[out], device="cuda")
    fn = compile_grouped_gemm(N=n, K=k, groups=groups, in_dtype=dtype, out_dtype=out)
    laid = torch.stack([_shuffled(x) for x in w])
    print(f"grouped M={rows} N={n} K={k} groups={groups} {dtype} {out} tile {tile_rows}", flush=True)
    fn.tile_rows = tile_rows
    try:
        fn(c, a, laid, sa, sb, torch.tensor(offsets, dtype=torch.int32).cuda(), rows, torch.cuda.current_stream())
        torch.cuda.synchronize()
    finally:
        fn.tile_rows = 0
    for e in range(groups):
        for at in range(offsets[e], offsets[e + 1], 2048):
            r = slice(at, min(at + 2048, offsets[e + 1]))
            want = a[r].double() @ w[e].double().t().contiguous()
            if sa is not None:
                want = want * sa[r, None].double() * sb[e].double()
            assert torch.equal(c[r], want.float().to(DT[out]))
    assert (c[offsets[-1] :] == GUARD).all()


@pytest.mark.parametrize("dtype,out,n,k", [("fp8", "bf16", 4112, 4096), ("int8", "fp16", 4112, 4160), ("bf16", "bf16", 2064, 4128), ("fp16", "fp16", 2064, 4096)])
@pytest.mark.parametrize("tile_rows", [16, 32, 64])
def test_weights_past_the_caches(tile_rows, dtype, out, n, k):
    """Eight weights of 135 MB together, rows for three quarters of a tile each: the builds that read W past the caches."""
    rows = tile_rows * 6
    sizes = [tile_rows, 1, 0, tile_rows - 1, tile_rows + 2, 5, 0]
    sizes.append(rows - 3 - sum(sizes))
    _exact_on_the_device(rows, n, k, 8, dtype, out, sizes, tile_rows)


@pytest.mark.parametrize("dtype,out", [("fp8", "bf16"), ("fp8", "fp16"), ("int8", "bf16"), ("int8", "fp16"), ("bf16", "bf16"), ("bf16", "fp16"), ("fp16", "bf16"), ("fp16", "fp16")])
def test_outputs_past_the_caches(dtype, out):
    """C of 176 MB, in ragged tiles of 128 rows and columns that end inside one."""
    _exact_on_the_device(22000, 4112, 192 if dtype in ("fp8", "int8") else 96, 5, dtype, out, [7000, 0, 129, 8255, 6600], 128)


@pytest.mark.parametrize("tile_rows", [0, 16, 32, 64, 128])
def test_groups_in_front_of_offsets_that_go_back(tile_rows):
    n, k = 272, 128
    a, w, sa, sb = _operands(90, n, k, 4, "fp8", 5)
    for offsets, sound in [([0, 30, 10, 10, 5], [0, 30, 30, 30, 30]), ([3, 20, 61, 7, 7], [3, 20, 61, 61, 61]), ([-4, 90, 80, 70, 0], [0, 90, 90, 90, 90])]:
        _check_exact(_run(a, w, sa, sb, offsets, "fp8", "bf16", tile_rows), a, w, sa, sb, sound, "bf16")
