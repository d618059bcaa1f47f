"""GPU tests of the products with 4-bit weights and group scales against their definition in 64 bits.

Exact inputs: activations are whole numbers up to 8 and scales powers of two, so that every partial sum (at most K * 8 * 15 steps of a quarter of the largest scale, below 2^24) is exact in fp32 whatever its order: the output
is the definition, rounded once to 16 bits, to the bit.
Random inputs: with u = 2^-23 for every addition in whatever order, a group's sum of codes and the sum of activations times 16 + zero are off by at most group * u * 31 * sum|a| each, the
groups' sums by another (K / group + 8) u of their magnitudes; then the rounding to 16 bits, and what the activation function makes of the error (its slope is at most 1.13)
and its own evaluation (2^-20, of exp2 and a reciprocal).
"""

import pytest
import torch

from flydsl_amd import layout, quant
from kernels.gemm.w4a16_gemm import compile_w4a16_gemm

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
HALF = {"bf16": 2.0**-8, "fp16": 2.0**-11}


def _weights(n, k, group, dt, zero_points, seed, exact):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8)
    if exact:
        scale = torch.exp2(-torch.randint(4, 7, (n, k // group), generator=g).float()).to(dt)
    else:
        scale = (0.002 + 0.01 * torch.rand(n, k // group, generator=g)).to(dt)
    zero = torch.randint(0, 16, (n, k // group), generator=g, dtype=torch.uint8) if zero_points else None
    return codes, scale, zero


def _deq(codes, scale, zero, group):
    z = torch.full(scale.shape, 8.0, dtype=torch.float64) if zero is None else zero.double()
    return (codes.double() - z.repeat_interleave(group, 1)) * scale.double().repeat_interleave(group, 1)


def _act(y, epi):
    if epi == "bias_relu":
        return y.clamp(min=0)
    if epi == "bias_silu":
        return y * torch.sigmoid(y)
    if epi == "bias_gelu":
        return 0.5 * y * (1 + torch.tanh(0.7978845608 * (y + 0.044715 * y**3)))
    return y


def _run(a, codes, scale, zero, bias, group, dtype, epi, guard=3):
    m, k = a.shape
    n = codes.shape[0]
    fn = compile_w4a16_gemm(N=n, K=k, group_size=group, in_dtype=dtype, zero_points=zero is not None, epilogue=epi)
    c = torch.full((m + guard, n), -77.0, dtype=DT[dtype], device="cuda")
    z = None if zero is None else layout.shuffle_group_zeros(zero).cuda()
    args = a.cuda(), layout.shuffle_weight_w4a16(codes).cuda(), layout.shuffle_group_scales(scale).cuda(), z, None if bias is None else bias.cuda(), m
    print(f"w4a16 M={m} N={n} K={k} group={group} {dtype} {epi}", flush=True)
    fn(c, *args, torch.cuda.current_stream())
    again = torch.empty_like(c[:m])
    fn(again, *args)  # the Python checks, the current stream
    torch.cuda.synchronize()
    assert (c[m:] == -77).all()
    assert torch.equal(c[:m].view(torch.int16), again.view(torch.int16))
    return c[:m].cpu()


SIZES = [(1, 16, 128), (1, 4096, 4096), (2, 2064, 1152), (5, 1040, 2176), (16, 48, 11008), (17, 512, 640), (32, 7168, 2048), (33, 272, 512), (100, 1024, 1024), (3, 28672, 256), (16, 8208, 384), (20, 1040, 4096), (16, 2064, 8192),
         (8, 528, 6144), (3, 32992, 5120), (1, 16, 32768), (9, 14352, 7168),
         (32, 8192, 4096), (17, 8176, 8192), (32, 8208, 6144), (40, 4112, 5120)]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("group,zero_points,dtype", [(128, False, "bf16"), (128, True, "fp16"), (64, True, "bf16"), (64, False, "fp16"), (32, False, "fp16"), (32, True, "bf16")])
def test_exact_sums(m, n, k, group, zero_points, dtype):
    if group < 128:
        k -= 128 - group if k > 128 else 0  # rows that end inside a block
    dt = DT[dtype]
    codes, scale, zero = _weights(n, k, group, dt, zero_points, m + n + k, True)
    a = torch.randint(-8, 9, (m, k), generator=torch.Generator().manual_seed(m)).to(dt)
    got = _run(a, codes, scale, zero, None, group, dtype, "none")
    want = (a.double() @ _deq(codes, scale, zero, group).t()).float()  # exact in fp32
    assert torch.equal(got, want.to(dt))


@pytest.mark.parametrize("m,n,k", [(16, 1040, 4224), (1, 528, 5120), (40, 272, 5120), (8, 1040, 5248), (9, 1040, 5376), (3, 4112, 6144), (16, 4112, 6144), (8, 528, 6272), (1, 8208, 7168), (7, 1040, 8192), (9, 1040, 8192)])
@pytest.mark.parametrize("group,zero_points,dtype", [(128, False, "fp16"), (128, True, "bf16"), (64, True, "fp16"), (64, False, "bf16")])
def test_exact_sums_of_five_to_eight_steps(m, n, k, group, zero_points, dtype):
    test_exact_sums(m, n, k, group, zero_points, dtype)


@pytest.mark.parametrize("m,n,k", [(17, 528, 2176), (23, 1040, 2688), (24, 4112, 2944), (25, 528, 2944), (32, 1040, 3200), (24, 272, 4096)])
@pytest.mark.parametrize("group,zero_points,dtype", [(128, True, "bf16"), (64, False, "bf16"), (64, True, "fp16"), (32, False, "bf16"), (32, True, "fp16")])
def test_exact_sums_of_three_and_four_steps(m, n, k, group, zero_points, dtype):
    test_exact_sums(m, n, k, group, zero_points, dtype)


@pytest.mark.parametrize("m,n,k", [(1, 528, 896), (16, 28688, 1024), (33, 1040, 1024), (17, 528, 768), (8, 4112, 2816), (16, 28688, 2560), (7, 1040, 7168), (1, 528, 9216), (16, 4112, 8832), (9, 16912, 9216), (3, 17424, 8320),
                                   (24, 8720, 6144), (17, 528, 5248), (20, 16400, 4224)])
@pytest.mark.parametrize("group,zero_points,dtype", [(128, False, "bf16"), (64, True, "bf16"), (32, False, "fp16"), (32, True, "bf16")])
def test_exact_sums_of_other_steps_and_passes(m, n, k, group, zero_points, dtype):
    test_exact_sums(m, n, k, group, zero_points, dtype)


@pytest.mark.parametrize("epi", ["none", "bias", "bias_relu", "bias_silu", "bias_gelu"])
@pytest.mark.parametrize("m,n,k,group,zero_points,dtype", [(1, 1024, 4096, 128, True, "bf16"), (9, 528, 2080, 32, True, "fp16"), (31, 320, 960, 64, False, "bf16")])
def test_random_values_and_epilogues(m, n, k, group, zero_points, dtype, epi):
    dt = DT[dtype]
    codes, scale, zero = _weights(n, k, group, dt, zero_points, 5, False)
    g = torch.Generator().manual_seed(6)
    a, bias = torch.randn(m, k, generator=g).to(dt), (0.5 * torch.randn(n, generator=g)).to(dt)
    got = _run(a, codes, scale, zero, None if epi == "none" else bias, group, dtype, epi).double()
    w = _deq(codes, scale, zero, group)
    y = a.double() @ w.t()
    u = 2.0**-23
    mags = (a.double().abs().view(m, -1, group).sum(-1)) @ scale.double().t()
    slack = 2 * group * u * 31 * mags + (k // group + 8) * u * (a.double().abs() @ w.abs().t())
    if epi != "none":
        y = y + bias.double()
        slack = slack + u * y.abs()
    want = _act(y, epi)
    slack = 1.13 * slack + (2.0**-20 * y.abs() if epi in ("bias_silu", "bias_gelu") else 0)
    assert ((got - want).abs() <= HALF[dtype] * (want.abs() + slack) + slack + 2.0**-25).all()


def test_quantised_weights_and_outlier_rows():
    """What the quantiser makes, with an activation row of zeros and one that is not finite beside the others."""
    g = torch.Generator().manual_seed(8)
    w = 0.02 * torch.randn(256, 1024, generator=g)
    a = torch.randn(6, 1024, generator=g).to(torch.bfloat16)
    a[1] = 0
    a[4, 7] = float("nan")
    for zero_points in (False, True):
        codes, scale, zero = quant.pergroup_w4_quant(w, 64, zero_points)
        got = _run(a, codes, scale, zero, None, 64, "bf16", "none").float()
        keep = [0, 2, 3, 5]
        want = (a[keep].double() @ _deq(codes, scale, zero, 64).t()).float()
        assert (got[1] == 0).all() and torch.isnan(got[4]).all()
        assert (got[keep] - want).abs().max() <= 2.0**-7 * want.abs().max()
        # and the weights are what they were quantised from: 15 or 16 steps over a group's range of about 5 deviations, sqrt(1/12) of a step each
        full = a[keep].double() @ w.double().t()
        assert (got[keep] - full).norm() / full.norm() < 0.13


def test_graph_replays():
    m, n, k = 4, 1024, 2048
    fn = compile_w4a16_gemm(N=n, K=k, group_size=128)
    codes, scale, _ = _weights(n, k, 128, torch.bfloat16, False, 3, True)
    w, s = layout.shuffle_weight_w4a16(codes).cuda(), layout.shuffle_group_scales(scale).cuda()
    a = torch.randint(-8, 9, (m, k)).to(torch.bfloat16).cuda()
    c, eager = (torch.empty(m, n, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        fn(c, a, w, s, None, None, m, side)
    for _ in range(3):
        a.copy_(torch.randint(-8, 9, (m, k)).to(torch.bfloat16))
        graph.replay()
        fn(eager, a, w, s, None, None, m)
        torch.cuda.synchronize()
        assert torch.equal(c, eager)
        want = (a.cpu().double() @ _deq(codes, scale, None, 128).t()).float().to(torch.bfloat16)
        assert torch.equal(c.cpu(), want)


def test_refusals():
    fn = compile_w4a16_gemm(N=64, K=256, zero_points=True, epilogue="bias")
    b = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt, device="cuda")
    good = dict(C=b(4, 64), A=b(4, 256), W=b(64, 128, dt=torch.uint8), scales=b(4, 2, 16), zeros=b(4, 2, 8, dt=torch.uint8), bias=b(64))
    for stream in (None, torch.cuda.current_stream()):
        fn(*good.values(), 4, stream)
        for name, bad in [("C", b(3, 64)), ("A", b(4, 255)), ("W", b(63, 128, dt=torch.uint8)), ("scales", b(4, 2, 15)), ("zeros", b(4, 2, 7, dt=torch.uint8)), ("bias", b(63)),
                          ("A", b(4, 256, dt=torch.float16)), ("scales", b(4, 2, 16, dt=torch.float16)), ("zeros", None), ("bias", None), ("W", b(64, 256, dt=torch.uint8)[:, ::2]),
                          ("A", b(4, 512)[:, :256])]:
            with pytest.raises(ValueError, match=name):
                fn(*{**good, name: bad}.values(), 4, stream)
        with pytest.raises(ValueError, match="aligned"):
            fn(*{**good, "A": b(4 * 256 + 4)[4:]}.values(), 4, stream)
        with pytest.raises(ValueError, match="outside"):
            fn(*good.values(), 0, stream)


@pytest.mark.parametrize("m,n,k,group,zero_points,dtype", [(6, 528, 1024, 128, False, "bf16"), (6, 272, 2080, 32, True, "fp16"), (20, 1040, 2560, 64, False, "bf16"), (31, 528, 4096, 128, True, "bf16"), (9, 2064, 9216, 128, True, "bf16"),
                                                         (22, 1040, 6144, 32, False, "fp16"), (40, 272, 5120, 64, True, "bf16")])
def test_infinities_and_sums_beyond_fp32(m, n, k, group, zero_points, dtype):
    """An infinity in a row of A is one in the columns whose weight of it is not zero; finite rows have finite products, also where a group's sum of 16 + code is beyond fp32.  Rows beside them are what
    they are without."""
    dt = DT[dtype]
    codes, scale, zero = _weights(n, k, group, dt, zero_points, m + n, True)
    a = torch.randint(-8, 9, (m, k), generator=torch.Generator().manual_seed(m)).to(dt)
    inf = float("inf")
    a[0, 7], a[1, k - 1] = inf, -inf
    a[3, 5], a[3, k // 2] = inf, inf
    a[m - 1, 0], a[m - 1, 33] = inf, -inf
    if dtype == "bf16":
        a[4] = 0
        a[4, 1:4], a[4, k - 2] = 2.0**124, -(2.0**124)  # times up to 31 beyond 2^128, times (q - z) s at most 2^124 4 15 / 16
    got = _run(a, codes, scale, zero, None, group, dtype, "none")
    w = _deq(codes, scale, zero, group)
    rows = [i for i in range(m) if torch.isfinite(a[i]).all()]
    want = torch.empty(m, n, dtype=torch.float64)
    want[rows] = a[rows].double() @ w.t()
    for i in set(range(m)) - set(rows):  # (the library's product may take an infinity times zero out of a sum)
        want[i] = (a[i].double() * w)[:, ~torch.isfinite(a[i])].sum(1)
    want = want.float().to(dt)
    assert torch.isfinite(want[rows]).all() and torch.isinf(want[[0, 1]]).any() and torch.isnan(want[m - 1]).any()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(7.0, inf, -inf), want.nan_to_num(7.0, inf, -inf))


# one size for every build of the kernel that the sizes above do not take: three steps of up to 24 rows, passes of two steps of up to 24 rows, of three and of two steps of 16
BUILDS = [(24, 2048, 2560, 128, False), (20, 8720, 5248, 128, True), (17, 8208, 5184, 64, False), (16, 4112, 9216, 128, True), (9, 1040, 9152, 64, False), (3, 33024, 8320, 128, False), (16, 32784, 8320, 128, True),
          (5, 33040, 7232, 64, False), (1, 32784, 7232, 64, True)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("m,n,k,group,zero_points", BUILDS)
def test_exact_sums_of_the_other_builds(m, n, k, group, zero_points, dtype):
    dt = DT[dtype]
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    codes = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8, device="cuda")
    scale = torch.exp2(-torch.randint(4, 7, (n, k // group), generator=g, device="cuda").float()).to(dt)
    zero = torch.randint(0, 16, (n, k // group), generator=g, dtype=torch.uint8, device="cuda") if zero_points else None
    a = torch.randint(-8, 9, (m, k), generator=g, device="cuda").to(dt)
    got = _run(a, codes, scale, zero, None, group, dtype, "none")
    for n0 in range(0, n, 4096):  # (8 bytes a weight here)
        c = slice(n0, n0 + 4096)
        z = torch.full_like(scale[c], 8.0, dtype=torch.float64) if zero is None else zero[c].double()
        w = (codes[c].double() - z.repeat_interleave(group, 1)) * scale[c].double().repeat_interleave(group, 1)
        want = (a.double() @ w.t().contiguous()).float()
        assert torch.equal(got[:, c], want.to(dt).cpu())
