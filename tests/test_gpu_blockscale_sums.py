"""GPU tests of the block-scaled products on operands of very different sizes, every tile, and of one token's few rows on many groups.

Tolerance: the matrix instruction adds the products of eight consecutive elements of K in one step, aligned to the largest of their exponents with 13 bits below it, so a group of eight is off by seven units of
2^-13 of its largest product at most, which is at most the largest |a| times the largest |w| of the eight.  Then 15 additions of groups of eight, the scales' product and its use, an addition for every block
and, in slices, seven of them, 2^-23 of the magnitudes each at most, and the rounding to 16 bits, half a unit.
"""

import functools

import pytest
import torch

from flydsl_amd import layout, quant
from kernels.gemm.blockscale_gemm import compile_blockscale_gemm, compile_grouped_blockscale_gemm

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn
DT = {"bf16": (torch.bfloat16, 2.0**-8), "fp16": (torch.float16, 2.0**-11)}
TILES = [(0, 0), (1, 0), (16, 0), (32, 0), (64, 0), (128, 0), (128, 128), (16, 16), (16, 32), (32, 32), (32, 64), (64, 64)]


def _far_apart(g, *shape):
    """Normal numbers times powers of two from 2^-7 to 2^7, another for every element."""
    return torch.randn(*shape, generator=g) * torch.exp2(torch.randint(-7, 8, shape, generator=g).float())


@functools.lru_cache(maxsize=4)
def _operands(rows, n, k, groups, seed):
    g = torch.Generator().manual_seed(seed)
    a, sa = quant.per_1x128_f8_quant(_far_apart(g, rows, k))
    w, sb = quant.per_128x128_f8_quant(0.02 * _far_apart(g, groups, n, k))
    return a, w, sa, sb


def _check(c, a, w, sa, sb, half):
    n, k = w.shape
    av = a.double() * sa.double().t().repeat_interleave(128, 1)[:, :k]
    wv = (w.double() * sb.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]).t().contiguous()
    largest = av.abs().view(-1, k // 8, 8).amax(-1) @ wv.abs().view(k // 8, 8, n).amax(1)
    want, slack = av @ wv, 7 * 2.0**-13 * largest + (15 + 2 + 7 + -(-k // 128)) * 2.0**-23 * (av.abs() @ wv.abs())
    assert ((c.double() - want).abs() <= half * (want.abs() + slack) + slack + 2.0**-25).all()


def _launch(fn, tile, c, *args):
    fn.tile = tile
    try:
        fn(c, *args, torch.cuda.current_stream())
        torch.cuda.synchronize()
    finally:
        fn.tile = (0, 0)
    return c.cpu()


def _laid(w):
    return layout.shuffle_weight(w.view(torch.int8)).view(FP8).contiguous().cuda()


@pytest.mark.parametrize("m,n,k", [(3, 144, 64), (70, 288, 1088), (150, 272, 4096)])
@pytest.mark.parametrize("out", ["bf16", "fp16"])
@pytest.mark.parametrize("tile", TILES)
def test_values_far_apart(m, n, k, tile, out):
    a, w, sa, sb = _operands(m, n, k, 1, m)
    dt, half = DT[out]
    print(f"blockscale M={m} N={n} K={k} tile {tile} {out}", flush=True)
    c = _launch(compile_blockscale_gemm(N=n, K=k, out_dtype=out), tile, torch.empty(m, n, dtype=dt, device="cuda"), a.cuda(), _laid(w[0]), sa.cuda(), sb[0].contiguous().cuda(), m)
    _check(c, a, w[0], sa, sb[0], half)


@pytest.mark.parametrize("tile", [t for t in TILES if t[0] != 1])
@pytest.mark.parametrize("groups,live", [(256, [1] * 8), (256, [2, 1, 1, 3, 1]), (160, [6]), (4096, [1] * 6)])
def test_a_token_on_many_groups(groups, live, tile):
    """The rows of one token or two, most groups empty: the first, the last and ones between have rows."""
    n, k, m = 80, 320, sum(live)
    a, w, sa, sb = _operands(m, n, k, groups, m)
    at = [round(i * (groups - 1) / max(len(live) - 1, 1)) for i in range(len(live))]
    sizes = [0] * groups
    for e, s in zip(at, live):
        sizes[e] = s
    offsets = torch.tensor([0] + sizes).cumsum(0)
    print(f"blockscale {m} rows on {groups} tile {tile}", flush=True)
    c = _launch(compile_grouped_blockscale_gemm(N=n, K=k, groups=groups), tile, torch.full((m + 2, n), -77.0, dtype=torch.bfloat16, device="cuda"), a.cuda(), _laid(w), sa.cuda(), sb.cuda(),
                offsets.int().cuda(), m)
    for e, s in zip(at, live):
        r = slice(int(offsets[e]), int(offsets[e]) + s)
        _check(c[r], a[r], w[e], sa[:, r], sb[e], 2.0**-8)
    assert (c[m:] == -77).all()
