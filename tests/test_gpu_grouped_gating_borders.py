"""GPU tests of the routing by groups where its 32 bits meet its definition in 64: zeros of both signs at the border of the top-k, groups whose two
best cancel, and the weights.

Expected experts come from the definition in 64 bits by stable sorts, lower index first of equal ones, and have to be equal.
"""

import pytest
import torch

from kernels.moe.grouped_topk_gating import build_grouped_topk_gating_module

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _launch(x, bias, topk, dtype="f32", **options):
    t, e = x.shape
    fn = build_grouped_topk_gating_module(e, topk, dtype, **options)
    w, ids = torch.full((t, topk), -7.0, device="cuda"), torch.full((t, topk), -7, dtype=torch.int32, device="cuda")
    print(f"route {t}x{e} top {topk} {dtype} {options}", flush=True)
    fn(x.to(DT[dtype]).cuda(), None if bias is None else bias.cuda(), w, ids, t, stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    return w.cpu(), ids.cpu().long()


def _first(c, k):
    """Indices of the k largest of every row, the lower of equal ones first (0.0 and -0.0 are equal)."""
    return torch.sort(c, dim=-1, descending=True, stable=True)[1][..., :k]


def _scores(x, scores):
    x = x.double()
    return 1 / (1 + torch.exp(-x)) if scores == "sigmoid" else torch.softmax(x, 1)


@pytest.mark.parametrize("scores", ["sigmoid", "softmax"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("t,e,topk", [(1, 2, 1), (1, 64, 8), (37, 64, 8), (50, 256, 30), (9001, 256, 30), (5, 1023, 32), (20, 17, 3)])
def test_zeros_of_both_signs_are_equal(t, e, topk, dtype, scores):
    """Logits times a mask leave zeros of both signs, and the last experts taken are among them: fewer logits are above zero than are taken, half of all are
    zeros; 9001 tokens share wavefronts by twos."""
    g = torch.Generator().manual_seed(t + e)
    u = torch.rand(t, e, generator=g)
    x = torch.where(u < 0.1 * topk / e, 1.0, torch.where(u < 0.5, -1.0, torch.where(u < 0.75, -0.0, 0.0)))
    if e == 2:
        x = torch.tensor([[-0.0, 0.0]])
    w, ids = _launch(x, None, topk, dtype, scores=scores, renormalize=False)
    assert torch.equal(ids, _first(x.double() + 0.0, topk))
    if e > 2:  # (half the experts of a run at most are above zero, and every run has zeros)
        for groups, kept in ((1, 1),) + (((8, 4),) if e % 8 == 0 else ()):
            c = x.double() + 0.0
            if groups > 1:
                parts = c.view(t, groups, -1)
                keep = torch.zeros(t, groups, dtype=torch.bool).scatter_(1, _first(parts.amax(-1), kept), True)
                c = parts.masked_fill(~keep.unsqueeze(-1), -float("inf")).view(t, e)
            assert torch.equal(_launch(x, None, topk, dtype, scores=scores, groups=groups, topk_groups=kept, group_score="max")[1], _first(c, topk))


def _by_group_sums(x, bias, topk, scores, groups, kept):
    c = _scores(x, scores) + bias.double()
    parts = c.view(x.shape[0], groups, -1)
    best = parts.topk(2, -1)[0]
    keep = torch.zeros(x.shape[0], groups, dtype=torch.bool).scatter_(1, _first(best[..., 0] + best[..., 1], kept), True)
    return _first(parts.masked_fill(~keep.unsqueeze(-1), -float("inf")).view_as(c), topk)


def test_two_groups_whose_sums_cancel():
    """Sums of +1000 and -1000: 0.70155918 and 0.70154750 in 64 bits, and in 32 the other way round by five times that."""
    x = torch.tensor([[-0.9691795, -0.2960838, -0.9690792, -0.29621333]])
    bias = torch.tensor([1000.0, -1000.0, 1000.0, -1000.0])
    assert torch.equal(_launch(x, bias, 2, groups=2, topk_groups=1)[1], torch.tensor([[0, 1]]))


@pytest.mark.parametrize("scores", ["sigmoid", "softmax"])
@pytest.mark.parametrize("e,groups,kept,topk", [(4, 2, 1, 2), (32, 8, 4, 8), (256, 8, 4, 8), (120, 40, 11, 6), (1023, 33, 5, 17)])
@pytest.mark.parametrize("size", [64.0, 1000.0, 4096.0, 2.0**20])
def test_groups_whose_two_best_cancel(size, e, groups, kept, topk, scores):
    """Biases of both signs in every group, so that a group's worth is what two far larger numbers leave; logits of a token that are close to each other, and ones that are not; wavefronts of one token
    and of more.  (In 64 bits a worth is off by 2^-32 at most; the worths are some 1e-5 apart, by softmax of many experts 1e-7.)"""
    g = torch.Generator().manual_seed(e)
    bias = torch.full((groups, e // groups), -size)
    bias[:, :: max(e // groups, 1)] = size
    bias = bias.flatten()
    for t in (50, 9000 if e <= 256 else 500):
        x = torch.randn(t, 1, generator=g) + torch.where(torch.rand(t, 1, generator=g) < 0.7, 1e-4, 1.5) * torch.randn(t, e, generator=g)
        assert torch.equal(_launch(x, bias, topk, scores=scores, groups=groups, topk_groups=kept)[1], _by_group_sums(x, bias, topk, scores, groups, kept))


@pytest.mark.parametrize("scores", ["sigmoid", "softmax"])
def test_one_group_far_from_the_others(scores):
    """One group's biases cancel at 10^4, 10^31 or 3 * 10^38, the others' are ordinary: what its worth may be off is its own."""
    g = torch.Generator().manual_seed(3)
    x = 0.3 + 1e-4 * torch.randn(300, 64, generator=g)
    for size in (1e4, 1e31, 3e38):
        bias = 0.25 * torch.ones(64)
        bias[24:32] = -size
        bias[26] = size
        assert torch.equal(_launch(x, bias, 8, scores=scores, groups=8, topk_groups=4)[1], _by_group_sums(x, bias, 8, scores, 8, 4))


@pytest.mark.parametrize("scores", ["sigmoid", "softmax"])
@pytest.mark.parametrize("first", [24, 25, 31])
@pytest.mark.parametrize("mask", [-30.0, -1e4, -1e9, -1e37])
def test_experts_masked_by_their_bias(mask, first, scores):
    """A run whose experts a bias masks, all of them, all but one, and one of them; the others close to each other and not."""
    g = torch.Generator().manual_seed(first)
    bias = 0.1 * torch.randn(64, generator=g)
    bias[first:32] = mask
    for spread in (1e-5, 1.5):
        x = 0.3 + spread * torch.randn(400, 64, generator=g)
        assert torch.equal(_launch(x, bias, 8, scores=scores, groups=8, topk_groups=4)[1], _by_group_sums(x, bias, 8, scores, 8, 4))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("scores,renormalize", [("sigmoid", True), ("sigmoid", False), ("softmax", True), ("softmax", False)])
@pytest.mark.parametrize("t,e,groups,kept,topk", [(40, 256, 8, 4, 8), (9000, 256, 8, 4, 8), (33, 1024, 1, 1, 32), (300, 8, 1, 1, 8), (7, 1023, 33, 5, 17), (200, 160, 8, 3, 1)])
def test_weights_are_rounded_once(t, e, groups, kept, topk, scores, renormalize, dtype):
    """Scores, their sum, the quotient and the product with the scale in 64 bits, one rounding to 32: half a unit, 2^-24 of the value, and some 64 units of 64 bits, 2^-46, for all that is in front of it."""
    g = torch.Generator().manual_seed(t + e)
    x = (1.5 * torch.randn(t, e, generator=g)).to(DT[dtype]).float()
    bias = 0.1 * torch.randn(e, generator=g)
    w, ids = _launch(x, bias, topk, dtype, scores=scores, groups=groups, topk_groups=kept, group_score="max" if topk == 1 else "top2", renormalize=renormalize, scale=2.5)
    want = _scores(x, scores).gather(1, ids)
    if renormalize:
        want = want / want.sum(1, keepdim=True)
    assert ((w.double() - 2.5 * want).abs() <= (2.0**-24 + 2.0**-46) * 2.5 * want).all()
