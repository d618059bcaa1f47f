"""GPU tests of the routing with a bias and groups of experts against its definition in 64 bits.

The experts have to be equal.  Without a bias they are compared by their logits, exactly; with one the definition's scores and the kernel's are both in 64 bits, so they order the same but where two differ
by some 2^-52, which these inputs do not have: logits are random in 24 bits, or on a grid where equal ones are equal in both.  Weights: the score rounded to fp32, topk of them added, a division and a product: topk + 3 roundings of 2^-24.
"""

import math

import pytest
import torch

from kernels.moe.grouped_topk_gating import build_grouped_topk_gating_module

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
INF, NAN = float("inf"), float("nan")


def _want(x, bias, topk, scores, groups, topk_groups, group_score, renorm, scale):
    x = x.double().cpu()
    t, e = x.shape
    masked = x.isnan() | (x == -INF)
    x = x.masked_fill(masked, -INF)
    if scores == "sigmoid":
        s = 1 / (1 + torch.exp(-x))
    else:
        top = x.amax(1, keepdim=True)
        p = torch.where(x == top, torch.ones_like(x), torch.exp(x - top)).masked_fill(masked, 0)
        s = p / p.sum(1, keepdim=True)
    c = x if bias is None else s + bias.double().cpu()  # (without a bias the logits themselves, which order like their scores)
    masked = masked | c.isnan()
    c = c.masked_fill(masked, -INF)
    s = s.masked_fill(masked, 0)
    if topk_groups < groups:
        parts = (s.masked_fill(masked, -INF) if bias is None and group_score == "top2" else c).view(t, groups, -1)
        best = parts.topk(min(2, e // groups), -1)[0]
        worth = best[..., 0] if group_score == "max" else torch.where(best[..., 1] == -INF, best[..., 1], best[..., 0] + best[..., 1])
        order = torch.sort(worth, dim=1, descending=True, stable=True)[1]
        keep = torch.zeros(t, groups, dtype=torch.bool).scatter_(1, order[:, :topk_groups], True).repeat_interleave(e // groups, 1)
        c, s = c.masked_fill(~keep, -INF), s.masked_fill(~keep, 0)
    ids = torch.sort(c, dim=1, descending=True, stable=True)[1][:, :topk]
    w = s.gather(1, ids)
    if renorm:
        w = w / w.sum(1, keepdim=True).clamp(min=1e-20)
    return ids, w * scale


def _run(x, bias, topk, scores="sigmoid", groups=1, topk_groups=1, group_score="top2", renorm=True, scale=1.0, dtype="f32"):
    t, e = x.shape
    fn = build_grouped_topk_gating_module(e, topk, dtype, scores=scores, groups=groups, topk_groups=topk_groups, group_score=group_score, renormalize=renorm, scale=scale)
    ids = torch.full((t + 2, topk), -7, dtype=torch.int32, device="cuda")
    w = torch.full((t + 2, topk), -7.0, device="cuda")
    print(f"route {t}x{e} top {topk} {scores} {topk_groups} of {groups} {group_score} {dtype}", flush=True)
    dx, db = x.to(DT[dtype]).cuda(), None if bias is None else bias.cuda()
    fn(dx, db, w, ids, t, stream=torch.cuda.current_stream())
    again = torch.full_like(ids, -7), torch.full_like(w, -7.0)
    fn(dx, db, again[1], again[0], t)
    torch.cuda.synchronize()
    assert torch.equal(ids, again[0]) and torch.equal(w.view(torch.int32), again[1].view(torch.int32))
    assert (ids[t:] == -7).all() and (w[t:] == -7).all()
    want, ww = _want(dx, bias, topk, scores, groups, topk_groups, group_score, renorm, scale)
    assert torch.equal(ids[:t].cpu().long(), want)
    assert ((w[:t].double().cpu() - ww).abs() <= (topk + 3) * 2.0**-24 * ww.abs() + 2.0**-148).all()


def _x(t, e, seed, std=1.5):
    return std * torch.randn(t, e, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("scores", ["sigmoid", "softmax"])
@pytest.mark.parametrize("t,e,topk,groups,topk_groups", [
    (1, 256, 8, 8, 4), (5, 256, 8, 1, 1), (300, 256, 8, 8, 4), (3, 160, 6, 8, 3), (70, 160, 6, 1, 1), (9, 1024, 32, 1, 1), (9, 1024, 32, 64, 2), (4, 1023, 17, 33, 5), (4, 1020, 9, 17, 4), (4, 645, 5, 5, 2),
    (1, 1, 1, 1, 1), (7, 2, 2, 1, 1), (3, 3, 1, 1, 1), (11, 64, 4, 32, 2), (2, 65, 8, 1, 1), (5, 72, 8, 4, 1), (33, 512, 10, 16, 16), (2, 17, 17, 1, 1), (1000, 32, 4, 4, 2), (6, 120, 1, 40, 1),
])
def test_sizes(t, e, topk, groups, topk_groups, scores):
    for group_score, bias, renorm, scale in (("top2", True, True, 2.5), ("max", False, False, 1.0)):
        _run(_x(t, e, e + topk), _x(1, e, 5, 0.1)[0] if bias else None, topk, scores, groups, topk_groups, group_score, renorm, scale)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("bias", [False, True])
def test_types_and_ties(dtype, bias):
    """Logits on a grid of a quarter: most of a token's are equal to another's, and lower experts and groups go first."""
    x = (_x(200, 256, 3) * 4).round() / 4
    b = (_x(1, 256, 4, 0.3)[0] * 4).round() / 4 if bias else None
    for groups, kept, score in ((1, 1, "top2"), (8, 4, "max"), (8, 4, "top2")):
        if score == "top2" and not bias:
            continue  # (sums of two scores that are equal but for their rounding)
        if bias:
            x = torch.round(x)  # (equal sums of a score and a bias come from equal terms)
            b = torch.zeros(256)
            b[::2] = 0.5
        if score == "top2":
            b = _x(1, 8, 4, 0.3)[0].repeat_interleave(32)  # (a group's own, so that no two groups' sums meet)
        _run(x, b, 8, "sigmoid", groups, kept, score, dtype=dtype)
        if not bias:
            _run(x, b, 8, "softmax", groups, kept, score, dtype=dtype)


def test_all_equal():
    _run(torch.zeros(5, 160), None, 6, "softmax", 8, 3, "max")
    _run(torch.zeros(5, 160), torch.zeros(160), 6, "sigmoid", 8, 3, "top2")


@pytest.mark.parametrize("scores", ["sigmoid", "softmax"])
def test_masked_experts(scores):
    """-Inf and NaN among the logits, rows with fewer left than are taken, and rows with nothing left."""
    x = _x(40, 64, 9)
    g = torch.Generator().manual_seed(2)
    for r in range(40):
        x[r, torch.randperm(64, generator=g)[: 64 * r // 39]] = -INF if r % 2 else NAN
    bias = _x(1, 64, 6, 0.2)[0]
    for groups, kept in ((1, 1), (8, 2), (4, 3)):
        for b in (None, bias):
            for score in ("top2", "max"):
                _run(x, b, 8, scores, groups, kept, score)
    bias[3], bias[9], bias[17] = NAN, INF, -INF
    _run(x, bias, 8, scores, 8, 4, "top2")
    x[::3, 5] = INF
    x[::5, 6] = INF
    _run(x, None, 8, scores, 8, 4, "max")
    if scores == "sigmoid":
        _run(x, bias, 8, scores, 8, 4, "top2")


@pytest.mark.parametrize("scores", ["sigmoid", "softmax"])
def test_scores_far_from_one(scores):
    """Scores below the smallest number of fp32 order all the same, and a sum that rounds to nothing leaves weights of nothing."""
    x = torch.linspace(-300, -100, 64).repeat(3, 1)
    x[1] = x[1].flip(0)
    x[2, 7] = 0.0
    _run(x, None, 8, scores, renorm=False)
    _run(x, None, 4, scores, 4, 2, "max", renorm=False)


@pytest.mark.parametrize("scores", ["sigmoid", "softmax"])
def test_saturated_scores_order_by_their_logits(scores):
    """sigmoid(40) and sigmoid(60) are both 1 in 64 bits, exp(-800) and exp(-900) both 0: the logits tell them apart."""
    x = torch.linspace(40, 60, 64)[torch.randperm(64, generator=torch.Generator().manual_seed(0))].repeat(3, 1)
    x[1] = -x[1] * 20
    x[2, 5] = INF
    _run(x, None, 8, scores)
    _run(x, None, 8, scores, 8, 4, "max")


def test_close_scores():
    """Values a few units of the 32-bit scores apart, inside the last bits that the selection's numbers drop, equal ones among them: what is taken again in 64 bits."""
    g = torch.Generator().manual_seed(4)
    for e, groups, kept in ((64, 1, 1), (256, 8, 4), (17, 1, 1), (1024, 1, 1)):
        x = 0.5 + torch.randint(0, 40, (50, e), generator=g) * 2.0**-22
        _run(x, None, 8, "sigmoid", groups, kept, "max")
        _run(x, None, 8, "softmax", groups, kept, "max")
        bias = torch.randint(0, 3, (e,), generator=g) * 2.0**-30
        _run(x, bias, 8, "sigmoid", groups, kept, "max")
    x = _x(50, 64, 3).bfloat16().float()
    for dtype in ("bf16", "f32"):
        _run(x, torch.zeros(64), 8, "sigmoid", dtype=dtype)
        _run(x, torch.zeros(64), 8, "softmax", 8, 3, "max", dtype=dtype)


def test_border_that_32_bits_do_not_see():
    """Scores of which sigmoid and bias in fp32 would be equal, or the other way round."""
    x = torch.zeros(2, 64)
    x[:, :] = -20 - torch.arange(64) * 1e-4
    bias = torch.full((64,), 1.0)  # 1 + 2e-9 is 1 in fp32
    _run(x, bias, 8)
    _run(x.flip(1), bias, 8)


def test_no_tokens_and_refusals():
    fn = build_grouped_topk_gating_module(64, 4, "bf16", groups=8, topk_groups=2)
    e = lambda *s, dt=torch.float32, dev="cuda": torch.zeros(*s, dtype=dt, device=dev)
    good = [e(3, 64, dt=torch.bfloat16), e(64), e(3, 4), e(3, 4, dt=torch.int32)]
    fn(good[0][:0], good[1], good[2][:0], good[3][:0], 0)
    for stream in (None, torch.cuda.current_stream()):
        fn(*good, 0, stream=stream)
        for at, bad in ((0, e(3, 64)), (0, e(2, 64, dt=torch.bfloat16)), (0, e(64, 3, dt=torch.bfloat16).t()), (1, e(63)), (1, e(64, dt=torch.float16)), (1, e(64, dev="cpu")), (2, e(3, 3)), (2, e(3, 4, dt=torch.int32)),
                        (3, e(3, 4)), (3, e(3, 4, dt=torch.int64)), (3, None), (2, None), (0, None)):
            args = list(good)
            args[at] = bad
            with pytest.raises(ValueError):
                fn(*args, 3, stream=stream)
        with pytest.raises(ValueError):
            fn(*good, 1 << 24, stream=stream)


def test_replayed():
    x, bias = _x(37, 256, 1).cuda(), _x(1, 256, 2, 0.1)[0].cuda()
    fn = build_grouped_topk_gating_module(256, 8, "f32", groups=8, topk_groups=4)
    w, ids = torch.empty(37, 8, device="cuda"), torch.empty(37, 8, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        fn(x, bias, w, ids, 37, stream=side)
    for k in range(3):
        x.copy_(_x(37, 256, 20 + k))
        bias.copy_(_x(1, 256, 30 + k, 0.1)[0])
        graph.replay()
        torch.cuda.synchronize()
        want, ww = _want(x, bias, 8, "sigmoid", 8, 4, "top2", True, 1.0)
        assert torch.equal(ids.cpu().long(), want) and ((w.double().cpu() - ww).abs() <= 11 * 2.0**-24 * ww).all()


def test_most_tokens():
    """2^24 - 1 tokens, logits of more than 2^32 bytes: tokens at the front, about the border and at the end."""
    t, e = (1 << 24) - 1, 130
    x = _x(65521, e, 3).bfloat16().cuda().repeat(-(-t // 65521), 1)[:t]
    bias = _x(1, e, 4, 0.1)[0]
    fn = build_grouped_topk_gating_module(e, 4, "bf16", scores="sigmoid", groups=10, topk_groups=3, group_score="top2", scale=1.5)
    ids, w = torch.full((t + 1, 4), -7, dtype=torch.int32, device="cuda"), torch.full((t + 1, 4), -7.0, device="cuda")
    print(f"route {t}x{e}", flush=True)
    fn(x, bias.cuda(), w, ids, t, stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    rows = torch.tensor([r for at in (0, 2**31 // (2 * e), 2**32 // (2 * e), t) for r in range(max(at - 40, 0), min(at + 40, t))], device="cuda")
    want, ww = _want(x[rows], bias, 4, "sigmoid", 10, 3, "top2", True, 1.5)
    assert torch.equal(ids[rows].cpu().long(), want)
    assert ((w[rows].double().cpu() - ww).abs() <= 7 * 2.0**-24 * ww.abs()).all()
    assert (ids[t] == -7).all() and (w[t] == -7).all()
