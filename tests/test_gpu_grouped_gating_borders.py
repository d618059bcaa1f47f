"""GPU tests of the routing by groups where its choice in 32 bits meets its definition in 64: zeros of both signs at the border of the top-k.

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
    """Logits times a mask leave zeros of both signs, and the last experts taken are among them: about a tenth of the logits are above zero, half of them zeros; 9001 tokens share wavefronts by twos."""
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
