"""The norm, the grouped products and the 4-bit products one behind the other, as a decoder layer has them: residual addition and norm in front of a router and an expert layer, whose output a
projection with 4-bit weights takes back to the residual stream.

Every stage is checked against its definition in 64 bits on what the stage in front of it wrote, with the tolerances of its own tests, and the launches are captured into graphs and
replayed on other tokens.
"""

import pytest
import torch

from flydsl_amd import layout, quant, quant_device
from kernels.gemm.grouped_gemm import compile_grouped_gemm
from kernels.gemm.w4a16_gemm import compile_w4a16_gemm
from kernels.moe.topk_gating_softmax_kernel import build_topk_gating_softmax_module

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn
U = 2.0**-24


class Layer:
    def __init__(self, tokens, dim, inter, experts, topk, seed):
        g = torch.Generator().manual_seed(seed)
        rnd = lambda *s, std=1.0: std * torch.randn(*s, generator=g)
        self.tokens, self.dim, self.inter, self.experts, self.topk = tokens, dim, inter, experts, topk
        self.norm_w = (1 + rnd(dim, std=0.2)).bfloat16().cuda()
        self.router = rnd(experts, dim, std=0.05).bfloat16().cuda()
        w = rnd(experts, inter, dim, std=0.02)
        self.w_scale = (w.abs().amax(-1) / 448).cuda()
        self.w = (w / self.w_scale.cpu().unsqueeze(-1)).to(FP8).cuda()
        self.w_laid = layout.shuffle_weight(self.w.view(torch.int8)).view(FP8).contiguous()
        self.codes, self.scale, self.zero = quant.pergroup_w4_quant(rnd(dim, inter, std=0.02).cuda(), 64, True)
        self.down = layout.shuffle_weight_w4a16(self.codes), layout.shuffle_group_scales(self.scale), layout.shuffle_group_zeros(self.zero)
        self.gate = build_topk_gating_softmax_module(experts, topk, "bf16", True)
        self.grouped = compile_grouped_gemm(N=inter, K=dim, groups=experts)
        self.back = compile_w4a16_gemm(N=dim, K=inter, group_size=64, zero_points=True)
        b = lambda *s, dt=torch.bfloat16: torch.empty(*s, dtype=dt, device="cuda")
        rows = tokens * topk
        self.h, self.normed, self.q, self.qs = b(tokens, dim), b(tokens, dim), b(tokens, dim, dt=FP8), b(tokens, 1, dt=torch.float32)
        self.weights, self.ids, self.tei = b(tokens, topk, dt=torch.float32), b(tokens, topk, dt=torch.int32), b(tokens, topk, dt=torch.int32)
        self.up, self.out, self.mix = b(rows, inter), b(tokens, dim), b(tokens, inter)
        self.a, self.as_, self.offsets = b(rows, dim, dt=FP8), b(rows, 1, dt=torch.float32), torch.zeros(experts + 1, dtype=torch.int32, device="cuda")

    # the layer's launches of this library; what torch does between them is in run()
    def norm(self, x, residual, stream):
        quant_device.rmsnorm_quant(x, self.norm_w, 1e-6, residual=residual, residual_out=self.h, normed=self.normed, stream=stream, out=(self.q, self.qs))

    def experts_up(self, stream):
        self.grouped(self.up, self.a, self.w_laid, self.as_, self.w_scale, self.offsets, self.tokens * self.topk, stream)

    def project(self, stream):
        self.back(self.out, self.mix, *self.down, None, self.tokens, stream)

    def run(self, x, residual, stream, norm=None, experts_up=None, project=None):
        (norm or (lambda: self.norm(x, residual, stream)))()
        logits = self.normed @ self.router.t().contiguous()
        self.gate(logits, self.weights, self.ids, self.tei, self.tokens, stream=stream)
        flat = self.ids.view(-1).long()
        self.order = torch.argsort(flat, stable=True)
        self.offsets[1:] = torch.nn.functional.one_hot(flat, self.experts).cumsum(0)[-1].cumsum(0)
        token = self.order // self.topk
        self.a.copy_(self.q.view(torch.uint8)[token].view(FP8))
        self.as_.copy_(self.qs[token])
        (experts_up or (lambda: self.experts_up(stream)))()
        mixed = (torch.nn.functional.silu(self.up.float()) * self.weights.view(-1)[self.order].unsqueeze(1))
        back = torch.empty_like(mixed)
        back[self.order] = mixed
        self.mix.copy_(back.view(self.tokens, self.topk, self.inter).sum(1))
        (project or (lambda: self.project(stream)))()
        return self.out

    def check(self, x, residual):
        h = (x.float() + residual.float()).bfloat16()
        assert torch.equal(self.h, h)
        y = h.double() * self.norm_w.double() / (h.double().square().mean(-1, keepdim=True) + 1e-6).sqrt()
        tol = (self.dim / 64 + 40) * U
        assert ((self.normed.double() - y).abs() <= (2.0**-8 + tol) * y.abs()).all()
        s = y.abs().amax(-1, keepdim=True) / 448
        assert ((self.qs.double() - s).abs() <= tol * s).all()
        assert ((self.q.double() - y / s).abs() <= torch.clamp(2.0**-4 * (1 + 4 * U) * (y / s).abs(), min=2.0**-10) + 4 * U * (y / s).abs()).all()
        off = self.offsets.tolist()
        assert off[0] == 0 and off[-1] == self.tokens * self.topk
        for e in range(self.experts):
            r = slice(off[e], off[e + 1])
            assert (self.ids.view(-1)[self.order[r]] == e).all()
            if off[e] == off[e + 1]:
                continue
            scale = self.as_[r].double() * self.w_scale[e].double()
            a, w = self.a[r].double(), self.w[e].double().t().contiguous()
            want, mags = a @ w * scale, a.abs() @ w.abs() * scale
            assert ((self.up[r].double() - want).abs() <= 2.0**-8 * want.abs() + (self.dim + 3) * 2.0**-23 * 1.01 * mags).all()
        w = (self.codes.double() - self.zero.double().repeat_interleave(64, 1)) * self.scale.double().repeat_interleave(64, 1)
        a = self.mix.double()
        want = a @ w.t().contiguous()
        mags = a.abs().view(self.tokens, -1, 64).sum(-1) @ self.scale.double().t().contiguous()
        slack = 2 * 64 * 2.0**-23 * 31 * mags + (self.inter // 64 + 8) * 2.0**-23 * (a.abs() @ w.abs().t().contiguous())
        assert ((self.out.double() - want).abs() <= 2.0**-8 * (want.abs() + slack) + slack).all()


@pytest.mark.parametrize("tokens,dim,inter,experts,topk", [(1, 1024, 512, 8, 2), (13, 2048, 768, 16, 4), (64, 1024, 1536, 32, 8), (300, 512, 320, 8, 2)])
def test_layer(tokens, dim, inter, experts, topk):
    layer = Layer(tokens, dim, inter, experts, topk, seed=tokens)
    for seed in range(2):
        g = torch.Generator().manual_seed(seed)
        x, r = torch.randn(tokens, dim, generator=g).bfloat16().cuda(), (2 * torch.randn(tokens, dim, generator=g)).bfloat16().cuda()
        print(f"layer {tokens} {dim} {inter} {experts} {topk}", flush=True)
        layer.run(x, r, torch.cuda.current_stream())
        torch.cuda.synchronize()
        layer.check(x, r)


def test_layer_in_graphs():
    """The launches recorded once and replayed on other tokens and other groups."""
    tokens, dim = 20, 1024
    layer, eager = (Layer(tokens, dim, 512, 16, 4, seed=3) for _ in range(2))
    x, r = (torch.randn(tokens, dim, device="cuda").bfloat16() for _ in range(2))
    now = torch.cuda.current_stream()
    layer.run(x, r, now)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(now)
    replays = []
    for launch in (lambda: layer.norm(x, r, side), lambda: layer.experts_up(side), lambda: layer.project(side)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            launch()
        replays.append(graph.replay)
    for k in range(4):
        x.copy_(torch.randn(tokens, dim, device="cuda").bfloat16())
        layer.run(x, r, now, *replays)
        eager.run(x, r, now)
        torch.cuda.synchronize()
        assert torch.equal(layer.out.view(torch.int16), eager.out.view(torch.int16)), k
        eager.check(x, r)
