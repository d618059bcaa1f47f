"""Routing by groups, the block quantiser and the block-scaled products one behind the other, as an expert layer has them: every token's rows to its experts' gate-up product, the gate and its rounding
to fp8, the experts' second product, and beside them a shared expert through the dense products.

Every stage is checked against its definition in 64 bits on what the stage in front of it wrote, and the launches are captured into graphs and replayed on other tokens.

Tolerances are those of the stages' own tests, but for the products' (gated activations are further apart than normal ones).  The matrix instruction adds the products of eight consecutive elements of K in
one step, aligned to the largest of their exponents with 13 bits below it: next to 2^16 - 2^16 in one group of eight, 2^3 is kept whole and 2^2 is lost, while products of other groups are kept to 2^-24
(checked on the machine, product by product).  The largest's own six fraction bits fit, so a group is off by seven units of 2^-13 of its largest product at most, and that is at most the largest |a| times the
largest |w| of the eight; then come 15 additions of groups, the scales' product and its use, and an addition for every block, 2^-23 of the magnitudes each at most.
"""

import pytest
import torch

from flydsl_amd import layout, quant, quant_device
from kernels.gemm.blockscale_gemm import compile_blockscale_gemm, compile_grouped_blockscale_gemm
from kernels.moe.grouped_topk_gating import build_grouped_topk_gating_module

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn
U = 2.0**-24


def _wide(s, size):
    """[blocks, rows] scales as [rows, size]"""
    return s.double().t().repeat_interleave(128, 1)[:, :size]


class Layer:
    def __init__(self, tokens, dim, inter, experts, topk, groups, topk_groups, seed):
        g = torch.Generator().manual_seed(seed)
        rnd = lambda *s, std=1.0: std * torch.randn(*s, generator=g)
        self.tokens, self.dim, self.inter, self.experts, self.topk, self.groups, self.topk_groups = tokens, dim, inter, experts, topk, groups, topk_groups
        self.router, self.bias = rnd(experts, dim, std=dim**-0.5).cuda(), rnd(experts, std=0.1).cuda()
        self.w, self.laid, self.sw = {}, {}, {}
        for name, shape in (("gate_up", (experts, 2 * inter, dim)), ("down", (experts, dim, inter)), ("shared_gate_up", (1, 2 * inter, dim)), ("shared_down", (1, dim, inter))):
            w, s = quant.per_128x128_f8_quant(rnd(*shape, std=shape[-1] ** -0.5))
            self.w[name], self.sw[name] = w.cuda(), s.cuda()
            self.laid[name] = layout.shuffle_weight(self.w[name].view(torch.int8)).view(FP8).contiguous()
        self.route = build_grouped_topk_gating_module(experts, topk, "f32", scores="sigmoid", groups=groups, topk_groups=topk_groups, group_score="top2", renormalize=True, scale=2.5)
        sizes = {"gate_up": dict(N=2 * inter, K=dim), "down": dict(N=dim, K=inter)}
        self.grouped = {k: compile_grouped_blockscale_gemm(groups=experts, **v) for k, v in sizes.items()}
        self.dense = {k: compile_blockscale_gemm(**v) for k, v in sizes.items()}
        b = lambda *s, dt=torch.bfloat16: torch.empty(*s, dtype=dt, device="cuda")
        rows, kd, ki = tokens * topk, -(-dim // 128), -(-inter // 128)
        self.logits, self.weights, self.ids = b(tokens, experts, dt=torch.float32), b(tokens, topk, dt=torch.float32), b(tokens, topk, dt=torch.int32)
        self.q, self.qs = b(tokens, dim, dt=FP8), b(kd, tokens, dt=torch.float32)
        self.a, self.as_, self.offsets = b(rows, dim, dt=FP8), b(kd, rows, dt=torch.float32), torch.zeros(experts + 1, dtype=torch.int32, device="cuda")
        self.up, self.h, self.hs, self.out = b(rows, 2 * inter), b(rows, inter, dt=FP8), b(ki, rows, dt=torch.float32), b(rows, dim)
        self.sup, self.sh, self.shs, self.sout = b(tokens, 2 * inter), b(tokens, inter, dt=FP8), b(ki, tokens, dt=torch.float32), b(tokens, dim)

    # the layer's launches of this library; what torch does between them is in run()
    def front(self, x, stream):
        self.route(self.logits, self.bias, self.weights, self.ids, self.tokens, stream=stream)
        quant_device.per_1x128_f8_quant(x, stream=stream, out=(self.q, self.qs))

    def products(self, stream):
        rows = self.tokens * self.topk
        self.grouped["gate_up"](self.up, self.a, self.laid["gate_up"], self.as_, self.sw["gate_up"], self.offsets, rows, stream)
        quant_device.per_1x128_f8_quant(self.up, gated=True, stream=stream, out=(self.h, self.hs))
        self.grouped["down"](self.out, self.h, self.laid["down"], self.hs, self.sw["down"], self.offsets, rows, stream)
        self.dense["gate_up"](self.sup, self.q, self.laid["shared_gate_up"], self.qs, self.sw["shared_gate_up"], self.tokens, stream)
        quant_device.per_1x128_f8_quant(self.sup, gated=True, stream=stream, out=(self.sh, self.shs))
        self.dense["down"](self.sout, self.sh, self.laid["shared_down"], self.shs, self.sw["shared_down"], self.tokens, stream)

    def run(self, x, stream, front=None, products=None):
        self.logits.copy_(x.float() @ self.router.t().contiguous())
        (front or (lambda: self.front(x, stream)))()
        flat = self.ids.view(-1).long()
        self.order = torch.argsort(flat, stable=True)
        self.offsets[1:] = torch.nn.functional.one_hot(flat, self.experts).cumsum(0)[-1].cumsum(0)
        token = self.order // self.topk
        self.a.copy_(self.q.view(torch.uint8)[token].view(FP8))
        self.as_.copy_(self.qs[:, token])
        (products or (lambda: self.products(stream)))()
        back = torch.empty_like(self.out, dtype=torch.float32)
        back[self.order] = self.out.float() * self.weights.view(-1)[self.order].unsqueeze(1)
        return back.view(self.tokens, self.topk, self.dim).sum(1) + self.sout.float()

    def check(self, x):
        # (comparisons in 64 bits on both sides, as the routing's own tests have them)
        s = 1 / (1 + torch.exp(-self.logits.double()))
        c = s + self.bias.double()
        worth = c.view(self.tokens, self.groups, -1).topk(2, -1)[0].sum(-1)
        keep = torch.zeros_like(worth, dtype=torch.bool).scatter_(1, worth.topk(self.topk_groups, 1)[1], True).repeat_interleave(self.experts // self.groups, 1)
        ids = c.masked_fill(~keep, -float("inf")).topk(self.topk, 1)[1]
        assert torch.equal(self.ids.long(), ids)
        w = s.gather(1, ids)
        w = w / w.sum(1, keepdim=True) * 2.5
        assert ((self.weights.double() - w).abs() <= (self.topk + 3) * U * w).all()
        want, scale = quant.per_1x128_f8_quant(x.cpu())
        assert torch.equal(self.q.view(torch.uint8).cpu(), want.view(torch.uint8)) and torch.equal(self.qs.cpu(), scale)
        off = self.offsets.tolist()
        assert off[0] == 0 and off[-1] == self.tokens * self.topk
        for e in range(self.experts):
            r = slice(off[e], off[e + 1])
            assert (self.ids.view(-1)[self.order[r]] == e).all()
            self.check_product(self.up[r], self.a[r], self.as_[:, r], "gate_up", e)
            self.check_product(self.out[r], self.h[r], self.hs[:, r], "down", e)
        self.check_product(self.sup, self.q, self.qs, "shared_gate_up", 0)
        self.check_product(self.sout, self.sh, self.shs, "shared_down", 0)
        self.check_gate(self.up, self.h, self.hs)
        self.check_gate(self.sup, self.sh, self.shs)

    def check_product(self, c, a, sa, name, e):
        n, k = self.w[name].shape[1:]
        av = a.double() * _wide(sa, k)
        wv = (self.w[name][e].double() * self.sw[name][e].double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]).t().contiguous()
        largest = av.abs().view(-1, k // 8, 8).amax(-1) @ wv.abs().view(k // 8, 8, n).amax(1)
        want, slack = av @ wv, 7 * 2.0**-13 * largest + (16 + 3 + -(-k // 128)) * 2.0**-23 * (av.abs() @ wv.abs())
        assert ((c.double() - want).abs() <= 2.0**-8 * (want.abs() + slack) + slack).all()

    def check_gate(self, up, q, s):
        g, u = up.double().split(self.inter, 1)
        y = g / (1 + torch.exp(-g)) * u
        b = torch.nn.functional.pad(y, (0, -self.inter % 128)).view(y.shape[0], -1, 128)
        want = b.abs().amax(-1) / 448
        want[want == 0] = 1
        assert ((s.double().t() - want).abs() <= 11.5 * U * want).all()
        v = (b / want.unsqueeze(-1)).view(y.shape[0], -1)[:, : self.inter]
        assert ((q.double() - v).abs() <= torch.clamp(2.0**-4 * v.abs(), min=2.0**-10) * (1 + 2.0**-4) + 24 * U * v.abs()).all()


def _tokens(tokens, dim, seed):
    return torch.randn(tokens, dim, generator=torch.Generator().manual_seed(seed)).bfloat16().cuda()


@pytest.mark.parametrize("tokens,dim,inter,experts,topk,groups,topk_groups", [(1, 1024, 512, 16, 4, 4, 2), (7, 832, 320, 24, 6, 3, 2), (64, 1024, 256, 64, 8, 8, 4), (300, 576, 704, 8, 2, 4, 2)])
def test_layer(tokens, dim, inter, experts, topk, groups, topk_groups):
    layer = Layer(tokens, dim, inter, experts, topk, groups, topk_groups, seed=tokens)
    for seed in range(2):
        x = _tokens(tokens, dim, seed)
        print(f"layer {tokens} {dim} {inter} {experts} {topk}", flush=True)
        layer.run(x, torch.cuda.current_stream() if seed else None)
        torch.cuda.synchronize()
        layer.check(x)


def test_layer_in_graphs():
    """The launches recorded once and replayed on other tokens and other groups."""
    tokens, dim = 20, 1024
    layer, eager = (Layer(tokens, dim, 384, 16, 4, 4, 2, seed=3) for _ in range(2))
    x = _tokens(tokens, dim, 0)
    layer.run(x, torch.cuda.current_stream())
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    for part in (lambda: layer.front(x, side), lambda: layer.products(side)):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side):
            part()
    for seed in range(1, 4):
        x.copy_(_tokens(tokens, dim, seed))
        got = layer.run(x, None, front=graphs[0].replay, products=graphs[1].replay)
        want = eager.run(x, torch.cuda.current_stream())
        torch.cuda.synchronize()
        layer.check(x)
        for a, b in ((layer.ids, eager.ids), (layer.weights, eager.weights), (layer.up, eager.up), (layer.out, eager.out), (layer.sout, eager.sout), (got, want)):
            assert torch.equal(a, b)


def test_two_layers_at_once():
    """Two layers of the same sizes on two streams: no launch keeps anything that another's could meet."""
    layers = [Layer(96, 1024, 256, 16, 4, 4, 2, seed=5 + i) for i in range(2)]
    xs = [_tokens(96, 1024, i) for i in range(2)]
    for layer, x in zip(layers, xs):
        layer.run(x, torch.cuda.current_stream())
    torch.cuda.synchronize()
    want = [(l.up.clone(), l.out.clone(), l.sout.clone()) for l in layers]
    streams = [torch.cuda.Stream() for _ in layers]
    for _ in range(20):
        for layer, x, stream in zip(layers, xs, streams):
            layer.front(x, stream)
            layer.products(stream)
    torch.cuda.synchronize()
    for layer, x, kept in zip(layers, xs, want):
        layer.check(x)
        assert all(torch.equal(a, b) for a, b in zip((layer.up, layer.out, layer.sout), kept))
