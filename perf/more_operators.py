"""What the router and the block-scaled fp8 products of this library are measured on.

Four operators of an expert layer whose weights and activations are e4m3 with one fp32 scale for each block of 128:

  route     router scores (sigmoid or softmax), a bias for balance, groups of experts, top-k, renormalised weights (``build_grouped_topk_gating_module``)
  quant     16- or 32-bit rows to e4m3 with a scale for every 128 columns, a gated activation in front (``quant_device.per_1x128_f8_quant``)
  block     rows times a weight with a scale for every 128 x 128 of it (``compile_blockscale_gemm``)
  experts   the same with rows sorted by expert and the expert's own weight, ragged sizes on the device (``compile_grouped_blockscale_gemm``)

``own`` chooses between the library's kernels and plain torch operations on the same inputs.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "f16": torch.float16, "f32": torch.float32}
FP8 = torch.float8_e4m3fn
QMAX = 448.0
BLOCK = 128


def listed():
    return [
        # ---- route ----
        # one token in decode: the launch is everything
        dict(name="route_t1", op="route", tokens=1, experts=256, topk=8, dtype="f32", scores="sigmoid", groups=8, topk_groups=4, group_score="top2", bias=True, renorm=True, scale=2.5),
        # a chunk of a prompt, 16-bit logits, softmax scores, the best expert speaks for its group, weights as they are
        dict(name="route_t777", op="route", tokens=777, experts=160, topk=6, dtype="bf16", scores="softmax", groups=8, topk_groups=3, group_score="max", bias=False, renorm=False, scale=16.0),
        # a long prefill
        dict(name="route_t16384", op="route", tokens=16384, experts=256, topk=8, dtype="f32", scores="sigmoid", groups=8, topk_groups=4, group_score="top2", bias=True, renorm=True, scale=2.5),
        # ---- quant ----
        # a decode batch's expert rows behind the gate-up product
        dict(name="quant_t40_gated", op="quant", rows=40, dim=1536, dtype="bf16", gated=True, strided=False),
        # a chunk of a prompt in fp16, a width that ends inside a block, x a slice of a wider buffer
        dict(name="quant_t777_odd", op="quant", rows=777, dim=2056, dtype="fp16", gated=False, strided=True),
        # prefill in front of the widest products
        dict(name="quant_t8192", op="quant", rows=8192, dim=8192, dtype="bf16", gated=False, strided=False),
        # ---- block ----
        # single-stream decode of one projection
        dict(name="block_m1", op="block", M=1, N=6144, K=4096, out="bf16"),
        # a ragged batch, N and K that end inside a block
        dict(name="block_m333_odd", op="block", M=333, N=2832, K=2240, out="fp16"),
        # prefill of one projection
        dict(name="block_m8192", op="block", M=8192, N=4096, K=4096, out="bf16"),
        # ---- experts ----
        # 64 tokens x top-8 on 32 experts: bound by the experts' weights
        dict(name="experts_decode", op="experts", rows=512, N=3584, K=4096, groups=32, empty=2, tail=0, out="bf16"),
        # ragged groups, sizes off the blocks, rows behind the last group
        dict(name="experts_ragged", op="experts", rows=1500, N=2816, K=1088, groups=17, empty=3, tail=37, out="bf16"),
        # 4096 tokens x top-8 on 32 experts: bound by the matrix cores
        dict(name="experts_prefill", op="experts", rows=32768, N=4096, K=1536, groups=32, empty=0, tail=0, out="bf16"),
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of `step` between lo and hi, spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(hi // step, max(-(-lo // step), int(round(v / step)))) * step


def draw(rng):
    op = rng.choice(["route", "quant", "block", "block", "experts", "experts"])
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8, 16])
        experts = groups * _log(rng, 8, 512 // groups)  # 8 to 512, groups of 8 and more
        topk_groups = rng.randint(1, groups)
        topk = rng.randint(1, min(16, experts // groups * topk_groups))
        bias = rng.random() < 0.6
        return dict(op=op, tokens=min(_log(rng, 1, 16384), 16384 * 256 // experts), experts=experts, topk=topk, dtype=rng.choice(["f32", "bf16", "f16"]), scores=rng.choice(["sigmoid", "softmax"]),
                    groups=groups, topk_groups=topk_groups, group_score="top2" if bias else "max", bias=bias, renorm=rng.random() < 0.6, scale=rng.choice([1.0, 2.5]))
    if op == "quant":
        gated = rng.random() < 0.4
        dim = _log(rng, 128, 16384 if not gated else 8192, rng.choice([1, 8, 64, 128]))
        return dict(op=op, rows=min(_log(rng, 1, 32768), 8192 * 8192 // dim // (2 if gated else 1)), dim=dim, dtype=rng.choice(["bf16", "bf16", "fp16"]), gated=gated, strided=rng.random() < 0.3)
    most = 8192 * 4096 * 4096
    if op == "block":
        n, k = _log(rng, 256, 28672, 16), _log(rng, 256, 16384, rng.choice([64, 128]))
        while n * k > 28672 * 8192:
            n = n // 32 * 16
        return dict(op=op, M=min(_log(rng, 1, 8192), most // (n * k)), N=n, K=k, out=rng.choice(["bf16", "bf16", "fp16"]))
    groups = rng.choice([1, 4, 8, 17, 32, 64, 128])
    n, k = _log(rng, 512, 8192, 16), _log(rng, 256, 8192, rng.choice([64, 128]))
    while groups * n * k > 32 * 4096 * 4096:
        n, k = n // 32 * 16, k // 128 * 64
    rows = max(groups, min(_log(rng, 1, 32768), 32768 * 4096 * 1536 // (n * k)))
    return dict(op=op, rows=rows, N=n, K=k, groups=groups, empty=rng.randint(0, groups // 3), tail=rng.choice([0, 0, rng.randint(1, 200)]), out=rng.choice(["bf16", "bf16", "fp16"]))


# ---- inputs ----


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(std)


def _prepare_route(c, g):
    t, e, k = c["tokens"], c["experts"], c["topk"]
    # logits of a trained router: some experts are liked by most tokens
    logits = _randn(g, t, e, std=1.5).add_(_randn(g, e, std=0.5))
    return {"logits": logits.to(DT[c["dtype"]]), "bias": _randn(g, e, std=0.1) if c["bias"] else None, "weights": torch.empty(t, k, dtype=torch.float32, device="cuda"),
            "ids": torch.empty(t, k, dtype=torch.int32, device="cuda")}


def _prepare_quant(c, g):
    rows, dim, dt = c["rows"], c["dim"], DT[c["dtype"]]
    cols = 2 * dim if c["gated"] else dim
    # activations with a few channels far above the rest
    x = (_randn(g, rows, cols) * (1.0 + 20.0 * (torch.rand(cols, generator=g, device="cuda") < 0.004))).to(dt)
    if c["strided"]:
        wide = torch.zeros(rows, cols + 56, dtype=dt, device="cuda")
        wide[:, :cols] = x
        x = wide[:, :cols]
    return {"x": x, "q": torch.empty(rows, dim, dtype=FP8, device="cuda"), "scale": torch.empty(-(-dim // BLOCK), rows, dtype=torch.float32, device="cuda")}


def _blocks(t, dims):
    """`t` with the given dimensions filled up with zeros to whole blocks and split into (blocks, 128)."""
    pad = []
    for d in reversed(range(t.dim())):
        pad += [0, -t.shape[d] % BLOCK if d in dims else 0]
    t = torch.nn.functional.pad(t, pad)
    shape = []
    for d in range(t.dim()):
        shape += [t.shape[d] // BLOCK, BLOCK] if d in dims else [t.shape[d]]
    return t.view(shape)


def _quant_a(x):
    """Rows as the quantiser in front of a product leaves them: e4m3 [rows, K] and scales [blocks of K, rows]."""
    b = _blocks(x, (1,))
    s = b.abs().amax(-1) / QMAX
    return (b / s.unsqueeze(-1)).view(x.shape[0], -1)[:, : x.shape[1]].to(FP8).contiguous(), s.t().contiguous()


def _quant_w(w):
    """A weight [.., N, K] as a checkpoint holds it: e4m3 and scales [.., blocks of N, blocks of K]."""
    n, k = w.shape[-2:]
    b = _blocks(w.view(-1, n, k), (1, 2))
    s = b.abs().amax((2, 4)) / QMAX
    q = (b / s[:, :, None, :, None]).view(-1, -(-n // BLOCK) * BLOCK, -(-k // BLOCK) * BLOCK)[:, :n, :k].to(FP8)
    return q.contiguous().view(w.shape), s.view(*w.shape[:-2], s.shape[-2], s.shape[-1]).contiguous()


def _laid(q):
    """In the order that the library multiplies weights in: 1 KB blocks of 16 rows x 64 bytes, 16 bytes a lane."""
    n, k = q.shape[-2:]
    return q.view(torch.int8).view(-1, n // 16, 16, k // 64, 4, 16).permute(0, 1, 3, 4, 2, 5).contiguous().view(q.shape).view(FP8)


def _prepare_block(c, g):
    a, sa = _quant_a(_randn(g, c["M"], c["K"]))
    w, sb = _quant_w(_randn(g, c["N"], c["K"], std=0.02))
    return {"a": a, "sa": sa, "w": w, "sb": sb, "w_laid": _laid(w), "c": torch.empty(c["M"], c["N"], dtype=DT[c["out"]], device="cuda")}


def _sizes(c, seed):
    """Rows of every group: all but `empty` of them have some, as a router that prefers some experts gives them."""
    r = random.Random(seed)
    live = r.sample(range(c["groups"]), min(c["groups"] - c["empty"], c["rows"]))
    likes = [math.exp(r.gauss(0, 0.5)) for _ in live]
    left, total, sizes = c["rows"] - len(live), sum(likes), [0] * c["groups"]
    for i, (e, w) in enumerate(zip(live, likes)):
        take = left if i + 1 == len(live) else min(left, int(round(left * w / total)))
        sizes[e], left, total = 1 + take, left - take, total - w
    return sizes


def _prepare_experts(c, g, seed):
    n, k, sizes, rows = c["N"], c["K"], _sizes(c, seed), c["rows"] + c["tail"]
    a, sa = _quant_a(_randn(g, rows, k))
    w, sb = _quant_w(_randn(g, c["groups"], n, k, std=0.02))
    offsets = torch.tensor([0] + sizes, dtype=torch.int64).cumsum(0).to(torch.int32).cuda()
    return {"a": a, "sa": sa, "w": w, "sb": sb, "w_laid": _laid(w), "offsets": offsets, "rows": rows, "most": max(sizes), "c": torch.zeros(rows, n, dtype=DT[c["out"]], device="cuda")}


def prepare(case, seed):
    g, op = _gen(seed), case["op"]
    s = _prepare_route(case, g) if op == "route" else _prepare_quant(case, g) if op == "quant" else _prepare_block(case, g) if op == "block" else _prepare_experts(case, g, seed)
    s["case"], s["stream"], s["keep"] = case, torch.cuda.current_stream(), {}
    return s


# ---- one pass ----


def _run_route(s):
    c = s["case"]
    if own:
        fn = s["keep"].get("fn")
        if fn is None:
            from flydsl_amd.kernels.moe.grouped_topk_gating import build_grouped_topk_gating_module

            fn = s["keep"]["fn"] = build_grouped_topk_gating_module(c["experts"], c["topk"], c["dtype"], scores=c["scores"], groups=c["groups"], topk_groups=c["topk_groups"],
                                                                    group_score=c["group_score"], renormalize=c["renorm"], scale=c["scale"])
        fn(s["logits"], s["bias"], s["weights"], s["ids"], c["tokens"], stream=s["stream"])
        return {"ids": s["ids"], "weights": s["weights"]}
    # in 64 bits: which of two scores is the larger is a whole number's worth
    x = s["logits"].double()
    if c["scores"] == "sigmoid":
        score = 1.0 / (1.0 + torch.exp(-x))
    else:
        score = torch.exp(x - x.amax(-1, keepdim=True))
        score = score / score.sum(-1, keepdim=True)
    chosen = score if s["bias"] is None else score + s["bias"].double()
    if c["topk_groups"] < c["groups"]:
        parts = chosen.view(c["tokens"], c["groups"], -1)
        worth = parts.amax(-1) if c["group_score"] == "max" else torch.sort(parts, dim=-1, descending=True)[0][..., :2].sum(-1)
        best = torch.sort(worth, dim=-1, descending=True, stable=True)[1][:, : c["topk_groups"]]
        keep = torch.zeros(c["tokens"], c["groups"], dtype=torch.bool, device="cuda").scatter_(1, best, True)
        chosen = torch.where(keep.unsqueeze(-1), parts, torch.full_like(parts, -math.inf)).view_as(chosen)
    ids = torch.sort(chosen, dim=-1, descending=True, stable=True)[1][:, : c["topk"]]
    w = torch.gather(score, 1, ids)
    if c["renorm"]:
        w = w / w.sum(-1, keepdim=True).clamp(min=1e-20)
    return {"ids": ids.int(), "weights": (w * c["scale"]).float()}


def _run_quant(s):
    c = s["case"]
    if own:
        from flydsl_amd import quant_device

        q, scale = quant_device.per_1x128_f8_quant(s["x"], gated=c["gated"], stream=s["stream"], out=(s["q"], s["scale"]))
        return {"q": q, "scale": scale}
    y = s["x"].float()
    if c["gated"]:
        gate, up = y[:, : c["dim"]], y[:, c["dim"] :]
        y = gate * torch.sigmoid(gate) * up
    b = _blocks(y, (1,))
    scale = b.abs().amax(-1) / QMAX
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    q = (b / scale.unsqueeze(-1)).view(c["rows"], -1)[:, : c["dim"]].to(FP8)
    return {"q": q.contiguous(), "scale": scale.t().contiguous()}


def _wide(q, s):
    """The values that e4m3 weights and their scales stand for, in 32 bits."""
    n, k = q.shape[-2:]
    return q.float() * s.repeat_interleave(BLOCK, -2)[..., :n, :].repeat_interleave(BLOCK, -1)[..., :k]


def _wide_rows(q, s):
    return q.float() * s.t().repeat_interleave(BLOCK, 1)[:, : q.shape[1]]


def _run_block(s):
    c = s["case"]
    if own:
        fn = s["keep"].get("fn")
        if fn is None:
            from flydsl_amd.kernels.gemm.blockscale_gemm import compile_blockscale_gemm

            fn = s["keep"]["fn"] = compile_blockscale_gemm(N=c["N"], K=c["K"], out_dtype=c["out"])
        fn(s["c"], s["a"], s["w_laid"], s["sa"], s["sb"], c["M"], s["stream"])
        return s["c"]
    return torch.matmul(_wide_rows(s["a"], s["sa"]), _wide(s["w"], s["sb"]).t()).to(s["c"].dtype)


def _run_experts(s):
    c = s["case"]
    if own:
        fn = s["keep"].get("fn")
        if fn is None:
            from flydsl_amd.kernels.gemm.blockscale_gemm import compile_grouped_blockscale_gemm

            fn = s["keep"]["fn"] = compile_grouped_blockscale_gemm(N=c["N"], K=c["K"], groups=c["groups"], out_dtype=c["out"])
        fn(s["c"], s["a"], s["w_laid"], s["sa"], s["sb"], s["offsets"], s["rows"], s["stream"])
        return s["c"]
    # every group padded to the longest one, all of them in one batched product
    at = torch.arange(s["most"], device="cuda")
    row = (s["offsets"][:-1].long().unsqueeze(1) + at).clamp(max=s["rows"] - 1)
    y = torch.bmm(_wide_rows(s["a"], s["sa"])[row], _wide(s["w"], s["sb"]).transpose(1, 2))
    every = torch.arange(s["rows"], device="cuda")
    group = torch.searchsorted(s["offsets"][1:], every.int(), right=True).clamp(max=c["groups"] - 1)
    y = y[group, (every - s["offsets"][group]).clamp(max=s["most"] - 1)]
    return torch.where((every < s["offsets"][-1]).unsqueeze(1), y.to(s["c"].dtype), s["c"])


def run(state):
    op = state["case"]["op"]
    return _run_route(state) if op == "route" else _run_quant(state) if op == "quant" else _run_block(state) if op == "block" else _run_experts(state)


def work(case):
    c, op = case, case["op"]
    if op == "route":
        n = c["tokens"] * c["experts"]
        return {"bytes": n * (4 if c["dtype"] == "f32" else 2) + 8 * c["tokens"] * c["topk"] + (4 * c["experts"] if c["bias"] else 0), "flops": 8 * n}
    if op == "quant":
        n = c["rows"] * c["dim"]
        return {"bytes": n * ((2 * 2 if c["gated"] else 2) + 1) + 4 * c["rows"] * -(-c["dim"] // BLOCK), "flops": n * (8 if c["gated"] else 3)}
    n, k, kb, nb = c["N"], c["K"], -(-c["K"] // BLOCK), -(-c["N"] // BLOCK)
    rows = c["M"] if op == "block" else c["rows"]
    live = 1 if op == "block" else min(c["groups"] - c["empty"], c["rows"])
    return {"bytes": rows * (k + 4 * kb + 2 * n) + live * (n * k + 4 * nb * kb) + (0 if op == "block" else 4 * (c["groups"] + 1)), "flops": 2 * rows * n * k}


# ---- the definitions in 64 bits ----


def _exact_route(c, s):
    x = s["logits"].double()
    p = torch.sigmoid(x) if c["scores"] == "sigmoid" else torch.softmax(x, 1)
    key = p.clone()
    if c["bias"]:
        key += s["bias"].double()
    t, e, g = c["tokens"], c["experts"], c["groups"]
    rows = torch.arange(t, device="cuda")
    if c["topk_groups"] < g:
        inside = key.view(t, g, e // g)
        first, at = inside.max(2)
        worth = first
        if c["group_score"] == "top2":
            rest = inside.clone()
            rest.scatter_(2, at.unsqueeze(2), -math.inf)
            worth = first + rest.max(2)[0]
        out = torch.ones(t, g, dtype=torch.bool, device="cuda")
        for _ in range(c["topk_groups"]):
            best = (worth == worth.max(1, keepdim=True)[0]).int().argmax(1)  # the first of equal ones
            out[rows, best] = False
            worth[rows, best] = -math.inf
        key[out.repeat_interleave(e // g, 1)] = -math.inf
    ids = torch.empty(t, c["topk"], dtype=torch.int64, device="cuda")
    for j in range(c["topk"]):
        best = (key == key.max(1, keepdim=True)[0]).int().argmax(1)
        ids[:, j] = best
        key[rows, best] = -math.inf
    w = p[rows.unsqueeze(1), ids]
    if c["renorm"]:
        w = w / torch.maximum(w.sum(1, keepdim=True), torch.tensor(1e-20, dtype=torch.float64, device="cuda"))
    return {"ids": ids.int(), "weights": w * c["scale"]}


def _exact_quant(c, s):
    y = s["x"].double()
    if c["gated"]:
        y = y[:, : c["dim"]] / (1 + torch.exp(-y[:, : c["dim"]])) * y[:, c["dim"] :]
    q, scales = torch.empty_like(y), []
    for k0 in range(0, c["dim"], BLOCK):
        part = y[:, k0 : k0 + BLOCK]
        scale = part.abs().amax(1) / QMAX
        scale[scale == 0] = 1.0
        q[:, k0 : k0 + BLOCK] = part / scale.unsqueeze(1)
        scales.append(scale)
    return {"q": q.to(FP8), "scale": torch.stack(scales)}


def _exact_product(a, sa, w, sb):
    """sum over the blocks of K of (a block times w block) times both scales, a block at a time"""
    y = torch.zeros(a.shape[0], w.shape[0], dtype=torch.float64, device="cuda")
    for i in range(sa.shape[0]):
        k = slice(i * BLOCK, min((i + 1) * BLOCK, a.shape[1]))
        cols = sb[:, i].double().repeat_interleave(BLOCK)[: w.shape[0]]
        y += (a[:, k].double() * sa[i].double().unsqueeze(1)) @ (w[:, k].double() * cols.unsqueeze(1)).t().contiguous()
    return y


def _exact_experts(c, s, seed):
    y, at = s["c"].double(), 0
    for e, size in enumerate(_sizes(c, seed)):
        if size:
            r = slice(at, at + size)
            y[r] = _exact_product(s["a"][r], s["sa"][:, r], s["w"][e], s["sb"][e])
            at += size
    return y


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "block":
        return _exact_product(s["a"], s["sa"], s["w"], s["sb"])
    return _exact_route(case, s) if op == "route" else _exact_quant(case, s) if op == "quant" else _exact_experts(case, s, seed)
