"""What the norm, the 4-bit products and the grouped products of this library are measured on.

Three operators of a decoder layer in serving:

  norm      residual addition, root-mean-square norm and per-row quantisation to fp8 / int8 (``quant_device.rmsnorm_quant``)
  w4        a few rows times 4-bit weights with a 16-bit scale (and a zero point) per group along K (``compile_w4a16_gemm``)
  grouped   rows sorted by expert times the expert's own weight, ragged sizes on the device (``compile_grouped_gemm``)

``own`` chooses between the library's kernels and plain torch operations in fp32 on the same inputs.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp8": torch.float8_e4m3fn, "int8": torch.int8}
QMAX = {"fp8": 448.0, "int8": 127.0}
EPS = 1e-6


def listed():
    return [
        # ---- norm ----
        # one token in decode, where the launch is everything
        dict(name="norm_t1", op="norm", rows=1, dim=4096, dtype="bf16", quant="fp8", residual=True, normed=False, strided=False),
        # a decode batch in fp16 for int8 products; no residual (the first norm of a model)
        dict(name="norm_t67_int8", op="norm", rows=67, dim=8192, dtype="fp16", quant="int8", residual=False, normed=False, strided=False),
        # a chunk of a prompt with a width that is no multiple of anything, x a slice of a wider buffer
        dict(name="norm_t777_odd", op="norm", rows=777, dim=2051, dtype="bf16", quant="fp8", residual=True, normed=False, strided=True),
        # prefill in front of an MoE layer: the router reads the 16-bit rows too
        dict(name="norm_t8192", op="norm", rows=8192, dim=8192, dtype="bf16", quant="fp8", residual=True, normed=True, strided=False),
        # ---- w4 ----
        # single-stream decode of one projection
        dict(name="w4_m1", op="w4", M=1, N=6144, K=4096, group=128, dtype="bf16", zeros=False, epilogue="none"),
        # a ragged little batch, the finest groups, zero points and a fused activation, sizes off every tile
        dict(name="w4_m5_g32", op="w4", M=5, N=1040, K=2080, group=32, dtype="fp16", zeros=True, epilogue="bias_silu"),
        # the widest feed-forward layer in batched decode
        dict(name="w4_m16_ffn", op="w4", M=16, N=28672, K=8192, group=128, dtype="bf16", zeros=True, epilogue="none"),
        # a larger decode batch
        dict(name="w4_m32_g64", op="w4", M=32, N=7168, K=2048, group=64, dtype="bf16", zeros=False, epilogue="none"),
        # ---- grouped ----
        # 64 tokens x top-8 on 32 experts: bound by the experts' weights
        dict(name="grouped_decode", op="grouped", rows=512, N=3584, K=4096, groups=32, empty=2, tail=0, dtype="fp8", out="bf16"),
        # a few adapters or experts in 16 bits, ragged, with rows behind the last group
        dict(name="grouped_ragged", op="grouped", rows=1500, N=2816, K=1088, groups=17, empty=3, tail=37, dtype="bf16", out="bf16"),
        # 1024 tokens x top-4 on 128 small experts in int8
        dict(name="grouped_many", op="grouped", rows=4096, N=2048, K=768, groups=128, empty=9, tail=0, dtype="int8", out="fp16"),
        # 4096 tokens x top-8 on 32 experts: bound by the matrix cores
        dict(name="grouped_prefill", op="grouped", rows=32768, N=4096, K=1536, groups=32, empty=0, tail=0, dtype="fp8", out="bf16"),
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of `step` between lo and hi, spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(hi // step, max(-(-lo // step), int(round(v / step)))) * step


def draw(rng):
    op = rng.choice(["norm", "w4", "grouped"])
    if op == "norm":
        dim = _log(rng, 256, 16384, rng.choice([1, 8, 8, 64]))
        rows = min(_log(rng, 1, 8192), 8192 * 8192 // dim)
        return dict(op=op, rows=rows, dim=dim, dtype=rng.choice(["bf16", "fp16"]), quant=rng.choice(["fp8", "fp8", "int8"]), residual=rng.random() < 0.7,
                    normed=rng.random() < 0.3, strided=rng.random() < 0.3)
    if op == "w4":
        group = rng.choice([32, 64, 128])
        n = _log(rng, 512, 28672, 16)
        k = min(_log(rng, 512, 16384, group), 28672 * 8192 // n // group * group)
        return dict(op=op, M=_log(rng, 1, 32), N=n, K=k, group=group, dtype=rng.choice(["bf16", "bf16", "fp16"]), zeros=rng.random() < 0.5,
                    epilogue=rng.choice(["none", "none", "bias", "bias_relu", "bias_silu", "bias_gelu"]))
    dtype = rng.choice(["fp8", "fp8", "int8", "bf16", "fp16"])
    groups = rng.choice([1, 4, 8, 17, 32, 64, 128])
    n, k = _log(rng, 512, 8192, 16), _log(rng, 256, 8192, 64)
    while groups * n * k > 32 * 4096 * 1536:  # the weights of the largest listed layer are the most
        n, k = n // 32 * 16, k // 128 * 64
    rows = max(groups, min(_log(rng, 1, 32768), int(32768 * 4096 * 1536 / (n * k * (2 if dtype in ("bf16", "fp16") else 1)))))
    return dict(op=op, rows=rows, N=n, K=k, groups=groups, empty=rng.randint(0, groups // 3), tail=rng.choice([0, 0, rng.randint(1, 200)]), dtype=dtype,
                out=rng.choice(["bf16", "fp16"]) if dtype in ("fp8", "int8") else dtype)


# ---- inputs ----


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, std=1.0, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(std).to(dtype)


def _rows(t, strided):
    """`t` as it is, or as the first columns of a wider buffer."""
    if not strided:
        return t
    wide = torch.zeros(t.shape[0], t.shape[1] + 61, dtype=t.dtype, device=t.device)
    wide[:, : t.shape[1]] = t
    return wide[:, : t.shape[1]]


def _prepare_norm(c, g):
    dt, rows, dim = DT[c["dtype"]], c["rows"], c["dim"]
    # activations with a few channels far above the rest, as a residual stream has them
    loud = 1.0 + 20.0 * (torch.rand(dim, generator=g, device="cuda") < 0.004)
    s = {"x": _rows((_randn(g, rows, dim, dtype=torch.float32) * loud).to(dt), c["strided"]),
         "weight": (1.0 + _randn(g, dim, std=0.2, dtype=torch.float32)).to(dt)}
    s["residual"] = (_randn(g, rows, dim, std=3.0, dtype=torch.float32) * loud).to(dt) if c["residual"] else None
    s["h"] = torch.empty(rows, dim, dtype=dt, device="cuda") if c["residual"] else None
    s["normed"] = torch.empty(rows, dim, dtype=dt, device="cuda") if c["normed"] else None
    s["q"], s["scale"] = torch.empty(rows, dim, dtype=DT[c["quant"]], device="cuda"), torch.empty(rows, 1, dtype=torch.float32, device="cuda")
    return s


def _prepare_w4(c, g):
    m, n, k, gs, dt = c["M"], c["N"], c["K"], c["group"], DT[c["dtype"]]
    # 4-bit weights as a quantiser leaves them: N(0, 0.02) spread over the codes of every group
    w = _randn(g, n, k // gs, gs, std=0.02, dtype=torch.float32)
    if c["zeros"]:
        lo, hi = w.amin(2, keepdim=True).clamp_(max=0), w.amax(2, keepdim=True).clamp_(min=0)
        scale = ((hi - lo) / 15).to(dt)
        zero = torch.round(-lo / scale.float()).clamp_(0, 15)
    else:
        scale = (w.abs().amax(2, keepdim=True) / 7.5).to(dt)
        zero = torch.full_like(scale, 8.0, dtype=torch.float32)
    codes = torch.round(w.div_(scale.float()).add_(zero)).clamp_(0, 15).to(torch.uint8).view(n, k)
    del w
    scale, zero = scale.view(n, k // gs), zero.to(torch.uint8).view(n, k // gs)
    s = {"codes": codes, "scale": scale, "zero": zero}
    # the same weights in the order the library multiplies them in, laid out once
    kp = -(-k // 128) * 128
    v = torch.nn.functional.pad(codes, (0, kp - k)).view(n // 16, 16, kp // 128, 4, 4, 4, 2)  # n / 16, n % 16, k / 128, dword, lane group, pair, half
    v = v.permute(0, 2, 4, 1, 3, 6, 5).contiguous()  # blocks of [lane group][row][dword][half][pair]
    s["w_laid"] = (v[..., 0::2] | (v[..., 1::2] << 4)).contiguous().view(n, kp // 2)
    s["scale_laid"] = scale.view(n // 16, 16, k // gs).transpose(1, 2).contiguous()
    z = zero.view(n // 16, 16, k // gs).transpose(1, 2).contiguous()
    s["zero_laid"] = (z[..., 0::2] | (z[..., 1::2] << 4)).contiguous() if c["zeros"] else None
    s["a"] = _randn(g, m, k, dtype=dt)
    s["bias"] = _randn(g, n, std=0.1, dtype=dt) if c["epilogue"] != "none" else None
    s["c"] = torch.empty(m, n, dtype=dt, device="cuda")
    return s


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


def _quant_rows(t, kind):
    s = t.abs().amax(-1, keepdim=True) / QMAX[kind]
    q = t / s
    return (q if kind == "fp8" else q.trunc()).to(DT[kind]), s.squeeze(-1).contiguous()


def _prepare_grouped(c, g, seed):
    dt, out, n, k, groups = DT[c["dtype"]], DT[c["out"]], c["N"], c["K"], c["groups"]
    sizes, rows = _sizes(c, seed), c["rows"] + c["tail"]
    s = {"rows": rows, "most": max(sizes)}
    x = _randn(g, rows, k, dtype=torch.float32)
    w = _randn(g, groups, n, k, std=0.02, dtype=torch.float32)
    if c["dtype"] in QMAX:
        s["a"], s["sa"] = _quant_rows(x, c["dtype"])
        s["w"], s["sb"] = _quant_rows(w, c["dtype"])
    else:
        s["a"], s["w"], s["sa"], s["sb"] = x.to(dt), w.to(dt), None, None
    del x, w
    piece = 16 // s["w"].element_size()  # preshuffled: 1 KB blocks of 16 rows x 64 bytes, 16 bytes a lane
    v = s["w"].view(torch.int8 if piece == 16 else torch.int16).view(groups, n // 16, 16, k // (4 * piece), 4, piece)
    s["w_laid"] = v.permute(0, 1, 3, 4, 2, 5).contiguous().view(groups, n, k).view(dt)
    s["offsets"] = torch.tensor([0] + sizes, dtype=torch.int64).cumsum(0).to(torch.int32).cuda()
    s["c"] = torch.zeros(rows, n, dtype=out, device="cuda")
    return s


def prepare(case, seed):
    g = _gen(seed)
    s = _prepare_norm(case, g) if case["op"] == "norm" else _prepare_w4(case, g) if case["op"] == "w4" else _prepare_grouped(case, g, seed)
    s["case"], s["stream"], s["keep"] = case, torch.cuda.current_stream(), {}
    return s


# ---- one pass ----


def _norm_outputs(c, q, scale, h, normed):
    # int8 rows as the values that their codes stand for
    out = {"q": q if c["quant"] == "fp8" else q.to(torch.float16), "scale": scale}
    if h is not None:
        out["residual"] = h
    if normed is not None:
        out["normed"] = normed
    return out


def _run_norm(s):
    c = s["case"]
    if own:
        from flydsl_amd import quant_device

        quant_device.rmsnorm_quant(s["x"], s["weight"], EPS, residual=s["residual"], quant_dtype=DT[c["quant"]], residual_out=s["h"], normed=s["normed"],
                                   stream=s["stream"], out=(s["q"], s["scale"]))
        return _norm_outputs(c, s["q"], s["scale"], s["h"], s["normed"])
    h = s["x"].float()
    dt = s["x"].dtype
    kept = None
    if c["residual"]:
        kept = (h + s["residual"].float()).to(dt)  # what the layers behind see
        h = kept.float()
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * s["weight"].float()
    scale = y.abs().amax(-1, keepdim=True) / QMAX[c["quant"]]
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    q = y / scale
    q = (q if c["quant"] == "fp8" else q.trunc()).to(DT[c["quant"]])
    return _norm_outputs(c, q, scale, kept, y.to(dt) if c["normed"] else None)


def _activate(y, kind):
    if kind == "bias_relu":
        return y.clamp(min=0)
    if kind == "bias_silu":
        return y * torch.sigmoid(y)
    if kind == "bias_gelu":
        return 0.5 * y * (1.0 + torch.tanh(0.7978845608 * (y + 0.044715 * y * y * y)))
    return y


def _run_w4(s):
    c = s["case"]
    if own:
        fn = s["keep"].get("fn")
        if fn is None:
            from flydsl_amd.kernels.gemm.w4a16_gemm import compile_w4a16_gemm

            fn = s["keep"]["fn"] = compile_w4a16_gemm(N=c["N"], K=c["K"], group_size=c["group"], in_dtype=c["dtype"], zero_points=c["zeros"], epilogue=c["epilogue"])
        fn(s["c"], s["a"], s["w_laid"], s["scale_laid"], s["zero_laid"], s["bias"], c["M"], s["stream"])
        return s["c"]
    n, k, gs = c["N"], c["K"], c["group"]
    w = (s["codes"].view(n, k // gs, gs).float() - s["zero"].float().unsqueeze(-1)) * s["scale"].float().unsqueeze(-1)
    y = torch.matmul(s["a"].float(), w.view(n, k).t())
    if s["bias"] is not None:
        y = _activate(y + s["bias"].float(), c["epilogue"])
    return y.to(s["a"].dtype)


def _run_grouped(s):
    c = s["case"]
    if own:
        fn = s["keep"].get("fn")
        if fn is None:
            from flydsl_amd.kernels.gemm.grouped_gemm import compile_grouped_gemm

            fn = s["keep"]["fn"] = compile_grouped_gemm(N=c["N"], K=c["K"], groups=c["groups"], in_dtype=c["dtype"], out_dtype=c["out"])
        fn(s["c"], s["a"], s["w_laid"], s["sa"], s["sb"], s["offsets"], s["rows"], s["stream"])
        return s["c"]
    # every group padded to the longest one, all of them in one batched product
    at = torch.arange(s["most"], device="cuda")
    row = (s["offsets"][:-1].long().unsqueeze(1) + at).clamp(max=s["rows"] - 1)
    y = torch.bmm(s["a"].float()[row], s["w"].float().transpose(1, 2))
    every = torch.arange(s["rows"], device="cuda")
    group = torch.searchsorted(s["offsets"][1:], every.int(), right=True).clamp(max=c["groups"] - 1)
    y = y[group, (every - s["offsets"][group]).clamp(max=s["most"] - 1)]
    if s["sa"] is not None:
        y = y * s["sa"].unsqueeze(1) * s["sb"][group]
    return torch.where((every < s["offsets"][-1]).unsqueeze(1), y.to(s["c"].dtype), s["c"])


def run(state):
    op = state["case"]["op"]
    return _run_norm(state) if op == "norm" else _run_w4(state) if op == "w4" else _run_grouped(state)


def work(case):
    c = case
    if c["op"] == "norm":
        n = c["rows"] * c["dim"]
        return {"bytes": n * (2 + 1 + (4 if c["residual"] else 0) + (2 if c["normed"] else 0)) + 2 * c["dim"] + 4 * c["rows"], "flops": 8 * n}
    if c["op"] == "w4":
        m, n, k = c["M"], c["N"], c["K"]
        scales = n * (k // c["group"])
        return {"bytes": n * k // 2 + 2 * scales + (scales // 2 if c["zeros"] else 0) + 2 * m * k + 2 * m * n + (2 * n if c["epilogue"] != "none" else 0), "flops": 2 * m * n * k}
    size = 1 if c["dtype"] in QMAX else 2
    live = min(c["groups"] - c["empty"], c["rows"])
    scales = 4 * (c["rows"] + live * c["N"]) if c["dtype"] in QMAX else 0
    return {"bytes": size * (c["rows"] * c["K"] + live * c["N"] * c["K"]) + 2 * c["rows"] * c["N"] + scales + 4 * (c["groups"] + 1), "flops": 2 * c["rows"] * c["N"] * c["K"]}


# ---- the definitions in 64 bits ----


def _exact_norm(c, s):
    h = s["x"].double()
    kept = None
    if c["residual"]:
        kept = (h + s["residual"].double()).to(s["x"].dtype)
        h = kept.double()
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS) * s["weight"].double()
    scale = y.abs().amax(-1, keepdim=True) / QMAX[c["quant"]]
    scale[scale == 0] = 1.0
    q = y / scale
    out = {"q": q.to(DT["fp8"]) if c["quant"] == "fp8" else q.trunc(), "scale": scale}
    if kept is not None:
        out["residual"] = kept.double()
    if c["normed"]:
        out["normed"] = y
    return out


def _exact_w4(c, s):
    parts = []
    for n0 in range(0, c["N"], 4096):  # a slice of the columns at a time: the weights take 8 bytes each here
        q, sc, z = (s[k][n0 : n0 + 4096].double() for k in ("codes", "scale", "zero"))
        w = (q - z.repeat_interleave(c["group"], 1)) * sc.repeat_interleave(c["group"], 1)
        parts.append(s["a"].double() @ w.t().contiguous())
    y = torch.cat(parts, 1)
    if s["bias"] is not None:
        y = _activate(y + s["bias"].double(), c["epilogue"])
    return y


def _exact_grouped(c, s, seed):
    y, at = s["c"].double(), 0
    for e, size in enumerate(_sizes(c, seed)):
        if size:
            part = s["a"][at : at + size].double() @ s["w"][e].double().t().contiguous()
            if s["sa"] is not None:
                part = part * s["sa"][at : at + size, None].double() * s["sb"][e].double()
            y[at : at + size] = part
            at += size
    return y


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_norm(case, s) if case["op"] == "norm" else _exact_w4(case, s) if case["op"] == "w4" else _exact_grouped(case, s, seed)
