"""The operators around the MoE block that are timed: routing rules, residual add + RMSNorm with 8-bit output, products of a few rows with
4-bit weights.  `own` False computes them from elementary torch operations, True through the package's entry points.

Sizes are those of the repository's configurations (rows of 2880, 32 and 128 experts) and generic ones.  Kinds of case:

  route    router logits [T, E] -> experts and weights of every token
  norm     x + delta, its RMSNorm, the result as e4m3 with scales ("mx": e8m0 per 32 values, "g128": fp32 per 128, "row": fp32 per row) or bf16
  linear   y = x W^T + bias, W in 4 bits ("mxfp4": e2m1 with e8m0 per 32 values, "int4": 0..15 less a zero point, bf16 scales per group),
           rows x in bf16 or as e4m3 with e8m0 scales per 32 values ("mx8")
"""
import importlib

import numpy as np
import torch

own = False


def pkg():
    return importlib.import_module("gpt-oss-amd_amd")


def route(T, E, K, scoring="sigmoid", bias=True, groups=1, keep=1, top=2, renorm=True, scale=1.0, name=None):
    c = dict(kind="route", T=T, E=E, K=K, scoring=scoring, bias=bias, groups=groups, keep=keep, top=top, renorm=renorm, scale=scale)
    return dict(c, name=name) if name else c


def norm(B, H, out, delta=True, name=None):
    c = dict(kind="norm", B=B, H=H, out=out, delta=delta)
    return dict(c, name=name) if name else c


def linear(B, N, K, fmt, rows="bf16", group=32, zeros=False, bias=True, name=None):
    c = dict(kind="linear", B=B, N=N, K=K, fmt=fmt, rows=rows, group=group, zeros=zeros, bias=bias)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one user generating: one token's experts among many in groups
        route(1, 256, 8, groups=8, keep=4, scale=2.5, name="route1_256_groups"),
        # a ragged decode batch of the larger configuration, probabilities over all experts
        route(61, 128, 4, scoring="softmax", bias=False, name="route61_128"),
        # a prefill chunk of the smaller configuration with a bias for balance
        route(4096, 32, 4, name="route4096_32"),
        # prompts of several users prefilled together
        route(16384, 256, 8, groups=8, keep=4, scale=2.5, name="route16384_256_groups"),
        # a single token's row, ready for an 8-bit product
        norm(1, 2880, "mx", name="norm1_mx"),
        # a decode batch, one scale a row
        norm(256, 2880, "row", name="norm256_row"),
        # prefill: an odd number of rows in bf16 for the library's products, and the largest in groups whose last is shorter
        norm(1000, 2880, "bf16", name="norm1000_bf16"),
        norm(16384, 2880, "g128", name="norm16384_g128"),
        # one token through a square projection
        linear(1, 2880, 2880, "mxfp4", name="linear1_mxfp4"),
        # a handful of users, group scales with zero points
        linear(7, 5760, 2880, "int4", group=64, zeros=True, name="linear7_int4_g64"),
        # a decode batch in 8 bits
        linear(64, 5760, 2880, "mxfp4", rows="mx8", name="linear64_mx8"),
        # the output matrix over a large vocabulary for a small batch
        linear(16, 131072, 2880, "mxfp4", bias=False, name="linear16_head"),
    ]


def draw(rng):
    def log(lo, hi):  # whole numbers spread over the logarithm
        return max(lo, min(hi, int(round(2 ** rng.uniform(np.log2(lo), np.log2(hi))))))

    kind = rng.choice(["route", "norm", "linear", "linear"])
    if kind == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        size = rng.randint(8, 64) if groups > 1 else rng.randint(8, 384)
        E = groups * size
        keep = rng.randint(1, groups)
        T = log(1, min(16384, 16384 * 256 // E))
        return route(T, E, rng.randint(1, 8), rng.choice(["sigmoid", "softmax"]), rng.choice([True, False]), groups, keep, rng.choice([1, 2]),
                     rng.choice([True, False]), rng.choice([1.0, 2.5]))
    if kind == "norm":
        H = 32 * log(2, 256)
        return norm(log(1, min(16384, 16384 * 2880 // H)), H, rng.choice(["mx", "mx", "g128", "row", "bf16"]), rng.choice([True, True, False]))
    fmt = rng.choice(["mxfp4", "int4"])
    K = 32 * log(8, 512)
    most = 131072 * 2880 // K
    N = 64 * log(4, most // 64) if fmt == "mxfp4" else log(200, most // 2)
    return linear(log(1, 64), N, K, fmt, rng.choice(["bf16", "bf16", "mx8"]), 32 if fmt == "mxfp4" else rng.choice([32, 64, 128]),
                  fmt == "int4" and rng.choice([True, False]), rng.choice([True, False]))


# ---- inputs -------------------------------------------------------------------------------------
def inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device="cuda") * scale

    def whole(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=torch.uint8)

    s = {"case": case}
    if case["kind"] == "route":
        # some experts are liked by all tokens, as in a trained router; the bias for balance works against it
        s["logits"] = normal(case["T"], case["E"]) + normal(1, case["E"], scale=0.5)
        s["bias"] = normal(case["E"], scale=0.05) if case["bias"] else None
    elif case["kind"] == "norm":
        # a residual stream with some values far larger than the others, and what a layer adds to it
        H = case["H"]
        s["x"] = normal(case["B"], H, scale=4.0) * torch.exp(normal(1, H))
        s["delta"] = normal(case["B"], H) if case["delta"] else None
        s["w"] = (1.0 + normal(H, scale=0.2)).bfloat16()
    else:
        B, N, K = case["B"], case["N"], case["K"]
        s["codes"] = whole(0, 256, N, K // 2)
        if case["fmt"] == "mxfp4":
            s["scales"] = whole(119, 128, N, K // 32)
        else:
            n = -(-K // case["group"])
            s["scales"] = (0.01 * torch.exp(normal(N, n, scale=0.3))).bfloat16()
            s["zeros"] = whole(5, 11, N, n) if case["zeros"] else None
        s["b"] = normal(N, scale=0.02).bfloat16() if case["bias"] else None
        x = normal(B, K)
        if case["rows"] == "bf16":
            s["x"], s["x_scales"] = x.bfloat16(), None
        else:
            e = torch.floor(torch.log2(x.view(B, K // 32, 32).abs().amax(-1))) - 7
            s["x"] = torch.ldexp(x.view(B, K // 32, 32), -e[..., None]).to(torch.float8_e4m3fn).view(torch.uint8).view(B, K)
            s["x_scales"] = (e + 127).to(torch.uint8)
    return s


def prepare(case, seed):
    s = inputs(case, seed)
    if own:  # what a program that uses the package holds besides: weights laid out once, output buffers, the routing rule
        p = pkg()
        dev = torch.device("cuda")
        s["p"] = p
        if case["kind"] == "route":
            T, K = case["T"], case["K"]
            s["rule"] = p.RouteRule(scoring=case["scoring"], balance_bias=s["bias"], n_groups=case["groups"], groups_per_token=case["keep"],
                                    group_top=case["top"], renormalize=case["renorm"], scale=case["scale"])
            s["v"] = torch.empty((T, K), dtype=torch.float32, device=dev)
            s["i"] = torch.empty((T, K), dtype=torch.int32, device=dev)
        elif case["kind"] == "norm":
            B, H, out = case["B"], case["H"], case["out"]
            s["x_out"] = torch.empty_like(s["x"])
            if out == "bf16":
                s["o"] = torch.empty((B, H), dtype=torch.bfloat16, device=dev)
            else:
                s["q"] = torch.empty((B, H), dtype=torch.uint8, device=dev)
                s["group"] = {"mx": 32, "g128": 128, "row": 0}[out]
                n = {"mx": H // 32, "g128": -(-H // 128), "row": 1}[out]
                s["q_scales"] = torch.empty((B, n), dtype=torch.uint8 if out == "mx" else torch.float32, device=dev)
        else:
            B, N, K = case["B"], case["N"], case["K"]
            s["y"] = torch.empty((B, N), dtype=torch.float32, device=dev)
            if case["fmt"] == "mxfp4":
                s["tiled"] = p.mxfp4_repack(s["codes"].view(1, N, K // 32, 16), s["scales"].view(1, N, K // 32))
            else:
                s["tiled"] = p.int4_repack(s["codes"], s["scales"], s["zeros"], case["group"])
    return s


# ---- one pass -----------------------------------------------------------------------------------
def run(s):
    c = s["case"]
    if own:
        return run_own(s, c)
    if c["kind"] == "route":
        return plain_route(s, c)
    if c["kind"] == "norm":
        return plain_norm(s, c)
    return plain_linear(s, c)


def run_own(s, c):
    p = s["p"]
    if c["kind"] == "route":
        p.route(s["v"], s["i"], s["logits"], c["T"], c["E"], c["K"], s["rule"])
        return s["v"], s["i"]
    if c["kind"] == "norm":
        if c["out"] == "bf16":
            p.add_rmsnorm(s["x_out"], s["x"], s["w"], c["B"], c["H"], delta=s["delta"], o_bf16=s["o"])
            return s["x_out"], s["o"]
        p.add_rmsnorm(s["x_out"], s["x"], s["w"], c["B"], c["H"], delta=s["delta"], q=s["q"], q_scales=s["q_scales"], q_group=s["group"])
        scales = s["q_scales"].view(torch.float8_e8m0fnu) if c["out"] == "mx" else s["q_scales"]
        return s["x_out"], s["q"].view(torch.float8_e4m3fn), scales
    if c["fmt"] == "mxfp4":
        blocks, scales = s["tiled"]
        p.linear_mxfp4(s["y"], s["x"], blocks, scales, c["B"], c["K"], c["N"], bias=s["b"], x_scales=s["x_scales"])
    else:
        codes, scales, zeros = s["tiled"]
        p.linear_int4(s["y"], s["x"], codes, scales, c["B"], c["K"], c["N"], c["group"], tiled_zeros=zeros, bias=s["b"], x_scales=s["x_scales"])
    return s["y"]


def plain_route(s, c):
    T, E, K, G = c["T"], c["E"], c["K"], c["groups"]
    l = s["logits"].double()  # scores a rounding apart decide between experts
    if c["scoring"] == "softmax":
        e = torch.exp(l - l.amax(-1, keepdim=True))
        score = (e / e.sum(-1, keepdim=True)).float()
    else:
        score = (1.0 / (1.0 + torch.exp(-l))).float()
    choice = score + s["bias"] if c["bias"] else score
    if G > 1:
        best = torch.sort(choice.view(T, G, E // G), dim=-1, descending=True).values
        value = best[..., 0] + best[..., 1] if c["top"] == 2 else best[..., 0]
        kept = torch.sort(value, dim=-1, descending=True, stable=True).indices[:, : c["keep"]]
        in_kept = torch.zeros((T, G), dtype=torch.bool, device=choice.device).scatter_(1, kept, True)
        choice = torch.where(in_kept[..., None], choice.view(T, G, E // G), float("-inf")).view(T, E)
    index = torch.sort(choice, dim=-1, descending=True, stable=True).indices[:, :K]
    w = torch.gather(score, 1, index).double()
    if c["renorm"]:
        w = w / w.sum(-1, keepdim=True)
    return (w * c["scale"]).float(), index.int()


def plain_norm(s, c):
    B, H, out = c["B"], c["H"], c["out"]
    x = s["x"] + s["delta"] if c["delta"] else s["x"].clone()
    # sums and products in 64 bits, as the 8-bit values next to a border need; the factor itself is a 32-bit number
    mean = x.square().double().sum(-1, keepdim=True) / H + float(np.float32(1e-5))
    inv = 1.0 / torch.sqrt(mean.float())
    y = (s["w"].double() * (inv.double() * x.double())).float()
    if out == "bf16":
        return x, y.bfloat16()
    n = {"mx": 32, "g128": 128, "row": H}[out]
    yg = torch.nn.functional.pad(y, (0, -H % n)).view(B, -1, n)
    amax = yg.abs().amax(-1)
    if out == "mx":
        # the smallest power of two that brings the largest value to 448 or below
        m, e = torch.frexp(amax)
        e = torch.clamp(torch.where(m > 0.875, e - 8, e - 9), min=-126)
        q = torch.ldexp(yg, -e[..., None].float())
        scale = (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)
    else:
        amax = torch.clamp(amax, min=2.0 ** -100)
        q = yg * (448.0 / amax)[..., None]
        scale = amax / 448.0
    return x, q.reshape(B, -1)[:, :H].contiguous().to(torch.float8_e4m3fn), scale


E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def plain_linear(s, c):
    B, N, K, n = c["B"], c["N"], c["K"], c["group"]
    codes = torch.stack((s["codes"] & 15, s["codes"] >> 4), -1).view(N, K)  # the low half of a byte comes first
    if c["fmt"] == "mxfp4":
        w = torch.tensor(E2M1, device=codes.device)[codes.int()]
        scale = torch.exp2(s["scales"].float() - 127.0)
    else:
        zero = s["zeros"].float().repeat_interleave(n, -1)[:, :K] if c["zeros"] else 8.0
        w = codes.float() - zero
        scale = s["scales"].float()
    w = w * scale.repeat_interleave(n, -1)[:, :K]
    if c["rows"] == "bf16":
        x = s["x"].float()
    else:
        x = s["x"].view(torch.float8_e4m3fn).float() * torch.exp2(s["x_scales"].float() - 127.0).repeat_interleave(32, -1)
    y = x @ w.t()
    return y + s["b"].float() if c["bias"] else y


def work(case):
    if case["kind"] == "route":
        T, E, K = case["T"], case["E"], case["K"]
        return {"bytes": 4 * T * E + 8 * T * K + (4 * E if case["bias"] else 0), "flops": 8 * T * E}
    if case["kind"] == "norm":
        B, H, out = case["B"], case["H"], case["out"]
        per_row = 8 * H + (4 * H if case["delta"] else 0) + {"mx": H + H // 32, "g128": H + 4 * -(-H // 128), "row": H + 4, "bf16": 2 * H}[out]
        return {"bytes": B * per_row + 2 * H, "flops": 6 * B * H}
    B, N, K = case["B"], case["N"], case["K"]
    n = -(-K // case["group"])
    scales = N * n * (1 if case["fmt"] == "mxfp4" else 3 if case["zeros"] else 2)
    rows = B * K * 2 if case["rows"] == "bf16" else B * K + B * K // 32
    return {"bytes": N * K // 2 + scales + rows + 4 * B * N + (2 * N if case["bias"] else 0), "flops": 2 * B * N * K}


# ---- from the definitions, in 64 bits --------------------------------------------------------------
def exact(case, seed):
    s = inputs(case, seed)
    if case["kind"] == "route":
        return exact_route(s, case)
    if case["kind"] == "norm":
        return exact_norm(s, case)
    return exact_linear(s, case)


def exact_route(s, c):
    T, E, K, G = c["T"], c["E"], c["K"], c["groups"]
    l = s["logits"].cpu().numpy().astype(np.float64)
    if c["scoring"] == "softmax":
        p = np.exp(l - l.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
    else:
        p = np.where(l >= 0, 1.0 / (1.0 + np.exp(-np.abs(l))), np.exp(-np.abs(l)) / (1.0 + np.exp(-np.abs(l))))
    # experts are chosen by scores and sums in 32 bits: that is part of the definition
    choice = p.astype(np.float32)
    if c["bias"]:
        choice = choice + s["bias"].cpu().numpy()
    rows = np.arange(T)[:, None]
    if G > 1:
        by_group = choice.reshape(T, G, E // G)
        ranked = -np.sort(-by_group, axis=2)
        value = ranked[:, :, 0] + ranked[:, :, 1] if c["top"] == 2 else ranked[:, :, 0]
        order = np.argsort(-value, axis=1, kind="stable")
        lost = np.zeros((T, G), dtype=bool)
        lost[rows, order[:, c["keep"]:]] = True
        choice = np.where(np.repeat(lost, E // G, axis=1), np.float32(-np.inf), choice)
    index = np.argsort(-choice, axis=1, kind="stable")[:, :K]
    w = p[rows, index]
    if c["renorm"]:
        w = w / w.sum(1, keepdims=True)
    return torch.from_numpy(w * c["scale"]), torch.from_numpy(index.astype(np.int32))


def to_e4m3(v):
    """The nearest e4m3 value (ties to even) of |v| up to 448 and a rounding, as 64-bit numbers."""
    power = torch.clamp(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -40))), min=-6.0)
    step = torch.exp2(power - 3.0)
    return torch.clamp(torch.round(v / step) * step, -448.0, 448.0)


def exact_norm(s, c):
    B, H, out = c["B"], c["H"], c["out"]
    x = s["x"].double()
    if c["delta"]:
        x = x + s["delta"].double()
    y = s["w"].double() * x * torch.rsqrt((x * x).mean(1, keepdim=True) + 1e-5)
    if out == "bf16":
        return x, y
    n = {"mx": 32, "g128": 128, "row": H}[out]
    groups = [y[:, k : k + n] for k in range(0, H, n)]
    amax = torch.stack([v.abs().amax(1) for v in groups], 1)
    if out == "mx":
        scale = torch.exp2(torch.clamp(torch.ceil(torch.log2(amax / 448.0)), min=-126.0))
    else:
        scale = amax / 448.0
    q = torch.cat([to_e4m3(v / scale[:, i : i + 1]) for i, v in enumerate(groups)], 1)
    return x, q, scale


def exact_linear(s, c):
    B, N, K, n = c["B"], c["N"], c["K"], c["group"]
    dev = s["codes"].device
    x = s["x"].double() if c["rows"] == "bf16" else torch.ldexp(s["x"].view(torch.float8_e4m3fn).double().view(B, K // 32, 32), s["x_scales"].double()[..., None] - 127).view(B, K)
    if c["fmt"] == "mxfp4":
        magnitude = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=dev)
    y = torch.zeros((B, N), dtype=torch.float64, device=dev)
    for k in range(0, K, n):  # a group of the contraction at a time
        m = min(n, K - k)
        byte = s["codes"][:, k // 2 : (k + m) // 2].long()
        code = torch.cat([(byte % 16)[..., None], (byte // 16)[..., None]], 2).view(N, m)
        if c["fmt"] == "mxfp4":
            w = magnitude[code % 8] * (1 - 2 * (code // 8)) * torch.exp2(s["scales"][:, k // n].double() - 127)[:, None]
        else:
            w = (code - (s["zeros"][:, k // n].long()[:, None] if c["zeros"] else 8)).double() * s["scales"][:, k // n].double()[:, None]
        y += x[:, k : k + m] @ w.t()
    if c["bias"]:
        y += s["b"].double()
    return y
