"""The operators between a layer's projections and behind its output matrix that are timed: rotary embedding with the write into a paged
cache, attention of single tokens over that cache, attention over packed prompts, log probabilities of tokens.  `own` False computes
them from elementary torch operations, True through the package's entry points.

Sizes are generic ones and those of the repository's configurations (heads of 64, windows of 128, rope theta 150000).  Kinds of case:

  write     rows of a query/key/value projection [T, (Hq + 2 Hkv) D] -> rotated queries, keys and values in the cache (bf16, or "mx8": e4m3
            with e8m0 scales per 32 values) and, for prompts, keys and values as packed rows too
  decode    one query a sequence over the pages that its table lists
  prefill   prompts of different lengths one after another, causal; with `context` keys in front of each prompt's own
  logprobs  logits [T, V] -> log probability of a token a row, entropy, the largest alternatives
"""
import importlib
import math
import random

import numpy as np
import torch

own = False


def pkg():
    return importlib.import_module("gpt-oss-amd_amd")


def write(T, Hq, Hkv, D, fmt="bf16", page=64, prompt=False, rows="f32", name=None):
    c = dict(kind="write", T=T, Hq=Hq, Hkv=Hkv, D=D, fmt=fmt, page=page, prompt=prompt, rows=rows)
    return dict(c, name=name) if name else c


def decode(B, longest, Hq, Hkv, D, fmt="bf16", page=64, window=0, sinks=True, ragged=False, mix=1, name=None):
    c = dict(kind="decode", B=B, longest=longest, Hq=Hq, Hkv=Hkv, D=D, fmt=fmt, page=page, window=window, sinks=sinks, ragged=ragged, mix=mix)
    return dict(c, name=name) if name else c


def prefill(B, longest, Hq, Hkv, D, window=0, sinks=True, ragged=False, context=0, mix=1, name=None):
    c = dict(kind="prefill", B=B, longest=longest, Hq=Hq, Hkv=Hkv, D=D, window=window, sinks=sinks, ragged=ragged, context=context, mix=mix)
    return dict(c, name=name) if name else c


def logprobs(T, V, top, rows="f32", name=None):
    c = dict(kind="logprobs", T=T, V=V, top=top, rows=rows)
    return dict(c, name=name) if name else c


def lengths(case):
    """The sequences' lengths: all the longest, or spread over the logarithm with the longest among them."""
    if not case["ragged"]:
        return [case["longest"]] * case["B"]
    r = random.Random(case["mix"])
    some = [max(1, int(round(case["longest"] ** r.random()))) for _ in range(case["B"] - 1)]
    some.insert(r.randrange(case["B"]), case["longest"])
    return some


def listed():
    return [
        # a decode batch's new tokens into an 8-bit cache
        write(64, 64, 8, 64, fmt="mx8", name="write64_mx8"),
        # prompts of several users: the cache for later, packed rows for the attention that follows
        write(8192, 64, 8, 64, prompt=True, name="write8192_prompt"),
        # a handful of users in a layer with a short window
        decode(7, 4000, 64, 8, 64, window=128, ragged=True, name="decode7_window"),
        # one user with a long document
        decode(1, 131072, 64, 8, 64, name="decode1_128k"),
        # a batch in full flow: some have just begun, some have long histories
        decode(64, 16384, 64, 8, 64, ragged=True, name="decode64_ragged"),
        # a large batch over an 8-bit cache, larger heads, no sinks
        decode(128, 4096, 32, 8, 128, fmt="mx8", sinks=False, name="decode128_mx8"),
        # one short prompt of an odd length: what a user waits for
        prefill(1, 333, 64, 8, 64, name="prefill333"),
        # prompts of many lengths in a layer with a short window
        prefill(16, 3000, 64, 8, 64, window=128, ragged=True, name="prefill16_window"),
        # a long prompt
        prefill(1, 8192, 64, 8, 64, name="prefill8192"),
        # larger heads without sinks, the second part of each prompt: 2048 tokens behind 2048 that came before
        prefill(4, 2048, 32, 4, 128, sinks=False, context=2048, name="prefill4_d128"),
        # one generated token and its alternatives, as an interface shows them
        logprobs(1, 131072, 20, name="logprobs1_top20"),
        # scoring the tokens of a text, logits from a library product
        logprobs(1000, 200000, 5, rows="bf16", name="logprobs1000_bf16"),
    ]


def draw(rng):
    def log(lo, hi):  # whole numbers spread over the logarithm
        return max(lo, min(hi, int(round(2 ** rng.uniform(np.log2(lo), np.log2(max(lo, hi)))))))

    kind = rng.choice(["write", "decode", "decode", "prefill", "prefill", "logprobs"])
    D = rng.choice([64, 64, 128])
    Hkv = rng.choice([1, 2, 4, 8])
    Hq = Hkv * rng.choice([1, 3, 4, 8, 8, 16])
    page = rng.choice([16, 32, 64, 128, 256])
    window = rng.choice([0, 0, 128, log(1, 1024)])
    sinks = rng.choice([True, False])
    if kind == "write":
        T = log(1, 8192 * 80 * 64 // max(80 * 64, (Hq + 2 * Hkv) * D))
        return write(T, Hq, Hkv, D, rng.choice(["bf16", "mx8"]), page, rng.choice([True, False]), rng.choice(["f32", "f32", "bf16"]))
    if kind == "decode":
        fmt = rng.choice(["bf16", "mx8"])
        B = log(1, 256)
        keys = 4 * 131072 * 8 * 64 // (B * Hkv * D)  # up to the cache of the large batch
        return decode(B, log(1, max(1, min(131072, keys))), Hq, Hkv, D, fmt, page, window, sinks, rng.choice([True, True, False]), rng.randrange(1 << 20))
    if kind == "prefill":
        B = log(1, 16)
        context = rng.choice([0, 0, 0, log(1, 2048)])
        most = 64 * 8192 * 8192 // 2 * 64 // (Hq * D * B)  # longest^2 / 2 + longest * context pairs, as many as the long prompt has
        longest = max(1, int(math.sqrt(2 * most + context ** 2) - context))
        return prefill(B, log(1, min(8192, longest)), Hq, Hkv, D, window, sinks, rng.choice([True, True, False]), context, rng.randrange(1 << 20))
    rows = rng.choice(["f32", "bf16"])
    V = log(64, 262144)
    return logprobs(log(1, max(1, min(4096, 1000 * 200000 // (2 * V)))), V, rng.choice([0, 1, 5, 20, 32]), rows)


# ---- inputs -------------------------------------------------------------------------------------
def to_mx8(x):
    """e4m3 codes and e8m0 scales per 32 values, as torch's types, of fp32 values: the smallest power of two that leaves 448 or less."""
    g = x.reshape(*x.shape[:-1], -1, 32)
    amax = g.abs().amax(-1)
    m, e = torch.frexp(amax)
    e = torch.where(m > 0.875, e - 8, e - 9)
    e = torch.where(amax == 0, -126, torch.clamp(e, min=-126))
    codes = torch.ldexp(g, -e[..., None].float()).to(torch.float8_e4m3fn).reshape(x.shape)
    return codes, (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device="cuda") * scale

    def whole(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    s = {"case": case}
    if case["kind"] == "logprobs":
        # a few tokens stand out from the many
        T, V = case["T"], case["V"]
        l = normal(T, V, scale=2.0)
        l.add_(torch.exp(normal(1, V, scale=0.5)))
        s["logits"] = l if case["rows"] == "f32" else l.bfloat16()
        s["tokens"] = torch.randint(0, V, (T,), generator=g, device="cuda", dtype=torch.int32)
        return s
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    if case["kind"] == "write":
        T, page = case["T"], case["page"]
        # keys have channels that are larger than others
        rows = normal(T, Hq + 2 * Hkv, D) * torch.exp(normal(1, 1, D, scale=0.5))
        s["qkv"] = rows.view(T, -1) if case["rows"] == "f32" else rows.view(T, -1).bfloat16()
        s["positions"] = torch.randint(0, 131072, (1,), generator=g, device="cuda", dtype=torch.int32) + torch.arange(T, device="cuda", dtype=torch.int32)
        s["inv_freq"] = (150000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)).float().cuda()
        s["rope_scale"] = 0.1 * math.log(32.0) + 1.0
        n_pages = -(-T // page) + 3
        s["slots"] = torch.randperm(n_pages * page, generator=g, device="cuda")[:T].int() if not case["prompt"] else (
            torch.randperm(n_pages, generator=g, device="cuda").int()[:, None] * page + torch.arange(page, device="cuda", dtype=torch.int32)).view(-1)[:T].contiguous()
        cache = [torch.zeros((n_pages, Hkv, page, D), device="cuda") for _ in range(2)]
    elif case["kind"] == "decode":
        lens, page = lengths(case), case["page"]
        per = [-(-n // page) for n in lens]
        n_pages = sum(per) + 3
        free = torch.randperm(n_pages, generator=g, device="cuda").int()
        table = np.zeros((len(lens), max(per)), np.int64)
        at = 0
        for b, n in enumerate(per):
            table[b, :n] = np.arange(at, at + n)
            at += n
        s["table"] = free[torch.from_numpy(table).cuda()].contiguous()
        s["lens"] = whole(lens)
        s["q"] = normal(len(lens), Hq, D).bfloat16()
        cache = [normal(n_pages, Hkv, page, D), normal(n_pages, Hkv, page, D)]
        cache[0] *= torch.exp(normal(1, 1, 1, D, scale=0.5))
    else:
        lens = lengths(case)
        tq, tk = sum(lens), sum(lens) + len(lens) * case["context"]
        s["q"] = normal(tq, Hq, D).bfloat16()
        s["k"] = (normal(tk, Hkv, D) * torch.exp(normal(1, 1, D, scale=0.5))).bfloat16()
        s["v"] = normal(tk, Hkv, D).bfloat16()
        s["q_starts"] = whole(np.concatenate([[0], np.cumsum(lens)]).tolist())
        s["k_starts"] = whole(np.concatenate([[0], np.cumsum(np.array(lens) + case["context"])]).tolist())
        s["longest"] = max(lens), max(lens) + case["context"]
        cache = None
    if cache is not None:
        if case["fmt"] == "mx8":
            s["k"], s["k_scales"] = to_mx8(cache[0])
            s["v"], s["v_scales"] = to_mx8(cache[1])
        else:
            s["k"], s["v"] = cache[0].bfloat16(), cache[1].bfloat16()
            s["k_scales"] = s["v_scales"] = None
    if case["kind"] != "write":
        s["sinks"] = normal(Hq).bfloat16() if case["sinks"] else None
        s["scale"] = D ** -0.5
    return s


def prepare(case, seed):
    s = inputs(case, seed)
    if own:  # what a program that uses the package holds besides: the cache's handle, output buffers, a workspace
        p = pkg()
        s["p"] = p

        def empty(*shape, dtype=torch.float32):
            return torch.empty(shape, dtype=dtype, device="cuda")

        bf16 = torch.bfloat16
        if case["kind"] == "logprobs":
            T, top = case["T"], case["top"]
            s["logp"], s["entropy"] = empty(T), empty(T)
            s["top_logp"], s["top_index"] = (empty(T, top), empty(T, top, dtype=torch.int32)) if top else (None, None)
            s["workspace"] = empty(p.token_logprobs_workspace_bytes(T, case["V"], top), dtype=torch.uint8)
            return s
        Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
        if case["kind"] != "prefill":
            s["cache"] = p.KvCache(s["k"], s["v"], s["k_scales"], s["v_scales"])
        if case["kind"] == "write":
            T = case["T"]
            s["q"] = empty(T, Hq, D, dtype=bf16)
            s["k_rows"], s["v_rows"] = (empty(T, Hkv, D, dtype=bf16), empty(T, Hkv, D, dtype=bf16)) if case["prompt"] else (None, None)
        else:
            s["out"] = torch.empty_like(s["q"])
            if case["kind"] == "decode":
                s["workspace"] = empty(p.attention_decode_workspace_bytes(case["B"], Hq, Hkv, D), dtype=torch.uint8)
    return s


# ---- one pass -----------------------------------------------------------------------------------
def run(s):
    c = s["case"]
    if own:
        return run_own(s, c)
    return {"write": plain_write, "decode": plain_decode, "prefill": plain_prefill, "logprobs": plain_logprobs}[c["kind"]](s, c)


def run_own(s, c):
    p = s["p"]
    if c["kind"] == "logprobs":
        p.token_logprobs(s["logits"], s["tokens"], c["T"], c["V"], logprobs=s["logp"], entropy=s["entropy"], top_logprobs=s["top_logp"],
                         top_indices=s["top_index"], top_k=c["top"], workspace=s["workspace"])
        return (s["logp"], s["entropy"], s["top_logp"], s["top_index"]) if c["top"] else (s["logp"], s["entropy"])
    Hq, Hkv, D = c["Hq"], c["Hkv"], c["D"]
    if c["kind"] == "write":
        p.rope_kv_write(s["q"], s["qkv"], s["positions"], s["inv_freq"], c["T"], Hq, Hkv, D, rope_scale=s["rope_scale"], k=s["k_rows"], v=s["v_rows"],
                        cache=s["cache"], slots=s["slots"])
        out = [s["q"], s["k"], s["v"]]
        if c["fmt"] == "mx8":
            out += [s["k_scales"], s["v_scales"]]
        return out + [s["k_rows"], s["v_rows"]] if c["prompt"] else out
    if c["kind"] == "decode":
        p.attention_decode(s["out"], s["q"], s["cache"], s["table"], s["lens"], c["B"], Hq, s["scale"], s["workspace"], window=c["window"],
                           sinks=s["sinks"])
    else:
        p.attention_prefill(s["out"], s["q"], s["k"], s["v"], s["q_starts"], s["k_starts"], c["B"], Hq, Hkv, D, s["scale"], window=c["window"],
                            sinks=s["sinks"])
    return s["out"]


def plain_write(s, c):
    T, Hq, Hkv, D, page = c["T"], c["Hq"], c["Hkv"], c["D"], c["page"]
    angle = s["positions"].double()[:, None] * s["inv_freq"].double()  # far positions: in 32 bits nothing of the angle would be left
    cos, sin = ((f(angle) * s["rope_scale"]).float()[:, None] for f in (torch.cos, torch.sin))
    x = s["qkv"].float().view(T, Hq + 2 * Hkv, D)
    a, b = x[:, : Hq + Hkv, : D // 2], x[:, : Hq + Hkv, D // 2 :]
    r = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    q, k, v = r[:, :Hq].bfloat16(), r[:, Hq:], x[:, Hq + Hkv :]
    at, off = (s["slots"] // page).long(), (s["slots"] % page).long()

    def put(rows, codes, scales):
        new, new_scales = to_mx8(rows)
        codes.view(torch.uint8)[at, :, off] = new.view(torch.uint8)
        scales.view(torch.uint8)[at, :, off] = new_scales.view(torch.uint8)

    if c["fmt"] == "mx8":
        put(k, s["k"], s["k_scales"])
        put(v, s["v"], s["v_scales"])
        out = [q, s["k"], s["v"], s["k_scales"], s["v_scales"]]
    else:
        s["k"][at, :, off] = k.bfloat16()
        s["v"][at, :, off] = v.bfloat16()
        out = [q, s["k"], s["v"]]
    return out + [k.bfloat16(), v.bfloat16()] if c["prompt"] else out


def softmax_with_sink(scores, sinks):
    """Weights of scores [.., keys], a score of -infinity none, the sink's [..] left out; zeros where nothing is visible."""
    m = scores.amax(-1, keepdim=True)
    if sinks is not None:
        m = torch.maximum(m, sinks[..., None])
    m = torch.where(m == float("-inf"), 0.0, m)
    e = torch.exp(scores - m)
    total = e.sum(-1, keepdim=True)
    if sinks is not None:
        total = total + torch.exp(sinks[..., None] - m)
    return e / torch.clamp(total, min=torch.finfo(total.dtype).tiny)


def plain_decode(s, c):
    B, Hq, Hkv, D, page = c["B"], c["Hq"], c["Hkv"], c["D"], c["page"]
    lens = s["lens"].long()
    most = min(c["longest"], c["window"] or c["longest"])
    first = torch.clamp(lens - (c["window"] or c["longest"]), min=0)
    at = first[:, None] + torch.arange(most, device=lens.device)  # [B, keys]
    seen = at < lens[:, None]
    at = torch.minimum(at, lens[:, None] - 1)
    pages = torch.gather(s["table"].long(), 1, at // page)

    def rows(x, scales):  # [B, keys, Hkv, D]
        r = x.view(torch.uint8)[pages, :, at % page].view(x.dtype).float()
        if scales is None:
            return r
        e = scales.view(torch.uint8)[pages, :, at % page].float() - 127.0
        return (r.view(*r.shape[:-1], D // 32, 32) * torch.exp2(e)[..., None]).view(r.shape)

    k, v = rows(s["k"], s["k_scales"]), rows(s["v"], s["v_scales"])
    q = s["q"].float().view(B * Hkv, Hq // Hkv, D)
    k = k.permute(0, 2, 3, 1).reshape(B * Hkv, D, most)
    v = v.permute(0, 2, 1, 3).reshape(B * Hkv, most, D)
    scores = (torch.bmm(q, k) * s["scale"]).view(B, Hkv, Hq // Hkv, most)
    scores = torch.where(seen[:, None, None], scores, float("-inf"))
    sinks = None if s["sinks"] is None else s["sinks"].float().view(1, Hkv, Hq // Hkv)
    w = softmax_with_sink(scores, sinks)
    return torch.bmm(w.view(B * Hkv, Hq // Hkv, most), v).view(B, Hq, D).bfloat16()


def plain_prefill(s, c):
    B, Hq, Hkv, D = c["B"], c["Hq"], c["Hkv"], c["D"]
    g, (nq, nk) = Hq // Hkv, s["longest"]
    q_starts, k_starts = s["q_starts"].long(), s["k_starts"].long()
    lq, lk = q_starts[1:] - q_starts[:-1], k_starts[1:] - k_starts[:-1]
    i, j = torch.arange(nq, device=lq.device), torch.arange(nk, device=lq.device)

    def padded(x, starts, n, idx):  # rows of each prompt, the last one's repeated behind them: [B, idx, H, D]
        return x[starts[:-1, None] + torch.minimum(idx, n[:, None] - 1)].float()

    q = padded(s["q"], q_starts, lq, i).view(B, nq, Hkv, g, D).permute(0, 2, 3, 1, 4).reshape(B * Hkv, g * nq, D)
    k = padded(s["k"], k_starts, lk, j).permute(0, 2, 3, 1).reshape(B * Hkv, D, nk)
    v = padded(s["v"], k_starts, lk, j).permute(0, 2, 1, 3).reshape(B * Hkv, nk, D)
    last = i + (lk - lq)[:, None]  # [B, nq]: the last key that a query sees
    seen = j <= last[..., None]
    if c["window"]:
        seen &= j > last[..., None] - c["window"]
    scores = torch.bmm(q, k).mul_(s["scale"]).view(B, Hkv, g, nq, nk)
    scores.masked_fill_(~seen[:, None, None], float("-inf"))
    sinks = None if s["sinks"] is None else s["sinks"].float().view(1, Hkv, g, 1)
    w = softmax_with_sink(scores, sinks)
    del scores
    o = torch.bmm(w.view(B * Hkv, g * nq, nk), v).view(B, Hkv, g, nq, D).permute(0, 3, 1, 2, 4)
    return o[i < lq[:, None]].reshape(-1, Hq, D).bfloat16()


def plain_logprobs(s, c):
    l = s["logits"].float()
    m = l.amax(-1, keepdim=True)
    d = l - m
    e = torch.exp(d)
    z = e.sum(-1, keepdim=True, dtype=torch.float64)  # where one token has nearly all the weight, the others' is lost next to 1 in 32 bits
    log_z = torch.log(z)
    logp = (torch.gather(d, 1, s["tokens"].long()[:, None]) - log_z).float()
    entropy = (log_z - (e * d).sum(-1, keepdim=True, dtype=torch.float64) / z).float()
    if not c["top"]:
        return logp[:, 0], entropy[:, 0]
    order = torch.sort(s["logits"], dim=-1, descending=True, stable=True).indices[:, : c["top"]]
    return logp[:, 0], entropy[:, 0], (torch.gather(d, 1, order) - log_z).float(), order.int()


def pairs(case):
    """Visible pairs of a query and a key of one head, over all sequences."""
    w = case["window"]
    if case["kind"] == "decode":
        return sum(min(n, w or n) for n in lengths(case))
    total = 0
    for n in lengths(case):
        last = np.arange(n, dtype=np.int64) + 1 + case["context"]
        total += int((np.minimum(last, w) if w else last).sum())
    return total


def work(case):
    if case["kind"] == "logprobs":
        T, V = case["T"], case["V"]
        return {"bytes": T * V * (4 if case["rows"] == "f32" else 2) + 12 * T + 8 * T * case["top"], "flops": 6 * T * V}
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    if case["kind"] == "write":
        T = case["T"]
        each = D * 2 if case["fmt"] == "bf16" else D + D // 32
        row = (Hq + 2 * Hkv) * D * (4 if case["rows"] == "f32" else 2) + 2 * Hq * D + 2 * Hkv * each + (4 * Hkv * D if case["prompt"] else 0) + 8
        return {"bytes": T * row + 2 * D, "flops": 3 * T * (Hq + Hkv) * D}
    lens = lengths(case)
    n = pairs(case)
    if case["kind"] == "decode":
        each = D * 2 if case["fmt"] == "bf16" else D + D // 32
        return {"bytes": 2 * n * Hkv * each + 4 * len(lens) * Hq * D, "flops": 4 * n * Hq * D}
    keys = sum(lens) + len(lens) * case["context"]
    return {"bytes": 4 * sum(lens) * Hq * D + 4 * keys * Hkv * D, "flops": 4 * n * Hq * D}


# ---- from the definitions, in 64 bits --------------------------------------------------------------
def exact(case, seed):
    s = inputs(case, seed)
    return {"write": exact_write, "decode": exact_decode, "prefill": exact_prefill, "logprobs": exact_logprobs}[case["kind"]](s, case)


def e4m3_rounded(v):
    """The nearest e4m3 value (ties to even) of 64-bit numbers up to 448 and a rounding."""
    power = torch.clamp(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -40))), min=-6.0)
    step = torch.exp2(power - 3.0)
    return torch.clamp(torch.round(v / step) * step, -448.0, 448.0)


def exact_write(s, c):
    T, Hq, Hkv, D, page = c["T"], c["Hq"], c["Hkv"], c["D"], c["page"]
    x = s["qkv"].double().view(T, Hq + 2 * Hkv, D)
    turn = torch.polar(torch.full((T, D // 2), s["rope_scale"], dtype=torch.float64, device=x.device), s["positions"].double()[:, None] * s["inv_freq"].double()[None])
    z = torch.complex(x[:, : Hq + Hkv, : D // 2].contiguous(), x[:, : Hq + Hkv, D // 2 :].contiguous()) * turn[:, None]
    turned = torch.cat((z.real, z.imag), 2)
    q, k, v = turned[:, :Hq], turned[:, Hq:], x[:, Hq + Hkv :]
    out, scales = [q], []
    slots = s["slots"].long()
    for rows, held in ((k, s["k"]), (v, s["v"])):
        flat = torch.zeros((held.shape[0] * page, Hkv, D), dtype=torch.float64, device=x.device)
        if c["fmt"] == "mx8":
            groups = rows.reshape(T, Hkv, D // 32, 32)
            power = torch.clamp(torch.ceil(torch.log2(groups.abs().amax(3) / 448.0)), min=-126.0)
            rows = e4m3_rounded(groups / torch.exp2(power)[..., None]).reshape(T, Hkv, D)
            all_powers = torch.full((held.shape[0] * page, Hkv, D // 32), 2.0 ** -126, dtype=torch.float64, device=x.device)
            all_powers[slots] = torch.exp2(power)
            scales.append(all_powers.view(-1, page, Hkv, D // 32).transpose(1, 2).contiguous())
        flat[slots] = rows
        out.append(flat.view(-1, page, Hkv, D).transpose(1, 2).contiguous())
    return out + scales + ([k, v] if c["prompt"] else [])


def exact_attention(q, k, v, last, window, scale, sinks):
    """q [n, g, D] of heads that share k, v [m, D]; last [n]: the last key that a query sees.  [n, g, D]"""
    x = torch.matmul(q, k.t().contiguous()) * scale
    j = torch.arange(k.shape[0], device=k.device)
    hidden = j[None] > last[:, None]
    if window:
        hidden = hidden | (j[None] <= last[:, None] - window)
    x = x.masked_fill(hidden[:, None], float("-inf"))
    lse = torch.logsumexp(x, 2)
    if sinks is not None:
        lse = torch.logaddexp(lse, sinks[None].expand_as(lse))
    return torch.matmul(torch.exp(x - lse[..., None]), v)


def exact_decode(s, c):
    Hq, Hkv, D, page = c["Hq"], c["Hkv"], c["D"], c["page"]
    g = Hq // Hkv
    out = torch.zeros((c["B"], Hq, D), dtype=torch.float64, device=s["q"].device)
    sinks = None if s["sinks"] is None else s["sinks"].double()
    for b, n in enumerate(lengths(c)):
        pages = s["table"][b, : -(-n // page)].long()

        def all_rows(x, scales):  # [n, Hkv, D]
            r = x.view(torch.uint8)[pages].view(x.dtype).double()
            if scales is not None:
                r = torch.ldexp(r.view(*r.shape[:-1], D // 32, 32), scales.view(torch.uint8)[pages].double()[..., None] - 127).view(r.shape)
            return r.transpose(1, 2).reshape(-1, Hkv, D)[:n]

        k, v = all_rows(s["k"], s["k_scales"]), all_rows(s["v"], s["v_scales"])
        last = torch.tensor([n - 1], device=k.device)
        for h in range(Hkv):
            mine = slice(h * g, (h + 1) * g)
            out[b, mine] = exact_attention(s["q"][b : b + 1, mine].double(), k[:, h].contiguous(), v[:, h].contiguous(), last, c["window"], s["scale"],
                                           None if sinks is None else sinks[mine])[0]
    return out


def exact_prefill(s, c):
    Hq, Hkv, D = c["Hq"], c["Hkv"], c["D"]
    g, most = Hq // Hkv, 1024
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    sinks = None if s["sinks"] is None else s["sinks"].double()
    q_at = k_at = 0
    for n in lengths(c):
        m = n + c["context"]
        for h in range(Hkv):
            mine = slice(h * g, (h + 1) * g)
            k, v = s["k"][k_at : k_at + m, h].double().contiguous(), s["v"][k_at : k_at + m, h].double().contiguous()
            for i in range(0, n, most):  # so many queries at a time
                rows = torch.arange(i, min(n, i + most), device=k.device)
                end = int(rows.numel()) + i + m - n
                begin = max(0, i + m - n - c["window"] + 1) if c["window"] else 0
                out[q_at + i : q_at + i + rows.numel(), mine] = exact_attention(
                    s["q"][q_at + i : q_at + i + rows.numel(), mine].double(), k[begin:end], v[begin:end], rows + (m - n - begin), c["window"], s["scale"],
                    None if sinks is None else sinks[mine])
        q_at, k_at = q_at + n, k_at + m
    return out


def exact_logprobs(s, c):
    T, top = c["T"], c["top"]
    logp, entropy = (torch.zeros(T, dtype=torch.float64) for _ in range(2))
    best, index = torch.zeros((T, top), dtype=torch.float64), torch.zeros((T, top), dtype=torch.int32)
    for t in range(T):
        l = s["logits"][t].double()
        lp = l - torch.logsumexp(l, 0)
        logp[t] = lp[s["tokens"][t]].cpu()
        entropy[t] = -(torch.exp(lp) * lp).sum().cpu()
        if top:
            order = torch.sort(l, descending=True, stable=True).indices[:top]
            best[t], index[t] = lp[order].cpu(), order.int().cpu()
    return (logp, entropy, best, index) if top else (logp, entropy)
