"""The cache, attention and log probability operators as a program uses them: prompts into the cache and through their attention, then tokens one by one
with projections, norm, output matrix and scores around; eager, and captured and replayed."""
import numpy as np
import pytest
import torch

import attnref

pytestmark = pytest.mark.gpu

H, HQ, HKV, D, V, PAGE, TOP = 256, 8, 2, 64, 640, 16, 5
QKV = (HQ + 2 * HKV) * D


class Layer:
    """Weights of one attention layer and an output matrix, a cache, and room for B sequences."""

    def __init__(self, pkg, dev, B, fmt, window, seed=0):
        self.pkg, self.B, self.dev, self.window = pkg, B, dev, window
        g = torch.Generator(device="cpu").manual_seed(seed)
        codes = lambda n, k: torch.randint(0, 256, (1, n, k // 32, 16), generator=g, dtype=torch.uint8).to(dev)  # noqa: E731
        scales = lambda n, k: torch.randint(119, 123, (1, n, k // 32), generator=g, dtype=torch.uint8).to(dev)  # noqa: E731
        self.w_qkv, self.w_out, self.w_head = (pkg.mxfp4_repack(codes(n, k), scales(n, k)) for n, k in ((QKV, H), (H, HQ * D), (V, H)))
        self.norm = torch.ones(H, device=dev).bfloat16()
        self.inv = (150000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)).float().to(dev)
        self.sinks = torch.randn(HQ, generator=g).bfloat16().to(dev)
        n_pages, self.max_pages = 40 * B, 20
        self.table = torch.randperm(n_pages, generator=g)[: B * self.max_pages].view(B, self.max_pages).int().to(dev)
        u8 = lambda *s: torch.zeros(s, dtype=torch.uint8, device=dev)  # noqa: E731
        if fmt == "bf16":
            self.cache = pkg.KvCache(*(torch.zeros((n_pages, HKV, PAGE, D), dtype=torch.bfloat16, device=dev) for _ in range(2)))
        else:
            self.cache = pkg.KvCache(u8(n_pages, HKV, PAGE, D), u8(n_pages, HKV, PAGE, D), u8(n_pages, HKV, PAGE, D // 32), u8(n_pages, HKV, PAGE, D // 32))
        f = lambda *s, t=torch.float32: torch.empty(s, dtype=t, device=dev)  # noqa: E731
        bf = torch.bfloat16
        self.x = torch.randn((B, H), generator=g).to(dev)
        self.t, self.qkv, self.q, self.att, self.delta, self.x2, self.u, self.logits = (
            f(B, H, t=bf), f(B, QKV), f(B, HQ, D, t=bf), f(B, HQ, D, t=bf), f(B, H), f(B, H), f(B, H, t=bf), f(B, V))
        self.tokens, self.pos, self.lens, self.slots = (torch.zeros(B, dtype=torch.int32, device=dev) for _ in range(4))
        self.logp, self.ent, self.top, self.index = f(B), f(B), f(B, TOP), f(B, TOP, t=torch.int32)
        self.ws = torch.empty(pkg.attention_decode_workspace_bytes(B, HQ, HKV, D), dtype=torch.uint8, device=dev)

    def slots_of(self, b, positions):
        return self.table[b, positions // PAGE] * PAGE + positions % PAGE

    def step(self):
        """One token a sequence at positions self.pos: everything on the device."""
        p, B = self.pkg, self.B
        torch.add(self.pos, 1, out=self.lens)
        page = torch.gather(self.table, 1, (self.pos // PAGE).long()[:, None])[:, 0]
        torch.add(page * PAGE, self.pos % PAGE, out=self.slots)
        p.add_rmsnorm(self.x2, self.x, self.norm, B, H, o_bf16=self.t)
        p.linear_mxfp4(self.qkv, self.t, *self.w_qkv, B, H, QKV)
        p.rope_kv_write(self.q, self.qkv, self.pos, self.inv, B, HQ, HKV, D, rope_scale=1.1, cache=self.cache, slots=self.slots)
        p.attention_decode(self.att, self.q, self.cache, self.table, self.lens, B, HQ, D ** -0.5, self.ws, window=self.window, sinks=self.sinks)
        p.linear_mxfp4(self.delta, self.att.view(B, HQ * D), *self.w_out, B, HQ * D, H)
        p.add_rmsnorm(self.x2, self.x, self.norm, B, H, delta=self.delta, o_bf16=self.u)
        p.linear_mxfp4(self.logits, self.u, *self.w_head, B, H, V)
        p.token_logprobs(self.logits, self.tokens, B, V, logprobs=self.logp, entropy=self.ent, top_logprobs=self.top, top_indices=self.index, top_k=TOP)

    def outputs(self):
        return [t.clone() for t in (self.q, self.att, self.x2, self.logits, self.logp, self.ent, self.top, self.index, self.cache.k, self.cache.v)]


def prompts(layer, lens, seed):
    """Rows of the projection for prompts of these lengths, turned, in the cache and through their attention: (out, q, k, v) packed."""
    p, dev = layer.pkg, layer.dev
    T = sum(lens)
    g = torch.Generator(device="cpu").manual_seed(seed)
    qkv = torch.randn((T, QKV), generator=g).to(dev)
    pos = torch.cat([torch.arange(n, dtype=torch.int32) for n in lens]).to(dev)
    slots = torch.cat([layer.slots_of(b, torch.arange(n, device=dev)) for b, n in enumerate(lens)]).int()
    bf = torch.bfloat16
    q, k, v = (torch.empty((T, h, D), dtype=bf, device=dev) for h in (HQ, HKV, HKV))
    p.rope_kv_write(q, qkv, pos, layer.inv, T, HQ, HKV, D, rope_scale=1.1, k=k, v=v, cache=layer.cache, slots=slots)
    starts = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device=dev)
    out = torch.empty_like(q)
    p.attention_prefill(out, q, k, v, starts, starts, len(lens), HQ, HKV, D, D ** -0.5, window=layer.window, sinks=layer.sinks)
    return out, q, k, v


@pytest.mark.parametrize("window", [0, 20])
def test_the_last_token_of_a_prompt_both_ways(pkg, dev, window):
    """Decoding a prompt's last token over the cache that the prompt left is the last row of the prompt's attention: both within their bounds of the formula."""
    lens = [1, 40, 130, 300]
    layer = Layer(pkg, dev, len(lens), "bf16", window)
    out, q, k, v = prompts(layer, lens, 5)
    last = np.cumsum(lens) - 1
    layer.lens.copy_(torch.tensor(lens))
    q_last = q[torch.from_numpy(last).to(dev)].contiguous()
    pkg.attention_decode(layer.att, q_last, layer.cache, layer.table, layer.lens, layer.B, HQ, D ** -0.5, layer.ws, window=window, sinks=layer.sinks)
    qd, kd, vd, sinks, a, b = (t.double().cpu().numpy() for t in (q_last, k, v, layer.sinks, layer.att, out))
    for i, n in enumerate(lens):
        lo = last[i] + 1 - (min(n, window) if window else n)
        for h in range(HQ):
            g = h // (HQ // HKV)
            want, limit = attnref.attention_row(qd[i, h], kd[lo : last[i] + 1, g], vd[lo : last[i] + 1, g], D ** -0.5, sinks[h])
            assert (abs(a[i, h] - want) <= limit).all() and (abs(b[last[i], h] - want) <= limit).all()


@pytest.mark.parametrize("fmt", ["bf16", "mx8"])
@pytest.mark.parametrize("window", [0, 20])
def test_steps_eager_and_captured(pkg, dev, fmt, window):
    """Tokens one by one behind prompts; the captured step replayed for each gives what the eager one does."""
    lens = [7, 100, 33]
    eager, captured = (Layer(pkg, dev, len(lens), fmt, window) for _ in range(2))
    for layer in (eager, captured):
        prompts(layer, lens, 6)
        layer.pos.copy_(torch.tensor(lens))
    torch.cuda.synchronize()
    captured.step()  # writes the slots that the first replay writes again
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured.step()
    for i in range(5):
        for layer in (eager, captured):
            layer.x.copy_(torch.randn((layer.B, H), generator=torch.Generator().manual_seed(i)))
            layer.tokens.fill_(11 * i)
        eager.step()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(eager.outputs(), captured.outputs()):
            assert torch.equal(a, b)
        # every row of the step against the formulas, from what went into each operator
        for b in range(eager.B):
            logp, ent, limit, e_limit = attnref.logprobs(eager.logits[b].double().cpu().numpy())
            assert abs(eager.logp[b].item() - logp[11 * i]) <= limit[11 * i] and abs(eager.ent[b].item() - ent) <= e_limit
            assert eager.index[b].tolist() == np.argsort(-eager.logits[b].double().cpu().numpy(), kind="stable")[:TOP].tolist()
        if fmt == "bf16":
            q, sinks, got = (t.double().cpu().numpy() for t in (eager.q, eager.sinks, eager.att))
            for b in range(eager.B):
                n = int(eager.lens[b])
                s = eager.slots_of(b, torch.arange(max(0, n - window) if window else 0, n, device=dev)).long()
                kk, vv = (t[s // PAGE, :, s % PAGE].double().cpu().numpy() for t in (eager.cache.k, eager.cache.v))
                for h in range(HQ):
                    want, bound = attnref.attention_row(q[b, h], kk[:, h // (HQ // HKV)], vv[:, h // (HQ // HKV)], D ** -0.5, sinks[h])
                    assert (abs(got[b, h] - want) <= bound).all()
        for layer in (eager, captured):
            layer.pos += 1


def test_a_prompt_in_pieces(pkg, dev):
    """A prompt taken in pieces, each over all the keys so far, has the same bits as at once where the pieces end on tile borders."""
    layer = Layer(pkg, dev, 1, "bf16", 0)
    out, q, k, v = prompts(layer, [300], 7)
    for a, b in ((0, 128), (128, 256), (256, 300)):
        part = torch.empty((b - a, HQ, D), dtype=torch.bfloat16, device=dev)
        qs, ks = (torch.tensor([0, n], dtype=torch.int32, device=dev) for n in (b - a, b))
        pkg.attention_prefill(part, q[a:b], k[:b], v[:b], qs, ks, 1, HQ, HKV, D, D ** -0.5, sinks=layer.sinks)
        assert torch.equal(part, out[a:b])
