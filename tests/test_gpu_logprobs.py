"""moe_token_logprobs against its definition in 64 bits."""
import numpy as np
import pytest
import torch

import attnref

pytestmark = pytest.mark.gpu


def call(pkg, logits, tokens, top, stream=None, out=None, ws=None):
    T, V = logits.shape
    dev = logits.device
    if out is None:
        out = [torch.full((T + 1,), -9.0, device=dev), torch.full((T + 1,), -9.0, device=dev), torch.full((T + 1, max(top, 1)), -9.0, device=dev),
               torch.full((T + 1, max(top, 1)), -9, dtype=torch.int32, device=dev)]
    if ws is None:
        ws = torch.empty(pkg.token_logprobs_workspace_bytes(T, V, top), dtype=torch.uint8, device=dev).random_(0, 256)
    pkg.token_logprobs(logits, tokens, T, V, logprobs=out[0], entropy=out[1], top_logprobs=out[2] if top else None, top_indices=out[3] if top else None,
                       top_k=top, workspace=ws, stream=stream)
    return out


def check(logits, tokens, top, out):
    l = logits.double().cpu().numpy()
    logp, ent, best, index = (t.cpu().numpy() for t in out)
    for t, row in enumerate(l):
        want, entropy, limit, e_limit = attnref.logprobs(row)
        tok = int(tokens[t])
        assert logp[t] == want[tok] or abs(logp[t] - want[tok]) <= limit[tok], (t, logp[t], want[tok], limit[tok])
        assert abs(ent[t] - entropy) <= e_limit, (t, ent[t], entropy, e_limit)
        if top:
            order = np.argsort(-row, kind="stable")[:top]
            assert np.array_equal(index[t], order), (t, index[t], order)
            fine = want[order] == best[t]
            with np.errstate(invalid="ignore"):
                assert (fine | (abs(best[t] - want[order]) <= limit[order])).all()
    n = len(l)
    assert logp[n] == ent[n] == -9 and (best[n] == -9).all() and (index[n] == -9).all()


def rows(dev, T, V, kind, dtype, stride=0, seed=0):
    g = torch.Generator(device="cpu").manual_seed(seed + T + V)
    l = 2 * torch.randn((T, V), generator=g)
    if kind == "peaked":
        l += 12 * torch.exp(0.5 * torch.randn((1, V), generator=g))
    if kind == "ascending":
        l = l.sort(-1).values
    if kind == "equal":
        l.fill_(1.5)
    if kind == "masked":  # most are -infinity, some rows keep one or two
        keep = torch.rand((T, V), generator=g) < 0.05
        keep[:, V // 2] = True
        keep[::3] = False
        keep[::3, 0] = True
        l = torch.where(keep, l, float("-inf"))
    if kind == "far":
        l += 3000.0
    if kind == "zeros":  # both signs of zero are the same value
        l = torch.where(torch.rand((T, V), generator=g) < 0.5, 0.0, -0.0)
    wide = torch.full((T, max(V, stride)), 99.0, dtype=dtype)
    wide[:, :V] = l.to(dtype)
    return wide.to(dev)[:, :V], torch.randint(0, V, (T,), generator=g, dtype=torch.int32).to(dev)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,V,top,kind,stride", [
    (1, 1, 1, "normal", 0), (3, 2, 2, "normal", 0), (2, 31, 5, "normal", 0), (5, 65, 32, "masked", 71), (4, 511, 20, "normal", 0), (3, 513, 0, "peaked", 0),
    (7, 1000, 20, "normal", 1003), (2, 4096, 32, "equal", 0), (6, 4097, 7, "normal", 0), (1, 50021, 20, "normal", 0), (3, 131072, 20, "peaked", 0),
    (2, 100003, 32, "ascending", 100009), (2, 70000, 5, "masked", 0), (2, 30000, 20, "equal", 0), (3, 20000, 9, "far", 20001), (2, 9000, 32, "zeros", 0),
    (1030, 600, 3, "normal", 601), (1500, 64, 32, "masked", 0)])
def test_rows(pkg, dev, T, V, top, kind, stride, dtype):
    print(T, V, top, kind, stride, dtype, flush=True)
    l, tokens = rows(dev, T, V, kind, dtype, stride)
    check(l, tokens, top, call(pkg, l, tokens, top))


@pytest.mark.parametrize("V", [200, 60000])
def test_one_token_with_nearly_all_the_weight(pkg, dev, V):
    """Small entropies and log probabilities next to 0 keep their precision."""
    l, tokens = rows(dev, 4, V, "normal", torch.float32)
    for i, up in enumerate((15.0, 25.0, 40.0, 90.0)):
        l[i, 100 + i] += up + 8
        tokens[i] = 100 + i
    out = call(pkg, l, tokens, 4)
    check(l, tokens, 4, out)
    assert (out[1][:3] > 0).all() and (out[0][:3] < 0).all()


def test_alignments(pkg, dev):
    """Rows that begin anywhere: strides and first elements that are no multiples of 16 bytes."""
    for dtype in (torch.float32, torch.bfloat16):
        buf = torch.randn(9 * 5003 + 64, device=dev).to(dtype)
        for first in (0, 1, 2, 3, 5, 7):
            l = buf[first:].as_strided((9, 4999), (5003, 1))
            tokens = torch.arange(9, dtype=torch.int32, device=dev) * 500
            check(l, tokens, 12, call(pkg, l, tokens, 12))


def test_rows_without_probabilities_and_tokens_out_of_range(pkg, dev):
    inf = float("inf")
    for V in (50, 40000):
        l = torch.randn((7, V), device=dev)
        l[1, 7], l[2, 9], l[3] = float("nan"), inf, -inf
        l[4], l[5, 3], l[5, 20] = float("nan"), inf, float("nan")
        tokens = torch.tensor([0, 7, 9, 1, 0, 3, V], dtype=torch.int32, device=dev)
        logp, ent, best, index = call(pkg, l, tokens, 32)
        assert torch.isnan(logp[1:7]).all() and torch.isnan(ent[1:6]).all() and torch.isnan(best[1:6]).all()
        assert torch.isfinite(logp[0]) and torch.isfinite(ent[[0, 6]]).all() and torch.isfinite(best[[0, 6]]).all()
        for t in range(7):
            i = index[t].tolist()
            assert len(set(i)) == 32 and min(i) >= 0 and max(i) < V, (t, i)
        l[6, : V - 20], l[6, 5] = -inf, float("nan")  # a NaN among values without weight
        assert torch.isnan(call(pkg, l, tokens, 7)[1][6])
        tokens[6] = -1
        assert torch.isnan(call(pkg, l, tokens, 0)[0][6])


def test_each_output_alone(pkg, dev):
    l, tokens = rows(dev, 5, 9000, "normal", torch.float32)
    whole = call(pkg, l, tokens, 6)
    ws = torch.empty(pkg.token_logprobs_workspace_bytes(5, 9000, 6), dtype=torch.uint8, device=dev)
    a, b, c, d = (torch.zeros_like(t) for t in whole)
    pkg.token_logprobs(l, tokens, 5, 9000, logprobs=a, workspace=ws)
    pkg.token_logprobs(l, None, 5, 9000, entropy=b, workspace=ws)
    pkg.token_logprobs(l, None, 5, 9000, top_logprobs=c, top_indices=d, top_k=6, workspace=ws)
    for x, y in zip((a, b, c, d), whole):
        assert torch.equal(x[:5], y[:5])


def test_more_rows_than_a_launch_has_blocks(pkg, dev):
    T, V = (1 << 22) + 300, 3
    l = torch.randn((T, V), device=dev)
    tokens = torch.randint(0, V, (T,), device=dev, dtype=torch.int32)
    logp, ent, best, index = call(pkg, l, tokens, 2)
    lp = torch.log_softmax(l.double(), -1)
    assert torch.equal(index[:T].long(), torch.sort(l, dim=-1, descending=True, stable=True).indices[:, :2])
    # few terms: |l| below 8, a handful of roundings of values below 16
    assert (logp[:T] - lp.gather(1, tokens.long()[:, None])[:, 0]).abs().max() <= 2.0 ** -18
    assert (ent[:T] + (lp.exp() * lp).sum(-1)).abs().max() <= 2.0 ** -18


def test_past_32_bits(pkg, dev):
    V, tail = 131071, 40
    for T in ((1 << 31) // V + tail,):
        print("logprobs", T, V, flush=True)
        l = torch.empty((T, V), device=dev).normal_()
        tokens = torch.arange(T, dtype=torch.int32, device=dev)
        out = call(pkg, l, tokens, 8)
        again = call(pkg, torch.cat([l[-tail:]] * 30)[: 30 * tail], tokens[-tail:].repeat(30), 8)  # as many rows as are not cut into parts
        for a, b in zip(out, again):
            assert torch.equal(a[T - tail : T], b[:tail])


def test_captured_and_on_another_stream(pkg, dev):
    cases = [rows(dev, 3, 40000, "normal", torch.float32), rows(dev, 1, 60000, "normal", torch.bfloat16)]
    ws = torch.empty(max(pkg.token_logprobs_workspace_bytes(3, 40000, 8), pkg.token_logprobs_workspace_bytes(1, 60000, 8)), dtype=torch.uint8, device=dev)
    outs = [call(pkg, l, t, 8) for l, t in cases]
    graphs = []
    for (l, t), out in zip(cases, outs):
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            call(pkg, l, t, 8, out=out, ws=ws)
        graphs.append(g)
    for i in range(4):
        for (l, t), out, g in zip(cases, outs, graphs):
            l.normal_()
            want = call(pkg, l, t, 8)
            for o in out:
                o.fill_(-9)
            g.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b)
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            on_side = call(pkg, l, t, 8, stream=side, out=[torch.full_like(o, -9) for o in out], ws=ws) if i == 0 else None
            if on_side:
                torch.cuda.synchronize()
                for a, b in zip(on_side, want):
                    assert torch.equal(a, b)
