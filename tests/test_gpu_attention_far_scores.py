"""Attention with finite scores of any size.  Queries and keys have one dimension that counts and whole numbers in it, so that scores are exact; they lie so far
apart that a row is the value of its largest score, or the mean of several."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

Hkv, G = 2, 3
Hq = Hkv * G


def make(n, D, size, seed):
    """q [n, Hq, D], k, v [n, Hkv, D], and the numbers of the keys [n, Hkv]: scores of a head are +-2^size times a key's number."""
    r = np.random.default_rng(seed)
    number = np.stack([r.permutation(np.arange(1, n + 1)) % 199 for _ in range(Hkv)], 1).astype(np.float64)  # below 2^8, and equal ones from 200 on
    q, k = np.zeros((n, Hq, D)), np.zeros((n, Hkv, D))
    sign = np.where(r.random((n, Hq)) < 0.5, -1.0, 1.0)
    at = D // 2 + 3
    q[:, :, at] = sign * 2.0 ** (size - size // 2)
    k[:, :, at] = number * 2.0 ** (size // 2)
    v = 2.0 * r.integers(-60, 60, (n, Hkv, D))  # means of two are whole
    return q, k, v, sign, number


def expected(sign, number, v, first, last):
    """The mean of the values with the largest score, for every query over keys first .. last."""
    n = sign.shape[0]
    out, exact = np.zeros((n, Hq, v.shape[2])), np.zeros((n, Hq), bool)
    for i in range(n):
        for h in range(Hq):
            s = sign[i, h] * number[first[i] : last[i] + 1, h // G]
            best = np.flatnonzero(s == s.max())
            out[i, h] = v[first[i] + best, h // G].mean(0)
            exact[i, h] = len(best) <= 2
    assert exact.all()
    return out


def on(dev, *arrays):
    return [torch.from_numpy(a).bfloat16().to(dev) for a in arrays]


SIZES = [14, 20, 21, 24, 27, 30, 31, 33, 36, 40, 60, 100]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("window", [0, 50])
def test_prompts(pkg, dev, D, size, window):
    print(D, size, window, flush=True)
    n = 300
    q, k, v, sign, number = make(n, D, size, size)
    i = np.arange(n)
    want = expected(sign, number, v, np.maximum(0, i - window + 1) if window else 0 * i, i)
    dq, dk, dv = on(dev, q, k, v)
    starts = torch.tensor([0, n], dtype=torch.int32, device=dev)
    out = torch.empty_like(dq)
    pkg.attention_prefill(out, dq, dk, dv, starts, starts, 1, Hq, Hkv, D, 1.0, window=window)
    if size >= 20:
        assert torch.equal(out.double().cpu(), torch.from_numpy(want))
    else:
        # a weight is 2^d there, d what the product of the largest score lost: rounded to bf16 it is off by up to 2^-8, its sum is not, and the two of
        # a mean have the same; 120 is the largest value.  The result is rounded once more
        limit = 2.0 ** -8 * 120 + 2.0 ** -8 * (abs(want) + 2.0 ** -8 * 120)
        assert (abs(out.double().cpu().numpy() - want) <= limit).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("size", SIZES)
def test_single_tokens(pkg, dev, D, size):
    print(D, size, flush=True)
    n, page = 300, 16
    q, k, v, sign, number = make(n, D, size, size)
    i = np.arange(n)
    want = expected(sign, number, v, 0 * i, i)
    dq, dk, dv = on(dev, q, k, v)
    pages = -(-n // page)
    held = [torch.zeros((pages * page, Hkv, D), dtype=torch.bfloat16, device=dev) for _ in range(2)]
    for t, rows in zip(held, (dk, dv)):
        t[:n] = rows
    cache = pkg.KvCache(*(t.view(pages, page, Hkv, D).transpose(1, 2).contiguous() for t in held))
    table = torch.arange(pages, dtype=torch.int32, device=dev).repeat(n, 1)
    lens = torch.arange(1, n + 1, dtype=torch.int32, device=dev)
    out = torch.empty_like(dq)
    ws = torch.empty(pkg.attention_decode_workspace_bytes(n, Hq, Hkv, D), dtype=torch.uint8, device=dev)
    pkg.attention_decode(out, dq, cache, table, lens, n, Hq, 1.0, ws)
    assert torch.equal(out.double().cpu(), torch.from_numpy(want))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("size", [24, 30, 33, 40, 60])
def test_far_below_before_others(pkg, dev, D, size):
    """Keys far below come first: what they weighed is gone once others are seen."""
    n, low = 200, 70
    q, k = np.zeros((n, Hq, D)), np.zeros((n, Hkv, D))
    q[..., 5] = 1.0
    k[:low, :, 5] = -(2.0 ** size)
    v = np.full((n, Hkv, D), 3.0)
    v[:low] = 40.0
    dq, dk, dv = on(dev, q, k, v)
    starts = torch.tensor([0, n], dtype=torch.int32, device=dev)
    out = torch.empty_like(dq)
    pkg.attention_prefill(out, dq, dk, dv, starts, starts, 1, Hq, Hkv, D, 0.37)
    assert (out[:low] == 40.0).all() and (out[low:] == 3.0).all()


@pytest.mark.parametrize("D", [64, 128])
def test_rows_beside_far_ones_keep_their_bits(pkg, dev, D):
    """Some queries of a tile have far scores, over keys that all see: the others' results stay what they are without them."""
    n = 260
    g = torch.Generator().manual_seed(D)
    q, k, v = (torch.randn((n, h, D), generator=g).bfloat16().to(dev) for h in (Hq, Hkv, Hkv))
    starts = torch.tensor([0, n], dtype=torch.int32, device=dev)
    sinks = torch.randn(Hq, generator=g).bfloat16().to(dev)
    outs = []
    for far in (1.0, 2.0 ** 34):
        x = q.clone()
        x[::7] *= far
        out = torch.empty_like(x)
        pkg.attention_prefill(out, x, k, v, starts, starts, 1, Hq, Hkv, D, 0.125, sinks=sinks)
        outs.append(out)
    same = torch.arange(n, device=dev) % 7 != 0
    assert torch.equal(outs[0][same], outs[1][same])
    assert torch.isfinite(outs[1]).all()
