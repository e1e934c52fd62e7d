"""The precision of the weights in attention of single tokens, seen past the bf16 result: values that cancel but for what the weights are off by."""
import numpy as np
import pytest
import torch

import attnref

gpu = pytest.mark.gpu


def cancelling(n, D, seed):
    """Scores [n] that are bf16 numbers, values v [n, D] in bf16 whose weighted mean is about 2^-24 of that of |v|."""
    r = np.random.default_rng(seed)
    bf16 = lambda a: torch.from_numpy(np.asarray(a)).bfloat16().double().numpy()  # noqa: E731
    s = bf16(r.uniform(-2, 2, n))
    v = bf16(r.standard_normal((n, D)))
    w = attnref.softmax_rows(s, None)
    at = r.permutation(n)[:4]
    v[at] = 0
    for i in at:
        v[i] = bf16(-(w @ v) / w[i])  # what is left falls by 2^8 each time
    assert (abs(w @ v) < 2.0 ** -20 * (w @ abs(v))).all()
    return s, v, w


def limit(n, w, v, s):
    o, mean = w @ v, w @ abs(v)
    # scores are exact; times log2(e) and less the maximum two roundings, of up to |s| log2(e) and the difference; exp2 a step: in a weight twice, numerator and sum.
    # A weight as two bf16 numbers 2^-16.  Sums over n keys, joins of waves and the quotient: n + 12 roundings, twice
    size = 3 * abs(s).max() * 1.45
    error = mean * (attnref.U16 + 2 * (size + 2) * attnref.U24 + 2 * (n + 12) * attnref.U24)
    return o, error + attnref.U8 * (abs(o) + error)


CASES = [(24, 64), (40, 64), (100, 64), (40, 128), (100, 128)]


@gpu
@pytest.mark.parametrize("n,D", CASES)
def test_weights_are_good_to_16_bits(pkg, dev, n, D):
    print(n, D, flush=True)
    Hq, Hkv, page, B = 6, 2, 16, 5
    pages = -(-n // page)
    k, v = np.zeros((B, pages * page, Hkv, D)), np.zeros((B, pages * page, Hkv, D))
    want = np.zeros((2, B, Hkv, D))
    for b in range(B):
        for h in range(Hkv):
            s, v[b, :n, h], w = cancelling(n, D, 10 * b + h)
            k[b, :n, h, 3] = s
            want[:, b, h] = limit(n, w, v[b, :n, h], s)
    q = torch.zeros((B, Hq, D), dtype=torch.bfloat16, device=dev)
    q[..., 3] = 1.0
    cache = pkg.KvCache(*(torch.from_numpy(t).bfloat16().to(dev).view(B, pages, page, Hkv, D).transpose(2, 3).reshape(B * pages, Hkv, page, D).contiguous() for t in (k, v)))
    table = torch.arange(B * pages, dtype=torch.int32, device=dev).view(B, pages)
    lens = torch.full((B,), n, dtype=torch.int32, device=dev)
    out = torch.empty_like(q)
    ws = torch.empty(pkg.attention_decode_workspace_bytes(B, Hq, Hkv, D), dtype=torch.uint8, device=dev)
    pkg.attention_decode(out, q, cache, table, lens, B, Hq, 1.0, ws)
    o, off = (np.repeat(t, Hq // Hkv, 1) for t in want)
    assert (abs(out.double().cpu().numpy() - o) <= off).all()


@pytest.mark.parametrize("n,D", CASES)
def test_weights_of_8_bits_would_not_pass(n, D):
    s, v, w = cancelling(n, D, 1)
    o, off = limit(n, w, v, s)
    e = np.exp(s - s.max())
    rounded = torch.from_numpy(e).bfloat16().double().numpy()
    assert (abs(rounded @ v / e.sum() - o) > off).mean() > 0.5
    rest = torch.from_numpy(e - rounded).bfloat16().double().numpy()
    assert (abs((rounded + rest) @ v / e.sum() - o) <= off).all()
