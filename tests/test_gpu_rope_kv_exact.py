"""Keys for an 8-bit cache against the turn in 64 bits: scales the smallest that do, codes the nearest, to the bit."""
import numpy as np
import pytest
import torch

import opsref
import ropeexact

gpu = pytest.mark.gpu


def quantised(w):
    """Scales and values of groups of 32 of rows w [.., D] in 64 bits by the cache's rule."""
    g = w.reshape(*w.shape[:-1], -1, 32)
    power = np.maximum(np.ceil(np.log2(np.maximum(abs(g).max(-1), 2.0 ** -200) / 448.0)), -126.0)
    return power, opsref.to_e4m3(g / np.exp2(power)[..., None])


SCALE = 1.25


def make(T, D, far, seed):
    """Keys x [T, 1, D] whose turned values lie as close to the middle of two codes as fp32 keys allow, but for the largest of each group."""
    r = np.random.default_rng(seed)
    x = (r.standard_normal((T, 1, D)) * np.exp(r.standard_normal((1, 1, D)))).astype(np.float32)
    pos = r.integers(-far, far, T, dtype=np.int64).astype(np.int32)
    inv = (10000.0 ** (-np.arange(0, D, 2) / D)).astype(np.float32)
    w = ropeexact.turned(x.astype(np.float64), pos, inv, SCALE)
    power, values = quantised(w)
    step = np.exp2(np.maximum(np.floor(np.log2(np.maximum(abs(values), 2.0 ** -20))), -6.0) - 3.0)
    middle = (np.sign(values) * (abs(values) + step / 2) * np.exp2(power)[..., None]).reshape(w.shape)
    largest = (abs(values) > 200.0).reshape(w.shape)
    h = D // 2
    a = ropeexact.angles(pos, inv)[:, None]
    u = (middle[..., :h] / SCALE + x[..., h:].astype(np.float64) * np.sin(a)) / np.cos(a)
    fit = (abs(np.cos(a)) > 0.5) & ~largest[..., :h] & (abs(u - x[..., :h]) < 0.1 * abs(x[..., :h]))
    x[..., :h] = np.where(fit, u, x[..., :h]).astype(np.float32)
    assert fit.mean() > 0.25
    return x, pos, inv


def differing(x, pos, inv, power, values):
    """Places where codes or scales are not those of the turn in 64 bits, nor of a value as far from it as roundings in 64 bits make it."""
    D = x.shape[-1]
    w = ropeexact.turned(x.astype(np.float64), pos, inv, SCALE)
    # cosine and sine: the angle to 2^-52, the functions and their product with scale to 2^-51 together; two products and a sum: below 2^-49 of each
    off = 2.0 ** -49 * SCALE * (abs(x) + abs(np.roll(x, D // 2, -1))).astype(np.float64)
    wrong = np.ones(values.shape, bool)
    for d in (0.0, -off, off):
        p, v = quantised(w + np.sign(w) * d)
        wrong &= (v != values) | (p != power)[..., None]
    return int(wrong.sum())


FAR = [1, 4096, 200000, 2**31 - 1]


@gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("far", FAR)
def test_codes_of_turned_keys_are_the_nearest(pkg, dev, D, far):
    T, page = 2000, 64
    print(D, far, flush=True)
    x, pos, inv = make(T, D, far, D + far % 1000)
    n_pages = -(-T // page)
    rows = torch.from_numpy(np.concatenate([x, x, x], 1)).to(dev).view(T, -1)
    kv = [torch.zeros((n_pages, 1, page, D), dtype=torch.uint8, device=dev) for _ in range(2)]
    ss = [torch.zeros((n_pages, 1, page, D // 32), dtype=torch.uint8, device=dev) for _ in range(2)]
    i = torch.arange(T, dtype=torch.int32, device=dev)
    pkg.rope_kv_write(None, rows, torch.from_numpy(pos).to(dev), torch.from_numpy(inv).to(dev), T, 1, 1, D, rope_scale=SCALE, cache=pkg.KvCache(*kv, *ss), slots=i)
    values = opsref.e4m3_values(kv[0].view(-1, D)[:T].cpu().numpy()).reshape(T, 1, D // 32, 32)
    power = ss[0].view(-1, D // 32)[:T].cpu().numpy().astype(np.float64).reshape(T, 1, D // 32) - 127
    assert differing(x, pos, inv, power, values) == 0


@pytest.mark.parametrize("far", FAR[1:])
def test_the_codes_tell_less_exact_turns_apart(far):
    """Turns in 32 bits, and angles that lose what a product of 55 bits has past 53, give other codes of such keys."""
    T, D = 2000, 64
    x, pos, inv = make(T, D, far, D + far % 1000)
    a = ropeexact.angles(pos, inv)
    u, v = x[..., : D // 2], x[..., D // 2 :]

    def codes(c, s, dtype):
        c, s = c.astype(dtype)[:, None], s.astype(dtype)[:, None]
        w = np.concatenate([u.astype(dtype) * c - v.astype(dtype) * s, v.astype(dtype) * c + u.astype(dtype) * s], -1).astype(np.float64)
        return quantised(w)
    exact = [np.float64(np.float32(SCALE)) * f(a) for f in (np.cos, np.sin)]
    assert differing(x, pos, inv, *codes(*exact, np.float64)) == 0
    assert differing(x, pos, inv, *codes(*exact, np.float32)) > 1000
    if far > 2**30:
        b = pos.astype(np.float64)[:, None] * inv.astype(np.float64)[None]
        turns = b * 0.15915494309189533577
        b = (turns - np.rint(turns)) * (2 * np.pi)
        assert differing(x, pos, inv, *codes(*[np.float64(np.float32(SCALE)) * f(b) for f in (np.cos, np.sin)], np.float64)) > 1000
