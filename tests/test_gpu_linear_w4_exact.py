"""int4 weights are code - zero point, exactly: where those are small or none, so are the products' errors, whatever the codes are."""
import numpy as np
import pytest
import torch

import opsref

pytestmark = pytest.mark.gpu

# one tile of weight rows to a block, and blocks that go through several
SHAPES = [(1, 200, 2880), (7, 200, 2880), (20, 200, 2880), (2, 20033, 288), (20, 20033, 288)]


def product(pkg, dev, x, codes, scales, zeros, group, x_scales=None, bias=None):
    """codes [N, K] 0..15, scales [N, n] fp32 that bf16 holds, zeros [N, n] or None; x on the host."""
    N, K = codes.shape
    on = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
    t = pkg.int4_repack(on((codes[:, ::2] | codes[:, 1::2] << 4).astype(np.uint8)), on(scales).bfloat16(), None if zeros is None else on(zeros), group)
    y = torch.full((x.shape[0], N), -7.0, device=dev)
    pkg.linear_int4(y, x.to(dev), t[0], t[1], x.shape[0], K, N, group, tiled_zeros=t[2], bias=None if bias is None else bias.to(dev),
                    x_scales=None if x_scales is None else x_scales.to(dev))
    return y.cpu().numpy()


def zero_points(r, N, K, group, given):
    """([N, n] u8 or None, the same spread over [N, K])"""
    n = -(-K // group)
    z = r.integers(0, 16, (N, n), dtype=np.uint8) if given else np.full((N, n), 8, np.uint8)
    return (z if given else None), np.repeat(z, group, 1)[:, :K]


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("B,N,K", SHAPES)
def test_weights_of_zero_give_zero(pkg, dev, group, zeros, B, N, K):
    r = np.random.default_rng(B + N)
    z, spread = zero_points(r, N, K, group, zeros)
    scales = np.exp2(r.integers(-3, 3, (N, -(-K // group)))).astype(np.float32)
    x = torch.from_numpy(np.abs(r.standard_normal((B, K))).astype(np.float32)).bfloat16()
    print("weights of zero", group, zeros, B, N, K, flush=True)
    assert (product(pkg, dev, x, spread, scales, z, group) == 0).all()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("B,N,K", SHAPES)
@pytest.mark.parametrize("rows", ["bf16", "mx8"])
def test_rows_of_one_sign_against_few_weights(pkg, dev, group, zeros, B, N, K, rows):
    """One weight in 256 is not zero.  A result takes at most K / 8 + 64 roundings of half a step 2^-24 (the matrix instruction adds at least 8
    products at a time; a scale, the waves' sums), each of a partial sum of at most the sum of the magnitudes |x| |W|, which is small here."""
    r = np.random.default_rng(B + N)
    z, spread = zero_points(r, N, K, group, zeros)
    step = np.where(spread < 15, 1, -1)
    codes = (spread + step * (r.random((N, K)) < 1 / 256)).astype(np.uint8)
    n = -(-K // group)
    scales = torch.from_numpy((0.01 * np.exp(0.3 * r.standard_normal((N, n)))).astype(np.float32)).bfloat16().float().numpy()
    w = (codes.astype(np.float64) - spread) * np.repeat(scales.astype(np.float64), group, 1)[:, :K]
    v = np.abs(r.standard_normal((B, K))).astype(np.float32)
    if rows == "bf16":
        x, xs = torch.from_numpy(v).bfloat16(), None
        v = x.double().numpy()
    else:
        c = torch.from_numpy(v * 100).clamp(max=448).to(torch.float8_e4m3fn).view(torch.uint8)
        x, xs = c, torch.from_numpy(r.integers(117, 124, (B, K // 32), dtype=np.uint8))
        v = opsref.e4m3_values(c.numpy()) * np.repeat(np.exp2(xs.numpy().astype(np.float64) - 127), 32, 1)
    print("rows of one sign", group, zeros, B, N, K, rows, flush=True)
    got = product(pkg, dev, x, codes, scales, z, group, xs)
    assert (np.abs(got - v @ w.T) <= (K / 8 + 64) * 2.0 ** -24 * (v @ np.abs(w).T)).all()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("B,N", [(3, 80), (18, 80), (3, 20033)])
def test_large_finite_rows(pkg, dev, group, zeros, B, N):
    """Weights of -1, 0 and 1 on rows of 2^120: every partial sum is a multiple of 2^120 of at most 160 of them, finite and exact."""
    K = 160
    r = np.random.default_rng(N)
    z, spread = zero_points(r, N, K, group, zeros)
    codes = np.clip(spread.astype(np.int64) + r.integers(-1, 2, (N, K)), 0, 15).astype(np.uint8)
    x = torch.full((B, K), 2.0 ** 120).bfloat16()
    print("large rows", group, zeros, B, N, flush=True)
    got = product(pkg, dev, x, codes, np.ones((N, -(-K // group)), np.float32), z, group)
    want = 2.0 ** 120 * (codes.astype(np.float64) - spread).sum(1)
    assert np.array_equal(got.astype(np.float64), np.broadcast_to(want, (B, N)))


def test_every_code_and_zero_point(pkg, dev):
    """A one in one place of x reads out one weight, for every code with every zero point."""
    N, K = 256, 256
    r = np.random.default_rng(0)
    for group in (32, 64, 128):
        codes = ((np.arange(N)[:, None] + np.arange(K)[None] * 5) & 15).astype(np.uint8)
        z = ((np.arange(N)[:, None] >> 4) + np.arange(K // group)[None]).astype(np.uint8) & 15
        scales = np.exp2(r.integers(-2, 3, (N, K // group))).astype(np.float32)
        got = product(pkg, dev, torch.eye(K).bfloat16(), codes, scales, z, group)
        want = (codes.astype(np.float64) - np.repeat(z, group, 1)) * np.repeat(scales, group, 1)
        assert np.array_equal(got, want.T.astype(np.float32))
