"""moe_linear_mxfp4 and moe_linear_int4: bit for bit where every sum is exact in 32 bits, against 64 bits otherwise."""
import numpy as np
import pytest
import torch

import opsref

pytestmark = pytest.mark.gpu

ROWS = [1, 2, 15, 16, 17, 32, 33, 64, 65, 130]


class Weights:
    def __init__(self, pkg, dev, N, K, fmt, group=32, zeros=False, seed=0, exact=False):
        r = np.random.default_rng(seed)
        self.pkg, self.dev, self.N, self.K, self.fmt, self.group = pkg, dev, N, K, fmt, group
        codes = r.integers(0, 256, (N, K // 2), dtype=np.uint8)
        t = lambda a: torch.from_numpy(a).to(dev)  # noqa: E731
        if fmt == "mxfp4":
            scales = r.integers(126, 129, (N, K // 32), dtype=np.uint8) if exact else r.integers(119, 128, (N, K // 32), dtype=np.uint8)
            self.w = opsref.mxfp4_weights(codes, scales)
            self.bound = np.abs(self.w)
            self.tiled = pkg.mxfp4_repack(t(codes).view(1, N, K // 32, 16), t(scales).view(1, N, K // 32))
        else:
            n = -(-K // group)
            scales = np.exp2(r.integers(-1, 2, (N, n))).astype(np.float32) if exact else (0.01 * np.exp(0.3 * r.standard_normal((N, n)))).astype(np.float32)
            scales = torch.from_numpy(scales).bfloat16()
            z = r.integers(0, 16, (N, n), dtype=np.uint8) if zeros else None
            self.w, self.bound = opsref.int4_weights(codes, scales.double().numpy(), z, group)
            self.tiled = pkg.int4_repack(t(codes), scales.to(dev), None if z is None else t(z), group)

    def run(self, x, x_scales=None, bias=None, B=None, stream=None):
        B = x.shape[0] if B is None else B
        y = torch.full((B * self.N + 64,), -7.0, device=self.dev)
        if self.fmt == "mxfp4":
            self.pkg.linear_mxfp4(y, x, *self.tiled, B, self.K, self.N, bias=bias, x_scales=x_scales, stream=stream)
        else:
            self.pkg.linear_int4(y, x, self.tiled[0], self.tiled[1], B, self.K, self.N, self.group, tiled_zeros=self.tiled[2], bias=bias,
                                 x_scales=x_scales, stream=stream)
        assert (y[B * self.N:] == -7).all()
        return y[: B * self.N].view(B, self.N)


def mx8_rows(r, B, K, whole):
    """(codes, scale bytes, values) of rows in e4m3 with e8m0 scales; whole: small whole numbers."""
    if whole:
        v = r.integers(-8, 9, (B, K)).astype(np.float32)
        s = np.full((B, K // 32), 127, np.uint8)
        s[:, ::2] = 128
    else:
        v = (r.standard_normal((B, K)) * 100).astype(np.float32)
        s = r.integers(117, 124, (B, K // 32), dtype=np.uint8)
    codes = torch.from_numpy(v).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    return codes, torch.from_numpy(s), opsref.e4m3_values(codes.numpy()) * np.repeat(np.exp2(s.astype(np.float64) - 127), 32, 1)


FORMS = [("mxfp4", 32, False), ("int4", 32, True), ("int4", 64, False), ("int4", 64, True), ("int4", 128, False), ("int4", 128, True)]


@pytest.mark.parametrize("fmt,group,zeros", FORMS)
@pytest.mark.parametrize("N,K", [(64, 32), (64, 96), (128, 128), (64, 160), (192, 512), (64, 992), (128, 1056), (320, 2880), (64, 8224)])
def test_exact_sums(pkg, dev, fmt, group, zeros, N, K):
    """Small whole numbers and scales of 1/2, 1 and 2: every partial sum, in any order, is a multiple of 1/4 (MXFP4) or 1/2 (int4) of at most
    2^22 of them, and thus exact: MXFP4 4 * 12 * 8224 or 16 * 12 * 2880 < 2^20, int4 4 * 30 * 8224 or 16 * 30 * 2880 < 2^21 (and within a group
    16 * 31 * 128)."""
    w = Weights(pkg, dev, N, K, fmt, group, zeros, seed=N + K, exact=True)
    r = np.random.default_rng(K)
    for B in ROWS:
        print("exact sums", fmt, group, zeros, N, K, B, flush=True)
        x = r.integers(-4, 5, (B, K)).astype(np.float32)
        got = w.run(torch.from_numpy(x).bfloat16().to(dev))
        assert np.array_equal(got.cpu().numpy(), x.astype(np.float64) @ w.w.T)
        if K <= 2880:
            codes, scales, v = mx8_rows(r, B, K, True)
            got = w.run(codes.to(dev), scales.to(dev))
            assert np.array_equal(got.cpu().numpy(), v @ w.w.T)


@pytest.mark.parametrize("fmt,group,zeros", FORMS)
@pytest.mark.parametrize("N,K", [(4160, 96), (13056, 64), (20032, 288), (16448, 1184), (4800, 8224)])
def test_exact_sums_of_many_tiles(pkg, dev, fmt, group, zeros, N, K):
    """As above, for blocks that go through several tiles of weight rows: with waves side by side, the last block's tiles ending early, in one or
    more slabs of the contraction; against sums in 64 bits on the device."""
    w = Weights(pkg, dev, N, K, fmt, group, zeros, seed=N + K, exact=True)
    wt = torch.from_numpy(w.w).to(dev).t().contiguous()
    for B in (3, 20, 40):
        print("exact sums", fmt, group, zeros, N, K, B, flush=True)
        x = torch.randint(-4, 5, (B, K), device=dev, generator=torch.Generator(device=dev).manual_seed(B)).bfloat16()
        assert torch.equal(w.run(x).double(), x.double() @ wt)


@pytest.mark.parametrize("fmt,group,zeros", FORMS)
@pytest.mark.parametrize("B,N,K", [(1, 2880, 2880), (5, 64, 4096), (16, 1024, 1440), (40, 640, 2880), (64, 2880, 640), (100, 128, 5760)])
def test_against_64_bits(pkg, dev, fmt, group, zeros, B, N, K):
    w = Weights(pkg, dev, N, K, fmt, group, zeros, seed=B + N + K)
    r = np.random.default_rng(N)
    bias = torch.from_numpy(r.standard_normal(N).astype(np.float32)).bfloat16()
    for rows in ("bf16", "mx8"):
        print("against 64 bits", fmt, group, zeros, B, N, K, rows, flush=True)
        if rows == "bf16":
            x, xs = torch.from_numpy(r.standard_normal((B, K)).astype(np.float32)).bfloat16(), None
            v = x.double().numpy()
        else:
            x, xs, v = mx8_rows(r, B, K, False)
        for b in (None, bias):
            got = w.run(x.to(dev), None if xs is None else xs.to(dev), None if b is None else b.to(dev)).cpu().numpy()
            want = v @ w.w.T + (0 if b is None else b.double().numpy())
            # products are exact; at most K / 8 + 64 roundings of half a step 2^-24 on the way of a product to the result (the matrix
            # instruction adds at least 8 products at a time; a scale, a zero point, the waves' sums, the bias), each of at most the sum of
            # the magnitudes
            limit = (K / 8 + 64) * 2.0 ** -24 * (np.abs(v) @ w.bound.T + (0 if b is None else np.abs(b.double().numpy())))
            assert (np.abs(got - want) <= limit).all()
            # and as a whole below that: as many roundings of random sign, of partial sums of terms of random sign
            walk = (K / 8 + 64) ** 0.5 * 2.0 ** -24 * np.sqrt((w.bound ** 2).mean() / (w.w ** 2).mean())
            assert np.linalg.norm(got - want) <= walk * np.linalg.norm(want)


@pytest.mark.parametrize("N,K,group", [(1, 32, 32), (5, 64, 64), (17, 160, 128), (50, 1440, 64), (2881, 96, 32)])
def test_int4_any_number_of_rows(pkg, dev, N, K, group):
    w = Weights(pkg, dev, N, K, "int4", group, True, seed=N, exact=True)
    r = np.random.default_rng(K)
    for B in (1, 18):
        x = r.integers(-4, 5, (B, K)).astype(np.float32)
        assert np.array_equal(w.run(torch.from_numpy(x).bfloat16().to(dev)).cpu().numpy(), x.astype(np.float64) @ w.w.T)


@pytest.mark.parametrize("fmt,group", [("mxfp4", 32), ("int4", 64)])
@pytest.mark.parametrize("N,K", [(320, 2880), (4096, 640), (40960, 256)])
def test_rows_are_independent_and_deterministic(pkg, dev, fmt, group, N, K):
    """Same kernel family at every number of rows: a row's bits are those it has alone; a row that is not finite stays its own."""
    w = Weights(pkg, dev, N, K, fmt, group, True, seed=N)
    x = torch.randn((66, K), device=dev, generator=torch.Generator(device=dev).manual_seed(K)).bfloat16()
    y = w.run(x)
    assert torch.equal(y, w.run(x))
    for b in (0, 15, 16, 40, 65):
        assert torch.equal(w.run(x[b:b + 1].contiguous())[0], y[b])
    assert torch.equal(w.run(x[:31].contiguous()), y[:31])
    bad = x.clone()
    bad[3, 5] = float("nan")
    bad[20, K - 1] = float("inf")
    z = w.run(bad)
    keep = [i for i in range(66) if i not in (3, 20)]
    assert torch.equal(z[keep], y[keep])
    assert torch.isnan(z[3]).all() and not torch.isfinite(z[20]).all()


def test_every_code_and_scale(pkg, dev):
    """A one in one place of x reads out one weight: all codes, and every e8m0 byte from 1 that keeps bf16 and fp32 normal."""
    N, K = 256, 64
    codes = np.arange(N, dtype=np.uint8)[:, None] ^ np.arange(K // 2, dtype=np.uint8)[None] * 7
    codes = codes.astype(np.uint8)
    scales = np.clip(np.arange(N)[:, None] + np.array([0, 3]), 2, 250).astype(np.uint8)
    want = opsref.mxfp4_weights(codes, scales)
    t = lambda a: torch.from_numpy(a).to(dev)  # noqa: E731
    tiled = pkg.mxfp4_repack(t(codes).view(1, N, K // 32, 16), t(scales).view(1, N, K // 32))
    y = torch.empty((K, N), device=dev)
    pkg.linear_mxfp4(y, torch.eye(K, device=dev).bfloat16(), *tiled, K, K, N)
    assert np.array_equal(y.cpu().numpy().astype(np.float64), want.T)


def test_workspace_free_graph_and_streams(pkg, dev):
    """Captured with the norm that feeds it, replayed between eager calls; two streams at once."""
    B, K, N = 9, 2880, 1024
    w = Weights(pkg, dev, N, K, "mxfp4", seed=5)
    x = torch.randn((B, K), device=dev)
    d = torch.randn((B, K), device=dev)
    nw = torch.rand(K, device=dev).bfloat16()
    xo, q, qs = torch.empty_like(x), torch.empty((B, K), dtype=torch.uint8, device=dev), torch.empty((B, K // 32), dtype=torch.uint8, device=dev)
    y = torch.empty((B, N), device=dev)

    def step():
        pkg.add_rmsnorm(xo, x, nw, B, K, delta=d, q=q, q_scales=qs)
        pkg.linear_mxfp4(y, q, *w.tiled, B, K, N, x_scales=qs)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        x.copy_(torch.randn((B, K), device=dev) * (i + 1))
        step()
        want = y.clone(), xo.clone()
        y.fill_(float("nan"))
        xo.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[0]) and torch.equal(xo, want[1])
    rows = torch.randn((20, K), device=dev).bfloat16()
    want = w.run(rows)
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.empty((20, N), device=dev) for _ in sides]
    torch.cuda.synchronize()
    for s, o in zip(sides, outs):
        pkg.linear_mxfp4(o, rows, *w.tiled, 20, K, N, stream=s)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
