"""Blocks that go through many tiles of weight rows: every form of rows and bias, ragged numbers of weight rows, y at any address; every sum exact
in 32 bits, against 64 bits on the device."""
import numpy as np
import pytest
import torch

from test_gpu_linear_w4 import FORMS, Weights, mx8_rows

pytestmark = pytest.mark.gpu


def run(w, x, x_scales, bias, offset):
    """y at `offset` floats from the start of a buffer, which stays as it was around it."""
    B = x.shape[0]
    n = B * w.N
    buffer = torch.full((n + offset + 64,), -7.0, device=w.dev)
    y = buffer[offset:offset + n]
    if w.fmt == "mxfp4":
        w.pkg.linear_mxfp4(y, x, *w.tiled, B, w.K, w.N, bias=bias, x_scales=x_scales)
    else:
        w.pkg.linear_int4(y, x, w.tiled[0], w.tiled[1], B, w.K, w.N, w.group, tiled_zeros=w.tiled[2], bias=bias, x_scales=x_scales)
    assert (buffer[:offset] == -7).all() and (buffer[offset + n:] == -7).all()
    return y.view(B, w.N)


@pytest.mark.parametrize("fmt,group,zeros", FORMS)
@pytest.mark.parametrize("N,K", [(4160, 96), (13056, 64), (20033, 288), (16450, 1184), (13059, 2880), (4800, 8224)])
def test_every_form_of_rows_and_bias(pkg, dev, fmt, group, zeros, N, K):
    """Rows of whole numbers up to 16, a bias of halves up to 32, weights that are multiples of 1/4 up to 12 (MXFP4) or of 1/2 up to 30: partial sums
    are multiples of 1/4 below 16 * 12 * 8224 + 32 < 2^21, or of 1/2 below 16 * 30 * 8224 + 32 < 2^22, and thus exact in any order."""
    if fmt == "mxfp4":
        N = N // 64 * 64
    w = Weights(pkg, dev, N, K, fmt, group, zeros, seed=N + K, exact=True)
    wt = torch.from_numpy(w.w).to(dev).t().contiguous()
    r = np.random.default_rng(N)
    bias = torch.from_numpy(r.integers(-64, 65, N).astype(np.float32) / 2).bfloat16().to(dev)
    for B in (1, 3, 20, 40):
        print("many tiles", fmt, group, zeros, N, K, B, flush=True)
        x = torch.from_numpy(r.integers(-4, 5, (B, K)).astype(np.float32)).bfloat16().to(dev)
        codes, scales, v = mx8_rows(r, B, K, True)
        for rows, xs, values in ((x, None, x.double()), (codes.to(dev), scales.to(dev), torch.from_numpy(v).to(dev))):
            want = values @ wt
            assert torch.equal(run(w, rows, xs, None, 0).double(), want)
            assert torch.equal(run(w, rows, xs, bias, 4).double(), want + bias.double())
            assert torch.equal(run(w, rows, xs, bias, 1).double(), want + bias.double())


@pytest.mark.parametrize("fmt,group", [("mxfp4", 32), ("int4", 32), ("int4", 128)])
@pytest.mark.parametrize("N,K", [(128, 160), (16448, 288)])
def test_rows_in_8_bits_that_are_not_numbers(pkg, dev, fmt, group, N, K):
    """A group with an infinity, as moe_add_rmsnorm writes it: scale byte 255, every code a NaN.  Its row is NaN, the others as without it."""
    w = Weights(pkg, dev, N, K, fmt, group, True, seed=N, exact=True)
    B = 20
    codes, scales, _ = mx8_rows(np.random.default_rng(K), B, K, True)
    want = run(w, codes.to(dev), scales.to(dev), None, 0)
    x = torch.ones((1, K), device=dev)
    x[0, 40] = float("inf")
    q, s = torch.empty((1, K), dtype=torch.uint8, device=dev), torch.empty((1, K // 32), dtype=torch.uint8, device=dev)
    pkg.add_rmsnorm(x, x, torch.ones(K, device=dev).bfloat16(), 1, K, q=q, q_scales=s)
    assert s[0, 1] == 255 and ((q[0, 32:64] & 0x7F) == 0x7F).all()
    for b in (0, 7, 18):
        bad, bad_s = codes.to(dev), scales.to(dev)
        bad[b, 32:64], bad_s[b, 1] = q[0, 32:64], 255
        got = run(w, bad, bad_s, None, 0)
        keep = [i for i in range(B) if i != b]
        assert torch.isnan(got[b]).all() and torch.equal(got[keep], want[keep])
