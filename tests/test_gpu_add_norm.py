"""moe_add_rmsnorm against 64-bit arithmetic: every row length class, output and scale form, non-finite and tiny rows."""
import numpy as np
import pytest
import torch

import opsref

pytestmark = pytest.mark.gpu

GROUPS = [32, 128, 0]


def call(pkg, dev, x, w, group, delta=None, eps=1e-5, in_place=False, want=("o", "o_bf16", "q")):
    B, H = x.shape
    pad = 64
    bufs = {"o": torch.full((B * H + pad,), -7.0, device=dev), "o_bf16": torch.full((B * H + pad,), -7.0, dtype=torch.bfloat16, device=dev),
            "q": torch.full((B * H + pad,), 77, dtype=torch.uint8, device=dev)}
    n = B * (1 if group == 0 else -(-H // group))
    scales = torch.full((n + pad,), 77, dtype=torch.uint8 if group == 32 else torch.float32, device=dev)
    xo = x.clone() if in_place else torch.full((B, H), float("nan"), device=dev)
    kw = {k: bufs[k] for k in want}
    if "q" in want:
        kw.update(q_scales=scales, q_group=group)
    pkg.add_rmsnorm(xo, xo if in_place else x, w, B, H, delta=delta, eps=eps, **kw)
    for k, b in bufs.items():
        guard = 77 if k == "q" else -7.0
        assert (b[B * H:] == guard).all() and (k in want or (b == guard).all()), k
    assert (scales[n:] == 77).all()
    got = {k: b[: B * H].view(B, H) for k, b in bufs.items()}
    return xo, got, scales[:n].view(B, -1)


def check(pkg, dev, x, w, group, delta=None, eps=1e-5, in_place=False):
    xo, got, scales = call(pkg, dev, x, w, group, delta, eps, in_place)
    want_x = x + delta if delta is not None else x
    assert torch.equal(xo, want_x)
    y = got["o"].cpu().numpy()
    ref = opsref.rmsnorm(want_x.cpu().numpy(), w.float().cpu().numpy(), eps)
    # relative: fp32 squares and the rounding of their mean, halved by the root: 2^-24; root, quotient and result: half a step each
    assert (np.abs(y - ref) <= 4 * 2.0 ** -24 * np.abs(ref) + 2.0 ** -149).all()
    assert torch.equal(got["o_bf16"], got["o"].bfloat16())
    # the restatement's sum of squares is the kernel's up to 64-bit roundings, which move the fp32 mean once in 10^8 rows
    t = opsref.rmsnorm_products(want_x.cpu().numpy(), w.float().cpu().numpy(), eps)
    assert np.array_equal(t.astype(np.float32), y)
    wq, ws = opsref.quantise(t, group)
    gs = scales.cpu().numpy()
    gs = np.exp2(gs.astype(np.float64) - 127) if group == 32 else gs.astype(np.float64)
    assert np.array_equal(gs, ws)
    assert np.array_equal(opsref.e4m3_values(got["q"].cpu().numpy()), wq)
    return got


def rows(dev, B, H, seed, scale=4.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn((B, H), device=dev, generator=g) * scale * torch.exp(torch.randn((1, H), device=dev, generator=g))
    d = torch.randn((B, H), device=dev, generator=g)
    w = (1 + 0.2 * torch.randn(H, device=dev, generator=g)).bfloat16()
    return x, d, w


@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("B,H", [(1, 32), (3, 64), (2, 96), (5, 992), (4, 1024), (4, 1056), (3, 2880), (2, 4096), (2, 4128), (2, 5120), (1, 8192), (2, 16384),
                                 (1, 16416), (1, 40000)])
def test_add_rmsnorm(pkg, dev, group, B, H):
    x, d, w = rows(dev, B, H, B + H)
    a = check(pkg, dev, x, w, group, d)
    b = check(pkg, dev, x, w, group, d, in_place=True)
    assert all(torch.equal(a[k], b[k]) for k in a)
    check(pkg, dev, x, w, group, None, eps=1e-6)
    # a row does not depend on the rows around it
    for r in range(B):
        _, one, _ = call(pkg, dev, x[r:r + 1].contiguous(), w, group, d[r:r + 1].contiguous())
        assert all(torch.equal(one[k][0], a[k][r]) for k in a)


@pytest.mark.parametrize("group", [128, 0])
@pytest.mark.parametrize("H", [4, 36, 132, 260, 2884, 4100])
def test_odd_lengths(pkg, dev, group, H):
    x, d, w = rows(dev, 3, H, H)
    check(pkg, dev, x, w, group, d)


@pytest.mark.parametrize("H", [64, 2880, 5120])
def test_each_output_alone(pkg, dev, H):
    x, d, w = rows(dev, 3, H, H)
    _, every, scales = call(pkg, dev, x, w, 32, d)
    for k in ("o", "o_bf16", "q"):
        _, one, s = call(pkg, dev, x, w, 32, d, want=(k,))
        assert torch.equal(one[k], every[k]) and (k != "q" or torch.equal(s, scales))


def test_same_bits_as_rmsnorm(pkg, dev):
    for H in (64, 260, 512, 1024, 1028, 2048, 2880, 4096):
        x, _, w = rows(dev, 9, H, H)
        want = torch.empty_like(x)
        pkg.rmsnorm(want, x, w, 9, H)
        assert torch.equal(call(pkg, dev, x, w, 0)[1]["o"], want)


@pytest.mark.parametrize("B,H", [(30000, 1024), (8000, 2880), (3000, 8192), (1500, 16384)])
def test_rows_past_the_cache(pkg, dev, B, H):
    """More than 256 MiB of rows take other loads and stores: the bits of parts of the batch."""
    x, d, w = rows(dev, B, H, H)
    for group in GROUPS:
        xo, got, scales = call(pkg, dev, x, w, group, d)
        for a, b in ((0, 50), (B // 2, B // 2 + 50), (B - 50, B)):
            po, part, ps = call(pkg, dev, x[a:b].contiguous(), w, group, d[a:b].contiguous())
            assert torch.equal(po, xo[a:b]) and torch.equal(ps, scales[a:b]) and all(torch.equal(part[k], got[k][a:b]) for k in got)


@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("H", [256, 2880, 4352])
def test_zero_tiny_and_wide_rows(pkg, dev, group, H):
    x, _, w = rows(dev, 6, H, H)
    x[0] = 0
    x[1] *= 1e-30            # the mean is eps alone
    x[2, 5:] *= 1e-18        # groups far below the row's largest value
    x[3] *= 1e15
    x[4, : H // 2] = 0
    w[7] = 0
    check(pkg, dev, x, w, group)


@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("H", [256, 2880, 4352])
def test_scale_borders(pkg, dev, group, H):
    """Largest values at, just below and just above 448 times a power of two: y = x where the mean square is one and eps nothing."""
    x = torch.ones((3, H), device=dev)
    w = torch.ones(H, dtype=torch.bfloat16, device=dev)
    w[::32] = 1.75
    w[32::64] = 1.7578125
    w[100::128] = 224.0
    check(pkg, dev, x, w, group, eps=0.0)


@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("H", [256, 2880, 4352])
def test_non_finite_rows(pkg, dev, group, H):
    x, _, w = rows(dev, 4, H, H)
    x[1, 70] = float("inf")
    x[2, 3] = float("nan")
    _, got, scales = call(pkg, dev, x, w, group)
    q, o = got["q"].cpu().numpy(), got["o"]
    s = scales.cpu().numpy()
    for r in (1, 2):  # inf * 0 where the value itself is infinite, 0 for the others of its row; every value of a NaN's row
        n = H if group == 0 else group
        for i, k in enumerate(range(0, H, n)):
            finite = bool(torch.isfinite(o[r, k:k + n]).all())
            v = opsref.e4m3_values(q[r, k:k + n])
            assert np.isfinite(v).all() if finite else np.isnan(v).all()
            assert (s[r, i] != 255 if group == 32 else np.isfinite(s[r, i])) if finite else (s[r, i] == 255 if group == 32 else np.isnan(s[r, i]))
    good, gq, gs = call(pkg, dev, x[[0, 3]].contiguous(), w, group)
    assert torch.equal(gq["q"], got["q"][[0, 3]]) and torch.equal(gs, scales[[0, 3]])
