"""moe_rope_kv_write against its formula in 64 bits."""
import numpy as np
import pytest
import torch

import attnref
import opsref

pytestmark = pytest.mark.gpu

SENTINEL = 0x5A


def make(dev, T, Hq, Hkv, D, rows, seed, stride=None, far=200000):
    r = np.random.default_rng(seed)
    x = (r.standard_normal((T, Hq + 2 * Hkv, D)) * np.exp(r.standard_normal((1, 1, D)))).astype(np.float32)
    x = torch.from_numpy(x).to(torch.bfloat16 if rows == "bf16" else torch.float32)
    wide = torch.full((T, stride or x[0].numel()), 7.0, dtype=x.dtype)
    wide[:, : x[0].numel()] = x.view(T, -1)
    pos = torch.from_numpy(r.integers(0, far, T, dtype=np.int32))
    return x.double().numpy(), wide.to(dev)[:, : x[0].numel()], pos.to(dev)


def check_rows(got, want, bound):
    limit = attnref.U8 * (abs(want) + bound) + bound + 1e-40
    assert (abs(got.double().cpu().numpy() - want) <= limit).all()


def check_mx(codes, scales, want, bound):
    """Values held in 8 bits [.., D] of rows with the given fp32 error: the scale the smallest that does, the codes the nearest."""
    v = opsref.e4m3_values(codes)
    s = np.exp2(scales.astype(np.float64) - 127)
    w, b = (a.reshape(*a.shape[:-1], -1, 32) for a in (want, bound))
    most, off = abs(w).max(-1), b.max(-1)
    assert (448 * s >= most - off).all() and ((scales == 1) | (224 * s < most + off)).all()
    got = v.reshape(w.shape) * s[..., None]
    assert (abs(got - w) <= 2.0 ** -4 * (abs(w) + b) + 2.0 ** -10 * s[..., None] + b).all()


CASES = [  # T, Hq, Hkv, D, R, rows, fmt, page, stride
    (1, 64, 8, 64, 64, "f32", "bf16", 16, None),
    (1, 1, 1, 64, 64, "f32", "mx8", 16, None),
    (7, 8, 2, 128, 128, "bf16", "mx8", 32, None),
    (5, 3, 1, 64, 24, "f32", "bf16", 64, 324),
    (33, 4, 4, 128, 64, "f32", "mx8", 16, 1540),
    (64, 64, 8, 64, 64, "bf16", "mx8", 256, None),
    (300, 6, 2, 128, 8, "bf16", "bf16", 128, 1288),
    (129, 2, 1, 64, 0, "f32", "mx8", 64, None),
    (1000, 16, 2, 64, 64, "f32", "bf16", 1024, None),
]


@pytest.mark.parametrize("T,Hq,Hkv,D,R,rows,fmt,page,stride", CASES)
def test_rows_and_cache(pkg, dev, T, Hq, Hkv, D, R, rows, fmt, page, stride):
    print(T, Hq, Hkv, D, R, rows, fmt, page, stride, flush=True)
    x, qkv, pos = make(dev, T, Hq, Hkv, D, rows, T + D, stride)
    r = np.random.default_rng(3)
    inv = (150000.0 ** (-np.arange(0, R, 2) / max(R, 1))).astype(np.float32)
    n_pages = -(-T // page) + 2
    slots = r.permutation(n_pages * page)[:T].astype(np.int32)
    lost = np.arange(T) % 5 == 3  # tokens that go nowhere
    slots[lost] = np.where(np.arange(T)[lost] % 2, -1 - slots[lost], n_pages * page + slots[lost])
    width = 2 * D if fmt == "bf16" else D
    kv = [torch.full((n_pages, Hkv, page, width), SENTINEL, dtype=torch.uint8, device=dev) for _ in range(2)]
    ss = [torch.full((n_pages, Hkv, page, D // 32), SENTINEL, dtype=torch.uint8, device=dev) for _ in range(2)]
    cache = pkg.KvCache(*[t.view(torch.bfloat16) for t in kv]) if fmt == "bf16" else pkg.KvCache(*kv, *ss)
    q = torch.full((T + 1, Hq, D), -3.0, dtype=torch.bfloat16, device=dev)
    k, v = (torch.full((T + 1, Hkv, D), -3.0, dtype=torch.bfloat16, device=dev) for _ in range(2))
    pkg.rope_kv_write(q, qkv, pos, torch.from_numpy(inv).to(dev), T, Hq, Hkv, D, rotary_dim=R, rope_scale=1.25, k=k, v=v, cache=cache,
                      slots=torch.from_numpy(slots).to(dev))
    p = pos.cpu().numpy()
    qk, bound = attnref.rope(x[:, : Hq + Hkv], p, inv, R, 1.25)
    wv = x[:, Hq + Hkv :]
    check_rows(q[:T], qk[:, :Hq], bound[:, :Hq])
    check_rows(k[:T], qk[:, Hq:], bound[:, Hq:])
    assert torch.equal(v[:T].cpu(), torch.from_numpy(wv).bfloat16())
    assert all((t[T] == -3.0).all() for t in (q, k, v))
    # the cache by slots
    at = slots[~lost]
    flat = [t.cpu().numpy().transpose(0, 2, 1, 3).reshape(n_pages * page, Hkv, -1) for t in (*kv, *ss)]
    rest = np.ones(n_pages * page, bool)
    rest[at] = False
    assert all((f[rest] == SENTINEL).all() for f in (flat if fmt == "mx8" else flat[:2]))
    if fmt == "bf16":
        for f, rows_ in zip(flat, (k, v)):
            assert np.array_equal(f[at], rows_[:T].cpu().view(torch.uint8).numpy()[~lost])
    else:
        check_mx(flat[0][at], flat[2][at], qk[~lost, Hq:], bound[~lost, Hq:])
        for f, s, w in ((flat[1], flat[3], wv),) + (((flat[0], flat[2], x[:, Hq : Hq + Hkv]),) if R == 0 else ()):
            values, scales = opsref.quantise(w[~lost].reshape(-1, D), 32)
            assert np.array_equal(opsref.e4m3_values(f[at]).reshape(-1, D), values)
            assert np.array_equal(np.exp2(s[at].astype(np.float64) - 127).reshape(-1, D // 32), scales)


def test_far_positions_and_parts_asked_for(pkg, dev):
    """Positions up to 2^31 - 1 and negative ones; only what is asked for is written."""
    x, qkv, _ = make(dev, 6, 2, 1, 64, "f32", 1)
    pos = np.array([0, 1, 2**31 - 1, 2**24 + 1, -5, 1000003], np.int32)
    inv = (10000.0 ** (-np.arange(0, 64, 2) / 64)).astype(np.float32)
    want, bound = attnref.rope(x[:, :3], pos, inv, 64, 1.0)
    a, b = pos.astype(np.float64), inv.astype(np.float64)
    turns = abs(a[:, None] * b[None])  # the product and the turns of a position of 31 bits: two roundings of 2^-53 of the angle
    bound += np.concatenate([turns, turns], -1)[:, None] * 2.0 ** -51 * (abs(x[:, :3]) + abs(np.roll(x[:, :3], 32, -1)))
    q, k = torch.empty((6, 2, 64), dtype=torch.bfloat16, device=dev), torch.empty((6, 1, 64), dtype=torch.bfloat16, device=dev)
    args = (qkv, torch.from_numpy(pos).to(dev), torch.from_numpy(inv).to(dev), 6, 2, 1, 64)
    pkg.rope_kv_write(q, *args)
    check_rows(q, want[:, :2], bound[:, :2])
    pkg.rope_kv_write(None, *args, k=k)
    check_rows(k, want[:, 2:], bound[:, 2:])
    with pytest.raises(pkg.MoeError):
        pkg.rope_kv_write(None, *args)


def test_8_bit_groups_with_odd_values(pkg, dev):
    """Zeros, denormals, the largest values; an infinity or a NaN spoils its group alone."""
    T, D = 4, 64
    x = np.zeros((T, 3, D), np.float32)
    x[0, 2, 3] = np.inf
    x[1, 2, 40] = np.nan
    x[1, 2, 5] = 3e38
    x[2, 2, 7], x[2, 2, 8] = 1e-40, 448 * 2.0 ** -126
    x[3, 2, :32], x[3, 2, 32:] = 448.0, 449.0
    x[0, 2, 32:] = 1.0
    kv = [torch.zeros((1, 1, 16, D), dtype=torch.uint8, device=dev) for _ in range(2)]
    ss = [torch.zeros((1, 1, 16, 2), dtype=torch.uint8, device=dev) for _ in range(2)]
    i = torch.arange(T, dtype=torch.int32, device=dev)
    pkg.rope_kv_write(None, torch.from_numpy(x).to(dev).view(T, -1), i, None, T, 1, 1, D, rotary_dim=0, cache=pkg.KvCache(*kv, *ss), slots=i)
    codes, scales = kv[1].cpu().numpy()[0, 0, :T], ss[1].cpu().numpy()[0, 0, :T]
    values, want = opsref.quantise(x[:, 2].astype(np.float64), 32)
    assert np.array_equal(opsref.e4m3_values(codes), values, equal_nan=True)
    assert np.array_equal(np.where(scales == 255, np.nan, np.exp2(scales - 127.0)), want, equal_nan=True)
    assert (scales[0] == (255, 119)).all() and (scales[3] == (127, 128)).all()


def test_past_32_bits(pkg, dev):
    """Rows whose offsets pass 2^31 values and a cache of more than 2^32 bytes: the far end as a call on it alone."""
    Hq, Hkv, D, tail = 2, 1, 64, 50
    stride = 1 << 22
    T = (1 << 31) // stride + tail
    print("rope", T, stride, flush=True)
    buf = torch.zeros(T * stride, device=dev)
    qkv = buf.view(T, stride)[:, : 4 * D]
    qkv.copy_(torch.randn((T, 4 * D), device=dev))
    pos = torch.arange(T, dtype=torch.int32, device=dev)
    inv = torch.rand(32, device=dev)
    page = 1 << 20
    n_pages = (1 << 32) // (page * D * 2) + 1
    kv = [torch.zeros((n_pages, Hkv, page, D), dtype=torch.bfloat16, device=dev) for _ in range(2)]
    slots = n_pages * page - 1 - pos
    q = torch.empty((T, Hq, D), dtype=torch.bfloat16, device=dev)
    pkg.rope_kv_write(q, qkv, pos, inv, T, Hq, Hkv, D, cache=pkg.KvCache(*kv), slots=slots)
    qe, ke, ve = (torch.empty((tail, h, D), dtype=torch.bfloat16, device=dev) for h in (Hq, Hkv, Hkv))
    pkg.rope_kv_write(qe, qkv[-tail:].contiguous(), pos[-tail:].contiguous(), inv, tail, Hq, Hkv, D, k=ke, v=ve)
    assert torch.equal(q[-tail:], qe)
    at = (slots[-tail:] % page).long()
    assert torch.equal(kv[0][-1, 0, at], ke[:, 0]) and torch.equal(kv[1][-1, 0, at], ve[:, 0])
