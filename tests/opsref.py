"""The operators around the block restated in numpy, in 64 bits, a token, row or weight at a time: what moe_route, moe_add_rmsnorm and
moe_linear_* are held to."""
import numpy as np

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6])


def scores(row, scoring):
    """fp32 scores of one token's logits."""
    row = row.astype(np.float64)
    with np.errstate(all="ignore"):
        if scoring == "sigmoid":
            return (1.0 / (1.0 + np.exp(-row))).astype(np.float32)
        if (row == -np.inf).all():
            return np.zeros(len(row), np.float32)
        e = np.exp(row - row.max())
        return (e / e.sum()).astype(np.float32)


def ranked(values, allowed):
    """Allowed indices by value, descending; equal ones ascending, a NaN as +infinity."""
    return sorted(allowed, key=lambda i: (-np.inf if np.isnan(values[i]) else -values[i], i))


def route(logits, K, scoring="softmax", bias=None, n_groups=1, groups_per_token=1, group_top=1, renormalize=True, scale=1.0):
    T, E = logits.shape
    size = E // n_groups
    out_v, out_i = np.zeros((T, K), np.float32), np.zeros((T, K), np.int32)
    for t in range(T):
        s = scores(logits[t], scoring)
        with np.errstate(all="ignore"):
            c = s if bias is None else (s + bias).astype(np.float32)
            value = []
            for g in range(n_groups):
                order = ranked(c, range(g * size, (g + 1) * size))
                value.append(c[order[0]] + c[order[1]] if group_top == 2 and size > 1 else c[order[0]])
            kept = ranked(np.array(value, np.float32), range(n_groups))[:groups_per_token] if n_groups > 1 else [0]
            chosen = ranked(c, [e for g in sorted(kept) for e in range(g * size, (g + 1) * size)])[:K]
            w = s[chosen].astype(np.float64)
            if renormalize:
                w = w * 0 if w.sum() == 0 else w / w.sum()
            out_v[t], out_i[t] = (w * np.float64(np.float32(scale))).astype(np.float32), chosen
    return out_v, out_i


def rmsnorm(x, w, eps):
    """RMSNorm of fp32 rows in 64 bits."""
    x = x.astype(np.float64)
    return w.astype(np.float64) * x / np.sqrt((x * x).mean(1, keepdims=True) + np.float64(np.float32(eps)))


def rmsnorm_products(x, w, eps):
    """The same with the steps that moe_rmsnorm takes in fp32: the squares, the mean, its root and the reciprocal; not rounded."""
    with np.errstate(over="ignore"):
        mean = (x * x).astype(np.float64).mean(1, keepdims=True) + np.float64(np.float32(eps))
        inv = np.float32(1) / np.sqrt(mean.astype(np.float32))
    return w.astype(np.float64) * (inv.astype(np.float64) * x.astype(np.float64))


def to_e4m3(v):
    """Nearest e4m3 value (ties to even) of 64-bit numbers up to 448 and a rounding."""
    a = np.abs(v)
    step = np.exp2(np.maximum(np.floor(np.log2(np.maximum(a, 2.0 ** -60))), -6.0) - 3.0)
    return np.sign(v) * np.minimum(np.round(a / step) * step, 448.0)


def e4m3_values(codes):
    """The values of e4m3 codes: sign, four exponent bits of bias 7, three of mantissa, 0x7F not a number."""
    codes = codes.astype(np.int64)
    e, m = (codes >> 3) & 15, codes & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * np.exp2(e - 10.0))
    v = np.where((codes & 0x7F) == 0x7F, np.nan, v)
    return np.where(codes >> 7, -v, v)


def quantise(y, group):
    """(values the codes stand for without their scale, scales) of rows y in 64 bits by the rule of moe_add_rmsnorm."""
    B, H = y.shape
    n = H if group == 0 else group
    q, scales = np.zeros((B, H)), np.zeros((B, -(-H // n)))
    for b in range(B):
        for i, k in enumerate(range(0, H, n)):
            v = y[b, k:k + n]
            if not np.isfinite(v.astype(np.float32)).all():
                q[b, k:k + n] = scales[b, i] = np.nan
                continue
            a = np.abs(v).max()
            if group == 32:
                p = -126.0
                while np.float64(np.float32(a)) > 448.0 * 2.0 ** p:
                    p += 1
                scales[b, i] = 2.0 ** p
                q[b, k:k + n] = to_e4m3(v / 2.0 ** p)
            else:
                a = np.maximum(a, 2.0 ** -100)
                scales[b, i] = np.float32(a) / np.float32(448)
                q[b, k:k + n] = to_e4m3(v / (a / 448.0))
    return q, scales


def nibbles(codes):
    """[N, K / 2] bytes -> [N, K] codes, low half first."""
    return np.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1)


def mxfp4_weights(codes, scales):
    return E2M1[nibbles(codes)] * np.repeat(np.exp2(scales.astype(np.float64) - 127), 32, 1)


def int4_weights(codes, scales, zeros, group):
    """(weights, and what the products of the kernel's two sums are bounded by per |x|: scale * (16 + code + 16 + zero))"""
    c = nibbles(codes).astype(np.float64)
    K = c.shape[1]
    s = np.repeat(scales.astype(np.float64), group, 1)[:, :K]
    z = np.full_like(c, 8.0) if zeros is None else np.repeat((zeros & 15).astype(np.float64), group, 1)[:, :K]
    return (c - z) * s, (32 + c + z) * np.abs(s)
