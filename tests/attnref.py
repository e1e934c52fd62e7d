"""Rotary embedding, attention and log probabilities restated in numpy, in 64 bits, with what the kernels' roundings may add up to."""
import numpy as np

U8, U16, U24 = 2.0 ** -8, 2.0 ** -16, 2.0 ** -24  # half a step of bf16, and of fp32, relative to a value


def rope(x, positions, inv_freq, R, scale):
    """(turned rows, bound of the fp32 error) of heads x [T, H, D]."""
    out, bound = x.copy(), np.zeros_like(x)
    h = R // 2
    a = positions.astype(np.float64)[:, None, None] * inv_freq.astype(np.float64)[None, None, :]
    u, v = x[..., :h], x[..., h:R]
    scale = np.float64(np.float32(scale))
    out[..., :h] = scale * (u * np.cos(a) - v * np.sin(a))
    out[..., h:R] = scale * (v * np.cos(a) + u * np.sin(a))
    # cosine and sine to 2^-22, times scale and the two products rounded: 2^-22 + 3 * 2^-24 of each product, below 2^-21
    bound[..., :h] = bound[..., h:R] = scale * (abs(u) + abs(v)) * 2.0 ** -21
    return out, bound


def softmax_rows(s, sink):
    """Weights of scores s [n], with a sink's score or None; zeros where nothing is visible."""
    m = max(s.max() if len(s) else -np.inf, -np.inf if sink is None else sink)
    if m == -np.inf:
        return np.zeros_like(s)
    e = np.exp(s - m)
    return e / (e.sum() + (0.0 if sink is None else np.exp(sink - m)))


def attention_row(q, k, v, scale, sink):
    """(result, bound) of one query row q [D] over the keys k, v [n, D] that it sees."""
    D, n = q.shape[0], k.shape[0]
    if n == 0:
        return np.zeros(D), np.zeros(D)
    scale = np.float64(np.float32(scale))
    s = scale * (k @ q)
    w = softmax_rows(s, sink)
    o, mean = w @ v, w @ abs(v)
    # a score: D products added in fp32, times scale and log2(e), less the maximum: (D + 4) roundings of up to the sum of the products, which the
    # largest score bounds too; in a weight it counts twice (numerator and sum).  exp2 and the sums over keys, in which a weight takes part in
    # n additions at most: n + 8 roundings, twice.  The weight itself is rounded to bf16
    spread = scale * (abs(k) @ abs(q)).max() + (0.0 if sink is None else abs(sink))
    relative = U8 + 2 * (D + 4) * U24 * spread + 2 * (n + 8) * U24
    error = mean * relative
    return o, error + U8 * (abs(o) + error) + 1e-40


def visible(i, n_q, n_k, window):
    last = i + n_k - n_q
    first = max(0, last - window + 1) if window else 0
    return first, max(first, last + 1)


def logprobs(row):
    """(log p [V], entropy, bound of log p, bound of the entropy) of one row of finite or -infinite logits."""
    row = row.astype(np.float64)
    m = row.max()
    d = row - m
    with np.errstate(invalid="ignore"):
        e = np.exp(d)
        moment = np.where(e > 0, e * d, 0.0)
    ties = (d == 0).sum()
    rest = e[d < 0].sum()
    z = ties + rest
    log_z = np.log1p(ties - 1 + rest)
    logp = d - log_z
    entropy = log_z - moment.sum() / z
    # a term: the difference and its product with log2(e) rounded, exp2 off by up to a step: (2 |d| + 2) half steps; sums: a lane's terms and those of
    # 64 lanes, 8 waves and the parts, fewer than n / 512 + 200 additions of a term
    n = len(row) / 512 + 200
    size = np.where(e > 0, abs(np.where(e > 0, d, 0.0)), 0.0)
    # a term below 2^-126, the least normal number, is 0: |d| is above 87 there, and e |d| falls with |d|, so that its moment is below 88 * 2^-126
    off_rest = U24 * ((e * (2 * size + 2))[d < 0].sum() + n * rest) + len(row) * 2.0 ** -126
    off_moment = U24 * ((e * size * (2 * size + 4)).sum() + n * abs(moment.sum())) + 88 * len(row) * 2.0 ** -126
    off_log = off_rest / z + 4 * U24 * log_z
    off_entropy = off_log + off_moment / z + abs(moment.sum()) / z * (off_rest / z + 2 * U24) + 2 * U24 * (entropy + log_z)
    with np.errstate(invalid="ignore"):
        return logp, entropy, off_log + U24 * abs(logp) + 1e-40, off_entropy + 1e-40
