"""moe_route against a token-at-a-time restatement: both scorings, bias, groups, ties, masked and non-finite logits, and the block that
runs with a rule."""
import numpy as np
import pytest
import torch

import opsref

pytestmark = pytest.mark.gpu


def run(pkg, dev, logits, K, **kw):
    T, E = logits.shape
    bias = kw.pop("bias", None)
    rule = pkg.RouteRule(balance_bias=None if bias is None else torch.from_numpy(bias).to(dev), **kw)
    v = torch.full((T + 1, K), -7.0, device=dev)
    i = torch.full((T + 1, K), -7, dtype=torch.int32, device=dev)
    pkg.route(v, i, torch.from_numpy(logits).to(dev), T, E, K, rule)
    assert (v[T] == -7).all() and (i[T] == -7).all()  # rows behind the last are left alone
    return v[:T].cpu().numpy(), i[:T].cpu().numpy()


def check(pkg, dev, logits, K, **kw):
    v, i = run(pkg, dev, logits, K, **dict(kw))
    wv, wi = opsref.route(logits, K, **kw)
    assert np.array_equal(i, wi)
    # half a step for the final rounding, one for a score next to a border that two exponentials round differently
    assert np.array_equal(np.isnan(v), np.isnan(wv))
    assert (np.abs(v - wv) <= 1.5 * 2.0 ** -23 * np.abs(wv))[~np.isnan(wv)].all()


def logits_of(T, E, seed):
    r = np.random.default_rng(seed)
    return (r.standard_normal((T, E)) * 1.5).astype(np.float32), (r.standard_normal(E) * 0.1).astype(np.float32)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,K", [(1, 1, 1), (3, 5, 5), (65, 8, 2), (130, 32, 4), (33, 64, 8), (7, 65, 6), (40, 128, 8), (5, 160, 8), (9, 256, 8),
                                   (6, 300, 3), (5, 513, 8), (4, 1000, 8), (3, 1024, 1)])
def test_route(pkg, dev, scoring, T, E, K):
    logits, bias = logits_of(T, E, T + E)
    for b in (None, bias):
        for renorm, scale in ((True, 1.0), (False, 2.5)):
            check(pkg, dev, logits, K, scoring=scoring, bias=b, renormalize=renorm, scale=scale)


@pytest.mark.parametrize("E,G,keep,K", [(8, 8, 3, 3), (16, 2, 1, 8), (32, 4, 2, 4), (64, 8, 4, 6), (64, 64, 8, 8), (120, 5, 3, 8), (160, 8, 3, 6), (256, 8, 4, 8),
                                        (256, 2, 2, 8), (512, 16, 1, 8), (960, 3, 2, 8), (1024, 64, 2, 8), (66, 33, 7, 8), (1000, 10, 10, 8), (990, 33, 4, 8),
                                        (36, 3, 2, 5), (100, 10, 3, 8), (200, 2, 1, 7), (768, 2, 1, 8), (72, 9, 4, 6)])
def test_route_groups(pkg, dev, E, G, keep, K):
    logits, bias = logits_of(37, E, E + G)
    for top in (1, 2):
        check(pkg, dev, logits, K, scoring="sigmoid", bias=bias, n_groups=G, groups_per_token=keep, group_top=top, scale=2.5)
    check(pkg, dev, logits, K, scoring="softmax", n_groups=G, groups_per_token=keep, renormalize=False)


@pytest.mark.parametrize("T", [1601, 3307])  # 32 and 16 lanes to a token
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,G,keep,K", [(5, 1, 1, 2), (16, 4, 2, 4), (32, 1, 1, 4), (60, 5, 2, 6), (128, 8, 3, 8), (192, 8, 4, 8), (256, 8, 4, 8), (256, 1, 1, 8),
                                        (258, 3, 2, 8), (400, 16, 5, 8), (512, 32, 3, 8), (768, 1, 1, 8), (1024, 8, 4, 8), (990, 33, 4, 8)])
def test_many_tokens_as_few(pkg, dev, scoring, E, G, keep, K, T):
    """Batches large enough for several tokens to a wave: the bits of the same rows in small batches, and those of the restatement."""
    logits, bias = logits_of(T, E, E + G)
    kw = dict(scoring=scoring, bias=bias, n_groups=G, groups_per_token=keep, group_top=2, scale=2.5)
    v, i = run(pkg, dev, logits, K, **dict(kw))
    for a, b in ((0, 30), (1000, 1031), (T - 33, T)):
        sv, si = run(pkg, dev, logits[a:b].copy(), K, **dict(kw))
        assert np.array_equal(i[a:b], si) and np.array_equal(v[a:b], sv)
        check(pkg, dev, logits[a:b].copy(), K, **dict(kw))


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_ties_go_to_the_lower_index(pkg, dev, scoring):
    for E, G, keep in ((12, 1, 1), (64, 8, 3), (256, 8, 4), (1024, 16, 5)):
        logits = np.zeros((5, E), np.float32)
        logits[1, ::3] = 1.0
        logits[2] = -np.arange(E) // 4
        logits[3] = np.arange(E) // 4
        logits[4, -1] = -0.0
        check(pkg, dev, logits, 4, scoring=scoring, n_groups=G, groups_per_token=keep, group_top=2)
        check(pkg, dev, logits, 4, scoring=scoring, n_groups=G, groups_per_token=keep, bias=np.full(E, -0.5, np.float32))


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T", [9, 1700, 3300])
@pytest.mark.parametrize("E,G,keep", [(16, 1, 1), (64, 8, 2), (256, 8, 4), (320, 4, 3), (960, 3, 2)])
def test_route_masked_and_far_logits(pkg, dev, scoring, E, G, keep, T):
    lowest = np.finfo(np.float32).min
    logits, bias = logits_of(9, E, E)
    logits[0] = -np.inf                  # nothing to choose from
    logits[1] = lowest                   # the type's lowest value everywhere
    logits[2, : E - 3] = -np.inf         # fewer experts than are wanted
    logits[3, ::2] = lowest
    logits[4] *= 200                     # scores that underflow, and that round to one
    logits[5, 1] = np.nan
    logits[6, E - 1] = np.nan
    if scoring == "sigmoid":
        logits[7, 2] = np.inf
    bias[3] = -np.inf                    # an expert that is switched off
    for b in (None, bias):
        for renorm in (True, False):
            kw = dict(scoring=scoring, n_groups=G, groups_per_token=keep, group_top=2, renormalize=renorm)
            check(pkg, dev, logits, 4, bias=b, **kw)
            many = np.concatenate([logits, logits_of(T - 9, E, 1)[0]])
            v, i = run(pkg, dev, many, 4, bias=b, **kw)
            assert np.array_equal(i[:9], opsref.route(logits, 4, bias=b, **kw)[1])
            assert (i >= 0).all() and (i < E).all() and all(len(set(r)) == 4 for r in i)
    v, _ = run(pkg, dev, logits, 4, scoring="softmax")
    assert (v[0] == 0).all()


def test_route_large_batch_and_streams(pkg, dev):
    """Every row of a large batch as the same rows alone, on two streams at once and from a replayed graph."""
    T, E, K = 20001, 256, 8
    logits = torch.randn((T, E), device=dev, generator=torch.Generator(device=dev).manual_seed(1))
    bias = 0.1 * torch.randn(E, device=dev, generator=torch.Generator(device=dev).manual_seed(2))
    rule = pkg.RouteRule("sigmoid", bias, 8, 4, 2, True, 2.5)
    v, i = torch.empty((T, K), device=dev), torch.empty((T, K), dtype=torch.int32, device=dev)
    pkg.route(v, i, logits, T, E, K, rule)
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    out = [(torch.empty((500, K), device=dev), torch.empty((500, K), dtype=torch.int32, device=dev)) for _ in sides]
    starts = (0, T - 500)
    parts = [logits[s:s + 500].contiguous() for s in starts]
    torch.cuda.synchronize()
    for st, o, p in zip(sides, out, parts):
        pkg.route(o[0], o[1], p, 500, E, K, rule, stream=st)
    torch.cuda.synchronize()
    for s, o in zip(starts, out):
        assert torch.equal(o[0], v[s:s + 500]) and torch.equal(o[1], i[s:s + 500])
    sv, si = opsref.route(logits[:64].cpu().numpy(), K, "sigmoid", bias.cpu().numpy(), 8, 4, 2, True, 2.5)
    assert np.array_equal(i[:64].cpu().numpy(), si)


def torch_block(wl, shape, raw, x, ti, tv):
    """The experts of given routing in 64 bits: rows and SwiGLU outputs rounded to bf16, as the block does."""
    w1, b1 = raw["w_mlp1"].double(), raw["b_mlp1"].double()
    w2, b2 = raw["w_mlp2"].double(), raw["b_mlp2"].double()
    out = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    xr = x.bfloat16().double()
    for t in range(x.shape[0]):
        for k in range(ti.shape[1]):
            e = int(ti[t, k])
            z = (w1[e] * xr[t]).sum(1) + b1[e]
            gate, up = z[0::2].clamp(max=7.0), z[1::2].clamp(-7.0, 7.0)
            h = (gate * torch.sigmoid(1.702 * gate) * (up + 1)).bfloat16().double()
            out[t] += ((w2[e] * h).sum(1) + b2[e]) * tv[t, k].double()
    return out


@pytest.mark.parametrize("T", [1, 7, 33, 200])
def test_block_with_a_rule(pkg, wl, dev, T):
    E, K, H, I = 32, 4, 256, 128
    shape = wl.MoeShape("rule", T=T, H=H, I=I, E=E, K=K, fmt="bf16", seed=T)
    blk, raw = wl.make_device_layer(shape, pkg.normal_table(), dev)
    x = wl.make_device_input(shape, pkg.normal_table(), dev)
    bias = 0.05 * torch.randn(E, device=dev, generator=torch.Generator(device=dev).manual_seed(3))
    plain = blk.forward(x)
    # probabilities over all experts, renormalised over the chosen: softmax over the chosen
    blk.route = pkg.RouteRule("softmax")
    y, ti, tv = blk.forward(x)
    assert torch.equal(ti, plain[1])
    # scores rounded to 32 bits, divided, rounded; the block's own are rounded exponentials, divided, rounded; logits rounded up to 2^-24
    # of |logit| < 16 move both: 2^-21
    assert ((tv - plain[2]).abs() <= 2.0 ** -21 * plain[2]).all()
    assert (y - plain[0]).abs().max().item() <= 1e-5 * max(1.0, plain[0].abs().max().item())
    logits = torch.empty((T, E), device=dev)
    pkg.gemm_router(logits, x, raw["w_router"], raw["b_router"], T, H, E)
    rule = pkg.RouteRule("sigmoid", bias, 8, 3, 2, True, 2.5)
    blk.route = rule
    scores = torch.empty((T, E), device=dev)
    x0 = torch.randn((T, H), device=dev)
    res = x0.clone()
    y, ti, tv = blk.forward(x, router_score=scores, residual_x=res)
    assert torch.equal(res, x0 + y)
    assert (scores - logits).abs().max().item() <= 2.0 ** -20  # |logit| < 16, rounded and the bias added
    v, i = torch.empty((T, K), device=dev), torch.empty((T, K), dtype=torch.int32, device=dev)
    pkg.route(v, i, scores, T, E, K, rule)
    assert torch.equal(i, ti) and torch.equal(v, tv)
    y2, ti2, tv2 = blk.forward(x)  # logits in the workspace
    assert torch.equal(y, y2) and torch.equal(ti, ti2) and torch.equal(tv, tv2)
    want = torch_block(wl, shape, raw, x, ti, tv)
    # bf16 SwiGLU outputs one step apart, fp32 sums: as for the block's other tests
    assert (y.double() - want).abs().max().item() <= 1e-2 * want.abs().max().item()
    name = blk.describe(blk.params(x, y, ti, tv))["router"]
    assert name.endswith("+ route_kernel")
