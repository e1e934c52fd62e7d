"""The block under a rule with either kind of weights, through the decode and the prefill kernels, with logits summed in one order, and with groups that
leave lanes of the routing kernel idle."""
import numpy as np
import pytest
import torch

from test_gpu_route import torch_block

pytestmark = pytest.mark.gpu


def dense(pkg, raw, blk, fmt):
    """The experts' weights as the kernels use them: bf16 values of either format."""
    if fmt == "bf16":
        return raw
    out = dict(raw)
    for name, rows, k in (("w_mlp1", 2 * blk.I, blk.H), ("w_mlp2", blk.H, blk.I)):
        t, s = blk.tensors[name], blk.tensors[name + "_scales"]
        out[name] = pkg.mxfp4_tiled_to_bf16(t, s, blk.E, rows, k).view(blk.E, rows, k)
    return out


@pytest.mark.parametrize("fmt", ["bf16", "mxfp4"])
@pytest.mark.parametrize("T,E,K,G,keep,flag", [(600, 32, 4, 8, 3, None), (2500, 32, 4, 8, 3, None), (50, 32, 4, 8, 3, "FORCE_TILED"), (5, 32, 4, 8, 3, "ROUTER_STRICT_ORDER"),
                                               (300, 128, 8, 8, 4, "ROUTER_STRICT_ORDER"), (300, 128, 4, 8, 4, None), (41, 128, 4, 1, 1, "FORCE_STREAM"),
                                               (20, 960, 4, 3, 2, None), (70, 960, 4, 3, 2, "FORCE_TILED"), (9, 32, 4, 4, 2, "FORCE_BUCKET_LAUNCH"),
                                               (64, 32, 4, 4, 2, "FUSED_GEMM_LAUNCH")])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_block(pkg, wl, dev, fmt, T, E, K, G, keep, flag, scoring):
    H, I = 128, 64
    flags = getattr(pkg, "MOE_FLAG_" + flag) if flag else 0
    print("block", fmt, T, E, K, G, keep, flag, scoring, flush=True)
    shape = wl.MoeShape("rule", T=T, H=H, I=I, E=E, K=K, fmt=fmt, seed=T + E)
    blk, raw = wl.make_device_layer(shape, pkg.normal_table(), dev)
    x = wl.make_device_input(shape, pkg.normal_table(), dev)
    r = np.random.default_rng(E)
    bias = torch.from_numpy((0.05 * r.standard_normal(E)).astype(np.float32)).to(dev)
    blk.route = rule = pkg.RouteRule(scoring, bias, G, keep, 2, True, 2.5)
    scores, nw = torch.full((T, E), float("nan"), device=dev), (1 + torch.rand(H, device=dev)).bfloat16()
    x0 = torch.randn((T, H), device=dev)
    res, norm = x0.clone(), torch.empty_like(x0)
    y, ti, tv = blk.forward(x, router_score=scores, residual_x=res, next_norm_weight=nw, next_norm_out=norm, flags=flags)
    # the scores are the exact logits, fp32-rounded twice (|logit| < 16, and the bias added), in whatever order they are summed in 64 bits
    exact = x.double() @ raw["w_router"].double().t() + raw["b_router"].double()
    assert (scores.double() - exact).abs().max().item() <= 2.0 ** -20
    v, i = torch.empty((T, K), device=dev), torch.empty((T, K), dtype=torch.int32, device=dev)
    pkg.route(v, i, scores, T, E, K, rule)
    assert torch.equal(i, ti) and torch.equal(v, tv)
    assert torch.equal(res, x0 + y)
    want_norm = torch.empty_like(norm)
    pkg.rmsnorm(want_norm, res, nw, T, H)
    assert torch.equal(norm, want_norm)
    some = torch.unique(torch.linspace(0, T - 1, 24, device=dev).long())
    want = torch_block(wl, shape, dense(pkg, raw, blk, fmt), x[some], ti[some], tv[some])
    # bf16 SwiGLU outputs one step apart, fp32 sums: as for the block's other tests
    assert (y[some].double() - want).abs().max().item() <= 1e-2 * want.abs().max().item()
    # logits in the workspace, and without what follows the block
    y2, ti2, tv2 = blk.forward(x, flags=flags)
    assert torch.equal(y, y2) and torch.equal(ti, ti2) and torch.equal(tv, tv2)


@pytest.mark.parametrize("fmt,T", [("bf16", 3), ("mxfp4", 3), ("bf16", 600), ("mxfp4", 600)])
def test_captured(pkg, wl, dev, fmt, T):
    """Replays between eager calls on other inputs; the captured call's rule object is gone by then."""
    shape = wl.MoeShape("captured", T=T, H=128, I=64, E=32, K=4, fmt=fmt, seed=T)
    blk, _ = wl.make_device_layer(shape, pkg.normal_table(), dev)
    x = wl.make_device_input(shape, pkg.normal_table(), dev)
    bias = 0.05 * torch.randn(32, device=dev)
    out = [torch.empty((T, 128), device=dev), torch.empty((T, 4), dtype=torch.int32, device=dev), torch.empty((T, 4), device=dev)]
    blk.route = pkg.RouteRule("sigmoid", bias, 8, 3, 2, True, 2.5)
    blk.forward(x, *out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        blk.forward(x, *out)
    for n in range(4):
        x.normal_()
        bias.normal_().mul_(0.05)
        blk.route = pkg.RouteRule("sigmoid", bias, 8, 3, 2, True, 2.5)
        want = [t.clone() for t in blk.forward(x)]
        for t in out:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
