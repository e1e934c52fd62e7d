"""Batches of more rows than one launch holds (2^32 threads, which the runtime refuses): rows on both sides of where launches meet, and the last, as in
a batch of their own."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_route(pkg, dev, scoring):
    T, E, K = (1 << 28) + 5, 2, 1  # 16 lanes to a token
    print("route", T, E, scoring, flush=True)
    logits = torch.empty((T, E), device=dev).normal_(generator=torch.Generator(device=dev).manual_seed(1))
    rule = pkg.RouteRule(scoring, renormalize=False)

    def run(part):
        n = part.shape[0]
        v, i = torch.full((n, K), -7.0, device=dev), torch.full((n, K), -7, dtype=torch.int32, device=dev)
        pkg.route(v, i, part, n, E, K, rule)
        return v, i
    v, i = run(logits)
    assert (i >= 0).all() and (i < E).all() and (v > 0).all()
    for at in [0, T - 70] + [(1 << b) - 35 for b in range(24, 29)]:
        for a, b in zip((v, i), run(logits[at:at + 70].clone())):
            assert torch.equal(a[at:at + 70], b)


@pytest.mark.parametrize("B,H,group", [((1 << 26) + 5, 4, 128), ((1 << 23) + 5, 1028, 0)])
def test_add_rmsnorm(pkg, dev, B, H, group):
    """64 and 256 threads to a row."""
    print("add_rmsnorm", B, H, group, flush=True)
    x = torch.empty((B, H), device=dev).normal_(generator=torch.Generator(device=dev).manual_seed(1))
    w = (1 + torch.rand(H, device=dev)).bfloat16()

    def run(part, **kw):
        n = part.shape[0]
        out = torch.empty((n, H), dtype=torch.bfloat16, device=dev)
        q, s = torch.zeros((n, H), dtype=torch.uint8, device=dev), torch.zeros((n, -(-H // (group or H))), device=dev)
        pkg.add_rmsnorm(part, part, w, n, H, o_bf16=out, q=q, q_scales=s, q_group=group, **kw)
        return out, q, s
    got = run(x)
    assert (got[2] > 0).all()
    for at in [0, B - 70] + [(1 << b) - 35 for b in range(20, 27) if (1 << b) + 35 < B]:
        for a, b in zip(got, run(x[at:at + 70].clone())):
            assert torch.equal(a[at:at + 70], b)
