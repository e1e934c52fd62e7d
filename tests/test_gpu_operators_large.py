"""The operators around the block on tensors whose offsets pass 32 bits: the far end as a call on it alone."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TAIL = 96


def test_route_past_32_bits(pkg, dev):
    E, K = 512, 8
    T = (1 << 31) // E + TAIL  # more than 2^31 logits
    print("route", T, E, flush=True)
    logits = torch.empty((T, E), device=dev).normal_()
    v, i = torch.empty((T, K), device=dev), torch.empty((T, K), dtype=torch.int32, device=dev)
    rule = pkg.RouteRule("sigmoid", None, 8, 4, 2)
    pkg.route(v, i, logits, T, E, K, rule)
    end = logits[-TAIL:].contiguous()
    ve, ie = torch.empty((TAIL, K), device=dev), torch.empty((TAIL, K), dtype=torch.int32, device=dev)
    pkg.route(ve, ie, end, TAIL, E, K, rule)
    assert torch.equal(v[-TAIL:], ve) and torch.equal(i[-TAIL:], ie)


@pytest.mark.parametrize("H,group", [(2880, 32), (20480, 128)])
def test_add_rmsnorm_past_32_bits(pkg, dev, H, group):
    B = (1 << 31) // H + TAIL
    print("add_rmsnorm", B, H, flush=True)
    x, d = torch.empty((B, H), device=dev).normal_(), torch.empty((B, H), device=dev).normal_()
    w = torch.ones(H, device=dev).bfloat16()
    end, d_end = x[-TAIL:].clone(), d[-TAIL:].clone()

    def run(x, d):
        n = x.shape[0]
        q = torch.empty((n, H), dtype=torch.uint8, device=dev)
        s = torch.empty((n, H // group), dtype=torch.uint8 if group == 32 else torch.float32, device=dev)
        pkg.add_rmsnorm(x, x, w, n, H, delta=d, q=q, q_scales=s, q_group=group)
        return x, q, s
    for a, b in zip(run(x, d), run(end, d_end)):
        assert torch.equal(a[-TAIL:], b)


@pytest.mark.parametrize("B", [2, 40])
def test_int4_weights_past_32_bits(pkg, dev, B):
    K, group = 8192, 128
    N = (1 << 32) // (K // 2) + TAIL  # more than 2^32 bytes of codes
    print("int4", N, K, flush=True)
    codes = torch.empty((N, K // 2), dtype=torch.uint8, device=dev).random_(0, 256)
    scales = torch.rand((N, K // group), device=dev).bfloat16()
    zeros = torch.empty((N, K // group), dtype=torch.uint8, device=dev).random_(0, 16)
    x = torch.randn((B, K), device=dev).bfloat16()

    def run(c, s, z):
        n = c.shape[0]
        t = pkg.int4_repack(c, s, z, group)
        y = torch.empty((B, n), device=dev)
        pkg.linear_int4(y, x, t[0], t[1], B, K, n, group, tiled_zeros=t[2])
        return y
    y = run(codes, scales, zeros)
    assert torch.equal(y[:, -TAIL:], run(codes[-TAIL:].contiguous(), scales[-TAIL:].contiguous(), zeros[-TAIL:].contiguous()))


def test_results_past_32_bits(pkg, dev):
    """More than 2^31 values of y."""
    B, K = 65, 64
    N = ((1 << 31) // (B - 1) // 64 + 2) * 64
    print("results", B, N, flush=True)
    codes = torch.empty((1, N, K // 32, 16), dtype=torch.uint8, device=dev).random_(0, 256)
    scales = torch.full((1, N, K // 32), 124, dtype=torch.uint8, device=dev)
    t = pkg.mxfp4_repack(codes, scales)
    x = torch.randn((B, K), device=dev).bfloat16()
    y = torch.empty((B, N), device=dev)
    pkg.linear_mxfp4(y, x, *t, B, K, N)
    n = 128
    te = pkg.mxfp4_repack(codes[:, -n:].contiguous(), scales[:, -n:].contiguous())
    end = torch.empty((B, n), device=dev)
    pkg.linear_mxfp4(end, x, *te, B, K, n)
    assert torch.equal(y[:, -n:], end)
