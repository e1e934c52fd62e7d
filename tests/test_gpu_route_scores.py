"""Scores of moe_route as numbers of their own: fp64's accuracy, rounded to fp32 once, and the same bits in a batch of any size."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def exponentials(x):
    """exp of 64-bit numbers, in numpy's extended precision (2^-63)."""
    return np.exp(x.astype(np.longdouble))


def assert_rounded(got, exact, sure_share):
    """fp32 of the exact value, unless that lies within 2^-51 of the middle of two fp32 numbers: fp64's roundings of an exponential, a sum and a
    quotient, half a step 2^-53 and a little each."""
    want = exact.astype(np.float32)
    below, above = (exact * (1 - np.longdouble(2) ** -51)).astype(np.float32), (exact * (1 + np.longdouble(2) ** -51)).astype(np.float32)
    sure = below == above
    assert sure.mean() > sure_share
    assert np.array_equal(got[sure], want[sure])


# 2^-26 of random scores are not sure, and those of two logits d < 2^-15 apart (at most 2^-17 of the pairs here): 1/2 + d/4 - d^3/48 is next to a
# multiple of 2^-25
RANDOM = 1 - 2.0 ** -16


def test_sigmoid_scores_next_to_the_middle(pkg, dev):
    """Scores 1/2 - l/4 + l^3/48 of logits -l in steps of 2^-26: every second or so is l^3/48 from the middle of two fp32 numbers."""
    logits = (torch.arange(1, 4096, dtype=torch.float64) * -(2.0 ** -26)).float().to(dev)
    T = logits.numel()
    v, i = torch.empty((T, 1), device=dev), torch.empty((T, 1), dtype=torch.int32, device=dev)
    pkg.route(v, i, logits, T, 1, 1, pkg.RouteRule("sigmoid", renormalize=False))
    assert_rounded(v.cpu().numpy()[:, 0], 1 / (1 + exponentials(-logits.cpu().numpy().astype(np.float64))), 0.5)


@pytest.mark.parametrize("scale", [1.5, 20.0])
def test_sigmoid_scores(pkg, dev, scale):
    T = 1 << 23
    logits = torch.randn(T, device=dev, generator=torch.Generator(device=dev).manual_seed(int(scale))) * scale
    v, i = torch.empty((T, 1), device=dev), torch.empty((T, 1), dtype=torch.int32, device=dev)
    pkg.route(v, i, logits, T, 1, 1, pkg.RouteRule("sigmoid", renormalize=False))
    assert_rounded(v.cpu().numpy()[:, 0], 1 / (1 + exponentials(-logits.cpu().numpy().astype(np.float64))), RANDOM)


@pytest.mark.parametrize("E", [2, 8, 130])
def test_softmax_scores(pkg, dev, E):
    T, K = (1 << 22) // min(E, 8), min(E, 8)
    logits = torch.randn((T, E), device=dev, generator=torch.Generator(device=dev).manual_seed(E)) * 3
    v, i = torch.empty((T, K), device=dev), torch.empty((T, K), dtype=torch.int32, device=dev)
    pkg.route(v, i, logits, T, E, K, pkg.RouteRule("softmax", renormalize=False))
    l = logits.cpu().numpy().astype(np.float64)
    e = exponentials(l - l.max(1, keepdims=True))
    chosen = np.take_along_axis(e / e.sum(1, keepdims=True), i.cpu().numpy().astype(np.int64), 1)
    assert_rounded(v.cpu().numpy(), chosen, RANDOM)


@pytest.mark.parametrize("E,G", [(256, 8), (130, 1), (960, 3), (1000, 1)])
def test_softmax_scores_in_batches_of_any_size(pkg, dev, E, G):
    """4, 16 and more tokens to a block: the rows' bits are those of few."""
    K, T = 8, 40000
    rule = pkg.RouteRule("softmax", None, G, 1, 2, False)
    logits = torch.randn((T, E), device=dev, generator=torch.Generator(device=dev).manual_seed(E)) * 2

    def run(part):
        n = part.shape[0]
        v, i = torch.empty((n, K), device=dev), torch.empty((n, K), dtype=torch.int32, device=dev)
        pkg.route(v, i, part, n, E, K, rule)
        return v, i
    whole = run(logits)
    for size in (500, 2000):
        for at in range(0, T, size):
            v, i = run(logits[at:at + size])
            assert torch.equal(v, whole[0][at:at + size]) and torch.equal(i, whole[1][at:at + size])
