"""Attention with values as large as its sums have room for, scores and sinks of -infinity."""
import numpy as np
import pytest
import torch

import test_gpu_attention_decode as decode
import test_gpu_attention_prefill as prefill

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("spread", [0.3, 1.0, 3.0])
def test_large_values_in_prompts(pkg, dev, D, spread):
    """Keys times the largest |value| next to 2^115; scores that rise along the keys, so that maxima stay behind."""
    print(D, spread, flush=True)
    n = 500
    c = prefill.Case(pkg, dev, [n], 4, 2, D, 0, True, seed=D, spread=spread)
    rise = torch.linspace(0.5, 1.5, n, device=dev)[:, None, None]
    c.k[:n] = (c.k[:n] * rise).bfloat16()
    c.v[:n] = (2.0 ** 105 * (1 + torch.rand((n, 2, D), generator=torch.Generator().manual_seed(1)))).bfloat16().to(dev)  # up to 2^106, 500 < 2^9
    c.run()
    c.check(rows=[0, 1, 63, 64, 127, 128, 200, 383, 499])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [1, 500, 4000])
def test_large_values_over_a_cache(pkg, dev, D, n):
    """Keys times the largest |value| next to 2^127, whole and in parts."""
    print(D, n, flush=True)
    c = decode.Case(pkg, dev, [n], 4, 2, D, page=16, sinks=True, seed=n)
    room = 127 - int(np.ceil(np.log2(n)))
    v = (2.0 ** (room - 1) * (1 + torch.rand(c.cache.v.shape, generator=torch.Generator().manual_seed(1)))).bfloat16()
    v = torch.where(v >= 2.0 ** room, torch.tensor(2.0 ** room * (1 - 2.0 ** -8)).bfloat16(), v)
    c.v = v.double().numpy()
    c.cache.v.copy_(v.to(dev))
    c.run()
    c.check()


@pytest.mark.parametrize("sink", [float("-inf"), None])
def test_nothing_has_weight(pkg, dev, sink):
    """All scores of -infinity, and sinks of -infinity or none: zeros."""
    inf = float("inf")
    c = decode.Case(pkg, dev, [40, 3000], 4, 2, 64, page=16, seed=1)
    p = prefill.Case(pkg, dev, [70], 4, 2, 64, 0, False, seed=2, behind=0)
    for case in (c, p):
        case.sinks = None if sink is None else torch.full((4,), sink, dtype=torch.bfloat16, device=dev)
        case.q.fill_(1.0)
    c.cache.k.fill_(-inf)
    c.cache.v.fill_(1.0)
    p.k.fill_(-inf)
    c.run()
    p.run()
    assert (c.out[:2] == 0).all() and (p.out == 0).all()


def test_a_sink_of_minus_infinity_is_none(pkg, dev):
    for case in (decode.Case(pkg, dev, [0, 40, 3000], 4, 2, 64, page=16, seed=3), prefill.Case(pkg, dev, [30, 0, 170], 4, 2, 64, 0, False, [-10], seed=4)):
        case.run()
        want = case.out.clone()
        case.sinks = torch.full((4,), float("-inf"), dtype=torch.bfloat16, device=dev)
        case.run()
        assert torch.equal(case.out, want)
