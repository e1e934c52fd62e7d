"""moe_attention_prefill with windows as long as a sequence and longer, up to the largest, also where there are more queries than keys."""
import pytest
import torch

import test_gpu_attention_prefill as prefill

pytestmark = pytest.mark.gpu

LENS, CONTEXT = [40, 300, 5, 150], [-20, -170, 60, 0]  # 20, 130, 65 and 150 keys


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window", [2**31 - 1, 2**31 - 2, 2**31 - 100, 2**30, 365 + 3, 365, 150])
def test_a_window_past_all_keys_is_none(pkg, dev, D, window):
    print(D, window, flush=True)
    c = prefill.Case(pkg, dev, LENS, 4, 2, D, window, True, CONTEXT, seed=D)
    c.run()
    c.check()
    out = c.out.clone()
    c.window = 0
    c.run()
    assert torch.equal(c.out, out)


@pytest.mark.parametrize("window", [149, 131, 130, 129, 66, 65, 64, 20, 19])
def test_windows_around_the_sequences_lengths(pkg, dev, window):
    print(window, flush=True)
    c = prefill.Case(pkg, dev, LENS, 2, 1, 64, window, False, CONTEXT, seed=window)
    c.run()
    c.check()
