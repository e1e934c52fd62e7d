"""moe_token_logprobs with the most rows that it takes."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_the_most_rows(pkg, dev):
    """2^31 - 256 rows of one logit: all the weight is on it. ."""
    T = 0x7FFFFF00
    print("logprobs", T, flush=True)
    logits = torch.zeros((T, 1), dtype=torch.bfloat16, device=dev)
    logits[-3:, 0] = torch.tensor([5.0, -7.0, float("-inf")])
    tokens = torch.zeros(T, dtype=torch.int32, device=dev)
    tokens[[0, T // 2, T - 2]] = torch.tensor([1, -1, 2], dtype=torch.int32, device=dev)  # no such tokens
    out = torch.full((T + 1,), -9.0, device=dev)
    pkg.token_logprobs(logits, tokens, T, 1, logprobs=out)
    bad = torch.tensor([0, T // 2, T - 2, T - 1], device=dev)
    assert torch.isnan(out[bad]).all() and out[T] == -9
    out[bad] = 0
    assert int(torch.count_nonzero(out[:T])) == 0
