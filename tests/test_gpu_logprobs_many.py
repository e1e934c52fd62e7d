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


def check_selected(l, top, index):
    """The top_k by value, lower indices first, of rows of any size."""
    order = torch.sort(l, dim=-1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(index.long(), order)


def of_kind(kind, T, V, dtype, dev):
    g = torch.Generator(device=dev).manual_seed(V)
    l = 2 * torch.randn((T, V), generator=g, device=dev)
    if kind in ("masked", "clamped"):
        l = torch.where(torch.rand((T, V), generator=g, device=dev) < 40.0 / V, l, float("-inf") if kind == "masked" else -10000.0)
        l[:, V // 2] = 1.0
    if kind == "equal":
        l.fill_(-2.5)
    if kind == "two values":
        l = (l > 4).float()
    if kind == "coarse":
        l = torch.round(l)
    if kind == "ascending":
        l = l.sort(-1).values
    if kind == "descending":
        l = l.sort(-1, descending=True).values
    if kind == "largest last":  # equal ones in front of the border values at a row's end, which are taken first
        l.fill_(-1.0)
        l[:, -100:] = 1.0
    return l.to(dtype)


KINDS = ["random", "masked", "clamped", "equal", "two values", "coarse", "ascending", "descending", "largest last"]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,V", [(600, 20011), (3, 70007), (520, 2500), (1, 300000)])
@pytest.mark.parametrize("kind", KINDS)
def test_selection_of_rows_with_many_equal_logits(pkg, dev, kind, T, V, dtype):
    print(kind, T, V, dtype, flush=True)
    l = of_kind(kind, T, V, dtype, dev)
    lp = torch.log_softmax(l.double(), -1)
    for top in (1, 5, 32):
        best, index = torch.empty((T, top), device=dev), torch.empty((T, top), dtype=torch.int32, device=dev)
        ws = torch.empty(pkg.token_logprobs_workspace_bytes(T, V, top), dtype=torch.uint8, device=dev)
        pkg.token_logprobs(l, None, T, V, top_logprobs=best, top_indices=index, top_k=top, workspace=ws)
        check_selected(l, top, index)
        want = lp.gather(1, index.long())
        # a sum of V terms of up to 1 in lanes and waves: V / 256 + 200 roundings of 2^-24 of log Z's argument at the most, and its own and the result's
        limit = (V / 256 + 200) * 2.0 ** -24 + 2.0 ** -22 * want.abs()
        assert ((best.double() - want).abs() <= limit)[torch.isfinite(want)].all() and torch.equal(torch.isfinite(best), torch.isfinite(want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_time_does_not_hang_on_equal_logits(pkg, dev, dtype):
    """Rows of which most are equal take no longer than others by more than a few times (every value entered into a list one by one: 50 times)."""
    T, V, top = 600, 100000, 20
    best, index = torch.empty((T, top), device=dev), torch.empty((T, top), dtype=torch.int32, device=dev)
    ws = torch.empty(pkg.token_logprobs_workspace_bytes(T, V, top), dtype=torch.uint8, device=dev)
    took = {}
    for kind in KINDS:
        l = of_kind(kind, T, V, dtype, dev)
        times = []
        for _ in range(7):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            pkg.token_logprobs(l, None, T, V, top_logprobs=best, top_indices=index, top_k=top, workspace=ws)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        took[kind] = min(times)
    print(took, flush=True)
    assert all(took[kind] < 10 * took["random"] for kind in KINDS if kind != "ascending"), took
