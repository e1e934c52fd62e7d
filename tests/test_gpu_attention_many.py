"""The cache and attention operators on more rows than a launch has blocks, and the most sequences that a call takes."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_rope_kv_write(pkg, dev):
    """The rows of the second launch as a call on them alone."""
    Hq, Hkv, D, tail = 62, 1, 64, 300
    T = (1 << 23) + tail  # 512 units a token, so a block each
    print("rope", T, flush=True)
    qkv = torch.zeros((T, (Hq + 2 * Hkv) * D), dtype=torch.bfloat16, device=dev)
    qkv[-2 * tail :].normal_()
    pos = torch.arange(T, dtype=torch.int32, device=dev)
    inv = torch.rand(D // 2, device=dev)
    page = 1 << 10
    kv = [torch.zeros((T // page + 1, Hkv, page, D), dtype=torch.bfloat16, device=dev) for _ in range(2)]
    k, v = (torch.empty((T, Hkv, D), dtype=torch.bfloat16, device=dev) for _ in range(2))
    pkg.rope_kv_write(None, qkv, pos, inv, T, Hq, Hkv, D, k=k, v=v, cache=pkg.KvCache(*kv), slots=pos)
    n = 2 * tail
    ke, ve = (torch.empty((n, Hkv, D), dtype=torch.bfloat16, device=dev) for _ in range(2))
    pkg.rope_kv_write(None, qkv[-n:], pos[-n:], inv, n, Hq, Hkv, D, k=ke, v=ve)
    assert torch.equal(k[-n:], ke) and torch.equal(v[-n:], ve)
    for held, rows in zip(kv, (k, v)):
        assert torch.equal(held.view(-1, D)[T - n : T], rows[-n:, 0])


@pytest.mark.parametrize("heads", [129, 4])
def test_attention_decode(pkg, dev, heads):
    """65535 sequences of one to three keys on shared pages, a long one among them: those of one key have its value, and rows do not depend on the batch."""
    B, D, page = 65535, 64, 16
    print("decode", heads, flush=True)
    k, v = (torch.randn((40, heads, page, D), device=dev).bfloat16() for _ in range(2))
    cache = pkg.KvCache(k, v)
    table = (torch.arange(B, device=dev, dtype=torch.int32)[:, None] + torch.arange(30, device=dev, dtype=torch.int32)) % 40
    lens = torch.arange(B, device=dev, dtype=torch.int32) % 3 + 1
    lens[B - 9] = 450
    q = torch.randn((B, heads, D), device=dev).bfloat16()
    out = torch.empty_like(q)
    ws = torch.empty(pkg.attention_decode_workspace_bytes(B, heads, heads, D), dtype=torch.uint8, device=dev)
    pkg.attention_decode(out, q, cache, table, lens, B, heads, 0.125, ws)
    one = lens == 1
    assert torch.equal(out[one], v[table[one, 0].long(), :, 0])
    for a, b in ((0, 60), (B - 60, B)):  # in short batches, where a piece is as long
        part = torch.empty_like(q[a:b])
        pkg.attention_decode(part, q[a:b].contiguous(), cache, table[a:b].contiguous(), lens[a:b].contiguous(), b - a, heads, 0.125, ws)
        same = lens[a:b] <= 3
        assert torch.equal(out[a:b][same], part[same])
        # the long one's sum may be cut elsewhere: a few roundings of 2^-24 before the one to bf16, a step of 2^-7 of the value at the most
        d = (out[a:b].float() - part.float()).abs()
        assert (d <= 2.0 ** -7 * part.float().abs() + 2.0 ** -16).all()


def test_attention_prefill(pkg, dev):
    """65535 prompts of one token: each has its value."""
    n, heads, D = 65535, 256, 64
    print("prefill", n, heads, flush=True)
    q = torch.randn((n, heads, D), device=dev).bfloat16()
    k, v = (torch.randn((n, 8, D), device=dev).bfloat16() for _ in range(2))
    starts = torch.arange(n + 1, dtype=torch.int32, device=dev)
    out = torch.empty_like(q)
    pkg.attention_prefill(out, q, k, v, starts, starts, n, heads, 8, D, 0.125)
    assert torch.equal(out.view(n, 8, heads // 8, D), v[:, :, None].expand(n, 8, heads // 8, D))
