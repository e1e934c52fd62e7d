"""Refusals and sizes of the cache, attention and log probability operators, without a device: every check comes before the first launch."""
import ctypes

import numpy as np
import pytest
import torch

import attnref


def cache(pkg, **kw):
    p = pkg.KvCacheParams(ctypes.sizeof(pkg.KvCacheParams), 4, 16, 2, 64, 16, 16, None, None)
    for k, v in kw.items():
        setattr(p, k, v)
    return ctypes.addressof(p), p


BAD_CACHES = [(dict(struct_bytes=8), -5), (dict(k=None), -1), (dict(v=None), -1), (dict(k_scales=16), -1), (dict(n_pages=0), -2), (dict(page_size=0), -2),
              (dict(page_size=8), -2), (dict(page_size=48), -2), (dict(page_size=-16), -2), (dict(page_size=1 << 21), -3),
              (dict(n_pages=1 << 27), -3), (dict(head_dim=96), -2), (dict(n_kv_heads=0), -2), (dict(n_kv_heads=1025), -3), (dict(k=8), -6), (dict(v=24), -6)]


def test_rope_kv_write_refuses(pkg):
    ok = dict(qkv=16, t=0, stride=384, pos=16, inv=16, T=2, Hq=2, Hkv=2, D=64, R=64, scale=1.0, q=16, k=16, v=16, cache=None, slots=None)

    def call(**kw):
        a = dict(ok, **kw)
        return pkg.lib.moe_rope_kv_write(*[a[n] for n in ok], None)
    good, held = cache(pkg)
    assert call(qkv=None) == call(pos=None) == call(inv=None) == call(slots=16) == call(cache=good) == call(q=None, k=None, v=None) == -1
    assert call(t=2) == -5
    assert call(T=0) == call(R=72) == call(R=12) == call(R=-8) == call(D=32, R=32) == call(Hq=0) == call(Hkv=0) == call(stride=380) == call(stride=386) == -2
    assert call(Hq=1025, stride=1 << 20) == call(T=0x7FFFFF01) == -3
    assert call(qkv=8) == call(q=8) == call(k=4) == call(v=8) == call(pos=2) == call(inv=2) == -6
    for bad, code in BAD_CACHES:
        address, held = cache(pkg, **bad)
        assert call(cache=address, slots=16) == code, bad
    address, held = cache(pkg, n_kv_heads=4)
    assert call(cache=address, slots=16) == -2
    address, held = cache(pkg, k_scales=16, v_scales=16)
    assert call(cache=address, slots=16, R=32) == -2  # a group of 32 values would be turned in part


def test_attention_decode_refuses(pkg):
    good, held = cache(pkg)
    ok = dict(out=16, q=16, cache=good, table=16, lens=16, B=2, Hq=4, max_pages=4, window=0, scale=0.125, sinks=None, ws=16, n=1 << 30)

    def call(**kw):
        a = dict(ok, **kw)
        return pkg.lib.moe_attention_decode(*[a[n] for n in ok], None)
    assert call(out=None) == call(q=None) == call(cache=None) == call(table=None) == call(lens=None) == -1
    assert call(B=0) == call(Hq=3) == call(Hq=0) == call(max_pages=0) == call(window=-1) == -2
    assert call(B=65536) == call(Hq=1026) == call(max_pages=(1 << 26) + 1) == -3
    assert call(ws=None) == call(ws=8) == call(n=pkg.attention_decode_workspace_bytes(2, 4, 2, 64) - 1) == -4
    assert call(scale=0.0) == call(scale=-1.0) == call(scale=float("nan")) == call(scale=float("inf")) == -5
    assert call(out=8) == call(q=8) == call(table=2) == call(lens=2) == call(sinks=1) == -6
    for bad, code in BAD_CACHES:
        address, held = cache(pkg, **bad)
        assert call(cache=address) == code, bad


def test_attention_decode_workspace(pkg):
    f = pkg.attention_decode_workspace_bytes
    assert f(0, 4, 2, 64) == f(2, 3, 2, 64) == f(2, 4, 2, 80) == f(70000, 4, 2, 64) == 0
    for heads in ((64, 8), (1, 1), (40, 8), (1024, 1), (1024, 1024)):
        sizes = [f(b, *heads, 64) for b in (1, 2, 7, 64, 1000, 65535)]
        assert all(a <= b for a, b in zip(sizes, sizes[1:])) and sizes[0] > 0


def test_attention_prefill_refuses(pkg):
    ok = dict(out=16, q=16, k=16, v=16, qs=16, ks=16, n=2, tq=8, tk=8, Hq=4, Hkv=2, D=64, so=256, sq=256, sk=128, sv=128, window=0, scale=0.125, sinks=None)

    def call(**kw):
        a = dict(ok, **kw)
        return pkg.lib.moe_attention_prefill(*[a[n] for n in ok], None)
    assert all(call(**{name: None}) == -1 for name in ("out", "q", "k", "v", "qs", "ks"))
    assert all(call(**bad) == -2 for bad in (dict(n=0), dict(tq=0), dict(tk=0), dict(Hq=3), dict(D=72), dict(window=-1), dict(so=248), dict(sq=248), dict(sk=120),
                                             dict(sv=120), dict(so=260), dict(sk=132)))
    assert call(n=65536) == call(tq=1 << 28) == call(Hq=1026, Hkv=2, so=1 << 20, sq=1 << 20) == call(sk=(1 << 23) + 8) == call(sv=(1 << 23) + 8) == -3
    assert call(scale=0.0) == call(scale=float("nan")) == -5
    assert all(call(**bad) == -6 for bad in (dict(out=8), dict(q=8), dict(k=8), dict(v=8), dict(qs=2), dict(ks=2), dict(sinks=1)))


def test_token_logprobs_refuses(pkg):
    ok = dict(l=16, t=0, stride=100, tokens=16, T=2, V=100, K=3, lp=16, e=16, tl=16, ti=16, ws=None, n=0)

    def call(**kw):
        a = dict(ok, **kw)
        return pkg.lib.moe_token_logprobs(*[a[n] for n in ok], None)
    assert call(l=None) == call(tokens=None) == call(tl=None) == call(ti=None) == call(K=0) == call(lp=None, e=None, tl=None, ti=None, K=0) == -1
    assert call(t=2) == -5
    assert call(T=0) == call(V=0) == call(K=-1) == call(V=2, stride=2) == call(stride=99) == -2
    assert call(K=33) == call(T=0x7FFFFF01) == call(V=(1 << 30) + 1, stride=1 << 31) == -3
    assert call(V=100000, stride=100000) == call(V=100000, stride=100000, ws=8, n=1 << 30) == -4
    assert call(V=100000, stride=100000, ws=16, n=pkg.token_logprobs_workspace_bytes(2, 100000, 3) - 1) == -4
    assert call(l=18) == call(l=17, t=1) == call(tokens=2) == call(lp=2) == call(e=2) == call(tl=2) == call(ti=2) == -6


def test_token_logprobs_workspace(pkg):
    f = pkg.token_logprobs_workspace_bytes
    assert f(0, 100, 3) == f(1, 100, 101) == f(1, 100, 33) == f(5, 2048, 3) == 0
    sizes = [f(t, 131072, 20) for t in (1, 2, 3, 100, 1000, 1023, 1024, 5000)]
    assert all(0 < a <= b for a, b in zip(sizes, sizes[1:]))


def test_wrappers_refuse_tensors_that_do_not_fit(pkg):
    z = torch.zeros
    with pytest.raises(ValueError, match="expected \\[n_pages"):
        pkg.KvCache(z(4, 16, 64), z(4, 16, 64))
    with pytest.raises(ValueError, match="both or neither"):
        pkg.KvCache(z(4, 2, 16, 64), z(4, 2, 16, 64), k_scales=z(4, 2, 16, 2))
    with pytest.raises(ValueError, match="k: expected 8192 values of torch.bfloat16"):
        pkg.KvCache(z(4, 2, 16, 64), z(4, 2, 16, 64))
    with pytest.raises(ValueError, match="k_scales: expected 256 values"):
        c = z(4, 2, 16, 64, dtype=torch.uint8)
        pkg.KvCache(c, c, z(4, dtype=torch.uint8), z(4, dtype=torch.uint8))
    c = pkg.KvCache(z(4, 2, 16, 64).bfloat16(), z(4, 2, 16, 64).bfloat16())
    i = z(2, 4, dtype=torch.int32)
    with pytest.raises(ValueError, match="qkv: expected 2 rows of 512 values"):
        pkg.rope_kv_write(None, z(2, 500), i, None, 2, 4, 2, 64)
    with pytest.raises(ValueError, match="page_table: expected \\[batch, max_pages\\]"):
        pkg.attention_decode(None, None, c, i[0], i[0], 2, 4, 1.0, None)
    with pytest.raises(ValueError, match="current device"):
        pkg.attention_decode(z(2, 4, 64).bfloat16(), z(2, 4, 64).bfloat16(), c, i, i[0], 2, 4, 1.0, z(8, dtype=torch.uint8))
    with pytest.raises(ValueError, match="out: expected 2 rows of 256 values"):
        pkg.attention_prefill(z(2, 3, 64).bfloat16(), z(2, 4, 64).bfloat16(), z(2, 2, 64).bfloat16(), z(2, 2, 64).bfloat16(), i, i, 1, 4, 2, 64, 1.0)
    with pytest.raises(ValueError, match="logits: expected 3 rows of 64 values"):
        pkg.token_logprobs(z(2, 64), i, 3, 64)
    with pytest.raises(ValueError, match="logits: expected 2 rows of 64 values of torch.float32, got \\(2, 64\\) of torch.float16"):
        pkg.token_logprobs(z(2, 64).half(), i, 2, 64)


def test_reference_agrees_with_torch():
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(n, 64, generator=g, dtype=torch.float64) for n in (5, 7, 7))
    # query i of 5 sees the keys up to i + 2
    mask = torch.ones(5, 7, dtype=torch.bool).tril(2)
    want = torch.nn.functional.scaled_dot_product_attention(q, k, v, attn_mask=mask, scale=0.25)
    for i in range(5):
        a, b = attnref.visible(i, 5, 7, 0)
        got, _ = attnref.attention_row(q[i].numpy(), k[a:b].numpy(), v[a:b].numpy(), 0.25, None)
        assert np.allclose(got, want[i].numpy(), rtol=1e-13)
    l = 3 * torch.randn(1000, generator=g, dtype=torch.float64)
    logp, entropy, _, _ = attnref.logprobs(l.numpy())
    assert np.allclose(logp, torch.log_softmax(l, 0).numpy(), rtol=1e-13)
    assert np.isclose(entropy, torch.distributions.Categorical(logits=l).entropy().item(), rtol=1e-12)
