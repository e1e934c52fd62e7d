"""The most rows that the attention and log probability operators take, without a device: what they refuse, before the first launch."""


def test_prefill_refuses_keys_that_whole_tiles_cannot_count(pkg):
    call = lambda tk, scale=0.125: pkg.lib.moe_attention_prefill(16, 16, 16, 16, 16, 16, 1, 8, tk, 4, 2, 64, 256, 256, 128, 128, 0, scale, None, None)  # noqa: E731
    assert call(0x7FFFFF01) == call(0x7FFFFFFF) == -3
    assert call(0x7FFFFF00, 0.0) == -5  # the largest gets past the sizes: a scale that is none stops it


def test_scales_that_log2_e_takes_past_fp32_are_refused(pkg):
    import ctypes
    held = pkg.KvCacheParams(ctypes.sizeof(pkg.KvCacheParams), 4, 16, 2, 64, 16, 16, None, None)
    prefill = lambda scale: pkg.lib.moe_attention_prefill(16, 16, 16, 16, 16, 16, 1, 8, 8, 4, 2, 64, 256, 256, 128, 128, 0, scale, 1, None)  # noqa: E731
    decode = lambda scale: pkg.lib.moe_attention_decode(16, 16, ctypes.addressof(held), 16, 16, 2, 4, 4, 0, scale, 1, 16, 1 << 30, None)  # noqa: E731
    for call in (prefill, decode):
        assert call(1.8e38) == call(3.4e38) == -5
        assert call(2.0 ** 127) == call(1e-45) == -6  # past the scale's check: the sinks' address stops them


def test_a_missing_workspace_is_the_library_s_error(pkg, monkeypatch):
    import pytest
    import torch
    monkeypatch.setattr(pkg, "_device", lambda: -1)  # host tensors pass for the current device's: the call ends before it reads them
    z = torch.zeros
    cache = pkg.KvCache(z(4, 2, 16, 64).bfloat16(), z(4, 2, 16, 64).bfloat16())
    q, i = z(2, 4, 64).bfloat16(), z(2, 4, dtype=torch.int32)
    with pytest.raises(pkg.MoeError):
        pkg.attention_decode(q, q, cache, i, i[0], 2, 4, 1.0, None, stream=0)
    with pytest.raises(pkg.MoeError):
        pkg.token_logprobs(z(2, 5000), i, 2, 5000, logprobs=z(2), stream=0)
