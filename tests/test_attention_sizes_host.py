"""The most rows that the attention and log probability operators take, without a device: what they refuse, before the first launch."""


def test_prefill_refuses_keys_that_whole_tiles_cannot_count(pkg):
    call = lambda tk, scale=0.125: pkg.lib.moe_attention_prefill(16, 16, 16, 16, 16, 16, 1, 8, tk, 4, 2, 64, 256, 256, 128, 128, 0, scale, None, None)  # noqa: E731
    assert call(0x7FFFFF01) == call(0x7FFFFFFF) == -3
    assert call(0x7FFFFF00, 0.0) == -5  # the largest gets past the sizes: a scale that is none stops it
