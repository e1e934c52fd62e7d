"""Rows in 8 bits as bytes and in torch's own types for them."""
import pytest
import torch


def test_types_that_do_not_fit_are_refused(pkg):
    """The looks at the 8-bit tensors alone, on tensors of the host, whose device index is -1."""
    q, s = torch.zeros(2, 64, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8)
    e4m3, e8m0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
    assert pkg._bytes_arg("q", q, e4m3, 128, -1) == pkg._bytes_arg("q", q.view(e4m3), e4m3, 128, -1) == q.data_ptr()
    assert pkg._bytes_arg("s", s.view(e8m0), e8m0, 4, -1) == s.data_ptr() and pkg._bytes_arg("s", None, e8m0, 4, -1) is None
    for bad in (q.view(torch.float8_e5m2), q.view(e8m0), q.view(torch.int8), q[:1], q.view(e4m3)[:1]):
        with pytest.raises(ValueError, match="^q: expected 128 values of torch.uint8"):
            pkg._bytes_arg("q", bad, e4m3, 128, -1)
    with pytest.raises(ValueError, match="^q: expected a contiguous tensor"):
        pkg._bytes_arg("q", torch.zeros(64, 2, dtype=torch.uint8).t(), e4m3, 128, -1)


@pytest.mark.gpu
def test_the_same_bits(pkg, dev):
    B, K, N = 5, 160, 128
    g = torch.Generator(device=dev).manual_seed(1)
    x, w = torch.randn((B, K), device=dev, generator=g), torch.rand(K, device=dev, generator=g).bfloat16()
    codes, scales = torch.randint(0, 256, (1, N, K // 32, 16), dtype=torch.uint8, device=dev, generator=g), torch.full((1, N, K // 32), 124, dtype=torch.uint8, device=dev)
    mx = pkg.mxfp4_repack(codes, scales)
    int4 = pkg.int4_repack(codes.view(N, K // 2), torch.rand((N, 2), device=dev, generator=g).bfloat16(), None, 128)
    out = []
    for e4m3, e8m0 in ((torch.uint8, torch.uint8), (torch.float8_e4m3fn, torch.float8_e8m0fnu)):
        xo, y, z = torch.empty_like(x), torch.empty((B, N), device=dev), torch.empty((B, N), device=dev)
        q, s = torch.empty((B, K), dtype=e4m3, device=dev), torch.empty((B, K // 32), dtype=e8m0, device=dev)
        pkg.add_rmsnorm(xo, x, w, B, K, q=q, q_scales=s)
        pkg.linear_mxfp4(y, q, *mx, B, K, N, x_scales=s)
        pkg.linear_int4(z, q, int4[0], int4[1], B, K, N, 128, x_scales=s)
        out.append((q.view(torch.uint8), s.view(torch.uint8), y, z))
    assert all(torch.equal(a, b) for a, b in zip(*out))
