"""Rows in 8 bits: every code with every scale byte, as one weight reads it out."""
import numpy as np
import pytest
import torch

import opsref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N", [64, 16448])  # a tile to a block, and several
@pytest.mark.parametrize("fmt", ["mxfp4", "int4"])
def test_every_code_and_scale_byte(pkg, dev, fmt, N):
    """Row c holds code c and zeros; the weights are a power of two that keeps the result a normal number.  It is the code times 2^(byte - 127)
    rounded to bf16 (to nearest even; no rounding from 2^-126 on)."""
    K = 32
    codes = np.arange(256, dtype=np.uint8)
    rows = np.zeros((256, K), np.uint8)
    rows[:, 5] = codes
    rows = torch.from_numpy(rows).to(dev)
    y = torch.empty((256, N), device=dev)
    for power in (20, -27):
        if fmt == "mxfp4":
            w = pkg.mxfp4_repack(torch.full((1, N, 1, 16), 0x22, dtype=torch.uint8, device=dev), torch.full((1, N, 1), 127 + power, dtype=torch.uint8, device=dev))
        else:
            w = pkg.int4_repack(torch.full((N, K // 2), 0x99, dtype=torch.uint8, device=dev), torch.full((N, 1), 2.0 ** power, device=dev).bfloat16(), None, 32)
        for b in range(0, 100) if power == 20 else range(100, 256):
            scales = torch.full((256, 1), b, dtype=torch.uint8, device=dev)
            if fmt == "mxfp4":
                pkg.linear_mxfp4(y, rows, *w, 256, K, N, x_scales=scales)
            else:
                pkg.linear_int4(y, rows, w[0], w[1], 256, K, N, 32, x_scales=scales)
            with np.errstate(over="ignore"):
                x = (opsref.e4m3_values(codes) * (2.0 ** (b - 127) if b < 255 else np.nan)).astype(np.float32)
            want = torch.from_numpy(x).bfloat16().double() * 2.0 ** power
            got = y.double().cpu()
            assert torch.equal(got.nan_to_num(nan=7.0), want[:, None].expand(256, N).nan_to_num(nan=7.0)), b
