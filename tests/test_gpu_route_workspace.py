"""The block under a rule that keeps its logits in the workspace: over the experts' rows, or behind them where these are shorter."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,H,I,E,K", [(5, 64, 64, 128, 1), (70, 64, 64, 256, 1), (70, 256, 128, 32, 4)])
@pytest.mark.parametrize("fmt", ["bf16", "mxfp4"])
def test_logits_in_the_workspace(pkg, wl, dev, T, H, I, E, K, fmt):
    shape = wl.MoeShape("workspace", T=T, H=H, I=I, E=E, K=K, fmt=fmt, seed=T)
    blk, _ = wl.make_device_layer(shape, pkg.normal_table(), dev)
    x = wl.make_device_input(shape, pkg.normal_table(), dev)
    behind = 4 * T * E > T * K * (2 * I + 4 * H)
    assert pkg.block_workspace_bytes(T, H, I, E, K) <= blk.workspace.numel()
    plain = [t.clone() for t in blk.forward(x)]
    blk.route = pkg.RouteRule("sigmoid", None, 8, 4, 2, True, 2.5)
    scores = torch.empty((T, E), device=dev)
    want = [t.clone() for t in blk.forward(x, router_score=scores)]
    got = blk.forward(x)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # what a block without a rule needs, guarded: enough without a rule, and with one that has its logits elsewhere
    whole = pkg.block_workspace_bytes(T, H, I, E, K)
    least = whole - (T * E * 4 + 255) // 256 * 256 if behind else whole
    guarded = torch.full((least + 256,), 0x5A, dtype=torch.uint8, device=dev)
    blk.workspace = guarded[:least]
    assert all(torch.equal(a, b) for a, b in zip(blk.forward(x, router_score=scores), want))
    if behind:
        with pytest.raises(pkg.MoeError):
            blk.forward(x)
    else:
        assert all(torch.equal(a, b) for a, b in zip(blk.forward(x), want))
    blk.route = None
    assert all(torch.equal(a, b) for a, b in zip(blk.forward(x), plain))
    torch.cuda.synchronize()
    assert (guarded[least:] == 0x5A).all()
