"""Refusals and sizes of the operators around the block, without a device: every check comes before the first launch."""
import ctypes

import numpy as np
import pytest

import opsref


def rule(pkg, **kw):
    p = pkg.RouteParams(struct_bytes=ctypes.sizeof(pkg.RouteParams), scoring=0, n_groups=1, groups_per_token=1, group_top=1, renormalize=1, scale=1.0)
    for k, v in kw.items():
        setattr(p, k, v)
    return ctypes.byref(p)


def test_route_refuses(pkg):
    f = pkg.lib.moe_route
    assert f(None, 16, 16, 4, 32, 4, rule(pkg), None) == f(16, 16, 16, 4, 32, 4, None, None) == -1
    assert f(16, 16, 16, 0, 32, 4, rule(pkg), None) == f(16, 16, 16, 4, 3, 4, rule(pkg), None) == f(16, 16, 16, 4, 32, 0, rule(pkg), None) == -2
    assert f(16, 16, 16, 4, 1025, 4, rule(pkg), None) == f(16, 16, 16, 4, 32, 9, rule(pkg), None) == -3
    assert f(16, 16, 16, 0x7FFFFF01, 1, 1, rule(pkg), None) == -3
    assert f(16, 16, 16, 4, 520, 4, rule(pkg, n_groups=65, groups_per_token=4), None) == -3
    assert f(16, 16, 16, 4, 32, 4, rule(pkg, scoring=2), None) == f(16, 16, 16, 4, 32, 4, rule(pkg, struct_bytes=8), None) == -5
    for bad in (dict(n_groups=0), dict(n_groups=5), dict(n_groups=4, groups_per_token=0), dict(n_groups=4, groups_per_token=5), dict(group_top=0),
                dict(group_top=3), dict(n_groups=16, groups_per_token=1)):  # the last: two experts stay, four are wanted
        assert f(16, 16, 16, 4, 32, 4, rule(pkg, **bad), None) == -2, bad


def test_block_refuses_a_bad_rule(pkg):
    r = pkg.RouteParams(struct_bytes=ctypes.sizeof(pkg.RouteParams), scoring=0, n_groups=3, groups_per_token=1, group_top=1)
    p = pkg.BlockParams(struct_bytes=ctypes.sizeof(pkg.BlockParams), n_tokens=4, hidden_dim=64, intermediate_dim=64, n_experts=4,
                        experts_per_token=2, route=ctypes.addressof(r))
    assert pkg.lib.moe_block_forward(ctypes.byref(p), None) == -2
    r.n_groups = 1
    assert pkg.lib.moe_block_forward(ctypes.byref(p), None) == -1  # the rule is fine, the tensors are NULL
    p.struct_bytes = pkg.BlockParams.route.offset  # a caller of the struct without the member: what lies there is not looked at
    r.n_groups = 3
    assert pkg.lib.moe_block_forward(ctypes.byref(p), None) == -1


def test_describe_names_the_rule_kernel(pkg):
    r = pkg.RouteParams(struct_bytes=ctypes.sizeof(pkg.RouteParams))
    for T, E, router in ((1, 32, "router_scores_kernel + route_kernel"), (300, 128, "router_partial_kernel + router_finalize_kernel + route_kernel")):
        p = pkg.BlockParams(struct_bytes=ctypes.sizeof(pkg.BlockParams), n_tokens=T, hidden_dim=2880, intermediate_dim=2880, n_experts=E,
                            experts_per_token=4, weight_format=1, route=ctypes.addressof(r))
        text = ctypes.create_string_buffer(1024)
        assert pkg.lib.moe_block_describe(ctypes.byref(p), text, len(text)) == 0
        assert text.value.decode().startswith("router=%s; " % router)


def test_add_rmsnorm_refuses(pkg):
    f = pkg.lib.moe_add_rmsnorm
    ok = dict(x_out=16, x=16, delta=16, w=16, batch=2, size=64, eps=1e-5, o=16, ob=16, q=16, qs=16, group=32)

    def call(**kw):
        a = dict(ok, **kw)
        return f(a["x_out"], a["x"], a["delta"], a["w"], a["batch"], a["size"], a["eps"], a["o"], a["ob"], a["q"], a["qs"], a["group"], None)
    assert call(x_out=None) == call(x=None) == call(w=None) == call(q=None) == call(qs=None) == call(o=None, ob=None, q=None, qs=None) == -1
    assert call(batch=0) == call(size=0) == call(size=66) == call(size=68) == -2  # the last: no multiple of 32 for scales of 32
    assert call(batch=0x7FFFFF01, size=4, group=0) == -3
    assert call(group=64) == -5
    assert call(x=8) == call(x_out=8) == call(delta=4) == call(o=8) == call(w=4) == call(ob=4) == call(q=2) == call(qs=2, group=0) == -6


def test_linear_refuses(pkg):
    f, g = pkg.lib.moe_linear_mxfp4, pkg.lib.moe_linear_int4
    assert f(None, 16, None, 16, 16, None, 1, 64, 64, None) == f(16, 16, None, 16, None, None, 1, 64, 64, None) == -1
    assert f(16, 16, None, 16, 16, None, 0, 64, 64, None) == f(16, 16, None, 16, 16, None, 1, 48, 64, None) == -2
    assert f(16, 16, None, 16, 16, None, 1, 64, 32, None) == -2  # rows of tiled MXFP4 come in groups of 64
    assert f(16, 16, None, 16, 16, None, 65536, 64, 64, None) == f(16, 16, None, 16, 16, None, 1, 64, 2**26 + 64, None) == -3
    assert f(16, 8, None, 16, 16, None, 1, 64, 64, None) == f(2, 16, None, 16, 16, None, 1, 64, 64, None) == f(16, 16, None, 16, 16, 1, 1, 64, 64, None) == -6
    assert g(16, None, None, 16, 16, None, None, 1, 64, 5, 32, None) == -1
    assert g(16, 16, None, 16, 16, None, None, 1, 64, 0, 32, None) == -2
    assert g(16, 16, None, 16, 16, None, None, 1, 64, 5, 16, None) == -5
    assert g(16, 16, None, 16, 16, 8, None, 1, 64, 5, 32, None) == -6


def test_int4_repack_refuses_and_sizes(pkg):
    assert pkg.int4_tiled_bytes(17, 160, 64) == (2 * 2 * 1024, 2 * 4 * 32, 2 * 4 * 16)
    assert pkg.int4_tiled_bytes(16, 128, 128) == (1024, 2 * 32, 2 * 16)
    assert pkg.int4_tiled_bytes(0, 128, 128) == pkg.int4_tiled_bytes(16, 48, 32) == pkg.int4_tiled_bytes(16, 64, 48) == (0, 0, 0)
    f = pkg.lib.moe_int4_repack
    assert f(None, 16, None, 16, 64, 32, 16, 16, None, None) == f(16, 16, 16, 16, 64, 32, 16, 16, None, None) == -1
    assert f(16, 16, None, 16, 40, 32, 16, 16, None, None) == -2
    assert f(16, 16, None, 16, 64, 33, 16, 16, None, None) == -5
    assert f(2, 16, None, 16, 64, 32, 16, 16, None, None) == f(16, 16, None, 16, 64, 32, 8, 16, None, None) == -6


def test_wrappers_refuse_tensors_that_do_not_fit(pkg):
    import torch
    x = torch.zeros(2, 64)
    with pytest.raises(ValueError, match="x_out: expected 128 values of torch.float32, got 128 of torch.bfloat16"):
        pkg.add_rmsnorm(x.bfloat16(), x, x.bfloat16(), 2, 64, o=x)
    with pytest.raises(ValueError, match="x_out: expected 192 values"):
        pkg.add_rmsnorm(x, x, x.bfloat16(), 3, 64, o=x)
    with pytest.raises(ValueError, match="x: expected a tensor on the current device"):
        pkg.linear_mxfp4(x, x.bfloat16(), x, x, 2, 64, 64)
    with pytest.raises(ValueError, match="x: expected 128 values of torch.uint8"):  # 8-bit rows come with their scales
        pkg.linear_int4(x, x.bfloat16(), x, x, 2, 64, 64, 32, x_scales=x)


def test_a_rule_is_softmax_or_sigmoid(pkg):
    with pytest.raises(ValueError, match="scoring: expected softmax or sigmoid, got 'tanh'"):
        pkg.RouteRule("tanh")


def test_oracle_e4m3_and_scales_agree_with_torch():
    import torch
    v = np.concatenate([np.linspace(-448, 448, 4001), np.exp2(np.linspace(-14, 8.8, 999))])
    want = torch.from_numpy(v).to(torch.float8_e4m3fn)
    assert np.array_equal(opsref.to_e4m3(v), want.double().numpy())
    codes = np.arange(256, dtype=np.uint8)
    both = opsref.e4m3_values(codes), torch.from_numpy(codes).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(both[0], both[1], equal_nan=True)
