"""What a routing rule's address stands in keeps the rule."""
import ctypes
import gc
import weakref

import torch


def block(pkg, rule):
    """A MoeBlock without tensors: its parameter blocks are made and packed, not launched."""
    blk = pkg.MoeBlock.__new__(pkg.MoeBlock)
    blk.H = blk.I = 64
    blk.E, blk.K, blk.fmt, blk.swiglu_limit, blk.alpha, blk.max_tokens = 4, 2, 0, 7.0, 1.702, 4
    blk.tensors, blk.workspace, blk.route = {}, torch.zeros(256, dtype=torch.uint8), rule
    return blk


def test_prepared_blocks_keep_their_rules(pkg, monkeypatch):
    monkeypatch.setattr(pkg, "_ptr", lambda t: None if t is None else t.data_ptr())  # tensors of the host
    t, i = torch.zeros(2, 64), torch.zeros(2, 2, dtype=torch.int32)
    blk = block(pkg, pkg.RouteRule("sigmoid", scale=2.5))
    rules = [weakref.ref(blk.route)]
    params = [blk.params(t, t, i, t)]
    blk.route = pkg.RouteRule("softmax", scale=1.5)
    rules.append(weakref.ref(blk.route))
    params.append(blk.params(t, t, i, t))
    blk.route = None
    params.append(blk.params(t, t, i, t))
    packed = pkg.pack_layer_params(params)
    addresses = [p.route for p in params]
    del params, blk
    gc.collect()
    assert all(r() is not None for r in rules) and addresses[2] is None
    for p, address, scale in zip(packed, addresses, (2.5, 1.5)):
        assert p.route == address and pkg.RouteParams.from_address(address).scale == scale
    del packed, p
    gc.collect()
    assert all(r() is None for r in rules)


def test_a_rule_keeps_the_bias_that_its_parameters_hold(pkg, monkeypatch):
    monkeypatch.setattr(pkg, "_device", lambda: -1)  # tensors of the host
    rule = pkg.RouteRule("sigmoid", torch.zeros(4))
    rule.of(4)
    first = weakref.ref(rule.balance_bias)
    address = rule.balance_bias.data_ptr()
    rule.balance_bias = torch.ones(8)  # until the next call the parameters hold the first one's address
    gc.collect()
    assert first() is not None and rule.params.balance_bias == address
    rule.of(8)
    gc.collect()
    assert first() is None and rule.params.balance_bias == rule.balance_bias.data_ptr()


def test_route_refuses_addresses_between_values(pkg):
    rule = ctypes.byref(pkg.RouteParams(struct_bytes=ctypes.sizeof(pkg.RouteParams), n_groups=1, groups_per_token=1, group_top=1))
    for bad in ((2, 16, 16), (16, 2, 16), (16, 16, 2)):
        assert pkg.lib.moe_route(*bad, 4, 32, 4, rule, None) == -6
