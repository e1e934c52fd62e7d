"""A routing rule takes no room in the block's workspace that its experts' rows do not have."""
import ctypes

import pytest


@pytest.mark.parametrize("shape,nbytes", [((1, 2880, 2880, 32, 4), 82176), ((256, 2880, 2880, 32, 4), 20232448), ((4096, 2880, 2880, 32, 4), 318632448),
                                          ((4096, 2880, 2880, 128, 4), 322563584), ((16384, 2880, 2880, 128, 8), 2411650816),
                                          ((300, 64, 64, 16, 2), 316416)])
def test_sizes_are_those_of_the_block_without_rules(pkg, shape, nbytes):
    assert pkg.block_workspace_bytes(*shape) == nbytes


def test_logits_longer_than_the_rows_have_room_of_their_own(pkg):
    """64 experts' rows of one bf16 and one fp32 row a token against 128 and 1024 logits: T * E * 4 bytes more."""
    assert pkg.block_workspace_bytes(8, 64, 64, 128, 1) == 18688 + 8 * 128 * 4
    assert pkg.block_workspace_bytes(500, 64, 64, 1024, 1) == 4392448 + 500 * 1024 * 4


def test_int4_sizes_past_32_bits(pkg):
    """More than 64 GiB of codes; rows and lengths that whole tiles take past 32 bits are refused."""
    assert pkg.int4_tiled_bytes(1 << 26, 4096, 128) == ((1 << 26) * 2048, (1 << 26) * 64, (1 << 26) * 32)
    assert pkg.int4_tiled_bytes(0x7FFFFF01, 128, 128) == pkg.int4_tiled_bytes(16, 0x7FFFFF20, 128) == (0, 0, 0)
    assert pkg.lib.moe_int4_repack(16, 16, None, 0x7FFFFF01, 64, 32, 16, 16, None, None) == -3


@pytest.mark.parametrize("E,G,kernel", [(960, 3, "route_any_kernel"), (990, 33, "route_any_kernel"), (1000, 10, "route_any_kernel"), (1024, 1, "route_kernel"),
                                        (960, 4, "route_kernel"), (256, 8, "route_kernel"), (512, 32, "route_kernel")])
def test_describe_names_the_routing_kernel_that_runs(pkg, E, G, kernel):
    """Groups of more experts than 16 to each of the lanes that a group has of 64."""
    r = pkg.RouteParams(struct_bytes=ctypes.sizeof(pkg.RouteParams), n_groups=G, groups_per_token=G, group_top=1)
    lanes = 1
    while 2 * lanes * G <= 64:
        lanes *= 2
    assert (kernel == "route_any_kernel") == (-(-(E // G) // lanes) > 16)
    for T, before in ((1, "router_scores_kernel"), (300, "router_partial_kernel + router_finalize_kernel")):
        p = pkg.BlockParams(struct_bytes=ctypes.sizeof(pkg.BlockParams), n_tokens=T, hidden_dim=128, intermediate_dim=64, n_experts=E,
                            experts_per_token=4, route=ctypes.addressof(r))
        text = ctypes.create_string_buffer(1024)
        assert pkg.lib.moe_block_describe(ctypes.byref(p), text, len(text)) == 0
        assert text.value.decode().startswith("router=%s + %s; " % (before, kernel))
