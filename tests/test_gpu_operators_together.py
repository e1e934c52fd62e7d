"""The operators around the block as a decode step uses them: a 4-bit projection, residual add + norm, the block under a routing rule, the next
norm in 8 bits and the product that reads it; eager, layer by layer in one call, and captured and replayed."""
import numpy as np
import pytest
import torch

import opsref

pytestmark = pytest.mark.gpu

H, I, E, K, N = 256, 128, 32, 4, 640


class Step:
    def __init__(self, pkg, wl, dev, T):
        self.pkg, self.T = pkg, T
        r = np.random.default_rng(T)
        on = lambda a: torch.from_numpy(a).to(dev)  # noqa: E731
        codes, scales = r.integers(0, 256, (H, H // 2), dtype=np.uint8), (0.01 * np.exp(0.3 * r.standard_normal((H, H // 64)))).astype(np.float32)
        zeros = r.integers(0, 16, (H, H // 64), dtype=np.uint8)
        scales = torch.from_numpy(scales).bfloat16()
        self.proj_w, self.proj_bound = opsref.int4_weights(codes, scales.double().numpy(), zeros, 64)
        self.proj = pkg.int4_repack(on(codes), scales.to(dev), on(zeros), 64)
        codes, scales = r.integers(0, 256, (N, H // 2), dtype=np.uint8), r.integers(119, 128, (N, H // 32), dtype=np.uint8)
        self.head_w = opsref.mxfp4_weights(codes, scales)
        self.head = pkg.mxfp4_repack(on(codes).view(1, N, H // 32, 16), on(scales).view(1, N, H // 32))
        self.block, _ = wl.make_device_layer(wl.MoeShape("step", T=T, H=H, I=I, E=E, K=K, fmt="bf16", seed=T), pkg.normal_table(), dev)
        self.bias = 0.05 * on(r.standard_normal(E).astype(np.float32))
        self.block.route = pkg.RouteRule("sigmoid", self.bias, 8, 3, 2, True, 2.5)
        self.norms = [(1 + 0.2 * torch.from_numpy(r.standard_normal(H).astype(np.float32))).bfloat16().to(dev) for _ in range(2)]
        f = lambda *s: torch.empty(s, device=dev)  # noqa: E731
        self.attn, self.x = f(T, H).bfloat16(), f(T, H)
        self.delta, self.x1, self.t, self.agg, self.scores, self.x2, self.logits = f(T, H), f(T, H), f(T, H), f(T, H), f(T, E), f(T, H), f(T, N)
        self.ti, self.tv = torch.empty((T, K), dtype=torch.int32, device=dev), f(T, K)
        self.q, self.qs = torch.empty((T, H), dtype=torch.uint8, device=dev), torch.empty((T, H // 32), dtype=torch.uint8, device=dev)

    def fill(self, seed):
        g = torch.Generator(device=self.x.device).manual_seed(seed)
        self.x.normal_(generator=g)
        self.attn.normal_(generator=g)

    def run(self):
        p, T = self.pkg, self.T
        p.linear_int4(self.delta, self.attn, self.proj[0], self.proj[1], T, H, H, 64, tiled_zeros=self.proj[2])
        p.add_rmsnorm(self.x1, self.x, self.norms[0], T, H, delta=self.delta, o=self.t)
        self.block.forward(self.t, self.agg, self.ti, self.tv, router_score=self.scores, residual_x=self.x1)
        p.add_rmsnorm(self.x2, self.x1, self.norms[1], T, H, q=self.q, q_scales=self.qs)
        p.linear_mxfp4(self.logits, self.q, *self.head, T, H, N, x_scales=self.qs)

    def outputs(self):
        return [t.clone() for t in (self.delta, self.x1, self.t, self.agg, self.ti, self.tv, self.q, self.qs, self.logits)]

    def spoil(self):
        for t in (self.delta, self.x1, self.t, self.agg, self.tv, self.scores, self.x2, self.logits):
            t.fill_(float("nan"))
        for t in (self.ti, self.q, self.qs):
            t.zero_()


@pytest.mark.parametrize("T", [1, 5, 40])
def test_decode_step(pkg, wl, dev, T):
    s = Step(pkg, wl, dev, T)
    s.fill(1)
    s.spoil()
    s.run()
    # every operator on what it was given.  The bounds of the products: K / 8 + 64 roundings of half a step 2^-24, as for the products alone
    limit = (H / 8 + 64) * 2.0 ** -24
    attn = s.attn.double().cpu().numpy()
    assert (np.abs(s.delta.cpu().numpy() - attn @ s.proj_w.T) <= limit * (np.abs(attn) @ s.proj_bound.T)).all()
    before = s.x + s.delta
    t = opsref.rmsnorm_products(before.cpu().numpy(), s.norms[0].float().cpu().numpy(), 1e-5)
    assert np.array_equal(t.astype(np.float32), s.t.cpu().numpy())
    wv, wi = opsref.route(s.scores.cpu().numpy(), K, "sigmoid", s.bias.cpu().numpy(), 8, 3, 2, True, 2.5)
    assert np.array_equal(wi, s.ti.cpu().numpy())
    assert (np.abs(s.tv.cpu().numpy() - wv) <= 2.0 ** -23 * wv).all()  # the same 64-bit quotient up to its roundings, rounded once
    assert torch.equal(s.x1, before + s.agg) and torch.equal(s.x2, s.x1)
    wq, ws = opsref.quantise(opsref.rmsnorm_products(s.x2.cpu().numpy(), s.norms[1].float().cpu().numpy(), 1e-5), 32)
    assert np.array_equal(opsref.e4m3_values(s.q.cpu().numpy()), wq) and np.array_equal(np.exp2(s.qs.cpu().numpy() - 127.0), ws)
    rows = wq * np.repeat(ws, 32, 1)
    assert (np.abs(s.logits.cpu().numpy() - rows @ s.head_w.T) <= limit * (np.abs(rows) @ np.abs(s.head_w).T)).all()


@pytest.mark.parametrize("T", [1, 40])
def test_captured_steps_that_alternate(pkg, wl, dev, T):
    steps = [Step(pkg, wl, dev, T), Step(pkg, wl, dev, T + 3)]
    graphs = []
    for s in steps:
        s.fill(7)
        s.run()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s.run()
        graphs.append(g)
    for i in range(4):
        for s, g in zip(steps, graphs):
            s.fill(20 + i)
            s.run()
            want = s.outputs()
            s.spoil()
            g.replay()
            torch.cuda.synchronize()
            for a, b in zip(s.outputs(), want):
                assert torch.equal(a, b)


def test_layers_with_their_own_rules(pkg, wl, dev):
    """A rule per layer in one call, the last one's left out: as the layers one by one."""
    T = 6
    rules = [pkg.RouteRule("sigmoid", scale=1.5), pkg.RouteRule("softmax", n_groups=8, groups_per_token=2, group_top=2, renormalize=False), None]
    blocks, xs = [], []
    for i, rule in enumerate(rules):
        shape = wl.MoeShape("layers", T=T, H=H, I=I, E=E, K=K, fmt="bf16", seed=i)
        b, _ = wl.make_device_layer(shape, pkg.normal_table(), dev)
        b.route = rule
        blocks.append(b)
        xs.append(wl.make_device_input(shape, pkg.normal_table(), dev))
    want = [b.forward(x) for b, x in zip(blocks, xs)]
    got = [[torch.full_like(o, -1) for o in w] for w in want]
    packed = pkg.pack_layer_params([b.params(x, *o) for b, x, o in zip(blocks, xs, got)])
    pkg.forward_layers(packed, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    for w, o in zip(want, got):
        for a, b in zip(w, o):
            assert torch.equal(a, b)
