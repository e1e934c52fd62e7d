"""moe_attention_prefill against its formula in 64 bits: prompts of every length around the tile borders, keys in front of them, queries without keys."""
import numpy as np
import pytest
import torch

import attnref

pytestmark = pytest.mark.gpu


class Case:
    def __init__(self, pkg, dev, lens, Hq, Hkv, D, window=0, sinks=False, context=None, seed=0, pad=0, spread=1.0, behind=3):
        r = np.random.default_rng(seed)
        self.pkg, self.Hq, self.Hkv, self.D, self.window, self.lens = pkg, Hq, Hkv, D, window, lens
        self.keys = [n + (context[i % len(context)] if context else 0) for i, n in enumerate(lens)]
        self.keys = [max(0, n) for n in self.keys]
        tq, tk = sum(lens) + behind, sum(self.keys) + behind

        def rows(n, H, poison):
            t = torch.full((n, H * D + pad), float("nan"), dtype=torch.bfloat16)
            t[: n - poison, : H * D] = torch.from_numpy(spread * r.standard_normal((n - poison, H * D))).bfloat16()
            return t.to(dev)[:, : H * D].view(n, H, D) if not pad else t.to(dev).as_strided((n, H, D), (H * D + pad, D, 1))
        self.q, self.k, self.v = rows(tq, Hq, behind), rows(tk, Hkv, behind), rows(tk, Hkv, behind)
        self.out = torch.full((tq, Hq * D + pad), -3.0, dtype=torch.bfloat16, device=dev).as_strided((tq, Hq, D), (Hq * D + pad, D, 1))
        starts = lambda n: np.concatenate([[0], np.cumsum(n)]).astype(np.int32)  # noqa: E731
        self.qs, self.ks = starts(lens), starts(self.keys)
        self.d_qs, self.d_ks = torch.from_numpy(self.qs).to(dev), torch.from_numpy(self.ks).to(dev)
        self.sinks = torch.from_numpy(r.standard_normal(Hq) + 1).bfloat16().to(dev) if sinks else None
        self.scale = D ** -0.5

    def run(self, stream=None):
        self.pkg.attention_prefill(self.out, self.q, self.k, self.v, self.d_qs, self.d_ks, len(self.lens), self.Hq, self.Hkv, self.D, self.scale,
                                   window=self.window, sinks=self.sinks, stream=stream)

    def check(self, rows=None):
        assert (self.out[self.qs[-1]:] == -3.0).all()
        got, q, k, v = (t.double().cpu().numpy() for t in (self.out, self.q, self.k, self.v))
        sinks = None if self.sinks is None else self.sinks.double().cpu().numpy()
        g = self.Hq // self.Hkv
        for s, n in enumerate(self.lens):
            m = self.keys[s]
            for i in range(n) if rows is None else sorted({x for x in rows if -n <= x < n}):
                i %= n
                a, b = attnref.visible(i, n, m, self.window)
                b = max(a, b)
                for h in range(self.Hq):
                    kk, vv = k[self.ks[s] + a : self.ks[s] + b, h // g], v[self.ks[s] + a : self.ks[s] + b, h // g]
                    want, limit = attnref.attention_row(q[self.qs[s] + i, h], kk, vv, self.scale, None if sinks is None else sinks[h])
                    e = abs(got[self.qs[s] + i, h] - want)
                    assert (e <= limit).all(), (s, n, m, i, h, e.max(), limit.max())


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hkv,window,sinks", [(4, 1, 0, False), (3, 3, 0, True), (8, 2, 20, True), (16, 2, 1, False), (2, 1, 130, False)])
def test_lengths(pkg, dev, D, Hq, Hkv, window, sinks):
    print(D, Hq, Hkv, window, sinks, flush=True)
    c = Case(pkg, dev, [1, 0, 31, 33, 64, 5, 127, 129, 1, 66], Hq, Hkv, D, window, sinks, seed=D + Hq, pad=8 * (Hq % 3))
    c.run()
    c.check()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,sinks", [(0, True), (70, False), (257, True)])
def test_keys_in_front_and_queries_without_keys(pkg, dev, D, window, sinks):
    """More keys than queries, as many, fewer (the first queries see nothing and have zeros), none."""
    print(D, window, sinks, flush=True)
    lens, context = [3, 40, 130, 70, 9, 1], [500, -20, 64, -70, 1, 300]
    c = Case(pkg, dev, lens, 4, 2, D, window, sinks, context, seed=window)
    c.run()
    c.check()
    at = c.qs[1]
    assert (c.out[at : at + 20] == 0).all() and (c.out[c.qs[3] : c.qs[4]] == 0).all()


def test_long_prompts(pkg, dev):
    for D, window in ((64, 0), (128, 0), (64, 128)):
        print(D, window, flush=True)
        c = Case(pkg, dev, [1500, 700], 8, 1, D, window, True, seed=D)
        c.run()
        c.check(rows=[0, 1, 127, 128, 129, 255, 256, 511, 640, -1, -2, -130])


def test_many_short_prompts_and_large_scores(pkg, dev):
    for lens, Hq, Hkv, spread in (([2, 3] * 70, 2, 1, 1.0), ([140], 40, 40, 1.0), ([150, 90], 8, 2, 5.0)):
        c = Case(pkg, dev, lens, Hq, Hkv, 64, 0, True, seed=len(lens), spread=spread)
        c.run()
        c.check(rows=[0, 1, 2, 77, -1])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("window", [0, 40])
def test_what_a_row_does_not_see_does_not_matter(pkg, dev, D, value, window):
    """Keys and values that are not finite reach the rows that see them and no others."""
    c = Case(pkg, dev, [150, 100, 90], 4, 2, D, window, True, seed=11)
    c.run()
    want = c.out.clone()
    place = {0: 70, 1: 99}
    for s, j in place.items():
        c.v[c.ks[s] + j, 0, 3] = value
        c.k[c.ks[s] + j, 1, 5] = value
    c.run()
    torch.cuda.synchronize()
    row = torch.arange(c.out.shape[0], device=dev)
    for s in range(3):
        for i in range(c.lens[s]):
            at, j = c.qs[s] + i, place.get(s, 10**6)
            if j <= i and (not window or j > i - window):
                # an infinity may cancel or spoil; dimension 3 of the heads that read the value holds it
                assert not torch.isfinite(c.out[at, :2, 3]).any()
                keep = [d for d in range(D) if d != 3]
                assert torch.equal(c.out[at, :2][:, keep], want[at, :2][:, keep])
            else:
                assert torch.equal(c.out[at], want[at]), (s, i)
    assert torch.equal(c.out[c.qs[-1]:], want[c.qs[-1]:])


def test_strided_rows_of_one_tensor(pkg, dev):
    """Queries, keys and values as views of the rows of one projection."""
    T, Hq, Hkv, D = 200, 6, 2, 64
    x = torch.randn((T, Hq + 2 * Hkv, D), device=dev).bfloat16()
    starts = torch.tensor([0, 77, T], dtype=torch.int32, device=dev)
    outs = []
    for q, k, v in ((x[:, :Hq], x[:, Hq : Hq + Hkv], x[:, Hq + Hkv :]), [t.contiguous() for t in (x[:, :Hq], x[:, Hq : Hq + Hkv], x[:, Hq + Hkv :])]):
        out = torch.empty((T, Hq, D), dtype=torch.bfloat16, device=dev)
        pkg.attention_prefill(out, q, k, v, starts, starts, 2, Hq, Hkv, D, 0.125)
        outs.append(out)
    assert torch.equal(*outs)


def test_a_row_does_not_depend_on_other_sequences(pkg, dev):
    c = Case(pkg, dev, [90, 200, 17], 4, 2, 64, sinks=True, seed=12)
    c.run()
    a, b = int(c.qs[1]), int(c.qs[2])
    one = torch.tensor([0, b - a], dtype=torch.int32, device=dev)
    out = torch.empty((b - a, 4, 64), dtype=torch.bfloat16, device=dev)
    pkg.attention_prefill(out, c.q[a:b], c.k[a:b], c.v[a:b], one, one, 1, 4, 2, 64, c.scale, sinks=c.sinks)
    assert torch.equal(out, c.out[a:b])


def test_starts_outside_the_rows_are_cut(pkg, dev):
    c = Case(pkg, dev, [50, 40], 2, 1, 64, seed=13, behind=0)
    c.run()
    want = c.out.clone()
    c.d_qs[2], c.d_ks[2] = 2**31 - 1, 2**31 - 1
    c.d_qs[0], c.d_ks[0] = -5, -(2**31)
    c.out.fill_(0)
    c.run()
    assert torch.equal(c.out, want)


def test_captured_with_starts_that_change(pkg, dev):
    c = Case(pkg, dev, [300, 40, 160], 4, 2, 64, sinks=True, seed=14)
    c.run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.run()
    for cut in (0, 13, 100, 299):
        c.d_qs[1] = c.d_ks[1] = 300 - cut
        c.out.fill_(-1)
        c.run()
        want = c.out.clone()
        c.out.fill_(-1)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(c.out, want)


def test_past_32_bits(pkg, dev):
    """Rows whose offsets pass 2^31 values: the far end as a call on it alone."""
    Hq, Hkv, D, tail, stride = 2, 1, 64, 150, 1 << 23
    T = (1 << 31) // stride + tail
    print("prefill", T, stride, flush=True)
    buf = torch.zeros(T * stride, dtype=torch.bfloat16, device=dev)
    x = buf.as_strided((T, Hq + 2 * Hkv, D), (stride, D, 1))
    x.copy_(torch.randn((T, Hq + 2 * Hkv, D), device=dev))
    out = buf.as_strided((T, Hq, D), (stride, D, 1), 4096)
    starts = torch.tensor([0, T - tail, T], dtype=torch.int32, device=dev)
    pkg.attention_prefill(out, x[:, :Hq], x[:, Hq : Hq + Hkv], x[:, Hq + Hkv :], starts, starts, 2, Hq, Hkv, D, 0.125)
    e = x[-tail:].contiguous()
    one = torch.tensor([0, tail], dtype=torch.int32, device=dev)
    want = torch.empty((tail, Hq, D), dtype=torch.bfloat16, device=dev)
    pkg.attention_prefill(want, e[:, :Hq], e[:, Hq : Hq + Hkv], e[:, Hq + Hkv :], one, one, 1, Hq, Hkv, D, 0.125)
    assert torch.equal(out[-tail:], want)
