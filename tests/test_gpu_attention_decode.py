"""moe_attention_decode against its formula in 64 bits.  Whatever a query does not see is NaN: slots behind a sequence's last key and in front of its
window, pages that no table lists, scales; tables hold nonsense behind their last page."""
import numpy as np
import pytest
import torch

import attnref
import opsref

pytestmark = pytest.mark.gpu


class Case:
    def __init__(self, pkg, dev, lens, Hq, Hkv, D, fmt="bf16", page=16, window=0, sinks=False, seed=0, spread=1.0):
        r = np.random.default_rng(seed)
        self.pkg, self.lens, self.Hq, self.Hkv, self.D, self.window, self.B = pkg, lens, Hq, Hkv, D, window, len(lens)
        used = [-(-max(n, 0) // page) for n in lens]
        max_pages = max(max(used), 1) + 2
        self.n_pages = sum(used) + 3
        order = r.permutation(self.n_pages)
        table = np.array([[-1, 2**31 - 1, self.n_pages, -(2**31)][i % 4] for i in range(self.B * max_pages)], np.int32).reshape(self.B, max_pages)
        shape = (self.n_pages, Hkv, page, D)
        k, v = (spread * r.standard_normal(shape) for _ in range(2))
        seen = np.zeros((self.n_pages, page), bool)
        at = 0
        for b, n in enumerate(lens):
            table[b, : used[b]] = order[at : at + used[b]]
            at += used[b]
            j = np.arange(max(0, n - window) if window else 0, max(n, 0))
            seen[table[b, j // page], j % page] = True
        self.table, self.page = table, page
        if fmt == "bf16":
            kb, vb = (torch.from_numpy(np.where(seen[:, None, :, None], t, np.nan)).bfloat16() for t in (k, v))
            self.k, self.v = kb.double().numpy(), vb.double().numpy()
            self.cache = pkg.KvCache(kb.to(dev), vb.to(dev))
        else:
            held = []
            for t in (k, v):
                codes = torch.from_numpy(np.clip(t * 40, -448, 448)).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
                scales = r.integers(119, 125, (*shape[:3], D // 32), dtype=np.uint8)
                codes, scales = np.where(seen[:, None, :, None], codes, 0x7F), np.where(seen[:, None, :, None], scales, 255).astype(np.uint8)
                held.append((codes.astype(np.uint8), scales))
            self.k, self.v = (opsref.e4m3_values(c) * np.repeat(np.exp2(s - 127.0), 32, -1) for c, s in held)
            on = [torch.from_numpy(a).to(dev) for c in held for a in c]
            self.cache = pkg.KvCache(on[0].view(torch.float8_e4m3fn), on[2].view(torch.float8_e4m3fn), on[1].view(torch.float8_e8m0fnu), on[3])
        self.scale = D ** -0.5
        self.q = torch.from_numpy(spread * r.standard_normal((self.B, Hq, D))).bfloat16().to(dev)
        self.sinks = torch.from_numpy(r.standard_normal(Hq) + 1).bfloat16().to(dev) if sinks else None
        self.d_table = torch.from_numpy(table).to(dev)
        self.d_lens = torch.tensor(lens, dtype=torch.int32, device=dev)
        self.ws = torch.empty(pkg.attention_decode_workspace_bytes(self.B, Hq, Hkv, D), dtype=torch.uint8, device=dev).random_(0, 256)
        self.out = torch.full((self.B + 1, Hq, D), -3.0, dtype=torch.bfloat16, device=dev)

    def run(self, stream=None):
        self.pkg.attention_decode(self.out, self.q, self.cache, self.d_table, self.d_lens, self.B, self.Hq, self.scale, self.ws, window=self.window,
                                  sinks=self.sinks, stream=stream)

    def check(self, gone=()):
        assert (self.out[self.B] == -3.0).all()
        got = self.out[: self.B].double().cpu().numpy()
        q = self.q.double().cpu().numpy()
        sinks = None if self.sinks is None else self.sinks.double().cpu().numpy()
        g = self.Hq // self.Hkv
        for b, n in enumerate(self.lens):
            j = np.arange(max(0, n - self.window) if self.window else 0, max(n, 0))
            j = j[~np.isin(self.table[b, j // self.page], gone)] if len(gone) else j
            pages, slots = self.table[b, j // self.page], j % self.page
            for h in range(self.Hq):
                k, v = self.k[pages, h // g, slots], self.v[pages, h // g, slots]
                want, limit = attnref.attention_row(q[b, h], k, v, self.scale, None if sinks is None else sinks[h])
                assert (abs(got[b, h] - want) <= limit).all(), (b, n, h, abs(got[b, h] - want).max(), limit.max())


LENGTHS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 511, 513, 1000, -7]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("fmt", ["bf16", "mx8"])
@pytest.mark.parametrize("Hq,Hkv,page,window,sinks", [(8, 1, 16, 0, False), (4, 4, 32, 0, True), (6, 2, 64, 128, True), (17, 1, 16, 1, False),
                                                      (40, 2, 128, 33, True), (16, 1, 1024, 0, True)])
def test_lengths_and_heads(pkg, dev, D, fmt, Hq, Hkv, page, window, sinks):
    print(D, fmt, Hq, Hkv, page, window, sinks, flush=True)
    c = Case(pkg, dev, LENGTHS, Hq, Hkv, D, fmt, page, window, sinks, seed=Hq)
    c.run()
    c.check()


@pytest.mark.parametrize("lens,Hq,Hkv,D,fmt,page,window", [
    ([20000], 8, 1, 64, "bf16", 64, 0), ([9001], 16, 2, 128, "mx8", 32, 0), ([5000, 1, 700, 0, 64, 3333], 8, 2, 64, "mx8", 16, 0),
    ([6000, 40], 4, 2, 128, "bf16", 256, 2500), ([1] * 70 + [4000] + [3] * 70, 2, 1, 64, "bf16", 16, 0), ([300] * 200, 2, 2, 64, "bf16", 16, 0),
    ([5] * 300 + [3000] + [40] * 100, 2, 1, 64, "mx8", 16, 0), ([5] * 520 + [4100, 0] + [40] * 100, 2, 1, 64, "bf16", 16, 0)])
def test_long_ones_in_parts(pkg, dev, lens, Hq, Hkv, D, fmt, page, window):
    print(lens[:3], Hq, Hkv, D, fmt, page, window, flush=True)
    for sinks in (False, True):
        c = Case(pkg, dev, lens, Hq, Hkv, D, fmt, page, window, sinks, seed=page)
        c.run()
        c.check()


def test_many_heads_and_large_scores(pkg, dev):
    for Hq, Hkv, spread in ((1024, 8, 1.0), (130, 130, 1.0), (8, 2, 6.0)):
        print(Hq, Hkv, spread, flush=True)
        c = Case(pkg, dev, [70, 400], Hq, Hkv, 64, page=32, sinks=True, seed=5, spread=spread)
        c.run()
        c.check()


def test_pages_that_do_not_exist(pkg, dev):
    """A page number out of range is a page without keys, also where all of a sequence's are."""
    c = Case(pkg, dev, [300, 48, 16], 4, 2, 64, page=16, sinks=True, seed=9)
    for at, bad in (((0, 3), -1), ((0, 7), c.n_pages), ((0, 18), 2**31 - 1), ((2, 0), -(2**31))):
        c.table[at] = bad
    c.d_table.copy_(torch.from_numpy(c.table))
    c.run()
    c.check(gone=[-1, c.n_pages, 2**31 - 1, -(2**31)])
    assert (c.out[2] == 0).all()


def test_lengths_past_the_table_are_cut(pkg, dev):
    c = Case(pkg, dev, [64, 32], 4, 2, 64, page=16, seed=2)
    short = c.d_table[:, :4].contiguous()
    c.table = short.cpu().numpy()
    c.table[1, 2:] = c.table[0, :2]
    c.d_table = torch.from_numpy(c.table).to(dev)
    c.d_lens = torch.tensor([2**31 - 1, 2**30 + 5], dtype=torch.int32, device=dev)
    c.lens = [64, 64]
    c.run()
    c.check()


def test_keys_of_minus_infinity_and_nan_where_seen(pkg, dev):
    c = Case(pkg, dev, [100, 200], 4, 1, 64, page=16, seed=3)
    c.q.fill_(1.0)
    page, slot = c.table[0, 2], 5
    c.cache.k[page, 0, slot] = float("-inf")  # a weight of nothing
    c.cache.v[c.table[1, 1], 0, 3, 7] = float("nan")
    c.run()
    assert torch.isfinite(c.out[0]).all()
    bad = torch.isnan(c.out[1])
    assert bad[:, 7].all() and int(bad.sum()) == 4
    c.k[page, 0, slot] = -1e6
    c.v[c.table[1, 1], 0, 3, 7] = 0
    c.out[1, :, 7] = 0
    got = c.out.clone()
    c.cache.v[c.table[1, 1], 0, 3, 7] = 0
    c.run()
    assert torch.equal(c.out[0], got[0])
    c.check()


def test_other_stream_same_bits(pkg, dev):
    c = Case(pkg, dev, [3000, 5, 777], 8, 2, 64, "mx8", 16, sinks=True, seed=4)
    c.run()
    want = c.out.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        c.out[: c.B] = 0
        side.wait_stream(torch.cuda.current_stream())
        c.run(stream=side)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(c.out, want)


def test_captured_calls_that_share_a_workspace(pkg, dev):
    """Two captured calls, replayed in turn with lengths that change on the device; eager calls between them."""
    cases = [Case(pkg, dev, [2000, 9, 500], 8, 2, 64, page=16, seed=6), Case(pkg, dev, [100, 4000, 1], 8, 2, 64, "mx8", 16, seed=7)]
    cases[1].ws = cases[0].ws
    graphs = []
    for c in cases:
        c.run()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.run()
        graphs.append(g)
    for i in range(4):
        for c, g in zip(cases, graphs):
            c.lens = [max(0, n - 37 * i) for n in c.lens]
            c.d_lens.copy_(torch.tensor(c.lens, dtype=torch.int32))
            c.run()
            want = c.out.clone()
            c.out[: c.B] = -1
            c.ws.random_(0, 256)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(c.out, want)
    for c in cases:
        c.check()


@pytest.mark.parametrize("fmt", ["bf16", "mx8"])
def test_cache_past_32_bits(pkg, dev, fmt):
    """The last pages of a cache of more than 2^32 bytes a tensor: as those pages alone."""
    Hkv, D, page, n = 8, 64, 64, 700
    per = Hkv * page * D * (2 if fmt == "bf16" else 1)
    n_pages = (1 << 32) // per + 40
    print("decode", n_pages, per, flush=True)
    used = -(-n // page)
    c = Case(pkg, dev, [n], 64, Hkv, D, fmt, page, seed=8)
    c.run()
    want = c.out.clone()
    small = c.d_table[0, :used].long()
    parts = []
    for t in (c.cache.k, c.cache.v, c.cache.k_scales, c.cache.v_scales):
        if t is None:
            parts.append(None)
            continue
        big = torch.empty((n_pages, *t.shape[1:]), dtype=t.dtype, device=dev)
        big.view(torch.uint8)[-used:] = t.view(torch.uint8)[small]
        parts.append(big)
    c.cache = pkg.KvCache(*parts)
    c.d_table[0, :used] = torch.arange(n_pages - used, n_pages, dtype=torch.int32, device=dev)
    c.out[:1] = 0
    c.run()
    assert torch.equal(c.out, want)
