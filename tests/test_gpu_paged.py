"""The paged KV cache on the GPU against its restatement in 64 bits (oracle/pagedref.py).

Whatever is planned, stored or selected is exact: tables, slots, cache bytes, bounds and pages
are compared value for value, with what a call does not write included.

Attention is compared by relative 2-norm. Its scores are sums of head_dim products that are
exact in f32 (an f16 value times one of the two f16 terms of q, which keep q to 2^-22), so a
score is off by the sums' roundings: about sqrt(2 head_dim) 2^-24 of the partial sums' size.
With |q| |k| / sqrt(head_dim) up to about 60 here (head_dim 256, |q| 1.2 and |k| 2 a value)
that is sqrt(512) * 6e-8 * 60 = 8e-5 at the very worst, and 2^-24 sqrt(512) |s| = 1e-5 for
the scores |s| <= 8 that weigh anything; a softmax weight is off by the same share, and the
sum over slots averages it. TOL is 2e-5.
"""
import ctypes as C

import numpy as np
import pytest

import pagedref as ref
from conftest import rel_l2
from voxgen_amd import abi
from voxgen_amd.paged import NONE, PagedCache
from voxgen_amd.runtime import Context

pytestmark = pytest.mark.gpu
TOL = 2e-5


def rows_of(rng, *shape):
    """Keys or values with channel means of their own, as trained models have."""
    return (rng.standard_normal(shape) + 1.5 * rng.standard_normal(shape[-1])).astype(np.float32)


class Side:
    """A cache on the device and the same here: pages of random rows, in slots that hold no token random bits (NaN and
    infinities among them), tables in any order, and the step's counts."""

    def __init__(self, ctx, heads, page_size, lengths, counts, seed, layers=1, spare=3, max_rows=None, max_count=None,
                 bounds=False, width=None):
        self.ctx, self.rng = ctx, np.random.default_rng(seed)
        rng = self.rng
        self.q_heads, self.kv_heads, self.hd = heads
        self.ps, self.layers = page_size, layers
        self.lengths, self.counts = np.array(lengths, np.uint32), np.array(counts, np.uint32)
        n = len(lengths)
        have = [-(-a // page_size) for a in lengths]
        want = [-(-(a + c) // page_size) for a, c in zip(lengths, counts)]
        self.width = max(want) + 2 if width is None else width
        self.pages = max(sum(want) + spare, 1)
        self.max_rows = sum(counts) if max_rows is None else max_rows
        self.max_rows = max(self.max_rows, 1)
        any_page = rng.permutation(self.pages).astype(np.uint32)
        self.tables = np.full((n, self.width), NONE, np.uint32)
        used = 0
        for i, k in enumerate(have):
            self.tables[i, :k] = any_page[used:used + k]
            used += k
        self.pool = np.concatenate([[self.pages - used], any_page[used:], rng.integers(0, 1 << 32, used)]).astype(np.uint32)
        self.dev = PagedCache(ctx, layers, self.pages, page_size, self.kv_heads, self.hd, n, self.width, self.max_rows,
                              self.q_heads, max_count=max(max(counts), 1) if max_count is None else max_count, bounds=bounds)
        geom = (layers, self.pages, page_size, self.kv_heads, self.hd)
        bits = lambda shape: rng.integers(0, 1 << 16, shape, dtype=np.uint16).view(np.float16)  # noqa: E731
        self.k, self.v = bits(ref.k_shape(*geom)), bits(ref.v_shape(*geom))
        self.bounds = bits((layers, self.pages, self.kv_heads, 2, self.hd)) if bounds else None
        for i, a in enumerate(lengths):
            for col in range(have[i]):
                for layer in range(layers):
                    for h in range(self.kv_heads):
                        for cache, is_v in ((self.k, False), (self.v, True)):
                            m = min(page_size, a - col * page_size)
                            for s, x in enumerate(rows_of(rng, m, self.hd)):
                                ref.put(cache, layer, self.tables[i, col], h, s, x, is_v)
                        if bounds:
                            x = ref.page_rows(self.k, layer, self.tables[i, col], h, False)[:m]
                            self.bounds[layer, self.tables[i, col], h] = ref.bounds_of(x)
        self.send()

    def send(self):
        d = self.dev
        for buf, x in ((d.k, self.k), (d.v, self.v), (d.lengths, self.lengths), (d.counts, self.counts), (d.tables, self.tables),
                       (d.pool, self.pool), (d.bounds, self.bounds)):
            if buf is not None:
                buf.upload(x)

    def plan(self):
        self.dev.plan()
        self.want = ref.plan(self.lengths, self.counts, self.tables, self.pool, self.pages, self.ps, self.max_rows,
                             self.dev.max_count)
        self.tables = self.want["tables"]
        return self.want

    def check_plan(self):
        got = self.dev.read_plan()
        got["tables"] = self.dev.tables.download(np.uint32).reshape(self.tables.shape)
        for name, x in self.want.items():
            assert np.array_equal(got[name], x), (name, got[name], x)

    def put_rows(self, layer, k, v):
        """Rows [max_rows, kv_heads, hd] into the plan's slots, and the bounds of their pages, here."""
        touched = {}
        for r, slot in enumerate(self.want["slots"]):
            if slot == NONE:
                continue
            page, s = slot // self.ps, slot % self.ps
            touched[page] = max(touched.get(page, 0), s + 1)
            for h in range(self.kv_heads):
                ref.put(self.k, layer, page, h, s, k[r, h], False)
                ref.put(self.v, layer, page, h, s, v[r, h], True)
        if self.bounds is not None:
            for page, n in touched.items():
                for h in range(self.kv_heads):
                    self.bounds[layer, page, h] = ref.bounds_of(ref.page_rows(self.k, layer, page, h, False)[:n])

    def store(self, layer=0, k=None, v=None):
        """The step's rows, in both."""
        shape = (self.max_rows, self.kv_heads, self.hd)
        k = rows_of(self.rng, *shape) if k is None else k
        v = rows_of(self.rng, *shape) if v is None else v
        self.dev.store(layer, self.ctx.array(k), self.ctx.array(v))
        self.put_rows(layer, k, v)

    def check_bytes(self):
        for name, buf, want in (("k", self.dev.k, self.k), ("v", self.dev.v, self.v), ("bounds", self.dev.bounds, self.bounds)):
            if buf is None:
                continue
            got = buf.download(np.uint16).view(np.float16).reshape(want.shape)
            same = (got == want) | (np.isnan(got) & np.isnan(want))
            assert same.all(), (name, np.argwhere(~same)[:5])

    def queries(self):
        return (self.rng.standard_normal((self.max_rows, self.kv_heads, self.q_heads // self.kv_heads, self.hd)) * 1.2).astype(np.float32)

    def expect(self, q, layer=0, pages=None, out=None):
        """Rows that take part; the others as in `out`."""
        got = np.zeros(q.shape) if out is None else out.astype(np.float64).reshape(q.shape)
        row = 0
        for i, c in enumerate(self.counts):
            c = int(c)
            if self.want["granted"][i]:
                got[row:row + c] = ref.attention(q[row:row + c], self.k, self.v, layer, self.tables[i], int(self.lengths[i]),
                                                 None if pages is None else pages[row:row + c])
            row += c
        return got

    def attend(self, q, layer=0, selected=None, budget=0):
        """(output rows, their values before)"""
        out = self.rng.standard_normal(q.shape).astype(np.float32)
        buf = self.ctx.array(out)
        self.dev.attention(layer, self.ctx.array(q), buf, selected=selected, budget=budget)
        return buf.download(np.float32).reshape(q.shape), out

    def check_attention(self, layer=0, q=None):
        q = self.queries() if q is None else q
        got, before = self.attend(q, layer)
        want = self.expect(q, layer, out=before)
        assert not np.isnan(got).any()
        takes = self.want["requests"] != NONE
        assert np.array_equal(got[~takes], before[~takes])
        for r in np.flatnonzero(takes):
            assert rel_l2(got[r], want[r]) < TOL, (r, rel_l2(got[r], want[r]))


def strided(rng, x, stride, base):
    """x's rows in a flat array at `base`, `stride` apart, random numbers between."""
    x = x.reshape(len(x), -1)
    flat = rng.standard_normal(base + (len(x) - 1) * stride + x.shape[1]).astype(np.float32)
    for i, r in enumerate(x):
        flat[base + i * stride:base + i * stride + len(r)] = r
    return flat


# ----------------------------------------------------------------- plans
@pytest.mark.parametrize("n,page_size,tokens,spare,seed", [
    (1, 16, 1, 3, 1), (1, 128, 300, 2, 2), (3, 32, 5, 0, 3), (16, 64, 1, 1, 4), (70, 16, 40, 8, 5), (300, 32, 3, 100, 6),
    (1025, 16, 2, 400, 7), (4096, 256, 1, 2000, 8), (2500, 16, 9, 9000, 9)])
@pytest.mark.parametrize("short", [False, True])
def test_plan(ctx, n, page_size, tokens, spare, seed, short):
    """Requests of any length, idle ones, ones that are refused for each reason; pages in any order."""
    rng = np.random.default_rng(seed)
    width = 9
    cap = width * page_size
    lengths = rng.integers(0, cap + 1, n).astype(np.uint32)
    counts = np.where(rng.random(n) < 0.2, 0, rng.integers(1, tokens + 1, n)).astype(np.uint32)
    counts[rng.random(n) < 0.05] = tokens + 1                       # more rows than one request may have
    if n > 3:
        lengths[1], counts[1] = 0xFFFFFFF0, 1                       # a length that no table holds
        counts[n // 2 if short else n - 1] = 0xFFFFFFFF
    have = np.minimum(-(-lengths.astype(np.int64) // page_size), width)
    pages = int(have.sum()) + spare + 3
    any_page = rng.permutation(pages).astype(np.uint32)
    tables = np.full((n, width), NONE, np.uint32)
    at = 0
    for i, k in enumerate(have):
        tables[i, :k] = any_page[at:at + k]
        at += k
    tables[rng.random((n, width)) < 0.02] = pages + 7               # entries that are no page
    free = spare // 3 if short else spare
    pool = np.concatenate([[free], any_page[at:], np.zeros(at, np.uint32)]).astype(np.uint32)
    real = counts[counts <= tokens + 1].sum()
    max_rows = max(1, int(real) - (3 if short else -5), tokens)
    c = PagedCache(ctx, 1, pages, page_size, 2, 64, n, width, max_rows, 4, max_count=tokens)
    for buf, x in ((c.lengths, lengths), (c.counts, counts), (c.tables, tables), (c.pool, pool)):
        buf.upload(x)
    want = ref.plan(lengths, counts, tables, pool, pages, page_size, max_rows, tokens)
    for _ in range(2):                                              # a plan can be made again
        c.plan()
        got = c.read_plan()
        got["tables"] = c.tables.download(np.uint32).reshape(tables.shape)
        for name, x in want.items():
            assert np.array_equal(got[name], x), name
    assert np.array_equal(c.lengths.download(np.uint32), lengths) and np.array_equal(c.pool.download(np.uint32), pool)
    c.advance()
    assert np.array_equal(c.lengths.download(np.uint32), lengths + want["granted"])
    assert c.pool.download(np.uint32, 1)[0] == free - want["pages"]


def test_pool_of_more_than_there_is(ctx):
    """A pool that says it has more pages than the cache is taken to be full."""
    c = PagedCache(ctx, 1, 4, 16, 1, 64, 2, 8, 80, 1, max_count=80)
    c.pool.upload(np.array([0xFFFFFFFF, 3, 2, 1, 0], np.uint32))
    c.counts.upload(np.array([70, 1], np.uint32))
    c.plan()
    assert list(c.read_plan()["granted"]) == [0, 0]
    c.counts.upload(np.array([64, 1], np.uint32))
    c.plan()
    got = c.read_plan()
    assert list(got["granted"]) == [64, 0] and list(got["slots"][:64]) == list(range(64)) and (got["slots"][64:] == NONE).all()


def test_life_of_requests(ctx):
    """Steps of any counts, with what is taken back, against the restatement: no page is ever in two places."""
    rng = np.random.default_rng(3)
    n, pages, ps, width = 37, 150, 16, 20
    c = PagedCache(ctx, 1, pages, ps, 1, 64, n, width, 200, 1, max_count=60)
    lengths, tables = np.zeros(n, np.uint32), np.full((n, width), NONE, np.uint32)
    pool = np.concatenate([[pages], np.arange(pages)[::-1]]).astype(np.uint32)
    assert np.array_equal(c.pool.download(np.uint32), pool) and not c.lengths.download(np.uint32).any()
    for step in range(30):
        counts = np.where(rng.random(n) < 0.5, 0, rng.integers(1, 12, n)).astype(np.uint32)
        if step % 7 == 3:
            counts[rng.integers(n)] = 60
        c.counts.upload(counts)
        c.plan()
        want = ref.plan(lengths, counts, tables, pool, pages, ps, 200, 60)
        assert np.array_equal(c.read_plan()["slots"], want["slots"])
        c.advance()
        lengths, tables = lengths + want["granted"], want["tables"]
        pool[0] -= want["pages"]
        keep = np.where(rng.random(n) < 0.6, 0xFFFFFFFF, np.where(rng.random(n) < 0.3, 0, rng.integers(0, 200, n))).astype(np.uint32)
        if step % 3 == 2:
            c.cut(ctx.array(keep))
            lengths, tables, pool = ref.cut(keep, lengths, tables, pool, ps)
        assert np.array_equal(c.lengths.download(np.uint32), lengths)
        assert np.array_equal(c.tables.download(np.uint32).reshape(n, width), tables)
        assert np.array_equal(c.pool.download(np.uint32)[:pool[0] + 1], pool[:pool[0] + 1])
        everywhere = np.concatenate([tables[tables != NONE], pool[1:pool[0] + 1]])
        assert len(everywhere) == pages and len(set(everywhere.tolist())) == pages
    c.cut(ctx.array(np.zeros(n, np.uint32)))
    assert c.pool.download(np.uint32, 1)[0] == pages and (c.tables.download(np.uint32) == NONE).all()


def test_cut_of_many_requests(ctx):
    rng = np.random.default_rng(4)
    n, ps, width = 3000, 16, 4
    lengths = rng.integers(0, 65, n).astype(np.uint32)
    tables, at = np.full((n, width), NONE, np.uint32), 0
    pages = 3000 * 4 + 5
    for i, a in enumerate(lengths):
        k = -(-int(a) // ps)
        tables[i, :k] = np.arange(at, at + k)
        at += k
    pool = np.concatenate([[pages - at], np.arange(at, pages), np.zeros(at)]).astype(np.uint32)
    c = PagedCache(ctx, 1, pages, ps, 1, 64, n, width, 8, 1)
    for buf, x in ((c.lengths, lengths), (c.tables, tables), (c.pool, pool)):
        buf.upload(x)
    keep = rng.integers(0, 70, n).astype(np.uint32)
    c.cut(ctx.array(keep))
    for buf, x in zip((c.lengths, c.tables, c.pool), ref.cut(keep, lengths, tables, pool, ps)):
        assert np.array_equal(buf.download(np.uint32), x.ravel())


# ----------------------------------------------------------------- rows
@pytest.mark.parametrize("bounds", [False, True])
@pytest.mark.parametrize("heads,page_size,lengths,counts", [
    ((16, 2, 128), 32, [0], [1]), ((16, 2, 128), 64, [300, 7, 63], [1, 1, 1]), ((3, 3, 64), 16, [7, 0, 21], [9, 40, 3]),
    ((4, 1, 256), 128, [31, 500], [2, 150]), ((16, 2, 128), 16, [5], [200]), ((2, 2, 64), 256, [250, 1], [300, 254]),
    ((16, 2, 128), 32, [13, 0, 0, 95], [6, 0, 33, 70]), ((4, 1, 256), 16, [0, 15, 16], [17, 1, 1])])
def test_store(ctx, heads, page_size, lengths, counts, bounds):
    side = Side(ctx, heads, page_size, lengths, counts, 11, layers=2, bounds=bounds, max_rows=sum(counts) + 2)
    side.plan()
    side.check_plan()
    side.store(1)
    side.check_bytes()


def test_store_of_strided_rows(ctx):
    side = Side(ctx, (8, 4, 64), 32, [9, 40], [30, 5], 12, bounds=True)
    side.plan()
    k, v = (rows_of(side.rng, 35, 4, 64) for _ in range(2))
    for k_stride, v_stride, k_base, v_base in ((260, 300, 8, 4), (257, 259, 1, 3), (256, 263, 0, 5)):
        side.dev.store(0, ctx.array(strided(side.rng, k, k_stride, k_base)), ctx.array(strided(side.rng, v, v_stride, v_base)),
                       k_stride, v_stride, k_base, v_base)
        side.put_rows(0, k, v)
        side.check_bytes()
        k, v = k + 1, v - 2


def test_store_of_values_beyond_f16(ctx):
    """Roundings are to nearest, ties to even; what is too large is infinite, and NaN stays."""
    side = Side(ctx, (2, 2, 64), 16, [3], [8], 13, bounds=True)
    side.plan()
    k = rows_of(side.rng, 8, 2, 64)
    k[0, 0, :7] = [65504, 65519.996, 65520, -1e30, np.inf, -np.inf, np.nan]
    k[1, 0, :6] = [2.0 ** -24, 2.0 ** -25, 1.5 * 2.0 ** -25, 1 + 2.0 ** -11, 1 + 3 * 2.0 ** -11, -0.0]
    side.store(0, k, k[::-1].copy())
    side.check_bytes()


def test_rows_without_a_page_are_not_stored(ctx):
    side = Side(ctx, (2, 2, 64), 16, [20, 5], [3, 2], 14, bounds=True)
    side.tables[0, 1] = side.pages + 3
    side.dev.tables.upload(side.tables)
    side.plan()
    side.check_plan()
    assert list(side.want["slots"][:3]) == [NONE] * 3
    side.store()
    side.check_bytes()


# ------------------------------------------------------------ attention
SHAPES = [(16, 2, 128), (16, 2, 64), (8, 8, 64), (32, 4, 128), (16, 1, 256), (10, 2, 128), (3, 3, 256), (64, 2, 64), (12, 1, 128)]


@pytest.mark.parametrize("page_size", [16, 32, 128])
@pytest.mark.parametrize("heads", SHAPES)
def test_single_tokens(ctx, heads, page_size):
    lengths = [0, 1, 15, 16, 31, 32, 33, 127, 300, 511, 70]
    side = Side(ctx, heads, page_size, lengths, [1] * 10 + [0], 21, max_rows=12, layers=2)
    side.plan()
    side.store(1)
    side.check_attention(1)


@pytest.mark.parametrize("heads,page_size,lengths", [
    ((16, 2, 128), 64, [5000]), ((16, 2, 128), 16, [2047, 9000, 3]), ((16, 1, 256), 32, [3001]), ((8, 8, 64), 256, [7000, 640]),
    ((1, 1, 128), 32, [12345]), ((16, 1, 64), 32, [6000, 50])])
def test_single_tokens_over_long_caches(ctx, heads, page_size, lengths):
    side = Side(ctx, heads, page_size, lengths, [1] * len(lengths), 22)
    side.plan()
    side.store()
    side.check_attention()


@pytest.mark.parametrize("heads", SHAPES)
@pytest.mark.parametrize("page_size,lengths,counts", [
    (16, [0, 40, 333], [5, 2, 7]), (32, [0], [130]), (64, [100, 31], [70, 33]), (32, [17, 0, 0], [1, 90, 3])])
def test_several_tokens(ctx, heads, page_size, lengths, counts):
    side = Side(ctx, heads, page_size, lengths, counts, 23, max_rows=sum(counts) + 1)
    side.plan()
    side.store()
    side.check_attention()


@pytest.mark.parametrize("heads,page_size,lengths,counts", [
    ((16, 2, 128), 32, [0], [700]), ((16, 2, 128), 64, [1500], [300]), ((8, 8, 64), 16, [0, 700], [400, 100]),
    ((16, 1, 256), 32, [200], [120]), ((2, 1, 64), 128, [2000], [900])])
def test_prompts(ctx, heads, page_size, lengths, counts):
    side = Side(ctx, heads, page_size, lengths, counts, 24)
    side.plan()
    side.store()
    side.check_attention()


@pytest.mark.parametrize("heads,page_size,lengths,counts,pages", [
    ((16, 2, 128), 256, [700, 3], [1, 1], 1030), ((32, 2, 128), 64, [3000, 90, 31], [1, 1, 1], 4100), ((8, 2, 64), 64, [400, 30], [2, 1], 8200),
    ((16, 1, 64), 32, [1700], [1], 33000), ((16, 2, 256), 16, [100, 40], [1, 1], 8200), ((12, 1, 256), 128, [2000], [1], 2050)])
def test_layers_beyond_the_caches(ctx, heads, page_size, lengths, counts, pages):
    """A layer of more than 256 MB, its pages anywhere."""
    side = Side(ctx, heads, page_size, lengths, counts, 28, spare=pages - sum(-(-(a + c) // page_size) for a, c in zip(lengths, counts)))
    assert side.k.nbytes + side.v.nbytes > 256 << 20
    side.plan()
    side.store()
    side.check_attention()


@pytest.mark.parametrize("heads,n,count", [((8, 4, 64), 128, 1), ((8, 2, 128), 300, 2), ((4, 4, 64), 40, 40)])
def test_parts_of_many_pages(ctx, heads, n, count):
    """So many requests that a part has more chunks than the plan lists pages of (32) and than a wave's share of a few:
    all of them over the same 4096 slots, each with a page of its own behind them."""
    side = Side(ctx, heads, 128, [4096] + [0] * (n - 1), [count] * n, 29, spare=0)
    side.tables[:, :32] = side.tables[0, :32]
    side.lengths[:] = 4096
    side.send()
    side.plan()
    assert (side.want["granted"] == count).all()
    side.store()
    side.check_attention()


def test_many_requests(ctx):
    rng = np.random.default_rng(25)
    lengths, counts = rng.integers(0, 150, 200).tolist(), rng.integers(0, 4, 200).tolist()
    side = Side(ctx, (4, 1, 64), 16, lengths, counts, 25, max_count=3)
    side.plan()
    side.store()
    side.check_attention()


def test_refused_requests_keep_their_rows(ctx):
    side = Side(ctx, (16, 2, 128), 16, [15, 40, 31, 8], [2, 3, 1, 4], 26, max_rows=10)
    side.pool[0] = 1                                                # for the first; the third wants one too
    side.dev.pool.upload(side.pool)
    side.plan()
    side.check_plan()
    assert list(side.want["granted"]) == [2, 3, 1, 4] and side.want["pages"] == 1
    side.counts = np.array([2, 3, 2, 4], np.uint32)
    side.max_rows = 10
    side.dev.counts.upload(side.counts)
    side.plan()
    side.check_plan()
    assert list(side.want["granted"]) == [2, 3, 0, 0]               # no page is left; the row buffer ends
    side.store()
    side.check_bytes()
    side.check_attention()


def test_layout_of_query_rows(ctx):
    """Any stride and base, and q and out in one buffer."""
    side = Side(ctx, (10, 2, 64), 16, [40, 700], [3, 2], 27)
    side.plan()
    side.store()
    q = side.queries()
    want = side.expect(q)
    for stride, base in ((640, 0), (643, 5), (1300, 4)):
        src = strided(side.rng, q, stride, base)
        out = side.rng.standard_normal(src.shape).astype(np.float32)
        ob = ctx.array(out)
        side.dev.attention(0, ctx.array(src), ob, q_stride=stride, out_stride=stride, q_base=base, out_base=base)
        got = ob.download(np.float32)
        for r in range(5):
            at = slice(base + r * stride, base + r * stride + 640)
            assert rel_l2(got[at], want[r]) < TOL
            out[at] = got[at]
        assert np.array_equal(got, out)                              # nothing between the rows
    both = np.concatenate([q.reshape(5, -1), np.zeros((5, 640), np.float32)], 1)
    buf = ctx.array(both)
    side.dev.attention(0, buf, buf, q_stride=1280, out_stride=1280, out_base=640)
    got = buf.download(np.float32).reshape(5, 1280)
    assert np.array_equal(got[:, :640], both[:, :640]) and rel_l2(got[:, 640:], want) < TOL


@pytest.mark.parametrize("heads", [(16, 2, 128), (2, 2, 64), (16, 1, 256), (32, 1, 64)])
def test_what_is_not_finite_stays_with_its_slot(ctx, heads):
    """NaN and infinities in K and V, of cached tokens and of the step's own: the rows that attend to the slot, and no
    other, have what IEEE arithmetic on the formula has."""
    side = Side(ctx, heads, 16, [0, 40, 90], [40, 9, 1], 28)
    side.plan()
    shape = (50, side.kv_heads, side.hd)
    k, v = rows_of(side.rng, *shape), rows_of(side.rng, *shape)
    v[20, 0, 3], v[25, 0, 3], v[22, 0, 5], v[23, 0, 6] = np.inf, -np.inf, -np.inf, np.nan
    k[30, 0, 7] = np.nan
    v[44, -1, 60] = np.inf
    side.store(0, k, v)
    ref.put(side.v, 0, side.tables[2, 1], 0, 3, np.full(side.hd, np.nan), True)
    side.dev.v.upload(side.v)
    q = side.queries()
    got, before = side.attend(q)
    want = side.expect(q, out=before)
    assert np.array_equal(np.isnan(got), np.isnan(want)), np.argwhere(np.isnan(got) != np.isnan(want))[:4]
    assert np.array_equal(np.isinf(got), np.isinf(want)) and np.array_equal(got[np.isinf(got)], want[np.isinf(want)])
    ok = np.isfinite(want)
    assert ok[:20].all() and not ok[30:40, 0].any()
    assert rel_l2(got[ok], want[ok]) < TOL


def test_queries_that_are_not_finite(ctx):
    side = Side(ctx, (16, 2, 128), 32, [100, 50], [1, 5], 29)
    side.plan()
    side.store()
    q = side.queries()
    q[0, 0, 3, 5] = np.nan
    q[2, 1, 0, 0] = np.inf
    q[3, 0, 7] = 1e30                                               # scores of any size are finite
    got, before = side.attend(q)
    want = side.expect(q, out=before)
    nan = np.isnan(got).any(-1)
    assert nan[0, 0, 3] and nan[2, 1, 0] and nan.sum() == 2
    nan[3, 0, 7] = True                                             # the largest score alone
    assert rel_l2(got[~nan], want[~nan]) < TOL


@pytest.mark.parametrize("scale", [0.0, 1e-6, 30.0, 3e3])
def test_scores_of_any_size(ctx, scale):
    """Uniform weights, and weights of which one is all."""
    side = Side(ctx, (8, 1, 128), 32, [700, 3], [2, 1], 30)
    side.plan()
    side.store()
    q = side.queries() * np.float32(scale)
    got, before = side.attend(q)
    want = side.expect(q, out=before)
    # a score of size |s| is off by up to 2^-22 |s|, its weight by that share: |s| reaches about 10 * scale
    assert rel_l2(got, want) < TOL + 10 * scale * 2.0 ** -22 * 4


def test_pages_that_are_not(ctx):
    """Table entries that are no page hold nothing; a row without any is 0."""
    side = Side(ctx, (16, 2, 128), 16, [100, 20, 50], [1, 3, 2], 31, max_rows=6)
    side.plan()
    side.store()
    side.tables[0, [0, 3]] = [side.pages, 0xFFFFFFFE]
    side.tables[1, :] = 0xFFFFFFFF
    side.dev.tables.upload(side.tables)
    q = side.queries()
    got, before = side.attend(q)
    want = side.expect(q, out=before)
    assert not got[1:4].any() and rel_l2(got, want) < TOL


def test_plan_of_any_content_stays_in_bounds(ctx):
    """The kernels bound whatever a plan's buffer holds: rows are anything, and nothing else is written."""
    side = Side(ctx, (16, 2, 128), 16, [100, 20], [1, 30], 32, bounds=True)
    side.plan()
    rng = np.random.default_rng(1)
    words = side.dev.plan_buffer.nbytes // 4
    for most in (8, 200, 1 << 12, 1 << 32):
        junk = rng.integers(0, most, words, dtype=np.uint64).astype(np.uint32)
        side.dev.plan_buffer.upload(junk)
        guard = side.rng.standard_normal((31 + 64, 2048)).astype(np.float32)
        out = ctx.array(guard)
        q, k = ctx.array(side.queries()), ctx.array(rows_of(rng, 31, 256))
        side.dev.store(0, k, k)
        side.dev.attention(0, q, out)
        sel = side.dev.selection(4)
        side.dev.select(0, q, sel, 4)
        side.dev.attention(0, q, out, selected=sel, budget=4)
        side.dev.advance()
        ctx.sync()
        got = out.download(np.float32).reshape(guard.shape)
        assert np.array_equal(got[31:], guard[31:])


def test_lists_of_any_content_stay_in_bounds(ctx):
    """The same of plans of single tokens over tables that are divided: pages of items and joins are anything too."""
    side = Side(ctx, (16, 2, 128), 16, [2000, 20, 900], [1, 1, 1], 34, width=200)
    side.plan()
    side.store()
    rng = np.random.default_rng(2)
    words = side.dev.plan_buffer.nbytes // 4
    for most in (2, 8, 64, 200, 2400, 1 << 32):
        side.dev.plan_buffer.upload(rng.integers(0, most, words, dtype=np.uint64).astype(np.uint32))
        guard = side.rng.standard_normal((3 + 64, 2048)).astype(np.float32)
        out, q = ctx.array(guard), ctx.array(side.queries())
        side.dev.attention(0, q, out)
        assert np.array_equal(out.download(np.float32).reshape(guard.shape)[3:], guard[3:])
    side.plan()
    side.check_attention()                                          # nothing of it is left


def test_offsets_beyond_32_bits(ctx):
    """Caches of more than 4 GiB each, their last layer and pages; a selection too."""
    layers, pages, ps = 3, 24000, 256
    c = PagedCache(ctx, layers, pages, ps, 2, 128, 2, 8, 2, 16, bounds=True)
    assert c.k.nbytes > 8 << 30
    rng = np.random.default_rng(33)
    tables = np.full((2, 8), NONE, np.uint32)
    tables[0, :4], tables[1, :3] = pages - 1 - np.arange(4), [5, 16384, 23990]
    lengths = np.array([900, 600], np.uint32)
    for buf, x in ((c.lengths, lengths), (c.tables, tables), (c.counts, np.array([1, 1], np.uint32))):
        buf.upload(x)
    one = ref.k_shape(1, 1, ps, 2, 128)
    pages_k, pages_v = {}, {}
    for page in (tables[tables != NONE]).tolist():
        k, v = np.zeros(one, np.float16), np.zeros(ref.v_shape(1, 1, ps, 2, 128), np.float16)
        for h in range(2):
            for s, (x, y) in enumerate(zip(rows_of(rng, ps, 128), rows_of(rng, ps, 128))):
                ref.put(k, 0, 0, h, s, x, False)
                ref.put(v, 0, 0, h, s, y, True)
        at = (2 * pages + page) * k.nbytes
        c.k.upload(k, at)
        c.v.upload(v, at)
        b = np.stack([ref.bounds_of(ref.page_rows(k, 0, 0, h, False)) for h in range(2)])
        c.bounds.upload(b, (2 * pages + page) * b.nbytes)
        pages_k[page], pages_v[page] = k, v
    c.plan()
    k, v = rows_of(rng, 2, 2, 128), rows_of(rng, 2, 2, 128)
    c.store(2, ctx.array(k), ctx.array(v))
    q = rng.standard_normal((2, 2, 8, 128)).astype(np.float32)
    out, sel = ctx.zeros(q.nbytes), c.selection(2)
    c.attention(2, ctx.array(q), out)
    got = out.download(np.float32).reshape(q.shape)
    c.select(2, ctx.array(q), sel, 2)
    c.attention(2, ctx.array(q), out, selected=sel, budget=2)
    sparse = out.download(np.float32).reshape(q.shape)
    chosen = sel.download(np.uint32).reshape(2, 2, 2)
    for i in range(2):
        n = int(lengths[i])
        mine = tables[i][:n // ps + 1]
        kc, vc = (np.concatenate([p[int(x)] for x in mine], 1) for p in (pages_k, pages_v))
        for h in range(2):
            ref.put(kc, 0, n // ps, h, n % ps, k[i, h], False)
            ref.put(vc, 0, n // ps, h, n % ps, v[i, h], True)
        at = np.arange(len(mine), dtype=np.uint32)
        assert rel_l2(got[i], ref.attention(q[i:i + 1], kc, vc, 0, at, n)) < TOL
        bounds = np.stack([[ref.bounds_of(ref.page_rows(kc, 0, p, h, False)[:n + 1 - p * ps]) for h in range(2)]
                           for p in range(len(mine))])[None]
        for h in range(2):
            want = ref.select(ref.scores(q[i, h], bounds, 0, at, n, ps, h), 2, 0, 1)
            assert np.array_equal(chosen[i, h], want)
        assert rel_l2(sparse[i], ref.attention(q[i:i + 1], kc, vc, 0, at, n, [chosen[i]])) < TOL


# ------------------------------------------------------------ selection
def check_selection(side, budget, sinks, recent, q=None, layer=0):
    q = side.queries() if q is None else q
    sel = side.dev.selection(budget)
    side.dev.select(layer, side.ctx.array(q), sel, budget, sinks, recent)
    got = sel.download(np.uint32).reshape(side.max_rows, side.kv_heads, budget)
    want = np.full(got.shape, NONE, np.uint32)
    for r in np.flatnonzero(side.want["requests"] != NONE):
        i, p = side.want["requests"][r], int(side.want["positions"][r])
        for h in range(side.kv_heads):
            want[r, h] = ref.select(ref.scores(q[r, h], side.bounds, layer, side.tables[i], p, side.ps, h), budget, sinks, recent)
    assert np.array_equal(got, want), [(x, got[tuple(x[:2])], want[tuple(x[:2])]) for x in np.argwhere(got != want)[:1]]
    out, before = side.attend(q, layer, sel, budget)
    expected = side.expect(q, layer, want, before)
    takes = side.want["requests"] != NONE
    assert np.array_equal(out[~takes], before[~takes])
    if np.isfinite(expected).all():
        for r in np.flatnonzero(takes):
            assert rel_l2(out[r], expected[r]) < TOL, r
    return got, out, expected


@pytest.mark.parametrize("heads,page_size,lengths,counts,budget,sinks,recent", [
    ((16, 2, 128), 32, [0, 31, 32, 700, 2000], [1] * 5, 8, 1, 2), ((16, 2, 128), 16, [1000, 40], [1, 3], 20, 0, 1),
    ((8, 8, 64), 64, [900, 130], [2, 1], 3, 1, 1), ((16, 1, 256), 16, [600], [1], 9, 2, 3), ((32, 4, 128), 128, [4000, 0], [1, 1], 5, 0, 5),
    ((10, 2, 128), 16, [3000], [1], 1, 0, 1), ((3, 3, 64), 16, [5000, 9], [1, 0], 100, 50, 50), ((64, 2, 64), 32, [800], [1], 7, 1, 1),
    ((4, 2, 64), 16, [0], [300], 6, 1, 2), ((16, 2, 128), 32, [100, 7], [1, 1], 50, 0, 1), ((16, 2, 128), 32, [5000, 3300], [1, 1], 100, 1, 4),
    ((40, 2, 128), 64, [6000], [1], 60, 0, 1), ((12, 1, 256), 16, [4000], [1], 200, 3, 5), ((8, 1, 256), 64, [5000, 40], [1, 2], 50, 1, 1)])
def test_selection(ctx, heads, page_size, lengths, counts, budget, sinks, recent):
    side = Side(ctx, heads, page_size, lengths, counts, 41, layers=2, bounds=True, max_rows=sum(counts) + 1,
                width=max(-(-(a + c) // page_size) for a, c in zip(lengths, counts)))
    side.plan()
    side.store(1)
    side.check_bytes()
    check_selection(side, budget, sinks, recent, layer=1)


def test_selection_of_many_pages(ctx):
    """More pages than a workgroup has threads, and than its registers hold; bounds only, K and V are not read."""
    rng = np.random.default_rng(42)
    n, ps = 20000, 16
    c = PagedCache(ctx, 1, n, ps, 1, 64, 2, n, 2, 2, bounds=True)
    bounds = np.sort(rng.standard_normal((1, n, 1, 2, 64)).astype(np.float16), axis=3)
    tables = np.stack([rng.permutation(n), rng.permutation(n)]).astype(np.uint32)
    lengths = np.array([n * ps - 1, 9000 * ps + 3], np.uint32)
    for buf, x in ((c.bounds, bounds), (c.tables, tables), (c.lengths, lengths), (c.counts, np.array([1, 1], np.uint32))):
        buf.upload(x)
    c.plan()
    q = rng.standard_normal((2, 2, 64)).astype(np.float32)
    for budget, sinks, recent in ((1, 0, 1), (37, 3, 4), (1024, 1, 1), (7000, 10, 500), (n, 0, 1)):
        sel = c.selection(budget)
        c.select(0, ctx.array(q), sel, budget, sinks, recent)
        got = sel.download(np.uint32).reshape(2, budget)
        for i in range(2):
            want = ref.select(ref.scores(q[i], bounds, 0, tables[i], int(lengths[i]), ps, 0), budget, sinks, recent)
            assert np.array_equal(got[i], want), (budget, i)


@pytest.mark.parametrize("n,hd", [(512, 128), (513, 64), (1024, 256), (1025, 128), (2048, 64), (5000, 128), (8192, 256), (8193, 64)])
def test_selection_by_the_width_of_tables(ctx, n, hd):
    """About the sizes at which a thread holds more orders."""
    rng = np.random.default_rng(46)
    c = PagedCache(ctx, 1, n, 16, 2, hd, 2, n, 2, 4, bounds=True)
    bounds = np.sort(rng.standard_normal((1, n, 2, 2, hd)).astype(np.float16), axis=3)
    tables = np.stack([rng.permutation(n), rng.permutation(n)]).astype(np.uint32)
    lengths = np.array([n * 16 - 1, n * 11], np.uint32)
    for buf, x in ((c.bounds, bounds), (c.tables, tables), (c.lengths, lengths), (c.counts, np.array([1, 1], np.uint32))):
        buf.upload(x)
    c.plan()
    q = rng.standard_normal((2, 2, 2, hd)).astype(np.float32)
    for budget, sinks, recent in ((2, 0, 1), (n // 8, 1, 4), (n - 1, 2, 1)):
        sel = c.selection(budget)
        c.select(0, ctx.array(q), sel, budget, sinks, recent)
        got = sel.download(np.uint32).reshape(2, 2, budget)
        for i in range(2):
            for h in range(2):
                want = ref.select(ref.scores(q[i, h], bounds, 0, tables[i], int(lengths[i]), 16, h), budget, sinks, recent)
                assert np.array_equal(got[i, h], want), (budget, i, h)


def test_equal_scores_go_to_the_lowest_pages(ctx):
    """Queries of 0, bounds that are equal, and both kinds of zero."""
    side = Side(ctx, (4, 1, 64), 16, [1000, 500], [1, 1], 43, bounds=True)
    side.plan()
    side.store()
    q = np.zeros((2, 1, 4, 64), np.float32)
    q[1] = -0.0
    got, _, _ = check_selection(side, 7, 1, 2, q)
    assert list(got[0, 0]) == [0, 1, 2, 3, 4, 61, 62] and list(got[1, 0]) == [0, 1, 2, 3, 4, 30, 31]
    side.bounds[:] = np.float16(0.25)
    side.bounds[0, side.tables[0, 40], 0] = np.float16(0.5)
    side.bounds[0, side.tables[0, 20:30], 0] = np.float16(-0.25)
    side.dev.bounds.upload(side.bounds)
    got, _, _ = check_selection(side, 5, 0, 1, np.abs(side.queries()))
    assert list(got[0, 0]) == [0, 1, 2, 40, 62]


def test_scores_that_are_not_finite(ctx):
    """NaN before all, then infinities in their order. A sum that is 0 (of queries of the other sign) times an infinite
    bound is NaN, as 0 * inf is."""
    side = Side(ctx, (2, 1, 64), 16, [800], [1], 44, bounds=True)
    side.plan()
    side.store()
    for page, dim, x in ((7, 3, np.nan), (30, 0, np.inf), (31, 0, -np.inf), (12, 5, np.nan)):
        side.bounds[0, side.tables[0, page], 0, :, dim] = x
    side.tables[0, 25] = side.pages + 1                             # no page
    side.dev.bounds.upload(side.bounds)
    side.dev.tables.upload(side.tables)
    q = np.abs(side.queries()) + np.float32(0.1)
    for budget in (2, 3, 4, 5, 6, 49, 50):
        got, _, _ = check_selection(side, budget, 0, 1, q)
    got, _, _ = check_selection(side, 5, 0, 1, q)
    assert list(got[0, 0]) == [7, 12, 25, 30, 50]
    got, _, _ = check_selection(side, 5, 0, 1, -q)
    assert list(got[0, 0]) == [7, 12, 25, 30, 50]
    both = q.copy()
    both[0, 0, 1] *= -1                                             # up and down are not 0: the bound's own sign
    for page, x in ((30, -np.inf), (31, np.inf)):
        side.bounds[0, side.tables[0, page], 0, :, 0] = [-1, x] if x > 0 else [x, -1]
    side.bounds[0, side.tables[0, 32], 0, 1, 0] = -np.inf
    side.dev.bounds.upload(side.bounds)
    got, _, _ = check_selection(side, 6, 0, 1, both)
    assert list(got[0, 0]) == [7, 12, 25, 30, 31, 50]
    for budget in (4, 5, 49, 50):
        check_selection(side, budget, 0, 1, both)
    q[0, 0, 0, 9] = np.nan
    got, _, _ = check_selection(side, 3, 0, 1, q)
    assert list(got[0, 0]) == [0, 1, 50]


@pytest.mark.parametrize("page_size", [16, 64])
@pytest.mark.parametrize("heads", [(16, 2, 128), (32, 1, 64), (6, 2, 256)])
def test_selections_of_ones_own(ctx, heads, page_size):
    """Any lists: in any order, entries that are no page of the row, none at all."""
    side = Side(ctx, heads, page_size, [1000, 300, 20], [1, 2, 1], 45, bounds=True)
    side.plan()
    side.store()
    budget, q = 15, side.queries()
    lists = np.full((4, side.kv_heads, budget), NONE, np.uint32)
    used = []
    for r, p in enumerate((1000, 300, 301, 20)):
        used.append([])
        for h in range(side.kv_heads):
            n = min(budget, p // page_size + 1)
            x = side.rng.permutation(p // page_size + 1)[:n].astype(np.uint32)
            x[side.rng.random(len(x)) < 0.3] = [NONE, 1 << 20, 0x80000000][h % 3]
            lists[r, h, :n] = x
            lists[r, h, n:] = 0                                     # behind those that count
            used[-1].append(x)
    lists[2, 0] = NONE
    used[2][0] = lists[2, 0]
    out, before = side.attend(q, 0, ctx.array(lists), budget)
    want = side.expect(q, 0, used, before)
    assert not out[2, 0].any() and rel_l2(out, want) < TOL


# ------------------------------------------------------------ together
def test_graph_of_a_step(ctx):
    """A captured step replays with the state of the day: each replay against an eager step of a cache that lives the
    same life, whose scratch is left dirty in between."""
    rng = np.random.default_rng(51)
    heads, layers, n = (16, 2, 128), 2, 5

    def make():
        return PagedCache(ctx, layers, 64, 32, 2, 128, n, 12, 12, 16, max_count=4, bounds=True)
    a, b = make(), make()
    rows, qs = 12 * 256, 12 * 2048
    bufs = [[ctx.zeros(4 * s) for s in (rows, rows, qs, qs, qs)] + [c.selection(3)] for c in (a, b)]

    def step(c, x):
        k, v, q, out, sparse, sel = x
        c.plan()
        for layer in range(layers):
            c.store(layer, k, v)
            c.attention(layer, q, out)
            c.select(layer, q, sel, 3, 1, 1)
            c.attention(layer, q, sparse, selected=sel, budget=3)
        c.advance()
    for c in (a, b):
        c.counts.upload(np.array([4, 1, 0, 3, 2], np.uint32))
    step(a, bufs[0])
    step(b, bufs[1])
    ctx.sync()
    ctx.graph_begin()
    step(a, bufs[0])
    g = ctx.graph_end()
    try:
        for turn in range(6):
            counts = rng.integers(0, 4, n).astype(np.uint32)
            x = [rng.standard_normal(s).astype(np.float32) for s in (rows, rows, qs)]
            for c, u in ((a, bufs[0]), (b, bufs[1])):
                c.counts.upload(counts)
                for buf, y in zip(u, x):
                    buf.upload(y)
                for buf in u[3:5]:
                    buf.upload(np.zeros(qs, np.float32))
            ctx.graph_launch(g)
            b._scratch.fill_u32(0x7FC00000)
            step(b, bufs[1])
            ctx.sync()
            for p, q in ((a.k, b.k), (a.v, b.v), (a.bounds, b.bounds)):
                assert p.nbytes == q.nbytes
            for u, w in zip(bufs[0][3:], bufs[1][3:]):
                assert np.array_equal(u.download(np.uint32), w.download(np.uint32)), turn
            assert np.array_equal(a.lengths.download(np.uint32), b.lengths.download(np.uint32))
            assert np.array_equal(a.pool.download(np.uint32)[:1], b.pool.download(np.uint32)[:1])
    finally:
        ctx.graph_free(g)


def test_results_do_not_depend_on_scratch_or_repetition(ctx):
    side = Side(ctx, (16, 2, 128), 32, [4000, 900, 33], [1, 1, 1], 52, bounds=True)
    side.plan()
    side.store()
    q = side.queries()
    first, _ = side.attend(q)
    sel = side.dev.selection(30)
    side.dev.select(0, ctx.array(q), sel, 30, 1, 2)
    chosen = sel.download(np.uint32)
    sparse, _ = side.attend(q, 0, sel, 30)
    for word in (0, 0xFFFFFFFF, 0x7F800000, 0x3F800000):
        side.dev._scratch.fill_u32(word)
        assert np.array_equal(side.attend(q)[0], first)
        side.dev._scratch.fill_u32(word)
        side.dev.select(0, ctx.array(q), sel, 30, 1, 2)
        assert np.array_equal(sel.download(np.uint32), chosen)
        side.dev._scratch.fill_u32(word)
        assert np.array_equal(side.attend(q, 0, sel, 30)[0], sparse)


def test_two_contexts_at_once(ctx):
    """Two caches on two contexts, their calls interleaved."""
    other = Context(ctx.device)
    try:
        sides = [Side(c, (16, 2, 128), 32, [900, 40, 0], [1, 2, 20], 53 + n) for n, c in enumerate((ctx, other))]
        qs = [s.queries() for s in sides]
        outs = [s.ctx.zeros(q.nbytes) for s, q in zip(sides, qs)]
        dev_q = [s.ctx.array(q) for s, q in zip(sides, qs)]
        for s in sides:
            s.plan()
            s.store()
        for _ in range(5):
            for s, q, o in zip(sides, dev_q, outs):
                s.dev.attention(0, q, o)
        for s, q, o in zip(sides, qs, outs):
            s.ctx.sync()
            assert rel_l2(o.download(np.float32), s.expect(q)) < TOL
        del sides, outs, dev_q
    finally:
        other.close()


def test_serving(ctx):
    """Requests of two layers that come, are prompted in chunks, decode, draft with some of it rejected, and end, in a cache
    that is too small for all: every step's outputs against what each request's own tokens say."""
    rng = np.random.default_rng(54)
    layers, heads, hd, ps, n = 2, (4, 2), 64, 16, 6
    c = PagedCache(ctx, layers, 18, ps, heads[1], hd, n, 20, 96, heads[0], max_count=64, bounds=True)
    said = [[] for _ in range(n)]                                   # per request: (k, v) [layers, kv_heads, hd] of every token
    refused = 0
    for step in range(25):
        counts = np.array([rng.choice([0, 1, 1, 1, 5, 30]) for _ in range(n)], np.uint32)
        keep = np.full(n, 0xFFFFFFFF, np.uint32)
        k, v = (rows_of(rng, layers, 96, heads[1], hd) for _ in range(2))
        q = rng.standard_normal((layers, 96, heads[1], 2, hd)).astype(np.float32)
        c.counts.upload(counts)
        c.plan()
        granted = c.read_plan()["granted"]
        refused += int(((granted == 0) & (counts > 0)).sum())
        outs = [ctx.zeros(q[0].nbytes) for _ in range(2 * layers)]
        sel = c.selection(4)
        for layer in range(layers):
            qb = ctx.array(q[layer])
            c.store(layer, ctx.array(k[layer]), ctx.array(v[layer]))
            c.attention(layer, qb, outs[layer])
            c.select(layer, qb, sel, 4, 1, 1)
            c.attention(layer, qb, outs[layers + layer], selected=sel, budget=4)
            chosen = sel.download(np.uint32).reshape(96, heads[1], 4)
            row = 0
            got, few = (o.download(np.float32).reshape(q[layer].shape) for o in (outs[layer], outs[layers + layer]))
            for i in range(n):
                for t in range(int(counts[i])):
                    if not granted[i]:
                        continue
                    r = row + t
                    now = said[i] + [(k[:, row + u], v[:, row + u]) for u in range(t + 1)]
                    for h in range(heads[1]):
                        kk, vv = (np.stack([x[w][layer, h] for x in now]).astype(np.float16).astype(np.float64) for w in (0, 1))
                        s = q[layer, r, h].astype(np.float64) @ kk.T / np.sqrt(hd)
                        for have, mask in ((got, np.ones(len(now), bool)), (few, np.isin(np.arange(len(now)) // ps, chosen[r, h]))):
                            e = np.exp(s[:, mask] - s[:, mask].max(-1, keepdims=True))
                            assert rel_l2(have[r, h], e / e.sum(-1, keepdims=True) @ vv[mask]) < TOL, (step, i, t, h)
                row += int(counts[i])
        c.advance()
        row = 0
        for i in range(n):
            if granted[i]:
                said[i] += [(k[:, row + u], v[:, row + u]) for u in range(int(counts[i]))]
                if counts[i] == 5:                                   # a draft: two of five stay
                    keep[i] = len(said[i]) - 3
                if rng.random() < 0.08 or len(said[i]) > 150:
                    keep[i] = 0
                said[i] = said[i][:int(min(keep[i], len(said[i])))]
            row += int(counts[i])
        c.cut(ctx.array(keep))
        assert list(c.lengths.download(np.uint32)) == [len(x) for x in said]
    assert refused
