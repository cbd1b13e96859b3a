"""The paged KV cache's attention where values or tables are out of the ordinary, on tiles of 8, 16 and 32
query rows of each head size: against the formula in 64 bits, element by element (a library's matrix product need not
keep to IEEE arithmetic where factors are infinite).

Finite outputs are compared by relative 2-norm with the bound that test_gpu_paged.py derives; a score of the path for
infinite keys is a sum of head_dim products in f32, off by sqrt(head_dim) 2^-24 of its terms' size, which is below
what that bound has for products of two terms.
"""
import ctypes as C

import numpy as np
import pytest

import pagedref as ref
from conftest import rel_l2
from test_gpu_paged import NONE, TOL, Side, rows_of
from voxgen_amd import abi
from voxgen_amd.paged import PagedCache

pytestmark = pytest.mark.gpu

# (heads, rows of a request): tokens x group is what a tile is chosen by
TILES = [((16, 2, 128), 1), ((8, 4, 64), 4), ((4, 1, 256), 2),            # 8 rows
         ((32, 2, 128), 1), ((16, 4, 64), 3), ((16, 1, 256), 1),          # 16
         ((16, 2, 128), 5), ((8, 1, 64), 9), ((6, 1, 256), 7)]            # 32


def by_formula(side, q, layer=0, pages=None, tables=None):
    """softmax(q . K / sqrt(head_dim)) . V of every row that takes part, NaN in the others."""
    out = np.full(q.shape, np.nan)
    tables = side.tables if tables is None else tables
    row = 0
    with np.errstate(all="ignore"):
        for i, count in enumerate(side.counts.tolist()):
            n = int(side.lengths[i]) + count
            for h in range(side.kv_heads):
                k, there = ref.rows(side.k, layer, tables[i], h, n, False)
                v, _ = ref.rows(side.v, layer, tables[i], h, n, True)
                for t in range(count if side.want["granted"][i] else 0):
                    sees = there & (np.arange(n) <= n - count + t)
                    if pages is not None:
                        sees &= np.isin(np.arange(n) // side.ps, pages[row + t][h])
                    for j in range(q.shape[2]):
                        s = (q[row + t, h, j].astype(np.float64) * k[sees]).sum(-1) / np.sqrt(side.hd)
                        e = np.exp(s - s.max()) if len(s) else s
                        out[row + t, h, j] = (e[:, None] / e.sum() * v[sees]).sum(0) if len(s) else 0
            row += count
    return out


def check(got, want):
    assert np.array_equal(np.isnan(got), np.isnan(want)), np.argwhere(np.isnan(got) != np.isnan(want))[:4]
    assert np.array_equal(np.isinf(got), np.isinf(want)) and np.array_equal(got[np.isinf(got)], want[np.isinf(want)])
    for r in np.ndindex(*got.shape[:3]):
        ok = np.isfinite(want[r])
        off = rel_l2(got[r][ok], want[r][ok])
        assert off < TOL, r


def mixed_signs(q, dim, sign):
    """Queries whose product with an infinity of that sign in dimension `dim` is -inf; of some rows, however small they
    are there; of some +inf or, where they are 0, NaN."""
    rows = q.reshape(-1, q.shape[-1])
    rows[:, dim] = -sign * (np.abs(rows[:, dim]) + np.float32(0.01))
    rows[1::5, dim] *= np.float32(1e-14)
    rows[3::11, dim] *= -1
    rows[7::11, dim] = 0
    return q


# ------------------------------------------------------------ infinite keys
@pytest.mark.parametrize("heads,count", TILES)
@pytest.mark.parametrize("sign", [1, -1])
def test_infinite_keys(ctx, heads, count, sign):
    """A key that is infinite (what is stored of 65520 or more is) has a score of -inf for queries of the other sign: a
    weight of 0, and the row is what its other slots make it. Cached ones, and the step's own, which its earlier rows do not
    attend to; one whose value is infinite too, for 0 times that is NaN."""
    side = Side(ctx, heads, 16, [90, 40, 33], [count] * 3, 61)
    side.plan()
    ref_k = np.full(side.hd, np.float32(0.5))
    ref_k[3] = sign * np.inf
    ref.put(side.k, 0, side.tables[0, 1], 0, 1, ref_k, False)
    ref.put(side.k, 0, side.tables[1, 0], 0, 11, ref_k, False)
    for slot, dim, x in ((11, 2, np.inf), (12, 6, -np.inf)):
        v = np.ones(side.hd, np.float32)
        v[dim] = x
        ref.put(side.v, 0, side.tables[1, 0], 0, slot, v, True)
    side.send()
    side.plan()
    k, v = (rows_of(side.rng, side.max_rows, side.kv_heads, side.hd) for _ in range(2))
    k[-1, -1, 3] = sign * 70000                                     # of the third request's last row
    side.store(0, k, v)
    assert np.isinf(side.k[0, side.tables[2, (33 + count - 1) // 16]]).any()
    q = mixed_signs(side.queries(), 3, sign)
    want = by_formula(side, q)
    assert np.isfinite(want[0, 0]).all(-1).any() and np.isnan(want).any()
    got, _ = side.attend(q)
    check(got, want)


@pytest.mark.parametrize("heads", [(16, 2, 128), (32, 2, 64), (8, 1, 256)])
def test_infinite_keys_of_divided_requests(ctx, heads):
    """Among parts that have none, and a part of which every slot has one."""
    side = Side(ctx, heads, 32, [3000, 2500, 0], [1] * 3, 62, width=100)
    side.plan()
    side.store()
    for i, slots in ((0, list(range(300)) + [2999]), (1, [1700])):
        for s in slots:
            for h in range(side.kv_heads):
                x = rows_of(side.rng, side.hd)
                x[9] = -np.inf
                ref.put(side.k, 0, side.tables[i, s // 32], h, s % 32, x, False)
    x = rows_of(side.rng, side.hd)
    x[9] = -np.inf
    ref.put(side.k, 0, side.tables[2, 0], 0, 0, x, False)           # all that a request has: -inf less -inf is NaN
    side.send()
    q = mixed_signs(side.queries(), 9, -1)
    want = by_formula(side, q)
    assert np.isfinite(want[:2]).all(-1).sum() > 5 and np.isnan(want[2, 0]).all()
    check(side.attend(q)[0], want)


@pytest.mark.parametrize("heads", [(16, 2, 128), (32, 2, 64), (24, 1, 256)])
def test_infinite_keys_of_selected_pages(ctx, heads):
    side = Side(ctx, heads, 16, [1500, 200], [1, 1], 63, width=120)
    side.plan()
    side.store()
    for i, s in ((0, 37), (0, 1490), (1, 60)):
        x = rows_of(side.rng, side.hd)
        x[9] = np.inf
        ref.put(side.k, 0, side.tables[i, s // 16], 0, s % 16, x, False)
    side.send()
    lists = np.full((2, side.kv_heads, 90), NONE, np.uint32)
    lists[0], lists[1, :, :6] = np.arange(2, 92), [3, 0, 9, 2, 1, 12]
    lists[0, :, -1] = 1490 // 16
    q = mixed_signs(side.queries(), 9, 1)
    want = by_formula(side, q, pages=lists)
    assert np.isfinite(want[:, 0]).all(-1).any() and np.isnan(want).any()
    check(side.attend(q, 0, ctx.array(lists), 90)[0], want)


# ------------------------------------------------------------ infinite values in parts that hardly count
@pytest.mark.parametrize("selected", [False, True])
def test_infinite_values_in_parts_of_little_weight(ctx, selected):
    """An infinite value reaches the rows that attend to it, whatever its weight, if all its part's are far below the
    others': 300 less in the exponent here, which 64 bits hold and 32 do not."""
    side = Side(ctx, (8, 1, 128), 32, [3000], [1], 64, width=100)
    side.plan()
    u = np.where(side.rng.random(128) < 0.5, -1, 1).astype(np.float32)
    for s in range(3000):
        x = u * (3 if s >= 1500 else -3) + 0.01 * side.rng.standard_normal(128).astype(np.float32)
        ref.put(side.k, 0, side.tables[0, s // 32], 0, s % 32, x, False)
    v = np.ones(128, np.float32)
    v[[4, 5]] = np.inf, -np.inf
    ref.put(side.v, 0, side.tables[0, 1], 0, 7, v, True)
    side.send()
    side.plan()
    side.store(0, u[None, None] * 3, rows_of(side.rng, 1, 1, 128))
    q = (np.ones((1, 1, 8, 128), np.float32) * u * 4.4).astype(np.float32)
    if selected:
        lists = np.arange(94, dtype=np.uint32).reshape(1, 1, 94)
        got, want = side.attend(q, 0, ctx.array(lists), 94)[0], by_formula(side, q, pages=lists)
    else:
        got, want = side.attend(q)[0], by_formula(side, q)
    assert np.isinf(want).sum() == 16 and not np.isnan(want).any()
    check(got, want)


# ------------------------------------------------------------ tables that change behind a plan
def edit(side, tables, i, gone, swapped):
    """Entries of request i that are no page, and two whose pages change places."""
    tables[i, gone] = [side.pages, 0xFFFFFFFE, NONE][:len(gone)]
    tables[i, swapped] = tables[i, swapped[::-1]]


@pytest.mark.parametrize("heads,count", TILES)
@pytest.mark.parametrize("before", [True, False])
def test_tables_of_the_call(ctx, heads, count, before):
    """Pages are those of the tables at the time of the attention, whether the plan was made of the same or not: the first
    ones of a part, those further on, and a request without any."""
    side = Side(ctx, heads, 16, [1400, 150, 20], [count] * 3, 65, max_rows=3 * count + 1, width=95)
    side.plan()
    side.store()
    tables = side.tables.copy()
    edit(side, tables, 0, [0, 3, 70], [1, 80])
    edit(side, tables, 1, [2], [4, 5])
    tables[2, :] = NONE
    side.dev.tables.upload(tables)
    if before:
        side.dev.plan()
    q = side.queries()
    want = by_formula(side, q, tables=tables)
    got, old = side.attend(q)
    assert not want[2 * count:3 * count].any()
    assert np.array_equal(got[3 * count:], old[3 * count:])
    check(got[:3 * count], want[:3 * count])


@pytest.mark.parametrize("heads", [(8, 4, 64), (16, 1, 128), (4, 1, 256)])
def test_tables_of_the_call_in_divided_requests(ctx, heads):
    side = Side(ctx, heads, 32, [6000, 2100], [1, 1], 66, width=200)
    side.plan()
    side.store()
    tables = side.tables.copy()
    edit(side, tables, 0, [0, 8, 101], [7, 150])
    edit(side, tables, 1, list(range(3)), [40, 60])
    tables[1, 8:16] = NONE                                          # a part's whole
    side.dev.tables.upload(tables)
    q = side.queries()
    check(side.attend(q)[0], by_formula(side, q, tables=tables))


@pytest.mark.parametrize("heads,page_size,lengths,count,pages", [
    ((16, 2, 128), 256, [900, 3], 1, 1030), ((32, 2, 64), 256, [600, 30], 1, 2060), ((16, 1, 256), 128, [500, 40], 1, 2060)])
def test_layers_beyond_the_caches(ctx, heads, page_size, lengths, count, pages):
    """Of more than 256 MB, which are read past the caches: infinite keys, and tables that change behind the plan."""
    need = [-(-(a + count) // page_size) for a in lengths]
    side = Side(ctx, heads, page_size, lengths, [count] * 2, 69, spare=pages - sum(need), width=12)
    assert side.k.nbytes + side.v.nbytes > 256 << 20
    side.plan()
    side.store()
    q = mixed_signs(side.queries(), 5, 1)
    x = rows_of(side.rng, side.hd)
    x[5] = np.inf
    ref.put(side.k, 0, side.tables[0, 0], 0, 7, x, False)
    side.dev.k.upload(side.k)
    want = by_formula(side, q)
    assert np.isfinite(want[0, 0]).all(-1).any() and np.isnan(want).any()
    check(side.attend(q)[0], want)
    tables = side.tables.copy()
    tables[0, [0, 1]] = tables[0, [1, 0]]
    tables[1, 0] = side.pages
    side.dev.tables.upload(tables)
    check(side.attend(q)[0], by_formula(side, q, tables=tables))


# ------------------------------------------------------------ two batches over one state
@pytest.mark.parametrize("heads", [(16, 2, 128), (16, 1, 256)])
def test_steps_of_two_batches_over_the_same_requests(ctx, heads):
    """Prompts by a batch that has room for them, single tokens by one of a row a request: lengths, tables, pool and pages are
    the same, plans and scratch each batch's own."""
    q_heads, kv_heads, hd = heads
    side = Side(ctx, heads, 16, [0, 700, 33], [40, 3, 0], 68, spare=8, max_rows=60, max_count=40, width=50)
    wide, state = side.dev, "k v lengths counts tables pool".split()
    narrow = PagedCache(ctx, 1, side.pages, 16, kv_heads, hd, 3, side.width, 3, q_heads)
    for name in state:
        setattr(narrow, name, getattr(wide, name))
    for dev, counts in ((wide, [40, 3, 0]), (narrow, [1, 0, 1]), (narrow, [1, 1, 1]), (wide, [0, 37, 5]), (narrow, [1, 1, 1])):
        side.dev, side.max_rows, side.counts = dev, dev.max_rows, np.array(counts, np.uint32)
        dev.counts.upload(side.counts)
        side.plan()
        side.check_plan()
        assert list(side.want["granted"]) == counts
        side.store()
        side.check_bytes()
        side.check_attention()
        dev.advance()
        side.lengths = side.lengths + side.want["granted"]
        side.pool[0] -= side.want["pages"]
        assert np.array_equal(wide.lengths.download(np.uint32), side.lengths) and wide.pool.download(np.uint32, 1)[0] == side.pool[0]


# ------------------------------------------------------------ what a call does not write
class Guarded:
    """Buffers of chosen sizes with words behind them that no call may change."""

    def __init__(self, ctx, rng):
        self.ctx, self.rng, self.all = ctx, rng, []

    def buffer(self, words):
        x = self.rng.integers(0, 1 << 32, words + 256, dtype=np.uint64).astype(np.uint32)
        b = self.ctx.array(x)
        self.all.append((b, words, x[words:]))
        return b

    def check(self):
        for b, words, x in self.all:
            assert np.array_equal(b.download(np.uint32, 256, 4 * words), x), words


@pytest.mark.parametrize("heads,max_count", [((16, 2, 128), 1), ((32, 2, 64), 1), ((8, 1, 256), 20), ((16, 2, 128), 20)])
def test_no_content_makes_a_call_write_behind_a_buffer(ctx, heads, max_count):
    """Plans, tables, lengths, pools and selections of any content, in buffers of just the sizes that a call asks for."""
    q_heads, kv_heads, hd = heads
    rng = np.random.default_rng(67)
    requests, width, rows, pages, ps, budget, layers = 3, 120, 21, 70, 16, 9, 2
    batch = abi.PagedBatch(abi.PagedGeom(layers, pages, ps, kv_heads, hd), requests, width, rows, max_count, q_heads)
    lib, wide, row = abi.load(), q_heads * hd, kv_heads * hd
    store = abi.PagedStorePush(batch, 1, row, row, 0, 0)
    attn, sparse = (abi.PagedAttentionPush(batch, 1, wide, wide, 0, 0, n) for n in (0, budget))
    pick = abi.PagedSelectPush(batch, 1, wide, 0, budget, 1, 2)
    g = Guarded(ctx, rng)
    nbytes = lib.vx_paged_cache_bytes(C.byref(batch.geom))
    need = lib.vx_paged_plan_bytes(C.byref(batch))
    kc, vc, bounds = (g.buffer(n // 4) for n in (nbytes, nbytes, lib.vx_paged_bounds_bytes(C.byref(batch.geom))))
    lengths, counts, keep, tables, pool = (g.buffer(n) for n in (requests, requests, requests, requests * width, pages + 1))
    plan, k, v, q, out, sel = (g.buffer(n) for n in (need // 4, rows * row, rows * row, rows * wide, rows * wide, rows * kv_heads * budget))
    scratch = [g.buffer(n // 4) for n in (lib.vx_paged_attention_scratch_bytes(C.byref(attn)), lib.vx_paged_attention_scratch_bytes(C.byref(sparse)),
                                          lib.vx_paged_select_scratch_bytes(C.byref(pick)))]
    h = lambda *x: [b.handle for b in x]  # noqa: E731
    for most in (3, 8, 70, 1900, 1 << 12, 1 << 32):
        fill = lambda b, words, top=most: b.upload(rng.integers(0, top, words, dtype=np.uint64).astype(np.uint32))  # noqa: E731
        for made in (False, True):
            fill(lengths, requests), fill(counts, requests, min(most, 30)), fill(keep, requests)
            fill(tables, requests * width), fill(pool, pages + 1), fill(plan, need // 4), fill(sel, rows * kv_heads * budget)
            if made:
                abi.call("vx_paged_plan", ctx.handle, *h(lengths, counts, tables, pool, plan), batch)
            abi.call("vx_paged_store", ctx.handle, *h(k, v, kc, vc, bounds, plan), store)
            abi.call("vx_paged_attention", ctx.handle, *h(q, kc, vc, out, tables, plan), None, scratch[0].handle, attn)
            abi.call("vx_paged_attention", ctx.handle, *h(q, kc, vc, out, tables, plan, sel, scratch[1]), sparse)
            abi.call("vx_paged_select", ctx.handle, *h(q, bounds, tables, plan, sel, scratch[2]), pick)
            abi.call("vx_paged_attention", ctx.handle, *h(q, kc, vc, out, tables, plan, sel, scratch[1]), sparse)
            abi.call("vx_paged_advance", ctx.handle, *h(plan, lengths, pool), batch)
            abi.call("vx_paged_cut", ctx.handle, *h(keep, lengths, tables, pool), batch)
            g.check()
    abi.call("vx_paged_reset", ctx.handle, *h(lengths, tables, pool), batch)
    g.check()
