"""PagedCache over the C ABI (vx_paged_*): an f16 KV cache in pages for many requests of
unequal length, its attention over all of a request's pages or over those that a cheap
score selects. No reference counterpart: the reference's caches are those of one sequence,
with room for its whole context. Failures raise abi.VxError.

A step of up to max_rows rows, counts[i] of them of request i:

    cache = PagedCache(ctx, layers, pages, page_size, kv_heads, head_dim, requests, table_width, max_rows, q_heads)
    cache.counts.upload(counts)                    # rows of each request in the step
    cache.plan()                                   # pages for them, slots, positions
    for layer in range(layers):
        ...                                        # k, v, q rows of the layer, RoPE applied
        cache.store(layer, k, v)
        cache.attention(layer, q, out)
    cache.advance()

With bounds=True, in place of the attention over everything:

        cache.select(layer, q, selected, budget, sinks=1, recent=4)
        cache.attention(layer, q, out, selected=selected, budget=budget)

cache.cut(keep) takes tokens back and returns their pages; not between a plan and its advance.
Lengths, counts, tables and pool live on the device, so a step captures into a graph.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import abi
from .runtime import Buffer, Context

NONE = abi.PAGED_NONE


class PagedCache:
    """K and V pages, with `bounds` those of their keys, and the state of the requests (u32):
    lengths and counts [requests], tables [requests][table_width], the pool of free pages, and
    the plan of the present step."""

    def __init__(self, ctx: Context, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int, requests: int,
                 table_width: int, max_rows: int, q_heads: int, max_count: int = 1, bounds: bool = False):
        self.ctx, self.layers, self.pages, self.page_size = ctx, layers, pages, page_size
        self.kv_heads, self.head_dim, self.requests, self.table_width = kv_heads, head_dim, requests, table_width
        self.max_rows, self.q_heads, self.max_count = max_rows, q_heads, max_count
        self.geom = abi.PagedGeom(layers, pages, page_size, kv_heads, head_dim)
        self.batch = abi.PagedBatch(self.geom, requests, table_width, max_rows, max_count, q_heads)
        lib = abi.load()
        nbytes, plan = lib.vx_paged_cache_bytes(C.byref(self.geom)), lib.vx_paged_plan_bytes(C.byref(self.batch))
        if not nbytes or not plan:
            raise abi.VxError(abi.STATUS_CODE["VX_ERR_SHAPE"], lib.vx_last_error().decode(), "vx_paged_plan_bytes")
        self.k, self.v = ctx.alloc(nbytes), ctx.alloc(nbytes)
        self.bounds = ctx.alloc(lib.vx_paged_bounds_bytes(C.byref(self.geom))) if bounds else None
        self.lengths, self.counts = ctx.alloc(4 * requests), ctx.zeros(4 * requests)
        self.tables, self.pool = ctx.alloc(4 * requests * table_width), ctx.alloc(4 * (pages + 1))
        self.plan_buffer = ctx.alloc(plan)
        self._batch = C.byref(self.batch)
        self._scratch, self._outgrown, self._pushes = None, [], {}
        self._plan, self._store, self._attention, self._select = (
            lib.vx_paged_plan, lib.vx_paged_store, lib.vx_paged_attention, lib.vx_paged_select)
        self.reset()

    @property
    def nbytes(self) -> int:
        """Device bytes of the two caches."""
        return self.k.nbytes + self.v.nbytes

    def reset(self) -> None:
        """Every request empty, every page free."""
        abi.call("vx_paged_reset", self.ctx.handle, self.lengths.handle, self.tables.handle, self.pool.handle, self._batch)

    def plan(self) -> None:
        """The step of self.counts: pages, slots and positions of its rows, and the attention's division."""
        status = self._plan(self.ctx.handle, self.lengths.handle, self.counts.handle, self.tables.handle, self.pool.handle,
                            self.plan_buffer.handle, self._batch)
        if status:
            abi.check(status, "vx_paged_plan")

    def plan_layout(self) -> dict:
        """(byte offset, words) of what a plan holds for its user."""
        at, out = abi.PAGED_PLAN_ROWS, {}
        for name, n in (("slots", self.max_rows), ("requests", self.max_rows), ("positions", self.max_rows),
                        ("granted", self.requests)):
            out[name] = (4 * at, n)
            at += n
        return out

    def read_plan(self) -> dict:
        """The plan on the host: rows, pages taken, requests and rows that take part, and the arrays of plan_layout()."""
        head = self.plan_buffer.download(np.uint32, 4)
        got = dict(zip(("rows", "pages", "taking", "rows_taking"), (int(x) for x in head)))
        for name, (offset, n) in self.plan_layout().items():
            got[name] = self.plan_buffer.download(np.uint32, n, offset)
        return got

    def advance(self) -> None:
        """Lengths and pool as the plan left them: once a plan, after the last layer, with no cut or reset since the plan."""
        abi.call("vx_paged_advance", self.ctx.handle, self.plan_buffer.handle, self.lengths.handle, self.pool.handle,
                 self._batch)

    def cut(self, keep: Buffer) -> None:
        """Requests down to keep (u32[requests]) tokens at most; their pages return to the pool. Before a plan or behind its
        advance: both go by the lengths and the pool that the plan found."""
        abi.call("vx_paged_cut", self.ctx.handle, keep.handle, self.lengths.handle, self.tables.handle, self.pool.handle,
                 self._batch)

    # A decode loop makes the same few calls over and over: their push structs are made once, by their fields.
    def _keep(self, key, push):
        if len(self._pushes) >= 4096:
            self._pushes.clear()
        self._pushes[key] = push
        return push

    def store(self, layer: int, k: Buffer, v: Buffer, k_stride: int | None = None, v_stride: int | None = None,
              k_base: int = 0, v_base: int = 0) -> None:
        """The step's rows into their slots, and the bounds of their pages."""
        key = ("store", layer, k_stride, v_stride, k_base, v_base)
        pc = self._pushes.get(key)
        if pc is None:
            width = self.kv_heads * self.head_dim
            pc = self._keep(key, C.byref(abi.PagedStorePush(
                self.batch, layer, width if k_stride is None else k_stride, width if v_stride is None else v_stride,
                k_base, v_base)))
        status = self._store(self.ctx.handle, k.handle, v.handle, self.k.handle, self.v.handle,
                             self.bounds.handle if self.bounds else None, self.plan_buffer.handle, pc)
        if status:
            abi.check(status, "vx_paged_store")

    def attention(self, layer: int, q: Buffer, out: Buffer, q_stride: int | None = None, out_stride: int | None = None,
                  q_base: int = 0, out_base: int = 0, selected: Buffer | None = None, budget: int = 0,
                  scratch: Buffer | None = None) -> None:
        """Attention of the step's rows, over all positions up to their own or those of the selected pages. The
        scratch is the cache's own unless one is given. It grows with the largest call, which a capture cannot do: call
        once with the same sizes before. A graph keeps the scratch that it was captured with."""
        key = ("attention", layer, q_stride, out_stride, q_base, out_base, budget)
        got = self._pushes.get(key)
        if got is None:
            width = self.q_heads * self.head_dim
            pc = abi.PagedAttentionPush(self.batch, layer, width if q_stride is None else q_stride,
                                        width if out_stride is None else out_stride, q_base, out_base, budget)
            got = self._keep(key, (C.byref(pc), abi.load().vx_paged_attention_scratch_bytes(pc)))
        pc, nbytes = got
        if scratch is None:
            scratch = self._room(nbytes)
        status = self._attention(self.ctx.handle, q.handle, self.k.handle, self.v.handle, out.handle, self.tables.handle,
                                 self.plan_buffer.handle, selected.handle if selected else None, scratch.handle, pc)
        if status:
            abi.check(status, "vx_paged_attention")

    def selection(self, budget: int) -> Buffer:
        """A buffer for select() and attention(): u32 [max_rows][kv_heads][budget]."""
        return self.ctx.alloc(4 * self.max_rows * self.kv_heads * budget)

    def select(self, layer: int, q: Buffer, selected: Buffer, budget: int, sinks: int = 0, recent: int = 1,
               q_stride: int | None = None, q_base: int = 0, scratch: Buffer | None = None) -> None:
        """The pages that each of the step's rows attends to."""
        if not self.bounds:
            raise abi.VxError(abi.STATUS_CODE["VX_ERR_STATE"], "the cache has no bounds", "vx_paged_select")
        key = ("select", layer, budget, sinks, recent, q_stride, q_base)
        got = self._pushes.get(key)
        if got is None:
            pc = abi.PagedSelectPush(self.batch, layer, self.q_heads * self.head_dim if q_stride is None else q_stride, q_base,
                                     budget, sinks, recent)
            got = self._keep(key, (C.byref(pc), abi.load().vx_paged_select_scratch_bytes(pc)))
        pc, nbytes = got
        if scratch is None:
            scratch = self._room(nbytes)
        status = self._select(self.ctx.handle, q.handle, self.bounds.handle, self.tables.handle, self.plan_buffer.handle,
                              selected.handle, scratch.handle, pc)
        if status:
            abi.check(status, "vx_paged_select")

    def _room(self, nbytes: int) -> Buffer:
        """The cache's own scratch, larger if need be. The smaller one stays allocated: a captured graph may hold it. Twice
        the size, where there is room: all that stay are then no more than the one in use."""
        old = self._scratch
        if old is not None and old.nbytes >= nbytes:
            return old
        double = 2 * old.nbytes if old is not None else 0
        try:
            self._scratch = self.ctx.alloc(max(4, nbytes, double))
        except abi.VxError as e:
            if e.name != "VX_ERR_OOM" or double <= nbytes:
                raise
            self._scratch = self.ctx.alloc(nbytes)
        if old is not None:
            self._outgrown.append(old)
        return self._scratch
