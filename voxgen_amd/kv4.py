"""Kv4Cache over the C ABI (vx_kv4_*): a KV cache held in 4 bits with its attention and
its eviction. No reference counterpart: the reference's caches are f16, and full at
VX_ERR_CONTEXT_FULL. Failures raise abi.VxError.

A step of every sequence, and what to do when the slots run out:

    cache = Kv4Cache(ctx, layers, sequences, kv_heads, head_dim, context, track=True)
    for layer in range(layers):
        ...                                        # k, v, q rows of the layer, RoPE applied
        cache.store(layer, k, v)
        cache.attention(layer, q, out, q_heads)    # accumulates cache.weights
    cache.advance()
    if about_to_be_full:
        cache.evict(plan, keep, sinks=4, recent=256)

Slot counts live on the device (cache.slots), so a step captures into a graph.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import abi
from .runtime import Buffer, Context

NO_SLOT = abi.KV4_NO_SLOT


class Kv4Cache:
    """K and V caches, the sequences' slot counts and next positions (u32[sequences]; a
    sequence set to NO_SLOT in `slots` is idle) and, with `track`, the accumulated
    weights and the positions of every slot."""

    def __init__(self, ctx: Context, layers: int, sequences: int, kv_heads: int, head_dim: int, context: int,
                 track: bool = False):
        self.ctx, self.layers, self.sequences, self.kv_heads = ctx, layers, sequences, kv_heads
        self.head_dim, self.context, self.track = head_dim, context, track
        self.geom = abi.Kv4Geom(layers, sequences, kv_heads, head_dim, context)
        nbytes = abi.load().vx_kv4_cache_bytes(C.byref(self.geom))
        if not nbytes:
            raise abi.VxError(abi.STATUS_CODE["VX_ERR_SHAPE"], "not a valid cache geometry", "vx_kv4_cache_bytes")
        self.k, self.v = ctx.alloc(nbytes), ctx.alloc(nbytes)
        self.slots, self.positions = ctx.zeros(4 * sequences), ctx.zeros(4 * sequences)
        table = 4 * layers * sequences * kv_heads * context
        self.weights = ctx.zeros(table) if track else None
        self.slot_positions = ctx.zeros(table) if track else None
        self._scratch = None
        self._outgrown = []
        self._pushes = {}
        lib = abi.load()
        self._store, self._load, self._attention = lib.vx_kv4_store, lib.vx_kv4_load, lib.vx_kv4_attention

    @property
    def nbytes(self) -> int:
        """Device bytes of the two caches."""
        return self.k.nbytes + self.v.nbytes

    def reset(self) -> None:
        """Every sequence empty, at position 0."""
        self.slots.fill_u32(0)
        self.positions.fill_u32(0)

    def _range(self, first, n):
        return first, self.sequences - first if n is None else n

    # A decode loop makes the same few calls over and over: their push structs are made once, by their fields.
    def _keep(self, key, push):
        if len(self._pushes) >= 4096:
            self._pushes.clear()
        self._pushes[key] = push
        return push

    def _rows(self, key):
        layer, tokens, first, n, k_stride, v_stride, k_base, v_base = key
        width = self.kv_heads * self.head_dim
        first, n = self._range(first, n)
        return self._keep(key, C.byref(abi.Kv4RowsPush(
            self.geom, layer, first, n, tokens, width if k_stride is None else k_stride,
            width if v_stride is None else v_stride, k_base, v_base)))

    def store(self, layer: int, k: Buffer, v: Buffer, tokens: int = 1, first: int = 0, n: int | None = None,
              k_stride: int | None = None, v_stride: int | None = None, k_base: int = 0, v_base: int = 0) -> None:
        """Rows of `tokens` tokens of each of n sequences from `first` on into their slots."""
        key = (layer, tokens, first, n, k_stride, v_stride, k_base, v_base)
        pc = self._pushes.get(key) or self._rows(key)
        if self.track:
            positions, table = self.positions.handle, self.slot_positions.handle
        else:
            positions = table = None
        status = self._store(self.ctx.handle, k.handle, v.handle, self.k.handle, self.v.handle, self.slots.handle,
                             positions, table, pc)
        if status:
            abi.check(status, "vx_kv4_store")

    def load(self, layer: int, k: Buffer | None, v: Buffer | None, tokens: int = 1, first: int = 0,
             n: int | None = None, k_stride: int | None = None, v_stride: int | None = None, k_base: int = 0,
             v_base: int = 0, slots: Buffer | None = None) -> None:
        """The values of the slots that store() with the same arguments fills, or of those from `slots` on."""
        key = (layer, tokens, first, n, k_stride, v_stride, k_base, v_base)
        pc = self._pushes.get(key) or self._rows(key)
        status = self._load(self.ctx.handle, self.k.handle, self.v.handle, k.handle if k else None,
                            v.handle if v else None, (slots or self.slots).handle, pc)
        if status:
            abi.check(status, "vx_kv4_load")

    def advance(self, tokens: int = 1, first: int = 0, n: int | None = None) -> None:
        """The sequences' slots and positions after `tokens` tokens went through every layer."""
        first, n = self._range(first, n)
        abi.call("vx_kv4_advance", self.ctx.handle, self.slots.handle, self.positions.handle, first, n, tokens,
                 self.context)

    def attention(self, layer: int, q: Buffer, out: Buffer, q_heads: int, tokens: int = 1, first: int = 0,
                  n: int | None = None, q_stride: int | None = None, out_stride: int | None = None, q_base: int = 0,
                  out_base: int = 0, decay: float = 1.0, scratch: Buffer | None = None) -> None:
        """Attention of the call's rows over the cache; with `track`, into self.weights too. The scratch is the
        cache's own unless one is given. It grows with the largest call, which a capture cannot do: call once with
        the same sizes before. A graph keeps the scratch that it was captured with."""
        key = (layer, q_heads, tokens, first, n, q_stride, out_stride, q_base, out_base, decay)
        pc, nbytes = self._pushes.get(key) or self._rows_of_queries(key)
        if scratch is None:
            scratch = self._scratch
            if scratch is None or scratch.nbytes < nbytes:
                scratch = self._grow(nbytes)
        status = self._attention(self.ctx.handle, q.handle, self.k.handle, self.v.handle, out.handle,
                                 self.weights.handle if self.track else None, self.slots.handle, scratch.handle, pc)
        if status:
            abi.check(status, "vx_kv4_attention")

    def _rows_of_queries(self, key):
        layer, q_heads, tokens, first, n, q_stride, out_stride, q_base, out_base, decay = key
        width = q_heads * self.head_dim
        first, n = self._range(first, n)
        pc = abi.Kv4AttentionPush(self.geom, layer, first, n, tokens, q_heads, width if q_stride is None else q_stride,
                                  width if out_stride is None else out_stride, q_base, out_base, decay)
        return self._keep(key, (C.byref(pc), abi.load().vx_kv4_attention_scratch_bytes(pc, 1 if self.track else 0)))

    def _grow(self, nbytes: int) -> Buffer:
        """The cache's own scratch, larger. The smaller one stays allocated: a captured graph may hold it. Twice the size,
        where there is room: all that stay are then no more than the one in use."""
        old = self._scratch
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

    def plan_moves(self, keep: int) -> int:
        """Moves that the plan of an eviction to `keep` slots has room for, per plane."""
        return min(keep, self.context - keep)

    def plan(self, keep: int, n: int | None = None) -> Buffer:
        """A buffer for select() and compact() of n sequences (default: all)."""
        n = self.sequences if n is None else n
        return self.ctx.alloc(max(8, 8 * self.layers * n * self.kv_heads * self.plan_moves(keep)))

    def select(self, plan: Buffer, keep: int, sinks: int = 0, recent: int = 0, first: int = 0,
               n: int | None = None) -> None:
        """Which slots stay when sequences of more than `keep` are cut to it, as moves in `plan`."""
        if not self.track:
            raise abi.VxError(abi.STATUS_CODE["VX_ERR_STATE"], "the cache tracks no weights", "vx_kv4_select")
        first, n = self._range(first, n)
        abi.call("vx_kv4_select", self.ctx.handle, self.weights.handle, self.slot_positions.handle, self.slots.handle,
                 plan.handle, abi.Kv4EvictPush(self.geom, first, n, keep, sinks, recent))

    def compact(self, plan: Buffer, keep: int, first: int = 0, n: int | None = None) -> None:
        """Carries out the moves of `plan`, and sets the slot counts."""
        first, n = self._range(first, n)
        abi.call("vx_kv4_compact", self.ctx.handle, plan.handle, self.k.handle, self.v.handle,
                 self.weights.handle if self.track else None, self.slot_positions.handle if self.track else None,
                 self.slots.handle, abi.Kv4EvictPush(self.geom, first, n, keep, 0, 0))

    def evict(self, plan: Buffer, keep: int, sinks: int = 0, recent: int = 0, first: int = 0,
              n: int | None = None) -> None:
        """select() and compact()."""
        self.select(plan, keep, sinks, recent, first, n)
        self.compact(plan, keep, first, n)

    def filled(self) -> np.ndarray:
        """The sequences' slot counts, read back."""
        return self.slots.download(np.uint32, self.sequences)
