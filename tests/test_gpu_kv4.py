"""The 4-bit KV cache on the GPU against its restatement in 64 bits (oracle/kv4ref.py).

Whatever is stored, moved or selected is exact: cache bytes, positions, plans and read-back
values are compared bit for bit, with the slots that a call does not fill included.

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

import kv4ref
from conftest import rel_l2
from voxgen_amd import abi
from voxgen_amd.kv4 import NO_SLOT, Kv4Cache
from voxgen_amd.runtime import Context

pytestmark = pytest.mark.gpu
TOL = 2e-5


def rows_of(rng, *shape):
    """Keys or values with channel means of their own, as trained models have."""
    return (rng.standard_normal(shape) + 1.5 * rng.standard_normal(shape[-1])).astype(np.float32)


class Side:
    """A cache on the device and the same bytes here, slots filled up to `bases` and random bits in the others."""

    def __init__(self, ctx, geom, bases, seed, track=False):
        self.ctx, self.rng = ctx, np.random.default_rng(seed)
        L, S, H, hd, context = geom
        self.geom, self.bases = geom, list(bases)
        self.dev = Kv4Cache(ctx, L, S, H, hd, context, track=track)
        self.k, self.v = (kv4ref.blank(L, S, H, hd, context, self.rng) for _ in range(2))
        for s, n in enumerate(self.bases):
            for layer in range(L):
                for h in range(H):
                    for cache, is_v in ((self.k, False), (self.v, True)):
                        c, d, o = kv4ref.encode(rows_of(self.rng, 0 if n == NO_SLOT else n, hd))
                        for j in range(len(c)):
                            kv4ref.put(cache, (layer, s, h), j, c[j], d[j], o[j], is_v)
        self.send()

    def send(self):
        self.dev.k.upload(self.k)
        self.dev.v.upload(self.v)
        self.dev.slots.upload(np.array(self.bases, np.uint32))

    def check_bytes(self):
        for buf, want in ((self.dev.k, self.k), (self.dev.v, self.v)):
            got = buf.download(np.uint32).reshape(want.shape)
            assert np.array_equal(got, want), np.argwhere(got != want)[:5]

    def put_rows(self, layer, x, tokens, is_v, first=0, n=None):
        """Rows [n * tokens, H * hd] into the slots they belong to, here."""
        L, S, H, hd, context = self.geom
        n = S - first if n is None else n
        for i in range(n):
            base = self.bases[first + i]
            for t in range(tokens):
                if base >= context or base + t >= context:
                    continue
                for h in range(H):
                    c, d, o = kv4ref.encode(x[i * tokens + t, h * hd:(h + 1) * hd])
                    kv4ref.put(self.v if is_v else self.k, (layer, first + i, h), base + t, c, d, o, is_v)


def strided(rng, x, stride, base):
    """x's rows in a flat array at `base`, `stride` apart, random numbers between."""
    flat = rng.standard_normal(base + (len(x) - 1) * stride + x.shape[1]).astype(np.float32)
    for i, r in enumerate(x):
        flat[base + i * stride:base + i * stride + len(r)] = r
    return flat


# ----------------------------------------------------------------- rows
@pytest.mark.parametrize("hd,H,bases,tokens,context,pad,base", [
    (128, 2, [0], 1, 1, 0, 0), (128, 2, [300], 1, 512, 0, 0), (64, 3, [7], 9, 40, 0, 0), (256, 1, [31], 2, 64, 4, 8),
    (128, 2, [0], 200, 256, 3, 1), (64, 2, [5, NO_SLOT, 0, 37], 6, 41, 1, 2), (128, 1, [40, 39, 33], 8, 40, 0, 4),
    (256, 2, [13, 26], 33, 70, 0, 0)])
def test_store_and_load_are_exact(ctx, hd, H, bases, tokens, context, pad, base):
    side = Side(ctx, (2, len(bases), H, hd, context), bases, 11, track=True)
    rng, width, n = side.rng, H * hd, len(bases) * tokens
    stride = width + pad
    k, v = rows_of(rng, n, width), rows_of(rng, n, width)
    positions = rng.integers(0, 1 << 20, len(bases), dtype=np.uint32)
    side.dev.positions.upload(positions)
    table = rng.integers(0, 1 << 32, (2, len(bases), H, context), dtype=np.uint32)
    side.dev.slot_positions.upload(table)
    kb, vb = ctx.array(strided(rng, k, stride, base)), ctx.array(strided(rng, v, width, 0))
    side.dev.store(1, kb, vb, tokens=tokens, k_stride=stride, k_base=base)
    side.put_rows(1, k, tokens, False)
    side.put_rows(1, v, tokens, True)
    for s, b in enumerate(bases):
        for t in range(tokens):
            if b < context and b + t < context:
                table[1, s, :, b + t] = positions[s] + t
    side.check_bytes()
    assert np.array_equal(side.dev.slot_positions.download(np.uint32).reshape(table.shape), table)
    # read back: rows with a slot have what they stand for, the others stay
    back = [rng.standard_normal(base + n * stride).astype(np.float32), rng.standard_normal(n * width).astype(np.float32)]
    ob = [ctx.array(b) for b in back]
    side.dev.load(1, ob[0], ob[1], tokens=tokens, k_stride=stride, k_base=base)
    for i, b in enumerate(bases):
        for t in range(tokens):
            if b < context and b + t < context:
                r = i * tokens + t
                back[0][base + r * stride:base + r * stride + width] = kv4ref.stored(k[r].reshape(H, hd)).ravel()
                back[1][r * width:(r + 1) * width] = kv4ref.stored(v[r].reshape(H, hd)).ravel()
    for b, want in zip(ob, back):
        assert np.array_equal(b.download(np.float32), want)


def test_store_of_special_values(ctx):
    """Zeros, one value, ties between codes, the least and the largest numbers, infinities, a NaN."""
    hd, rng = 128, np.random.default_rng(3)
    x = np.zeros((12, hd), np.float32)
    x[1] = 3.25
    x[2] = np.arange(hd) % 31 / 2                      # steps of 1 and ties at every half
    x[3] = rng.standard_normal(hd) * 1e-7              # f16 subnormals
    x[4] = rng.standard_normal(hd) * 1e-38
    x[5] = rng.standard_normal(hd) * 1e30
    x[6, ::3], x[6, 1::3] = np.inf, -np.inf
    x[7] = rng.standard_normal(hd)
    x[7, 40] = np.nan
    x[8] = 1000 + rng.standard_normal(hd) * 1e-3       # an offset far above the step
    x[9, 5] = 70000
    x[10] = -0.0
    x[11] = np.float32(1e-45)
    side = Side(ctx, (1, 1, 1, hd, 40), [3], 4)
    side.dev.store(0, ctx.array(x), ctx.array(x[::-1].copy()), tokens=12)
    side.put_rows(0, x, 12, False)
    side.put_rows(0, x[::-1], 12, True)
    side.check_bytes()
    back = ctx.zeros(x.nbytes)
    side.dev.load(0, back, None, tokens=12)
    assert np.array_equal(back.download(np.float32).reshape(x.shape), kv4ref.stored(x).astype(np.float32), equal_nan=True)
    assert np.isnan(back.download(np.float32).reshape(x.shape)[7]).sum() == 32


def test_rows_side_by_side_in_one_buffer(ctx):
    """k and v, and q and out, as the halves of rows of one buffer: what they give in buffers of their own."""
    hd, H, qh, tokens, context = 128, 2, 8, 37, 64
    rng, width, wide = np.random.default_rng(13), H * hd, qh * hd
    cache = Kv4Cache(ctx, 1, 1, H, hd, context)
    kv = rows_of(rng, tokens, 2 * width)
    both = ctx.array(kv)
    cache.store(0, both, both, tokens=tokens, k_stride=2 * width, v_stride=2 * width, v_base=width)
    back = ctx.zeros(kv.nbytes)
    cache.load(0, back, back, tokens=tokens, k_stride=2 * width, v_stride=2 * width, v_base=width)
    assert np.array_equal(back.download(np.float32).reshape(tokens, 2 * H, hd), kv4ref.stored(kv.reshape(tokens, 2 * H, hd)))
    q = rng.standard_normal((tokens, wide)).astype(np.float32)
    out = ctx.zeros(q.nbytes)
    cache.attention(0, ctx.array(q), out, qh, tokens=tokens)
    rows = ctx.array(np.concatenate([q, np.zeros_like(q)], 1))
    cache.attention(0, rows, rows, qh, tokens=tokens, q_stride=2 * wide, out_stride=2 * wide, out_base=wide)
    got = rows.download(np.float32).reshape(tokens, 2, wide)
    assert np.array_equal(got[:, 0], q) and np.array_equal(got[:, 1], out.download(np.float32).reshape(tokens, wide))


def test_advance(ctx):
    slots, pos = ctx.array(np.array([0, 5, NO_SLOT, 38, 40, 99], np.uint32)), ctx.array(np.arange(6, dtype=np.uint32) * 100)
    abi.call("vx_kv4_advance", ctx.handle, slots.handle, pos.handle, 1, 5, 3, 40)
    assert list(slots.download(np.uint32)) == [0, 8, NO_SLOT, 40, 40, 99]
    assert list(pos.download(np.uint32)) == [0, 103, 200, 303, 403, 503]


# ----------------------------------------------------------------- attention
def attend(side, layer, tokens, q_heads, first=0, n=None, pad=0, base=0, decay=1.0, q_scale=1.2, check=TOL):
    """Runs the attention and compares its rows (and weights) with the restatement; returns them."""
    ctx, rng = side.ctx, side.rng
    L, S, H, hd, context = side.geom
    n = S - first if n is None else n
    width, group = q_heads * hd, q_heads // H
    q = (rng.standard_normal((n * tokens, width)) * q_scale).astype(np.float32)
    before = rng.standard_normal(base + (n * tokens - 1) * (width + pad) + width).astype(np.float32)
    ob = ctx.array(before)
    table = None
    if side.dev.track:
        table = rng.random((L, S, H, context)).astype(np.float32)
        side.dev.weights.upload(table)
    side.dev.attention(layer, ctx.array(strided(rng, q, width + pad, base)), ob, q_heads, tokens=tokens, first=first, n=n,
                       q_stride=width + pad, out_stride=width + pad, q_base=base, out_base=base, decay=decay)
    got = ob.download(np.float32)
    out = np.zeros((n * tokens, width))
    if table is not None:
        weights = side.dev.weights.download(np.float32).reshape(table.shape)
        want_w, touched = table.astype(np.float64), np.zeros(table.shape, bool)
    for i in range(n):
        b = side.bases[first + i]
        x = q[i * tokens:(i + 1) * tokens].reshape(tokens, H, group, hd)
        o, w = kv4ref.attention(x, side.k, side.v, layer, first + i, b, context)
        out[i * tokens:(i + 1) * tokens] = o.reshape(tokens, width)
        if table is not None and w.shape[1]:
            m = w.shape[1]
            old = np.where(np.arange(m) < b, decay * want_w[layer, first + i, :, :m], 0.0)
            want_w[layer, first + i, :, :m] = old + w
            touched[layer, first + i, :, :m] = True
    at = base + np.arange(n * tokens)[:, None] * (width + pad) + np.arange(width)
    rows = got[at]
    between = np.ones(len(got), bool)
    between[at.ravel()] = False
    assert np.array_equal(got[between], before[between])
    for i in range(n * tokens):
        if not out[i].any():
            assert not rows[i].any(), i
    assert np.isfinite(rows).all()
    assert rel_l2(rows, out) < check, rel_l2(rows, out)
    # a row by itself too: a wrong row among many shows
    worst = max((rel_l2(rows[i], out[i]) for i in range(n * tokens) if out[i].any()), default=0.0)
    assert worst < 4 * check, worst
    if table is not None:
        assert np.array_equal(weights[~touched], table[~touched])
        if touched.any():
            assert rel_l2(weights[touched], want_w[touched]) < check
            return rows, weights
    return rows


HEADS = [(128, 16, 2), (64, 16, 2), (256, 4, 1), (64, 3, 3), (128, 10, 2), (128, 32, 1), (64, 20, 1)]


@pytest.mark.parametrize("hd,qh,H", HEADS)
@pytest.mark.parametrize("base", [0, 1, 30, 31, 32, 127, 700])
def test_single_token(ctx, hd, qh, H, base):
    side = Side(ctx, (1, 1, H, hd, base + 1 + base % 3), [base + 1], base + hd)
    side.bases = [base]
    side.send()
    attend(side, 0, 1, qh)


@pytest.mark.parametrize("hd,qh,H,tokens,base,context", [
    (128, 16, 2, 2, 100, 110), (64, 16, 2, 7, 0, 7), (128, 4, 4, 16, 31, 60), (256, 8, 1, 5, 64, 70), (128, 16, 2, 33, 0, 64),
    (64, 6, 2, 45, 3, 90), (128, 16, 2, 70, 300, 384), (128, 10, 2, 50, 129, 200), (256, 4, 2, 40, 20, 60),
    (64, 8, 8, 130, 0, 130), (128, 32, 1, 20, 77, 128), (128, 16, 2, 1, 2000, 2048)])
@pytest.mark.parametrize("track", [False, True])
def test_several_tokens_and_prompts(ctx, hd, qh, H, tokens, base, context, track):
    side = Side(ctx, (2, 1, H, hd, context), [min(base + tokens, context)], tokens + hd, track=track)
    side.bases = [base]
    side.send()
    attend(side, 1, tokens, qh, decay=0.5)


@pytest.mark.parametrize("tokens", [1, 3, 24])
@pytest.mark.parametrize("track,hd", [(True, 128), (False, 64), (True, 256)])
def test_ragged_sequences(ctx, tokens, track, hd):
    """Idle sequences and rows whose slot lies past the context are zeros; the sequences outside the call's range are
    neither read nor written."""
    H, context = 2, 260
    filled = [200, 1, 260, 0, 100, 260, 33]
    side = Side(ctx, (1, 7, H, hd, context), filled, tokens)
    if track:
        side = Side(ctx, (1, 7, H, hd, context), filled, tokens, track=True)
    side.bases = [200 - tokens, NO_SLOT, 258, 0, NO_SLOT, 260, max(0, 33 - tokens)]
    side.send()
    for s, b in ((3, 0), (6, side.bases[6])):    # slots that the call's own tokens fill
        for layer_rows, is_v in ((rows_of(side.rng, tokens, H * hd), False), (rows_of(side.rng, tokens, H * hd), True)):
            side.put_rows(0, layer_rows, tokens, is_v, first=s, n=1)
    side.send()
    attend(side, 0, tokens, 8, pad=1, base=3)
    attend(side, 0, tokens, 8, first=2, n=3, decay=0.0)


@pytest.mark.parametrize("track", [False, True])
@pytest.mark.parametrize("hd,qh,H,tokens,bases,context", [
    (128, 16, 2, 790, [0], 800), (64, 16, 2, 800, [37], 830), (128, 6, 2, 521, [70, NO_SLOT, 0, 300], 600),
    (64, 3, 3, 1400, [5, 0, 33], 1440)])
def test_long_prompts(ctx, hd, qh, H, tokens, bases, context, track):
    """Tiles of 64 rows, whose last tokens may lie past the context."""
    filled = [NO_SLOT if b == NO_SLOT else min(b + tokens, context) for b in bases]
    side = Side(ctx, (1, len(bases), H, hd, context), filled, tokens, track=track)
    side.bases = bases
    side.send()
    attend(side, 0, tokens, qh, pad=4, base=4, decay=0.25)


@pytest.mark.parametrize("track,pad", [(False, 0), (True, 0), (True, 1)])
@pytest.mark.parametrize("hd,qh,H,tokens,bases,context", [
    (128, 8, 1, 1, [700], 800), (64, 16, 2, 7, [1200, 3], 1250), (256, 2, 1, 3, [600], 700), (128, 16, 2, 200, [900], 1104),
    (128, 16, 2, 520, [1100], 1650),
    (128, 16, 2, 40, [3000], 3100), (256, 8, 1, 40, [1500], 1600), (64, 16, 2, 18, [2100, 64], 2200),
    (128, 16, 1, 1, [3000], 3001), (64, 6, 2, 4, [2000, 10, NO_SLOT], 2050), (256, 12, 1, 1, [1500], 1600),
    (128, 8, 1, 1, [12000], 12001)])
def test_long_caches(ctx, hd, qh, H, tokens, bases, context, track, pad):
    """Several splits of the slots, joined; weights of many blocks."""
    filled = [NO_SLOT if b == NO_SLOT else b + tokens for b in bases]
    side = Side(ctx, (1, len(bases), H, hd, context), filled, tokens, track=track)
    side.bases = bases
    side.send()
    attend(side, 0, tokens, qh, pad=pad, base=pad, decay=1.0)


@pytest.mark.parametrize("hd,qh,H,tokens,S,context", [
    # tiles of 32 rows of every head size, over one split of the slots and over several
    (256, 16, 1, 100, 1, 1104), (256, 16, 1, 300, 1, 320), (256, 12, 2, 131, 2, 840), (64, 16, 2, 200, 1, 1710),
    (64, 16, 2, 301, 1, 900), (64, 12, 3, 170, 2, 2075), (128, 16, 2, 140, 1, 1000), (128, 16, 2, 150, 1, 1155),
    # weights that need no second launch, because there are many slots or few rows
    (64, 1, 1, 1, 1, 1), (128, 32, 1, 1, 1, 1), (128, 1, 1, 17, 1, 700), (256, 1, 1, 17, 1, 400), (64, 3, 3, 120, 2, 6000),
    (64, 8, 8, 180, 3, 6000), (64, 8, 8, 600, 3, 6000), (128, 8, 8, 120, 2, 1100), (128, 8, 8, 180, 3, 6000),
    (128, 8, 8, 600, 3, 6000), (256, 8, 8, 120, 1, 1100), (256, 8, 8, 120, 3, 400),
    # and with it
    (128, 8, 1, 400, 1, 700), (256, 4, 1, 33, 1, 40)])
def test_kernels_by_size(ctx, hd, qh, H, tokens, S, context):
    """Every kernel that the rules on sizes may choose (test_kv4.py looks that none is missing), with weights and without:
    rows that vx_kv4_store has written, of sequences of unequal length."""
    rng, group = np.random.default_rng(hd + tokens), qh // H
    bases = [max(0, context - tokens - 45 * s) for s in range(S)]
    k, v = rows_of(rng, S, context, H * hd), rows_of(rng, S, context, H * hd)
    q = (rng.standard_normal((S, tokens, H, group, hd)) * 1.2).astype(np.float32)
    old = rng.random((S, H, context)).astype(np.float32)
    outs = []
    for track in (False, True):
        cache, out = Kv4Cache(ctx, 1, S, H, hd, context, track=track), ctx.zeros(q.nbytes)
        cache.store(0, ctx.array(k), ctx.array(v), tokens=context)
        cache.slots.upload(np.array(bases, np.uint32))
        if track:
            cache.weights.upload(old)
        cache.attention(0, ctx.array(q), out, qh, tokens=tokens, decay=0.5)
        outs.append(out.download(np.float32).reshape(q.shape))
    weights = cache.weights.download(np.float32).reshape(old.shape)
    for s, base in enumerate(bases):
        n = base + tokens
        hidden = np.arange(n) > base + np.arange(tokens)[:, None]
        for h in range(H):
            kk, vv = (kv4ref.stored(x[s, :n, h * hd:(h + 1) * hd]) for x in (k, v))
            total = np.where(np.arange(n) < base, 0.5 * old[s, h, :n].astype(np.float64), 0.0)
            for g in range(group):
                x = q[s, :, h, g].astype(np.float64) @ kk.T / np.sqrt(hd)
                x[hidden] = -np.inf
                p = np.exp(x - x.max(-1, keepdims=True))
                p /= p.sum(-1, keepdims=True)
                want = p @ vv
                for out in outs:
                    off = np.linalg.norm(out[s, :, h, g] - want, axis=-1) / np.linalg.norm(want, axis=-1)
                    assert off.max() < 4 * TOL, (s, h, g, off.argmax())
                    assert rel_l2(out[s, :, h, g], want) < TOL
                total += p.sum(0)
            assert rel_l2(weights[s, h, :n], total) < TOL, (s, h)
            assert np.array_equal(weights[s, h, n:], old[s, h, n:])


@pytest.mark.parametrize("track", [False, True])
@pytest.mark.parametrize("hd,qh,H,tokens,S,context", [
    (128, 8, 1, 1, 1, 512), (128, 8, 1, 1, 1, 513), (64, 24, 2, 1, 3, 4000), (128, 16, 2, 3, 2, 1500), (256, 5, 1, 17, 1, 700),
    (128, 16, 2, 9, 1, 900), (128, 16, 2, 130, 2, 2100), (64, 3, 3, 1300, 3, 1400), (128, 16, 2, 530, 1, 1600)])
def test_scratch_is_kept_to(ctx, hd, qh, H, tokens, S, context, track):
    """Nothing behind the bytes asked for is written, and what the scratch holds before a call does not matter."""
    cache = Kv4Cache(ctx, 1, S, H, hd, context, track=track)
    rng = np.random.default_rng(tokens)
    k = ctx.array(rows_of(rng, S * context, H * hd))
    cache.store(0, k, k, tokens=context)
    cache.slots.upload(np.array([context - tokens, 0, NO_SLOT][:S], np.uint32))
    pc = abi.Kv4AttentionPush(cache.geom, 0, 0, S, tokens, qh, qh * hd, qh * hd, 0, 0, 0.0)
    n = abi.load().vx_kv4_attention_scratch_bytes(pc, int(track)) // 4
    q, got = ctx.array(rng.standard_normal((S * tokens, qh * hd)).astype(np.float32)), []
    for fill in (0, 0x7FC00000):
        scratch = ctx.array(np.full(n + 4096, fill, np.uint32))
        out = ctx.zeros(S * tokens * qh * hd * 4)
        cache.attention(0, q, out, qh, tokens=tokens, decay=0.0, scratch=scratch)
        assert (scratch.download(np.uint32)[n:] == fill).all()
        got.append(out.download(np.float32))
        if track:
            got[-1] = np.concatenate([got[-1], cache.weights.download(np.float32)])
    assert np.isfinite(got[0]).all() and np.array_equal(got[0], got[1])


def test_graphs_that_share_a_scratch(ctx):
    """Two captured calls of one cache, replayed in turn and in either order, and a larger eager call in between whose
    scratch outgrows theirs."""
    hd, H, qh, context = 128, 2, 16, 2048
    side = Side(ctx, (1, 2, H, hd, context), [1990, 700], 8, track=True)
    tokens = (1, 5)
    qs = [ctx.array(side.rng.standard_normal((2 * t, qh * hd)).astype(np.float32)) for t in tokens]
    outs = [ctx.zeros(2 * t * qh * hd * 4) for t in tokens]
    side.bases = [1980, 650]
    side.send()
    calls = [lambda i=i: side.dev.attention(0, qs[i], outs[i], qh, tokens=tokens[i], decay=0.0) for i in range(2)]
    want = []
    for i in (1, 0):
        calls[i]()
    want = [o.download(np.float32) for o in outs]
    graphs = []
    for call in calls:
        ctx.graph_begin()
        call()
        graphs.append(ctx.graph_end())
    big = ctx.zeros(2 * 40 * qh * hd * 4)
    for turn in ((0, 1), (1, 0), (0, 0, 1, 1)):
        for o in outs:
            o.upload(np.zeros(o.nbytes // 4, np.float32))
        for i in turn:
            ctx.graph_launch(graphs[i])
        ctx.sync()
        for o, x in zip(outs, want):
            assert np.array_equal(o.download(np.float32), x)
        side.dev.attention(0, ctx.zeros(2 * 40 * qh * hd * 4), big, qh, tokens=40)
    for g in graphs:
        ctx.graph_free(g)


def test_unused_slots_do_not_matter(ctx):
    """Not a bit of a row depends on what lies behind its last slot, infinities and NaN in d and o among it."""
    outs = []
    for fill in (0x00000000, 0x7C007C00, 0x7E00FE00, 0xFFFFFFFF):
        side = Side(ctx, (1, 1, 2, 128, 96), [70], 5)
        for cache, is_v in ((side.k, False), (side.v, True)):
            for h in range(2):
                kept = [a.copy() for a in kv4ref.get(cache, (0, 0, h), 70, is_v)]
                cache[0, 0, h] = fill
                for j in range(70):
                    kv4ref.put(cache, (0, 0, h), j, *(a[j] for a in kept), is_v)
        side.bases = [69]
        side.send()
        side.rng = np.random.default_rng(9)
        outs.append(attend(side, 0, 1, 16))
    for o in outs[1:]:
        assert np.array_equal(o, outs[0])


@pytest.mark.parametrize("scale", [1e-30, 1e-4, 30.0, 1e4])
def test_queries_of_any_size(ctx, scale):
    """From weights that are all but equal to ones where one slot takes all. A score |s| of a large q is off by 2^-24 |s|
    sqrt(256), which moves the weights of near ties: with 1e4 only the largest score weighs, and rows where the two
    largest differ by less than 0.1 are left out by making none (seeded)."""
    side = Side(ctx, (1, 1, 2, 128, 512), [401], 21)
    side.bases = [400]
    side.send()
    # 30: |s| to 30 * 1.2 * 2 * sqrt(128) / 2 ~ 400, off by 400 * 16 * 6e-8 = 4e-4 at worst; 1e4 by 0.13
    tol = {30.0: 4e-4}.get(scale, TOL)
    if scale == 1e4:
        rng = np.random.default_rng(2)
        k = kv4ref.rows(side.k, (0, 0, 0), 401, False)
        q = np.zeros((1, 16 * 128), np.float32)
        for h in range(16):
            k = kv4ref.rows(side.k, (0, 0, h // 8), 401, False)
            q[0, h * 128:(h + 1) * 128] = 1e4 * (k[37 * h % 400] - k.mean(0) * 0.5 + 0.01 * rng.standard_normal(128))
        ob = ctx.zeros(q.nbytes)
        side.dev.attention(0, ctx.array(q), ob, 16)
        want, _ = kv4ref.attention(q.reshape(1, 2, 8, 128), side.k, side.v, 0, 0, 400, 512)
        assert rel_l2(ob.download(np.float32), want) < TOL
        return
    attend(side, 0, 1, 16, q_scale=1.2 * scale, check=tol)


@pytest.mark.parametrize("hd,qh,H,tokens,context", [(128, 16, 2, 1, 512), (64, 16, 2, 2, 700), (256, 4, 1, 1, 90), (128, 16, 2, 60, 1400),
                                                    (128, 8, 1, 800, 1600)])
@pytest.mark.parametrize("scale", [1e6, 1e8, 1e10, 1e20, 1e30])
def test_queries_whose_scores_pass_f32s_integers(ctx, hd, qh, H, tokens, context, scale):
    """Rows that point at one slot's K with scores of up to 2^117: it takes all the weight, and the row is its V. The
    scores are off by 2^-24 sqrt(512) of their size, and the two largest differ by a tenth and more. (The weights
    p <= 1 go in as two f16 terms, f16(p) being exact here; the row is then exact but for the reciprocal, 2^-24 twice.)"""
    side = Side(ctx, (1, 1, H, hd, context), [context], 3)
    base, group = context - tokens, qh // H
    side.bases = [base]
    side.send()
    q = np.zeros((tokens, H, group, hd), np.float32)
    want = np.zeros(q.shape)
    for h in range(H):
        k, v = (kv4ref.rows(c, (0, 0, h), context, is_v) for c, is_v in ((side.k, False), (side.v, True)))
        at = np.argsort(-(k ** 2).sum(-1))      # the longest first, so that nothing lies further along them
        for t in range(tokens):
            seen = at[at <= base + t]
            for g in range(group):
                x = (k[seen[(g + t) % 4]] - k.mean(0)).astype(np.float32)
                s = k[:base + t + 1] @ x
                second, most = np.sort(s)[-2:]
                assert most - second > 0.1 * most
                q[t, h, g] = x * np.float32(scale)
                want[t, h, g] = v[np.argmax(s)]
    out = ctx.zeros(q.nbytes)
    side.dev.attention(0, ctx.array(q.reshape(tokens, -1)), out, qh, tokens=tokens)
    assert rel_l2(out.download(np.float32).reshape(q.shape), want) < 2.0 ** -22


@pytest.mark.parametrize("hd,qh,H,base,tokens", [(128, 16, 2, 500, 1), (128, 24, 2, 500, 1), (64, 16, 2, 1200, 3), (256, 4, 1, 90, 1),
                                                 (128, 16, 2, 1400, 60), (128, 8, 1, 900, 800), (256, 8, 1, 2000, 100)])
@pytest.mark.parametrize("scale", [30.0, 1e3, 1e5, 1e8, 1e12, 1e30])
def test_weights_of_large_scores_add_up_to_the_rows(ctx, hd, qh, H, base, tokens, scale):
    """Scores that are off by 2^-24 of their size, so by more than a weight allows: the weights have to come from the very
    scores that the rows' sums were made of. Allowed is what test_weights_are_not_off_to_one_side allows, and per row the
    difference of two references and of a score and one, each rounded to 2^-24 of itself where scores are small beside
    them: exact otherwise."""
    context, r = base + tokens, tokens * qh // H
    side = Side(ctx, (1, 1, H, hd, context), [context], base + hd, track=True)
    side.bases = [base]
    side.send()
    q = (side.rng.standard_normal((tokens, qh * hd)) * scale).astype(np.float32)
    side.dev.attention(0, ctx.array(q), ctx.zeros(q.nbytes), qh, tokens=tokens, decay=0.0)
    got = side.dev.weights.download(np.float32).reshape(H, context).astype(np.float64)
    assert got.min() >= 0 and got.max() <= r * (1 + 1e-6)
    assert abs(got.sum(-1) / r - 1).max() < 2 * (3.7e-7 / r ** 0.5 + 2.0 ** -24)


def test_large_and_small_weights_of_one_row(ctx):
    """One slot with nearly all the weight, thousands with 2^-14 of it each and values that add up."""
    side = Side(ctx, (1, 1, 1, 64, 4096), [0], 8, track=True)
    k = np.zeros((4001, 64), np.float32)
    k[:, 0], k[1234, 0] = -1.0, 1.0
    v = (np.abs(side.rng.standard_normal((4001, 64))) + 0.5).astype(np.float32)
    for h, (x, cache, is_v) in enumerate(((k, side.k, False), (v, side.v, True))):
        side.put_rows(0, x, 4001, is_v)
    side.bases = [4000]
    side.send()
    q = np.zeros((1, 64), np.float32)
    q[0, 0] = 14 * np.log(2) * 4        # scores +-4.85: 2^-14 of the largest weight, then 2^-1.75
    for top in (q, q / 8):
        ob = side.ctx.zeros(256)
        side.dev.attention(0, ctx.array(top), ob, 1, decay=0.0)
        want, w = kv4ref.attention(top.reshape(1, 1, 1, 64), side.k, side.v, 0, 0, 4000, 4096)
        assert rel_l2(ob.download(np.float32), want) < TOL
        assert rel_l2(side.dev.weights.download(np.float32)[:4001], w) < TOL


@pytest.mark.parametrize("hd,qh,H,base,tokens", [(128, 16, 2, 2000, 1), (128, 16, 2, 2000, 2), (64, 16, 2, 3000, 1), (256, 4, 1, 700, 3),
                                                 (128, 16, 2, 1500, 200), (64, 6, 2, 1200, 130), (256, 4, 1, 500, 120),
                                                 (128, 8, 1, 0, 300), (128, 2, 2, 40, 1)])
def test_weights_are_not_off_to_one_side(ctx, hd, qh, H, base, tokens):
    """Rows that weigh all slots about alike (|s| < 0.1, so that scores are exact to 1e-8). The sum of all weights has to
    be the number of rows: a weight is v / l with the v that l is the sum of, so what errs to one side cancels. A row is
    off by its reciprocal (2^-24 = 6e-8), by the additions of l, of which a lane makes n <= 380 (0.4 2^-24 sqrt(n / 3) in
    the mean square, over 16 lanes or more: 7e-8), and by the exponentials that take a wave's and a split's sum to the
    row's reference (2^-23 = 1.2e-7 each): 3.7e-7, of either sign, so over r rows by r^1/2 less. The additions over rows
    may all round one way: 2^-24. A single weight is off by the rounding of its exponent, which lies near 7 (2^-22 ln 2 =
    1.65e-7, as 4..8 has steps of 2^-21), and its exponential (2^-23), both once more in l, by the row's 3.7e-7 and
    a product (2^-24): 1e-6 at the very most."""
    context = base + tokens
    side = Side(ctx, (1, 1, H, hd, context), [context], base + hd, track=True)
    side.bases = [base]
    side.send()
    side.dev.weights.upload(np.full(H * context, 7.0, np.float32))
    q = (side.rng.standard_normal((tokens, qh * hd)) * 0.005).astype(np.float32)
    side.dev.attention(0, ctx.array(q), ctx.zeros(q.nbytes), qh, tokens=tokens, decay=0.0)
    got = side.dev.weights.download(np.float32).reshape(H, context).astype(np.float64)
    _, want = kv4ref.attention(q.reshape(tokens, H, qh // H, hd), side.k, side.v, 0, 0, base, context)
    assert rel_l2(got, want) < 1e-6
    assert abs(got.sum(-1) / (tokens * qh // H) - 1).max() < 3.7e-7 / (tokens * qh // H) ** 0.5 + 2.0 ** -24


def test_a_nan_row_is_nan_and_others_are_not(ctx):
    side = Side(ctx, (1, 2, 1, 128, 64), [20, 20], 5)
    side.bases = [19, 19]
    side.send()
    q = side.rng.standard_normal((2, 4 * 128)).astype(np.float32)
    q[0, 130] = np.nan
    ob = ctx.zeros(q.nbytes)
    side.dev.attention(0, ctx.array(q), ob, 4)
    got = ob.download(np.float32).reshape(2, 4, 128)
    assert np.isnan(got[0, 1]).all() and np.isfinite(got[0, [0, 2, 3]]).all() and np.isfinite(got[1]).all()


@pytest.mark.parametrize("hd,qh,H,tokens,base", [(128, 16, 2, 1, 40), (128, 16, 2, 2, 40), (128, 16, 2, 12, 40),
                                                (64, 4, 2, 30, 0), (256, 2, 1, 30, 9), (128, 16, 2, 1600, 0)])
def test_a_stored_nan_reaches_the_rows_that_attend_to_it(ctx, hd, qh, H, tokens, base):
    """V of one group of a slot in the call's midst, and K of another slot: earlier rows keep their bits, rows that
    attend to the V have NaN in that group's dimensions alone, rows that attend to the K are NaN."""
    context, group = base + tokens + 5, qh // H
    rng = np.random.default_rng(5)
    cache = Kv4Cache(ctx, 1, 1, H, hd, context)
    k, v = rows_of(rng, base + tokens, H * hd), rows_of(rng, base + tokens, H * hd)
    q, out = ctx.array(rng.standard_normal((tokens, qh * hd)).astype(np.float32)), ctx.zeros(tokens * qh * hd * 4)
    got = []
    at_v, at_k = base + tokens // 2, base + (3 * tokens) // 4
    for bad in (False, True):
        if bad:
            v[at_v, hd * (H - 1) + 35] = np.nan
            if tokens > 1:
                k[at_k, 1] = np.nan      # KV head 0
        cache.slots.upload(np.array([0], np.uint32))
        cache.store(0, ctx.array(k), ctx.array(v), tokens=base + tokens)
        cache.slots.upload(np.array([base], np.uint32))
        cache.attention(0, q, out, qh, tokens=tokens)
        got.append(out.download(np.float32).reshape(tokens, H, group, hd))
    clean, dirty = got
    assert np.isfinite(clean).all()
    want = np.zeros(clean.shape, bool)
    want[at_v - base:, H - 1, :, 32:64] = True
    if tokens > 1:
        want[at_k - base:, 0] = True
    assert np.array_equal(np.isnan(dirty), want)
    assert np.array_equal(dirty[~want], clean[~want])


@pytest.mark.parametrize("hd,qh,H", [(128, 16, 2), (64, 4, 2), (256, 4, 1)])
@pytest.mark.parametrize("tokens", [3, 6, 30, 300])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, 3e38])
def test_weights_of_rows_that_take_no_part_are_left_out(ctx, hd, qh, H, tokens, bad):
    """Rows past the context hold anything: not a bit of the others' rows and weights depends on them."""
    base, got = 50 + tokens // 2, []
    context = base + (tokens + 1) // 2
    rng = np.random.default_rng(8)
    cache = Kv4Cache(ctx, 1, 1, H, hd, context, track=True)
    k = ctx.array(rows_of(rng, context, H * hd))
    cache.store(0, k, k, tokens=context)
    cache.slots.upload(np.array([base], np.uint32))
    q = rng.standard_normal((tokens, qh * hd)).astype(np.float32)
    old = rng.random((H, context)).astype(np.float32)
    for fill in (0.0, bad):
        q[context - base:] = fill
        out = ctx.zeros(q.nbytes)
        cache.weights.upload(old)
        cache.attention(0, ctx.array(q), out, qh, tokens=tokens, decay=0.5)
        got.append(np.concatenate([out.download(np.float32), cache.weights.download(np.float32)]))
    assert np.isfinite(got[0]).all() and np.array_equal(got[1], got[0])


@pytest.mark.parametrize("hd,qh,H", [(128, 16, 2), (64, 4, 2), (256, 4, 1)])
@pytest.mark.parametrize("tokens", [3, 6, 30, 300])
@pytest.mark.parametrize("where", ["q", "k"])
def test_weights_of_a_nan_row_end_at_its_last_slot(ctx, hd, qh, H, tokens, where):
    """A row with a NaN in q, or in a K that it attends to, makes NaN of the weights of the slots that it attends to. The
    slots of later tokens have what the rows that attend to them give: bit for bit, with the NaN in q."""
    base, at, got = 70, tokens // 2, []
    rng = np.random.default_rng(9)
    cache = Kv4Cache(ctx, 1, 1, H, hd, base + tokens, track=True)
    k, v = rows_of(rng, base + tokens, H * hd), ctx.array(rows_of(rng, base + tokens, H * hd))
    q = rng.standard_normal((tokens, qh * hd)).astype(np.float32)
    for bad in (False, True):
        if bad and where == "q":
            q[at, hd * (qh - 1) + 3] = np.nan      # the last KV head's
        elif bad:
            k[base + at, H * hd - 1] = np.nan
        cache.slots.upload(np.array([0], np.uint32))
        cache.store(0, ctx.array(k), v, tokens=base + tokens)
        cache.slots.upload(np.array([base], np.uint32))
        cache.weights.upload(np.ones((H, base + tokens), np.float32))
        cache.attention(0, ctx.array(q), ctx.zeros(q.nbytes), qh, tokens=tokens, decay=0.5)
        got.append(cache.weights.download(np.float32).reshape(H, -1))
    want = np.zeros(got[0].shape, bool)
    # every row from token `at` on attends to the slot of the K, and so has NaN for all that it attends to
    want[H - 1, :base + at + 1 if where == "q" else None] = True
    assert np.isfinite(got[0]).all()
    assert np.array_equal(np.isnan(got[1]), want)
    assert np.array_equal(got[1][~want], got[0][~want])


# ----------------------------------------------------------------- eviction
def tables(rng, geom, bases, ties=True):
    L, S, H, hd, context = geom
    w = (rng.random((L, S, H, context)) ** 6 * 40).astype(np.float32)
    if ties:
        w = np.where(rng.random(w.shape) < 0.5, np.floor(w * 4) / 4, w).astype(np.float32)
    at = np.argsort(rng.random((L, S, H, 2 * context)), -1)[..., :context].astype(np.uint32)
    return w, at


@pytest.mark.parametrize("L,bases,H,context,keep,sinks,recent", [
    (1, [40], 1, 64, 20, 0, 0), (2, [64, 33, NO_SLOT, 7, 20], 2, 64, 20, 2, 5), (3, [1500], 2, 1500, 700, 4, 64),
    (1, [2049, 3001], 3, 3001, 2048, 4, 256), (1, [100], 1, 101, 100, 3, 3), (1, [101], 2, 101, 100, 3, 97),
    (1, [9], 1, 9, 1, 1, 0), (1, [5000], 1, 5001, 5000, 0, 0), (2, [1024, 1025], 1, 1100, 1023, 0, 1023),
    (1, [20000, 16385], 1, 20001, 15000, 4, 64), (1, [16384, 16000], 1, 16384, 8192, 4, 64)])
def test_select_and_compact_are_exact(ctx, L, bases, H, context, keep, sinks, recent):
    hd = 64
    geom = (L, len(bases), H, hd, context)
    side = Side(ctx, geom, [0] * len(bases), 31, track=True)      # any bits serve as rows
    side.bases = list(bases)
    side.send()
    w, at = tables(side.rng, geom, bases)
    w[..., ::17] = 0.0
    w[0, 0, 0, :min(9, context):3] = np.nan
    w[0, 0, 0, 1] = -0.0
    side.dev.weights.upload(w)
    side.dev.slot_positions.upload(at)
    plan, moves = side.dev.plan(keep), side.dev.plan_moves(keep)
    side.dev.select(plan, keep, sinks, recent)
    got = plan.download(np.uint32, L * len(bases) * H * moves * 2).reshape(L, len(bases), H, moves, 2)
    for i in np.ndindex(L, len(bases), H):
        n = 0 if bases[i[1]] == NO_SLOT else min(bases[i[1]], context)
        want = kv4ref.select(w[i], at[i], n, keep, sinks, recent)
        full = np.full((moves, 2), NO_SLOT, np.uint32)
        full[:len(want)] = np.array(want, np.uint32).reshape(-1, 2)
        assert np.array_equal(got[i], full), i
        kv4ref.move(side.k, i, want, False)
        kv4ref.move(side.v, i, want, True)
        for f, t in want:
            w[i][t], at[i][t] = w[i][f], at[i][f]
    for again in range(2):      # a plan carried out twice moves the same rows to the same places
        side.dev.compact(plan, keep)
        side.check_bytes()
        assert np.array_equal(side.dev.weights.download(np.uint32).reshape(w.shape), w.view(np.uint32))
        assert np.array_equal(side.dev.slot_positions.download(np.uint32).reshape(at.shape), at)
        assert list(side.dev.filled()) == [b if b == NO_SLOT else min(b, keep) for b in bases]


@pytest.mark.parametrize("hd", [128, 256])
def test_compact_of_wide_heads_and_some_sequences(ctx, hd):
    geom, bases, keep = (2, 3, 2, hd, 90), [90, 80, 88], 41
    side = Side(ctx, geom, [0, 0, 0], 7, track=True)
    side.bases = bases
    side.send()
    w, at = tables(side.rng, geom, bases)
    side.dev.weights.upload(w)
    side.dev.slot_positions.upload(at)
    plan = side.dev.plan(keep, n=2)
    side.dev.evict(plan, keep, 1, 2, first=1, n=2)
    for i in np.ndindex(2, 3, 2):
        if i[1]:
            moves = kv4ref.select(w[i], at[i], bases[i[1]], keep, 1, 2)
            kv4ref.move(side.k, i, moves, False)
            kv4ref.move(side.v, i, moves, True)
    side.check_bytes()
    assert list(side.dev.filled()) == [90, 41, 41]


def test_a_plan_that_is_not_one_moves_nothing_out_of_place(ctx):
    """Pairs outside [keep, context) -> [0, keep) are not carried out."""
    geom, keep = (1, 1, 1, 128, 50), 20
    side = Side(ctx, geom, [0], 2, track=True)
    side.bases = [50]
    side.send()
    w, at = tables(side.rng, geom, [50])
    side.dev.weights.upload(w)
    side.dev.slot_positions.upload(at)
    pairs = [(30, 3), (50, 4), (19, 5), (31, 20), (NO_SLOT, 6), (32, NO_SLOT), (49, 7), (1 << 31, 8)]
    plan = np.full((20, 2), NO_SLOT, np.uint32)
    plan[:len(pairs)] = pairs
    side.dev.compact(ctx.array(plan), keep)
    for is_v, cache in ((False, side.k), (True, side.v)):
        kv4ref.move(cache, (0, 0, 0), [(30, 3), (49, 7)], is_v)
    side.check_bytes()
    w[0, 0, 0, 3], w[0, 0, 0, 7] = w[0, 0, 0, 30], w[0, 0, 0, 49]
    assert np.array_equal(side.dev.weights.download(np.float32).reshape(w.shape), w)


# ----------------------------------------------------------------- together
class Mirror:
    """A cache that goes through the same steps in 64 bits."""

    def __init__(self, geom, sequences):
        self.geom = geom
        rng = np.random.default_rng(0)
        L, S, H, hd, context = geom
        self.k, self.v = (kv4ref.blank(L, S, H, hd, context, rng) for _ in range(2))
        self.slots, self.pos = list(sequences), [0] * S
        self.w = np.zeros((L, S, H, context))
        self.at = np.zeros((L, S, H, context), np.uint32)

    def step(self, layer, k, v, q, tokens, group, decay):
        L, S, H, hd, context = self.geom
        out = np.zeros(q.shape)
        for s in range(S):
            b = self.slots[s]
            if b == NO_SLOT:
                continue
            for t in range(tokens):
                for h in range(H):
                    for cache, x, is_v in ((self.k, k, False), (self.v, v, True)):
                        c, d, o = kv4ref.encode(x[s * tokens + t, h * hd:(h + 1) * hd])
                        kv4ref.put(cache, (layer, s, h), b + t, c, d, o, is_v)
                    self.at[layer, s, h, b + t] = self.pos[s] + t
            x = q[s * tokens:(s + 1) * tokens].reshape(tokens, H, group, hd)
            o, w = kv4ref.attention(x, self.k, self.v, layer, s, b, context)
            out[s * tokens:(s + 1) * tokens] = o.reshape(tokens, -1)
            m = w.shape[1]
            self.w[layer, s, :, :m] = np.where(np.arange(m) < b, decay * self.w[layer, s, :, :m], 0) + w
        return out

    def advance(self, tokens):
        for s, b in enumerate(self.slots):
            if b != NO_SLOT:
                self.slots[s] += tokens
                self.pos[s] += tokens

    def evict(self, keep, sinks, recent, weights):
        """By the device's weights, whose last bits a selection may hang on."""
        for i in np.ndindex(*self.w.shape[:3]):
            b = self.slots[i[1]]
            moves = [] if b == NO_SLOT else kv4ref.select(weights[i], self.at[i], b, keep, sinks, recent)
            kv4ref.move(self.k, i, moves, False)
            kv4ref.move(self.v, i, moves, True)
            for f, t in moves:
                self.w[i][t], self.at[i][t] = self.w[i][f], self.at[i][f]
        self.slots = [b if b == NO_SLOT else min(b, keep) for b in self.slots]


def test_prompt_steps_and_evictions_together(ctx):
    """A prompt, then captured steps that store, attend in two layers and advance, with an eviction (a graph of its own)
    whenever the slots run out: every step's rows, weights and slots follow the restatement, and the program's own eager
    work and waits come between the replays."""
    L, S, H, hd, context, qh, keep = 2, 3, 2, 128, 72, 8, 50
    geom, group, decay = (L, S, H, hd, context), qh // H, 0.9
    rng = np.random.default_rng(77)
    cache, mirror = Kv4Cache(ctx, *geom, track=True), Mirror((L, S, H, hd, context), [0, NO_SLOT, 0])
    cache.slots.upload(np.array([0, NO_SLOT, 0], np.uint32))
    cache.k.upload(mirror.k)
    cache.v.upload(mirror.v)
    tokens = 41

    def fresh(n):
        return rows_of(rng, S * n, H * hd), rows_of(rng, S * n, H * hd), rng.standard_normal((S * n, qh * hd)).astype(np.float32)

    def check(got, want):
        assert np.array_equal(got[want.any(-1) == 0], want[want.any(-1) == 0])
        assert rel_l2(got, want) < TOL
        w = cache.weights.download(np.float32).reshape(L, S, H, context)
        for s, b in enumerate(mirror.slots):
            if b != NO_SLOT:
                assert rel_l2(w[:, s, :, :b], mirror.w[:, s, :, :b]) < TOL
        return w

    for layer in range(L):
        k, v, q = fresh(tokens)
        out = ctx.zeros(q.nbytes)
        kb, vb, qb = ctx.array(k), ctx.array(v), ctx.array(q)
        cache.store(layer, kb, vb, tokens=tokens)
        cache.attention(layer, qb, out, qh, tokens=tokens, decay=decay)
        want = mirror.step(layer, k, v, q, tokens, group, decay)
        assert rel_l2(out.download(np.float32).reshape(want.shape), want) < TOL
    cache.advance(tokens)
    mirror.advance(tokens)

    bufs = [[ctx.zeros(x.nbytes) for x in fresh(1)] + [ctx.zeros(S * qh * hd * 4)] for _ in range(L)]
    plan = cache.plan(keep)

    def step():
        for layer, (kb, vb, qb, ob) in enumerate(bufs):
            cache.store(layer, kb, vb)
            cache.attention(layer, qb, ob, qh, decay=decay)
        cache.advance()

    def evict():
        cache.evict(plan, keep, sinks=2, recent=8)

    # one eager step on copies of the state, so that what a capture must not allocate is there
    saved = [b.download(np.uint32) for b in (cache.k, cache.v, cache.slots, cache.positions, cache.weights, cache.slot_positions)]
    step()
    evict()
    for b, x in zip((cache.k, cache.v, cache.slots, cache.positions, cache.weights, cache.slot_positions), saved):
        b.upload(x)
    graphs = []
    for body in (step, evict):
        ctx.graph_begin()
        body()
        graphs.append(ctx.graph_end())
    evictions = 0
    for i in range(70):
        host = [fresh(1) for _ in range(L)]
        for layer, (k, v, q) in enumerate(host):
            for b, x in zip(bufs[layer], (k, v, q)):
                b.upload(x)
        ctx.graph_launch(graphs[0])
        wants = [mirror.step(layer, k, v, q, 1, group, decay) for layer, (k, v, q) in enumerate(host)]
        mirror.advance(1)
        ctx.sync()
        for layer in range(L):
            w = check(bufs[layer][3].download(np.float32).reshape(wants[layer].shape), wants[layer])
        assert list(cache.filled()) == mirror.slots
        if max(b for b in mirror.slots if b != NO_SLOT) == context:
            ctx.graph_launch(graphs[1])
            mirror.evict(keep, 2, 8, w)
            ctx.sync()
            evictions += 1
            assert list(cache.filled()) == mirror.slots
            got = cache.slot_positions.download(np.uint32).reshape(mirror.at.shape)
            assert np.array_equal(got[:, 0, :, :keep], mirror.at[:, 0, :, :keep])
            assert np.array_equal(got[:, 2, :, :keep], mirror.at[:, 2, :, :keep])
            mirror.w[:] = cache.weights.download(np.float32).reshape(mirror.w.shape)
    for g in graphs:
        ctx.graph_free(g)
    assert evictions == 2
    for s in (0, 2):
        for layer in range(L):
            for h in range(H):
                at = mirror.at[layer, s, h, :mirror.slots[s]]
                assert len(set(at)) == len(at) and {0, 1} <= set(at) and set(range(103, 111)) <= set(at)


def test_offsets_beyond_4_gib(ctx):
    """The last plane of caches of 5.4 GB each."""
    L, S, H, hd, context = 64, 8, 8, 128, 16416
    cache = Kv4Cache(ctx, L, S, H, hd, context)
    assert cache.k.nbytes > 1 << 32
    rng = np.random.default_rng(6)
    slots = np.full(S, NO_SLOT, np.uint32)
    slots[-1] = 16380
    cache.slots.upload(slots)
    tokens = 36
    k, v = rows_of(rng, tokens, H * hd), rows_of(rng, tokens, H * hd)
    cache.store(L - 1, ctx.array(k), ctx.array(v), tokens=tokens, first=S - 1)
    kb, vb = ctx.zeros(k.nbytes), ctx.zeros(v.nbytes)
    cache.load(L - 1, kb, vb, tokens=tokens, first=S - 1)
    for b, x in ((kb, k), (vb, v)):
        assert np.array_equal(b.download(np.float32).reshape(tokens, H, hd), kv4ref.stored(x.reshape(tokens, H, hd)))
    # attention over the whole of it: the slots below 16380 all alike
    same = rows_of(rng, 1, H * hd)
    slots[-1] = 0
    cache.slots.upload(slots)
    cache.store(L - 1, ctx.array(np.repeat(same, 16380, 0)), ctx.array(np.repeat(same, 16380, 0)), tokens=16380, first=S - 1)
    slots[-1] = 16380
    cache.slots.upload(slots)
    q = rng.standard_normal((tokens, H * hd)).astype(np.float32)
    out = ctx.zeros(q.nbytes)
    cache.attention(L - 1, ctx.array(q), out, H, tokens=tokens, first=S - 1)
    got = out.download(np.float32).reshape(tokens, H, hd)
    for h in range(H):
        one = kv4ref.stored(same.reshape(H, hd))[h]
        keys = np.concatenate([np.repeat(one[None], 16380, 0), kv4ref.stored(k.reshape(tokens, H, hd))[:, h]])
        vals = np.concatenate([np.repeat(one[None], 16380, 0), kv4ref.stored(v.reshape(tokens, H, hd))[:, h]])
        for t in (0, 17, tokens - 1):
            s = q.reshape(tokens, H, hd)[t, h].astype(np.float64) @ keys[:16381 + t].T / np.sqrt(hd)
            p = np.exp(s - s.max())
            assert rel_l2(got[t, h], p @ vals[:16381 + t] / p.sum()) < TOL


def test_two_contexts_with_scratch_of_their_own(ctx):
    """Calls that overlap on two streams, each with its cache's scratch, give what they give alone."""
    with Context(ctx.device) as other:
        sides = [Side(c, (1, 2, 2, 128, 2048), [2000, 900], 3 + i, track=True) for i, c in enumerate((ctx, other))]
        q = [c.ctx.array(c.rng.standard_normal((2, 16 * 128)).astype(np.float32)) for c in sides]
        outs = [[c.ctx.zeros(2 * 16 * 128 * 4) for _ in range(21)] for c in sides]
        for i, c in enumerate(sides):
            c.bases = [1999, 899]
            c.send()
            c.dev.attention(0, q[i], outs[i][20], 16, decay=0.0)
            c.ctx.sync()
        for j in range(20):
            for i, c in enumerate(sides):
                c.dev.attention(0, q[i], outs[i][j], 16, decay=0.0)
        for i, c in enumerate(sides):
            alone = outs[i][20].download(np.float32)
            for j in range(20):
                assert np.array_equal(outs[i][j].download(np.float32), alone)
        for x in q + outs[0] + outs[1]:
            x.free()
        for c in sides:
            for b in (c.dev.k, c.dev.v, c.dev.slots, c.dev.positions, c.dev.weights, c.dev.slot_positions, c.dev._scratch):
                b.free()
