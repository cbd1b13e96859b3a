"""The 4-bit KV cache restated with numpy in 64 bits, from the format's and the
operators' definitions (include/voxhip.h, vx_kv4_*): what the kernels are tested against.

A cache here is the bytes of one vx_buf as uint32 [layers, sequences, kv_heads, blocks,
5 * head_dim]; rows are [..., head_dim]."""
import numpy as np

NO_SLOT = 0xFFFFFFFF
LIMIT = np.float32(61440)
BIT = [4 * (e // 2) + 16 * (e % 2) for e in range(8)]


def encode(x):
    """Codes [..., head_dim] uint32, step and offset [..., groups] float16."""
    g = np.asarray(x, np.float32).reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    bad = np.isnan(g).any(-1)
    g = np.clip(np.where(np.isnan(g), np.float32(0), g), -LIMIT, LIMIT)
    lo, hi = g.min(-1), g.max(-1)
    d = ((hi - lo) / np.float32(15)).astype(np.float16)
    o = lo.astype(np.float16)
    df, of = d.astype(np.float32)[..., None], o.astype(np.float32)[..., None]
    with np.errstate(all="ignore"):
        c = np.where(df > 0, np.clip(np.rint((g - of) / df), 0, 15), 0)
    c = np.where(bad[..., None], 0, c).astype(np.uint32)
    return c.reshape(x.shape), np.where(bad, np.float16(0), d), np.where(bad, np.float16(np.nan), o)


def values(c, d, o):
    """float64 values, each an f16: the sum in 64 bits is exact, the conversion rounds once."""
    g = c.reshape(*c.shape[:-1], c.shape[-1] // 32, 32).astype(np.float64)
    with np.errstate(all="ignore"):
        v = (o.astype(np.float64)[..., None] + d.astype(np.float64)[..., None] * g).astype(np.float16)
    return v.astype(np.float64).reshape(c.shape)


def stored(x):
    """What rows stand for once they are stored."""
    return values(*encode(x))


def blank(layers, sequences, kv_heads, head_dim, context, rng):
    """A cache of random bits: what unused slots may hold."""
    return rng.integers(0, 1 << 32, (layers, sequences, kv_heads, (context + 31) // 32, 5 * head_dim), dtype=np.uint32)


def put(cache, plane, slot, c, d, o, is_v):
    """One slot's codes [head_dim], step and offset [groups] into plane (layer, sequence, head)."""
    hd = cache.shape[-1] // 5
    groups = hd // 32
    b = cache[plane][slot // 32]
    s = slot % 32
    halves = b[4 * hd:].view(np.float16)
    if not is_v:
        b[s * hd // 8:(s + 1) * hd // 8] = sum(c.reshape(-1, 8)[:, e] << np.uint32(BIT[e]) for e in range(8))
        halves[s * groups * 2:(s + 1) * groups * 2] = np.stack([d, o], -1).ravel()
        return
    octet, e = s // 8, s % 8
    at = (octet * 32 + np.arange(hd) % 32) * groups + np.arange(hd) // 32
    b[at] = (b[at] & ~np.uint32(15 << BIT[e])) | (c << np.uint32(BIT[e]))
    for g in range(groups):
        halves[(octet * groups + g) * 16 + e] = d[g]
        halves[(octet * groups + g) * 16 + 8 + e] = o[g]


def get(cache, plane, slots, is_v):
    """(codes, step, offset) of the first `slots` slots of a plane."""
    hd = cache.shape[-1] // 5
    groups, b = hd // 32, cache[plane]
    n = b.shape[0]
    codes = np.stack([b[:, :4 * hd] >> np.uint32(x) & 15 for x in BIT], -1)
    halves = np.ascontiguousarray(b[:, 4 * hd:]).view(np.float16)
    if is_v:   # [block, octet, dim % 32, group, slot] and [block, octet, group, (d, o), slot]
        codes = codes.reshape(n, 4, 32, groups, 8).transpose(0, 1, 4, 3, 2)
        halves = halves.reshape(n, 4, groups, 2, 8).transpose(0, 1, 4, 2, 3)
    codes, halves = codes.reshape(n * 32, hd)[:slots], halves.reshape(n * 32, groups, 2)[:slots]
    return codes, halves[..., 0], halves[..., 1]


def rows(cache, plane, slots, is_v):
    """float64 values [slots, head_dim] of a plane's first slots."""
    return values(*get(cache, plane, slots, is_v))


def attention(q, k_cache, v_cache, layer, sequence, base, context):
    """(out, weights) in 64 bits: q [tokens, kv_heads, group, head_dim]; out the same shape,
    weights [kv_heads, slots] the rows' softmax weights summed over tokens and group."""
    tokens, kv_heads, group, hd = q.shape
    out = np.zeros(q.shape)
    if base >= context:
        return out, np.zeros((kv_heads, 0))
    keys = min(base + tokens, context)
    total = np.zeros((kv_heads, keys))
    for h in range(kv_heads):
        k, v = (rows(c, (layer, sequence, h), keys, is_v) for c, is_v in ((k_cache, False), (v_cache, True)))
        for t in range(min(tokens, context - base)):
            n = base + t + 1
            s = q[t, h].astype(np.float64) @ k[:n].T / np.sqrt(hd)
            p = np.exp(s - s.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            out[t, h] = p @ v[:n]
            total[h, :n] += p.sum(0)
    return out, total


def select(weights, positions, n, keep, sinks, recent):
    """Moves [(from, to)] of one plane's first n slots."""
    if n <= keep:
        return []
    w, at = weights[:n], positions[:n].astype(np.int64)
    held = (at < sinks) | (at + recent > at.max())
    # the slots that are held, then by falling weight, then NaN; ties to the lower slot
    rank = sorted(range(n), key=lambda j: (0, 0.0, j) if held[j] else (2, 0.0, j) if np.isnan(w[j]) else (1, -w[j], j))
    stays = set(rank[:keep])
    holes = [j for j in range(keep) if j not in stays]
    sources = [j for j in range(keep, n) if j in stays]
    return list(zip(sources, holes))


def move(cache, plane, moves, is_v):
    """Carries moves out on one plane."""
    if not moves:
        return
    c, d, o = get(cache, plane, max(f for f, _ in moves) + 1, is_v)   # copies
    for f, t in moves:
        put(cache, plane, t, c[f], d[f], o[f], is_v)
