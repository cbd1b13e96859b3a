"""The 4-bit KV cache's operators as cases to measure: storing rows, attention over the
cache for prompts and single tokens, its accumulated weights, and the eviction by them.

A cache holds, for every layer, sequence and KV head, blocks of 32 slots. A row of
head_dim values is cut into groups of 32; a group has 4-bit codes c, a step d and an
offset o (both f16), and stands for the f16 values o + d * c. A block is 20 * head_dim
bytes, as dwords:

  K: [slot 32][head_dim / 8] dwords of 8 dimensions, then [slot 32][group] (d, o);
  V: [octet 4][dimension % 32][group] dwords of 8 slots, then [octet 4][group][d x 8, o x 8];

element e of a dword's eight is its bits 4 (e / 2) + 16 (e % 2) and the three above.
Slots that hold no row have whatever bits were there.
"""
import functools
import math

import numpy as np
import torch

own = False

GPU = "cuda"
NO_SLOT = -1            # a sequence that takes no part, as int32
LIMIT = 61440.0         # inputs are clamped to this before they are coded


# --------------------------------------------------------------------- the cases
def _attend(name, sequences, idle, tokens, length, context, heads, weights):
    q_heads, kv_heads, head_dim = heads
    return dict(name=name, kind="attend", sequences=sequences, idle=idle, tokens=tokens, length=length,
                context=context, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, weights=weights)


def listed():
    return [
        # The keys and values of one decode step, and of a long prompt's chunk, one layer.
        dict(name="store_token", kind="store", sequences=1, tokens=1, length=300, context=512, kv_heads=2, head_dim=128),
        dict(name="store_prompt_1900", kind="store", sequences=1, tokens=1900, length=0, context=2048, kv_heads=2,
             head_dim=128),
        # A decode step early in an utterance (the BaseLM's heads), and deep in its longest
        # context with the weights that an eviction goes by.
        _attend("decode_512", 1, 0, 1, 511, 512, (16, 2, 128), False),
        _attend("decode_8k_weights", 1, 0, 1, 8001, 8192, (16, 2, 128), True),
        # A server's step: sixteen requests of unequal length in one call, one of them idle.
        _attend("decode_batch16_32k", 16, 1, 1, 32700, 32768, (16, 2, 128), False),
        # Seven drafted tokens at once over a long cache, heads of 64.
        _attend("draft7_batch4_4k", 4, 0, 7, 4000, 4096, (16, 2, 64), False),
        # A short prompt, a long one, and a later chunk of a longer one with its weights.
        _attend("prompt_384", 1, 0, 384, 0, 512, (16, 2, 128), False),
        _attend("prompt_1900", 1, 0, 1900, 0, 2048, (16, 2, 128), False),
        _attend("chunk_1024_at_7000_weights", 1, 0, 1024, 7000, 8192, (16, 2, 128), True),
        # Every layer's choice of what stays when the context is full: half of it, and one step's single slot.
        dict(name="select_half_8k", kind="select", layers=28, sequences=1, length=8192, context=8192, kv_heads=2, keep=4096,
             sinks=4, recent=256),
        dict(name="select_one_batch4", kind="select", layers=8, sequences=4, length=2049, context=2304, kv_heads=2, keep=2048,
             sinks=4, recent=64),
        # The move that follows from it, for the ResidualLM's eight layers.
        dict(name="compact_half_4k", kind="compact", layers=8, sequences=1, length=4096, context=4096, kv_heads=2,
             head_dim=128, keep=2048, sinks=4, recent=256),
        # (a single slot's move is in the draws)
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "attend", "attend", "attend", "attend", "select", "compact"])
    q_heads, kv_heads, head_dim = rng.choice([(16, 2, 128), (16, 2, 128), (16, 2, 64), (8, 8, 64), (32, 4, 128),
                                              (10, 2, 128), (16, 1, 256)])
    if kind == "store":
        sequences = rng.choice([1, 1, 5, 16])
        tokens = _log(rng, 1, 2000 // sequences)
        length = rng.randint(0, 2048)
        return dict(kind=kind, sequences=sequences, tokens=tokens, length=length, context=length + tokens + rng.randint(0, 70),
                    kv_heads=kv_heads, head_dim=head_dim)
    if kind == "attend":
        form = rng.choice(["decode", "decode", "draft", "prompt"])
        if form == "prompt":
            sequences, tokens, length = rng.choice([1, 1, 2]), _log(rng, 17, 900), rng.choice([0, 0, _log(rng, 1, 4000)])
        else:
            sequences = rng.choice([1, 1, 3, 8])
            tokens = 1 if form == "decode" else rng.randint(2, 16)
            length = _log(rng, 1, 32000 if sequences < 8 else 16000)
        case = _attend("", sequences, rng.randint(0, sequences - 1) // 2, tokens, length, length + tokens + rng.randint(0, 90),
                       (q_heads, kv_heads, head_dim), rng.random() < 0.4)
        del case["name"]
        return case
    length = _log(rng, 40, 8192 if kind == "select" else 4096)
    keep = max(1, length - 1 if rng.random() < 0.3 else int(length * rng.uniform(0.2, 1.05)))
    sinks = rng.randint(0, min(8, keep))
    case = dict(kind=kind, layers=rng.choice([1, 8, 28] if kind == "select" else [1, 4, 8]), sequences=rng.choice([1, 1, 3]),
                length=length, context=max(length, keep) + rng.randint(1, 60), kv_heads=rng.choice([1, 2, 4]))
    if kind == "compact":
        case["head_dim"] = head_dim
    return dict(case, keep=keep, sinks=sinks, recent=rng.randint(0, (keep - sinks) // 2))


def _lengths(case):
    """Slots that each sequence has filled before the call; -1: the sequence is idle."""
    n = case["sequences"]
    got = [max(0, case["length"] - case["length"] * 2 * s // (3 * n)) for s in range(n)]
    return [NO_SLOT if s >= n - case.get("idle", 0) else v for s, v in enumerate(got)]


def work(case):
    kind, lengths = case["kind"], _lengths(case)
    if kind == "store":      # f32 rows in, blocks out, and back
        values = 2 * case["sequences"] * case["tokens"] * case["kv_heads"] * case["head_dim"]
        return dict(bytes=values * (4 + 0.625) * 2, flops=values * 4)
    if kind == "attend":
        t, qh, kh, hd = case["tokens"], case["q_heads"], case["kv_heads"], case["head_dim"]
        filled = sum(n + t for n in lengths if n >= 0)
        pairs = sum(t * n + t * (t + 1) // 2 for n in lengths if n >= 0) * qh
        rows = t * qh * case["sequences"]
        return dict(bytes=filled * kh * 1.25 * hd + rows * hd * 8 + (filled * kh * 4 if case["weights"] else 0),
                    flops=pairs * 4 * hd)
    planes = case["layers"] * case["kv_heads"]
    moves = planes * sum(min(case["keep"], max(0, n - case["keep"])) for n in lengths)
    filled = planes * sum(lengths)
    if kind == "select":
        return dict(bytes=filled * 8 + moves * 8, flops=filled * 4)
    kept = planes * len(lengths) * case["keep"]      # read back as f32
    return dict(bytes=kept * case["head_dim"] * 2 * (4 + 0.625) + moves * (case["head_dim"] * 2.5 + 24), flops=kept * case["head_dim"])


# ------------------------------------------------------------------- the format
def _code(x):
    """(codes, step, offset) of f32 rows [..., head_dim]; every step is an f32 operation rounded once."""
    g = x.float().unflatten(-1, (-1, 32)).clamp(-LIMIT, LIMIT)
    lo, hi = g.amin(-1), g.amax(-1)
    d = ((hi - lo).double() / 15).float().half()
    o = lo.half()
    steps = ((g - o.float().unsqueeze(-1)).double() / d.double().unsqueeze(-1)).float().round()
    c = torch.where(d.unsqueeze(-1) > 0, steps.clamp(0, 15), torch.zeros_like(steps))
    return c.flatten(-2).to(torch.int32), d, o


def _value(c, d, o):
    """The f16 values that codes stand for, as f32."""
    g = c.float().unflatten(-1, (-1, 32))
    return (g * d.float().unsqueeze(-1) + o.float().unsqueeze(-1)).half().float().flatten(-2)


def _pack8(c):
    shifts = torch.tensor([4 * (e // 2) + 16 * (e % 2) for e in range(8)], device=c.device)
    word = (c.to(torch.int64) << shifts).sum(-1)
    return torch.where(word >= 1 << 31, word - (1 << 32), word).to(torch.int32)


def _unpack8(w):
    shifts = torch.tensor([4 * (e // 2) + 16 * (e % 2) for e in range(8)], device=w.device, dtype=torch.int32)
    return (w.unsqueeze(-1) >> shifts) & 15


def _pack(c, d, o, values):
    """Blocks [..., blocks, 5 * head_dim] int32 of codes [..., slots, head_dim], slots a multiple of 32."""
    lead, slots, hd = c.shape[:-2], c.shape[-2], c.shape[-1]
    n, groups = slots // 32, hd // 32
    if not values:
        codes = _pack8(c.reshape(*lead, n, 32 * hd // 8, 8))
        scales = torch.stack([d, o], -1).contiguous().view(torch.int32).reshape(*lead, n, hd)
    else:
        codes = _pack8(c.reshape(*lead, n, 4, 8, groups, 32).movedim(-3, -1).transpose(-3, -2)).reshape(*lead, n, 4 * hd)
        scales = torch.stack([t.reshape(*lead, n, 4, 8, groups).transpose(-1, -2) for t in (d, o)], -2).contiguous()
        scales = scales.view(torch.int32).reshape(*lead, n, hd)
    return torch.cat([codes, scales], -1).contiguous()


def _unpack(blocks, values):
    """(codes, step, offset) of blocks, the inverse of _pack."""
    lead, n, hd = blocks.shape[:-2], blocks.shape[-2], blocks.shape[-1] // 5
    groups = hd // 32
    codes, scales = blocks[..., :4 * hd], blocks[..., 4 * hd:].contiguous().view(torch.float16)
    if not values:
        c = _unpack8(codes).reshape(*lead, n * 32, hd)
        scales = scales.reshape(*lead, n * 32, groups, 2)
        return c, scales[..., 0], scales[..., 1]
    c = _unpack8(codes).reshape(*lead, n, 4, 32, groups, 8).transpose(-3, -2).movedim(-1, -3).reshape(*lead, n * 32, hd)
    scales = scales.reshape(*lead, n, 4, groups, 2, 8).movedim(-1, -3)
    return c, scales[..., 0].reshape(*lead, n * 32, groups), scales[..., 1].reshape(*lead, n * 32, groups)


# ------------------------------------------------------------------- inputs
def _rng(seed):
    return torch.Generator(device=GPU).manual_seed(int(seed) & 0x7FFFFFFFFFFF)


def _rows(g, *shape):
    """Keys or values of trained models: channels with means of their own, a few of them large."""
    x = torch.randn(*shape, generator=g, device=GPU)
    mean = torch.randn(shape[-1], generator=g, device=GPU)
    mean[torch.randint(0, shape[-1], (2,), generator=g, device=GPU)] *= 4
    return x + mean


def _cache(g, planes, slots, filled, hd, blank=False):
    """K and V blocks [*planes, blocks, 5 * hd] whose slots below `filled` [*planes] hold rows; the others hold any bits,
    or zeros where `blank`."""
    blocks = []
    used = torch.arange(slots, device=GPU) < filled.unsqueeze(-1)
    for values in (False, True):
        c, d, o = _code(_rows(g, *planes, slots, hd))
        c = torch.where(used.unsqueeze(-1), c, torch.randint(0, 16, c.shape, generator=g, device=GPU, dtype=torch.int32))
        bits = [torch.randint(-32768, 32768, d.shape, generator=g, device=GPU, dtype=torch.int16).view(torch.float16)
                for _ in range(2)]
        if blank:
            bits = [torch.zeros_like(d), torch.zeros_like(d)]
        d, o = torch.where(used.unsqueeze(-1), d, bits[0]), torch.where(used.unsqueeze(-1), o, bits[1])
        blocks.append(_pack(c, d, o, values))
        del c, d, o, bits
    return blocks


def _tables(g, case):
    """Accumulated weights and positions of every slot, as steps and earlier evictions leave them."""
    shape = (case["layers"], case["sequences"], case["kv_heads"], case["context"])
    # heavy-tailed, and zero or equal for many slots
    w = torch.rand(shape, generator=g, device=GPU).pow(6) * 40
    w = torch.where(torch.rand(shape, generator=g, device=GPU) < 0.4, (w * 8).floor() / 8, w)
    # distinct positions, not in the slots' order
    order = torch.rand(shape, generator=g, device=GPU).argsort(-1)
    lengths = torch.tensor(_lengths(case), device=GPU).view(1, -1, 1, 1)
    at = torch.where(order < lengths, order, order + case["context"])
    return w.contiguous(), at.sort(-1).values.gather(-1, torch.rand(shape, generator=g, device=GPU).masked_fill(
        torch.arange(case["context"], device=GPU) >= lengths, 2.0).argsort(-1)).to(torch.int32).contiguous()


@functools.lru_cache(maxsize=1)
def _context():
    from voxgen_amd.runtime import Context
    torch.zeros(1, device=GPU)
    return Context(torch.cuda.current_device())


class _View:
    """Device memory of the library as a torch tensor; keeps its owner alive."""

    def __init__(self, owner, ptr, shape, typestr):
        self.owner = owner
        self.__cuda_array_interface__ = dict(shape=tuple(shape), typestr=typestr, data=(ptr, False), version=2)


def _view(buf, shape, dtype=torch.float32):
    typestr = {torch.float32: "<f4", torch.int32: "<i4"}[dtype]
    return torch.as_tensor(_View(buf, buf.device_ptr, shape, typestr), device=GPU)


def _device(x):
    """A buffer of the library with x's values."""
    b = _context().alloc(x.numel() * x.element_size())
    _view(b, x.shape, x.dtype).copy_(x)
    return b


def _empty(*shape, dtype=torch.float32):
    b = _context().alloc(math.prod(shape) * 4)
    return b, _view(b, shape, dtype)


def prepare(case, seed):
    kind, g = case["kind"], _rng(seed)
    seqs, kh = case["sequences"], case["kv_heads"]
    s = dict(case=case, slots=torch.tensor(_lengths(case), device=GPU, dtype=torch.int32))
    slots32 = (case["context"] + 31) // 32 * 32
    if kind == "store":
        hd, rows = case["head_dim"], seqs * case["tokens"]
        s["k"], s["v"] = _rows(g, rows, kh, hd).reshape(rows, kh * hd), _rows(g, rows, kh, hd).reshape(rows, kh * hd)
        filled = s["slots"].view(1, -1, 1).expand(1, seqs, kh)
        s["blocks"] = _cache(g, (1, seqs, kh), slots32, filled, hd)
    elif kind == "attend":
        hd, t = case["head_dim"], case["tokens"]
        s["q"] = torch.randn(seqs * t, case["q_heads"] * hd, generator=g, device=GPU) * 1.2
        filled = torch.where(s["slots"] >= 0, s["slots"] + t, 0).view(1, -1, 1).expand(1, seqs, kh)
        s["blocks"] = _cache(g, (1, seqs, kh), slots32, filled, hd)
        if case["weights"]:
            s["weights"] = torch.rand(1, seqs, kh, case["context"], generator=g, device=GPU)
    else:
        s["weights"], s["slot_positions"] = _tables(g, case)
        if kind == "compact":
            filled = s["slots"].view(1, -1, 1).expand(case["layers"], seqs, kh)
            s["blocks"] = _cache(g, (case["layers"], seqs, kh), slots32, filled, case["head_dim"], blank=True)
            s["plan"] = _plan(case, s)
    if own:   # the program's cache and buffers
        from voxgen_amd.kv4 import Kv4Cache
        c = s["cache"] = Kv4Cache(_context(), case.get("layers", 1), seqs, kh, case.get("head_dim", 64), case["context"],
                                  track="weights" in s)
        _view(c.slots, (seqs,), torch.int32).copy_(s["slots"])
        if "blocks" in s:
            for buf, x in zip((c.k, c.v), s.pop("blocks")):
                _view(buf, x.shape, torch.int32).copy_(x)
        for name in ("weights", "slot_positions"):
            if name in s:
                x = s[name]
                s[name] = _view(getattr(c, name), x.shape, x.dtype)
                s[name].copy_(x)
        if kind == "store":
            s["k"], s["v"] = _device(s["k"]), _device(s["v"])
            s["back"] = [_empty(rows, kh * hd) for _ in range(2)]
        elif kind == "attend":
            s["q"], s["out"] = _device(s["q"]), _empty(seqs * t, case["q_heads"] * hd)
        else:
            moves = c.plan_moves(case["keep"])
            s["plan_out"] = _empty(case["layers"], seqs, kh, moves, 2, dtype=torch.int32)
            if kind == "compact":
                s["plan_out"][1].copy_(s.pop("plan"))
                s["back"] = [_empty(case["layers"], seqs * case["keep"], kh * case["head_dim"]) for _ in range(2)]
                s["from_zero"] = _context().zeros(seqs * 4)
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    if own:
        return _run_own(case, s)
    return dict(store=_store, attend=_attention, select=_select, compact=_compact)[case["kind"]](case, s)


def _run_own(case, s):
    kind, c = case["kind"], s["cache"]
    if kind == "store":
        (kb, kt), (vb, vt) = s["back"]
        c.store(0, s["k"], s["v"], tokens=case["tokens"])
        c.load(0, kb, vb, tokens=case["tokens"])
        return dict(k=kt, v=vt)
    if kind == "attend":
        buf, out = s["out"]
        c.attention(0, s["q"], buf, case["q_heads"], tokens=case["tokens"], decay=0.0)
        return dict(out=out, weights=s["weights"]) if case["weights"] else out
    if kind == "select":
        buf, plan = s["plan_out"]
        c.select(buf, case["keep"], case["sinks"], case["recent"])
        return plan
    c.compact(s["plan_out"][0], case["keep"])
    (kb, kt), (vb, vt) = s["back"]
    for layer in range(case["layers"]):
        at = layer * kt[0].numel()
        c.load(layer, kb, vb, tokens=case["keep"], k_base=at, v_base=at, slots=s["from_zero"])
    return dict(k=kt, v=vt, weights=s["weights"], slot_positions=s["slot_positions"],
                slots=_view(c.slots, (case["sequences"],), torch.int32))


def _store(case, s):
    """The rows' values after a round through the cache's format."""
    shape = (-1, case["kv_heads"], case["head_dim"])
    return {n: _value(*_code(s[n].view(shape))).flatten(-2) for n in ("k", "v")}


def _attention(case, s):
    seqs, t, qh, kh, hd = (case[n] for n in ("sequences", "tokens", "q_heads", "kv_heads", "head_dim"))
    k, v = (_value(*_unpack(b[0], values)) for b, values in zip(s["blocks"], (False, True)))      # [seqs, kh, slots, hd]
    first = s["slots"].view(-1, 1, 1)
    last = first + torch.arange(t, device=GPU).view(1, -1, 1)                                       # [seqs, t, 1]
    seen = (torch.arange(k.shape[2], device=GPU) <= last) & (first >= 0)                            # [seqs, t, slots]
    some = seen.any(1)[:, None, :, None]
    k, v = torch.where(some, k, 0.0), torch.where(some, v, 0.0)
    group = qh // kh
    q = s["q"].view(seqs, t, kh, group, hd).permute(0, 2, 3, 1, 4).reshape(seqs, kh, group * t, hd)
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(hd)
    seen = seen.repeat(1, group, 1).unsqueeze(1)                                                    # [seqs, 1, group * t, slots]
    x = torch.where(seen, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    e = torch.where(seen, torch.exp(x - torch.where(top > -math.inf, top, 0.0)), 0.0)
    del x
    p = e / torch.where(seen.any(-1, keepdim=True), e.sum(-1, keepdim=True), 1.0)
    out = torch.matmul(p, v).view(seqs, kh, group, t, hd).permute(0, 3, 1, 2, 4).reshape(seqs * t, qh * hd)
    if not case["weights"]:
        return out
    w = p.sum(2)[..., :case["context"]]
    return dict(out=out, weights=torch.where(some[..., 0][..., :case["context"]], w, s["weights"][0]).unsqueeze(0))


def _ranked(case, s):
    """Truth of every slot that stays: the `keep` of the largest weights, ties to the lowest slot."""
    slot = torch.arange(case["context"], device=GPU)
    n = s["slots"].view(1, -1, 1, 1)
    at, filled = s["slot_positions"], slot < n
    newest = torch.where(filled, at, -1).amax(-1, keepdim=True)
    held = (at < case["sinks"]) | (at > newest - case["recent"])
    key = torch.where(filled, torch.where(held, math.inf, s["weights"]), -math.inf)
    order = key.sort(dim=-1, descending=True, stable=True).indices
    return torch.zeros_like(filled | held).scatter(-1, order[..., :case["keep"]], True) & filled, filled


def _plan(case, s):
    """Moves [layers, sequences, kv_heads, moves, 2] (from, to): the i-th slot that stays above `keep` goes to the
    i-th one below it that does not."""
    kept, filled = _ranked(case, s)
    keep, context = case["keep"], case["context"]
    moves = min(keep, context - keep)
    slot = torch.arange(context, device=GPU).expand(kept.shape)
    full = s["slots"].view(1, -1, 1, 1) > keep
    ends = []
    for which in (kept & (slot >= keep) & full, ~kept & (slot < keep) & full):
        rank = torch.where(which, which.cumsum(-1) - 1, moves)
        ends.append(torch.full((*kept.shape[:-1], moves + 1), NO_SLOT, device=GPU, dtype=torch.int32)
                    .scatter(-1, rank, slot.to(torch.int32))[..., :moves])
    return torch.stack(ends, -1).contiguous()


def _select(case, s):
    return _plan(case, s)


def _compact(case, s):
    keep, plan = case["keep"], s["plan"].long()
    src, dst = plan[..., 0], plan[..., 1]
    end = case["context"]
    at = torch.arange(end + 1, device=GPU).expand(*src.shape[:-1], end + 1)
    at = at.scatter(-1, torch.where(dst >= 0, dst, end), torch.where(src >= 0, src, end))[..., :end]   # slot -> where its row was
    rows = []
    for b, values in zip(s["blocks"], (False, True)):
        x = _value(*_unpack(b, values))
        x = x.gather(-2, at[..., :keep].unsqueeze(-1).expand(*at.shape[:-1], keep, x.shape[-1]))
        rows.append(x.permute(0, 1, 3, 2, 4).reshape(case["layers"], case["sequences"] * keep, -1))
    return dict(k=rows[0], v=rows[1], weights=s["weights"].gather(-1, at), slot_positions=s["slot_positions"].gather(-1, at),
                slots=s["slots"].clamp(max=keep))


# ------------------------------------------------------------------- in 64 bits
def _exact_rows(x, hd):
    """The values that rows [n, kv_dim] are stored as, from the format's definition with numpy."""
    g = np.clip(x.cpu().numpy().reshape(-1, 32), np.float32(-LIMIT), np.float32(LIMIT))
    lo = g.min(1)
    step = ((g.max(1) - lo) / np.float32(15)).astype(np.float16)
    base = lo.astype(np.float16)
    with np.errstate(divide="ignore", invalid="ignore"):
        code = np.rint((g - base.astype(np.float32)[:, None]) / step.astype(np.float32)[:, None])
    code = np.where(step[:, None] > 0, np.clip(code, 0, 15), 0).astype(np.float64)
    return (base.astype(np.float64)[:, None] + step.astype(np.float64)[:, None] * code).astype(np.float16).astype(np.float64).reshape(x.shape)


def _exact_block_values(blocks, hd, values):
    """f64 values [slots, hd] of one plane's blocks, dword by dword as the layout says."""
    n, groups = blocks.shape[0], hd // 32
    words = blocks.cpu().numpy().view(np.uint32)
    codes = np.stack([(words[:, :4 * hd] >> np.uint32(4 * (e // 2) + 16 * (e % 2))) & 15 for e in range(8)], -1)
    halves = np.ascontiguousarray(words[:, 4 * hd:]).view(np.float16)
    if values:
        codes = codes.reshape(n, 4, 32, groups, 8).transpose(0, 1, 4, 3, 2).reshape(n * 32, groups, 32)
        halves = halves.reshape(n, 4, groups, 2, 8).transpose(0, 1, 4, 2, 3).reshape(n * 32, groups, 2)
    else:
        codes, halves = codes.reshape(n * 32, groups, 32), halves.reshape(n * 32, groups, 2)
    halves = halves.astype(np.float64)
    with np.errstate(all="ignore"):
        return (halves[..., 1:] + halves[..., :1] * codes).astype(np.float16).astype(np.float64).reshape(n * 32, hd)


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    kind, lengths = case["kind"], _lengths(case)
    if kind == "select":
        return None
    hd = case["head_dim"]
    if kind == "store":
        return {n: _exact_rows(s[n], hd) for n in ("k", "v")}
    if kind == "compact":
        layers, seqs, kh, keep = case["layers"], case["sequences"], case["kv_heads"], case["keep"]
        plan = s["plan"].cpu().numpy()
        rows = [np.zeros((layers, seqs, keep, kh, hd)) for _ in range(2)]
        tables = s["weights"].cpu().numpy().astype(np.float64)
        for i in np.ndindex(layers, seqs, kh):
            moves = plan[i][plan[i][:, 1] >= 0]
            for b, values, to in zip(s["blocks"], (False, True), rows):
                x = _exact_block_values(b[i], hd, values)
                x[moves[:, 1]] = x[moves[:, 0]]
                to[i[0], i[1], :, i[2]] = x[:keep]
            tables[i][moves[:, 1]] = tables[i][moves[:, 0]]
        return dict(k=rows[0].reshape(layers, seqs * keep, kh * hd), v=rows[1].reshape(layers, seqs * keep, kh * hd),
                    weights=tables, slot_positions=None, slots=None)
    seqs, t, qh, kh = (case[n] for n in ("sequences", "tokens", "q_heads", "kv_heads"))
    if seqs * kh * (case["length"] + t) > 2_000_000:
        return None
    q = s["q"].double().view(seqs, t, kh, qh // kh, hd)
    out = torch.zeros(seqs, t, kh, qh // kh, hd, dtype=torch.float64, device=GPU)
    w = s["weights"].double() if case["weights"] else None
    for b in range(seqs):
        n = lengths[b] + t
        if lengths[b] < 0:
            continue
        hidden = torch.ones(t, n, device=GPU, dtype=torch.bool).triu(lengths[b] + 1)
        for h in range(kh):
            k, v = (torch.from_numpy(_exact_block_values(x[0, b, h], hd, values)[:n]).to(GPU)
                    for x, values in zip(s["blocks"], (False, True)))
            total = torch.zeros(n, dtype=torch.float64, device=GPU)
            for j in range(qh // kh):
                p = torch.softmax((q[b, :, h, j] @ k.T / math.sqrt(hd)).masked_fill(hidden, -math.inf), -1)
                out[b, :, h, j] = p @ v
                total += p.sum(0)
            if w is not None:
                w[0, b, h, :n] = total
    out = out.view(seqs * t, qh * hd)
    return out if w is None else dict(out=out, weights=w)
