"""The paged KV cache's operators as cases to measure: block tables and slot maps from
request lengths, storing rows, attention of new tokens over the pages, and attention over
the pages that a cheap score selects for each query.

K and V lie in pages of `page_size` slots, f16, per layer [page][kv_head], and within a page

  K: [slot / 16][head_dim / 8][slot % 16][8],   V: [slot / 8][head_dim][8];

a request's position p is slot p % page_size of page table[request][p // page_size]. A step
has rows of several requests one behind the other, counts[i] of request i, at its positions
lengths[i] and up; row t of them attends to positions 0..lengths[i] + t. Beside a page lie its
bounds, f16 [page][kv_head][lo, hi][head_dim]: each dimension's least and greatest key. Slots
that hold no row have finite values of earlier requests.
"""
import functools
import math

import numpy as np
import torch

own = False

GPU = "cuda"
NONE = -1               # no page, slot, request or position, as int32


# --------------------------------------------------------------------- the cases
def _case(name, kind, requests, length, tokens, page_size, heads, ragged=False, idle=0, **more):
    q_heads, kv_heads, head_dim = heads
    case = dict(name=name, kind=kind, requests=requests, length=length, tokens=tokens, page_size=page_size, q_heads=q_heads,
                kv_heads=kv_heads, head_dim=head_dim, ragged=ragged, idle=idle, **more)
    return case if name else {k: v for k, v in case.items() if k != "name"}


def listed():
    base = (16, 2, 128)      # the BaseLM's heads
    return [
        # The plan of one decode step of a few requests, and of a busy server's: single tokens, prompts in
        # chunks, idle requests, and fewer free pages than they all ask for.
        _case("plan_decode_16", "plan", 16, 8000, 1, 32, base, short=False),
        _case("plan_mixed_512", "plan", 512, 2000, 64, 16, base, ragged=True, idle=40, short=True),
        # One layer's keys and values of a decode step, and of prompts of several lengths together.
        _case("store_token_16", "store", 16, 1000, 1, 32, base, bounds=False),
        _case("store_prompts_4", "store", 4, 300, 700, 64, base, ragged=True, bounds=True),
        # Single tokens: early in an utterance, deep in the longest context, a batch of unequal lengths
        # with an idle request, and a large batch.
        _case("decode_one_512", "attend", 1, 511, 1, 32, base),
        _case("decode_one_32k", "attend", 1, 32700, 1, 64, base),
        _case("decode_batch16_8k", "attend", 16, 8001, 1, 16, base, idle=1),
        _case("decode_batch64_24k", "attend", 64, 24000, 1, 32, base),
        # Drafted tokens over heads of 64, and chunks of two prompts over what is cached of them.
        _case("draft5_batch8_4k", "attend", 8, 4000, 5, 32, (16, 2, 64)),
        _case("prompts_700_at_3000", "attend", 2, 3001, 700, 32, base, ragged=True),
        # Pages selected for each query: a token deep in a long context, and a batch of them.
        _case("sparse_one_32k", "sparse", 1, 32600, 1, 32, base, budget=64, sinks=1, recent=8),
        _case("sparse_batch16_32k", "sparse", 16, 32700, 1, 64, base, budget=32, sinks=1, recent=4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "store", "attend", "attend", "attend", "sparse", "sparse"])
    heads = rng.choice([(16, 2, 128), (16, 2, 128), (16, 2, 64), (8, 8, 64), (32, 4, 128), (10, 2, 128), (16, 1, 256)])
    page_size = rng.choice([16, 32, 32, 64, 128])
    ragged = rng.random() < 0.5
    if kind == "plan":
        requests = _log(rng, 1, 512)
        return _case("", kind, requests, rng.randint(1, 4000), _log(rng, 1, 64), page_size, heads, ragged,
                     rng.randint(0, requests - 1) // 4, short=rng.random() < 0.4)
    if kind == "store":
        requests = _log(rng, 1, 32)
        return _case("", kind, requests, rng.randint(0, 1500), _log(rng, 1, max(1, 2000 // requests)), page_size, heads, ragged,
                     rng.randint(0, requests - 1) // 3, bounds=rng.random() < 0.6)
    if kind == "attend":
        form = rng.choice(["decode", "decode", "draft", "prompt"])
        if form == "prompt":
            requests, tokens, length = rng.choice([1, 1, 3]), _log(rng, 17, 450), rng.choice([0, _log(rng, 1, 3000)])
        else:
            requests = _log(rng, 1, 32)
            tokens = 1 if form == "decode" else rng.randint(2, 16)
            length = _log(rng, 1, 32000 if requests < 8 else 10000)
        return _case("", kind, requests, length, tokens, page_size, heads, ragged, rng.randint(0, requests - 1) // 3)
    requests = _log(rng, 1, 24)
    length = _log(rng, 200, 60000 if requests < 4 else 30000)
    budget = _log(rng, 8, 2048 // page_size if page_size < 128 else 24)
    return _case("", kind, requests, length, rng.choice([1, 1, 1, rng.randint(2, 6)]), page_size, heads, ragged,
                 rng.randint(0, requests - 1) // 3, budget=budget, sinks=rng.randint(0, 2), recent=rng.randint(1, budget // 2))


def _shape(case):
    """(lengths, counts) of the requests, table width, rows and pages of a case."""
    n, tokens = case["requests"], case["tokens"]
    lengths = [max(0, case["length"] - case["length"] * 2 * ((5 * i) % n) // (3 * n)) for i in range(n)]
    counts = [0 if i >= n - case["idle"] else 1 + (i * 7919 + tokens - 1) % tokens if case["ragged"] else tokens
              for i in range(n)]
    ps = case["page_size"]
    pages = [-(-(a + c) // ps) for a, c in zip(lengths, counts)]
    return lengths, counts, max(max(pages), 1) + 1, sum(counts), sum(pages) + 5


def work(case):
    kind = case["kind"]
    lengths, counts, width, rows, pages = _shape(case)
    kh, qh, hd, ps = (case[n] for n in ("kv_heads", "q_heads", "head_dim", "page_size"))
    new = sum(-(-(a + c) // ps) - -(-a // ps) for a, c in zip(lengths, counts))
    if kind == "plan":       # lengths, counts and the free pages in; table entries and three words a row out
        return dict(bytes=case["requests"] * 12 + new * 8 + rows * 16, flops=case["requests"] * 4 + rows * 4)
    if kind == "store":      # f32 rows in, f16 rows out; the bounds of the pages that they lie in
        touched = sum(-(-(a + c) // ps) - a // ps for a, c in zip(lengths, counts) if c)
        return dict(bytes=2 * rows * kh * hd * 6 + (touched * kh * hd * 4 if case["bounds"] else 0), flops=2 * rows * kh * hd)
    taking = [(a, c) for a, c in zip(lengths, counts) if c]
    if kind == "attend":
        filled = sum(a + c for a, c in taking)
        pairs = sum(c * a + c * (c + 1) // 2 for a, c in taking) * qh
        return dict(bytes=filled * kh * hd * 4 + filled // ps * 4 + rows * qh * hd * 8, flops=pairs * 4 * hd)
    most = case["budget"] * ps
    held = sum(min(a + c, c * most) for a, c in taking)
    seen = sum(-(-(a + c) // ps) for a, c in taking)
    return dict(bytes=(seen + held) * kh * hd * 4 + rows * (qh * hd * 8 + kh * case["budget"] * 4),
                flops=sum(c * min(a + c, most) for a, c in taking) * qh * 4 * hd
                + sum(c * -(-(a + c) // ps) for a, c in taking) * kh * hd * 4)


# ------------------------------------------------------------------- inputs
def _rng(seed):
    return torch.Generator(device=GPU).manual_seed(int(seed) & 0x7FFFFFFFFFFF)


def _i32(x):
    return torch.as_tensor(np.asarray(x), device=GPU).to(torch.int32)


def _rows(g, *shape):
    """Keys or values of trained models: channels with means of their own, a few of them large."""
    mean = torch.randn(shape[-1], generator=g, device=GPU)
    mean[torch.randint(0, shape[-1], (2,), generator=g, device=GPU)] *= 4
    return torch.randn(*shape, generator=g, device=GPU) + mean


def _batch(case, seed):
    """Lengths, counts, block tables and the pool of free pages as earlier steps have left them, and the rows of
    the step: what a server holds when it begins one."""
    lengths, counts, width, rows, pages = _shape(case)
    rng = np.random.RandomState(seed & 0x7FFFFFFF)
    ps, n = case["page_size"], case["requests"]
    if case["kind"] == "plan":      # requests in any order, each some tokens behind
        order = rng.permutation(n)
        lengths = [max(0, lengths[i] - int(rng.randint(0, 3 * ps))) for i in order]
        counts = [counts[i] for i in order]
        rows += 7                   # the row buffer has some to spare
    any_page = rng.permutation(pages)
    tables = np.full((n, width), NONE, np.int64)
    have = [-(-a // ps) for a in lengths]
    used = 0
    for i, k in enumerate(have):
        tables[i, :k] = any_page[used:used + k]
        used += k
    free = list(any_page[used:])
    need = sum(-(-(a + c) // ps) - k for a, c, k in zip(lengths, counts, have))
    if case.get("short"):
        free = free[:max(1, need * 3 // 4)]
    pool = np.zeros(pages + 1, np.int64)
    pool[0] = len(free)
    pool[1:1 + len(free)] = free
    s = dict(case=case, width=width, rows=rows, pages=pages, lengths=_i32(lengths), counts=_i32(counts), tables=_i32(tables),
             pool=_i32(pool))
    if case["kind"] != "plan":      # the step's plan, in hand for all its layers
        s.update(zip(("tables", "slots", "requests", "positions", "granted"), _plan(case, s).values()))
        s["taking"] = [(i, a, c) for i, (a, c) in enumerate(zip(lengths, counts)) if c]
    return s


def _filled(case, s):
    """Slots of every page that hold rows, the step's own among them."""
    ps, total = case["page_size"], (s["lengths"] + s["counts"]).long()
    col = torch.arange(s["width"], device=GPU)
    held = (total[:, None] - col * ps).clamp(0, ps)
    out = torch.zeros(s["pages"], dtype=torch.long, device=GPU)
    at = s["tables"].long()
    return out.scatter_add(0, at[at >= 0], held[at >= 0])


def _caches(g, case, s, spread):
    """K and V of every page, as rows [pages, kv_heads, slots, head_dim] in their layouts."""
    kh, hd, ps, pages = case["kv_heads"], case["head_dim"], case["page_size"], s["pages"]
    k = _rows(g, pages, kh, ps, hd)
    if spread:               # what is said on a page has a direction of its own
        k += torch.randn(pages, kh, 1, hd, generator=g, device=GPU)
    v = _rows(g, pages, kh, ps, hd)
    return _lay_k(k.half()), _lay_v(v.half())


def _lay_k(x):
    return x.unflatten(-1, (-1, 8)).unflatten(-3, (-1, 16)).transpose(-3, -2).contiguous()


def _lay_v(x):
    return x.unflatten(-2, (-1, 8)).transpose(-2, -1).contiguous()


def _rows_k(x):
    return x.transpose(-3, -2).flatten(-2).flatten(-3, -2)


def _rows_v(x):
    return x.transpose(-2, -1).flatten(-3, -2)


def _bounds(case, s, k):
    """f16 [pages, kv_heads, 2, head_dim] over the filled slots; zeros where a page has none."""
    x = _rows_k(k)                                                                  # [pages, kv_heads, slots, head_dim]
    n = _filled(case, s).view(-1, 1, 1, 1)
    there = torch.arange(case["page_size"], device=GPU).view(1, 1, -1, 1) < n
    lo, hi = torch.where(there, x, math.inf).amin(-2), torch.where(there, x, -math.inf).amax(-2)
    return torch.where(n > 0, torch.stack([lo, hi], -2), 0.0).half()


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


def _view(buf, shape, dtype=torch.float32, offset=0):
    typestr = {torch.float32: "<f4", torch.float16: "<f2", torch.int32: "<i4"}[dtype]
    return torch.as_tensor(_View(buf, buf.device_ptr + offset, shape, typestr), device=GPU)


def _device(x):
    """A buffer of the library with x's values."""
    b = _context().alloc(x.numel() * x.element_size())
    _view(b, x.shape, x.dtype).copy_(x)
    return b


def prepare(case, seed):
    kind, g, s = case["kind"], _rng(seed), _batch(case, seed)
    kh, qh, hd, ps, rows = case["kv_heads"], case["q_heads"], case["head_dim"], case["page_size"], s["rows"]
    if kind != "plan":
        s["kc"], s["vc"] = _caches(g, case, s, kind == "sparse")
    if kind == "store":
        s["k"], s["v"] = _rows(g, rows, kh * hd), _rows(g, rows, kh * hd)
    if kind in ("attend", "sparse"):
        s["q"] = torch.randn(rows, qh * hd, generator=g, device=GPU) * 1.2
    if kind == "sparse" or case.get("bounds"):
        s["bounds"] = _bounds(case, s, s["kc"])
    if own:   # the program's cache and buffers
        from voxgen_amd.paged import PagedCache
        c = s["cache"] = PagedCache(_context(), 1, s["pages"], ps, kh, hd, case["requests"], s["width"], max(rows, 1), qh,
                                    max_count=case["tokens"], bounds="bounds" in s)
        for buf, name in ((c.lengths, "lengths"), (c.counts, "counts"), (c.tables, "tables"), (c.pool, "pool")):
            _view(buf, s[name].shape, torch.int32).copy_(s[name])
        for buf, name in ((c.k, "kc"), (c.v, "vc"), (c.bounds, "bounds")):
            if name in s:
                x = s[name]
                s[name] = _view(buf, x.shape, torch.float16)
                s[name].copy_(x)
        if kind == "plan":
            s["tables"] = _view(c.tables, s["tables"].shape, torch.int32)
            s["out"] = {n: _view(c.plan_buffer, (size,), torch.int32, offset) for n, (offset, size) in c.plan_layout().items()}
        else:
            torch.cuda.synchronize()
            c.plan()
        if kind == "store":
            s["k"], s["v"] = _device(s["k"]), _device(s["v"])
        elif kind != "plan":
            s["q"] = _device(s["q"])
            s["out"] = _context().alloc(rows * qh * hd * 4)
            s["out_view"] = _view(s["out"], (rows, qh * hd))
        if kind == "sparse":
            s["selected"] = c.selection(case["budget"])
            s["selected_view"] = _view(s["selected"], (rows, kh, case["budget"]), torch.int32)
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    if own:
        return _run_own(case, s)
    return dict(plan=_plan, store=_store, attend=_attend, sparse=_sparse)[case["kind"]](case, s)


def _run_own(case, s):
    kind, c = case["kind"], s["cache"]
    if kind == "plan":
        c.plan()
        return dict(tables=s["tables"], **s["out"])
    if kind == "store":
        c.store(0, s["k"], s["v"])
        return {n: s[n] for n in ("kc", "vc", "bounds") if n in s}
    if kind == "attend":
        c.attention(0, s["q"], s["out"])
        return s["out_view"]
    c.select(0, s["q"], s["selected"], case["budget"], case["sinks"], case["recent"])
    c.attention(0, s["q"], s["out"], selected=s["selected"], budget=case["budget"])
    return dict(pages=s["selected_view"], out=s["out_view"])


def _plan(case, s):
    """Every request's pages for its new tokens, where its rows' pages, those of all requests before it and the row
    buffer suffice; of each row its slot, request and position."""
    ps, width, rows = case["page_size"], s["width"], max(s["rows"], 1)
    a, c, free = s["lengths"].long(), s["counts"].long(), s["pool"][0].long()
    upto = c.cumsum(0)
    have = (a + ps - 1) // ps
    fits = (c > 0) & (c <= case["tokens"]) & (upto <= rows) & (a + c <= width * ps)
    need = torch.where(fits, (a + c + ps - 1) // ps - have, 0)
    pages_upto = need.cumsum(0)
    granted = fits & ((need == 0) | (pages_upto <= free))
    col = torch.arange(width, device=GPU)
    nth = (pages_upto - need)[:, None] + col - have[:, None]
    fresh = granted[:, None] & (col >= have[:, None]) & (col < (have + need)[:, None])
    tables = torch.where(fresh, s["pool"][(free - nth).clamp(1, s["pages"])].long(), s["tables"].long())
    r = torch.arange(rows, device=GPU)
    request = torch.searchsorted(upto, r, right=True).clamp(max=case["requests"] - 1)
    there = (r < upto[-1]) & granted[request]
    position = a[request] + r - (upto - c)[request]
    page = tables[request, (position // ps).clamp(0, width - 1)]
    slot = page * ps + position % ps
    got = dict(tables=tables, slots=torch.where(there, slot, NONE), requests=torch.where(there, request, NONE),
               positions=torch.where(there, position, NONE), granted=torch.where(granted, c, 0))
    return {n: x.to(torch.int32) for n, x in got.items()}


def _store(case, s):
    """The caches with the rows in their slots, and the bounds of the pages that they lie in."""
    kh, hd, ps = case["kv_heads"], case["head_dim"], case["page_size"]
    slot = s["slots"].long()
    page, at = slot // ps, slot % ps
    k, v = s["k"].view(-1, kh, hd).half(), s["v"].view(-1, kh, hd).half()
    kc, vc = s["kc"].clone(), s["vc"].clone()
    kc[page, :, at // 16, :, at % 16] = k.unflatten(-1, (-1, 8))
    vc[page, :, at // 8, :, at % 8] = v
    if "bounds" not in s:
        return dict(kc=kc, vc=vc)
    return dict(kc=kc, vc=vc, bounds=torch.where(torch.zeros(s["pages"], device=GPU, dtype=torch.bool).index_fill(0, page, True)
                                                 .view(-1, 1, 1, 1), _bounds(case, s, kc), s["bounds"]))


def _softmax(x, seen):
    x = torch.where(seen, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    e = torch.where(seen, torch.exp(x - torch.where(top > -math.inf, top, 0.0)), 0.0)
    return e / torch.where(seen.any(-1, keepdim=True), e.sum(-1, keepdim=True), 1.0)


def _attend(case, s):
    kh, hd, ps = case["kv_heads"], case["head_dim"], case["page_size"]
    group = case["q_heads"] // kh
    q, out, at = s["q"].view(-1, kh, group, hd), [], 0
    for i, a, c in s["taking"]:
        page = s["tables"][i, :-(-(a + c) // ps)].long()
        k = _rows_k(s["kc"][page]).transpose(0, 1).reshape(kh, -1, hd).float()      # [kv_heads, slots, head_dim]
        v = _rows_v(s["vc"][page]).transpose(0, 1).reshape(kh, -1, hd).float()
        rows = q[at:at + c].permute(1, 2, 0, 3).reshape(kh, group * c, hd)
        x = torch.matmul(rows, k.transpose(-1, -2).contiguous()) / math.sqrt(hd)
        seen = torch.arange(k.shape[1], device=GPU) <= a + torch.arange(c, device=GPU).unsqueeze(-1)
        seen = seen.repeat(group, 1).unsqueeze(0)
        v = torch.where(seen[0, -1].unsqueeze(-1), v, 0.0)
        p = _softmax(x, seen)
        out.append(torch.matmul(p, v).view(kh, group, c, hd).permute(2, 0, 1, 3).reshape(c, -1))
        at += c
    return torch.cat(out)


def _sparse(case, s):
    kh, hd, ps, budget = case["kv_heads"], case["head_dim"], case["page_size"], case["budget"]
    group = case["q_heads"] // kh
    q, pages, out, at = s["q"].view(-1, kh, group, hd), [], [], 0
    for i, a, c in s["taking"]:
        table = s["tables"][i, :-(-(a + c) // ps)].long()
        rows = q[at:at + c]
        # the most that a key of the page can score, summed over the group: choices are borders, hence 64 bits
        up, down = rows.double().clamp(min=0).sum(2), rows.double().clamp(max=0).sum(2)         # [c, kv_heads, head_dim]
        b = s["bounds"][table].double().permute(1, 0, 2, 3)                                     # [kv_heads, pages, 2, head_dim]
        score = (up.unsqueeze(2) * b[:, :, 1] + down.unsqueeze(2) * b[:, :, 0]).sum(-1)         # [c, kv_heads, pages]
        page = torch.arange(table.numel(), device=GPU)
        last = ((a + torch.arange(c, device=GPU)) // ps).view(-1, 1, 1)
        held = (page < case["sinks"]) | (page > last - case["recent"])
        key = torch.where(page <= last, torch.where(held, math.inf, score), -math.inf)
        order = key.sort(dim=-1, descending=True, stable=True).indices[..., :budget]
        order = torch.where(order <= last, order, table.numel()).sort(-1).values
        order = torch.cat([order, order.new_full((c, kh, budget - order.shape[-1]), table.numel())], -1)
        there = order < table.numel()
        pages.append(torch.where(there, order, NONE))
        # attention over the slots of those pages
        physical = table[torch.where(there, order, 0)]                                          # [c, kv_heads, budget]
        head = torch.arange(kh, device=GPU).view(1, -1, 1)
        k = _rows_k(s["kc"][physical, head]).flatten(2, 3).float()                             # [c, kv_heads, slots, head_dim]
        v = _rows_v(s["vc"][physical, head]).flatten(2, 3).float()
        position = (order.unsqueeze(-1) * ps + torch.arange(ps, device=GPU)).flatten(-2)
        seen = (there.unsqueeze(-1).expand(-1, -1, -1, ps).flatten(-2)
                & (position <= a + torch.arange(c, device=GPU).view(-1, 1, 1))).unsqueeze(2)
        x = torch.matmul(rows, k.transpose(-1, -2).contiguous()) / math.sqrt(hd)
        p = _softmax(x, seen)
        out.append(torch.matmul(p, torch.where(seen.transpose(-1, -2), v, 0.0)).reshape(c, -1))
        at += c
    return dict(pages=torch.cat(pages).to(torch.int32), out=torch.cat(out))


# ------------------------------------------------------------------- in 64 bits
def _one_row(cache, table, head, n, ps, values):
    """f64 rows [n, head_dim] of one request and KV head, slot by slot as the layouts say."""
    p = torch.arange(n, device=GPU)
    page, at = table[p // ps].long(), p % ps
    if values:
        return cache[page, head, at // 8, :, at % 8].double()
    return cache[page, head, at // 16, :, at % 16].reshape(n, -1).double()


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    kind = case["kind"]
    if kind == "plan":
        return None
    kh, qh, hd, ps = (case[n] for n in ("kv_heads", "q_heads", "head_dim", "page_size"))
    if kind == "store":
        kc, vc = s["kc"].cpu().numpy().astype(np.float64), s["vc"].cpu().numpy().astype(np.float64)
        rows = [s[n].cpu().numpy().reshape(-1, kh, hd) for n in ("k", "v")]
        for r, slot in enumerate(s["slots"].tolist()):
            kc[slot // ps, :, slot % ps // 16, :, slot % 16] = rows[0][r].astype(np.float16).reshape(kh, -1, 8)
            vc[slot // ps, :, slot % ps // 8, :, slot % 8] = rows[1][r].astype(np.float16)
        got = dict(kc=kc, vc=vc)
        if "bounds" in s:
            b = got["bounds"] = s["bounds"].cpu().numpy().astype(np.float64)
            tables = s["tables"].cpu().numpy()
            for i, a, c in s["taking"]:
                for col in range(a // ps, (a + c - 1) // ps + 1):
                    x = kc[tables[i, col]].swapaxes(2, 3).reshape(kh, ps, hd)[:, :min(ps, a + c - col * ps)]
                    b[tables[i, col]] = np.stack([x.min(1), x.max(1)], 1)
        return got
    if sum(a + c for _, a, c in s["taking"]) * kh > 4_000_000:
        return None if kind == "attend" else dict(pages=None, out=None)
    q = s["q"].double().view(-1, kh, qh // kh, hd)
    out = torch.zeros_like(q)
    at = 0
    for i, a, c in s["taking"]:
        n = a + c
        for h in range(kh):
            k, v = (_one_row(s[name], s["tables"][i], h, n, ps, values) for name, values in (("kc", False), ("vc", True)))
            hidden = torch.ones(c, n, device=GPU, dtype=torch.bool).triu(a + 1)
            if kind == "sparse":
                bounds = s["bounds"][s["tables"][i, :-(-n // ps)].long(), h].double()
                for t in range(c):
                    last = (a + t) // ps
                    reach = sum(torch.maximum(q[at + t, h, j] * bounds[:, 0], q[at + t, h, j] * bounds[:, 1]) for j in range(qh // kh)).sum(-1)
                    keep = {p for p in range(last + 1) if p < case["sinks"] or p > last - case["recent"]}
                    ranked = sorted(range(last + 1), key=lambda p, reach=reach.tolist(): (p not in keep, -reach[p] if p not in keep else 0.0, p))
                    chosen = torch.zeros(-(-n // ps), device=GPU, dtype=torch.bool)
                    chosen[ranked[:case["budget"]]] = True
                    hidden[t] |= ~chosen.repeat_interleave(ps)[:n]
            for j in range(qh // kh):
                p = torch.softmax((q[at:at + c, h, j] @ k.T / math.sqrt(hd)).masked_fill(hidden, -math.inf), -1)
                out[at:at + c, h, j] = p @ v
        at += c
    out = out.view(-1, qh * hd)
    return out if kind == "attend" else dict(pages=None, out=out)
