"""The paged KV cache's host side on the CPU: the restatement's own consistency, geometry and
argument checks (a stand-in for the HIP runtime counts launches, so that a refused call is
seen to launch nothing), and the Python class's pushes."""
import ctypes as C
import subprocess

import numpy as np
import pytest

import pagedref as ref
from test_kv4 import TWO_DEVICES, roomy  # noqa: F401  (fixture)
from test_refused_memory import HIP_INCLUDE, child, fake  # noqa: F401  (fixture)
from voxgen_amd import abi


@pytest.mark.parametrize("hd,ps", [(64, 16), (128, 32), (256, 128)])
def test_pages_hold_what_was_put(hd, ps):
    rng = np.random.default_rng(1)
    for is_v in (False, True):
        cache = rng.standard_normal((ref.v_shape if is_v else ref.k_shape)(2, 3, ps, 2, hd)).astype(np.float16)
        other = cache[0].copy(), cache[1, 0].copy()
        x = rng.standard_normal((ps, hd)).astype(np.float16)
        for s in rng.permutation(ps):
            ref.put(cache, 1, 2, 1, int(s), x[s], is_v)
        assert np.array_equal(ref.page_rows(cache, 1, 2, 1, is_v), x)
        assert np.array_equal(cache[0], other[0]) and np.array_equal(cache[1, 0], other[1])
        flat = cache.reshape(2, 3, 2, -1)[1, 2, 1]                   # the layouts, word for word
        for s in (0, 7, ps - 1):
            for d in (0, 9, hd - 1):
                at = (s // 8 * hd + d) * 8 + s % 8 if is_v else ((s // 16 * (hd // 8) + d // 8) * 16 + s % 16) * 8 + d % 8
                assert flat[at] == x[s, d]


def test_plans_of_the_restatement():
    tables = np.full((3, 4), ref.NONE, np.uint32)
    tables[0, 0], tables[1, :2] = 7, [3, 9]
    pool = np.array([3, 5, 6, 8, 0, 0, 0, 0, 0, 0, 0], np.uint32)
    got = ref.plan(np.array([16, 20, 0], np.uint32), np.array([2, 13, 17], np.uint32), tables, pool, 10, 16, 40, 20)
    assert list(got["granted"]) == [2, 13, 0] and got["pages"] == 2 and got["rows"] == 32
    assert got["tables"][0, 1] == 8 and got["tables"][1, 2] == 6     # the pool's last first
    assert list(got["slots"][:3]) == [128, 129, 9 * 16 + 4] and (got["slots"][15:] == ref.NONE).all()


def test_sizes():
    lib = abi.load()
    geom = lambda *g: abi.PagedGeom(*g)  # noqa: E731
    size = lambda *g: lib.vx_paged_cache_bytes(C.byref(geom(*g)))  # noqa: E731
    assert size(28, 100, 32, 2, 128) == 28 * 100 * 32 * 2 * 128 * 2
    assert lib.vx_paged_bounds_bytes(C.byref(geom(28, 100, 32, 2, 128))) == 28 * 100 * 2 * 2 * 128 * 2
    for bad in ((0, 1, 16, 1, 64), (1, 0, 16, 1, 64), (1, 1, 16, 0, 64), (1, 1, 8, 1, 64), (1, 1, 48, 1, 64), (1, 1, 512, 1, 64),
                (1, 1, 0, 1, 64), (1, 1, 16, 1, 96), (65536, 1, 16, 1, 64), (1, 1, 16, 65536, 64), (1, 1 << 28, 16, 1, 64),
                (1, 1 << 24, 256, 1, 64), (65535, 1 << 20, 256, 1, 256), (1, 1 << 23, 256, 64, 64)):
        assert size(*bad) == 0 and lib.vx_paged_bounds_bytes(C.byref(geom(*bad))) == 0, bad
    assert lib.vx_paged_cache_bytes(None) == 0 and lib.vx_paged_plan_bytes(None) == 0
    plan = lambda **kw: lib.vx_paged_plan_bytes(C.byref(abi.PagedBatch(geom(1, 100, 16, 2, 128), *dict(  # noqa: E731
        requests=4, table_width=10, max_rows=8, max_count=2, q_heads=16, **kw).values() if not kw else dict(
        dict(requests=4, table_width=10, max_rows=8, max_count=2, q_heads=16), **kw).values())))
    assert plan() >= 4 * (8 + 3 * 8 + 4)
    for bad in (dict(requests=0), dict(table_width=0), dict(max_rows=0), dict(max_count=0), dict(q_heads=0), dict(q_heads=3),
                dict(requests=4097), dict(table_width=(1 << 24) + 1), dict(max_count=9), dict(q_heads=2050),
                dict(max_rows=1 << 20), dict(max_rows=4294967295)):
        assert plan(**bad) == 0, bad


CALLS = """
from voxgen_amd.paged import PagedCache
lib = abi.load()
def kernels():
    return launches("k_paged")
G = dict(layers=2, pages=30, page_size=16, kv_heads=2, head_dim=128)
B = dict(requests=3, table_width=200, max_rows=6, max_count=4, q_heads=8)
def batch(**kw):
    return abi.PagedBatch(abi.PagedGeom(*[kw.get(n, v) for n, v in G.items()]), *[kw.get(n, v) for n, v in B.items()])
def store_push(**kw):
    return abi.PagedStorePush(batch(**kw), *[kw.get(n, v) for n, v in dict(layer=0, k_stride=256, v_stride=256, k_base=0, v_base=0).items()])
def attn_push(**kw):
    return abi.PagedAttentionPush(batch(**kw), *[kw.get(n, v) for n, v in dict(
        layer=0, q_stride=1024, out_stride=1024, q_base=0, out_base=0, budget=0).items()])
def select_push(**kw):
    return abi.PagedSelectPush(batch(**kw), *[kw.get(n, v) for n, v in dict(layer=0, q_stride=1024, q_base=0, budget=5, sinks=1, recent=2).items()])
cache = lib.vx_paged_cache_bytes(batch().geom)
kc, vc, bounds = ctx.alloc(cache), ctx.alloc(cache), ctx.alloc(lib.vx_paged_bounds_bytes(batch().geom))
k, v = ctx.alloc(6 * 256 * 4), ctx.alloc(6 * 256 * 4)
q, out = ctx.alloc(6 * 1024 * 4), ctx.alloc(6 * 1024 * 4)
lengths, counts, keep = ctx.alloc(12), ctx.alloc(12), ctx.alloc(12)
tables, pool, plan = ctx.alloc(2400), ctx.alloc(31 * 4), ctx.alloc(lib.vx_paged_plan_bytes(batch()))
selected = ctx.alloc(6 * 2 * 5 * 4)
scratch = ctx.alloc(1 << 26)
small = ctx.alloc(4)
H = lambda b: b.handle if b is not None else None
def reset(b=None, lengths=lengths, tables=tables, pool=pool):
    return refused(abi.call, "vx_paged_reset", ctx.handle, H(lengths), H(tables), H(pool), b or batch())
def make(b=None, lengths=lengths, counts=counts, tables=tables, pool=pool, plan=plan):
    return refused(abi.call, "vx_paged_plan", ctx.handle, H(lengths), H(counts), H(tables), H(pool), H(plan), b or batch())
def advance(b=None, plan=plan, lengths=lengths, pool=pool):
    return refused(abi.call, "vx_paged_advance", ctx.handle, H(plan), H(lengths), H(pool), b or batch())
def cut(b=None, keep=keep, lengths=lengths, tables=tables, pool=pool):
    return refused(abi.call, "vx_paged_cut", ctx.handle, H(keep), H(lengths), H(tables), H(pool), b or batch())
def store(pc=None, k=k, v=v, kc=kc, vc=vc, bounds=bounds, plan=plan):
    return refused(abi.call, "vx_paged_store", ctx.handle, H(k), H(v), H(kc), H(vc), H(bounds), H(plan), pc or store_push())
def attn(pc=None, q=q, kc=kc, vc=vc, out=out, tables=tables, plan=plan, selected=None, scratch=scratch):
    return refused(abi.call, "vx_paged_attention", ctx.handle, H(q), H(kc), H(vc), H(out), H(tables), H(plan), H(selected), H(scratch), pc or attn_push())
def sparse(pc=None, **kw):
    return attn(pc or attn_push(budget=5), **dict(dict(selected=selected), **kw))
def select(pc=None, q=q, bounds=bounds, tables=tables, plan=plan, selected=selected, scratch=scratch):
    return refused(abi.call, "vx_paged_select", ctx.handle, H(q), H(bounds), H(tables), H(plan), H(selected), H(scratch), pc or select_push())
"""


def test_calls_are_refused_before_a_launch(fake):  # noqa: F811
    child(fake, CALLS + """
bad = (("VX_ERR_INVALID_ARG", dict(layers=0)), ("VX_ERR_INVALID_ARG", dict(pages=0)), ("VX_ERR_INVALID_ARG", dict(requests=0)),
       ("VX_ERR_INVALID_ARG", dict(max_rows=0)), ("VX_ERR_INVALID_ARG", dict(max_count=0)), ("VX_ERR_INVALID_ARG", dict(table_width=0)),
       ("VX_ERR_UNSUPPORTED", dict(page_size=24)), ("VX_ERR_UNSUPPORTED", dict(page_size=8)), ("VX_ERR_UNSUPPORTED", dict(head_dim=32)),
       ("VX_ERR_UNSUPPORTED", dict(requests=4097)), ("VX_ERR_SHAPE", dict(max_count=7)), ("VX_ERR_SHAPE", dict(q_heads=3)),
       ("VX_ERR_SHAPE", dict(q_heads=0)), ("VX_ERR_UNSUPPORTED", dict(q_heads=2050)), ("VX_ERR_UNSUPPORTED", dict(max_rows=1 << 30)))
for want, kw in bad:
    for call in (reset, make, advance, cut):
        assert call(batch(**kw)) == want, (call, kw)
    assert store(store_push(**kw)) == want and attn(attn_push(**kw)) == want and select(select_push(**kw)) == want, kw
    assert lib.vx_paged_attention_scratch_bytes(attn_push(**kw)) == 0 and lib.vx_paged_select_scratch_bytes(select_push(**kw)) == 0
for call, names in ((reset, "lengths tables pool"), (make, "lengths counts tables pool plan"), (advance, "plan lengths pool"),
                    (cut, "keep lengths tables pool"), (store, "k v kc vc plan"), (attn, "q kc vc out tables plan scratch"),
                    (sparse, "q kc vc out tables plan selected"), (select, "q bounds tables plan selected scratch")):
    for name in names.split():
        assert call(**{name: small}) == "VX_ERR_BOUNDS" or (call, name) == (sparse, "scratch"), (call, name)
        assert call(**{name: None}) == "VX_ERR_INVALID_ARG", (call, name)
assert store(bounds=small) == "VX_ERR_BOUNDS"
for call, push in ((store, store_push), (attn, attn_push), (select, select_push)):
    assert call(push(layer=2)) == "VX_ERR_SHAPE"
    assert call(push(layers=3)) == "VX_ERR_BOUNDS" and call(push(pages=31)) == "VX_ERR_BOUNDS" and call(push(max_rows=7)) == "VX_ERR_BOUNDS"
for call, push, strides in ((store, store_push, (("k_stride", 256), ("v_stride", 256))),
                            (attn, attn_push, (("q_stride", 1024), ("out_stride", 1024))), (select, select_push, (("q_stride", 1024),))):
    for name, n in strides:
        base = name.replace("stride", "base")
        assert call(push(**{name: n - 1})) == "VX_ERR_SHAPE" and call(push(**{name: 0})) == "VX_ERR_SHAPE"
        assert call(push(**{name: n + 1})) == "VX_ERR_BOUNDS" and call(push(**{base: 1})) == "VX_ERR_BOUNDS"
        assert call(push(**{name: 4294967295, base: 4294967295})) == "VX_ERR_BOUNDS"
assert attn(attn_push(budget=5)) == "VX_ERR_INVALID_ARG" and attn(selected=selected) == "VX_ERR_INVALID_ARG"
assert sparse(attn_push(budget=(1 << 24) + 1)) == "VX_ERR_UNSUPPORTED" and sparse(attn_push(budget=6)) == "VX_ERR_BOUNDS"
for want, kw in (("VX_ERR_INVALID_ARG", dict(budget=0)), ("VX_ERR_INVALID_ARG", dict(recent=0)), ("VX_ERR_UNSUPPORTED", dict(budget=(1 << 24) + 1)),
                 ("VX_ERR_SHAPE", dict(sinks=4)), ("VX_ERR_SHAPE", dict(sinks=4294967295)), ("VX_ERR_SHAPE", dict(recent=4294967295)),
                 ("VX_ERR_BOUNDS", dict(budget=6))):
    assert select(select_push(**kw)) == want, kw
for name, args in (("vx_paged_reset", 3), ("vx_paged_plan", 5), ("vx_paged_advance", 3), ("vx_paged_cut", 4)):
    some = [H(scratch)] * args
    assert refused(abi.call, name, None, *some, batch()) == "VX_ERR_INVALID_ARG"
    assert refused(abi.call, name, ctx.handle, *some, None) == "VX_ERR_INVALID_ARG"
assert kernels() == 0
for call in (reset, make, advance, cut, store, select):
    assert call() == "VX_OK", call
assert store(bounds=None) == "VX_OK" and attn() == "VX_OK" and sparse() == "VX_OK"
assert kernels() >= 9
""")


def test_a_written_buffer_is_bound_once(fake):  # noqa: F811
    """Every pair of a buffer that a call writes and another of the call; q and out side by side in one buffer are two."""
    child(fake, CALLS + """
one = ctx.alloc(1 << 26)
def pairs(call, written, read, but=()):
    for a in written.split():
        for b in [n for n in written.split() if n != a] + read.split():
            if {a, b} != set(but):
                assert call(**{a: one, b: one}) == "VX_ERR_INVALID_ARG", (call, a, b)
pairs(reset, "lengths tables pool", "")
pairs(make, "tables plan", "lengths counts pool")
pairs(advance, "lengths pool", "plan")
pairs(cut, "lengths tables pool", "keep")
pairs(store, "kc vc bounds", "k v plan")
pairs(attn, "out scratch", "q kc vc tables plan", ("q", "out"))
pairs(sparse, "out scratch", "q kc vc tables plan selected", ("q", "out"))
pairs(select, "selected scratch", "q bounds tables plan")
assert kernels() == 0
both = ctx.alloc(18 * 1024 * 4)
for ok, v in ((True, (2048, 2048, 0, 1024)), (True, (1024, 1024, 0, 6 * 1024)), (True, (1024, 2048, 0, 6 * 1024)),
              (False, (2048, 2048, 0, 1023)), (False, (1024, 1024, 0, 0)), (False, (1024, 1024, 0, 1024)), (False, (1024, 2048, 0, 1024))):
    got = attn(attn_push(**dict(zip(("q_stride", "out_stride", "q_base", "out_base"), v))), q=both, out=both)
    assert got == ("VX_OK" if ok else "VX_ERR_INVALID_ARG"), v
assert store(k=one, v=one) == "VX_OK" and make(lengths=one, counts=one) == "VX_OK"      # read twice
""")


def test_python_class(fake):  # noqa: F811
    child(fake, CALLS + """
assert refused(PagedCache, ctx, 1, 30, 24, 2, 64, 1, 4, 1, 2) == "VX_ERR_SHAPE"
assert refused(PagedCache, ctx, 1, 30, 16, 2, 64, 1, 4, 1, 3) == "VX_ERR_SHAPE"
c = PagedCache(ctx, 2, 30, 16, 2, 128, 3, 10, 6, 8, max_count=4, bounds=True)
assert c.nbytes == 2 * cache
assert c.plan_layout() == dict(slots=(32, 6), requests=(56, 6), positions=(80, 6), granted=(104, 3))
sel = c.selection(5)
assert sel.nbytes == 6 * 2 * 5 * 4
def step():
    c.plan()
    c.store(1, k, v)
    c.attention(1, q, out)
    c.select(1, q, sel, 5, sinks=1, recent=2)
    c.attention(1, q, out, selected=sel, budget=5)
    c.advance()
    c.cut(keep)
step()
before = len(c._pushes)
step()
assert len(c._pushes) == before
assert refused(c.store, 2, k, v) == "VX_ERR_SHAPE" and refused(c.attention, 0, q, out, 1025) == "VX_ERR_BOUNDS"
bare = PagedCache(ctx, 1, 30, 16, 2, 128, 3, 10, 6, 8)
assert bare.bounds is None and refused(bare.select, 0, q, sel, 5) == "VX_ERR_STATE"
assert refused(c.select, 0, q, sel, 11) == "VX_ERR_BOUNDS" and refused(c.select, 0, q, c.selection(11), 11) == "VX_OK"
# scratch that is refused leaves the cache as it was
big = PagedCache(ctx, 1, 30, 16, 2, 128, 3, 200, 1024, 8)
qs, outs = ctx.alloc(1024 * 1024 * 4), ctx.alloc(1024 * 1024 * 4)
refuse(4096, 1 << 40)
assert refused(big.attention, 0, qs, outs) == "VX_ERR_OOM" and big._scratch is None
refuse(0, 0)
assert refused(big.attention, 0, qs, outs) == "VX_OK"
""")


def test_scratch_of_calls_that_divide_nothing(fake):  # noqa: F811
    """Tables of a few chunks: no partial sums, but a size that tells such a call from one that is not valid."""
    child(fake, CALLS + """
for kw in (dict(table_width=1), dict(table_width=96), dict(table_width=200, budget=5)):
    need = lib.vx_paged_attention_scratch_bytes(attn_push(**kw))
    assert need == 16, (kw, need)
few = dict(table_width=10)
p = ctx.alloc(lib.vx_paged_plan_bytes(batch(**few)))
assert attn(attn_push(**few), plan=p, scratch=small) == "VX_ERR_BOUNDS"
assert attn(attn_push(**few), plan=p, scratch=None) == "VX_ERR_INVALID_ARG"
assert attn(attn_push(**few), plan=p, scratch=ctx.alloc(16)) == "VX_OK"
assert lib.vx_paged_attention_scratch_bytes(attn_push()) > 16
""")


def test_scratch_is_what_the_kernels_reach(fake):  # noqa: F811
    """Parts of a step: never more than its share of workgroups makes, whatever lengths the plan finds (the kernel's
    arithmetic, here with the sizes that a batch fixes)."""
    rng = np.random.default_rng(5)
    for _ in range(300):
        kv = int(rng.choice([1, 2, 3, 8]))
        log2 = int(rng.choice([7, 8, 9, 10]))
        share = -(-(1 << log2) // kv)
        n = int(rng.integers(1, 200))
        chunks, tiles = rng.integers(1, 1 << int(rng.integers(1, 14)), n), rng.integers(1, 1 << int(rng.integers(1, 10)), n)
        per = max(int((int((chunks * tiles).sum()) * kv + (1 << log2) - 1) >> log2), int(rng.choice([4, 8, 16, 48])))
        splits = np.minimum(-(-chunks // per), 256)
        by = -(-chunks // splits)
        splits = -(-chunks // by)
        assert (tiles * splits).sum() <= tiles.sum() + share
        assert (tiles * splits)[splits > 1].sum() <= 2 * share and tiles[splits > 1].sum() <= share


def test_launches_are_on_the_contexts_device(fake, tmp_path):  # noqa: F811
    """With another device current, every call launches on its context's, and leaves the caller's current."""
    source, library = tmp_path / "two.c", tmp_path / "libtwo.so"
    source.write_text(TWO_DEVICES)
    subprocess.run(["gcc", "-std=gnu11", "-O1", "-w", "-shared", "-fPIC", "-I", str(HIP_INCLUDE), str(source),
                    "-Wl,--no-as-needed", str(fake),
                    f"-Wl,-rpath,{fake.parent}", "-o", str(library)], check=True)
    child(library, CALLS + """
now = C.c_int()
for call in (reset, make, advance, cut, store, attn, sparse, select):
    fake.hipSetDevice(1)
    assert call() == "VX_OK"
    fake.hipGetDevice(C.byref(now))
    assert now.value == 1 and fake.astray_launches() == 0
""")


def test_grids_are_within_limits(roomy):  # noqa: F811
    """The largest sizes that a batch may have launch grids below 2^32 threads (the stand-in refuses none; the launch
    wrapper's own arithmetic is what is checked: calls return, with buffers of any size)."""
    child(roomy, CALLS + """
for kw in (dict(max_rows=1 << 22, max_count=1 << 22, q_heads=1, kv_heads=1, pages=1 << 20, table_width=1 << 20),
           dict(max_rows=1 << 19, max_count=1, q_heads=8, kv_heads=8, pages=1 << 16, table_width=1 << 16, requests=4096),
           dict(max_rows=64, max_count=64, q_heads=65535, kv_heads=65535, pages=64, requests=64)):
    b = batch(**kw)
    g = b.geom
    need = lib.vx_paged_plan_bytes(b)
    assert need, (kw, lib.vx_last_error())
    wide = b.q_heads * g.head_dim
    plan = ctx.alloc(need)
    assert make(b, plan=plan, lengths=ctx.alloc(4 * b.requests), counts=ctx.alloc(4 * b.requests),
                tables=ctx.alloc(4 * b.requests * b.table_width), pool=ctx.alloc(4 * (g.pages + 1))) == "VX_OK"
    pc = attn_push(q_stride=wide, out_stride=wide, **kw)
    rows = b.max_rows * wide * 4
    big = [ctx.alloc(lib.vx_paged_cache_bytes(g)) for _ in range(2)]
    tab = ctx.alloc(4 * b.requests * b.table_width)
    assert attn(pc, q=ctx.alloc(rows), out=ctx.alloc(rows), kc=big[0], vc=big[1], tables=tab, plan=plan,
                scratch=ctx.alloc(lib.vx_paged_attention_scratch_bytes(pc))) == "VX_OK"
""")


def test_every_kernel_has_a_case_whose_values_are_compared(roomy):  # noqa: F811
    """The kernels of a call go by sizes. Each that the library holds is launched by a case of the GPU tests that compares
    values with the restatement, so that no change of a rule leaves a kernel untested, or one that no call reaches."""
    child(roomy, CALLS + """
import re
sys.path[:0] = ["tests", "oracle"]
import test_gpu_paged as gpu
from pathlib import Path
held = set(n.decode() for n in re.findall(rb"_ZN2vx[0-9A-Z_]*k_paged_[A-Za-z0-9_]+", Path(abi.LIB_PATH).read_bytes()) if b"device_stub" not in n)
names = set(re.search("k_paged_.*", n).group() for n in held)
names = set(n for n in names if not re.match("k_paged_(advance|cut|reset)", n))          # one each
assert len(names) > 40, names
def params(test):
    sets = [{}]
    for m in [m for m in test.pytestmark if m.name == "parametrize"]:
        keys = m.args[0].split(",")
        rows = [dict(zip(keys, v if len(keys) > 1 else (v,))) for v in m.args[1]]
        sets = [dict(s, **r) for s in sets for r in rows]
    return sets
big = {n: ctx.alloc(1 << 36) for n in ("a", "b", "c", "d", "e", "f", "g")}
def step(heads, page_size, lengths, counts, pages=None, budget=0, bounds=False, width=None):
    need = [-(-(a + c) // page_size) for a, c in zip(lengths, counts)]
    b = abi.PagedBatch(abi.PagedGeom(1, pages or sum(need) + 3, page_size, heads[1], heads[2]), len(lengths), width or max(need) + 2,
                       sum(counts), max(counts), heads[0])
    row, qrow = heads[1] * heads[2], heads[0] * heads[2]
    assert make(b, big["a"], big["b"], big["c"], big["d"], big["e"]) == "VX_OK"
    assert store(abi.PagedStorePush(b, 0, row, row, 0, 0), big["a"], big["b"], big["c"], big["d"], big["e"] if bounds else None, big["f"]) == "VX_OK"
    assert attn(abi.PagedAttentionPush(b, 0, qrow, qrow, 0, 0, budget), big["a"], big["b"], big["c"], big["d"], big["e"], big["f"],
                big["g"] if budget else None, ctx.alloc(1 << 36)) == "VX_OK"
    if budget:
        pc = abi.PagedSelectPush(b, 0, qrow, 0, budget, 0, 1)
        assert select(pc, big["a"], big["b"], big["c"], big["d"], big["e"], big["f"]) == "VX_OK"
for p in params(gpu.test_single_tokens):
    step(p["heads"], p["page_size"], [511, 300], [1, 1])
for p in params(gpu.test_single_tokens_over_long_caches):
    step(p["heads"], p["page_size"], p["lengths"], [1] * len(p["lengths"]))
for test in (gpu.test_several_tokens, gpu.test_prompts, gpu.test_layers_beyond_the_caches, gpu.test_store):
    for p in params(test):
        step(**p)
for p in params(gpu.test_selection):
    step(*[p[n] for n in ("heads", "page_size", "lengths", "counts")], budget=p["budget"], bounds=True)
for p in params(gpu.test_selection_by_the_width_of_tables):
    step((4, 2, p["hd"]), 16, [5, 5], [1, 1], pages=p["n"], budget=p["n"] // 8, width=p["n"])
for p in params(gpu.test_plan):
    step((4, 2, 64), p["page_size"], [5] * p["n"], [1] * p["n"])
missing = [n for n in names if not launches(n)]
assert not missing, missing
""")
