"""The 4-bit KV cache's host side on the CPU: the format's restatement, geometry and
argument checks (a stand-in for the HIP runtime counts launches, so that a refused call is
seen to launch nothing), and the Python class's pushes."""
import ctypes as C
import subprocess

import numpy as np
import pytest

import kv4ref
from test_refused_memory import HIP_INCLUDE, child, fake  # noqa: F401  (fixture)
from voxgen_amd import abi


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_format_round_trip_is_within_half_a_step(hd):
    """A value is off by at most half a step d, plus the roundings of o and of the value to f16
    (half a unit each: 2^-11 of the largest magnitude), plus 15 times d's own (2^-11 of d, or half
    of f16's least step 2^-24) at the far end."""
    rng = np.random.default_rng(hd)
    x = (rng.standard_normal((40, hd)) * np.exp(rng.uniform(-6, 6, (40, 1)))).astype(np.float32)
    c, d, o = kv4ref.encode(x)
    step = np.repeat(d.astype(np.float64), 32, -1)
    off = np.abs(kv4ref.values(c, d, o) - x)
    assert np.all(off <= step / 2 + 2 * 2.0 ** -11 * np.abs(x).max(-1, keepdims=True) + 15 * (step * 2.0 ** -11 + 2.0 ** -25))
    assert c.max() == 15 and c.min() == 0


@pytest.mark.parametrize("hd,context", [(64, 33), (128, 64), (256, 1)])
def test_blocks_hold_what_was_put(hd, context):
    rng = np.random.default_rng(1)
    for is_v in (False, True):
        cache = kv4ref.blank(2, 1, 2, hd, context, rng)
        other = cache[0].copy()
        x = rng.standard_normal((context, hd)).astype(np.float32)
        for s in rng.permutation(context):
            kv4ref.put(cache, (1, 0, 1), int(s), *(a[s] for a in kv4ref.encode(x)), is_v)
        assert np.array_equal(kv4ref.rows(cache, (1, 0, 1), context, is_v), kv4ref.stored(x))
        assert np.array_equal(cache[0], other)


def test_cache_bytes():
    lib = abi.load()
    size = lambda *g: lib.vx_kv4_cache_bytes(C.byref(abi.Kv4Geom(*g)))  # noqa: E731
    assert size(28, 1, 2, 128, 8192) == 28 * 2 * 8192 * 80
    assert size(1, 3, 5, 64, 33) == 3 * 5 * 2 * 20 * 64          # whole blocks of 32 slots
    assert size(1, 1, 1, 256, 1) == 20 * 256
    for bad in ((0, 1, 1, 64, 1), (1, 0, 1, 64, 1), (1, 1, 0, 64, 1), (1, 1, 1, 64, 0), (1, 1, 1, 96, 1),
                (1, 1, 1, 0, 1), (1, 1, 1, 128, (1 << 28) + 1), (1, 65536, 1, 64, 1), (1, 256, 256, 64, 1),
                (65535, 65535, 1, 256, 1 << 28)):
        assert size(*bad) == 0, bad
    assert lib.vx_kv4_cache_bytes(None) == 0


REFUSALS = """
from voxgen_amd.kv4 import Kv4Cache
import ctypes as C
lib = abi.load()
def kernels():
    return launches("k_kv4")
def row_push(**kw):
    f = dict(layer=0, first_sequence=0, n_sequences=2, tokens=3, k_stride=256, v_stride=256, k_base=0, v_base=0)
    g = dict(layers=2, sequences=2, kv_heads=2, head_dim=128, context=40)
    for n, v in kw.items():
        (g if n in g else f)[n] = v
    return abi.Kv4RowsPush(abi.Kv4Geom(*g.values()), *f.values())
def attn_push(**kw):
    f = dict(layer=0, first_sequence=0, n_sequences=2, tokens=3, q_heads=8, q_stride=1024, out_stride=1024, q_base=0,
             out_base=0, decay=1.0)
    g = dict(layers=2, sequences=2, kv_heads=2, head_dim=128, context=40)
    for n, v in kw.items():
        (g if n in g else f)[n] = v
    return abi.Kv4AttentionPush(abi.Kv4Geom(*g.values()), *f.values())
def evict_push(**kw):
    f = dict(first_sequence=0, n_sequences=2, keep=20, sinks=2, recent=4)
    g = dict(layers=2, sequences=2, kv_heads=2, head_dim=128, context=40)
    for n, v in kw.items():
        (g if n in g else f)[n] = v
    return abi.Kv4EvictPush(abi.Kv4Geom(*g.values()), *f.values())
cache_bytes = 2 * 2 * 2 * 2 * 20 * 128
kc, vc = ctx.alloc(cache_bytes), ctx.alloc(cache_bytes)
rows = 6 * 256 * 4
k, v = ctx.alloc(rows), ctx.alloc(rows)
slots, pos = ctx.alloc(8), ctx.alloc(8)
table = 2 * 2 * 2 * 40 * 4
w, sp = ctx.alloc(table), ctx.alloc(table)
q, out = ctx.alloc(6 * 1024 * 4), ctx.alloc(6 * 1024 * 4)
small = ctx.alloc(4)
H = lambda b: b.handle if b is not None else None
def store(pc, k=k, v=v, kc=kc, vc=vc, slots=slots, pos=pos, sp=sp):
    return refused(abi.call, "vx_kv4_store", ctx.handle, H(k), H(v), H(kc), H(vc), H(slots), H(pos), H(sp), pc)
def load(pc, k=k, v=v, kc=kc, vc=vc, slots=slots):
    return refused(abi.call, "vx_kv4_load", ctx.handle, H(kc), H(vc), H(k), H(v), H(slots), pc)
def attn(pc, q=q, out=out, kc=kc, vc=vc, w=w, slots=slots, scratch=None):
    need = lib.vx_kv4_attention_scratch_bytes(pc, 1 if w is not None else 0)
    s = ctx.alloc(max(need, 4)) if scratch is None else scratch
    return refused(abi.call, "vx_kv4_attention", ctx.handle, H(q), H(kc), H(vc), H(out), H(w), H(slots), H(s), pc)
def select(pc, w=w, sp=sp, slots=slots, plan=None):
    p = plan or ctx.alloc(max(4, lib.vx_kv4_plan_bytes(pc)))
    return refused(abi.call, "vx_kv4_select", ctx.handle, H(w), H(sp), H(slots), H(p), pc)
def compact(pc, kc=kc, vc=vc, w=w, sp=sp, slots=slots, plan=None):
    p = plan or ctx.alloc(max(4, lib.vx_kv4_plan_bytes(pc)))
    return refused(abi.call, "vx_kv4_compact", ctx.handle, H(p), H(kc), H(vc), H(w), H(sp), H(slots), pc)
"""


def test_row_calls_are_refused_before_a_launch(fake):  # noqa: F811
    child(fake, REFUSALS + """
for call in (store, load):
    for want, kw in (("VX_ERR_INVALID_ARG", dict(tokens=0)), ("VX_ERR_INVALID_ARG", dict(n_sequences=0)),
                     ("VX_ERR_INVALID_ARG", dict(layers=0)), ("VX_ERR_SHAPE", dict(layer=2)),
                     ("VX_ERR_SHAPE", dict(first_sequence=2)), ("VX_ERR_SHAPE", dict(first_sequence=1)),
                     ("VX_ERR_SHAPE", dict(n_sequences=4294967295, first_sequence=1)),
                     ("VX_ERR_SHAPE", dict(tokens=41)), ("VX_ERR_SHAPE", dict(k_stride=255)),
                     ("VX_ERR_SHAPE", dict(v_stride=0)), ("VX_ERR_UNSUPPORTED", dict(head_dim=96)),
                     ("VX_ERR_BOUNDS", dict(k_stride=257)), ("VX_ERR_BOUNDS", dict(k_base=1)),
                     ("VX_ERR_BOUNDS", dict(v_base=4294967295, v_stride=4294967295)),
                     ("VX_ERR_BOUNDS", dict(tokens=4)), ("VX_ERR_BOUNDS", dict(layers=3)),
                     ("VX_ERR_BOUNDS", dict(context=65)), ("VX_ERR_BOUNDS", dict(sequences=3)),
                     ("VX_ERR_UNSUPPORTED", dict(context=1 << 29))):
        assert call(row_push(**kw)) == want, (call, kw)
    for want, kw in (("VX_ERR_INVALID_ARG", dict(kc=None)), ("VX_ERR_INVALID_ARG", dict(slots=None)),
                     ("VX_ERR_INVALID_ARG", dict(vc=kc)), ("VX_ERR_BOUNDS", dict(slots=small)),
                     ("VX_ERR_BOUNDS", dict(vc=small)), ("VX_ERR_BOUNDS", dict(v=small))):
        assert call(row_push(), **kw) == want, (call, kw)
assert store(row_push(), k=None) == "VX_ERR_INVALID_ARG"
assert store(row_push(), pos=small) == "VX_ERR_BOUNDS"
assert store(row_push(), sp=small) == "VX_ERR_BOUNDS"
assert load(row_push(), k=None, v=None) == "VX_ERR_INVALID_ARG"
adv = lambda *a: refused(abi.call, "vx_kv4_advance", ctx.handle, *a)
for a, want in (((H(slots), None, 0, 0, 1, 40), "VX_ERR_INVALID_ARG"), ((H(slots), None, 0, 2, 0, 40), "VX_ERR_INVALID_ARG"),
                ((H(slots), None, 0, 2, 1, 0), "VX_ERR_INVALID_ARG"), ((H(slots), None, 0, 2, 41, 40), "VX_ERR_SHAPE"),
                ((H(slots), None, 1, 2, 1, 40), "VX_ERR_BOUNDS"), ((None, None, 0, 2, 1, 40), "VX_ERR_INVALID_ARG"),
                ((H(slots), H(small), 0, 2, 1, 40), "VX_ERR_BOUNDS"), ((H(slots), H(slots), 0, 2, 1, 40), "VX_ERR_INVALID_ARG"),
                ((H(slots), None, 4294967295, 4294967295, 1, 40), "VX_ERR_BOUNDS")):
    assert adv(*a) == want, a
assert refused(abi.call, "vx_kv4_store", None, H(k), H(v), H(kc), H(vc), H(slots), None, None, row_push()) == "VX_ERR_INVALID_ARG"
assert refused(abi.call, "vx_kv4_store", ctx.handle, H(k), H(v), H(kc), H(vc), H(slots), None, None, None) == "VX_ERR_INVALID_ARG"
assert kernels() == 0
assert store(row_push()) == "VX_OK" and store(row_push(), pos=None, sp=None) == "VX_OK"
assert load(row_push()) == "VX_OK" and load(row_push(), k=None) == "VX_OK" and load(row_push(), v=None) == "VX_OK"
assert adv(H(slots), H(pos), 0, 2, 1, 40) == "VX_OK"
assert kernels() == 6
""")


def test_attention_is_refused_before_a_launch(fake):  # noqa: F811
    child(fake, REFUSALS + """
for want, kw in (("VX_ERR_INVALID_ARG", dict(tokens=0)), ("VX_ERR_SHAPE", dict(q_heads=7)), ("VX_ERR_SHAPE", dict(q_heads=0)),
                 ("VX_ERR_SHAPE", dict(layer=2)), ("VX_ERR_SHAPE", dict(first_sequence=1)), ("VX_ERR_SHAPE", dict(tokens=41)),
                 ("VX_ERR_SHAPE", dict(q_stride=1023)), ("VX_ERR_SHAPE", dict(out_stride=1)),
                 ("VX_ERR_BOUNDS", dict(q_base=1)), ("VX_ERR_BOUNDS", dict(out_base=1)), ("VX_ERR_BOUNDS", dict(tokens=4)),
                 ("VX_ERR_UNSUPPORTED", dict(head_dim=32)), ("VX_ERR_UNSUPPORTED", dict(q_heads=2050)),
                 ("VX_ERR_INVALID_ARG", dict(decay=-0.1)), ("VX_ERR_INVALID_ARG", dict(decay=1.5)),
                 ("VX_ERR_INVALID_ARG", dict(decay=float("nan"))), ("VX_ERR_BOUNDS", dict(context=65))):
    pc = attn_push(**kw)
    assert attn(pc) == want, kw
for want, kw in (("VX_ERR_INVALID_ARG", dict(q=None)), ("VX_ERR_INVALID_ARG", dict(out=None)),
                 ("VX_ERR_INVALID_ARG", dict(out=q)), ("VX_ERR_INVALID_ARG", dict(slots=None)),
                 ("VX_ERR_INVALID_ARG", dict(vc=kc)), ("VX_ERR_BOUNDS", dict(w=small)), ("VX_ERR_BOUNDS", dict(slots=small)),
                 ("VX_ERR_BOUNDS", dict(scratch=small)), ("VX_ERR_INVALID_ARG", dict(w=out)), ("VX_ERR_INVALID_ARG", dict(w=q))):
    assert attn(attn_push(), **kw) == want, kw
large = ctx.alloc(lib.vx_kv4_attention_scratch_bytes(attn_push(), 1) + 12 * 1024 * 4)
for name in ("q", "kc", "vc", "out", "w", "slots"):
    assert attn(attn_push(), **{name: large, "scratch": large}) == "VX_ERR_INVALID_ARG", name
assert kernels() == 0
both = ctx.alloc(12 * 1024 * 4)                      # q and out in one buffer, apart
assert attn(attn_push(out_base=6 * 1024), q=both, out=both) == "VX_OK"
assert attn(attn_push(out_base=6 * 1024 - 1), q=both, out=both) == "VX_ERR_INVALID_ARG"
assert attn(attn_push()) == "VX_OK" and attn(attn_push(), w=None) == "VX_OK"
for kw in (dict(tokens=0), dict(q_heads=3), dict(layer=2)):
    assert lib.vx_kv4_attention_scratch_bytes(attn_push(**kw), 1) == 0
assert lib.vx_kv4_attention_scratch_bytes(None, 0) == 0
""")


def test_eviction_is_refused_before_a_launch(fake):  # noqa: F811
    child(fake, REFUSALS + """
for call in (select, compact):
    for want, kw in (("VX_ERR_SHAPE", dict(keep=0)), ("VX_ERR_SHAPE", dict(keep=40)), ("VX_ERR_SHAPE", dict(sinks=17)),
                     ("VX_ERR_SHAPE", dict(recent=4294967295)), ("VX_ERR_INVALID_ARG", dict(n_sequences=0)),
                     ("VX_ERR_SHAPE", dict(first_sequence=1)), ("VX_ERR_UNSUPPORTED", dict(head_dim=100)),
                     ("VX_ERR_INVALID_ARG", dict(kv_heads=0)), ("VX_ERR_BOUNDS", dict(context=41)),
                     ("VX_ERR_BOUNDS", dict(layers=3))):
        assert call(evict_push(**kw)) == want, (call, kw)
    for want, kw in (("VX_ERR_BOUNDS", dict(plan=small)), ("VX_ERR_BOUNDS", dict(w=small)), ("VX_ERR_BOUNDS", dict(sp=small)),
                     ("VX_ERR_BOUNDS", dict(slots=small)), ("VX_ERR_INVALID_ARG", dict(slots=None))):
        assert call(evict_push(), **kw) == want, (call, kw)
assert select(evict_push(), w=None) == "VX_ERR_INVALID_ARG" and select(evict_push(), sp=None) == "VX_ERR_INVALID_ARG"
assert select(evict_push(), plan=w, w=w) == "VX_ERR_INVALID_ARG"
assert compact(evict_push(), kc=None) == "VX_ERR_INVALID_ARG" and compact(evict_push(), vc=None) == "VX_ERR_INVALID_ARG"
assert compact(evict_push(), vc=kc) == "VX_ERR_INVALID_ARG" and compact(evict_push(), sp=w) == "VX_ERR_INVALID_ARG"
assert kernels() == 0
assert select(evict_push()) == "VX_OK" and compact(evict_push()) == "VX_OK"
assert compact(evict_push(), kc=None, vc=None, w=None, sp=None) == "VX_OK"
assert kernels() == 3
assert lib.vx_kv4_plan_bytes(evict_push()) == 2 * 2 * 2 * 20 * 8
assert lib.vx_kv4_plan_bytes(evict_push(keep=33)) == 2 * 2 * 2 * 7 * 8
assert lib.vx_kv4_plan_bytes(None) == 0
""")


def test_a_written_buffer_is_bound_once(fake):  # noqa: F811
    """Every pair of a buffer that a call writes and another of the call; rows side by side in one buffer are two."""
    child(fake, REFUSALS + """
one = ctx.alloc(1 << 20)
def pairs(call, push, written, read, rows=()):
    for a in written:
        for b in [n for n in written if n != a] + list(read):
            if {a, b} != set(rows):
                assert call(push(), **{a: one, b: one}) == "VX_ERR_INVALID_ARG", (call, a, b)
pairs(store, row_push, ("kc", "vc", "sp"), ("k", "v", "slots", "pos"))
pairs(load, row_push, ("k", "v"), ("kc", "vc", "slots"), rows=("k", "v"))
scratch = ctx.alloc(1 << 20)
pairs(lambda pc, **kw: attn(pc, **dict(dict(scratch=scratch), **kw)), attn_push, ("out", "w", "scratch"),
      ("q", "kc", "vc", "slots"), rows=("q", "out"))
pairs(select, evict_push, ("plan",), ("w", "sp", "slots"))
pairs(compact, evict_push, ("kc", "vc", "w", "sp", "slots"), ("plan",))
assert kernels() == 0
# k and v, or q and out, in rows of one buffer: of one stride side by side, or one behind the other
def row_pairs(call, push, width, rows, names):
    buf, launched = ctx.alloc(3 * rows * width * 4), kernels()
    s, b = [n + "_stride" for n in names], [n + "_base" for n in names]
    def run(*v):
        return call(push(**dict(zip(s + b, v))), **{n: buf for n in names})
    w = width
    for ok, v in ((True, (2 * w, 2 * w, 0, w)), (True, (2 * w, 2 * w, w, 0)), (True, (2 * w + 4, 2 * w + 4, 3, w + 5)),
                  (True, (w, w, 0, rows * w)), (True, (w, 2 * w, 0, rows * w)), (True, (2 * w, 2 * w, 0, 3 * w)),
                  (False, (2 * w, 2 * w, 0, w - 1)), (False, (2 * w, 2 * w, 0, w + 1)), (False, (2 * w, 2 * w, 1, 0)),
                  (False, (2 * w, 2 * w, 2 * w, 0)), (False, (w, w, 0, 0)), (False, (w, w, 0, w)),
                  (False, (w, w, 0, rows * w - 1)), (False, (w, 2 * w, 0, w))):
        assert run(*v) == ("VX_OK" if ok else "VX_ERR_INVALID_ARG"), (call, v)
    return kernels() - launched
assert row_pairs(load, row_push, 256, 6, ("k", "v")) == 6
row_pairs(lambda pc, **kw: attn(pc, scratch=scratch, w=None, **kw), attn_push, 1024, 6, ("q", "out"))
assert store(row_push(), k=one, v=one) == "VX_OK" and store(row_push(), pos=slots) == "VX_OK"     # read twice
""")


def test_python_class_checks_and_keeps_its_pushes(fake):  # noqa: F811
    child(fake, REFUSALS + """
assert refused(Kv4Cache, ctx, 1, 1, 1, 96, 8) == "VX_ERR_SHAPE"
c = Kv4Cache(ctx, 2, 2, 2, 128, 40, track=True)
assert c.nbytes == 2 * cache_bytes
c.store(1, k, v, tokens=3)
c.load(1, k, None, tokens=3)
c.attention(1, q, out, 8, tokens=3)
c.advance(3)
plan = c.plan(20)
assert plan.nbytes == 2 * 2 * 2 * 20 * 8 and c.plan_moves(33) == 7
c.evict(plan, 20, sinks=1, recent=2)
assert refused(c.store, 2, k, v) == "VX_ERR_SHAPE"
assert refused(c.attention, 0, q, out, 8, 4) == "VX_ERR_BOUNDS"
bare = Kv4Cache(ctx, 1, 1, 1, 64, 8)
assert refused(bare.select, plan, 4) == "VX_ERR_STATE"
before = len(c._pushes)
c.store(1, k, v, tokens=3)
assert len(c._pushes) == before
""")


def test_scratch_that_grows_stays_bounded(fake):  # noqa: F811
    """Calls of every length: the scratches that are kept for graphs are together no larger than the one in use, and that
    is at most twice what the largest call needs; exactly that where no more can be had, and nothing is lost to a call
    that fails for want of memory."""
    child(fake, REFUSALS + """
c = Kv4Cache(ctx, 1, 1, 2, 128, 2048, track=True)
q, out = ctx.alloc(2048 * 2048 * 4), ctx.alloc(2048 * 2048 * 4)
push = lambda t: attn_push(layers=1, sequences=1, context=2048, n_sequences=1, tokens=t, q_heads=16, q_stride=2048, out_stride=2048)
need = lambda t: lib.vx_kv4_attention_scratch_bytes(push(t), 1)
largest = 0
for t in range(20, 1500):
    c.attention(0, q, out, 16, tokens=t)
    largest = max(largest, need(t))
    assert largest <= c._scratch.nbytes <= 2 * largest
    assert sum(b.nbytes for b in c._outgrown) <= c._scratch.nbytes
kept = [b.handle for b in c._outgrown]
now = c._scratch.nbytes
t = next(t for t in range(1500, 2049) if need(t) > now)
refuse(need(t), 1 << 40)
assert refused(c.attention, 0, q, out, 16, t) == "VX_ERR_OOM"
assert c._scratch.nbytes == now and [b.handle for b in c._outgrown] == kept
refuse(2 * now, 1 << 40)
assert refused(c.attention, 0, q, out, 16, t) == "VX_OK" and c._scratch.nbytes == need(t)
""")


TWO_DEVICES = """
#define __HIP_PLATFORM_AMD__ 1
#include <hip/hip_runtime_api.h>
static int now, astray;
int astray_launches(void) { return astray; }
hipError_t hipGetDevice(int *d) { *d = now; return hipSuccess; }
hipError_t hipSetDevice(int d) { now = d; return hipSuccess; }
hipError_t hipLaunchKernel(const void *fn, dim3 g, dim3 b, void **a, size_t s, hipStream_t st) {
    astray += now != 0;
    return hipSuccess;
}
"""


def test_launches_are_on_the_contexts_device(fake, tmp_path):  # noqa: F811
    """With another device current, every call launches on its context's, and leaves the caller's current."""
    source, library = tmp_path / "two.c", tmp_path / "libtwo.so"
    source.write_text(TWO_DEVICES)
    subprocess.run(["gcc", "-std=gnu11", "-O1", "-w", "-shared", "-fPIC", "-I", str(HIP_INCLUDE), str(source),
                    "-Wl,--no-as-needed", str(fake),
                    f"-Wl,-rpath,{fake.parent}", "-o", str(library)], check=True)
    child(library, REFUSALS + """
plan, scratch = ctx.alloc(1 << 20), ctx.alloc(1 << 24)
now = C.c_int()
for call in (lambda: store(row_push()), lambda: load(row_push()), lambda: attn(attn_push(), scratch=scratch),
             lambda: select(evict_push(), plan=plan), lambda: compact(evict_push(), plan=plan),
             lambda: refused(abi.call, "vx_kv4_advance", ctx.handle, H(slots), H(pos), 0, 2, 1, 40)):
    fake.hipSetDevice(1)
    assert call() == "VX_OK"
    fake.hipGetDevice(C.byref(now))
    assert now.value == 1 and fake.astray_launches() == 0
""")


ROOMY = """
#define _GNU_SOURCE
#define __HIP_PLATFORM_AMD__ 1
#include <hip/hip_runtime_api.h>
#include <sys/mman.h>
hipError_t hipMalloc(void **p, size_t n) {   /* address space; nothing touches what is large */
    *p = mmap(0, n, PROT_READ | PROT_WRITE, MAP_PRIVATE | MAP_ANONYMOUS | MAP_NORESERVE, -1, 0);
    return *p == MAP_FAILED ? hipErrorOutOfMemory : hipSuccess;
}
hipError_t hipFree(void *p) { return hipSuccess; }
"""


@pytest.fixture(scope="module")
def roomy(fake, tmp_path_factory):  # noqa: F811
    """The stand-in with room for buffers of any size."""
    where = tmp_path_factory.mktemp("roomy")
    source, library = where / "roomy.c", where / "libroomy.so"
    source.write_text(ROOMY)
    subprocess.run(["gcc", "-std=gnu11", "-O1", "-w", "-shared", "-fPIC", "-I", str(HIP_INCLUDE), str(source),
                    "-Wl,--no-as-needed", str(fake),
                    f"-Wl,-rpath,{fake.parent}", "-o", str(library)], check=True)
    return library


def test_rows_whose_end_passes_64_bits_are_refused(roomy):
    """More than 2^30 rows in caches that a card holds (43 GB each), of a stride for which the bytes of the rows, taken
    modulo 2^64, would fit a buffer of 4 GB."""
    child(roomy, REFUSALS + """
g = dict(layers=1, sequences=257, kv_heads=1, head_dim=64, context=1 << 22)
nbytes = lib.vx_kv4_cache_bytes(C.byref(abi.Kv4Geom(*g.values())))
kc, vc, slots = ctx.alloc(nbytes), ctx.alloc(nbytes), ctx.alloc(4 * 257)
rows = 257 << 22
far = -(-(1 << 62) // (rows - 1))                     # the least stride that wraps
assert far < 1 << 32 and ((rows - 1) * far + 64) * 4 % (1 << 64) < 1 << 33
buf, whole = ctx.alloc(1 << 33), ctx.alloc(rows * 64 * 4)
near = dict(n_sequences=257, tokens=1 << 22, k_stride=64, v_stride=64, **g)
for call in (store, load):
    kw = dict(kc=kc, vc=vc, slots=slots)
    for name, at in (("k_stride", dict(k=buf, v=whole)), ("v_stride", dict(k=whole, v=buf))):
        for stride in (far, 4294967295):
            assert call(row_push(**dict(near, **{name: stride})), **kw, **at, **({} if call is load else dict(pos=None, sp=None))) == "VX_ERR_BOUNDS"
near = dict(n_sequences=257, tokens=1 << 22, q_heads=1, q_stride=64, out_stride=64, **g)
scratch = ctx.alloc(lib.vx_kv4_attention_scratch_bytes(attn_push(**near), 0))
for name, at in (("q_stride", dict(q=buf, out=whole)), ("out_stride", dict(q=whole, out=buf))):
    assert attn(attn_push(**dict(near, **{name: far})), **at, kc=kc, vc=vc, w=None, slots=slots, scratch=scratch) == "VX_ERR_BOUNDS"
assert kernels() == 0
""")


def test_every_kernel_has_a_case_whose_values_are_compared(roomy):
    """The kernels of a call go by sizes. All sets of them that a sweep of sizes launches are launched by a case of the
    GPU tests that compares values with the restatement, so that no change of a rule leaves a kernel untested."""
    child(roomy, REFUSALS + """
sys.path[:0] = ["tests", "oracle"]
import test_gpu_kv4 as gpu
names = ["k_kv4_attnILi%dELi%dELi%dELb%dE" % (hd, nt, 8 if nt > 1 else 4, pk) for hd in (64, 128, 256)
         for nt, pk in ((1, 1), (1, 0), (2, 0), (4, 0))]
names += [n % hd for hd in (64, 128, 256) for n in ("k_kv4_finishILi%dE", "k_kv4_weights_rowsILi%dE")] + ["k_kv4_add_weights"]
bufs = {n: ctx.alloc(1 << 33) for n in ("q", "out", "kc", "vc", "w", "slots", "scratch")}
def kernels_of(hd, qh, heads, tokens, S, context, track):
    before = [launches(n) for n in names]
    pc = abi.Kv4AttentionPush(abi.Kv4Geom(1, S, heads, hd, context), 0, 0, S, tokens, qh, qh * hd, qh * hd, 0, 0, 1.0)
    b = dict(bufs, w=bufs["w"] if track else None)
    assert attn(pc, **b) == "VX_OK"
    return frozenset(n for n, c in zip(names, before) if launches(n) > c)
def params(test):
    marks = [m for m in test.pytestmark if m.name == "parametrize"]
    sets = [{}]
    for m in marks:
        keys = m.args[0].split(",")
        rows = [dict(zip(keys, v if len(keys) > 1 else (v,))) for v in m.args[1]]
        sets = [dict(s, **r) for s in sets for r in rows]
    return sets
covered = set()
for p in params(gpu.test_single_token):
    covered.add(kernels_of(p["hd"], p["qh"], p["H"], 1, 1, p["base"] + 1 + p["base"] % 3, False))
for p in params(gpu.test_several_tokens_and_prompts):
    covered.add(kernels_of(p["hd"], p["qh"], p["H"], p["tokens"], 1, p["context"], p["track"]))
for p in params(gpu.test_long_prompts) + params(gpu.test_long_caches):
    covered.add(kernels_of(p["hd"], p["qh"], p["H"], p["tokens"], len(p["bases"]), p["context"], p["track"]))
for p in params(gpu.test_kernels_by_size):
    for track in (False, True):
        covered.add(kernels_of(p["hd"], p["qh"], p["H"], p["tokens"], p["S"], p["context"], track))
reached = {}
for hd in (64, 128, 256):
    for qh, heads in ((1, 1), (8, 1), (16, 2), (8, 8), (32, 1), (3, 3)):
        for S in (1, 3, 16):
            for tokens in (1, 2, 5, 9, 17, 33, 65, 120, 250, 600, 1500, 4000):
                for context in (1, 40, 130, 400, 1000, 1100, 1600, 4100, 20000):
                    if tokens <= context:
                        for track in (False, True):
                            reached.setdefault(kernels_of(hd, qh, heads, tokens, S, context, track), (hd, qh, heads, tokens, S, context, track))
missing = [v for k, v in reached.items() if k not in covered]
assert not missing, missing
assert {n for k in reached for n in k} == set(n for n in names if n != "k_kv4_attnILi256ELi4ELi8ELb0E")
""")
