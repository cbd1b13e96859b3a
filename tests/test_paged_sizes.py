"""The paged KV cache's sizes on the CPU, from the library's own arithmetic: small C++ programs over csrc/paged.h, linked
with the library, and the grids that its calls launch."""
import subprocess
from pathlib import Path

import pytest

from test_kv4 import roomy  # noqa: F401  (fixture)
from test_paged import CALLS
from test_refused_memory import HIP_INCLUDE, child, fake  # noqa: F401  (fixture)
from voxgen_amd import abi

ROOT = Path(__file__).resolve().parents[1]

PROGRAM = """
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <random>
using std::max;
using std::min;
#include "paged.h"
using namespace vx;
#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\\n", __LINE__, #x); std::exit(1); } } while (0)
"""


@pytest.fixture(scope="module")
def run(tmp_path_factory):
    if not (HIP_INCLUDE / "hip" / "hip_runtime.h").exists():
        pytest.skip(f"no HIP headers under {HIP_INCLUDE}")
    where = tmp_path_factory.mktemp("sizes")

    def go(name, code):
        source, program = where / f"{name}.cpp", where / name
        source.write_text(PROGRAM + code)
        lib = Path(abi.LIB_PATH).resolve()
        subprocess.run(["g++", "-std=c++17", "-O2", "-w", "-D__HIP_PLATFORM_AMD__", "-I", str(HIP_INCLUDE), "-I", str(ROOT / "voxgen_amd" / "csrc"),
                        str(source), "-o", str(program), str(lib), f"-Wl,-rpath,{lib.parent}"], check=True)
        p = subprocess.run([str(program)], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
        assert p.returncode == 0, p.stdout
    return go


def test_items_are_no_more_work_than_their_requests_hold(run):
    """Whatever a plan's buffer holds, a workgroup goes through chunks that its rows attend to and no others: tables of 2^28
    positions would otherwise let a word of it ask for 2^28 chunks."""
    run("items", """
int main() {
    std::mt19937 rng(1);
    auto any = [&](uint32_t most) { return rng() % 4 ? (uint32_t)(rng() % most) : (uint32_t)rng(); };
    const uint32_t caps[] = {16, 1600, 32768, 1u << 28};
    uint32_t taken = 0;
    for (int n = 0; n < 4000000; ++n) {
        const uint32_t requests = 1 + rng() % 5, max_rows = 1 + rng() % 40, group = 1 + rng() % 9, cap = caps[rng() % 4], parts = rng() % 100;
        const PagedItem it = {any(requests + 1), any(max_rows + 1), any(cap + 2), any(max_rows + 1), any(max_rows * group + 1),
                              any(cap / 32u + 2), any(cap / 32u + 2), rng() % 2 ? VX_PAGED_NONE : any(parts + 1)};
        if (!paged_is_item(it, requests, max_rows, group, cap, parts)) continue;
        ++taken;
        CHECK(it.request < requests && (uint64_t)it.row + it.count <= max_rows && (uint64_t)it.base + it.count <= cap);
        CHECK(it.tile < it.count * group && (it.part == VX_PAGED_NONE || it.part < parts));
        CHECK(((uint64_t)it.first + it.n) * 32u < (uint64_t)it.base + it.count + 32u);
    }
    CHECK(taken > 10000);
    const PagedItem whole = {0, 0, 1000, 5, 0, 0, 32, VX_PAGED_NONE};
    CHECK(paged_is_item(whole, 1, 5, 1, 4096, 0));
    for (uint32_t PagedItem::*field : {&PagedItem::first, &PagedItem::n})
        for (uint32_t x : {33u, 4096u, 1u << 28, 0xFFFFFFFFu}) {
            PagedItem it = whole;
            it.*field = x;
            CHECK(!paged_is_item(it, 1, 5, 1, 4096, 0));
        }
}
""")


def test_lists_and_scratch_hold_what_the_plan_makes(run):
    """The plan's lists and the attention's parts, sized by a batch, hold what the kernel's division makes of any step of it,
    with any of its requests refused for want of pages. For parts of tiles of every size, tables that are divided and that
    are not, and steps of which nothing is spare."""
    run("plans", """
int main() {
    std::mt19937_64 rng(2);
    auto pick = [&](uint64_t lo, uint64_t hi) { return (uint32_t)(lo + rng() % (hi - lo + 1)); };
    auto log = [&](uint32_t lo, uint32_t hi) { return (uint32_t)std::exp(std::log(lo) + (std::log(hi + 0.99) - std::log(lo)) * (rng() % 10000) / 10000.0); };
    uint64_t full[4] = {}, kinds[6] = {};
    for (int n = 0; n < 20000; ++n) {
        const uint32_t heads[] = {1, 2, 3, 8, 32}, dims[] = {64, 128, 256};
        vx_paged_batch b{};
        b.geom = {1, 1u << 20, 16u << pick(0, 4), heads[rng() % 5], dims[rng() % 3]};
        b.requests = log(1, 300);
        b.table_width = std::max(1u, log(1, 100000) / b.geom.page_size);
        b.max_rows = log(1, 2000);
        b.max_count = rng() % 2 ? 1u : std::min(b.max_rows, log(1, 500));
        b.q_heads = b.geom.kv_heads * log(1, 40);
        if (!vx_paged_plan_bytes(&b)) continue;
        const PagedShape s = paged_shape(b);
        const uint32_t group = b.q_heads / b.geom.kv_heads, ps = b.geom.page_size, cap = b.table_width * ps;
        kinds[s.tile_rows == 8 ? 0 : s.tile_rows == 16 ? 1 : s.waves == 8 ? 2 : 3]++;
        kinds[s.joins ? 4 : 5]++;
        for (int step = 0; step < 20; ++step) {
            // lengths: any, all alike, one long, all full, about some multiple of a part
            const int kind = rng() % 5;
            const uint32_t alike = pick(0, cap - 1);
            std::vector<uint32_t> length, count;
            uint32_t rows = 0;
            float work = 0.f;
            for (uint32_t i = 0; i < b.requests; ++i) {
                uint32_t c = rng() % 8 == 0 ? 0u : kind == 3 || rng() % 2 ? b.max_count : pick(1, b.max_count);
                c = std::min(std::min(c, b.max_rows - rows), cap);
                rows += c;
                const uint32_t most = cap - c;
                const uint32_t l = kind == 0 ? pick(0, most) : kind == 1 ? alike : kind == 2 ? (i == 0 ? most : pick(0, 40)) : kind == 3 ? most
                                   : pick(1, 4) * 32u * s.least + pick(0, 64);
                length.push_back(std::min(l, most));
                count.push_back(c);
                if (c) work += (float)((c * group + s.tile_rows - 1) / s.tile_rows) * (float)((length.back() + c + 31) / 32);
            }
            const uint32_t per = paged_per(s, b.geom.kv_heads, work);
            const bool refuse = rng() % 4 == 0;
            uint64_t runs = 0, items = 0, joins = 0, parts = 0;
            for (uint32_t i = 0; i < b.requests; ++i) {
                const uint32_t c = count[i], l = length[i];
                if (c == 0 || (refuse && rng() % 3 == 0)) continue;
                uint32_t splits;
                const uint32_t chunks = (l + c + 31) / 32, by = paged_divide(s, per, chunks, splits), tiles = (c * group + s.tile_rows - 1) / s.tile_rows;
                CHECK(splits >= 1 && splits <= kPagedMaxSplits && (uint64_t)by * splits >= chunks && (uint64_t)by * (splits - 1) < chunks);
                CHECK(splits == 1 || by % s.waves == 0);
                runs += (l + c - 1) / ps - l / ps + 1;
                items += (uint64_t)tiles * splits;
                joins += splits > 1 ? tiles : 0;
                parts += splits > 1 ? (uint64_t)tiles * splits : 0;
            }
            CHECK(runs <= s.runs && items <= s.items && joins <= s.joins && parts <= s.parts);
            full[0] += runs * 10 > s.runs * 9ull, full[1] += items * 2 > s.items, full[2] += s.joins && joins * 2 > s.joins;
            full[3] += s.parts && parts * 3 > s.parts;
            // what the attention allocates for the parts
            vx_paged_attention_push pc{};
            pc.batch = b;
            CHECK(vx_paged_attention_scratch_bytes(&pc) >= parts * b.geom.kv_heads * s.tile_rows * (b.geom.head_dim + 2) * 4);
        }
    }
    for (uint64_t x : full) CHECK(x > 100);      // sizes are not far above what is needed
    for (uint64_t x : kinds) CHECK(x > 100);
}
""")


GRIDS = """
#define __HIP_PLATFORM_AMD__ 1
#include <hip/hip_runtime_api.h>
static int seen, bad;
int grids_seen(void) { return seen; }
int grids_bad(void) { int n = bad; bad = 0; return n; }
hipError_t hipLaunchKernel(const void *fn, dim3 g, dim3 b, void **a, size_t s, hipStream_t st) {
    unsigned long long x = (unsigned long long)g.x * b.x;
    ++seen;
    bad += !g.x || !g.y || !g.z || x >= 1ull << 32 || g.y > 65535 || g.z > 65535 || b.x * b.y * b.z > 1024 || b.x % 64 || b.y * b.z != 1;
    return hipSuccess;
}
"""


def test_grids_of_every_call(roomy, tmp_path):  # noqa: F811
    """Launch grids at the largest sizes that a batch may have, and the least: some workgroups, fewer than 2^32 threads,
    in the other dimensions at most 65535."""
    source, library = tmp_path / "grids.c", tmp_path / "libgrids.so"
    source.write_text(GRIDS)
    subprocess.run(["gcc", "-std=gnu11", "-O1", "-w", "-shared", "-fPIC", "-I", str(HIP_INCLUDE), str(source), "-Wl,--no-as-needed", str(roomy),
                    f"-Wl,-rpath,{roomy.parent}", "-o", str(library)], check=True)
    child(library, CALLS + """
def one(**kw):
    b = batch(**kw)
    g = b.geom
    need = lib.vx_paged_plan_bytes(b)
    assert need, (kw, lib.vx_last_error())
    row, wide, budget = g.kv_heads * g.head_dim, b.q_heads * g.head_dim, min(b.table_width, 200)
    apc = attn_push(q_stride=wide, out_stride=wide, **kw)
    spc, pick = attn_push(q_stride=wide, out_stride=wide, budget=budget, **kw), select_push(q_stride=wide, budget=budget, sinks=0, recent=1, **kw)
    state = dict(lengths=ctx.alloc(4 * b.requests), tables=ctx.alloc(4 * b.requests * b.table_width), pool=ctx.alloc(4 * (g.pages + 1)))
    plan, other = ctx.alloc(need), ctx.alloc(4 * b.requests)
    caches = dict(kc=ctx.alloc(lib.vx_paged_cache_bytes(g)), vc=ctx.alloc(lib.vx_paged_cache_bytes(g)))
    lo_hi, rows = ctx.alloc(lib.vx_paged_bounds_bytes(g)), {n: ctx.alloc(4 * b.max_rows * row) for n in "kv"}
    qo = dict(q=ctx.alloc(4 * b.max_rows * wide), out=ctx.alloc(4 * b.max_rows * wide))
    sel = ctx.alloc(4 * b.max_rows * g.kv_heads * budget)
    room = lambda n: ctx.alloc(n)
    for call in (lambda: reset(b, **state), lambda: make(b, counts=other, plan=plan, **state),
                 lambda: advance(b, plan=plan, lengths=state["lengths"], pool=state["pool"]), lambda: cut(b, keep=other, **state),
                 lambda: store(store_push(k_stride=row, v_stride=row, **kw), bounds=lo_hi, plan=plan, **rows, **caches),
                 lambda: store(store_push(k_stride=row, v_stride=row, **kw), bounds=None, plan=plan, **rows, **caches),
                 lambda: attn(apc, tables=state["tables"], plan=plan, scratch=room(lib.vx_paged_attention_scratch_bytes(apc)), **qo, **caches),
                 lambda: attn(spc, tables=state["tables"], plan=plan, selected=sel, scratch=room(lib.vx_paged_attention_scratch_bytes(spc)), **qo, **caches),
                 lambda: select(pick, q=qo["q"], bounds=lo_hi, tables=state["tables"], plan=plan, selected=sel,
                                scratch=room(lib.vx_paged_select_scratch_bytes(pick)))):
        n, got = fake.grids_seen(), call()
        assert got == "VX_OK", (kw, got, lib.vx_last_error())
        assert fake.grids_seen() > n and fake.grids_bad() == 0, kw
many = dict(layers=1, head_dim=64)
one(max_rows=1 << 22, max_count=1 << 22, q_heads=1, kv_heads=1, pages=1 << 20, table_width=1 << 18, requests=1, **many)
one(max_rows=1 << 22, max_count=1, q_heads=1, kv_heads=1, pages=1 << 20, table_width=1 << 16, requests=4096, **many)
one(max_rows=1 << 19, max_count=1, q_heads=8, kv_heads=8, pages=1 << 16, table_width=1 << 12, requests=4096, **many)
one(max_rows=1 << 12, max_count=1 << 12, q_heads=1024, kv_heads=1, pages=1 << 16, table_width=1 << 12, requests=4096, **many)
one(max_rows=240, max_count=240, q_heads=17408, kv_heads=17, pages=64, table_width=64, requests=64, **many)
one(max_rows=64, max_count=64, q_heads=65535, kv_heads=65535, pages=64, table_width=64, requests=64, **many)
one(max_rows=64, max_count=1, q_heads=65535, kv_heads=65535, pages=64, table_width=64, requests=64, **many)
one(max_rows=64, max_count=1, q_heads=65535, kv_heads=65535, pages=1 << 12, table_width=1 << 18, requests=1, **many)
one(max_rows=1, max_count=1, q_heads=1, kv_heads=1, pages=1, table_width=1, requests=1, **many)
one(max_rows=1, max_count=1, q_heads=1024, kv_heads=1, pages=1, table_width=1 << 24, requests=1, layers=1, head_dim=256)
""")
