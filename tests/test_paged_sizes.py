"""The paged KV cache's sizes on the CPU, from the library's own arithmetic: small C++ programs over csrc/paged.h, linked
with the library."""
import subprocess
from pathlib import Path

import pytest

from test_refused_memory import HIP_INCLUDE
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
