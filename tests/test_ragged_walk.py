"""How the persistent int8 kernels over experts walk their tiles: the walk's own source (RaggedWalk, xcd_remap, the launch's grid), compiled for the host with a wave of 64 lanes
as fibers, over offsets that segments have and offsets that contradict each other, on devices of any number of compute units."""

import os
import random
import re
import shutil
import subprocess

import pytest
import torch

from tilegym_amd import ops

from .test_int8_forms import RING
from .test_int8_ops import BF16, codes, scales

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tilegym_amd", "csrc")

HARNESS = r"""
#include <ucontext.h>
#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <vector>
#define __device__
#define __forceinline__ inline
using std::min;
struct Int8GemmParams { int M, E; const int* m_indptr; };

// 64 fibers that meet at every operation across lanes
static ucontext_t g_main, g_lane[64];
static std::vector<char> g_stack[64];
static int g_now, g_done;
static int64_t g_slot[64];
static void meet() { swapcontext(&g_lane[g_now], &g_main); }
template <typename F> static auto across(int64_t v, F f) {
    const int lane = g_now;
    g_slot[lane] = v;
    meet();
    const auto r = f(lane);
    meet();
    return r;
}
static int __shfl_up(int v, int d) { return (int)across(v, [=](int l) { return l >= d ? g_slot[l - d] : g_slot[l]; }); }
static int read_lane(int v, int l) { return (int)across(v, [=](int) { return g_slot[l]; }); }
static unsigned long long __ballot(bool b) {
    return across(b, [](int) { unsigned long long m = 0; for (int i = 0; i < 64; ++i) m |= (unsigned long long)(g_slot[i] != 0) << i; return m; });
}
static int __ffsll(long long v) { return __builtin_ffsll(v); }
#define __builtin_amdgcn_readlane(v, l) read_lane(v, l)
#define __builtin_amdgcn_readfirstlane(v) read_lane(v, 0)

@SOURCE@

static Int8GemmParams g_p;
static int g_tiles_n, g_bm, g_grid, g_block;
static bool g_agree = true;
template <int BM> static void lane_main() {
    const int lane = g_now;
    RaggedWalk<BM> walk;
    const int total = walk.start(g_p, lane, g_tiles_n);
    for (int v = g_block; v < total; v += g_grid) {
        int expert, m0, rows, tile_n;
        const int pid = xcd_remap(v, total);
        walk.find(g_p, lane, pid, g_tiles_n, expert, m0, rows, tile_n);
        const int64_t mine = (((int64_t)expert * 1000003 + m0) * 1009 + rows) * 10007 + tile_n, first = across(mine, [](int) { return g_slot[0]; });
        if (first != mine) g_agree = false;
        if (lane == 0) printf("%d %d %d %d %d %d\n", g_block, pid, expert, m0, rows, tile_n);
    }
    ++g_done;
    for (;;) meet();
}
int main() {
    int units;
    std::vector<int> indptr;
    while (scanf("%d %d %d %d %d", &g_bm, &g_p.M, &g_p.E, &g_tiles_n, &units) == 5) {
        indptr.resize(g_p.E + 1);
        for (int& x : indptr)
            if (scanf("%d", &x) != 1) return 2;
        g_p.m_indptr = indptr.data();
        g_grid = (int)walking_grid(most_row_tiles(g_p.M, g_p.E, g_bm) * g_tiles_n, units);
        printf("grid %d\n", g_grid);
        for (g_block = 0; g_block < g_grid; ++g_block) {
            g_done = 0;
            for (int l = 0; l < 64; ++l) {
                g_stack[l].resize(32768);
                getcontext(&g_lane[l]);
                g_lane[l].uc_stack.ss_sp = g_stack[l].data(), g_lane[l].uc_stack.ss_size = g_stack[l].size(), g_lane[l].uc_link = &g_main;
                makecontext(&g_lane[l], g_bm == 32 ? lane_main<32> : lane_main<256>, 0);
            }
            while (g_done < 64)
                for (g_now = 0; g_now < 64; ++g_now) swapcontext(&g_main, &g_lane[g_now]);
        }
        printf("end %d\n", (int)g_agree);
    }
    return 0;
}
"""


def _entity(path, start):
    """The source from the line that begins with `start` to the brace that closes its body."""
    text = open(os.path.join(CSRC, path)).read()
    at = text.index("\n" + start) + 1
    depth, i = 0, text.index("{", at)
    while True:
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        i += 1
        if depth == 0:
            return text[at:i] + ("" if start.startswith(("constexpr", "__device__")) else ";") + "\n"


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    source = (_entity("tg_host.h", "constexpr int64_t most_row_tiles(") + _entity("tg_host.h", "constexpr int64_t walking_grid(") +
              _entity("tg_device.h", "__device__ __forceinline__ int xcd_remap(") + _entity("int8_device.h", "__device__ __forceinline__ int ragged_rows(") +
              "template <int BM>\n" + _entity("int8_device.h", "struct RaggedWalk "))
    folder = tmp_path_factory.mktemp("walk")
    (folder / "walk.cpp").write_text(HARNESS.replace("@SOURCE@", source))
    subprocess.run(["g++", "-O1", "-std=c++17", "-o", str(folder / "walk"), str(folder / "walk.cpp")], check=True, timeout=120)

    def run(cases):
        given = "\n".join(" ".join(map(str, [bm, m, len(ptr) - 1, tiles_n, units, *ptr])) for bm, m, ptr, tiles_n, units in cases)
        out = subprocess.run([str(folder / "walk")], input=given, capture_output=True, text=True, check=True, timeout=100).stdout
        made = re.findall(r"grid (\d+)\n((?:[-\d]+ [^\n]*\n)*)end 1\n", out)
        assert len(made) == len(cases)
        return [(int(grid), [tuple(map(int, line.split())) for line in tiles.splitlines()]) for grid, tiles in made]
    return run


def _offsets(rng, experts, rows):
    return sorted(rng.randint(0, rows) for _ in range(experts + 1))


UNITS = (256, 304, 250, 64, 33, 7)


def test_segments_are_covered_once(walk):
    """Every tile of every segment exactly once, whatever the number of compute units."""
    rng, cases = random.Random(1), []
    for units in UNITS:
        for experts in (1, 64, 70, 200):
            rows = rng.choice((1, 40, 700, 3000))
            cases.append((rng.choice((32, 256)), rows, _offsets(rng, experts, rows), rng.choice((1, 2, 5)), units))
    for (bm, rows, ptr, tiles_n, units), (grid, tiles) in zip(cases, walk(cases)):
        want = [(e, m, min(bm, hi - m), n) for e, (lo, hi) in enumerate(zip(ptr, ptr[1:])) for m in range(lo, hi, bm) for n in range(tiles_n)]
        assert sorted(t[2:] for t in tiles) == sorted(want), (bm, rows, tiles_n, units)
        assert grid <= max(units, 8) and (grid % 8 == 0 or grid >= (rows // bm + min(len(ptr) - 1, rows)) * tiles_n)


def test_offsets_that_contradict_each_other_stay_in_range(walk):
    """Segments that overlap or run backwards: which tiles are taken is not said, but each lies within the rows, the experts and the columns."""
    rng, cases = random.Random(2), []
    for units in UNITS:
        cases.append((32, 10, [0, 10] * 35 + [0], 1, units))         # 35 experts of all ten rows
        cases.append((32, 10, [0, 10] * 100 + [0], 3, units))
        cases.append((256, 700, [0, 700] * 80 + [0], 2, units))
        cases.append((32, 5, [5, -3, 9, 0, 100, -7] * 30, 2, units))
        cases.append((32, 300, [rng.randint(-50, 400) for _ in range(140)], 2, units))
    for (bm, rows, ptr, tiles_n, units), (grid, tiles) in zip(cases, walk(cases)):
        for _, pid, expert, m0, has, tile_n in tiles:
            assert pid >= 0 and 0 <= expert < len(ptr) - 1 and 0 <= tile_n < tiles_n, (bm, rows, units, pid, expert, tile_n)
            assert 1 <= has <= bm and ptr[expert] <= m0 and m0 + has <= min(ptr[expert + 1], rows)


@pytest.mark.gpu
@pytest.mark.parametrize("bm,bn", RING + [(256, 256)])
def test_overlapping_segments_of_many_experts(device, bm, bn):
    """More experts than a wave has lanes, each second one with all rows: what is written lies within the rows, and each element is one of the experts' products or untouched."""
    m, n, k, experts = 40, 264, 256, 70
    a, b = codes((m, k), 1).to(device), codes((experts, n, k), 2).to(device)
    sa, sb = scales(m, 3).to(device), scales((experts, n), 4).to(device)
    want = torch.stack([ops.int8_matmul(a, b[e], sa, sb[e]) for e in range(experts)])
    for ptr in ([0, m] * 35 + [0], [0, m, m, 0, 0, 5, 3] * 10 + [m], [m, 0] * 35 + [m]):
        around = torch.full((m + 600, n), 7.0, dtype=BF16, device=device)
        out = around[300:300 + m]
        indptr = torch.tensor(ptr, dtype=torch.int32, device=device)
        ops.ragged_int8_matmul(a, b, sa, sb, indptr, out=out, kernel_configs=dict(KERNEL="tiled", BLOCK_M=bm, BLOCK_N=bn))
        assert bool((around[:300] == 7).all()) and bool((around[300 + m:] == 7).all())
        assert bool(((out == want) | (out == 7)).any(0).all())
