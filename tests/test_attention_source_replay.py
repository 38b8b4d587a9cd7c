"""The tile moves and the block numbering of the cross attention kernels, run on the CPU: the text of
``csrc/attention.h`` itself is compiled with a recorder in place of the DMA, so a change to it is what is tested.

Every move must read inside the rows that are there and fill each 16-byte unit of the LDS tile once, with what the
fragment reads expect there."""

from __future__ import annotations

import re
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "pymsst_amd" / "csrc"

_PRELUDE = r"""
#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <vector>
#define __device__
#define __host__
#define __forceinline__ inline
#define __builtin_amdgcn_readfirstlane(x) (x)
using std::max;
using std::min;
typedef uint32_t u32x4_t __attribute__((vector_size(16)));
struct { unsigned x; } threadIdx, blockIdx;

alignas(16) static char g_lds[65536];
static const char* g_from[4096];  // the source of each 16-byte unit of LDS
static int g_times[4096];
static uint32_t lds_addr(const void* p) { return static_cast<uint32_t>(static_cast<const char*>(p) - g_lds); }
static void dma16_m0(const void* g, uint32_t lds) {
  const uint32_t unit = lds / 16 + (threadIdx.x & 63);
  if (lds % 16 || unit >= 4096) { printf("a move to byte %u of LDS\n", lds); exit(1); }
  g_from[unit] = static_cast<const char*>(g);
  ++g_times[unit];
}
#define CHECK(cond, ...) do { if (!(cond)) { printf(__VA_ARGS__); printf(" (%s)\n", #cond); exit(1); } } while (0)
"""

_DRIVER = r"""
// A pass over `rows` rows of a tensor with `pitch` elements between rows, as the kernels run it.
template <typename T, int DP, int BK, int NW>
void tiles(int d, int rows, int64_t pitch, int t0, bool zeros) {
  using Tl = Tile<T, DP, BK, NW>;
  constexpr int DB = DP * sizeof(T), U = DB / 16;
  const int d_units = d * sizeof(T) / 16;
  const T* base = reinterpret_cast<const T*>(uintptr_t{1} << 40);
  const T* past = zeros ? reinterpret_cast<const T*>(uintptr_t{1} << 20) : nullptr;
  std::vector<Tl> tile(64 * NW);
  auto at = [&](int i) { return i * pitch; };
  for (int i = 0; i < 64 * NW; ++i) {
    threadIdx.x = i;
    tile[i].start(base, t0 * BK, d_units, at);
  }
  for (int t = t0; t * BK < rows; ++t) {
    const bool whole = DB < 512 && t * BK + BK <= rows;
    memset(g_times, 0, sizeof(g_times));
    for (int i = 0; i < 64 * NW; ++i) {
      threadIdx.x = i;
      if (whole) tile[i].fetch(g_lds, BK * static_cast<int64_t>(sizeof(T)) * pitch);
      else tile[i].fetch_cut(g_lds, base, t * BK, rows, d_units, at, past);
    }
    for (int s = 0; s < 4096; ++s) {
      CHECK(g_times[s] == (s < BK * U), "unit %d moved %d times: %d-byte rows, %d waves", s, g_times[s], DB, NW);
      if (s >= BK * U) continue;
      const int row = s / U, unit = (s % U) ^ swz<DB>(row), byte = unit < d_units ? 16 * unit : 0;
      const int src = t * BK + row;
      const char* want = reinterpret_cast<const char*>(base + at(min(src, rows - 1))) + byte;
      if (zeros && src >= rows) want = reinterpret_cast<const char*>(past) + byte;
      CHECK(g_from[s] == want, "row %d unit %d of tile %d: %d-byte rows, d %d, %d rows", row, unit, t, DB, d, rows);
    }
  }
}

template <typename T, int DP, int BK, int NW>
void clears(int d) {
  using Tl = Tile<T, DP, BK, NW>;
  constexpr int DB = DP * sizeof(T), U = DB / 16;
  const int d_units = d * sizeof(T) / 16;
  Tl tile;
  uint64_t seen = 0x9E3779B97F4A7C15ull;
  for (int rows : {1, BK / 2 - 1, BK}) {
    memset(g_lds, 0xFF, BK * DB + 64);
    for (int i = 0; i < 64 * NW; ++i) {
      threadIdx.x = i;
      tile.clear(g_lds, seen, d_units);
      tile.clear_from(g_lds, rows);
    }
    for (int s = 0; s < BK * U + 4; ++s) {
      const int row = s / U, unit = (s % U) ^ swz<DB>(row);
      const bool zero = s < BK * U && (row >= rows || unit >= d_units || !((seen >> row) & 1));
      for (int b = 0; b < 16; ++b) CHECK(g_lds[16 * s + b] == (zero ? 0 : -1), "cleared unit %d of row %d", unit, row);
    }
    seen = ~seen;
  }
  // the fragments: 32 bytes of k, the lane's half of them
  for (int s = 0; s < BK * U; ++s) g_lds[16 * s] = static_cast<char>((s % U) ^ swz<DB>(s / U)), g_lds[16 * s + 1] = static_cast<char>(s / U);
  for (int row = 0; row < BK; ++row) {
    for (int f = 0; f < U; ++f) {
      const u32x4_t u = row_frag<DB>(g_lds, row, f / 2, f % 2);
      CHECK((u[0] & 0xFF) == static_cast<uint32_t>(f) && ((u[0] >> 8) & 0xFF) == static_cast<uint32_t>(row), "fragment %d of row %d", f, row);
    }
  }
}

template <typename T, int DP, int BK, int NW>
void both() {
  for (int d = DP == 32 ? 8 : DP / 2 + 8; d <= DP; d += 8) {
    clears<T, DP, BK, NW>(d);
    for (int rows : {1, 31, 32, 33, 63, 64, 65, 128, 130, 257}) {
      for (int64_t pitch : {int64_t{d}, int64_t{8} * d + 16, int64_t{1} << 25}) {
        for (int t0 : {0, 1}) {
          for (bool zeros : {false, true}) tiles<T, DP, BK, NW>(d, rows, pitch, t0, zeros);
        }
      }
    }
  }
}

void numbering(int64_t pairs, int64_t per) {
  const Grid g = make_grid(pairs, per);
  CHECK(grid_fits(pairs, per), "%ld x %ld", long(pairs), long(per));
  const int64_t blocks = grid_blocks(g);
  CHECK(blocks < int64_t{1} << 24, "%ld blocks", long(blocks));
  std::vector<int> times(pairs * per);
  for (int64_t x = 0; x < blocks; ++x) {
    blockIdx.x = static_cast<unsigned>(x);
    uint32_t pair, sub;
    if (!locate(g, pair, sub)) continue;
    CHECK(pair < pairs && sub < per, "pair %u block %u", pair, sub);
    ++times[pair * per + sub];
  }
  for (int64_t i = 0; i < pairs * per; ++i) CHECK(times[i] == 1, "block %ld visited %d times", long(i), times[i]);
}

int main(int argc, char** argv) {
  if (argc > 1) {
    for (int64_t per : {1, 2, 3, 7, 8, 30, 513}) numbering(atoi(argv[1]), per);
    return 0;
  }
  // the tiles that the kernels use: 64 rows, 32 of 512-byte rows; 2 and 4 waves (512 bytes: 4)
  both<uint16_t, 32, 64, 2>(); both<uint16_t, 32, 64, 4>(); both<uint16_t, 64, 64, 2>(); both<uint16_t, 64, 64, 4>();
  both<uint16_t, 128, 64, 2>(); both<uint16_t, 128, 64, 4>();
  both<float, 32, 64, 2>(); both<float, 32, 64, 4>(); both<float, 64, 64, 2>(); both<float, 64, 64, 4>();
  both<float, 128, 32, 4>();
  return 0;
}
"""


def _block(text: str, start: str) -> str:
    """From the line that holds ``start`` (with a template line before it) to its closing brace."""
    at = text.index(start)
    assert text.count(start) == 1, start
    line = text.rindex("\n", 0, at) + 1
    before = text.rindex("\n", 0, line - 1) + 1
    if text[before:line].startswith("template"):
        line = before
    depth, i = 0, text.index("{", at)
    while True:
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        i += 1
        if depth == 0:
            break
    return text[line:i] + (";\n" if text[i:i + 1] == ";" else "\n")


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    header, common = (CSRC / "attention.h").read_text(), (CSRC / "common.h").read_text()
    parts = [_block(common, "struct FastDiv {")]
    parts += [_block(header, s) for s in ("constexpr int swz(int r)", "u32x4_t row_frag(", "struct Tile {", "struct Grid {",
                                          "inline Grid make_grid(", "inline bool grid_fits(", "inline int64_t grid_blocks(",
                                          "bool locate(")]
    folder = tmp_path_factory.mktemp("attention")
    source = _PRELUDE + "\n".join(parts) + _DRIVER
    (folder / "replay.cpp").write_text(source)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wno-unknown-pragmas", "-Wno-ignored-attributes", "-o", str(folder / "replay"),
                    str(folder / "replay.cpp")], check=True)
    return folder


def _run(program, *args):
    res = subprocess.run([str(program / "replay"), *map(str, args)], capture_output=True, text=True)
    assert res.returncode == 0, res.stdout


def test_tiles_read_their_rows_and_fill_lds_once(program):
    _run(program)


@pytest.mark.parametrize("pairs", [1, 7, 8, 16, 63, 64, 65, 100, 511, 512, 513, 576, 992, 2047, 2048, 2049, 8256])
def test_numbering_visits_every_block_once(program, pairs):
    _run(program, pairs)


def test_the_replay_uses_the_kernels_tiles():
    """The tile sizes that the driver instantiates are those of the sources."""
    fwd, bwd = (CSRC / "cross_attention.hip").read_text(), (CSRC / "cross_attention_bwd.hip").read_text()
    assert "constexpr int fwd_keys() { return DP * sizeof(T) == 512 ? 32 : 64; }" in fwd
    assert "constexpr int bwd_tile() { return DP * sizeof(T) == 512 ? 32 : 64; }" in bwd
    used = set(re.findall(r"Tile<T, DP, (\w+), (\w+)>", fwd + bwd))
    assert used == {("BK", "NW"), ("BQ", "NW"), ("64", "2")}


@pytest.mark.parametrize("old,new", [("min(row0 + row_of(i), rows - 1)", "row0 + row_of(i)"),
                                     ("return u < d_units ? 16 * u : 0;", "return 16 * u;"),
                                     ("(row0 + row_of(i))) + byte_of", "(row0 + row_of(i) + 1)) + byte_of"),
                                     ("ptr[i] += step;", "ptr[i] += step + 16;"),
                                     ("((local >> 3) * 8 + xcd) * 8 + (local & 7)",
                                      "((local >> 3) * 8 + xcd) * 8 + (local & 3)")])
def test_planted_mistakes_are_found(program, old, new):
    """In the replay's copy of the source: a row past the end, padding read, a wrong start, a wrong step, blocks
    visited twice."""
    text = (program / "replay.cpp").read_text()
    assert old in text
    (program / "bad.cpp").write_text(text.replace(old, new))
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wno-unknown-pragmas", "-Wno-ignored-attributes", "-o", str(program / "bad"),
                    str(program / "bad.cpp")], check=True)
    assert subprocess.run([str(program / "bad"), *(["2048"] if "local" in old else [])], capture_output=True).returncode == 1
