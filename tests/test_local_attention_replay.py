"""What the local attention kernels visit, run on the CPU: the text of ``csrc/local_attention.h`` itself is compiled, and
its tiles, masks and table indexes are held against the rule, pair by pair."""

from __future__ import annotations

import subprocess

import pytest

from tests.test_attention_source_replay import CSRC, _block

_PRELUDE = r"""
#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <vector>
#define __device__
#define __forceinline__ inline
using std::max;
using std::min;
#define CHECK(cond, ...) do { if (!(cond)) { printf(__VA_ARGS__); printf(" (%s)\n", #cond); exit(1); } } while (0)
constexpr int kPad = 64;
"""

_DRIVER = r"""
struct Case { Window w; int start, queries, count, frames; };

static bool rule(const Case& c, int n, int j) {
  const int64_t p = int64_t{c.start} + n;
  if (j >= c.count) return false;
  if (c.w.right >= 0 && j > p + c.w.right) return false;
  return c.w.left < 0 || j >= p - c.w.left || j < c.w.sinks;
}

template <int BK>
void forward(const Case& c, int rows) {
  for (int n0 = 0; n0 < c.queries; n0 += rows) {
    const int last = min(n0 + rows, c.queries) - 1;
    const TileList list = tiles_of<BK>(c.w, c.start + n0, c.start + last, c.count);
    CHECK(list.total >= 0 && list.sink >= 0 && list.sink <= list.total, "list");
    std::vector<int> there((c.count + BK - 1) / BK + 1);
    for (int i = 0; i < list.total; ++i) {
      const int t = list.at(i);
      CHECK(t >= 0 && t * BK < c.count, "tile %d of %d frames", t, c.count);
      CHECK(i == 0 || t > list.at(i - 1), "tiles fall");
      CHECK(i >= list.sink || t == i, "sink tiles start at 0");
      there[t] = 1;
    }
    for (int n = n0; n <= last; ++n) {
      for (int j = 0; j < c.count; ++j) CHECK(!rule(c, n, j) || there[j / BK], "query %d frame %d not visited", n, j);
    }
    for (int w0 = n0; w0 <= last; w0 += 32) {
      for (int i = 0; i < list.total * (BK / 32); ++i) {
        const int key0 = list.at(i / (BK / 32)) * BK + 32 * (i % (BK / 32)), p0 = c.start + w0;
        const Sees what = sees(c.w, p0, key0, c.count);
        for (int n = w0; n < w0 + 32; ++n) {
          const int low = low_of(c.w, c.start + n), high = high_of(c.w, c.start + n, c.count);
          const uint32_t bits = frames_seen(low, high, c.w.sinks, key0);
          for (int k = 0; k < 32; ++k) {
            const bool seen = rule(c, n, key0 + k);
            CHECK(what != Sees::kNone || !seen || n > last, "passed over: query %d frame %d", n, key0 + k);
            CHECK(what != Sees::kAll || seen, "taken whole: query %d frame %d", n, key0 + k);
            CHECK(((bits >> k) & 1) == seen, "mask: query %d frame %d", n, key0 + k);
          }
        }
      }
    }
  }
}

template <int BQ>
void backward(const Case& c, int block, int group, int splits, int chunks, int chunk) {
  const int sink_tiles = c.w.sinks > 0 ? min((c.w.sinks + block - 1) / block, (c.frames + block - 1) / block) : 0;
  for (int tile = 0; tile * block < c.count; ++tile) {
    const int key0 = tile * block, end = min(key0 + block, c.count), all = (c.queries + BQ - 1) / BQ;
    std::vector<int> times(all * group);
    for (int slot = 0; slot < splits + (tile < sink_tiles ? chunks : 0); ++slot) {
      const RowTiles r = rows_of<BQ>(c.w, c.start, c.queries, group, key0, end, slot, splits, chunks, chunk);
      CHECK(r.from >= 0 && r.from <= r.to && r.to <= r.tiles * group, "range %d %d of %d", r.from, r.to, r.tiles);
      for (int i = r.from; i < r.to; ++i) {
        const int g = i / r.tiles, t = r.first + i % r.tiles;
        CHECK(t >= 0 && t < all, "tile %d of %d", t, all);
        ++times[g * all + t];
      }
    }
    for (int g = 0; g < group; ++g) {
      for (int t = 0; t < all; ++t) {
        CHECK(times[g * all + t] <= 1, "tile %d twice", t);
        if (times[g * all + t]) continue;
        for (int n = t * BQ; n < min(c.queries, t * BQ + BQ); ++n) {
          for (int j = key0; j < end; ++j) CHECK(!rule(c, n, j), "query %d of frame %d not visited", n, j);
        }
      }
    }
    for (int j = key0; j < end; ++j) {
      for (int row0 = 0; row0 < c.queries; row0 += 32) {
        const uint32_t bits = queries_seeing(c.w, c.start, j, row0);
        for (int n = row0; n < min(c.queries, row0 + 32); ++n) CHECK(((bits >> (n - row0)) & 1) == rule(c, n, j), "query %d frame %d", n, j);
      }
    }
  }
}

void table(int distance) {
  const int entries = 2 * distance + 1 + 2 * kPad;
  for (int gap = -distance - 300; gap <= distance + 300; ++gap) {  // key0 - p0
    bool upper;
    const bool far = bias_far(gap - 31, distance, upper);
    for (int q = 0; q < 32; ++q) {
      for (int k = 0; k < 32; ++k) {
        const int d = gap + k - q;
        if (far) CHECK(upper ? d >= distance : d <= -distance, "distance %d taken for an end of %d", d, distance);
        else CHECK(d + distance + kPad >= 0 && d + distance + kPad < entries && kPad + distance - d >= 0 && kPad + distance - d < entries,
                   "distance %d of %d", d, distance);
      }
    }
  }
}

int main() {
  for (int d : {0, 1, 7, 31, 32, 48, 128, 1024}) table(d);
  uint64_t state = 12345;
  auto below_n = [&](int n) { state = state * 6364136223846793005ull + 1442695040888963407ull; return static_cast<int>((state >> 33) % n); };
  for (int i = 0; i < 700; ++i) {
    Case c{};
    c.queries = 1 + below_n(i % 3 ? 200 : 420);
    c.frames = below_n(2) ? c.queries : 1 + below_n(420);
    c.count = below_n(3) ? c.frames : below_n(c.frames + 1);
    c.start = below_n(2) ? 0 : below_n(600) - 150;
    c.w.left = below_n(4) ? below_n(below_n(2) ? 20 : 300) : -1;
    c.w.right = below_n(4) ? below_n(below_n(2) ? 20 : 300) : -1;
    if (below_n(3) == 0) c.w.right = 0;
    c.w.sinks = c.w.left < 0 ? 0 : below_n(3) ? below_n(10) : below_n(150);
    for (int rows : {64, 128}) {
      forward<32>(c, rows);
      forward<64>(c, rows);
      backward<32>(c, rows, 1 + i % 3, 1 + below_n(5), 1 + below_n(4), 1 + below_n(9));
      backward<64>(c, rows, 1 + i % 3, 1 + below_n(5), 1 + below_n(4), 1 + below_n(9));
    }
  }
  // the far ends of the documented ranges: no sum passes 32 bits
  for (int start : {-(1 << 29), 1 << 29}) {
    for (int left : {-1, 0, 1 << 29}) {
      for (int right : {-1, 0, 1 << 29}) {
        const Window w{left, right, left < 0 ? 0 : 1 << 28, nullptr};
        const int count = 1 << 28;
        const TileList l = tiles_of<64>(w, start, start + (1 << 28) - 1, count);
        CHECK(l.total >= 0 && (l.total == 0 || (l.at(0) >= 0 && l.at(l.total - 1) * int64_t{64} < count)), "far tiles");
        const RowTiles r = rows_of<64>(w, start, 1 << 28, 1, count - 128, count, 0, 1, 1, 8);
        CHECK(r.first >= 0 && r.first + r.tiles <= (1 << 22), "far rows");
      }
    }
  }
  return 0;
}
"""

_PIECES = ["struct Window {", "int low_of(", "int high_of(", "struct TileList {", "TileList tiles_of(", "uint32_t below(int x)",
           "uint32_t span_bits(", "uint32_t frames_seen(", "uint32_t queries_seeing(", "enum class Sees {", "Sees sees(",
           "bool bias_far(", "struct RowTiles {", "RowTiles rows_of("]


def _source():
    header = (CSRC / "local_attention.h").read_text()
    assert f"constexpr int kPad = 64;" in header
    return _PRELUDE + "\n".join(_block(header, p) for p in _PIECES) + _DRIVER


def _run(folder, source):
    (folder / "replay.cpp").write_text(source)
    subprocess.run(["g++", "-std=c++17", "-O2", "-fsanitize=undefined", "-fno-sanitize-recover=undefined", "-o",
                    str(folder / "replay"), str(folder / "replay.cpp")], check=True)
    return subprocess.run([str(folder / "replay")], capture_output=True, text=True)


def test_every_seen_pair_is_visited_once_and_masked_right(tmp_path):
    res = _run(tmp_path, _source())
    assert res.returncode == 0, res.stdout + res.stderr


def test_the_kernels_use_the_tested_pieces():
    fwd, bwd = ((CSRC / f).read_text() for f in ("local_attention.hip", "local_attention_bwd.hip"))
    for text in (fwd, bwd):
        assert "tiles_of<BK>(a.w, start + n0, start + min(n0 + 32 * NW, s.N) - 1, count)" in text
        assert "frames_seen(low, high, a.w.sinks, key0)" in text and "sees(a.w, p0, key0, count)" in text
        assert "bias_far(key0 - p0 - 31, a.bias.distance, upper)" in text
    assert "queries_seeing(a.w, start, ki, row0)" in bwd and "rows_of<BQ>(a.w, start, s.N, s.G, block_key0, block_end" in bwd


@pytest.mark.parametrize("old,new", [("j < w.sinks", "j <= w.sinks"), ("p + w.right + 1", "p + w.right"),
                                     ("min(sinks, l.first)", "sinks"), ("key + w.left - start + 1", "key + w.left - start"),
                                     ("key0 - w.right - start)", "key0 - start)"), ("lo + 62 <= -distance", "lo + 32 <= -distance"),
                                     ("r.first += r.tiles;", "r.first += r.tiles + 1;")])
def test_planted_mistakes_are_found(tmp_path, old, new):
    text = _source()
    if old == "j < w.sinks":  # in the rule of this file's copy
        old, new = "j < c.w.sinks", "j <= c.w.sinks"
    assert old in text
    assert _run(tmp_path, text.replace(old, new)).returncode != 0
