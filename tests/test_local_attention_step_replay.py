"""Which frames a step of the local attention reads and writes, and what it may be given, run on the CPU: the text of
``csrc/local_attention_step.hip`` itself is compiled and held against brute force."""

from __future__ import annotations

import ctypes
import re
import subprocess

import pytest

from pymsst_amd import _lib
from tests.test_attention_source_replay import CSRC, _block

_PRELUDE = r"""
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <set>
#define CHECK(cond, ...) do { if (!(cond)) { printf(__VA_ARGS__); printf(" (%s)\n", #cond); exit(1); } } while (0)
"""

_MEET_DRIVER = r"""
static uint64_t state = 9;
static int64_t below(int64_t n) { state = state * 6364136223846793005ull + 1442695040888963407ull; return static_cast<int64_t>((state >> 33) % n); }

static std::set<int64_t> bytes_of(const RowSet& r) {
  std::set<int64_t> all;
  for (int64_t i = 0; i < r.size[0]; ++i)
    for (int64_t j = 0; j < r.size[1]; ++j)
      for (int64_t k = 0; k < r.size[2]; ++k)
        for (int64_t c = 0; c < r.bytes; ++c) all.insert(static_cast<int64_t>(r.at) + i * r.apart[0] + j * r.apart[1] + k * r.apart[2] + c);
  return all;
}

static RowSet draw(int64_t at) {
  RowSet r{};
  r.bytes = 1 + below(6);
  int order[3] = {0, 1, 2};
  for (int i = 2; i > 0; --i) { const int j = below(i + 1), t = order[i]; order[i] = order[j]; order[j] = t; }
  int64_t extent = r.bytes;
  for (int i = 0; i < 3; ++i) {
    r.size[order[i]] = 1 + below(4);
    r.apart[order[i]] = below(8) == 0 ? below(6) : extent + below(2) * below(9);  // now and then rows that overlap
    if (below(12) == 0) r.apart[order[i]] = -r.apart[order[i]];
    extent = extent + labs(r.apart[order[i]]) * (r.size[order[i]] - 1);
  }
  r.at = 100000 + at;
  return r;
}

int main() {
  int meet = 0, apart = 0;
  for (int n = 0; n < 60000; ++n) {
    RowSet a = draw(0), b = draw(below(160) - 80);
    if (below(2)) {  // parts of one buffer
      for (int i = 0; i < 3; ++i) { b.apart[i] = a.apart[i]; b.size[i] = 1 + below(4); }
    }
    if (below(50) == 0) b.size[below(3)] = 0;
    const auto x = bytes_of(a), y = bytes_of(b);
    bool want = false;
    for (int64_t v : x) want |= y.count(v) != 0;
    CHECK(rows_meet(a, b) == want && rows_meet(b, a) == want, "sets %d", n);
    want ? ++meet : ++apart;
  }
  CHECK(meet > 8000 && apart > 8000, "%d meet, %d do not", meet, apart);
  // caches side by side in one buffer, by row, by head and by frame; a frame of a cache; far apart
  const int64_t d = 128, hk = 4, slots = 5000, batch = 60;
  for (int64_t pitch : {2 * d, 2 * d * hk, 2 * d * hk * slots}) {
    const int64_t head = pitch == 2 * d ? 2 * d : d, slot = pitch == 2 * d ? hk * head : pitch == 2 * d * hk ? pitch : hk * d;
    const int64_t row = pitch == 2 * d * hk * slots ? pitch : slots * slot;
    const RowSet k{1 << 20, {batch, slots, hk}, {row, slot, head}, d};
    RowSet v = k, one = k;
    v.at += pitch / 2;
    one.size[1] = 2;
    one.at += 4000 * slot;
    CHECK(!rows_meet(k, v) && !rows_meet(v, k), "side by side");
    CHECK(rows_meet(k, one) && rows_meet(one, k) && rows_meet(k, k), "a part of itself");
    v.at -= 16;
    CHECK(rows_meet(k, v), "side by side but for 16 bytes");
    one.at += int64_t{1} << 45;
    CHECK(!rows_meet(k, one), "elsewhere");
  }
  // numbers whose products pass 64 bits
  const RowSet wide{4096, {2, 2, 2}, {INT64_MAX - 15, INT64_MAX - 15, 16}, 16}, near{4096 + 32, {1, 1, 1}, {0, 0, 0}, 16};
  CHECK(!rows_meet(wide, near) && rows_meet(wide, wide), "wide");
  return 0;
}
"""


_ORDER_DRIVER = r"""
struct Ring { uint32_t d; uint32_t mod(uint32_t n) const { return n % d; } };
struct Row { int64_t n; };
struct Args {
  int32_t left, sinks, ring;
  Ring by_ring;
  Row kcs, vcs, ks, vs;
  struct { int32_t distance; } bias;
};
struct Sizes { int32_t N; };
typedef int32_t T;

static uint64_t state = 31;
static int below(int n) { state = state * 6364136223846793005ull + 1442695040888963407ull; return static_cast<int>((state >> 33) % n); }

static bool rule(const Args& a, int64_t query, int64_t frame) { return frame <= query && (frame >= query - a.left || frame < a.sinks); }
static int64_t slot_of(const Args& a, int64_t frame) { return frame < a.sinks ? frame : a.sinks + (frame - a.sinks) % a.ring; }

static void stream(const Args& a, const Sizes& s, int32_t now) {
  // K's cache holds frame numbers, V's their negatives; slots of frames that no query sees hold others
  std::vector<T> k_cache(a.sinks + a.ring, -7), v_cache(k_cache), k_new(s.N), v_new(s.N);
  for (int64_t f = 0; f < a.sinks && f < now; ++f) k_cache[f] = static_cast<T>(f);
  for (int64_t f = std::max<int64_t>(a.sinks, int64_t{now} - a.left); f < now; ++f) k_cache[slot_of(a, f)] = static_cast<T>(f);
  for (size_t i = 0; i < k_cache.size(); ++i) v_cache[i] = -k_cache[i];
  for (int n = 0; n < s.N && now >= 0; ++n) { k_new[n] = now + n; v_new[n] = -(now + n); }
  const T *kc = k_cache.data(), *vc = v_cache.data(), *kn = k_new.data(), *vn = v_new.data();
@ORDER@
  auto query_of = [](int n) { return n; };
  CHECK(now >= 0 || total == 0, "idle");
  std::set<int64_t> read, visited;
  for (int x = 0; x < total; ++x) {
    const T *kp, *vp;
    locate_frame(x, kp, vp);
    const int64_t f = frame_of(x);
    if (x < old_frames) {
      CHECK(kp - kc >= 0 && kp - kc < a.sinks + a.ring && vp - vc == kp - kc, "slot %ld", static_cast<long>(kp - kc));
      read.insert(kp - kc);
    } else {
      CHECK(kp - kn == x - old_frames && vp - vn == x - old_frames && x - old_frames < s.N, "new frame %d", x);
    }
    CHECK(*kp == f && *vp == -f, "frame %d of the order: %ld for %d", x, static_cast<long>(f), *kp);
    CHECK(visited.insert(f).second, "frame %ld twice", static_cast<long>(f));
  }
  for (int n = 0; n < s.N && now >= 0; ++n) {
    const int64_t p = int64_t{now} + n;
    for (int64_t f = 0; f <= p && f < a.sinks; ++f) CHECK(visited.count(f), "sink %ld of query %d", static_cast<long>(f), n);
    for (int64_t f = std::max<int64_t>(0, p - a.left); f <= p; ++f) CHECK(visited.count(f), "frame %ld of query %d", static_cast<long>(f), n);
@WRITTEN@
    CHECK(slot == slot_of(a, p) && slot < static_cast<uint32_t>(a.sinks + a.ring), "frame %ld goes to %u", static_cast<long>(p), slot);
    CHECK(!read.count(slot), "slot %u is read and written", slot);
  }
  for (int i = 0; i < 60 && total > 0; ++i) {
    const int x1 = below(3) ? total : 1 + below(total), base = below(x1), last = base + 1 + below(below(2) ? 8 : 64);
@WHOLE@
    const bool far = @FAR@;
    for (int x = base; x < last; ++x) {
      const int frame = x < total ? frame_of(x) : 0;
      for (int r = 0; r < s.N; ++r) {
        const bool want = x < x1 && rule(a, int64_t{now} + r, frame);
        CHECK(!whole || want, "taken whole: frame %d of the order, query %d", x, r);
        CHECK(!far || int64_t{now} + r - frame >= a.bias.distance, "taken for far: frame %d of the order", x);
@MASK@
        if (x < total) CHECK(seen == want, "mask: frame %d of the order, query %d", x, r);
        if (x >= x1) CHECK(!seen, "past the end");
      }
    }
  }
}

int main() {
  for (int i = 0; i < 6000; ++i) {
    Args a{};
    a.left = below(below(3) ? 12 : 120);
    a.sinks = below(3) ? below(9) : below(80);
    Sizes s{1 + below(below(2) ? 1 : 9)};
    a.ring = a.left + s.N + (below(2) ? 0 : below(20));
    a.by_ring.d = a.ring;
    a.kcs.n = a.vcs.n = a.ks.n = a.vs.n = 1;
    a.bias.distance = below(40);
    const int held = a.sinks + a.ring;
    const int32_t most = INT32_MAX - s.N + 1;  // the last frame a stream may stand at
    for (int32_t now : {0, -1, -2147483647 - 1, below(held + 3), held, held + below(5 * held), 1000003 + below(held), most - below(held), most}) stream(a, s, now);
  }
  return 0;
}
"""


def _compile_and_run(folder, source):
    (folder / "replay.cpp").write_text(source)
    subprocess.run(["g++", "-std=c++17", "-O2", "-fsanitize=undefined", "-fno-sanitize-recover=undefined", "-o",
                    str(folder / "replay"), str(folder / "replay.cpp")], check=True)
    return subprocess.run([str(folder / "replay")], capture_output=True, text=True)


def _meet_source():
    text = (CSRC / "local_attention_step.hip").read_text()
    return _PRELUDE + _block(text, "struct RowSet {") + "\n" + _block(text, "bool rows_meet(") + _MEET_DRIVER


def _between(text, start, end):
    assert text.count(start) == 1 and end in text[text.index(start):], (start, end)
    at = text.index(start)
    return text[at:text.index(end, at)]


def _order_source():
    """The kernel's own lines about frames and slots, between stand-ins for its arguments."""
    text = (CSRC / "local_attention_step.hip").read_text()
    order = _between(text, "  // the stream's frames in the order they are visited", "  const T* kc = ")
    order += _between(text, "  // where frame number x of the order lies", "\n\n  u32x4_t kf[kUnroll]")
    written = _between(text, "      const uint32_t frame = static_cast<uint32_t>(now)", "      *reinterpret_cast<u32x4_t*>(static_cast<T*>(a.k_cache)")
    whole = _between(text, "    const bool whole = ", "\n    if constexpr (BIAS)")
    far = re.search(r"if \((whole && base >= sink_frames && .* >= a\.bias\.distance)\) \{", text).group(1)
    mask = _between(text, "          const int back = now + query_of(r) - frame;", "w[r][u] = x < x1")
    mask += "const bool seen = " + re.search(r"w\[r\]\[u\] = (x < x1 && back >= 0 .*) \? w\[r\]\[u\] : -kInf;", text).group(1) + ";"
    parts = {"@ORDER@": order, "@WRITTEN@": written, "@WHOLE@": whole, "@FAR@": far, "@MASK@": mask}
    source = _PRELUDE + "#include <algorithm>\n#include <vector>\nusing std::max;\nusing std::min;\n" + _ORDER_DRIVER
    for name, part in parts.items():
        source = source.replace(name, part)
    return source


def test_a_step_reads_the_frames_it_sees_and_writes_the_new_ones(tmp_path):
    """Over random windows, sinks, rings and positions up to the last: every seen frame is visited once and read from the
    slot that holds it, the new ones go to their own slots, which are not read, and masks and shortcuts follow the rule."""
    res = _compile_and_run(tmp_path, _order_source())
    assert res.returncode == 0, res.stdout + res.stderr


@pytest.mark.parametrize("old,new", [("if (slot >= static_cast<uint32_t>(a.ring)) slot -= a.ring;", ""), ("max(now, 0) - a.left", "max(now, 0) - a.left + 1"),
                                     ("base >= sink_frames + s.N - 1", "base >= sink_frames"), ("back <= a.left", "back < a.left"),
                                     ("static_cast<uint32_t>(window_first - a.sinks)", "static_cast<uint32_t>(window_first)"),
                                     ("window_first + (last - 1 - sink_frames)", "window_first + (base - sink_frames)"),
                                     ("a.by_ring.mod(frame - static_cast<uint32_t>(a.sinks))", "a.by_ring.mod(frame)")])
def test_planted_mistakes_in_the_order_are_found(tmp_path, old, new):
    text = _order_source()
    assert old in text
    assert _compile_and_run(tmp_path, text.replace(old, new)).returncode != 0


def test_rows_that_share_memory_are_told(tmp_path):
    res = _compile_and_run(tmp_path, _meet_source())
    assert res.returncode == 0, res.stdout + res.stderr


@pytest.mark.parametrize("old,new", [("- a.bytes", "+ 0 * a.bytes"), ("1 - b.size[i], 0", "0, b.size[i] - 1"), ("terms[i].hi += hi;", "")])
def test_planted_mistakes_are_found(tmp_path, old, new):
    text = _meet_source()
    assert old in text
    assert _compile_and_run(tmp_path, text.replace(old, new)).returncode != 0


def test_caches_that_share_memory_are_refused():
    """Caches that overlap each other, or that q, k or v lie in: one block of the kernel would read what another writes."""
    lib = _lib.load_library()
    at = lambda n: ctypes.c_void_p(1 << 30 | n)  # noqa: E731  never dereferenced: every call below is refused
    strides = lambda *s: (ctypes.c_int64 * 3)(*s)  # noqa: E731
    b, slots, h, hk, d = 3, 20, 4, 2, 64
    held = b * slots * hk * d * 2  # bytes

    def step(q=None, k=None, v=None, kc=None, vc=None, cs=None):
        places = [at(x) if x is not None else at((8 + i) << 20) for i, x in enumerate((q, k, v, kc, vc))]
        return lib.pmsst_local_attention_step(places[0], None, places[1], None, places[2], None, places[3], cs, places[4], cs, at(0), 9, 4,
                                              None, 0, None, 0, 0, at(64 << 20), b, 2, slots, h, hk, d, 1.0, 2, None, 0, None)

    base = 11 << 20
    for kw in (dict(vc=base + held - 16), dict(vc=base - held + 16), dict(vc=base + 256), dict(k=base), dict(v=base + held // 2),
               dict(q=base + held - 16), dict(k=base - 2 * b * hk * d * 2 + 16), dict(v=(12 << 20) + 1024),
               dict(cs=strides(2 * slots * hk * d, 2 * hk * d, 2 * d), vc=base + 112)):
        assert step(**kw) == -1, kw
        assert b"share memory" in lib.pmsst_last_error() or b"lies in a cache" in lib.pmsst_last_error()
