// Shared pieces of the local attention kernels (local_attention.hip, local_attention_bwd.hip): which frames a
// query sees, the frames' tiles that a block visits, and the learned bias by distance.
//
// Query n of batch row b stands at frame p = starts[b] + n.  It sees frame j < count(b) where the key mask lets it,
//   j <= p + right  and  (j >= p - left  or  j < sinks).
// The frames that a run of queries sees are one run of frames and the first few: a block visits the tiles of
// both and nothing between them.  Rows are those of one head (unlike the cross attention's): a wave's 32 rows
// then stand at 32 frames in a row, and the bias of a 32 x 32 tile is 63 neighbouring numbers of one table.
//
// The bias enters as the starting value of the score's accumulator: b / scale, so that adding it costs no
// instruction of the vector unit, only the reads that fill the accumulator (zeros otherwise).  With the lane's
// query fixed, its 8 + 8 keys are two runs of the table, which lies in LDS by distance, one number a distance,
// padded so that a tile that touches the range of distances never reads past it.  Tiles beyond the range on
// either side start from one number.
#pragma once

#include "attention.h"

namespace pmsst {
namespace attn {

constexpr int kMaxDistance = 1024;
constexpr int kMaxBuckets = 1024;
constexpr int kPad = 64;                    // table entries past either end: a tile spans 63 distances
constexpr int32_t kMaxFrames = 1 << 28;     // sums of two frames and a limit fit 32 bits
constexpr float kBiasMost = 1048576.f;      // finite entries are cut to this,
constexpr float kBiasHides = -1e30f;        // and those not above this hide their bucket's frames

struct Window {
  int32_t left, right;    // -1: no limit
  int32_t sinks;          // 0 where left is none
  const int32_t* starts;  // [B] or NULL: 0
};

struct BiasArgs {
  const void* table;         // [buckets, H], NULL: no bias
  const int32_t* bucket_of;  // [2 distance + 1]: the bucket of distance i - distance
  int32_t buckets, distance;  // `distance` is cut to what a call reaches, and bucket_of moved along
  int32_t f32;               // the table's type: fp32, or that of q
};

inline int bias_entries(int distance) { return 2 * distance + 1 + 2 * kPad; }

__device__ __forceinline__ int start_of(const Window& w, int b) {
  if (w.starts == nullptr) return 0;
  constexpr int kMost = 1 << 29;
  const int s = w.starts[b];
  return s < -kMost ? -kMost : s > kMost ? kMost : s;
}

// The frames [lo, hi) of the window of a query at frame p, of `count`.
__device__ __forceinline__ int low_of(const Window& w, int p) { return w.left < 0 ? 0 : max(0, p - w.left); }
__device__ __forceinline__ int high_of(const Window& w, int p, int count) {
  return w.right < 0 ? count : min(count, p + w.right + 1);
}

// The tiles of BK frames that the queries at p0 .. p1 see any frame of: those of the sinks, then the window's.
struct TileList {
  int first;  // the first `sink` tiles are 0 ..., the others first + i - sink
  int sink;
  int total;
  __device__ __forceinline__ int at(int i) const { return i < sink ? i : first + i - sink; }
};
template <int BK>
__device__ __forceinline__ TileList tiles_of(const Window& w, int p0, int p1, int count) {
  const int hi = high_of(w, p1, count), lo = low_of(w, p0);
  TileList l;
  l.first = lo / BK;
  const int end = hi > lo ? (hi + BK - 1) / BK : l.first;
  const int sinks = (max(0, min(w.sinks, hi)) + BK - 1) / BK;
  l.sink = hi > lo ? min(sinks, l.first) : sinks;
  l.total = l.sink + end - l.first;
  return l;
}

// Bits [from, to) of 32.
__device__ __forceinline__ uint32_t below(int x) { return x >= 32 ? ~0u : x <= 0 ? 0u : (1u << x) - 1u; }
__device__ __forceinline__ uint32_t span_bits(int from, int to) { return below(to) & ~below(from); }

// Bits of the 32 frames from key0 on that a query with the window [low, high) sees.
__device__ __forceinline__ uint32_t frames_seen(int low, int high, int sinks, int key0) {
  return span_bits(low - key0, high - key0) | below(min(sinks, high) - key0);
}
// Bits of the 32 queries from row0 on that see frame `key`.
__device__ __forceinline__ uint32_t queries_seeing(const Window& w, int start, int key, int row0) {
  const int from = w.right < 0 ? 0 : key - w.right - start - row0;
  const int to = w.left < 0 || key < w.sinks ? 32 : key + w.left - start + 1 - row0;
  return span_bits(from, to);
}

// What a wave's 32 queries (from frame p0 on) see of the 32 frames from key0 on by window and sinks alone.
enum class Sees { kNone, kSome, kAll };
__device__ __forceinline__ Sees sees(const Window& w, int p0, int key0, int count) {
  const int hi_last = high_of(w, p0 + 31, count);
  if (key0 >= hi_last || (key0 + 31 < low_of(w, p0) && key0 >= w.sinks)) return Sees::kNone;
  if (key0 + 32 <= high_of(w, p0, count) && (key0 >= low_of(w, p0 + 31) || key0 + 32 <= w.sinks)) return Sees::kAll;
  return Sees::kSome;
}

// A bucket's entry of the bias.
__device__ __forceinline__ float bias_entry(const BiasArgs& t, int dtype, int heads, int head, int bucket) {
  bucket = bucket < 0 ? 0 : bucket >= t.buckets ? t.buckets - 1 : bucket;
  const int64_t at = static_cast<int64_t>(bucket) * heads + head;
  return t.f32                ? static_cast<const float*>(t.table)[at]
         : dtype == PMSST_F16 ? static_cast<float>(static_cast<const f16*>(t.table)[at])
                              : static_cast<float>(static_cast<const bf16*>(t.table)[at]);
}
// As the kernels take it, in units of 1 / unit.
__device__ __forceinline__ float bias_value(float v, float unit) {
  if (v <= kBiasHides) return -kInf;
  return (v > kBiasMost ? kBiasMost : v < -kBiasMost ? -kBiasMost : v) * unit;  // NaN stays
}

// Fills `table` by distance, kPad + distance entries on either side of 0 (falling distances if DOWN).  Two loads, one
// waiting for the other, make an entry: four are on their way at once.  True if one of this thread's hides its frames.
template <typename T, bool DOWN>
__device__ __forceinline__ bool fill_bias(float* table, const BiasArgs& t, int heads, int head, float unit, int threads) {
  const int entries = 2 * t.distance + 1 + 2 * kPad;
  bool hides = false;
  for (int base = threadIdx.x; base < entries; base += 4 * threads) {
    int bucket[4];
    float value[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int d = min(max(min(base + j * threads, entries - 1) - kPad - t.distance, -t.distance), t.distance);
      bucket[j] = t.bucket_of[t.distance + (DOWN ? -d : d)];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) value[j] = bias_entry(t, dtype_code<T>(), heads, head, bucket[j]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float v = bias_value(value[j], unit);
      hides |= v == -kInf;
      if (base + j * threads < entries) table[base + j * threads] = v;
    }
  }
  return hides;
}

// Bits of the 32 frames from key0 on that the bias (a table by rising distance) does not hide from a query at frame `pos`.
__device__ __forceinline__ uint32_t bias_shows(const float* table, int distance, int pos, int key0) {
  uint32_t bits = 0;
#pragma unroll 4
  for (int i = 0; i < 32; ++i) {
    const int d = min(max(key0 + i - pos, -distance), distance);
    bits |= (table[d + distance + kPad] != -kInf ? 1u : 0u) << i;
  }
  return bits;
}

// Whether the distances lo .. lo + 62 of a tile are all on one end of the table (that end's entry), or not.
__device__ __forceinline__ bool bias_far(int lo, int distance, bool& upper) {
  upper = lo >= distance;
  return upper || lo + 62 <= -distance;
}

// The first frame's distance to the first query of a tile, cut to where the table's ends begin: a tile beyond it reads
// its end's entries, all alike.
__device__ __forceinline__ int bias_gap(int gap, int distance) { return min(max(gap, -distance - 31), distance + 31); }

// The accumulator of a score tile: `table` entries from this lane's first one on, in the order of the registers.
__device__ __forceinline__ f32x16_t bias_tile(const float* first) {
  f32x16_t acc;
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i] = first[reg_key(i)];
  return acc;
}

// mma_rows with a starting value.
template <typename T, int DP>
__device__ __forceinline__ f32x16_t mma_rows_from(f32x16_t acc, const char* tile, int sub, const u32x4_t (&frag)[DP * sizeof(T) / 32],
                                                  int lane) {
  constexpr int DB = DP * sizeof(T);
  const int row = 32 * sub + key_row(lane & 31);
#pragma unroll
  for (int s = 0; s < DB / 32; ++s) {
    acc = mma<T>(row_frag<DB>(tile, row, s, lane >> 5), frag[s], acc);
    if constexpr (sizeof(T) == 4) hold(DB == 512 ? s % 2 == 1 : s % 4 == 3);
  }
  return acc;
}

// Moves a tile's pointers on by `bytes`.
template <typename TileT>
__device__ __forceinline__ void skip(TileT& t, int64_t bytes) {
#pragma unroll
  for (int i = 0; i < TileT::CH; ++i) t.ptr[i] += bytes;
}

// The tiles of BQ queries that a block with the frames [key0, key_end) passes over: of those that see any by the window,
// of every head in turn, the slot's share (slots below `splits`), or of those past the window, that see sinks alone,
// `chunk_tiles` a slot (the others, `chunks` in number).
struct RowTiles {
  int first, tiles;  // of a head
  int from, to;      // of the tiles of all heads in turn
};
template <int BQ>
__device__ __forceinline__ RowTiles rows_of(const Window& w, int start, int queries, int group, int key0, int key_end, int slot,
                                            int splits, int chunks, int chunk_tiles) {
  const int all = (queries + BQ - 1) / BQ;
  const int low = w.right < 0 ? 0 : max(0, key0 - w.right - start);
  const int high = w.left < 0 ? queries : min(queries, key_end + w.left - start);
  RowTiles r;
  r.first = min(low / BQ, all);
  r.tiles = high <= low ? 0 : max(0, (high + BQ - 1) / BQ - r.first);
  if (slot < splits) {
    const int64_t total = static_cast<int64_t>(r.tiles) * group;
    r.from = static_cast<int>(total * slot / splits);
    r.to = static_cast<int>(total * (slot + 1) / splits);
  } else {
    r.first += r.tiles;
    r.tiles = all - r.first;
    r.from = min((slot - splits) * chunk_tiles, r.tiles * group);
    r.to = slot + 1 == splits + chunks ? r.tiles * group : min(r.from + chunk_tiles, r.tiles * group);
  }
  return r;
}

// ---------------------------------------------------------------- host
// Checks and arguments that the forward and the backward share.
struct LocalArgs {
  Shape s;
  Window w;
  BiasArgs bias;
  int32_t cut;  // the distances cut off on either side of bucket_of
};
// The largest distance that a pair can have, up to `distance`.
inline int64_t reach_of(const Shape& s, const Window& w, int64_t distance) {
  if (w.starts == nullptr) distance = std::min<int64_t>(distance, std::max<int64_t>(std::max(s.N, s.M) - 1, 0));
  if (w.left >= 0 && w.right >= 0 && w.sinks == 0) distance = std::min<int64_t>(distance, std::max(w.left, w.right));
  return distance;
}
int make_local(const char* what, int64_t batch, int64_t queries, int64_t keys, int64_t heads, int64_t kv_heads, int64_t head_dim,
               int64_t left, int64_t right, int64_t sinks, const int32_t* starts, const void* bias, int bias_dtype,
               const int32_t* bucket_of, int64_t buckets, int64_t distance, double scale, int dtype, LocalArgs& out);

}  // namespace attn
}  // namespace pmsst
