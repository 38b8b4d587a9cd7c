// Shared pieces of the cross attention kernels (cross_attention.hip, cross_attention_bwd.hip).
//
// Rows: the queries of one (batch, key head) pair, r = n * group + g for query n and query head
// hk * group + g, so heads that share a key head share its tiles.  A wave owns 32 rows (or, where the
// keys' gradients are summed, 32 keys) and multiplies 32 x 32 tiles on the matrix cores.
//
// Products run "transposed": a tile of scores is computed as K Q^T, keys down and rows across, because
// lane l of a 32x32 result holds column l % 32 and rows 8 a + 4 (l / 32) + c (a, c = 0..3, register
// 4 a + c).  Each lane then owns one query and 16 keys: the softmax reduces inside a lane and once across
// the two halves, and its statistics are one register each.  With the K rows fed in the order key_row()
// gives, those 16 keys are 8 + 8 consecutive ones in exactly the places the next product wants its second
// operand (16-bit: column l % 32, k = 8 (l / 32) + 0..7 of each 16; fp32: any k per half), so P never leaves
// its registers.
//
// LDS tiles hold whole rows of the head dimension (DB bytes, zero-filled past head_dim), their 16-byte
// units XOR-swizzled by swz(row); see swz.
#pragma once

#include <algorithm>

#include "common.h"
#include "gemm.h"
#include "mfma.h"
#include "philox.h"
#include "ring.h"

namespace pmsst {
namespace attn {

typedef float f32x16_t __attribute__((ext_vector_type(16)));

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLn2 = 0.693147180559945309f;
constexpr float kInf = __builtin_inff();

// Element strides {batch, position, head} of a [B, N, H, D] tensor whose last axis is dense.
struct Strides {
  int64_t b, n, h;
};

struct Shape {
  int32_t B, N, M, H, Hk, D;
  int32_t G;      // H / Hk
  int32_t R;      // rows of one (batch, key head): N * G
  FastDiv by_g;
};

struct KeyMask {
  const uint8_t* mask;     // [B, M], 0 = not attended; NULL: all
  int64_t stride;          // between batch rows
  const int32_t* lengths;  // [B]; NULL: M
};

// The 16-byte unit u of LDS row r sits at unit u ^ swz(r).  A b128 fragment read takes one unit of 16 rows
// that differ in r % 16 each cycle, a transpose read 64 bytes (an aligned group of 4 units) of rows
// 4 i .. 4 i + 3; 64 banks hold 256 bytes, so rows that share r % (256 / DB) must differ in the swizzle, and
// of four consecutive rows those that start on the same bank in its group bits (the upper ones).
template <int DB>
__device__ __forceinline__ constexpr int swz(int r) {
  if constexpr (DB == 64) return (r >> 2) & 3;
  else if constexpr (DB == 128) return (((r >> 1) & 1) << 2) | (((r >> 2) & 1) << 1) | ((r >> 3) & 1);
  else return ((r & 3) << 2) | ((r >> 2) & 3);
}

// Key (inside 32) that row `rho` of a score tile's first operand holds.  Result register r of half h is row
// 8 (r / 4) + 4 h + r % 4, so a lane's registers 0-7 and 8-15 are the 8 consecutive keys 8 h + 0..7 of
// either 16: one operand fragment of a 16-bit product, and one block of the dropout's bits.
__device__ __forceinline__ constexpr int key_row(int rho) {
  return (rho & 16) | ((rho & 4) << 1) | ((rho & 8) >> 1) | (rho & 3);
}
// Key of register r, without the half's 8 h.
__device__ __forceinline__ constexpr int reg_key(int r) { return 16 * (r >> 3) + (r & 7); }

// acc += A (32 rows) B^T (32 columns) over the 32 bytes of k that a 16-byte fragment per lane spans.
template <typename T>
__device__ __forceinline__ f32x16_t mma(const u32x4_t& a, const u32x4_t& b, f32x16_t acc) {
  if constexpr (std::is_same<T, bf16>::value) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), acc,
                                                   0, 0, 0);
  } else if constexpr (std::is_same<T, f16>::value) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), acc, 0,
                                                  0, 0);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t ai = a[i], bi = b[i];
      acc = __builtin_amdgcn_mfma_f32_32x32x2f32(__builtin_bit_cast(float, ai), __builtin_bit_cast(float, bi), acc, 0, 0,
                                                 0);
    }
    return acc;
  }
}

// This lane's value and that of lane l ^ 32 combined, the lower lane's first: one exchange of register halves.
__device__ __forceinline__ void halves(float v, float& lo, float& hi) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t a = r[0], b = r[1];
  lo = __builtin_bit_cast(float, a);
  hi = __builtin_bit_cast(float, b);
}
__device__ __forceinline__ float half_max(float v) {
  float lo, hi;
  halves(v, lo, hi);
  return fmaxf(lo, hi);
}
__device__ __forceinline__ float half_sum(float v) {
  float lo, hi;
  halves(v, lo, hi);
  return lo + hi;
}

// Two fp32 rounded to nearest into one register of 16-bit values.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  typedef T v2 __attribute__((ext_vector_type(2)));
  const v2 v{static_cast<T>(lo), static_cast<T>(hi)};
  return __builtin_bit_cast(uint32_t, v);
}

// Eight score-tile registers (one 16-key step of a lane) as the second operand of the next product.
template <typename T>
__device__ __forceinline__ u32x4_t pack8(const f32x16_t& p, int step) {
  return u32x4_t{pack2<T>(p[8 * step], p[8 * step + 1]), pack2<T>(p[8 * step + 2], p[8 * step + 3]),
                 pack2<T>(p[8 * step + 4], p[8 * step + 5]), pack2<T>(p[8 * step + 6], p[8 * step + 7])};
}

// Eight elements (16-bit) or four (fp32) of a 16-byte unit.
template <typename T>
__device__ __forceinline__ void unpack(const u32x4_t& u, float (&o)[16 / sizeof(T)]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = u[i];
    if constexpr (std::is_same<T, bf16>::value) {
      o[2 * i] = __builtin_bit_cast(float, w << 16);
      o[2 * i + 1] = __builtin_bit_cast(float, w & 0xFFFF0000u);
    } else if constexpr (std::is_same<T, f16>::value) {
      o[2 * i] = static_cast<float>(__builtin_bit_cast(f16, static_cast<uint16_t>(w)));
      o[2 * i + 1] = static_cast<float>(__builtin_bit_cast(f16, static_cast<uint16_t>(w >> 16)));
    } else {
      o[i] = __builtin_bit_cast(float, w);
    }
  }
}

// ---------------------------------------------------------------- LDS fragments

// Fragment s (32 bytes of k) of tile row `row`: this lane's unit 2 s + h.
template <int DB>
__device__ __forceinline__ u32x4_t row_frag(const char* tile, int row, int s, int h) {
  return *reinterpret_cast<const u32x4_t*>(tile + row * DB + 16 * ((2 * s + h) ^ swz<DB>(row)));
}

// Transposed tile as first operand (16-bit): the product's rows are the head-dimension columns 32 dt + 0..31,
// its k the tile rows k0 + 8 h + 0..7 by two transpose reads; the columns of a 16-lane group come in the order
// 0-3, 8-11, 4-7, 12-15, so that a result lane holds 8 consecutive ones.
template <int DB>
__device__ __forceinline__ u32x4_t col_frag(const char* tile, int k0, int dt, int lane) {
  const int j = lane & 15, h = lane >> 5;
  const int row = k0 + 8 * h + (j >> 2);
  const int unit = 4 * dt + 2 * ((lane >> 4) & 1) + (j & 1);
  const int byte = 8 * ((j >> 1) & 1);
  typedef __attribute__((address_space(3))) s16x4_t lds_s16x4;
  const char* p0 = tile + row * DB + 16 * (unit ^ swz<DB>(row)) + byte;
  const char* p1 = tile + (row + 4) * DB + 16 * (unit ^ swz<DB>(row + 4)) + byte;
  const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p0));
  const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p1));
  const uint2 a = __builtin_bit_cast(uint2, lo), b = __builtin_bit_cast(uint2, hi);
  return u32x4_t{a.x, a.y, b.x, b.y};
}

// fp32 tiles are read by as many instructions as the matrix cores run: nothing is scheduled across this, or
// the reads of a whole tile would be hoisted and spill.
__device__ __forceinline__ void hold(bool here) {
  if (here) __builtin_amdgcn_sched_barrier(0);
}

// The lane index, unknown to the compiler for rows of 256 bytes and more: the up to 80 swizzled addresses of a tile, which do not
// change from tile to tile, would be kept in registers that those kernels do not have.
template <int DB>
__device__ __forceinline__ int fresh(int lane) {
  if constexpr (DB >= 256) asm volatile("" : "+v"(lane));
  return lane;
}

// acc[dt] += (tile rows sub*32 .. + 31)^T * b, b the two 16-row fragments of a score tile (16-bit types).
template <typename T, int DP>
__device__ __forceinline__ void mma_cols(const char* tile, int sub, const u32x4_t (&b)[2], f32x16_t (&acc)[DP / 32], int lane) {
#pragma unroll
  for (int s = 0; s < 2; ++s) {
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) {
      acc[dt] = mma<T>(col_frag<DP * sizeof(T)>(tile, 32 * sub + 16 * s, dt, lane), b[s], acc[dt]);
    }
  }
}

// acc[dt] += (tile rows sub*32 .. + 31)^T * p, for every 32 columns of the head dimension: p is a score tile
// whose k index is the tile's row.
template <typename T, int DP>
__device__ __forceinline__ void mma_cols(const char* tile, int sub, const f32x16_t& p, f32x16_t (&acc)[DP / 32], int lane) {
  constexpr int DB = DP * sizeof(T);
  if constexpr (sizeof(T) == 2) {
    const u32x4_t b[2] = {pack8<T>(p, 0), pack8<T>(p, 1)};
    mma_cols<T, DP>(tile, sub, b, acc, lane);
  } else {
    const int h = lane >> 5, d = lane & 31;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int row = 32 * sub + reg_key(r) + 8 * h;
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt) {
        const float a = *reinterpret_cast<const float*>(tile + row * DB + 16 * ((8 * dt + (d >> 2)) ^ swz<DB>(row)) +
                                                        4 * (d & 3));
        acc[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, p[r], acc[dt], 0, 0, 0);
      }
      hold(DB == 512 ? r % 2 == 1 : r % 4 == 3);
    }
  }
}

// (tile rows sub*32 + key_row(l % 32)) * frag^T
template <typename T, int DP>
__device__ __forceinline__ f32x16_t mma_rows(const char* tile, int sub, const u32x4_t (&frag)[DP * sizeof(T) / 32], int lane) {
  constexpr int DB = DP * sizeof(T);
  const int row = 32 * sub + key_row(lane & 31);
  f32x16_t acc{};
#pragma unroll
  for (int s = 0; s < DB / 32; ++s) {
    acc = mma<T>(row_frag<DB>(tile, row, s, lane >> 5), frag[s], acc);
    if constexpr (sizeof(T) == 4) hold(DB == 512 ? s % 2 == 1 : s % 4 == 3);
  }
  return acc;
}

// ---------------------------------------------------------------- global access

// A row's fragments from global memory: unit 2 s + h of each 32 bytes; zero past head_dim or where !valid.
template <typename T, int DP>
__device__ __forceinline__ void load_frags(const T* row, bool valid, int d_units, int h,
                                           u32x4_t (&f)[DP * sizeof(T) / 32]) {
  constexpr int NS = DP * sizeof(T) / 32;
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    f[s] = u32x4_t{0, 0, 0, 0};
    if (valid && 2 * s + h < d_units) f[s] = *reinterpret_cast<const u32x4_t*>(reinterpret_cast<const char*>(row) + 32 * s + 16 * h);
  }
}

// BK rows of a tile, moved from global memory straight into LDS (16 bytes a lane to a wave's base + 16 * lane:
// the lane that fills unit p of row r fetches unit p ^ swz(r)).  Whole tiles step a pointer per unit by a
// constant; a cut one (and rows whose heads do not divide the tile, and fp32 rows of 512 bytes, which leave no
// registers for pointers) computes its addresses, rows past the end
// clamped to the last, and what is not to be seen is zeroed afterwards by the lanes that moved it.
template <typename T, int DP, int BK, int NW>
struct Tile {
  static constexpr int DB = DP * sizeof(T);
  static constexpr int UNITS = DB / 16;
  static constexpr int CH = BK * UNITS / (64 * NW);  // moves of a wave
  static constexpr int STEP = 64 * NW / UNITS;       // rows between them
  static_assert(CH >= 1 && CH * 64 * NW == BK * UNITS && 64 % UNITS == 0, "whole rows per move");
  const char* ptr[CH];

  static __device__ __forceinline__ int row_of(int i) { return static_cast<int>(threadIdx.x) / UNITS + i * STEP; }

  // The unit this lane moves of its row (unit 0 in place of those past head_dim).
  static __device__ __forceinline__ int unit_of(int i) {
    return (static_cast<int>(threadIdx.x) % UNITS) ^ swz<DB>(row_of(i));
  }
  static __device__ __forceinline__ int byte_of(int i, int d_units) {
    const int u = unit_of(i);
    return u < d_units ? 16 * u : 0;
  }

  // at(row): element offset of a row from `base`
  template <typename F>
  __device__ __forceinline__ void start(const T* base, int row0, int d_units, F at) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      ptr[i] = reinterpret_cast<const char*>(base + at(row0 + row_of(i))) + byte_of(i, d_units);
    }
  }
  static __device__ __forceinline__ uint32_t target(const char* tile, int i) {
    return __builtin_amdgcn_readfirstlane(lds_addr(tile) + static_cast<uint32_t>(threadIdx.x) / 64 * 1024) + i * NW * 1024;
  }
  // Starts a whole tile's move; the pointers go on by `step` bytes.
  __device__ __forceinline__ void fetch(const char* tile, int64_t step) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      dma16_m0(ptr[i], target(tile, i));
      ptr[i] += step;
    }
  }
  // The tile at row0, of which only rows below `rows` (> 0) are there: those past the end are the last one again, or
  // what `past` (a row) holds.
  template <typename F>
  __device__ __forceinline__ void fetch_cut(const char* tile, const T* base, int row0, int rows, int d_units, F at,
                                            const T* past = nullptr) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int row = min(row0 + row_of(i), rows - 1);
      const T* from = past != nullptr && row0 + row_of(i) >= rows ? past : base + at(row);
      dma16_m0(reinterpret_cast<const char*>(from) + byte_of(i, d_units), target(tile, i));
    }
  }
  // Zeroes this lane's units of rows whose bit is 0, and those past head_dim; the moves must have arrived.
  __device__ __forceinline__ void clear(char* tile, uint64_t seen, int d_units) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      if (unit_of(i) >= d_units || !((seen >> row_of(i)) & 1)) {
        *reinterpret_cast<u32x4_t*>(tile + (i * 64 * NW + static_cast<int>(threadIdx.x)) * 16) = u32x4_t{0, 0, 0, 0};
      }
    }
  }
  // Zeroes this lane's units of the rows from `rows` on; the moves must have arrived.
  __device__ __forceinline__ void clear_from(char* tile, int rows) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int at = (i * 64 * NW + static_cast<int>(threadIdx.x)) * 16;
      if (at >= rows * DB) *reinterpret_cast<u32x4_t*>(tile + at) = u32x4_t{0, 0, 0, 0};
    }
  }
};

// Tiles lie in two stages: while one is multiplied, the next one's move fills the other.  (Three stages hold more
// LDS than the wait they save is worth: 124 x 948 queries, forward 365 us against 330 when the third was given up.)
constexpr int kStages = 2;

// Uses a loaded register here, so that the compiler waits for the load here and not (for every load in flight)
// inside the loop.
template <int N>
__device__ __forceinline__ void arrive(u32x4_t (&f)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(f[i]));
}

// Bits of BK <= 64 rows from row0 that lie below `rows`.
__device__ __forceinline__ uint64_t range_bits(int row0, int rows) {
  const int left = rows - row0;
  return left >= 64 ? ~uint64_t{0} : left <= 0 ? 0 : (uint64_t{1} << left) - 1;
}

// Keys of batch row b that count: its length (cut to [0, M]) and its row of the mask.
__device__ __forceinline__ int key_count(const KeyMask& km, int b, int M) {
  if (km.lengths == nullptr) return M;
  const int len = km.lengths[b];
  return len < 0 ? 0 : len > M ? M : len;
}

// `v` where bit k of `bits` is set, else `other`: a sign-extended bit and a bit select.
__device__ __forceinline__ float where_bit(uint32_t bits, int k, float v, float other) {
  const uint32_t m = static_cast<uint32_t>(__builtin_amdgcn_sbfe(static_cast<int>(bits), k, 1));
  return __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, v) & m) | (__builtin_bit_cast(uint32_t, other) & ~m));
}

// Stores a transposed accumulator (rows = head dimension, columns = positions): lane's position row at `row`.
template <typename T, int DP>
__device__ __forceinline__ void store_cols(T* row, const f32x16_t (&acc)[DP / 32], float scale, int d, int h) {
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int at = 32 * dt + 16 * j + 8 * h;
        if (at < d) {
          float o[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] = acc[dt][8 * j + i] * scale;
          store_pack<T, 8>(row + at, o);
        }
      }
    } else {
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const int at = 32 * dt + 8 * a + 4 * h;
        if (at < d) {
          float o[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) o[i] = acc[dt][4 * a + i] * scale;
          store_pack<T, 4>(row + at, o);
        }
      }
    }
  }
}

// The same, unrounded, into a partial sum's fp32 row; T is the type whose column order the accumulator has.
template <typename T, int DP>
__device__ __forceinline__ void store_cols_f32(float* row, const f32x16_t (&acc)[DP / 32], float scale, int d, int h) {
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt) {
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const int at = 32 * dt + (sizeof(T) == 2 ? reg_key(4 * a) + 8 * h : 8 * a + 4 * h);
      if (at < d) {
        float o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = acc[dt][4 * a + i] * scale;
        store_pack<float, 4>(row + at, o);
      }
    }
  }
}

// ---------------------------------------------------------------- block numbering
// Blocks of one (batch, key head) share its keys: they run on one XCD (the hardware deals block i to XCD
// i % 8) where the pairs fill the XCDs evenly; few pairs are spread block by block instead.  Many pairs are dealt
// eight at a time: the heads of a batch row, whose rows are neighbours in memory, follow each other on one XCD
// (1032 x 62 queries over 62 keys, 8 heads, forward and backward in turn: one by one 196 us, by eights 177); fewer go
// one by one, so that the heads of a long batch row are spread (2 rows of 8 heads over 8192 and 4096 keys: 240 us, by
// eights, all on two XCDs, 827).
struct Grid {
  uint32_t pairs;  // batch * key heads
  uint32_t per;    // blocks of a pair
  uint32_t by_xcd, by_eight;
  FastDiv by_per;
};

inline Grid make_grid(int64_t pairs, int64_t per) {
  Grid g;
  g.pairs = static_cast<uint32_t>(pairs);
  g.per = static_cast<uint32_t>(per);
  g.by_xcd = pairs % 8 == 0 || pairs >= 64;
  g.by_eight = pairs >= 2048 || (pairs >= 512 && pairs % 64 == 0);
  g.by_per = FastDiv(g.per);
  return g;
}
// A launch has less than 2^32 work-items: 2^24 blocks of up to 256.
inline bool grid_fits(int64_t pairs, int64_t per) { return per < (int64_t{1} << 24) / (pairs + 64); }
inline int64_t grid_blocks(const Grid& g) {
  const int64_t step = g.by_eight ? 64 : g.by_xcd ? 8 : 1;
  return (int64_t{g.pairs} + step - 1) / step * step * g.per;
}
// (pair, block of the pair); false: past the last pair.
__device__ __forceinline__ bool locate(const Grid& g, uint32_t& pair, uint32_t& sub) {
  const uint32_t x = blockIdx.x;
  if (g.by_xcd) {
    const uint32_t i = x >> 3, local = g.by_per.div(i), xcd = x & 7;
    sub = i - local * g.per;
    pair = g.by_eight ? ((local >> 3) * 8 + xcd) * 8 + (local & 7) : local * 8 + xcd;
  } else {
    pair = g.by_per.div(x);
    sub = x - pair * g.per;
  }
  return pair < g.pairs;
}

// ---------------------------------------------------------------- dropout of the weights
// Weight (b, head, n, key) is element ((b H + head) N + n) * pitch + key of the dropout's numbering, pitch =
// M rounded up to 8: a lane's 8 consecutive keys are one Philox block.
__device__ __forceinline__ uint64_t drop_row(const Shape& s, int b, int head, int n) {
  return ((static_cast<uint64_t>(b) * s.H + head) * s.N + n) * ((static_cast<uint32_t>(s.M) + 7) / 8);
}

// Head dimension a kernel is built for.
inline int padded_dim(int d) { return d <= 32 ? 32 : d <= 64 ? 64 : 128; }

// Host checks, in cross_attention.hip.
int make_shape(const char* what, int64_t batch, int64_t queries, int64_t keys, int64_t heads, int64_t kv_heads,
               int64_t head_dim, int dtype, Shape& s);
int make_strides(const char* what, const void* p, const int64_t* strides, int64_t positions, int64_t heads, int64_t dim,
                 int dtype, Strides& out);

}  // namespace attn
}  // namespace pmsst
