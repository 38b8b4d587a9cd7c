// Cross attention backward.  With P the weights, recomputed from the saved lse, f the dropout's factor of each
// weight (keep / (1 - p)) and dO the output's gradient:
//   D  = rowsum(dO o O)              dV = (P o f)^T dO
//   dS = P o ((dO V^T) o f - D)      dQ = scale dS K,   dK = scale dS^T Q
//
// Two kernels, so that every sum has one owner and no atomic is needed:
//  * attn_dq_kernel: a wave owns 32 rows (its Q and dO in registers) and passes over the key tiles; it also
//    writes D, which it forms from O and dO;
//  * attn_dkv_kernel: a wave owns 32 keys (its K and V in registers) and passes over the row tiles of every
//    query head that shares the key head.
// Both recompute S and dO V^T (7 products in all; one kernel would need 5 and atomics, or dQ partials, to sum dQ).
// Bound as the forward: 124 x 948 over 948, 8 heads of 64, fp16: dQ 451 us (758 TFLOP/s of its 3 products), dK and dV
// 615 us (742 of their 4), together 1066 (535 of the 5 that are needed); the least of six passes 426 and 573.
// Few owners over a long axis are split over it: fp32 partial sums in the workspace, added in a fixed order.
//
// fp16 only: P and dS are rounded to 16 bits as operands, and fp16 loses digits below 2^-14.  Both are scaled by
// powers of two that cannot overflow, from the bound |dO V^T o f - D| <= 2 max|V| |dO row|_1 / (1 - p); a small
// kernel before the others takes the maxima.
#include "attention.h"

namespace pmsst {
namespace {

using namespace attn;

struct BwdArgs {
  const void *q, *k, *v, *out, *dout;
  Strides qs, ks, vs, os, gs;
  KeyMask km;
  const float* lse;  // [B, H, N]
  void *dq, *dk, *dv;
  float *base, *delta;         // [pairs, rows_pad]: -lse in log2 units (- inf: no weight), D
  int32_t rows_pad;            // R rounded up to 64
  float *vmax, *l1;            // fp16: [pairs, kParts] maxima of |V| over the seen keys and of |dO row|_1
  float *part_q, *part_k, *part_v;  // partial sums [splits, pairs, R or M, D], NULL: not split
  Shape s;
  Grid grid;
  uint32_t tiles;              // owner tiles (rows or keys) of a pair; grid.per = tiles * splits
  int32_t tiles_per_split;
  float scale, scale_log2;
  Dropout drop;
};

constexpr int kParts = 16;
constexpr uint32_t kBoundPairs = 1u << 18;  // pairs of a grid row of attn_bound_kernel: 2^30 work-items

// Rows of a passing tile: 64, or 32 where its two LDS tiles, twice, would pass 64 KB.
template <typename T, int DP>
constexpr int bwd_tile() { return DP * sizeof(T) == 512 ? 32 : 64; }

// What stands for dO past the last row: these rows have no weight, but 0 times the last one's infinities is none.
__device__ const u32x4_t zero_row[32] = {};

// Largest power of two that keeps bound * 2^e <= 2^top (0 where the bound says nothing).
__device__ __forceinline__ int scale_exponent(float bound, int top) {
  if (!(bound > 0.f) || bound > 3e38f) return 0;
  int x;
  frexpf(bound, &x);
  const int e = top - x;
  return e < -100 ? -100 : e > 100 ? 100 : e;
}

__device__ __forceinline__ float parts_max(const float* parts) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < kParts; ++i) m = fmaxf(m, parts[i]);
  return m;
}

// fp16: dK's power of two, of a pair (P is held at 2^14 there, so dS at 2^(14 + this)).
__device__ __forceinline__ int pair_exponent(const BwdArgs& a, uint32_t pair) {
  return scale_exponent(2.f * parts_max(a.l1 + pair * kParts) * parts_max(a.vmax + pair * kParts) * a.drop.factor, 1);
}

// ---------------------------------------------------------------- one key
// Where a query sees one key alone, P is 1 whatever the score: dS, and with it dQ and dK, is zero exactly, while
// P from lse and D from O (rounded, and divided by 1 - p) would leave their rounding errors.  The sums are
// stored times 0 there: one that is no finite number (dP - dP is none then) stays none.

// Whether a key of this batch row outside [from, to) is seen.  Asked only where one key inside is: a scan that ends
// at the next one.
__device__ __forceinline__ bool seen_outside(const uint8_t* mask, int count, int from, int to) {
  if (mask == nullptr) return from > 0 || to < count;
  const int lane = threadIdx.x & 63;
  // 256 keys a step, so that four loads are on their way; an index past either end stands for the last (first) key,
  // which lies outside as well
  for (int t = to; t < count; t += 256) {
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < 256; i += 64) any |= mask[min(t + i + lane, count - 1)];
    if (__any(any != 0)) return true;
  }
  for (int t = from - 1; t >= 0; t -= 256) {
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < 256; i += 64) any |= mask[max(t - i - lane, 0)];
    if (__any(any != 0)) return true;
  }
  return false;
}

// ---------------------------------------------------------------- fp16 bounds

template <typename T>
__global__ __launch_bounds__(256) void attn_bound_kernel(BwdArgs a) {
  __shared__ float red[2][4];
  const Shape& s = a.s;
  const uint32_t pair = blockIdx.y * kBoundPairs + blockIdx.x / kParts;
  const int part = static_cast<int>(blockIdx.x % kParts);
  if (pair >= static_cast<uint32_t>(s.B) * s.Hk) return;
  const int b = static_cast<int>(pair) / s.Hk, hk = static_cast<int>(pair) - b * s.Hk;
  // 4, 8 or 16 lanes a row, 16 bytes each
  const int units = s.D / 8, log_lanes = units <= 4 ? 2 : units <= 8 ? 3 : 4;
  const int lane_u = threadIdx.x & ((1 << log_lanes) - 1), row_u = threadIdx.x >> log_lanes, step = 256 >> log_lanes;
  const int count = key_count(a.km, b, s.M);
  const T* vb = static_cast<const T*>(a.v) + b * a.vs.b + hk * a.vs.h;
  const T* gb = static_cast<const T*>(a.dout) + b * a.gs.b;
  float vm = 0.f, lm = 0.f;
#pragma unroll 4
  for (int64_t m = part * step + row_u; m < count; m += step * kParts) {
    if (a.km.mask && a.km.mask[b * a.km.stride + m] == 0) continue;
    if (lane_u < units) {
      float x[8];
      load_pack<T, 8>(vb + m * a.vs.n + 8 * lane_u, x);
#pragma unroll
      for (int i = 0; i < 8; ++i) vm = fmaxf(vm, fabsf(x[i]));
    }
  }
#pragma unroll 4
  for (int64_t r = part * step + row_u; r < s.R; r += step * kParts) {
    const int n = static_cast<int>(s.by_g.div(static_cast<uint32_t>(r))), head = hk * s.G + static_cast<int>(r) - n * s.G;
    float sum = 0.f;
    if (lane_u < units) {
      float x[8];
      load_pack<T, 8>(gb + n * a.gs.n + head * a.gs.h + 8 * lane_u, x);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += fabsf(x[i]);
    }
    lm = fmaxf(lm, group_sum(sum, 1 << log_lanes));
  }
  for (int off = 32; off > 0; off >>= 1) {
    vm = fmaxf(vm, __shfl_xor(vm, off, kWave));
    lm = fmaxf(lm, __shfl_xor(lm, off, kWave));
  }
  if ((threadIdx.x & 63) == 0) {
    red[0][threadIdx.x >> 6] = vm;
    red[1][threadIdx.x >> 6] = lm;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    a.vmax[pair * kParts + part] = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    a.l1[pair * kParts + part] = fmaxf(fmaxf(red[1][0], red[1][1]), fmaxf(red[1][2], red[1][3]));
  }
}

// ---------------------------------------------------------------- dQ

template <typename T, int DP, int NW, bool DROP>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(DP * sizeof(T) > 256 ? 1 : 2))) void attn_dq_kernel(BwdArgs a) {
  constexpr int DB = DP * sizeof(T), NS = DB / 32, DT = DP / 32;
  constexpr int BK = bwd_tile<T, DP>(), SUBS = BK / 32;
  __shared__ __attribute__((aligned(16))) char lds[kStages][2][BK * DB];
  const int lane = threadIdx.x & 63, h = lane >> 5, wave = threadIdx.x >> 6;
  uint32_t pair, sub_block;
  if (!locate(a.grid, pair, sub_block)) return;
  const uint32_t split = sub_block / a.tiles, row_tile = sub_block - split * a.tiles;
  const Shape& s = a.s;
  const int b = static_cast<int>(pair) / s.Hk, hk = static_cast<int>(pair) - b * s.Hk;
  const int d_units = s.D * static_cast<int>(sizeof(T)) / 16;

  const int r = static_cast<int>(row_tile) * 32 * NW + wave * 32 + (lane & 31);
  const bool row_ok = r < s.R;
  const bool idle = __builtin_amdgcn_readfirstlane(r) >= s.R;  // no row of this wave is there: it only moves tiles
  const int n = static_cast<int>(s.by_g.div(static_cast<uint32_t>(r))), head = hk * s.G + (r - n * s.G);
  u32x4_t qf[NS], gf[NS];
  float delta = 0.f, l1 = 0.f;
  load_frags<T, DP>(static_cast<const T*>(a.dout) + b * a.gs.b + (row_ok ? n * a.gs.n + head * a.gs.h : 0), row_ok,
                    d_units, h, gf);
  {
    u32x4_t of[NS];
    load_frags<T, DP>(static_cast<const T*>(a.out) + b * a.os.b + (row_ok ? n * a.os.n + head * a.os.h : 0), row_ok,
                      d_units, h, of);
    constexpr int E = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      float x[E], y[E];
      unpack<T>(of[i], x);
      unpack<T>(gf[i], y);
#pragma unroll
      for (int j = 0; j < E; ++j) {
        delta = fmaf(x[j], y[j], delta);
        if constexpr (std::is_same<T, f16>::value) l1 += fabsf(y[j]);
      }
    }
    delta = half_sum(delta);
  }
  hold(true);
  load_frags<T, DP>(static_cast<const T*>(a.q) + b * a.qs.b + (row_ok ? n * a.qs.n + head * a.qs.h : 0), row_ok, d_units,
                    h, qf);
  // -lse in log2 units: a row that sees no key (and one past the end) has no weight
  float base = -kInf;
  if (row_ok) {
    const float lse = a.lse[(static_cast<int64_t>(b) * s.H + head) * s.N + n];
    base = lse == -kInf ? -kInf : -lse * kLog2e;
  }
  if (h == 0 && split == 0 && r < a.rows_pad) {
    // for the other kernel, in the order and form it takes them; rows past the end have no weight
    float d = delta;
    if constexpr (std::is_same<T, f16>::value) d = ldexpf(d, pair_exponent(a, pair));
    const int64_t at = static_cast<int64_t>(pair) * a.rows_pad + r;
    a.base[at] = base + (std::is_same<T, f16>::value ? 14.f : 0.f);
    a.delta[at] = d;
  }
  int e = 0;
  if constexpr (std::is_same<T, f16>::value) {
    e = scale_exponent(2.f * half_sum(l1) * parts_max(a.vmax + pair * kParts) * a.drop.factor, 15);
    base += static_cast<float>(e);
  }

  const int count = key_count(a.km, b, s.M);
  const int all_tiles = (count + BK - 1) / BK;
  const int t0 = static_cast<int>(split) * a.tiles_per_split;
  const int t1 = min(all_tiles, t0 + a.tiles_per_split);
  const T* kb = static_cast<const T*>(a.k) + b * a.ks.b + hk * a.ks.h;
  const T* vb = static_cast<const T*>(a.v) + b * a.vs.b + hk * a.vs.h;
  const uint8_t* mask = a.km.mask ? a.km.mask + b * a.km.stride : nullptr;
  PhiloxKey key{};
  uint64_t drop0 = 0;
  if constexpr (DROP) {
    key = philox_key(a.drop.rng);
    drop0 = drop_row(s, b, head, n);
  }

  f32x16_t acc[DT]{};
  int found = 0;  // keys seen so far
  Tile<T, DP, BK, NW> kt, vt;
  auto k_at = [&](int i) { return i * a.ks.n; };
  auto v_at = [&](int i) { return i * a.vs.n; };
  kt.start(kb, t0 * BK, d_units, k_at);
  vt.start(vb, t0 * BK, d_units, v_at);
  uint8_t byte_now = 1, byte_next = 1;  // this lane's key of the mask
  auto mask_byte = [&](int t) { return mask[min(t * BK + lane, count - 1)]; };
  auto fetch = [&](int t, int stage) {
    const int key0 = t * BK;
    if (DB < 512 && key0 + BK <= count) {
      kt.fetch(lds[stage][0], BK * static_cast<int64_t>(sizeof(T)) * a.ks.n);
      vt.fetch(lds[stage][1], BK * static_cast<int64_t>(sizeof(T)) * a.vs.n);
    } else {
      kt.fetch_cut(lds[stage][0], kb, key0, count, d_units, k_at);
      vt.fetch_cut(lds[stage][1], vb, key0, count, d_units, v_at);
    }
  };
  arrive(qf);
  arrive(gf);
  asm volatile("" : "+v"(base), "+v"(delta));
  if (mask && t0 < t1) byte_next = mask_byte(t0);
  if (t0 < t1) fetch(t0, 0);
  int stage = 0;
  for (int t = t0; t < t1; ++t) {
    char* kl = lds[stage][0];
    char* vl = lds[stage][1];
    uint64_t seen = range_bits(t * BK, count);
    if (mask) {
      byte_now = byte_next;
      seen &= __ballot(byte_now != 0);
      if (t + 1 < t1) byte_next = mask_byte(t + 1);
    }
    if constexpr (BK == 32) seen &= 0xFFFFFFFFu;
    found += __popcll(seen);
    constexpr uint64_t kAll = BK == 64 ? ~uint64_t{0} : 0xFFFFFFFFu;
    vm_wait<0>();  // this wave's moves of the tile have arrived
    if (seen != kAll || d_units != kt.UNITS) {
      kt.clear(kl, seen, d_units);
      vt.clear(vl, seen, d_units);
    }
    __syncthreads();
    if (t + 1 < t1) fetch(t + 1, stage ^ 1);
    stage ^= 1;
    if (idle) continue;
#pragma unroll
    for (int u = 0; u < SUBS; ++u) {
      const uint32_t sub_seen = static_cast<uint32_t>(seen >> (32 * u));
      if (sub_seen == 0) continue;
      const int at_lane = fresh<DB>(lane);
      f32x16_t p = mma_rows<T, DP>(kl, u, qf, at_lane);
      f32x16_t dp = mma_rows<T, DP>(vl, u, gf, at_lane);
      if constexpr (DROP) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint32_t w[4];
          philox7(key, drop0 + static_cast<uint32_t>(t * (BK / 8) + 4 * u + 2 * j + h), w);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            dp[8 * j + i] = philox_keep(w, i, a.drop.limit) ? dp[8 * j + i] * a.drop.factor : 0.f;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        p[i] = __builtin_amdgcn_exp2f(fmaf(p[i], a.scale_log2, base)) * (dp[i] - delta);
      }
      if (sub_seen != 0xFFFFFFFFu) {
#pragma unroll
        for (int i = 0; i < 16; ++i) p[i] = where_bit(sub_seen >> (8 * h), reg_key(i), p[i], 0.f);
      }
      mma_cols<T, DP>(kl, u, p, acc, at_lane);
    }
  }
  const bool lone = found == 1 && !seen_outside(mask, count, t0 * BK, t1 * BK);
  if (!row_ok) return;
  const float out_scale = lone ? 0.f : std::is_same<T, f16>::value ? ldexpf(a.scale, -e) : a.scale;
  if (a.part_q) {
    const int64_t at = (static_cast<int64_t>(split) * a.grid.pairs + pair) * s.R + r;
    store_cols_f32<T, DP>(a.part_q + at * s.D, acc, out_scale, s.D, h);
  } else {
    const int64_t at = (static_cast<int64_t>(b) * s.N + n) * s.H + head;
    store_cols<T, DP>(static_cast<T*>(a.dq) + at * s.D, acc, out_scale, s.D, h);
  }
}

// ---------------------------------------------------------------- dK, dV

template <typename T, int DP, int NW, bool DROP>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(DP == 128 ? 1 : 2))) void attn_dkv_kernel(BwdArgs a) {
  constexpr int DB = DP * sizeof(T), NS = DB / 32, DT = DP / 32;
  constexpr int BQ = bwd_tile<T, DP>(), SUBS = BQ / 32;
  constexpr bool kHalf = std::is_same<T, f16>::value;
  __shared__ __attribute__((aligned(16))) char lds[kStages][2][BQ * DB];
  __shared__ __attribute__((aligned(16))) float stat[kStages][2][64];  // -lse (log2 units), D
  __shared__ __attribute__((aligned(16))) uint32_t kept[DROP ? NW : 1][DROP ? 32 : 4];
  const int lane = threadIdx.x & 63, h = lane >> 5, wave = threadIdx.x >> 6;
  uint32_t pair, sub_block;
  if (!locate(a.grid, pair, sub_block)) return;
  const uint32_t split = sub_block / a.tiles, key_tile = sub_block - split * a.tiles;
  const Shape& s = a.s;
  const int b = static_cast<int>(pair) / s.Hk, hk = static_cast<int>(pair) - b * s.Hk;
  const int d_units = s.D * static_cast<int>(sizeof(T)) / 16;
  const int count = key_count(a.km, b, s.M);
  const int block_key0 = static_cast<int>(key_tile) * 32 * NW;
  const int key0 = block_key0 + wave * 32, ki = key0 + (lane & 31);
  const bool seen = ki < count && (a.km.mask == nullptr || a.km.mask[b * a.km.stride + ki] != 0);

  const bool idle = __builtin_amdgcn_readfirstlane(key0) >= count;  // no key of this wave counts: it only moves tiles

  const int wave_key0 = __builtin_amdgcn_readfirstlane(key0);
  // (a key has two lanes)
  const int lone = __builtin_amdgcn_readfirstlane(
      __popcll(__ballot(seen)) == 2 &&
      !seen_outside(a.km.mask ? a.km.mask + b * a.km.stride : nullptr, count, wave_key0, wave_key0 + 32));

  f32x16_t dk[DT]{}, dv[DT]{};
  float k_scale = a.scale, v_scale = DROP ? a.drop.factor : 1.f;
  if (block_key0 < count) {
    u32x4_t kf[NS], vf[NS];
    load_frags<T, DP>(static_cast<const T*>(a.k) + b * a.ks.b + hk * a.ks.h + (seen ? ki * a.ks.n : 0), seen, d_units, h, kf);
    load_frags<T, DP>(static_cast<const T*>(a.v) + b * a.vs.b + hk * a.vs.h + (seen ? ki * a.vs.n : 0), seen, d_units, h, vf);
    // P' = 2^14 P (in base), dS' = P' 2^e (...): see the head of this file
    float dp_scale = DROP ? a.drop.factor : 1.f;
    if constexpr (kHalf) {
      const int e = pair_exponent(a, pair);
      dp_scale = ldexpf(dp_scale, e);
      k_scale = ldexpf(a.scale, -e - 14);
      v_scale = ldexpf(v_scale, -14);
    }

    const int tiles = (s.R + BQ - 1) / BQ;
    const int t0 = static_cast<int>(split) * a.tiles_per_split;
    const int t1 = min(tiles, t0 + a.tiles_per_split);
    const T* qb = static_cast<const T*>(a.q) + b * a.qs.b;
    const T* gb = static_cast<const T*>(a.dout) + b * a.gs.b;
    PhiloxKey key{};
    if constexpr (DROP) key = philox_key(a.drop.rng);

    Tile<T, DP, BQ, NW> qt, gt;
    auto at = [&](int i, const Strides& st) {
      const int n = static_cast<int>(s.by_g.div(static_cast<uint32_t>(i)));
      return n * st.n + (hk * s.G + (i - n * s.G)) * st.h;
    };
    auto q_at = [&](int i) { return at(i, a.qs); };
    auto g_at = [&](int i) { return at(i, a.gs); };
    const bool steps = BQ % s.G == 0;  // a tile further on is the same head again
    const int64_t q_step = BQ / s.G * static_cast<int64_t>(sizeof(T)) * a.qs.n;
    const int64_t g_step = BQ / s.G * static_cast<int64_t>(sizeof(T)) * a.gs.n;
    qt.start(qb, t0 * BQ, d_units, q_at);
    gt.start(gb, t0 * BQ, d_units, g_at);
    // waves 0 and 1 also move a tile's 64 (32) pairs of statistics, 4 bytes a lane
    const int wave0 = __builtin_amdgcn_readfirstlane(wave);
    const float* stat_src = (wave0 == 0 ? a.base : a.delta) + static_cast<int64_t>(pair) * a.rows_pad + lane;
    auto fetch = [&](int t, int stage) {
      const int row0 = t * BQ;
      if (DB < 512 && steps && row0 + BQ <= s.R) {
        qt.fetch(lds[stage][0], q_step);
        gt.fetch(lds[stage][1], g_step);
      } else {
        qt.fetch_cut(lds[stage][0], qb, row0, s.R, d_units, q_at);
        gt.fetch_cut(lds[stage][1], gb, row0, s.R, d_units, g_at, reinterpret_cast<const T*>(zero_row));
      }
      if (wave0 < 2 && (BQ == 64 || lane < BQ)) dma4_m0(stat_src + row0, __builtin_amdgcn_readfirstlane(lds_addr(stat[stage]) + 256 * wave0));
    };
    arrive(kf);
    arrive(vf);
    if (t0 < t1) fetch(t0, 0);
    int stage = 0;
    for (int t = t0; t < t1; ++t) {
      char* ql = lds[stage][0];
      char* gl = lds[stage][1];
      const float* base = stat[stage][0];
      const float* delta = stat[stage][1];
      vm_wait<0>();  // this wave's moves of the tile have arrived
      if (d_units != qt.UNITS) {
        qt.clear(ql, ~uint64_t{0}, d_units);
        gt.clear(gl, ~uint64_t{0}, d_units);
      }
      __syncthreads();
      if (t + 1 < t1) fetch(t + 1, stage ^ 1);
      stage ^= 1;
      if (idle) continue;
#pragma unroll
      for (int u = 0; u < SUBS; ++u) {
        if (t * BQ + 32 * u >= s.R) continue;
        if constexpr (DROP) {
          // 32 rows x 4 blocks of 8 keys: a lane draws 2 of them, one byte of kept bits each
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int idx = lane + 64 * j, row = idx >> 2, blk = idx & 3;
            const int i = min(t * BQ + 32 * u + row, s.R - 1);
            const int n = static_cast<int>(s.by_g.div(static_cast<uint32_t>(i)));
            uint32_t w[4];
            philox7(key, drop_row(s, b, hk * s.G + (i - n * s.G), n) + static_cast<uint32_t>(key0 / 8 + blk), w);
            reinterpret_cast<uint8_t*>(kept[wave])[idx] = static_cast<uint8_t>(philox_kept8(w, a.drop.limit));
          }
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
        hold(sizeof(T) == 4);
        const int at_lane = fresh<DB>(lane);
        f32x16_t p = mma_rows<T, DP>(ql, u, kf, at_lane);
        f32x16_t ds = mma_rows<T, DP>(gl, u, vf, at_lane);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int row = reg_key(i) + 8 * h;
          p[i] = __builtin_amdgcn_exp2f(fmaf(p[i], a.scale_log2, base[32 * u + row]));
          if constexpr (DROP) {
            const uint32_t keep = kept[wave][row];
            ds[i] = p[i] * (where_bit(keep, lane & 31, ds[i] * dp_scale, 0.f) - delta[32 * u + row]);
            p[i] = where_bit(keep, lane & 31, p[i], 0.f);
          } else {
            ds[i] = p[i] * fmaf(ds[i], dp_scale, -delta[32 * u + row]);
          }
        }
        if constexpr (DROP) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        hold(sizeof(T) == 4);
        mma_cols<T, DP>(gl, u, p, dv, at_lane);
        mma_cols<T, DP>(ql, u, ds, dk, at_lane);
      }
    }
  }
  if (ki >= s.M) return;
  if (lone) k_scale = 0.f;
  if (!seen) {
    // nothing was learnt about a key that is not seen, whatever its columns of the tiles hold
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      dk[dt] = f32x16_t{};
      dv[dt] = f32x16_t{};
    }
  }
  if (a.part_k) {
    const int64_t at = ((static_cast<int64_t>(split) * a.grid.pairs + pair) * s.M + ki) * s.D;
    store_cols_f32<T, DP>(a.part_k + at, dk, k_scale, s.D, h);
    store_cols_f32<T, DP>(a.part_v + at, dv, v_scale, s.D, h);
  } else {
    const int64_t at = ((static_cast<int64_t>(b) * s.M + ki) * s.Hk + hk) * s.D;
    store_cols<T, DP>(static_cast<T*>(a.dk) + at, dk, k_scale, s.D, h);
    store_cols<T, DP>(static_cast<T*>(a.dv) + at, dv, v_scale, s.D, h);
  }
}

// ---------------------------------------------------------------- up to 64 keys, 16 bits

// All gradients in one pass where a tile holds every key: a block of 2 waves keeps K and V in LDS and passes over
// the row tiles of its pair.  A wave takes 32 rows: its whole row of P and dP is in registers, so D is summed from
// them (unrounded, and O is not read: with few keys a rounded O would cost dQ and dK half a rounding more).  P and dS
// then go through LDS, rows down and keys across, to be the other operand of dV and dK, of which each wave owns 32
// keys.  5 products instead of 7, and every tensor is moved once: 1032 x 62 queries over 62 keys, bf16, 8 heads of 64
// take 105 us, of which the bytes need 88.
// fp16: P is held at 2^14; dS at a power of two from its own largest magnitude in the row tile, and dK's sum is
// brought to a tile's power when that is the smaller one.
// Waves that share a SIMD: fp16's scaling and the dropped bits together pass the registers of two.
template <typename T, int DP, bool DROP>
constexpr int few_waves() { return DP == 128 || (DP == 64 && DROP && std::is_same<T, f16>::value) ? 1 : 2; }

template <typename T, int DP, bool DROP>
__global__ __launch_bounds__(128) __attribute__((amdgpu_waves_per_eu(few_waves<T, DP, DROP>()))) void attn_bwd_few_kernel(BwdArgs a) {
  constexpr int DB = DP * sizeof(T), NS = DB / 32, DT = DP / 32, PB = 64 * sizeof(T);
  constexpr bool kHalf = std::is_same<T, f16>::value;
  __shared__ __attribute__((aligned(16))) char kv[2][64 * DB];
  __shared__ __attribute__((aligned(16))) char rows[2][64 * DB];
  __shared__ __attribute__((aligned(16))) char ps[2][64 * PB];
  __shared__ float most[2];
  const int lane = threadIdx.x & 63, h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t pair, split;
  if (!locate(a.grid, pair, split)) return;
  const Shape& s = a.s;
  const int b = static_cast<int>(pair) / s.Hk, hk = static_cast<int>(pair) - b * s.Hk;
  const int d_units = s.D * static_cast<int>(sizeof(T)) / 16;
  const int count = key_count(a.km, b, s.M);
  uint64_t seen = range_bits(0, count);
  if (a.km.mask) seen &= __ballot(a.km.mask[b * a.km.stride + min(lane, s.M - 1)] != 0);
  const bool lone = __popcll(seen) == 1;
  const int tiles = (s.R + 63) / 64;
  const int t0 = static_cast<int>(split) * a.tiles_per_split;
  const int t1 = min(tiles, t0 + a.tiles_per_split);
  PhiloxKey key{};
  if constexpr (DROP) key = philox_key(a.drop.rng);
  const float factor = DROP ? a.drop.factor : 1.f;

  Tile<T, DP, 64, 2> tile;  // no state: every move computes its addresses
  tile.fetch_cut(kv[0], static_cast<const T*>(a.k) + b * a.ks.b + hk * a.ks.h, 0, s.M, d_units, [&](int i) { return i * a.ks.n; });
  tile.fetch_cut(kv[1], static_cast<const T*>(a.v) + b * a.vs.b + hk * a.vs.h, 0, s.M, d_units, [&](int i) { return i * a.vs.n; });

  f32x16_t dk[DT]{}, dv[DT]{};
  constexpr int kNoSum = 101;  // above every exponent (scale_exponent's end at 100): nothing but zeros so far
  int e_sum = kNoSum;          // dk is held at 2^e_sum
  for (int t = t0; t < t1; ++t) {
    if (t > t0) __syncthreads();  // the tiles of the rows before these have been read
    auto at = [&](int i, const Strides& st) {
      const int n = static_cast<int>(s.by_g.div(static_cast<uint32_t>(i)));
      return n * st.n + (hk * s.G + (i - n * s.G)) * st.h;
    };
    tile.fetch_cut(rows[0], static_cast<const T*>(a.q) + b * a.qs.b, t * 64, s.R, d_units, [&](int i) { return at(i, a.qs); });
    tile.fetch_cut(rows[1], static_cast<const T*>(a.dout) + b * a.gs.b, t * 64, s.R, d_units, [&](int i) { return at(i, a.gs); });
    const int r = t * 64 + 32 * wave + (lane & 31);
    const bool row_ok = r < s.R;
    const int n = static_cast<int>(s.by_g.div(static_cast<uint32_t>(r))), head = hk * s.G + (r - n * s.G);
    float base = -kInf;  // -lse in log2 units: a row that sees no key (and one past the end) has no weight
    if (row_ok) {
      const float lse = a.lse[(static_cast<int64_t>(b) * s.H + head) * s.N + n];
      base = lse == -kInf ? -kInf : -lse * kLog2e;
    }
    vm_wait<0>();
    if (t == t0 && (seen != ~uint64_t{0} || d_units != tile.UNITS)) {
      tile.clear(kv[0], seen, d_units);
      tile.clear(kv[1], seen, d_units);
    }
    if (d_units != tile.UNITS) {
      tile.clear(rows[0], ~uint64_t{0}, d_units);
      tile.clear(rows[1], ~uint64_t{0}, d_units);
    }
    // rows past the end hold the last one again, whose infinities would meet their weights of 0
    if (t * 64 + 64 > s.R) tile.clear_from(rows[1], s.R - t * 64);
    __syncthreads();

    const int at_lane = fresh<256>(lane);  // whatever DB: this kernel has no registers for addresses
    uint32_t kept[2] = {0, 0};  // bit i: register i of the sub-tile
    if constexpr (DROP) {
      const uint64_t drop0 = drop_row(s, b, head, n);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t w[4];
        philox7(key, drop0 + static_cast<uint32_t>(2 * j + h), w);
        kept[j >> 1] |= philox_kept8(w, a.drop.limit) << (8 * (j & 1));
      }
      hold(true);
    }
    f32x16_t p[2], ds[2];
    {
      u32x4_t f[NS];
#pragma unroll
      for (int i = 0; i < NS; ++i) f[i] = row_frag<DB>(rows[0], 32 * wave + (at_lane & 31), i, h);
#pragma unroll
      for (int u = 0; u < 2; ++u) p[u] = mma_rows<T, DP>(kv[0], u, f, at_lane);
#pragma unroll
      for (int i = 0; i < NS; ++i) f[i] = row_frag<DB>(rows[1], 32 * wave + (at_lane & 31), i, h);
#pragma unroll
      for (int u = 0; u < 2; ++u) ds[u] = mma_rows<T, DP>(kv[1], u, f, at_lane);
    }
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint32_t bits = static_cast<uint32_t>(seen >> (32 * u)) >> (8 * h);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float w = where_bit(bits, reg_key(i), __builtin_amdgcn_exp2f(fmaf(p[u][i], a.scale_log2, base)), 0.f);
        const float dw = DROP ? where_bit(kept[u], i, ds[u][i] * factor, 0.f) : ds[u][i];
        sum[i & 1] = fmaf(w, dw, sum[i & 1]);
        ds[u][i] = dw;
        p[u][i] = w;
      }
    }
    const float delta = half_sum(sum[0] + sum[1]);
    float top = 0.f;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        ds[u][i] = p[u][i] * (ds[u][i] - delta);
        if constexpr (DROP) p[u][i] = where_bit(kept[u], i, p[u][i], 0.f);
        if constexpr (kHalf) top = fmaxf(top, fabsf(ds[u][i]));
      }
    }
    int e = 0;
    if constexpr (kHalf) {
      for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, kWave));
      if (lane == 0) most[wave] = top;
      __syncthreads();
      top = fmaxf(most[0], most[1]);
      e = top == 0.f ? kNoSum : scale_exponent(top, 15);
      const float power = ldexpf(1.f, e);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          ds[u][i] *= power;
          p[u][i] *= 16384.f;
        }
      }
      // dk stays at the smaller power of two; this tile's dS are stored at it below
      if (e < e_sum) {
        const float down = e_sum == kNoSum ? 0.f : ldexpf(1.f, e - e_sum);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
          for (int i = 0; i < 16; ++i) dk[dt][i] *= down;
        }
        e_sum = e;
      }
    }

    f32x16_t dq[DT]{};
#pragma unroll
    for (int u = 0; u < 2; ++u) mma_cols<T, DP>(kv[0], u, ds[u], dq, at_lane);
    const int row = 32 * wave + (at_lane & 31);
    if (row_ok) {
      const float dq_scale = lone ? 0.f : kHalf ? ldexpf(a.scale, -e) : a.scale;
      const int64_t to = (static_cast<int64_t>(b) * s.N + n) * s.H + head;
      store_cols<T, DP>(static_cast<T*>(a.dq) + to * s.D, dq, dq_scale, s.D, h);
    }

    // [row][key] tiles: a lane writes its row's keys, 8 consecutive ones a unit
    const float shift = kHalf ? ldexpf(1.f, e_sum - e) : 1.f;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if constexpr (kHalf) {
#pragma unroll
        for (int i = 0; i < 16; ++i) ds[u][i] *= shift;
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int to = row * PB + 16 * ((4 * u + 2 * j + h) ^ swz<PB>(row));
        *reinterpret_cast<u32x4_t*>(ps[0] + to) = pack8<T>(p[u], j);
        *reinterpret_cast<u32x4_t*>(ps[1] + to) = pack8<T>(ds[u], j);
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const u32x4_t pf = col_frag<PB>(ps[0], 16 * k, wave, at_lane), sf = col_frag<PB>(ps[1], 16 * k, wave, at_lane);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        dv[dt] = mma<T>(col_frag<DB>(rows[1], 16 * k, dt, at_lane), pf, dv[dt]);
        dk[dt] = mma<T>(col_frag<DB>(rows[0], 16 * k, dt, at_lane), sf, dk[dt]);
      }
    }
  }
  // a transposed read hands lane l the key key_row(l % 32)
  const int ki = 32 * wave + key_row(lane & 31);
  if (ki >= s.M) return;
  const float k_scale = lone ? 0.f : kHalf ? ldexpf(a.scale, -e_sum) : a.scale, v_scale = kHalf ? factor / 16384.f : factor;
  if (a.part_k) {
    const int64_t to = ((static_cast<int64_t>(split) * a.grid.pairs + pair) * s.M + ki) * s.D;
    store_cols_f32<T, DP>(a.part_k + to, dk, k_scale, s.D, h);
    store_cols_f32<T, DP>(a.part_v + to, dv, v_scale, s.D, h);
  } else {
    const int64_t to = ((static_cast<int64_t>(b) * s.M + ki) * s.Hk + hk) * s.D;
    store_cols<T, DP>(static_cast<T*>(a.dk) + to, dk, k_scale, s.D, h);
    store_cols<T, DP>(static_cast<T*>(a.dv) + to, dv, v_scale, s.D, h);
  }
}

// ---------------------------------------------------------------- partial sums

// out[b, position, head, d] = sum over splits of part[split, pair, row, d]; positions x group rows per pair
// (group 1 for the keys, whose two gradients are the grid's y).  A thread takes 4 columns.
template <typename T>
__global__ __launch_bounds__(256) void attn_sum_kernel(const float* part, void* out, const float* part1, void* out1, int splits, int64_t pairs,
                                                       int32_t heads, int32_t kv_heads, int32_t group, int32_t positions,
                                                       int32_t dim) {
  if (blockIdx.y != 0) {
    part = part1;
    out = out1;
  }
  const int64_t quads = dim / 4, rows = static_cast<int64_t>(positions) * group, total = pairs * rows * quads;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= total) return;
  const int64_t row = i / quads, quad = i - row * quads, pair = row / rows, r = row - pair * rows;
  const int64_t b = pair / kv_heads, hk = pair - b * kv_heads, n = r / group, head = hk * group + (r - n * group);
  float o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int k = 0; k < splits; ++k) {
    float x[4];
    load_pack<float, 4>(part + ((k * pairs * rows + row) * quads + quad) * 4, x);
#pragma unroll
    for (int c = 0; c < 4; ++c) o[c] += x[c];
  }
  store_pack<T, 4>(static_cast<T*>(out) + ((b * positions + n) * heads + head) * dim + 4 * quad, o);
}

// ---------------------------------------------------------------- host

struct BwdPlan {
  bool few;  // up to 64 keys of 16-bit types: attn_bwd_few_kernel (fp32's tiles would leave a CU one block of 2 waves)
  int nw_q, nw_k;
  int64_t q_tiles, q_splits, q_per, k_tiles, k_splits, k_per;
};

// Splits as in the forward: as many as give every CU two blocks, of at least 128 keys (rows) each.
BwdPlan plan_backward(const Shape& s, int dtype) {
  const bool wide = padded_dim(s.D) * static_cast<int>(dtype_size(dtype)) == 512;
  const int64_t bk = wide ? 32 : 64;
  const int64_t pairs = int64_t{s.B} * s.Hk, want = 2 * num_cus();
  auto split = [&](int64_t owners, int64_t along, int64_t& splits, int64_t& per) {
    const int64_t tiles = std::max<int64_t>(1, (along + bk - 1) / bk);
    splits = 1;
    if (owners < want) splits = std::max<int64_t>(1, std::min((want + owners - 1) / owners, along / 128));
    per = (tiles + splits - 1) / splits;
    splits = (tiles + per - 1) / per;
  };
  BwdPlan p;
  p.nw_q = s.R <= 64 && !wide ? 2 : 4;
  p.nw_k = s.M <= 64 && dtype == PMSST_F32 && !wide ? 2 : 4;  // (16-bit types with so few keys take p.few)
  p.q_tiles = (int64_t{s.R} + 32 * p.nw_q - 1) / (32 * p.nw_q);
  p.k_tiles = (int64_t{s.M} + 32 * p.nw_k - 1) / (32 * p.nw_k);
  p.few = s.M > 0 && s.M <= 64 && dtype != PMSST_F32;
  split(pairs * p.q_tiles, s.M, p.q_splits, p.q_per);
  split(std::max<int64_t>(1, pairs * (p.few ? 1 : p.k_tiles)), s.R, p.k_splits, p.k_per);
  return p;
}

struct BwdSpace {
  size_t delta, bound, part_q, part_k, total;
};

BwdSpace bwd_space(const Shape& s, const BwdPlan& p, int dtype) {
  const size_t pairs = static_cast<size_t>(s.B) * s.Hk;
  BwdSpace w;
  w.delta = p.few ? 0 : align_up(pairs * align_up(s.R, 64) * 4, 256);
  w.bound = dtype == PMSST_F16 && !p.few ? align_up(pairs * kParts * 4, 256) : 0;
  w.part_q = p.q_splits > 1 ? align_up(static_cast<size_t>(p.q_splits) * pairs * s.R * s.D * 4, 256) : 0;
  w.part_k = p.k_splits > 1 ? align_up(static_cast<size_t>(p.k_splits) * pairs * s.M * s.D * 4, 256) : 0;
  w.total = 2 * w.delta + 2 * w.bound + w.part_q + 2 * w.part_k;
  return w;
}

template <typename T, int DP, int NW>
int launch_dq(const BwdArgs& a, bool drop, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(grid_blocks(a.grid)));
  if (drop) attn_dq_kernel<T, DP, NW, true><<<grid, 64 * NW, 0, stream>>>(a);
  else attn_dq_kernel<T, DP, NW, false><<<grid, 64 * NW, 0, stream>>>(a);
  return check_launch("attn_dq_kernel");
}

template <typename T, int DP>
int launch_dq(const BwdArgs& a, int nw, bool drop, hipStream_t stream) {
  if constexpr (DP * sizeof(T) != 512) {
    if (nw == 2) return launch_dq<T, DP, 2>(a, drop, stream);
  }
  return launch_dq<T, DP, 4>(a, drop, stream);
}

template <typename T, int DP, int NW>
int launch_dkv(const BwdArgs& a, bool drop, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(grid_blocks(a.grid)));
  if (drop) attn_dkv_kernel<T, DP, NW, true><<<grid, 64 * NW, 0, stream>>>(a);
  else attn_dkv_kernel<T, DP, NW, false><<<grid, 64 * NW, 0, stream>>>(a);
  return check_launch("attn_dkv_kernel");
}

template <typename T, int DP>
int launch_dkv(const BwdArgs& a, int nw, bool drop, hipStream_t stream) {
  if constexpr (sizeof(T) == 4 && DP < 128) {
    if (nw == 2) return launch_dkv<T, DP, 2>(a, drop, stream);
  }
  return launch_dkv<T, DP, 4>(a, drop, stream);
}

template <typename T>
int sum_rows(const BwdArgs& a, const BwdPlan& p, hipStream_t stream) {
  const Shape& s = a.s;
  const int64_t pairs = int64_t{s.B} * s.Hk, blocks = (pairs * s.R * (s.D / 4) + 255) / 256;
  attn_sum_kernel<T><<<dim3(static_cast<uint32_t>(blocks)), 256, 0, stream>>>(
      a.part_q, a.dq, nullptr, nullptr, static_cast<int>(p.q_splits), pairs, s.H, s.Hk, s.G, s.N, s.D);
  return check_launch("attn_sum_kernel");
}

template <typename T>
int sum_keys(const BwdArgs& a, const BwdPlan& p, hipStream_t stream) {
  const Shape& s = a.s;
  const int64_t pairs = int64_t{s.B} * s.Hk, blocks = (pairs * s.M * (s.D / 4) + 255) / 256;
  attn_sum_kernel<T><<<dim3(static_cast<uint32_t>(blocks), 2), 256, 0, stream>>>(
      a.part_k, a.dk, a.part_v, a.dv, static_cast<int>(p.k_splits), pairs, s.Hk, s.Hk, 1, s.M, s.D);
  return check_launch("attn_sum_kernel");
}

template <typename T, int DP>
int run_bwd(BwdArgs& a, const BwdPlan& p, hipStream_t stream) {
  const bool drop = a.drop.limit != 0;
  const int64_t pairs = int64_t{a.s.B} * a.s.Hk;
  if constexpr (sizeof(T) == 2) {
    if (p.few) {
      a.tiles_per_split = static_cast<int32_t>(p.k_per);
      a.grid = make_grid(pairs, p.k_splits);
      const dim3 grid(static_cast<uint32_t>(grid_blocks(a.grid)));
      if (drop) attn_bwd_few_kernel<T, DP, true><<<grid, 128, 0, stream>>>(a);
      else attn_bwd_few_kernel<T, DP, false><<<grid, 128, 0, stream>>>(a);
      const int rc = check_launch("attn_bwd_few_kernel");
      return rc == PMSST_OK && a.part_k ? sum_keys<T>(a, p, stream) : rc;
    }
  }
  if constexpr (std::is_same<T, f16>::value) {
    const dim3 grid(static_cast<uint32_t>(std::min<int64_t>(pairs, kBoundPairs) * kParts),
                    static_cast<uint32_t>((pairs + kBoundPairs - 1) / kBoundPairs));
    attn_bound_kernel<T><<<grid, 256, 0, stream>>>(a);
    const int rc = check_launch("attn_bound_kernel");
    if (rc != PMSST_OK) return rc;
  }
  a.tiles = static_cast<uint32_t>(p.q_tiles);
  a.tiles_per_split = static_cast<int32_t>(p.q_per);
  a.grid = make_grid(pairs, p.q_tiles * p.q_splits);
  int rc = launch_dq<T, DP>(a, p.nw_q, drop, stream);
  if (rc == PMSST_OK && a.part_q) rc = sum_rows<T>(a, p, stream);
  if (rc != PMSST_OK || a.s.M == 0) return rc;
  a.tiles = static_cast<uint32_t>(p.k_tiles);
  a.tiles_per_split = static_cast<int32_t>(p.k_per);
  a.grid = make_grid(pairs, p.k_tiles * p.k_splits);
  rc = launch_dkv<T, DP>(a, p.nw_k, drop, stream);
  return rc == PMSST_OK && a.part_k ? sum_keys<T>(a, p, stream) : rc;
}

template <typename T>
int run_bwd(BwdArgs& a, const BwdPlan& p, hipStream_t stream) {
  return a.s.D <= 32 ? run_bwd<T, 32>(a, p, stream) : a.s.D <= 64 ? run_bwd<T, 64>(a, p, stream) : run_bwd<T, 128>(a, p, stream);
}

}  // namespace
}  // namespace pmsst

extern "C" {

size_t pmsst_cross_attention_backward_workspace_size(int64_t batch, int64_t queries, int64_t keys, int64_t heads,
                                                     int64_t kv_heads, int64_t head_dim, int dtype) {
  pmsst::attn::Shape s;
  if (pmsst::attn::make_shape("pmsst_cross_attention_backward", batch, queries, keys, heads, kv_heads, head_dim, dtype,
                              s) != PMSST_OK ||
      s.B == 0 || s.N == 0)
    return 0;
  return pmsst::bwd_space(s, pmsst::plan_backward(s, dtype), dtype).total;
}

int pmsst_cross_attention_backward(const void* grad_out, const int64_t* grad_out_strides, const void* q,
                                   const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v,
                                   const int64_t* v_strides, const void* out, const float* lse, const uint8_t* key_mask,
                                   int64_t key_mask_stride, const int32_t* key_lengths, void* grad_q, void* grad_k,
                                   void* grad_v, int64_t batch, int64_t queries, int64_t keys, int64_t heads,
                                   int64_t kv_heads, int64_t head_dim, double scale, double dropout_p, const int64_t* rng,
                                   int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace pmsst;
  using namespace pmsst::attn;
  const char* what = "pmsst_cross_attention_backward";
  BwdArgs a{};
  int rc = make_shape(what, batch, queries, keys, heads, kv_heads, head_dim, dtype, a.s);
  if (rc != PMSST_OK) return rc;
  PMSST_REQUIRE(scale > 0.0 && scale < 1e30, "%s: scale must be positive", what);
  PMSST_REQUIRE(dropout_p >= 0.0 && dropout_p < 1.0, "%s: the dropout probability must lie in [0, 1)", what);
  if (batch == 0) return PMSST_OK;
  PMSST_REQUIRE(queries > 0, "%s: queries must be positive (the keys' gradients are zero without any)", what);
  PMSST_REQUIRE(grad_out && q && out && lse && grad_q && (keys == 0 || (k && v && grad_k && grad_v)), "%s: null pointer",
                what);
  if ((rc = make_strides(what, grad_out, grad_out_strides, queries, heads, head_dim, dtype, a.gs)) != PMSST_OK) return rc;
  if ((rc = make_strides(what, out, nullptr, queries, heads, head_dim, dtype, a.os)) != PMSST_OK) return rc;
  if ((rc = make_strides(what, q, q_strides, queries, heads, head_dim, dtype, a.qs)) != PMSST_OK) return rc;
  if ((rc = make_strides(what, k, k_strides, keys, kv_heads, head_dim, dtype, a.ks)) != PMSST_OK) return rc;
  if ((rc = make_strides(what, v, v_strides, keys, kv_heads, head_dim, dtype, a.vs)) != PMSST_OK) return rc;
  PMSST_REQUIRE(((reinterpret_cast<uintptr_t>(grad_q) | reinterpret_cast<uintptr_t>(grad_k) |
                  reinterpret_cast<uintptr_t>(grad_v)) & 15) == 0,
                "%s: gradients must be 16-byte aligned", what);
  a.drop = make_dropout(dropout_p, rng);
  PMSST_REQUIRE(rng || a.drop.limit == 0, "%s: null pointer (rng)", what);
  const BwdPlan p = plan_backward(a.s, dtype);
  const BwdSpace w = bwd_space(a.s, p, dtype);
  if (w.total > 0 && (workspace == nullptr || workspace_bytes < w.total))
    return fail(PMSST_EWORKSPACE, "%s: workspace of %zu bytes needed, %zu given", what, w.total, workspace_bytes);
  PMSST_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "%s: workspace must be 16-byte aligned", what);
  a.q = q;
  a.k = k;
  a.v = v;
  a.out = out;
  a.dout = grad_out;
  a.km = {key_mask, key_mask_stride, key_lengths};
  a.lse = lse;
  a.dq = grad_q;
  a.dk = grad_k;
  a.dv = grad_v;
  char* at = static_cast<char*>(workspace);
  a.rows_pad = static_cast<int32_t>(align_up(a.s.R, 64));
  a.base = reinterpret_cast<float*>(at);
  at += w.delta;
  a.delta = reinterpret_cast<float*>(at);
  at += w.delta;
  a.vmax = reinterpret_cast<float*>(at);
  at += w.bound;
  a.l1 = reinterpret_cast<float*>(at);
  at += w.bound;
  if (w.part_q) a.part_q = reinterpret_cast<float*>(at);
  at += w.part_q;
  if (w.part_k) {
    a.part_k = reinterpret_cast<float*>(at);
    a.part_v = reinterpret_cast<float*>(at + w.part_k);
  }
  const int64_t per = p.few ? p.k_splits : std::max(p.q_tiles * p.q_splits, p.k_tiles * p.k_splits);
  PMSST_REQUIRE(grid_fits(batch * kv_heads, per), "%s: too many rows for one call", what);
  a.scale = static_cast<float>(scale);
  a.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case PMSST_F32: return run_bwd<float>(a, p, st);
    case PMSST_F16: return run_bwd<f16>(a, p, st);
    default: return run_bwd<bf16>(a, p, st);
  }
}

}  // extern "C"
