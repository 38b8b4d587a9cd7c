// Local attention backward.  With P the weights, recomputed from the saved lse, and dO the output's gradient:
//   D  = rowsum(dO o O)          dV = P^T dO          dS = P o (dO V^T - D)
//   dQ = scale dS K              dK = scale dS^T Q    dbias[c] = sum of dS over the pairs whose distance has bucket c
//
// Two kernels as in the cross attention, so that every sum has one owner: local_dq_kernel (a wave owns 32 queries and
// passes over the frames they see; it also writes D) and local_dkv_kernel (a wave owns 32 frames
// and passes over the queries that see them).
//
// The first frames (sinks) are seen by every later query: the block of their keys would pass over all rows while others
// pass over a window's.  Their rows past the window go to blocks of their own, as many tiles each as an ordinary block
// has; the sums meet in fp32 in the workspace and a third kernel adds them.  So do the sums of blocks that are split over
// their queries, where there are few of them.
//
// The bias's gradient sums dS along diagonals, in local_dkv_kernel.  A wave's 32 x 32 tile holds 63 of them, with one
// frame a lane and queries in registers: 31 additions with a lane move in the operand bring every diagonal into one lane
// (add_diagonals), and two more add them to the wave's own bins in LDS, one a distance.  Tiles beyond the table's
// distances add up in registers.  Every block leaves its bins in the workspace, and two small kernels add the blocks and the
// distances of a bucket, in a fixed order.  (With the bins summed by bucket in every block, that sum took half of the
// kernel's time: 16 x 2760 queries, window of 1024, 320 buckets, 1074 us against 552.)
#include "attention_bwd.h"
#include "local_attention.h"

namespace pmsst {
namespace {

using namespace attn;

struct BwdArgs {
  const void *q, *k, *v, *out, *dout;
  Strides qs, ks, vs, os, gs;
  KeyMask km;
  Window w;
  BiasArgs bias;
  const int32_t *order, *first;  // bucket_of's indexes by bucket, and where each bucket's begin
  int32_t cut;                   // indexes cut off on either side of the bias's table
  const float* lse;  // [B, H, N]
  void *dq, *dk, *dv, *dbias;
  float *base, *delta;  // [B * H, rows_pad]: -lse in log2 units (- inf: no weight), D
  uint32_t* lone;       // [B * H, rows_pad / 32]: a bit for each query that sees one frame alone
  int32_t rows_pad;     // N rounded up to 64
  float *vmax, *l1;     // fp16: [pairs, kParts] maxima of |V| over the seen frames and of |dO row|_1
  // of the keys that several blocks share: [splits, pairs, part_keys, D], then the sinks' later rows' [chunks, pairs, sink_rows, D]
  float *part_k, *part_v;
  float* part_bias;     // [H, B * blocks of a pair in local_dkv_kernel, span]: sums by falling distance
  float* sum_bias;      // [H, groups of kSumRows of those, span]
  Shape s;
  Grid grid;
  uint32_t row_begin, row_end;  // the row tiles of a launch of local_dq_kernel
  uint32_t key_tiles, splits, sink_tiles, chunks;
  int32_t chunk_tiles, part_keys, sink_rows;
  bool late_first;
  float scale, scale_log2, bias_unit;
  struct { float factor; } drop;  // what attn_bound_kernel's bound is multiplied by: no dropout here
};

// Rows of a passing tile: 64, or 32 where its two LDS tiles, twice, would pass 64 KB.
template <typename T, int DP>
constexpr int local_tile() { return DP * sizeof(T) == 512 ? 32 : 64; }

// fp16: dK's power of two, of a pair (P is held at 2^14 there, so dS at 2^(14 + this)).
__device__ __forceinline__ int pair_exponent(const BwdArgs& a, uint32_t pair) {
  return scale_exponent(2.f * parts_max(a.l1 + pair * kParts) * parts_max(a.vmax + pair * kParts), 1);
}

// ---------------------------------------------------------------- diagonals
constexpr int kBinPad = 16;  // places on either side of a wave's bins that add_diagonals adds zeros to

// x of lane l + N (l - N for N < 0) of the same row of 16 lanes; 0 past its ends.
template <int N>
__device__ __forceinline__ float row_moved(float x) {
  if constexpr (N == 0) return x;
  constexpr int kCtrl = N > 0 ? 0x100 + N : 0x110 - N;  // row_shl, row_shr
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), kCtrl, 0xF, 0xF, true));
}
__device__ __forceinline__ float keep_bits(float x, uint32_t m) {
  return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x) & m);
}

// Adds 8 queries c = C .. 7 in a row over a row of 16 frames r: those with r >= c to lane r - c of `on`, the others to
// lane r - c + 16 of `past`.
template <int C>
__device__ __forceinline__ void add_run(const float (&x)[8], float& on, float& past) {
  on += row_moved<C>(x[C]);
  if constexpr (C > 0) past += row_moved<C - 16>(x[C]);
  if constexpr (C < 7) add_run<C + 1>(x, on, past);
}

// Adds the diagonals of x (lane l: frame l % 32, queries reg_key(i) + 8 (l / 32)) to bins[query - frame], this wave's alone
// (or with frames and queries exchanged, to bins[frame - query]).
// A query's value moves to the lane of its diagonal inside its row of 16 lanes, in the operand of the addition; what
// leaves the row's low end goes on 16 lanes up in the next sum.  With h = l / 32, p = l / 16 % 2 and i = l % 16, the three
// sums then hold frame - query = 16 p - 8 h + i less 0, 16 and 32.  The rows' parts that mean the same are added, and
// exchanging the halves leaves -32 + l of the lower half in one register and -40 + l of the upper half in another.
__device__ __forceinline__ void add_diagonals(float* bins, const f32x16_t& x, int lane) {
  float near[8], far[8];
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    near[c] = x[c];
    far[c] = x[8 + c];
  }
  float a = 0.f, b = 0.f, c = 0.f;
  add_run<0>(near, a, b);
  add_run<0>(far, b, c);
  uint32_t even = (lane & 16) ? 0u : ~0u;
  asm volatile("" : "+v"(even));  // a register's mask, not one of the few scalar pairs
  const uint32_t u = __builtin_bit_cast(uint32_t, b);
  const auto rows = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t of_even = rows[0], of_odd = rows[1];  // in odd rows the even ones' b, in even rows the odd ones'
  a += keep_bits(__builtin_bit_cast(float, of_odd), even);
  c += keep_bits(__builtin_bit_cast(float, of_even), ~even);
  const auto halves = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, c), __builtin_bit_cast(uint32_t, a), false, false);
  const uint32_t first = halves[0], second = halves[1];
  // Lanes beyond the diagonals add 0, up to 9 places past them.  A lane's places in the two additions differ, and the
  // compiler may not read the second before it writes the first: they are other lanes'.
  asm volatile("" ::: "memory");
  bins[32 - lane] += __builtin_bit_cast(float, first);
  asm volatile("" ::: "memory");
  bins[40 - lane] += __builtin_bit_cast(float, second);
  asm volatile("" ::: "memory");
}

// ---------------------------------------------------------------- dQ

// TWICE: a pass for D before the one for dQ (16 bits; see the loop).
template <typename T, int DP, int NW, bool BIAS, bool TWICE>
__global__ __launch_bounds__(64 * NW)
__attribute__((amdgpu_waves_per_eu(DP * sizeof(T) > 256 || (TWICE && DP == 128) ? 1 : 2))) void local_dq_kernel(BwdArgs a) {
  constexpr int DB = DP * sizeof(T), NS = DB / 32, DT = DP / 32;
  constexpr int BK = local_tile<T, DP>(), SUBS = BK / 32;
  constexpr bool kHalf = std::is_same<T, f16>::value;
  __shared__ __attribute__((aligned(16))) char lds[kStages][2][BK * DB];
  extern __shared__ float table[];  // the bias by distance, then for each wave whether it saw an entry that hides
  const int lane = threadIdx.x & 63, h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t pair, sub_block;
  if (!locate(a.grid, pair, sub_block)) return;
  const Shape& s = a.s;
  const uint32_t tile_up = s.by_g.div(sub_block), g = sub_block - tile_up * static_cast<uint32_t>(s.G);
  const uint32_t row_tile = a.late_first ? a.row_end - 1 - tile_up : a.row_begin + tile_up;
  const int b = static_cast<int>(pair) / s.Hk, hk = static_cast<int>(pair) - b * s.Hk, head = hk * s.G + static_cast<int>(g);
  const int d_units = s.D * static_cast<int>(sizeof(T)) / 16;
  const int64_t bh = static_cast<int64_t>(b) * s.H + head;

  const int n0 = static_cast<int>(row_tile) * 32 * NW, n = n0 + wave * 32 + (lane & 31);
  const bool row_ok = n < s.N;
  const bool idle = n0 + wave * 32 >= s.N;  // no query of this wave is there: it only moves tiles
  const int n_at = row_ok ? n : 0;
  u32x4_t qf[NS], gf[NS];
  float delta = 0.f, l1 = 0.f;
  load_frags<T, DP>(static_cast<const T*>(a.dout) + b * a.gs.b + head * a.gs.h + n_at * a.gs.n, row_ok, d_units, h, gf);
  {
    u32x4_t of[NS];
    load_frags<T, DP>(static_cast<const T*>(a.out) + b * a.os.b + head * a.os.h + n_at * a.os.n, row_ok, d_units, h, of);
    constexpr int E = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      float x[E], y[E];
      unpack<T>(of[i], x);
      unpack<T>(gf[i], y);
#pragma unroll
      for (int j = 0; j < E; ++j) {
        delta = fmaf(x[j], y[j], delta);
        if constexpr (kHalf) l1 += fabsf(y[j]);
      }
    }
    delta = half_sum(delta);
  }
  hold(true);
  load_frags<T, DP>(static_cast<const T*>(a.q) + b * a.qs.b + head * a.qs.h + n_at * a.qs.n, row_ok, d_units, h, qf);
  // -lse in log2 units: a row that sees no frame (and one past the end) has no weight
  float base = -kInf;
  if (row_ok) {
    const float lse = a.lse[bh * s.N + n];
    base = lse == -kInf ? -kInf : -lse * kLog2e;
  }

  const int count = key_count(a.km, b, s.M);
  const int start = start_of(a.w, b);
  const int p0 = start + n0 + wave * 32, pos = start + n;
  const TileList list = tiles_of<BK>(a.w, start + n0, start + min(n0 + 32 * NW, s.N) - 1, count);
  const T* kb = static_cast<const T*>(a.k) + b * a.ks.b + hk * a.ks.h;
  const T* vb = static_cast<const T*>(a.v) + b * a.vs.b + hk * a.vs.h;
  const uint8_t* mask = a.km.mask ? a.km.mask + b * a.km.stride : nullptr;
  const int low = low_of(a.w, pos), high = high_of(a.w, pos, count);
  const int sinks = min(a.w.sinks, high);
  auto mask_byte = [&](int t) { return mask[min(t * BK + lane, count - 1)]; };
  constexpr uint64_t kAll = BK == 64 ? ~uint64_t{0} : 0xFFFFFFFFu;

  // Where a query sees one frame alone, P is 1 whatever the score: dS, and with it dQ and dK, is zero exactly, while P
  // from lse and D from O would leave their rounding errors.  (What the bias hides is taken off below, with its table.)
  int found = 0;
  if (mask == nullptr) {
    found = max(0, high - low) + max(0, min(sinks, low));
  } else {
    for (int i = 0; i < list.total; ++i) {  // ends where every query has two
      const int key0 = list.at(i) * BK;
      uint64_t seen = range_bits(key0, count) & __ballot(mask_byte(list.at(i)) != 0) & kAll;
#pragma unroll
      for (int u = 0; u < SUBS; ++u) {
        const int at = key0 + 32 * u;
        found += __popc(static_cast<uint32_t>(seen >> (32 * u)) & frames_seen(low, high, a.w.sinks, at));
      }
      if (!__any(row_ok && found < 2)) break;
    }
  }
  uint32_t lone = static_cast<uint32_t>(__ballot(found == 1));
  float alive = found == 1 ? 0.f : 1.f;

  const float row_base = base;
  int e = 0;
  if constexpr (kHalf) {
    e = scale_exponent(2.f * half_sum(l1) * parts_max(a.vmax + pair * kParts), 15);
    base += static_cast<float>(e);
  }

  f32x16_t acc[DT]{};
  Tile<T, DP, BK, NW> kt, vt;
  auto k_at = [&](int i) { return i * a.ks.n; };
  auto v_at = [&](int i) { return i * a.vs.n; };
  const int64_t k_step = BK * static_cast<int64_t>(sizeof(T)) * a.ks.n, v_step = BK * static_cast<int64_t>(sizeof(T)) * a.vs.n;
  uint8_t byte_now = 1, byte_next = 1;  // this lane's key of the mask
  auto fetch = [&](int i, int stage) {
    const int key0 = list.at(i) * BK;
    if (DB < 512 && key0 + BK <= count) {
      if (i == list.sink && i != 0) {
        skip(kt, (list.first - i) * k_step);
        skip(vt, (list.first - i) * v_step);
      }
      kt.fetch(lds[stage][0], k_step);
      vt.fetch(lds[stage][1], v_step);
    } else {
      kt.fetch_cut(lds[stage][0], kb, key0, count, d_units, k_at);
      vt.fetch_cut(lds[stage][1], vb, key0, count, d_units, v_at);
    }
  };
  arrive(qf);
  arrive(gf);
  asm volatile("" : "+v"(base), "+v"(delta));
  auto begin = [&] {
    if (list.total == 0) return;
    kt.start(kb, list.at(0) * BK, d_units, k_at);
    vt.start(vb, list.at(0) * BK, d_units, v_at);
    if (mask) byte_next = mask_byte(list.at(0));
    fetch(0, 0);
  };
  begin();
  const float* lane_table = nullptr;  // this lane's entry for frame 0
  float far_low = 0.f, far_high = 0.f, rest[2] = {0.f, 0.f};
  if constexpr (BIAS) {
    const int entries = 2 * a.bias.distance + 1 + 2 * kPad;
    const bool own = __any(fill_bias<T, false>(table, a.bias, s.H, head, a.bias_unit, 64 * NW));
    if (lane == 0) table[entries + wave] = own ? 1.f : 0.f;
    __syncthreads();
    far_low = table[0];
    far_high = table[entries - 1];
    lane_table = table + (a.bias.distance + kPad + 8 * h - pos);
    float hides = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) hides += table[entries + w];
    if (hides != 0.f) {
      // frames that the bias hides are not seen: counted again, until every query has two
      found = 0;
      for (int i = 0; i < list.total && __any(row_ok && found < 2); ++i) {
        const int key0 = list.at(i) * BK;
        uint64_t seen = range_bits(key0, count) & kAll;
        if (mask) seen &= __ballot(mask_byte(list.at(i)) != 0);
#pragma unroll
        for (int u = 0; u < SUBS; ++u) {
          const int at = key0 + 32 * u;
          found += __popc(static_cast<uint32_t>(seen >> (32 * u)) & frames_seen(low, high, a.w.sinks, at) &
                          bias_shows(table, a.bias.distance, pos, at));
        }
      }
      lone = static_cast<uint32_t>(__ballot(found == 1));
      alive = found == 1 ? 0.f : 1.f;
    }
  }
  // What a row's dS adds up to is 0 but for D's error (out is rounded, and so were the weights it is a sum of); with it, D is
  // rowsum(P o dP) to fp32's precision.  Of 16-bit rows that see few frames, D's error would be as large as the roundings
  // of dS and dQ together (windows of 39 frames: dQ 1.53 times one rounding's error, with the pass 1.42), so their
  // blocks pass over the tiles once for D alone; where many are seen it is lost among them.  (A kernel of its own: the two
  // passes hold the registers of a third wave, 456 us against 620 for 124 x 948 queries.)
#pragma unroll 1
  for (bool first_pass = TWICE;; first_pass = false) {
    int stage = 0;
    for (int i = 0; i < list.total; ++i) {
      const int t = list.at(i);
      char* kl = lds[stage][0];
      char* vl = lds[stage][1];
      uint64_t seen = range_bits(t * BK, count);
      if (mask) {
        byte_now = byte_next;
        seen &= __ballot(byte_now != 0);
        if (i + 1 < list.total) byte_next = mask_byte(list.at(i + 1));
      }
      seen &= kAll;
      vm_wait<0>();  // this wave's moves of the tile have arrived
      if (seen != kAll || d_units != kt.UNITS) {
        kt.clear(kl, seen, d_units);
        vt.clear(vl, seen, d_units);
      }
      __syncthreads();
      if (i + 1 < list.total) fetch(i + 1, stage ^ 1);
      stage ^= 1;
      if (idle) continue;
#pragma unroll
      for (int u = 0; u < SUBS; ++u) {
        const int key0 = t * BK + 32 * u;
        const uint32_t sub_seen = static_cast<uint32_t>(seen >> (32 * u));
        const Sees what = sees(a.w, p0, key0, count);
        if (sub_seen == 0 || what == Sees::kNone) continue;
        const int at_lane = fresh<DB>(lane);
        f32x16_t p;
        if constexpr (BIAS) {
          bool upper;
          if (bias_far(key0 - p0 - 31, a.bias.distance, upper)) {
            const float far = upper ? far_high : far_low;
#pragma unroll
            for (int r = 0; r < 16; ++r) p[r] = far;
          } else {
            p = bias_tile(lane_table + key0);
          }
          p = mma_rows_from<T, DP>(p, kl, u, qf, at_lane);
        } else {
          p = mma_rows<T, DP>(kl, u, qf, at_lane);
        }
        const f32x16_t dp = mma_rows<T, DP>(vl, u, gf, at_lane);
        if (what == Sees::kSome || sub_seen != 0xFFFFFFFFu) {
          uint32_t bits = sub_seen;
          if (what == Sees::kSome) bits &= frames_seen(low, high, a.w.sinks, key0);
          bits >>= 8 * h;
#pragma unroll
          for (int r = 0; r < 16; ++r) p[r] = where_bit(bits, reg_key(r), p[r], -kInf);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          p[r] = __builtin_amdgcn_exp2f(fmaf(p[r], a.scale_log2, base)) * (dp[r] - delta);
        }
        if (lone != 0) {
#pragma unroll
          for (int r = 0; r < 16; ++r) p[r] *= alive;
        }
        if constexpr (BIAS || TWICE) {
#pragma unroll
          for (int r = 0; r < 16; ++r) rest[r & 1] += p[r];
        }
        if (TWICE && first_pass) continue;
        mma_cols<T, DP>(kl, u, p, acc, at_lane);
      }
    }
    if (!TWICE || !first_pass) break;
    const float total = half_sum(rest[0] + rest[1]);
    delta += kHalf ? ldexpf(total, -e) : total;
    rest[0] = rest[1] = 0.f;
    __syncthreads();  // every wave has read the last tile
    begin();
  }
  if (row_ok) {
    const float out_scale = kHalf ? ldexpf(a.scale, -e) : a.scale;
    const int64_t at = (static_cast<int64_t>(b) * s.N + n) * s.H + head;
    store_cols<T, DP>(static_cast<T*>(a.dq) + at * s.D, acc, out_scale, s.D, h);
  }
  // for the other kernel, in the form it takes them; rows past the end have no weight
  if constexpr (BIAS) {
    // the bias's gradient needs D to fp32's precision (with D from out it is 3e-4 off)
    const float total = half_sum(rest[0] + rest[1]);
    delta += kHalf ? ldexpf(total, -e) : total;
  }
  if (h == 0 && n < a.rows_pad) {
    if constexpr (kHalf) delta = ldexpf(delta, pair_exponent(a, pair));
    const int64_t at = bh * a.rows_pad + n;
    a.base[at] = row_base + (kHalf ? 14.f : 0.f);
    a.delta[at] = delta;
    if (lane == 0) a.lone[at / 32] = lone;
  }
}

// The blocks' bins become the buckets' sums in two steps, each in a fixed order: `rows` blocks' at a time by distance,
// then those sums by bucket.
constexpr int kSumRows = 256;
__global__ __launch_bounds__(1024) void local_bins_sum_kernel(const float* bins, float* sums, int64_t blocks, int64_t parts, int span) {
  __shared__ float red[16][64];
  const int x = threadIdx.x & 63, y = threadIdx.x >> 6, at = static_cast<int>(blockIdx.y) * 64 + x;
  const int64_t head = blockIdx.x / parts, part = blockIdx.x - head * parts, from = part * kSumRows;
  const int64_t to = from + kSumRows < blocks ? from + kSumRows : blocks;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  if (at < span) {
    const float* bin = bins + head * blocks * span + at;
    int64_t k = from + y;
    for (; k + 48 < to; k += 64) {
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[j] += bin[(k + 16 * j) * span];
    }
    for (; k < to; k += 16) sum[0] += bin[k * span];
  }
  red[y][x] = (sum[0] + sum[1]) + (sum[2] + sum[3]);
  __syncthreads();
  if (y != 0 || at >= span) return;
  float t = 0.f;
#pragma unroll
  for (int j = 0; j < 16; ++j) t += red[j][x];
  sums[blockIdx.x * static_cast<int64_t>(span) + at] = t;
}

// dbias[bucket, head]; a wave a bucket (one with 800 distances: 6.7 us, 12.7 without four loads at a time).  `order` and
// `first` are by the whole table's indexes, of which `cut` lie off either end; the sums are by falling distance.
template <typename B>
__global__ __launch_bounds__(256) void local_bias_sum_kernel(const float* sums, B* out, const int32_t* order, const int32_t* first,
                                                             int parts, int span, int cut, int buckets, int heads) {
  const int x = threadIdx.x & 63, c = static_cast<int>(blockIdx.y) * 4 + static_cast<int>(threadIdx.x >> 6), all = span + 2 * cut;
  if (c >= buckets) return;
  const float* from = sums + static_cast<int64_t>(blockIdx.x) * parts * span;
  const int begin = max(0, first[c]), end = min(all, first[c + 1]);
  float sum = 0.f;
  for (int base = begin + x; base < end; base += 4 * 64) {  // two loads, one waiting for the other: four at a time
    int at[4];
    float value[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) at[j] = span - 1 - (order[min(base + j * 64, end - 1)] - cut);
    for (int z = 0; z < parts; ++z) {
#pragma unroll
      for (int j = 0; j < 4; ++j) value[j] = from[static_cast<int64_t>(z) * span + min(max(at[j], 0), span - 1)];
#pragma unroll
      for (int j = 0; j < 4; ++j) sum += base + j * 64 < end && at[j] >= 0 && at[j] < span ? value[j] : 0.f;
    }
  }
  sum = group_sum(sum, kWave);
  if (x == 0) out[static_cast<int64_t>(c) * heads + blockIdx.x] = from_f32<B>(sum);
}

// ---------------------------------------------------------------- dK, dV

// Waves that share a SIMD: fp32 rows of 64 with a bias pass the registers of two by a few.
template <typename T, int DP, bool BIAS>
constexpr int dkv_waves() { return DP == 128 || (DP == 64 && BIAS && sizeof(T) == 4) ? 1 : 2; }

template <typename T, int DP, int NW, bool BIAS>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(dkv_waves<T, DP, BIAS>()))) void local_dkv_kernel(BwdArgs a) {
  constexpr int DB = DP * sizeof(T), NS = DB / 32, DT = DP / 32;
  constexpr int BQ = local_tile<T, DP>(), SUBS = BQ / 32;
  constexpr bool kHalf = std::is_same<T, f16>::value;
  __shared__ __attribute__((aligned(16))) char lds[kStages][2][BQ * DB];
  __shared__ __attribute__((aligned(16))) float stat[kStages][2][64];  // -lse (log2 units), D
  extern __shared__ float table[];  // the bias by falling distance, then each wave's bins
  const int lane = threadIdx.x & 63, h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t pair, sub_block;
  if (!locate(a.grid, pair, sub_block)) return;
  const Shape& s = a.s;
  // the ordinary blocks, then those of the sinks' later rows
  const uint32_t ordinary = a.key_tiles * a.splits;
  const uint32_t of = sub_block < ordinary ? a.key_tiles : a.sink_tiles, i = sub_block < ordinary ? sub_block : sub_block - ordinary;
  const uint32_t key_tile = i % of, slot = i / of + (sub_block < ordinary ? 0u : a.splits);
  const int b = static_cast<int>(pair) / s.Hk, hk = static_cast<int>(pair) - b * s.Hk;
  const int d_units = s.D * static_cast<int>(sizeof(T)) / 16;
  const int count = key_count(a.km, b, s.M);
  const int start = start_of(a.w, b);
  const int block_key0 = static_cast<int>(key_tile) * 32 * NW, block_end = min(block_key0 + 32 * NW, count);
  const int key0 = block_key0 + wave * 32, ki = key0 + (lane & 31);
  const bool seen = ki < count && (a.km.mask == nullptr || a.km.mask[b * a.km.stride + ki] != 0);
  const bool idle = key0 >= count;  // no frame of this wave counts: it only moves tiles
  const bool any_unseen = __any(!seen);

  const RowTiles rows = rows_of<BQ>(a.w, start, s.N, s.G, block_key0, block_end, static_cast<int>(slot),
                                    static_cast<int>(a.splits), static_cast<int>(a.chunks), a.chunk_tiles);
  const int first = rows.first, tiles = rows.tiles, from = rows.from, to = block_key0 < count ? rows.to : rows.from;
  float* part_bias = nullptr;  // of the pair's first head; further heads lie part_step apart
  int64_t part_step = 0;
  if constexpr (BIAS) {
    const int span = 2 * a.bias.distance + 1;
    part_step = static_cast<int64_t>(s.B) * a.grid.per * span;
    part_bias = a.part_bias + hk * s.G * part_step + (static_cast<int64_t>(b) * a.grid.per + sub_block) * span;
    // the heads that have no tile here
    const int g_from = from < to ? from / tiles : 0, g_to = from < to ? (to - 1) / tiles + 1 : 0;
    for (int g = 0; g < s.G; ++g) {
      if (g >= g_from && g < g_to) continue;
      for (int i = threadIdx.x; i < span; i += 64 * NW) part_bias[g * part_step + i] = 0.f;
    }
  }

  f32x16_t dk[DT]{}, dv[DT]{};
  float k_scale = a.scale, v_scale = 1.f;
  if (from < to) {
    u32x4_t kf[NS], vf[NS];
    load_frags<T, DP>(static_cast<const T*>(a.k) + b * a.ks.b + hk * a.ks.h + (seen ? ki * a.ks.n : 0), seen, d_units, h, kf);
    load_frags<T, DP>(static_cast<const T*>(a.v) + b * a.vs.b + hk * a.vs.h + (seen ? ki * a.vs.n : 0), seen, d_units, h, vf);
    // P' = 2^14 P (in base), dS' = P' 2^e (...): as in the cross attention
    float dp_scale = 1.f, dp_unscale = 1.f;
    if constexpr (kHalf) {
      const int e = pair_exponent(a, pair);
      dp_scale = ldexpf(1.f, e);
      dp_unscale = ldexpf(1.f, -e);
      k_scale = ldexpf(a.scale, -e - 14);
      v_scale = ldexpf(1.f, -14);
    }
    const T* qb = static_cast<const T*>(a.q) + b * a.qs.b;
    const T* gb = static_cast<const T*>(a.dout) + b * a.gs.b;
    const int64_t q_step = BQ * static_cast<int64_t>(sizeof(T)) * a.qs.n, g_step = BQ * static_cast<int64_t>(sizeof(T)) * a.gs.n;
    Tile<T, DP, BQ, NW> qt, gt;
    auto q_at = [&](int i) { return i * a.qs.n; };
    auto g_at = [&](int i) { return i * a.gs.n; };
    const T *q_head = nullptr, *g_head = nullptr;
    // waves 0 and 1 also move a tile's 64 (32) pairs of statistics, 4 bytes a lane
    const float* stat_head = nullptr;
    const uint32_t* lone_head = nullptr;
    uint32_t lone_next[2] = {0, 0};  // the tile's queries that see one frame alone
    auto fetch = [&](int t, int stage) {
      const int row0 = t * BQ;
      if (DB < 512 && row0 + BQ <= s.N) {
        qt.fetch(lds[stage][0], q_step);
        gt.fetch(lds[stage][1], g_step);
      } else {
        qt.fetch_cut(lds[stage][0], q_head, row0, s.N, d_units, q_at);
        gt.fetch_cut(lds[stage][1], g_head, row0, s.N, d_units, g_at, reinterpret_cast<const T*>(zero_row));
      }
      if (wave < 2 && (BQ == 64 || lane < BQ)) dma4_m0(stat_head + row0, __builtin_amdgcn_readfirstlane(lds_addr(stat[stage]) + 256 * wave));
#pragma unroll
      for (int u = 0; u < SUBS; ++u) lone_next[u] = lone_head[row0 / 32 + u];
    };
    arrive(kf);
    arrive(vf);
    const float* lane_table = nullptr;  // this lane's entry for a query at frame 0
    float sum_low = 0.f, sum_high = 0.f;
    const int entries = 2 * a.bias.distance + 1 + 2 * kPad;
    float* bins = nullptr;
    auto begin_table = [&](int g) {
      fill_bias<T, true>(table, a.bias, s.H, hk * s.G + g, a.bias_unit, 64 * NW);
      for (int i = lane; i < entries; i += 64) bins[i] = 0.f;
      sum_low = sum_high = 0.f;
    };
    // a head's bins, over the waves
    auto end_table = [&](int g) {
      // past the table's ends, and the far tiles' sums: into the end bins
      const float above = group_sum(sum_high + bins[lane], kWave);
      const float under = group_sum(sum_low + bins[entries - kPad + lane], kWave);
      if (lane == 0) {
        bins[kPad] += above;
        bins[entries - 1 - kPad] += under;
      }
      __syncthreads();
      const float unscale = kHalf ? v_scale * dp_unscale : 1.f;
      for (int i = threadIdx.x; i < 2 * a.bias.distance + 1; i += 64 * NW) {
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) sum += table[entries + kBinPad + w * (entries + 2 * kBinPad) + kPad + i];
        part_bias[g * part_step + i] = sum * unscale;
      }
    };
    if constexpr (BIAS) {
      bins = table + entries + kBinPad + wave * (entries + 2 * kBinPad);
      lane_table = table + (a.bias.distance + kPad + 8 * h - ki);
    }
    // head by head: a loop over all tiles would hold what changes with the head in scalar registers that it does not have
    for (int at = from; at < to;) {
      const int g = at / tiles, head = hk * s.G + g, t0 = first + at - g * tiles, t1 = min(first + tiles, t0 + to - at);
      if (at > from) __syncthreads();  // every wave is past the head before: its tiles, table and bins
      at += t1 - t0;
      q_head = qb + head * a.qs.h;
      g_head = gb + head * a.gs.h;
      qt.start(q_head, t0 * BQ, d_units, q_at);
      gt.start(g_head, t0 * BQ, d_units, g_at);
      const int64_t stat_at = (static_cast<int64_t>(b) * s.H + head) * a.rows_pad;
      stat_head = (wave == 0 ? a.base : a.delta) + stat_at + lane;
      lone_head = a.lone + stat_at / 32;
      fetch(t0, 0);
      if constexpr (BIAS) begin_table(g);
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
        const uint32_t lone_now[2] = {lone_next[0], lone_next[1]};
        if (t + 1 < t1) fetch(t + 1, stage ^ 1);
        stage ^= 1;
        const int row_tile0 = t * BQ;
        if (idle) continue;
#pragma unroll
        for (int u = 0; u < SUBS; ++u) {
          const int row0 = row_tile0 + 32 * u, p0 = start + row0;
          if (row0 >= s.N) continue;
          const Sees what = sees(a.w, p0, key0, count);
          if (what == Sees::kNone) continue;
          hold(sizeof(T) == 4);
          const int at_lane = fresh<DB>(lane);
          f32x16_t p{}, ds{};
          bool near = false, upper = false;
          // 16 bits: every fragment of the two products is on its way before the first of them (a read at a time leaves the
          // matrix cores waiting for LDS; the registers are there, as two waves share a SIMD either way)
          u32x4_t fq[sizeof(T) == 2 ? NS : 1], fg[sizeof(T) == 2 ? NS : 1];
          if constexpr (sizeof(T) == 2) {
            const int row = 32 * u + key_row(at_lane & 31);
#pragma unroll
            for (int i = 0; i < NS; ++i) fq[i] = row_frag<DB>(ql, row, i, at_lane >> 5);
#pragma unroll
            for (int i = 0; i < NS; ++i) fg[i] = row_frag<DB>(gl, row, i, at_lane >> 5);
          }
          if constexpr (BIAS) {
            near = !bias_far(key0 - p0 - 31, a.bias.distance, upper);
            p = bias_tile(lane_table + (key0 - bias_gap(key0 - p0, a.bias.distance)));
          }
          if constexpr (sizeof(T) == 2) {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < NS; ++i) p = mma<T>(fq[i], kf[i], p);
#pragma unroll
            for (int i = 0; i < NS; ++i) ds = mma<T>(fg[i], vf[i], ds);
          } else {
            p = mma_rows_from<T, DP>(p, ql, u, kf, at_lane);
            ds = mma_rows<T, DP>(gl, u, vf, at_lane);
          }
          // (what lanes of unseen frames hold is dropped at the end, but for the bias's sums)
          if (what == Sees::kSome || (BIAS && any_unseen)) {
            uint32_t bits = queries_seeing(a.w, start, ki, row0) >> (8 * h);
            if constexpr (BIAS) bits = seen ? bits : 0u;
#pragma unroll
            for (int r = 0; r < 16; ++r) p[r] = where_bit(bits, reg_key(r), p[r], -kInf);
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int row = 32 * u + reg_key(r) + 8 * h;
            p[r] = __builtin_amdgcn_exp2f(fmaf(p[r], a.scale_log2, base[row]));
            // (not as one sum with the product, begun at -D: the matrix cores' roundings then lean to D's side, and the bias's
            // gradient of 124 x 948 queries is 1e-5 off instead of 6e-7)
            ds[r] = p[r] * fmaf(ds[r], dp_scale, -delta[row]);
          }
          const uint32_t sub_lone = lone_now[u];
          if (sub_lone != 0) {
#pragma unroll
            for (int r = 0; r < 16; ++r) ds[r] = where_bit(sub_lone >> (8 * h), reg_key(r), ds[r] * 0.f, ds[r]);
          }
          hold(sizeof(T) == 4);
          mma_cols<T, DP>(gl, u, p, dv, at_lane);
          mma_cols<T, DP>(ql, u, ds, dk, at_lane);
          if constexpr (BIAS) {
            if (near) {
              add_diagonals(bins + (a.bias.distance + kPad + p0 - key0), ds, lane);
            } else {
              float sum[2] = {0.f, 0.f};
#pragma unroll
              for (int r = 0; r < 16; ++r) sum[r & 1] += ds[r];
              const float both = sum[0] + sum[1];
              sum_high += upper ? both : 0.f;
              sum_low += upper ? 0.f : both;
            }
          }
        }
      }
      if constexpr (BIAS) end_table(g);
    }
  }
  if (ki >= s.M) return;
  if (!seen) {
    // nothing was learnt about a frame that is not seen, whatever its columns of the tiles hold
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      dk[dt] = f32x16_t{};
      dv[dt] = f32x16_t{};
    }
  }
  if (a.splits > 1 || key_tile < a.sink_tiles) {
    if (slot >= a.splits && ki >= a.sink_rows) return;  // no row past the window sees this frame
    int64_t row = (static_cast<int64_t>(min(slot, a.splits)) * a.grid.pairs + (slot < a.splits ? pair : 0u)) * a.part_keys + ki;
    if (slot >= a.splits) row += (static_cast<int64_t>(slot - a.splits) * a.grid.pairs + pair) * a.sink_rows;
    const int64_t at = row * s.D;
    store_cols_f32<T, DP>(a.part_k + at, dk, k_scale, s.D, h);
    store_cols_f32<T, DP>(a.part_v + at, dv, v_scale, s.D, h);
  } else {
    const int64_t at = ((static_cast<int64_t>(b) * s.M + ki) * s.Hk + hk) * s.D;
    store_cols<T, DP>(static_cast<T*>(a.dk) + at, dk, k_scale, s.D, h);
    store_cols<T, DP>(static_cast<T*>(a.dv) + at, dv, v_scale, s.D, h);
  }
}

// ---------------------------------------------------------------- up to 64 frames, 16 bits

// All gradients in one pass where a tile holds every frame, as in the cross attention: a block of 2 waves keeps K and V of
// a (batch row, key head) in LDS and passes over the query tiles of its heads; P and dS go through LDS to be the other
// operand of dV and dK.  A wave's whole rows of P and dP are in registers, so D is their sum, in fp32.  5 products instead
// of 7, and every tensor is moved once: 1032 x 62 queries over 62 frames with a bias, bf16, 8 heads of 64, 132 us (HBM, 3.5
// TB/s at 6 waves a CU: 48 KB of LDS a block) against 119 + 116 of the two kernels.  The same holds with many queries, which a
// block takes in turn (the whole backward, over 64 frames): 256 x 512, 8 heads, 147 us against 285; 256 x 4096, one head,
// 239 against 294; 64 x 2100 over 50, 4 heads, no bias, 86 against 137.
// (Waves that share a SIMD: fp16's scaling and a bias together pass the registers of two.)
template <typename T, int DP, bool BIAS>
constexpr int few_waves() { return DP == 128 || (DP == 64 && BIAS && std::is_same<T, f16>::value) ? 1 : 2; }

template <typename T, int DP, bool BIAS>
__global__ __launch_bounds__(128) __attribute__((amdgpu_waves_per_eu(few_waves<T, DP, BIAS>()))) void local_few_kernel(BwdArgs a) {
  constexpr int DB = DP * sizeof(T), NS = DB / 32, DT = DP / 32, PB = 64 * sizeof(T);
  constexpr bool kHalf = std::is_same<T, f16>::value;
  __shared__ __attribute__((aligned(16))) char kv[2][64 * DB];
  __shared__ __attribute__((aligned(16))) char rows[2][64 * DB];
  __shared__ __attribute__((aligned(16))) char ps[2][64 * PB];
  __shared__ float most[2];
  extern __shared__ float table[];  // the bias by distance, each wave's bins, and whether it saw an entry that hides
  const int lane = threadIdx.x & 63, h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t pair, sub;
  if (!locate(a.grid, pair, sub)) return;
  const Shape& s = a.s;
  const int b = static_cast<int>(pair) / s.Hk, hk = static_cast<int>(pair) - b * s.Hk;
  const int d_units = s.D * static_cast<int>(sizeof(T)) / 16;
  const int count = key_count(a.km, b, s.M);
  const int start = start_of(a.w, b);
  uint64_t kept = range_bits(0, count);
  if (a.km.mask) kept &= __ballot(a.km.mask[b * a.km.stride + min(lane, s.M - 1)] != 0);
  const int entries = 2 * a.bias.distance + 1 + 2 * kPad;
  float* bins = table + entries + kBinPad + wave * (entries + 2 * kBinPad);
  float* hides = table + 3 * entries + 4 * kBinPad;  // of 2 waves

  Tile<T, DP, 64, 2> tile;  // no state: every move computes its addresses
  tile.fetch_cut(kv[0], static_cast<const T*>(a.k) + b * a.ks.b + hk * a.ks.h, 0, s.M, d_units, [&](int i) { return i * a.ks.n; });
  tile.fetch_cut(kv[1], static_cast<const T*>(a.v) + b * a.vs.b + hk * a.vs.h, 0, s.M, d_units, [&](int i) { return i * a.vs.n; });

  f32x16_t dk[DT]{}, dv[DT]{};
  constexpr int kNoSum = 101;  // above every exponent (scale_exponent's end at 100): nothing but zeros so far
  int e_sum = kNoSum;          // dk is held at 2^e_sum
  const int tiles = (s.N + 63) / 64;
  for (int g = 0; g < s.G; ++g) {
    const int head = hk * s.G + g;
    float far_low = 0.f, far_high = 0.f, sum_low = 0.f, sum_high = 0.f;
    bool some_hidden = false;
    for (int t = 0; t < tiles; ++t) {
      if (g > 0 || t > 0) __syncthreads();  // the tiles of the rows before these have been read, and the table
      tile.fetch_cut(rows[0], static_cast<const T*>(a.q) + b * a.qs.b + head * a.qs.h, t * 64, s.N, d_units, [&](int i) { return i * a.qs.n; });
      tile.fetch_cut(rows[1], static_cast<const T*>(a.dout) + b * a.gs.b + head * a.gs.h, t * 64, s.N, d_units, [&](int i) { return i * a.gs.n; });
      const int n0 = t * 64 + 32 * wave, n = n0 + (lane & 31), p0 = start + n0, pos = start + n;
      const bool row_ok = n < s.N;
      // -lse in log2 units: a row that sees no frame (and one past the end) has no weight.  (On its way before the bias.)
      float lse = -kInf;
      if (row_ok) lse = a.lse[(static_cast<int64_t>(b) * s.H + head) * s.N + n];
      if constexpr (BIAS) {
        if (t == 0) {
          const bool own = __any(fill_bias<T, false>(table, a.bias, s.H, head, a.bias_unit, 128));
          hides[wave] = own ? 1.f : 0.f;
          for (int i = lane; i < entries; i += 64) bins[i] = 0.f;
          __syncthreads();
          some_hidden = __builtin_amdgcn_readfirstlane(hides[0] + hides[1] != 0.f);
        }
      }
      const float base = lse == -kInf ? -kInf : -lse * kLog2e;
      const int low = low_of(a.w, pos), high = high_of(a.w, pos, count);
      uint32_t seen[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) seen[u] = static_cast<uint32_t>(kept >> (32 * u)) & frames_seen(low, high, a.w.sinks, 32 * u);
      int found = __popc(seen[0]) + __popc(seen[1]);
      if constexpr (BIAS) {
        // frames that the bias hides are not seen (here, before the wait for the tiles: behind it 256 x 4096 queries take
        // 250 us, not 239)
        if (some_hidden) {
          found = 0;
#pragma unroll
          for (int u = 0; u < 2; ++u) found += __popc(seen[u] & bias_shows(table, a.bias.distance, pos, 32 * u));
        }
      }
      vm_wait<0>();
      if (g == 0 && t == 0 && (kept != ~uint64_t{0} || d_units != tile.UNITS)) {
        tile.clear(kv[0], kept, d_units);
        tile.clear(kv[1], kept, d_units);
      }
      if (d_units != tile.UNITS) {
        tile.clear(rows[0], ~uint64_t{0}, d_units);
        tile.clear(rows[1], ~uint64_t{0}, d_units);
      }
      // rows past the end hold the last one again, whose infinities would meet their weights of 0
      if (t * 64 + 64 > s.N) tile.clear_from(rows[1], s.N - t * 64);
      __syncthreads();

      const int at_lane = fresh<256>(lane);  // whatever DB: this kernel has no registers for addresses
      if constexpr (BIAS) {
        far_low = table[0];
        far_high = table[entries - 1];
      }
      f32x16_t p[2], ds[2];
      bool near[2] = {false, false}, upper[2] = {false, false};
      {
        u32x4_t f[NS];
#pragma unroll
        for (int i = 0; i < NS; ++i) f[i] = row_frag<DB>(rows[0], 32 * wave + (at_lane & 31), i, h);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          if constexpr (BIAS) {
            near[u] = !bias_far(32 * u - p0 - 31, a.bias.distance, upper[u]);
            if (near[u]) {
              p[u] = bias_tile(table + (a.bias.distance + kPad + 8 * h - pos + 32 * u));
            } else {
              const float far = upper[u] ? far_high : far_low;
#pragma unroll
              for (int r = 0; r < 16; ++r) p[u][r] = far;
            }
            p[u] = mma_rows_from<T, DP>(p[u], kv[0], u, f, at_lane);
          } else {
            p[u] = mma_rows<T, DP>(kv[0], u, f, at_lane);
          }
        }
#pragma unroll
        for (int i = 0; i < NS; ++i) f[i] = row_frag<DB>(rows[1], 32 * wave + (at_lane & 31), i, h);
#pragma unroll
        for (int u = 0; u < 2; ++u) ds[u] = mma_rows<T, DP>(kv[1], u, f, at_lane);
      }
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint32_t bits = seen[u] >> (8 * h);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float w = where_bit(bits, reg_key(i), __builtin_amdgcn_exp2f(fmaf(p[u][i], a.scale_log2, base)), 0.f);
          sum[i & 1] = fmaf(w, ds[u][i], sum[i & 1]);
          p[u][i] = w;
        }
      }
      const float delta = half_sum(sum[0] + sum[1]), alive = found == 1 ? 0.f : 1.f;
      float top = 0.f;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          ds[u][i] = p[u][i] * ((ds[u][i] - delta) * alive);
          if constexpr (kHalf) top = fmaxf(top, fabsf(ds[u][i]));
        }
        if constexpr (BIAS) {
          if (near[u]) {
            add_diagonals(bins + (a.bias.distance + kPad + 32 * u - p0), ds[u], lane);
          } else {
            float far[2] = {0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 16; ++i) far[i & 1] += ds[u][i];
            const float both = far[0] + far[1];
            sum_high += upper[u] ? both : 0.f;
            sum_low += upper[u] ? 0.f : both;
          }
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
        const float dq_scale = kHalf ? ldexpf(a.scale, -e) : a.scale;
        const int64_t to = (static_cast<int64_t>(b) * s.N + n) * s.H + head;
        store_cols<T, DP>(static_cast<T*>(a.dq) + to * s.D, dq, dq_scale, s.D, h);
      }

      // [row][frame] tiles: a lane writes its row's frames, 8 consecutive ones a unit
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
    if constexpr (BIAS) {
      // the head's bins, past the table's ends into the end ones, over the waves (the table's next fill waits at the
      // head's first barrier, as does the clearing of the bins, which are a wave's own until then)
      const float under = group_sum(sum_low + bins[lane], kWave);
      const float above = group_sum(sum_high + bins[entries - kPad + lane], kWave);
      if (lane == 0) {
        bins[kPad] += under;
        bins[entries - 1 - kPad] += above;
      }
      __syncthreads();
      const int span = 2 * a.bias.distance + 1;
      float* part = a.part_bias + (static_cast<int64_t>(head) * s.B + b) * span;
      for (int i = threadIdx.x; i < span; i += 128) {  // by falling distance
        const float* bin = table + entries + kBinPad + entries - 1 - kPad - i;
        part[i] = bin[0] + bin[entries + 2 * kBinPad];
      }
    }
  }
  // a transposed read hands lane l the frame key_row(l % 32)
  const int ki = 32 * wave + key_row(lane & 31);
  if (ki >= s.M) return;
  const float k_scale = kHalf ? ldexpf(a.scale, -e_sum) : a.scale, v_scale = kHalf ? 1.f / 16384.f : 1.f;
  const int64_t to = ((static_cast<int64_t>(b) * s.M + ki) * s.Hk + hk) * s.D;
  store_cols<T, DP>(static_cast<T*>(a.dk) + to, dk, k_scale, s.D, h);
  store_cols<T, DP>(static_cast<T*>(a.dv) + to, dv, v_scale, s.D, h);
}

// dk, dv of the keys that several blocks share = the sum of their parts, in order.  A thread takes 4 columns, `per` blocks a
// pair; the grid's y is the gradient.  (4 x 317 fp32 keys of 2 heads of 64 in eight parts: latency.  Four parts' loads at a
// time and no division of 64 bits: 8.4 -> 4.8 us.)
template <typename T>
__global__ __launch_bounds__(256) void local_parts_sum_kernel(BwdArgs a, uint32_t keys, uint32_t per, FastDiv by_quads) {
  const Shape& s = a.s;
  const uint32_t quads = by_quads.d, pair = blockIdx.x / per, i = (blockIdx.x - pair * per) * 256u + threadIdx.x;
  if (i >= keys * quads) return;  // (fits: the parts of 2^32 threads would take more memory than there is)
  const int64_t key = by_quads.div(i), quad = i - static_cast<uint32_t>(key) * quads;
  const float* from = (blockIdx.y != 0 ? a.part_v : a.part_k) + ((static_cast<int64_t>(pair) * a.part_keys + key) * quads + quad) * 4;
  const int64_t step = static_cast<int64_t>(a.grid.pairs) * a.part_keys * s.D;
  const int64_t sink_step = static_cast<int64_t>(a.grid.pairs) * a.sink_rows * s.D;
  float o[4] = {0.f, 0.f, 0.f, 0.f};
  auto add = [&](const float* first, int64_t apart, int parts) {
    for (int c = 0; c < parts; c += 4) {
      float x[4][4];
#pragma unroll
      for (int k = 0; k < 4; ++k) load_pack<float, 4>(first + min(c + k, parts - 1) * apart, x[k]);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] += c + k < parts ? x[k][j] : 0.f;
      }
    }
  };
  add(from, step, static_cast<int>(a.splits));
  if (key < a.sink_rows) {
    add(from + a.splits * step + static_cast<int64_t>(pair) * (a.sink_rows - a.part_keys) * s.D, sink_step, static_cast<int>(a.chunks));
  }
  const uint32_t b = pair / static_cast<uint32_t>(s.Hk), hk = pair - b * static_cast<uint32_t>(s.Hk);
  T* out = static_cast<T*>(blockIdx.y != 0 ? a.dv : a.dk);
  store_pack<T, 4>(out + ((static_cast<int64_t>(b) * s.M + key) * s.Hk + hk) * s.D + 4 * quad, o);
}

// ---------------------------------------------------------------- host

struct BwdPlan {
  bool few;  // local_few_kernel
  int nw_q, nw_k;
  int64_t twice_tiles;  // the first row tiles, whose queries see few frames: local_dq_kernel passes twice
  int64_t row_tiles, key_tiles, splits, sink_tiles, chunks, chunk_tiles;
  int64_t blocks() const { return few ? 1 : key_tiles * splits + sink_tiles * chunks; }  // of a pair, that leave bins
  int64_t sink_keys() const { return sink_tiles * 32 * nw_k; }
  int64_t part_keys() const { return few ? 0 : splits > 1 ? key_tiles * 32 * nw_k : sink_keys(); }
  static int64_t sink_rows(const Shape& s, const Window& w) { return std::min(w.sinks, s.M); }
};

// The frames' blocks are split over their queries where they are fewer than two a CU, into shares of at least two tiles:
// fp32, 4 x 317 queries and frames, 8 heads on 2, local_dkv_kernel 38 us and a sum of 5 against 186 and 4.  The sinks'
// rows in blocks of their own: 16 x 2760 queries, window of 1024, 4 sinks, 339 us and a sum of 5 against 357 and 4 (more
// with narrower windows, where a sinks' block passes over more times as many rows as another).
BwdPlan plan_backward(const Shape& s, const Window& w, int dtype) {
  const bool wide = padded_dim(s.D) * static_cast<int>(dtype_size(dtype)) == 512;
  const int64_t bq = wide ? 32 : 64, want = 2 * num_cus(), pairs = int64_t{s.B} * s.Hk;
  BwdPlan p{};
  p.nw_q = s.N <= 64 && !wide ? 2 : 4;
  p.nw_k = s.M <= 64 && !wide ? 2 : 4;
  const int64_t block_keys = 32 * p.nw_k;
  p.row_tiles = (int64_t{s.N} + 32 * p.nw_q - 1) / (32 * p.nw_q);
  p.key_tiles = (int64_t{s.M} + block_keys - 1) / block_keys;
  if (s.M <= 96 || (w.left >= 0 && w.right >= 0 && int64_t{w.left} + w.right + w.sinks < 96)) {
    p.twice_tiles = p.row_tiles;
  } else if (w.starts == nullptr && w.right >= 0 && w.right < 32) {
    p.twice_tiles = std::min<int64_t>(p.row_tiles, 256 / (32 * p.nw_q));  // a past that grows
  }
  // row tiles of an ordinary block
  const int64_t all = (int64_t{s.N} + bq - 1) / bq * s.G;
  int64_t usual = all;
  if (w.left >= 0 && w.right >= 0) usual = std::min(all, (int64_t{w.left} + w.right + block_keys + bq - 1) / bq * s.G);
  const int64_t blocks = std::max<int64_t>(1, pairs * p.key_tiles);
  // (few pairs: a block each would leave CUs without any)
  p.few = s.M > 0 && s.M <= 64 && dtype != PMSST_F32 && pairs >= num_cus();
  p.splits = blocks < want ? std::max<int64_t>(1, std::min((want + blocks - 1) / blocks, usual / 2)) : 1;
  if (w.sinks > 0) {
    p.sink_tiles = std::min<int64_t>(p.key_tiles, (w.sinks + block_keys - 1) / block_keys);
    // as many tiles a block as an ordinary one has, at least 8 (about 10 us) where those are not split; past 64 MB, no
    // more parts than the frames' own gradients would take in fp32 (16 x 8192 queries, windows of 128 either way, 2048
    // sinks, 4 parts in place of 16: the backward takes 2382 us in place of 2969, and 0.7 GB in place of 2.2)
    p.chunk_tiles = std::max<int64_t>(p.splits > 1 ? 2 : 8, usual / p.splits);
    const int64_t sinks = p.sink_rows(s, w), part_bytes = 8 * pairs * sinks * s.D;
    if (part_bytes > 0) {
      const int64_t most = std::max<int64_t>({1, (int64_t{64} << 20) / part_bytes, s.M / sinks});
      p.chunk_tiles = std::max(p.chunk_tiles, (all + most - 1) / most);
    }
    p.chunks = (all + p.chunk_tiles - 1) / p.chunk_tiles;
  }
  return p;
}

struct BwdSpace {
  size_t stat, bound, part_k, part_bias, sum_bias, total;
};

// span: distances of the bias, 0 without one
BwdSpace bwd_space(const Shape& s, const Window& win, const BwdPlan& p, int64_t span, int dtype) {
  const size_t pairs = static_cast<size_t>(s.B) * s.Hk;
  BwdSpace w;
  w.stat = p.few ? 0 : static_cast<size_t>(s.B) * s.H * align_up(s.N, 64) * 4;
  w.bound = dtype == PMSST_F16 && !p.few ? align_up(pairs * kParts * 4, 256) : 0;
  const int64_t sink_parts = p.few ? 0 : p.chunks * p.sink_rows(s, win);
  w.part_k = align_up(pairs * (p.splits * p.part_keys() + sink_parts) * s.D * 4, 256);
  const size_t blocks = static_cast<size_t>(s.B) * p.blocks();
  w.part_bias = align_up(s.H * blocks * span * 4, 256);
  w.sum_bias = align_up(s.H * ((blocks + kSumRows - 1) / kSumRows) * span * 4, 256);
  w.total = align_up(2 * w.stat + w.stat / 32, 256) + 2 * w.bound + 2 * w.part_k + w.part_bias + w.sum_bias;
  return w;
}

// LDS of a bias's table and the bins of `waves`.
size_t bins_bytes(const BwdArgs& a, int waves) { return (bias_entries(a.bias.distance) * (1 + waves) + 2 * kBinPad * waves) * 4; }

template <typename T, int DP, int NW, bool TWICE>
int launch_dq(BwdArgs& a, int64_t begin, int64_t end, hipStream_t stream) {
  if (begin == end) return PMSST_OK;
  a.row_begin = static_cast<uint32_t>(begin);
  a.row_end = static_cast<uint32_t>(end);
  a.grid = make_grid(int64_t{a.s.B} * a.s.Hk, (end - begin) * a.s.G);
  const dim3 grid(static_cast<uint32_t>(grid_blocks(a.grid)));
  if (a.bias.table) {
    local_dq_kernel<T, DP, NW, true, TWICE><<<grid, 64 * NW, (bias_entries(a.bias.distance) + NW) * 4, stream>>>(a);
  } else {
    local_dq_kernel<T, DP, NW, false, TWICE><<<grid, 64 * NW, 0, stream>>>(a);
  }
  return check_launch("local_dq_kernel");
}

template <typename T, int DP, int NW>
int launch_dq(BwdArgs& a, const BwdPlan& p, hipStream_t stream) {
  if constexpr (sizeof(T) == 2) {
    const int rc = launch_dq<T, DP, NW, true>(a, 0, p.twice_tiles, stream);
    return rc != PMSST_OK ? rc : launch_dq<T, DP, NW, false>(a, p.twice_tiles, p.row_tiles, stream);
  } else {
    return launch_dq<T, DP, NW, false>(a, 0, p.row_tiles, stream);
  }
}

template <typename T, int DP, int NW>
int launch_dkv(const BwdArgs& a, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(grid_blocks(a.grid)));
  if (a.bias.table) {
    local_dkv_kernel<T, DP, NW, true><<<grid, 64 * NW, bins_bytes(a, NW), stream>>>(a);
  } else {
    local_dkv_kernel<T, DP, NW, false><<<grid, 64 * NW, 0, stream>>>(a);
  }
  return check_launch("local_dkv_kernel");
}

template <typename T, int DP>
int launch_dq(BwdArgs& a, const BwdPlan& p, hipStream_t stream) {
  if constexpr (DP * sizeof(T) != 512) {
    if (p.nw_q == 2) return launch_dq<T, DP, 2>(a, p, stream);
  }
  return launch_dq<T, DP, 4>(a, p, stream);
}

template <typename T, int DP>
int launch_dkv(const BwdArgs& a, const BwdPlan& p, hipStream_t stream) {
  if constexpr (DP * sizeof(T) != 512) {
    if (p.nw_k == 2) return launch_dkv<T, DP, 2>(a, stream);
  }
  return launch_dkv<T, DP, 4>(a, stream);
}

template <typename T, int DP>
int run_bwd(BwdArgs& a, const BwdPlan& p, hipStream_t stream) {
  const int64_t pairs = int64_t{a.s.B} * a.s.Hk;
  const int64_t per = p.blocks();
  int rc = PMSST_OK;
  if (p.few) {
    if constexpr (sizeof(T) == 2) {
      a.grid = make_grid(pairs, 1);
      const dim3 grid(static_cast<uint32_t>(grid_blocks(a.grid)));
      if (a.bias.table) {
        local_few_kernel<T, DP, true><<<grid, 128, bins_bytes(a, 2) + 8, stream>>>(a);
      } else {
        local_few_kernel<T, DP, false><<<grid, 128, 0, stream>>>(a);
      }
      if ((rc = check_launch("local_few_kernel")) != PMSST_OK) return rc;
    }
  } else {
    if constexpr (std::is_same<T, f16>::value) rc = launch_bound<T>(a, pairs, stream);
    if (rc != PMSST_OK) return rc;
    if ((rc = launch_dq<T, DP>(a, p, stream)) != PMSST_OK) return rc;
    if (per > 0) {
      a.grid = make_grid(pairs, per);
      if ((rc = launch_dkv<T, DP>(a, p, stream)) != PMSST_OK) return rc;
    }
  }
  if (a.bias.table) {
    const int span = 2 * a.bias.distance + 1;
    const int64_t blocks = int64_t{a.s.B} * per, parts = (blocks + kSumRows - 1) / kSumRows;  // none without frames: zeros
    if (parts > 0) {
      const dim3 grid(static_cast<uint32_t>(a.s.H * parts), static_cast<uint32_t>((span + 63) / 64));
      local_bins_sum_kernel<<<grid, 1024, 0, stream>>>(a.part_bias, a.sum_bias, blocks, parts, span);
      if ((rc = check_launch("local_bins_sum_kernel")) != PMSST_OK) return rc;
    }
    const dim3 grid(static_cast<uint32_t>(a.s.H), static_cast<uint32_t>((a.bias.buckets + 3) / 4));
    if (a.bias.f32) {
      local_bias_sum_kernel<float><<<grid, 256, 0, stream>>>(a.sum_bias, static_cast<float*>(a.dbias), a.order, a.first,
                                                             static_cast<int>(parts), span, a.cut, a.bias.buckets, a.s.H);
    } else {
      local_bias_sum_kernel<T><<<grid, 256, 0, stream>>>(a.sum_bias, static_cast<T*>(a.dbias), a.order, a.first,
                                                         static_cast<int>(parts), span, a.cut, a.bias.buckets, a.s.H);
    }
    if ((rc = check_launch("local_bias_sum_kernel")) != PMSST_OK) return rc;
  }
  const int keys = std::min(a.part_keys, a.s.M);
  if (keys == 0) return rc;
  const uint32_t quads = a.s.D / 4, sum_blocks = static_cast<uint32_t>((int64_t{keys} * quads + 255) / 256);
  local_parts_sum_kernel<T><<<dim3(static_cast<uint32_t>(pairs) * sum_blocks, 2), 256, 0, stream>>>(a, keys, sum_blocks, FastDiv(quads));
  return check_launch("local_parts_sum_kernel");
}

template <typename T>
int run_bwd(BwdArgs& a, const BwdPlan& p, hipStream_t stream) {
  return a.s.D <= 32 ? run_bwd<T, 32>(a, p, stream) : a.s.D <= 64 ? run_bwd<T, 64>(a, p, stream) : run_bwd<T, 128>(a, p, stream);
}

}  // namespace
}  // namespace pmsst

extern "C" {

size_t pmsst_local_attention_backward_workspace_size(int64_t batch, int64_t queries, int64_t keys, int64_t heads, int64_t kv_heads,
                                                     int64_t head_dim, int64_t left, int64_t right, int64_t sinks,
                                                     int has_starts, int64_t max_distance, int dtype) {
  using namespace pmsst::attn;
  LocalArgs l;
  static const int32_t some = 0;
  if (make_local("pmsst_local_attention_backward", batch, queries, keys, heads, kv_heads, head_dim, left, right, sinks,
                 has_starts ? &some : nullptr, nullptr, 0, nullptr, 0, 0, 1.0, dtype, l) != PMSST_OK ||
      max_distance > kMaxDistance || l.s.B == 0 || l.s.N == 0)
    return 0;
  const int64_t span = max_distance < 0 ? 0 : 2 * reach_of(l.s, l.w, max_distance) + 1;
  return pmsst::bwd_space(l.s, l.w, pmsst::plan_backward(l.s, l.w, dtype), span, dtype).total;
}

int pmsst_local_attention_backward(const void* grad_out, const int64_t* grad_out_strides, const void* q, const int64_t* q_strides,
                                   const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides,
                                   const void* out, const float* lse, const uint8_t* key_mask, int64_t key_mask_stride,
                                   const int32_t* key_lengths, const int32_t* query_starts, int64_t left,
                                   int64_t right, int64_t sinks, const void* bias, int bias_dtype, const int32_t* bucket_of,
                                   const int32_t* bucket_order, const int32_t* bucket_first, int64_t buckets,
                                   int64_t max_distance, void* grad_q, void* grad_k, void* grad_v, void* grad_bias, int64_t batch,
                                   int64_t queries, int64_t keys, int64_t heads, int64_t kv_heads, int64_t head_dim, double scale,
                                   int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace pmsst;
  using namespace pmsst::attn;
  const char* what = "pmsst_local_attention_backward";
  LocalArgs l;
  int rc = make_local(what, batch, queries, keys, heads, kv_heads, head_dim, left, right, sinks, query_starts, bias, bias_dtype,
                      bucket_of, buckets, max_distance, scale, dtype, l);
  if (rc != PMSST_OK) return rc;
  if (batch == 0) return PMSST_OK;
  PMSST_REQUIRE(queries > 0, "%s: queries must be positive (the other gradients are zero without any)", what);
  PMSST_REQUIRE(grad_out && q && out && lse && grad_q && (keys == 0 || (k && v && grad_k && grad_v)), "%s: null pointer", what);
  PMSST_REQUIRE(bias == nullptr || (grad_bias && bucket_order && bucket_first), "%s: null pointer (bias)", what);
  BwdArgs a{};
  a.s = l.s;
  a.w = l.w;
  a.bias = l.bias;
  a.order = bucket_order;
  a.first = bucket_first;
  a.cut = l.cut;
  if ((rc = make_strides(what, grad_out, grad_out_strides, queries, heads, head_dim, dtype, a.gs)) != PMSST_OK) return rc;
  if ((rc = make_strides(what, out, nullptr, queries, heads, head_dim, dtype, a.os)) != PMSST_OK) return rc;
  if ((rc = make_strides(what, q, q_strides, queries, heads, head_dim, dtype, a.qs)) != PMSST_OK) return rc;
  if ((rc = make_strides(what, k, k_strides, keys, kv_heads, head_dim, dtype, a.ks)) != PMSST_OK) return rc;
  if ((rc = make_strides(what, v, v_strides, keys, kv_heads, head_dim, dtype, a.vs)) != PMSST_OK) return rc;
  PMSST_REQUIRE(((reinterpret_cast<uintptr_t>(grad_q) | reinterpret_cast<uintptr_t>(grad_k) | reinterpret_cast<uintptr_t>(grad_v)) &
                 15) == 0,
                "%s: gradients must be 16-byte aligned", what);
  const BwdPlan p = plan_backward(a.s, a.w, dtype);
  const BwdSpace w = bwd_space(a.s, a.w, p, bias ? 2 * a.bias.distance + 1 : 0, dtype);
  if (w.total > 0 && (workspace == nullptr || workspace_bytes < w.total))  // few frames without a bias: none is needed
    return fail(PMSST_EWORKSPACE, "%s: workspace of %zu bytes needed, %zu given", what, w.total, workspace_bytes);
  PMSST_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0 || w.total == 0, "%s: workspace must be 16-byte aligned", what);
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
  a.dbias = grad_bias;
  char* at = static_cast<char*>(workspace);
  a.rows_pad = static_cast<int32_t>(align_up(a.s.N, 64));
  a.base = reinterpret_cast<float*>(at);
  a.delta = reinterpret_cast<float*>(at + w.stat);
  a.lone = reinterpret_cast<uint32_t*>(at + 2 * w.stat);
  at += align_up(2 * w.stat + w.stat / 32, 256);
  a.vmax = reinterpret_cast<float*>(at);
  at += w.bound;
  a.l1 = reinterpret_cast<float*>(at);
  at += w.bound;
  a.part_k = reinterpret_cast<float*>(at);
  at += w.part_k;
  a.part_v = reinterpret_cast<float*>(at);
  at += w.part_k;
  a.part_bias = reinterpret_cast<float*>(at);
  a.sum_bias = reinterpret_cast<float*>(at + w.part_bias);
  a.key_tiles = static_cast<uint32_t>(p.key_tiles);
  a.sink_tiles = static_cast<uint32_t>(p.sink_tiles);
  a.chunks = static_cast<uint32_t>(p.chunks);
  a.chunk_tiles = static_cast<int32_t>(p.chunk_tiles);
  a.splits = static_cast<uint32_t>(p.splits);
  a.part_keys = static_cast<int32_t>(p.part_keys());
  a.sink_rows = static_cast<int32_t>(p.sink_rows(a.s, a.w));
  a.late_first = a.w.right >= 0 && a.w.left < 0;
  const int64_t per = std::max(p.row_tiles * a.s.G, p.blocks());
  PMSST_REQUIRE(grid_fits(batch * kv_heads, per), "%s: too many rows for one call", what);
  PMSST_REQUIRE(batch * kv_heads * a.part_keys * (head_dim / 4) < int64_t{1} << 31, "%s: too many sinks for one call", what);
  a.scale = static_cast<float>(scale);
  a.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  a.bias_unit = static_cast<float>(1.0 / scale);
  a.drop.factor = 1.f;
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case PMSST_F32: return run_bwd<float>(a, p, st);
    case PMSST_F16: return run_bwd<f16>(a, p, st);
    default: return run_bwd<bf16>(a, p, st);
  }
}

}  // extern "C"
