// Local attention forward: O = softmax(scale Q K^T + bias over the seen frames) V, where a query sees the frames of a
// window around its own and a few first ones (sinks); local_attention.h has the rule and the bias.
//
// One pass over the tiles that hold a seen frame, with a running maximum and sum, as in cross_attention.hip.  A block is
// NW waves of 32 queries of one head; blocks of a (batch row, key head) run on one XCD, so that the heads that share
// its keys find them in its L2.  Work goes by the seen frames: tiles between the sinks and the window are not visited,
// 32 x 32 sub-tiles that a wave's queries do not see are passed over, those they see whole take no mask.
//
// Few queries over many frames are split over the tiles and joined by a second kernel.
//
// What bounds it.  Heads of 64 in 16 bits, all frames seen: the cross attention's pass (products, exponentials and the
// tiles' LDS reads share a clock of 1.7 GHz) and, with a bias, 16 LDS reads a sub-tile more: 124 x 948, 8 heads, fp16,
// 366 us, 623 TFLOP/s.  Windows of a tile or two: HBM, and the tiles at the window's ends that are partly seen: 248 x 258
// queries, 8 heads, windows of 64 either way, bf16, 71 us, 3.7 TB/s.  Long rows with a window of 1024 (16 x 2760 queries, 8
// heads, bias, bf16): 151 us, 500 TFLOP/s of the pairs that are seen.  Few blocks: the latency of the tiles a block takes
// in turn.
#include "local_attention.h"

#include <cmath>

namespace pmsst {
namespace {

using namespace attn;

struct FwdArgs {
  const void *q, *k, *v;
  Strides qs, ks, vs;
  KeyMask km;
  Window w;
  BiasArgs bias;
  void* out;
  float* lse;       // [B, H, N] or NULL
  float* part_o;    // [splits, B * H, N, D], NULL: not split
  float* part_lse;  // [splits, B * H, N]
  Shape s;
  Grid grid;        // pairs (batch row, key head); per = row tiles * group * splits
  uint32_t row_tiles;
  int32_t splits, tiles_per_split;
  bool late_first;  // the last row tiles are the longest
  float scale_log2, bias_unit;
};

// Keys of a tile: 64, but 32 for fp32 rows of 512 bytes, whose four tiles fill 64 KB.
template <typename T, int DP>
constexpr int local_keys() { return DP * sizeof(T) == 512 ? 32 : 64; }

// As in the cross attention: the maximum may lag by kLag, and fp16's weights are shifted away from its subnormal numbers.
constexpr float kLag = 8.f;
template <typename T>
constexpr float p_shift() { return std::is_same<T, f16>::value ? 6.f : 0.f; }

template <typename T, int DP, int NW, bool BIAS>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(DP * sizeof(T) > 256 ? 1 : 2))) void local_fwd_kernel(FwdArgs a) {
  constexpr int DB = DP * sizeof(T), NS = DB / 32, DT = DP / 32;
  constexpr int BK = local_keys<T, DP>(), SUBS = BK / 32;
  __shared__ __attribute__((aligned(16))) char lds[kStages][2][BK * DB];
  extern __shared__ float table[];
  const int lane = threadIdx.x & 63, h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t pair, sub_block;
  if (!locate(a.grid, pair, sub_block)) return;
  const Shape& s = a.s;
  const uint32_t group = static_cast<uint32_t>(s.G);
  const uint32_t rest = s.by_g.div(sub_block), g = sub_block - rest * group;
  const uint32_t split = rest / a.row_tiles;
  uint32_t row_tile = rest - split * a.row_tiles;
  if (a.late_first) row_tile = a.row_tiles - 1 - row_tile;
  const int b = static_cast<int>(pair) / s.Hk, hk = static_cast<int>(pair) - b * s.Hk, head = hk * s.G + static_cast<int>(g);
  const int d_units = s.D * static_cast<int>(sizeof(T)) / 16;

  const int n0 = static_cast<int>(row_tile) * 32 * NW, n = n0 + wave * 32 + (lane & 31);
  const bool row_ok = n < s.N;
  const bool idle = n0 + wave * 32 >= s.N;  // no query of this wave is there: it only moves tiles
  u32x4_t qf[NS];
  load_frags<T, DP>(static_cast<const T*>(a.q) + b * a.qs.b + head * a.qs.h + (row_ok ? n * a.qs.n : 0), row_ok, d_units, h, qf);

  const int count = key_count(a.km, b, s.M);
  const int start = start_of(a.w, b);
  const int p0 = start + n0 + wave * 32, pos = start + n;
  const TileList list = tiles_of<BK>(a.w, start + n0, start + min(n0 + 32 * NW, s.N) - 1, count);
  const int i0 = static_cast<int>(split) * a.tiles_per_split;
  const int i1 = static_cast<int>(split) + 1 == a.splits ? list.total : min(list.total, i0 + a.tiles_per_split);
  const T* kb = static_cast<const T*>(a.k) + b * a.ks.b + hk * a.ks.h;
  const T* vb = static_cast<const T*>(a.v) + b * a.vs.b + hk * a.vs.h;
  const uint8_t* mask = a.km.mask ? a.km.mask + b * a.km.stride : nullptr;
  const int low = low_of(a.w, pos), high = high_of(a.w, pos, count);

  f32x16_t o[DT]{};
  float ref = -kInf;           // the maximum (in log2 units) P is taken against
  float l[2] = {0.f, 0.f};     // this lane's part of the sum

  Tile<T, DP, BK, NW> kt, vt;
  auto k_at = [&](int i) { return i * a.ks.n; };
  auto v_at = [&](int i) { return i * a.vs.n; };
  const int64_t k_step = BK * static_cast<int64_t>(sizeof(T)) * a.ks.n, v_step = BK * static_cast<int64_t>(sizeof(T)) * a.vs.n;
  kt.start(kb, list.at(i0) * BK, d_units, k_at);
  vt.start(vb, list.at(i0) * BK, d_units, v_at);
  uint8_t byte_now = 1, byte_next = 1;  // this lane's key of the mask
  auto mask_byte = [&](int t) { return mask[min(t * BK + lane, count - 1)]; };
  auto fetch = [&](int i, int stage) {
    const int key0 = list.at(i) * BK;
    if (DB < 512 && key0 + BK <= count) {
      if (i == list.sink && i != i0) {
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
  if (mask && i0 < i1) byte_next = mask_byte(list.at(i0));
  if (i0 < i1) fetch(i0, 0);
  const float* lane_table = nullptr;  // this lane's entry for frame 0
  float far_low = 0.f, far_high = 0.f;
  if constexpr (BIAS) {
    if (i0 < i1) {
      fill_bias<T, false>(table, a.bias, s.H, head, a.bias_unit, 64 * NW);
      __syncthreads();
      far_low = table[0];
      far_high = table[2 * a.bias.distance + 2 * kPad];
    }
    lane_table = table + (a.bias.distance + kPad + 8 * h - pos);
  }
  int stage = 0;
  for (int i = i0; i < i1; ++i) {
    const int t = list.at(i);
    char* kl = lds[stage][0];
    char* vl = lds[stage][1];
    uint64_t seen = range_bits(t * BK, count);
    if (mask) {
      byte_now = byte_next;
      seen &= __ballot(byte_now != 0);
      if (i + 1 < i1) byte_next = mask_byte(list.at(i + 1));
    }
    if constexpr (BK == 32) seen &= 0xFFFFFFFFu;
    constexpr uint64_t kAll = BK == 64 ? ~uint64_t{0} : 0xFFFFFFFFu;
    vm_wait<0>();  // this wave's moves of the tile have arrived
    if (seen != kAll || d_units != kt.UNITS) {
      kt.clear(kl, seen, d_units);
      vt.clear(vl, seen, d_units);
    }
    __syncthreads();
    if (i + 1 < i1) fetch(i + 1, stage ^ 1);
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
      if (what == Sees::kSome || sub_seen != 0xFFFFFFFFu) {
        uint32_t bits = sub_seen;
        if (what == Sees::kSome) bits &= frames_seen(low, high, a.w.sinks, key0);
        bits >>= 8 * h;
#pragma unroll
        for (int r = 0; r < 16; ++r) p[r] = where_bit(bits, reg_key(r), p[r], -kInf);
      }
      float top = fmaxf(p[0], p[1]), top2 = fmaxf(p[2], p[3]);
#pragma unroll
      for (int r = 4; r < 16; r += 4) {
        top = fmaxf(fmaxf(top, p[r]), p[r + 1]);
        top2 = fmaxf(fmaxf(top2, p[r + 2]), p[r + 3]);
      }
      top = half_max(fmaxf(top, top2)) * a.scale_log2;
      if (__any(top > ref + kLag)) {
        const float next = fmaxf(ref, top);
        const float alpha = next == -kInf ? 1.f : __builtin_amdgcn_exp2f(ref - next);
        ref = next;
        l[0] *= alpha;
        l[1] *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
          for (int r = 0; r < 16; ++r) o[dt][r] *= alpha;
        }
      }
      const float base = ref == -kInf ? 0.f : p_shift<T>() - ref;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        p[r] = __builtin_amdgcn_exp2f(fmaf(p[r], a.scale_log2, base));
        l[r & 1] += p[r];
      }
      mma_cols<T, DP>(vl, u, p, o, at_lane);
    }
  }

  const float sum = half_sum(l[0] + l[1]);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  if (!row_ok) return;
  const float lse = sum == 0.f ? -kInf : (ref - p_shift<T>() + __log2f(sum)) * kLn2;
  const int64_t bh = static_cast<int64_t>(b) * s.H + head;
  if (a.part_o) {
    const int64_t at = (static_cast<int64_t>(split) * s.B * s.H + bh) * s.N + n;
    store_cols_f32<T, DP>(a.part_o + at * s.D, o, inv, s.D, h);
    if (h == 0) a.part_lse[at] = lse;
    return;
  }
  const int64_t at = ((static_cast<int64_t>(b) * s.N + n) * s.H + head) * s.D;
  store_cols<T, DP>(static_cast<T*>(a.out) + at, o, inv, s.D, h);
  if (a.lse && h == 0) a.lse[bh * s.N + n] = lse;
}

// Joins the splits: a thread takes 4 columns of a row.  lse = log sum exp(lse_i), O = sum exp(lse_i - lse) O_i.
template <typename T>
__global__ __launch_bounds__(256) void local_join_kernel(FwdArgs a, uint32_t quads_per_row, FastDiv by_quads, uint32_t total) {
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  if (i >= total) return;
  const uint32_t row = by_quads.div(i), quad = i - row * quads_per_row;
  const Shape& s = a.s;
  const int64_t rows = static_cast<int64_t>(s.B) * s.H * s.N;
  float top = -kInf, sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int k = 0; k < a.splits; k += 4) {  // four splits' loads at a time
    float l[4], x[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t at = min(k + j, a.splits - 1) * rows + row;
      l[j] = a.part_lse[at];
      load_pack<float, 4>(a.part_o + at * s.D + 4 * quad, x[j]);
    }
    float next = top;
#pragma unroll
    for (int j = 0; j < 4; ++j) next = fmaxf(next, l[j]);
    const float f = top == -kInf ? 0.f : __builtin_amdgcn_exp2f((top - next) * kLog2e);
    top = next;
    sum *= f;
#pragma unroll
    for (int c = 0; c < 4; ++c) o[c] *= f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // a split without frames (or, where none is seen, every one) has no weight; NaN stays NaN
      const float w = k + j >= a.splits || l[j] == -kInf ? 0.f : __builtin_amdgcn_exp2f((l[j] - top) * kLog2e);
      sum += w;
#pragma unroll
      for (int c = 0; c < 4; ++c) o[c] = w == 0.f ? o[c] : fmaf(w, x[j][c], o[c]);
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const uint32_t bh = row / static_cast<uint32_t>(s.N), n = row - bh * static_cast<uint32_t>(s.N);
  const uint32_t b = bh / static_cast<uint32_t>(s.H), head = bh - b * static_cast<uint32_t>(s.H);
  const int64_t at = ((static_cast<int64_t>(b) * s.N + n) * s.H + head) * s.D + 4 * quad;
#pragma unroll
  for (int c = 0; c < 4; ++c) o[c] *= inv;
  store_pack<T, 4>(static_cast<T*>(a.out) + at, o);
  if (a.lse && quad == 0) a.lse[row] = sum == 0.f ? -kInf : top + __log2f(sum) * kLn2;
}

// ---------------------------------------------------------------- host

struct FwdPlan {
  int nw;
  int64_t row_tiles, splits, tiles_per_split;
};

// Waves of a block: 2 where that covers the queries (fp32 rows of 512 bytes keep 4): 1032 x 62 queries, 8 heads of 64, 74 us
// against 78; with more queries 4 read each tile half as often (248 x 258: 102 against 150; 124 x 948: 376 against 575).
// Splits: of at least 128 frames, up to 4 blocks of 4 waves (2 of 2 waves) a CU: 2 x 64 queries, 16 heads on 4,
// window of 4095, 15.4 us and a join of 4.4 against 82 without; fp32, 4 x 317 queries, 24 and 4.3 against 32.  More and
// smaller splits cost the join what the pass gains (14.0 and 6.1).
FwdPlan plan_forward(const Shape& s, const Window& w, int dtype) {
  FwdPlan p;
  const bool wide = padded_dim(s.D) * static_cast<int>(dtype_size(dtype)) == 512;
  p.nw = s.N <= 64 && !wide ? 2 : 4;
  const int64_t bk = wide ? 32 : 64, rows = 32 * p.nw;
  p.row_tiles = (int64_t{s.N} + rows - 1) / rows;
  // the most tiles that a block visits
  int64_t tiles = std::max<int64_t>(1, (int64_t{s.M} + bk - 1) / bk);
  if (w.left >= 0 && w.right >= 0) {
    tiles = std::min(tiles, (int64_t{w.left} + w.right + std::min<int64_t>(rows, s.N) + bk - 1) / bk + 1 + (w.sinks + bk - 1) / bk);
  }
  const int64_t blocks = int64_t{s.B} * s.H * p.row_tiles, want = (p.nw == 4 ? 4 : 2) * num_cus();
  p.splits = 1;
  if (blocks < want) p.splits = std::max<int64_t>(1, std::min((want + blocks - 1) / blocks, tiles * bk / 128));
  p.tiles_per_split = (tiles + p.splits - 1) / p.splits;
  p.splits = (tiles + p.tiles_per_split - 1) / p.tiles_per_split;
  return p;
}

template <typename T, int DP, int NW>
int launch_fwd(const FwdArgs& a, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(grid_blocks(a.grid)));
  if (a.bias.table) {
    local_fwd_kernel<T, DP, NW, true><<<grid, 64 * NW, bias_entries(a.bias.distance) * 4, stream>>>(a);
  } else {
    local_fwd_kernel<T, DP, NW, false><<<grid, 64 * NW, 0, stream>>>(a);
  }
  return check_launch("local_fwd_kernel");
}

template <typename T, int DP>
int launch_fwd(const FwdArgs& a, const FwdPlan& p, hipStream_t stream) {
  if constexpr (DP * sizeof(T) != 512) {
    if (p.nw == 2) return launch_fwd<T, DP, 2>(a, stream);
  }
  return launch_fwd<T, DP, 4>(a, stream);
}

template <typename T>
int run_fwd(const FwdArgs& a, const FwdPlan& p, hipStream_t stream) {
  const int rc = a.s.D <= 32   ? launch_fwd<T, 32>(a, p, stream)
                 : a.s.D <= 64 ? launch_fwd<T, 64>(a, p, stream)
                               : launch_fwd<T, 128>(a, p, stream);
  if (rc != PMSST_OK || p.splits == 1) return rc;
  const uint32_t quads = static_cast<uint32_t>(a.s.D / 4);
  const uint32_t total = static_cast<uint32_t>(a.s.B) * a.s.H * a.s.N * quads;
  local_join_kernel<T><<<dim3((total + 255) / 256), 256, 0, stream>>>(a, quads, FastDiv(quads), total);
  return check_launch("local_join_kernel");
}

size_t fwd_workspace(const Shape& s, const FwdPlan& p) {
  if (p.splits == 1) return 0;
  const size_t rows = static_cast<size_t>(p.splits) * s.B * s.H * s.N;
  return align_up(rows * s.D * 4, 256) + align_up(rows * 4, 256);
}

}  // namespace

namespace attn {

int make_local(const char* what, int64_t batch, int64_t queries, int64_t keys, int64_t heads, int64_t kv_heads, int64_t head_dim,
               int64_t left, int64_t right, int64_t sinks, const int32_t* starts, const void* bias, int bias_dtype,
               const int32_t* bucket_of, int64_t buckets, int64_t distance, double scale, int dtype, LocalArgs& out) {
  const int rc = make_shape(what, batch, queries, keys, heads, kv_heads, head_dim, dtype, out.s);
  if (rc != PMSST_OK) return rc;
  PMSST_REQUIRE(scale > 0.0 && scale < 1e30, "%s: scale must be positive", what);
  PMSST_REQUIRE(queries <= kMaxFrames && keys <= kMaxFrames, "%s: more than 2^28 queries or frames", what);
  PMSST_REQUIRE(left >= -1 && left <= 2 * kMaxFrames && right >= -1 && right <= 2 * kMaxFrames,
                "%s: left and right must be -1 (no limit) or lie in [0, 2^29]", what);
  PMSST_REQUIRE(sinks >= 0 && sinks <= kMaxFrames, "%s: sinks must lie in [0, 2^28]", what);
  // limits that nothing lies beyond are none
  if (starts == nullptr && left >= queries - 1) left = -1;
  if (starts == nullptr && right >= keys - 1) right = -1;
  out.w = {static_cast<int32_t>(left), static_cast<int32_t>(right), left < 0 ? 0 : static_cast<int32_t>(sinks), starts};
  out.bias = {};
  out.cut = 0;
  if (bias == nullptr) return PMSST_OK;
  PMSST_REQUIRE(bucket_of != nullptr, "%s: null pointer (bucket_of)", what);
  PMSST_REQUIRE(buckets >= 1 && buckets <= kMaxBuckets, "%s: the bias has 1 to %d buckets", what, kMaxBuckets);
  PMSST_REQUIRE(distance >= 0 && distance <= kMaxDistance, "%s: the bias's largest distance must lie in [0, %d]", what, kMaxDistance);
  PMSST_REQUIRE(scale >= 0x1p-20 && scale <= 0x1p20, "%s: with a bias, scale must lie in [2^-20, 2^20]", what);
  if (bias_dtype != PMSST_F32 && bias_dtype != dtype) return fail(PMSST_EDTYPE, "%s: the bias must be fp32 or of q's dtype", what);
  const int64_t reach = reach_of(out.s, out.w, distance);
  out.cut = static_cast<int32_t>(distance - reach);
  out.bias = {bias, bucket_of + out.cut, static_cast<int32_t>(buckets), static_cast<int32_t>(reach), bias_dtype == PMSST_F32};
  return PMSST_OK;
}

}  // namespace attn
}  // namespace pmsst

extern "C" {

size_t pmsst_local_attention_forward_workspace_size(int64_t batch, int64_t queries, int64_t keys, int64_t heads, int64_t kv_heads,
                                                    int64_t head_dim, int64_t left, int64_t right, int64_t sinks, int has_starts,
                                                    int dtype) {
  pmsst::attn::LocalArgs l;
  static const int32_t some = 0;
  if (pmsst::attn::make_local("pmsst_local_attention_forward", batch, queries, keys, heads, kv_heads, head_dim, left, right, sinks,
                              has_starts ? &some : nullptr, nullptr, 0, nullptr, 0, 0, 1.0, dtype, l) != PMSST_OK ||
      l.s.B == 0 || l.s.N == 0)
    return 0;
  return pmsst::fwd_workspace(l.s, pmsst::plan_forward(l.s, l.w, dtype));
}

int pmsst_local_attention_forward(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v,
                                  const int64_t* v_strides, const uint8_t* key_mask, int64_t key_mask_stride,
                                  const int32_t* key_lengths, const int32_t* query_starts, int64_t left, int64_t right,
                                  int64_t sinks, const void* bias, int bias_dtype, const int32_t* bucket_of, int64_t buckets,
                                  int64_t max_distance, void* out, float* lse, int64_t batch, int64_t queries, int64_t keys,
                                  int64_t heads, int64_t kv_heads, int64_t head_dim, double scale, int dtype,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  using namespace pmsst;
  using namespace pmsst::attn;
  const char* what = "pmsst_local_attention_forward";
  LocalArgs l;
  int rc = make_local(what, batch, queries, keys, heads, kv_heads, head_dim, left, right, sinks, query_starts, bias, bias_dtype,
                      bucket_of, buckets, max_distance, scale, dtype, l);
  if (rc != PMSST_OK) return rc;
  if (batch == 0 || queries == 0) return PMSST_OK;
  PMSST_REQUIRE(q && out && (keys == 0 || (k && v)), "%s: null pointer", what);
  FwdArgs a{};
  a.s = l.s;
  a.w = l.w;
  a.bias = l.bias;
  if ((rc = make_strides(what, q, q_strides, queries, heads, head_dim, dtype, a.qs)) != PMSST_OK) return rc;
  if ((rc = make_strides(what, k, k_strides, keys, kv_heads, head_dim, dtype, a.ks)) != PMSST_OK) return rc;
  if ((rc = make_strides(what, v, v_strides, keys, kv_heads, head_dim, dtype, a.vs)) != PMSST_OK) return rc;
  PMSST_REQUIRE((reinterpret_cast<uintptr_t>(out) & 15) == 0, "%s: out must be 16-byte aligned", what);
  const FwdPlan p = plan_forward(a.s, a.w, dtype);
  const size_t need = fwd_workspace(a.s, p);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return fail(PMSST_EWORKSPACE, "%s: workspace of %zu bytes needed, %zu given", what, need, workspace_bytes);
  PMSST_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0 || need == 0, "%s: workspace must be 16-byte aligned", what);
  a.q = q;
  a.k = k;
  a.v = v;
  a.km = {key_mask, key_mask_stride, key_lengths};
  a.out = out;
  a.lse = lse;
  if (need > 0) {
    a.part_o = static_cast<float*>(workspace);
    const size_t rows = static_cast<size_t>(p.splits) * a.s.B * a.s.H * a.s.N;
    a.part_lse = reinterpret_cast<float*>(static_cast<char*>(workspace) + align_up(rows * a.s.D * 4, 256));
  }
  a.row_tiles = static_cast<uint32_t>(p.row_tiles);
  a.splits = static_cast<int32_t>(p.splits);
  a.tiles_per_split = static_cast<int32_t>(p.tiles_per_split);
  a.late_first = a.w.right >= 0 && a.w.left < 0;
  const int64_t pairs = batch * kv_heads, per = p.row_tiles * a.s.G * p.splits;
  PMSST_REQUIRE(grid_fits(pairs, per), "%s: too many rows for one call", what);
  a.grid = make_grid(pairs, per);
  a.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  a.bias_unit = static_cast<float>(1.0 / scale);
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case PMSST_F32: return run_fwd<float>(a, p, st);
    case PMSST_F16: return run_fwd<f16>(a, p, st);
    default: return run_fwd<bf16>(a, p, st);
  }
}

}  // extern "C"
