// Cross attention forward: O = softmax(scale Q K^T over the seen keys) V, with the weights' dropout.
//
// One pass over the keys with a running maximum and sum (per row, fp32): with s the scores of a tile,
//   m' = max(m, max s),  l' = l exp(m - m') + sum exp(s - m'),  O' = O exp(m - m') + exp(s - m') V,
// and O / l at the end.  attention.h describes the tiles.  A block is NW waves of 32 rows; K and V tiles of BK
// keys are moved from memory straight into two LDS stages in turn, so that a tile is on its way while the one
// before it is multiplied.
//
// Bound: with many rows the matrix cores and the vector unit together (exponentials, sums and conversions of a tile take
// about as long as its products), at the clock that this mix leaves, 1.7 to 1.9 GHz of 2.4: 124 x 948 queries over 948
// keys, 8 heads of 64, fp16, 334 us = 680 TFLOP/s (a library product of 8192^3 reaches 1100).  With short rows HBM:
// 1032 x 62 over 62, bf16, 62 us = 4.2 TB/s in a training step (50 us where the call before has left its tensors in the
// last-level cache).  With single queries of 16 bits HBM as well: 16 x 8 heads over up to 16500 keys, 84 us = 4.8 TB/s.
// In fp32 their empty rows bound them: a wave multiplies 32 rows for the one that is there (8 x 8 heads over up to
// 16500 keys, as many bytes, 192 us).
//
// Few rows over many keys (single queries) are split over the keys: every split leaves its normalised O and
// its lse in the workspace, and a second kernel adds them with weights exp(lse_i - lse).
#include "attention.h"

namespace pmsst {
namespace {

using namespace attn;

struct FwdArgs {
  const void *q, *k, *v;
  Strides qs, ks, vs;
  KeyMask km;
  void* out;
  float* lse;       // [B, H, N] or NULL
  float* part_o;    // [splits, B * Hk, R, D], NULL: not split
  float* part_lse;  // [splits, B * Hk, R]
  Shape s;
  Grid grid;        // per = row tiles * splits
  uint32_t row_tiles;
  int32_t tiles_per_split;
  float scale_log2;  // scale * log2(e)
  Dropout drop;
};

// Keys of a tile: 64, but 32 for fp32 rows of 512 bytes, whose four tiles fill 64 KB.
template <typename T, int DP>
constexpr int fwd_keys() { return DP * sizeof(T) == 512 ? 32 : 64; }

// P is rounded to 16 bits as the next product's operand.  Its values are exp2(s - m + kShift): the maximum a
// row's values are taken against may lag by kLag before O is rescaled (a rescale is skipped for as long as no
// row of the wave needs one), and fp16 is shifted so that the least of what counts is no subnormal number.
constexpr float kLag = 8.f;
template <typename T>
constexpr float p_shift() { return std::is_same<T, f16>::value ? 6.f : 0.f; }

template <typename T, int DP, int NW, bool DROP>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(DP * sizeof(T) > 256 ? 1 : 2))) void attn_fwd_kernel(FwdArgs a) {
  constexpr int DB = DP * sizeof(T), NS = DB / 32, DT = DP / 32;
  constexpr int BK = fwd_keys<T, DP>(), SUBS = BK / 32;
  __shared__ __attribute__((aligned(16))) char lds[kStages][2][BK * DB];
  const int lane = threadIdx.x & 63, h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t pair, sub_block;
  if (!locate(a.grid, pair, sub_block)) return;
  const uint32_t split = sub_block / a.row_tiles, row_tile = sub_block - split * a.row_tiles;
  const Shape& s = a.s;
  const int b = static_cast<int>(pair) / s.Hk, hk = static_cast<int>(pair) - b * s.Hk;
  const int d_units = s.D * static_cast<int>(sizeof(T)) / 16;

  const int r = static_cast<int>(row_tile) * 32 * NW + wave * 32 + (lane & 31);
  const bool row_ok = r < s.R;
  const bool idle = __builtin_amdgcn_readfirstlane(r) >= s.R;  // no row of this wave is there: it only moves tiles
  const int n = static_cast<int>(s.by_g.div(static_cast<uint32_t>(r))), head = hk * s.G + (r - n * s.G);
  u32x4_t qf[NS];
  load_frags<T, DP>(static_cast<const T*>(a.q) + b * a.qs.b + (row_ok ? n * a.qs.n + head * a.qs.h : 0), row_ok, d_units,
                    h, qf);

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

  f32x16_t o[DT]{};
  float ref = -kInf;           // the maximum (in log2 units) P is taken against
  float l[2] = {0.f, 0.f};     // this lane's part of the sum

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
      if (sub_seen != 0xFFFFFFFFu) {
#pragma unroll
        for (int i = 0; i < 16; ++i) p[i] = where_bit(sub_seen >> (8 * h), reg_key(i), p[i], -kInf);
      }
      float top = fmaxf(p[0], p[1]), top2 = fmaxf(p[2], p[3]);
#pragma unroll
      for (int i = 4; i < 16; i += 4) {
        top = fmaxf(fmaxf(top, p[i]), p[i + 1]);
        top2 = fmaxf(fmaxf(top2, p[i + 2]), p[i + 3]);
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
          for (int i = 0; i < 16; ++i) o[dt][i] *= alpha;
        }
      }
      const float base = ref == -kInf ? 0.f : p_shift<T>() - ref;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        p[i] = __builtin_amdgcn_exp2f(fmaf(p[i], a.scale_log2, base));
        l[i & 1] += p[i];
      }
      if constexpr (DROP && sizeof(T) == 2) {
        // a word of random bits is two elements, as a word of the packed weights is
        u32x4_t pb[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint32_t w[4];
          philox7(key, drop0 + static_cast<uint32_t>(t * (BK / 8) + 4 * u + 2 * j + h), w);
          pb[j] = pack8<T>(p, j);
#pragma unroll
          for (int i = 0; i < 4; ++i) pb[j][i] &= ~philox_dropped(w[i], a.drop.limit);
        }
        mma_cols<T, DP>(vl, u, pb, o, at_lane);
        continue;
      }
      if constexpr (DROP) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint32_t w[4];
          philox7(key, drop0 + static_cast<uint32_t>(t * (BK / 8) + 4 * u + 2 * j + h), w);
#pragma unroll
          for (int i = 0; i < 8; ++i) p[8 * j + i] = philox_keep(w, i, a.drop.limit) ? p[8 * j + i] : 0.f;
        }
      }
      mma_cols<T, DP>(vl, u, p, o, at_lane);
    }
  }

  const float sum = half_sum(l[0] + l[1]);
  const float inv = sum == 0.f ? 0.f : (DROP ? a.drop.factor : 1.f) / sum;
  if (!row_ok) return;
  const float lse = sum == 0.f ? -kInf : (ref - p_shift<T>() + __log2f(sum)) * kLn2;
  if (a.part_o) {
    const int64_t at = (static_cast<int64_t>(split) * a.grid.pairs + pair) * s.R + r;
    store_cols_f32<T, DP>(a.part_o + at * s.D, o, inv, s.D, h);
    if (h == 0) a.part_lse[at] = lse;
    return;
  }
  const int64_t at = (static_cast<int64_t>(b) * s.N + n) * s.H + head;
  store_cols<T, DP>(static_cast<T*>(a.out) + at * s.D, o, inv, s.D, h);
  if (a.lse && h == 0) a.lse[(static_cast<int64_t>(b) * s.H + head) * s.N + n] = lse;
}

// Joins the splits: a thread takes 4 columns of a row.  lse = log sum exp(lse_i), O = sum exp(lse_i - lse) O_i.
template <typename T>
__global__ __launch_bounds__(256) void attn_join_kernel(FwdArgs a, int splits, uint32_t quads_per_row, FastDiv by_quads,
                                                        uint32_t total) {
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  if (i >= total) return;
  const uint32_t row = by_quads.div(i), quad = i - row * quads_per_row;
  const Shape& s = a.s;
  const int64_t rows = static_cast<int64_t>(a.grid.pairs) * s.R;
  float top = -kInf;
  for (int k = 0; k < splits; ++k) top = fmaxf(top, a.part_lse[k * rows + row]);
  float sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int k = 0; k < splits; ++k) {
    const float li = a.part_lse[k * rows + row];
    // a split without keys (or, where no key is seen, every one) has no weight; NaN stays NaN
    const float w = li == -kInf ? 0.f : __builtin_amdgcn_exp2f((li - top) * kLog2e);
    float x[4];
    load_pack<float, 4>(a.part_o + (k * rows + row) * s.D + 4 * quad, x);
    sum += w;
#pragma unroll
    for (int c = 0; c < 4; ++c) o[c] = fmaf(w, x[c], o[c]);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int c = 0; c < 4; ++c) o[c] *= inv;
  const uint32_t pair = row / static_cast<uint32_t>(s.R);
  const int r = static_cast<int>(row - pair * static_cast<uint32_t>(s.R));
  const int b = static_cast<int>(pair) / s.Hk, hk = static_cast<int>(pair) - b * s.Hk;
  const int n = static_cast<int>(s.by_g.div(static_cast<uint32_t>(r))), head = hk * s.G + (r - n * s.G);
  const int64_t at = (static_cast<int64_t>(b) * s.N + n) * s.H + head;
  store_pack<T, 4>(static_cast<T*>(a.out) + at * s.D + 4 * quad, o);
  if (a.lse && quad == 0) {
    a.lse[(static_cast<int64_t>(b) * s.H + head) * s.N + n] = sum == 0.f ? -kInf : top + __log2f(sum) * kLn2;
  }
}

// ---------------------------------------------------------------- host

struct FwdPlan {
  int nw;
  int bk;
  int64_t row_tiles, splits, tiles_per_split;
};

// Waves of a block: 2 where that covers the rows (half a block of 4 would idle; fp32 rows of 512 bytes keep 4,
// whose lanes hold half as much of a tile on its way), else 4.  Splits: of at least 128 keys, up to 4 blocks of 4
// waves a CU, whose products bound them and whose ragged ends so even out (2760 queries over up to 8192 keys,
// heads of 128: 240 us; with 2 blocks a CU 272, with 8 258), or of at least 512 keys, up to 2 blocks of 2 waves, which the
// keys' bytes bound in 16 bits (16 single queries over up to 16500 keys: 89 us; with 4 blocks 100, with 1 134; a tile of 64
// keys takes about 1 us and the second kernel 5).  fp32's single queries, bound by the products of empty rows, gain
// nothing by more blocks either (8 over up to 16500 keys: 192 us; with 4 blocks 203); rows of 512 bytes come under the first
// rule (16 over up to 4097 keys, heads of 128: 101 us; with 2 blocks 108, with 8 102).
FwdPlan plan_forward(const Shape& s, int dtype) {
  FwdPlan p;
  const bool wide = padded_dim(s.D) * static_cast<int>(dtype_size(dtype)) == 512;
  p.nw = s.R <= 64 && !wide ? 2 : 4;
  p.bk = wide ? 32 : 64;
  p.row_tiles = (int64_t{s.R} + 32 * p.nw - 1) / (32 * p.nw);
  const int64_t tiles = std::max<int64_t>(1, (int64_t{s.M} + p.bk - 1) / p.bk);
  const int64_t blocks = int64_t{s.B} * s.Hk * p.row_tiles, want = (p.nw == 4 ? 4 : 2) * num_cus();
  p.splits = 1;
  if (blocks < want) p.splits = std::max<int64_t>(1, std::min((want + blocks - 1) / blocks, int64_t{s.M} / (p.nw == 4 ? 128 : 512)));
  p.tiles_per_split = (tiles + p.splits - 1) / p.splits;
  p.splits = (tiles + p.tiles_per_split - 1) / p.tiles_per_split;
  return p;
}

template <typename T, int DP, int NW>
int launch_fwd(const FwdArgs& a, bool drop, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(grid_blocks(a.grid)));
  if (drop) attn_fwd_kernel<T, DP, NW, true><<<grid, 64 * NW, 0, stream>>>(a);
  else attn_fwd_kernel<T, DP, NW, false><<<grid, 64 * NW, 0, stream>>>(a);
  return check_launch("attn_fwd_kernel");
}

template <typename T, int DP>
int launch_fwd(const FwdArgs& a, const FwdPlan& p, bool drop, hipStream_t stream) {
  if constexpr (DP * sizeof(T) != 512) {
    if (p.nw == 2) return launch_fwd<T, DP, 2>(a, drop, stream);
  }
  return launch_fwd<T, DP, 4>(a, drop, stream);
}

template <typename T>
int run_fwd(const FwdArgs& a, const FwdPlan& p, bool drop, hipStream_t stream) {
  const int rc = a.s.D <= 32   ? launch_fwd<T, 32>(a, p, drop, stream)
                 : a.s.D <= 64 ? launch_fwd<T, 64>(a, p, drop, stream)
                               : launch_fwd<T, 128>(a, p, drop, stream);
  if (rc != PMSST_OK || p.splits == 1) return rc;
  const uint32_t quads = static_cast<uint32_t>(a.s.D / 4);
  const uint32_t total = a.grid.pairs * static_cast<uint32_t>(a.s.R) * quads;
  attn_join_kernel<T><<<dim3((total + 255) / 256), 256, 0, stream>>>(a, static_cast<int>(p.splits), quads, FastDiv(quads),
                                                                      total);
  return check_launch("attn_join_kernel");
}

size_t fwd_workspace(const Shape& s, const FwdPlan& p) {
  if (p.splits == 1) return 0;
  const size_t rows = static_cast<size_t>(p.splits) * s.B * s.Hk * s.R;
  return align_up(rows * s.D * 4, 256) + align_up(rows * 4, 256);
}

}  // namespace

namespace attn {

int make_shape(const char* what, int64_t batch, int64_t queries, int64_t keys, int64_t heads, int64_t kv_heads,
               int64_t head_dim, int dtype, Shape& s) {
  if (!dtype_ok(dtype)) return fail(PMSST_EDTYPE, "%s: unsupported dtype %d", what, dtype);
  constexpr int64_t kMax = int64_t{1} << 30;
  PMSST_REQUIRE(batch >= 0 && queries >= 0 && keys >= 0 && heads > 0 && kv_heads > 0, "%s: bad size", what);
  PMSST_REQUIRE(heads % kv_heads == 0, "%s: kv_heads must divide heads", what);
  PMSST_REQUIRE(head_dim >= 8 && head_dim <= 128 && head_dim % 8 == 0, "%s: head_dim must be a multiple of 8 in [8, 128]",
                what);
  PMSST_REQUIRE(batch <= kMax && queries <= kMax && keys <= kMax && heads <= kMax, "%s: size above 2^30", what);
  const int64_t g = heads / kv_heads;
  PMSST_REQUIRE(queries == 0 || g <= kMax / queries, "%s: more than 2^30 rows share a key head", what);
  PMSST_REQUIRE(batch == 0 || kv_heads <= kMax / batch, "%s: more than 2^30 batch rows and key heads", what);
  s.B = static_cast<int32_t>(batch);
  s.N = static_cast<int32_t>(queries);
  s.M = static_cast<int32_t>(keys);
  s.H = static_cast<int32_t>(heads);
  s.Hk = static_cast<int32_t>(kv_heads);
  s.D = static_cast<int32_t>(head_dim);
  s.G = static_cast<int32_t>(g);
  s.R = static_cast<int32_t>(g * queries);
  s.by_g = FastDiv(static_cast<uint32_t>(s.G));
  return PMSST_OK;
}

int make_strides(const char* what, const void* p, const int64_t* strides, int64_t positions, int64_t heads, int64_t dim,
                 int dtype, Strides& out) {
  out = strides ? Strides{strides[0], strides[1], strides[2]} : Strides{positions * heads * dim, heads * dim, dim};
  const int64_t unit = 16 / static_cast<int64_t>(dtype_size(dtype));
  PMSST_REQUIRE((reinterpret_cast<uintptr_t>(p) & 15) == 0 && out.b % unit == 0 && out.n % unit == 0 && out.h % unit == 0,
                "%s: tensors and their strides must be whole 16 bytes", what);
  return PMSST_OK;
}

}  // namespace attn
}  // namespace pmsst

extern "C" {

size_t pmsst_cross_attention_forward_workspace_size(int64_t batch, int64_t queries, int64_t keys, int64_t heads,
                                                    int64_t kv_heads, int64_t head_dim, int dtype) {
  pmsst::attn::Shape s;
  if (pmsst::attn::make_shape("pmsst_cross_attention_forward", batch, queries, keys, heads, kv_heads, head_dim, dtype, s) !=
          PMSST_OK ||
      s.B == 0 || s.N == 0)
    return 0;
  return pmsst::fwd_workspace(s, pmsst::plan_forward(s, dtype));
}

int pmsst_cross_attention_forward(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                                  const void* v, const int64_t* v_strides, const uint8_t* key_mask,
                                  int64_t key_mask_stride, const int32_t* key_lengths, void* out, float* lse,
                                  int64_t batch, int64_t queries, int64_t keys, int64_t heads, int64_t kv_heads,
                                  int64_t head_dim, double scale, double dropout_p, const int64_t* rng, int dtype,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  using namespace pmsst;
  using namespace pmsst::attn;
  const char* what = "pmsst_cross_attention_forward";
  FwdArgs a{};
  int rc = make_shape(what, batch, queries, keys, heads, kv_heads, head_dim, dtype, a.s);
  if (rc != PMSST_OK) return rc;
  PMSST_REQUIRE(scale > 0.0 && scale < 1e30, "%s: scale must be positive", what);
  PMSST_REQUIRE(dropout_p >= 0.0 && dropout_p < 1.0, "%s: the dropout probability must lie in [0, 1)", what);
  if (batch == 0 || queries == 0) return PMSST_OK;
  PMSST_REQUIRE(q && out && (keys == 0 || (k && v)), "%s: null pointer", what);
  if ((rc = make_strides(what, q, q_strides, queries, heads, head_dim, dtype, a.qs)) != PMSST_OK) return rc;
  if ((rc = make_strides(what, k, k_strides, keys, kv_heads, head_dim, dtype, a.ks)) != PMSST_OK) return rc;
  if ((rc = make_strides(what, v, v_strides, keys, kv_heads, head_dim, dtype, a.vs)) != PMSST_OK) return rc;
  PMSST_REQUIRE((reinterpret_cast<uintptr_t>(out) & 15) == 0, "%s: out must be 16-byte aligned", what);
  a.drop = make_dropout(dropout_p, rng);
  PMSST_REQUIRE(rng || a.drop.limit == 0, "%s: null pointer (rng)", what);
  const FwdPlan p = plan_forward(a.s, dtype);
  const size_t need = fwd_workspace(a.s, p);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return fail(PMSST_EWORKSPACE, "%s: workspace of %zu bytes needed, %zu given", what, need, workspace_bytes);
  PMSST_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0 || need == 0, "%s: workspace must be 16-byte aligned",
                what);
  a.q = q;
  a.k = k;
  a.v = v;
  a.km = {key_mask, key_mask_stride, key_lengths};
  a.out = out;
  a.lse = lse;
  if (need > 0) {
    a.part_o = static_cast<float*>(workspace);
    const size_t rows = static_cast<size_t>(p.splits) * a.s.B * a.s.Hk * a.s.R;
    a.part_lse = reinterpret_cast<float*>(static_cast<char*>(workspace) + align_up(rows * a.s.D * 4, 256));
  }
  a.row_tiles = static_cast<uint32_t>(p.row_tiles);
  a.tiles_per_split = static_cast<int32_t>(p.tiles_per_split);
  const int64_t pairs = batch * kv_heads, per = p.row_tiles * p.splits;
  PMSST_REQUIRE(grid_fits(pairs, per), "%s: too many rows for one call", what);
  a.grid = make_grid(pairs, per);
  a.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool drop = a.drop.limit != 0;
  switch (dtype) {
    case PMSST_F32: return run_fwd<float>(a, p, drop, st);
    case PMSST_F16: return run_fwd<f16>(a, p, drop, st);
    default: return run_fwd<bf16>(a, p, drop, st);
  }
}

}  // extern "C"
