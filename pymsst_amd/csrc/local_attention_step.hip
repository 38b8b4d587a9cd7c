// Local attention frame by frame: a few new frames of each stream are written into its ring caches and attended to with
// the first frames (sinks) and the last ones that the caches hold, in one launch, or two where blocks are split.
//
// The bytes of the keys and values bound it, so there are no matrix instructions and no LDS tiles: a row of K is
// spread over the lanes of a group, 16 bytes each, and a wave's load takes 64 / group rows.  Every lane keeps the
// products' columns it loads: its part of q, of the sums O, and its group's own maximum and sum of the weights.  Groups
// meet once, at the end: within the wave by lane exchanges, between waves through LDS, between blocks (where few
// streams have long windows) through the workspace and a second kernel.
//
// A block takes up to 8 rows (query heads that share the key head, times new frames) so that each K and V is read once
// for all of them.
//
// The slots that are written hold frames that no query of the call sees (slots - sinks >= left + frames), and the new
// frames are read from k and v, not from the caches: no block waits for another.
//
// One row: HBM and the launch; 8 rows of a shared key head: the same (200 MB of fp16 keys and values of 128 in 47 us, 4.3
// TB/s).  Four rows with a bias: the vector unit (219 MB in 58 us, 3.8 TB/s; a padded table that saves the lookups' cuts changes
// nothing).  The smallest call's kernel is 5 us and its enqueue 15.  Waves of a block: 8 in place of 4 took 50 us for 47, 2 took 80; loads in
// flight a lane: kUnroll of 2 and 8 took 48 and 50.
#include "local_attention.h"

namespace pmsst {
namespace {

using namespace attn;

struct StepArgs {
  const void *q, *k, *v;
  void *k_cache, *v_cache;
  Strides qs, ks, vs, kcs, vcs;
  const int32_t* positions;
  int32_t left, sinks, ring;
  BiasArgs bias;
  void* out;
  float *part_o, *part_m, *part_l;  // [splits, B * Hk, R, D] and [splits, B * Hk, R]: sums, maxima, sums of weights
  Shape s;                          // N: new frames; R = G * N rows of a (stream, key head), r = n * G + g
  Grid grid;                        // per = row chunks * splits
  FastDiv by_ring;
  uint32_t splits;
  int32_t per_split;                // frames
  float scale_log2;
};

// f of this lane's value and that of lane l ^ 16, the lower lane's first.
template <typename F>
__device__ __forceinline__ float rows_join(float v, F f) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t a = r[0], b = r[1];
  return f(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}

// Sum over the aligned groups of LPR lanes, by lane moves in the adder's own operand.
template <int LPR>
__device__ __forceinline__ float lanes_sum(float v) {
  v += dpp_mov<0xB1>(v);                                    // quad_perm [1,0,3,2]
  v += dpp_mov<0x4E>(v);                                    // quad_perm [2,3,0,1]
  if constexpr (LPR >= 8) v += dpp_mov<0x141>(v);           // row_half_mirror
  if constexpr (LPR >= 16) v += dpp_mov<0x140>(v);          // row_mirror
  if constexpr (LPR >= 32) v = rows_join(v, [](float x, float y) { return x + y; });
  return v;
}

// f over the lanes that share (lane % LPR).
template <int LPR, typename F>
__device__ __forceinline__ float groups_join(float v, F f) {
  if constexpr (LPR <= 4) v = f(v, dpp_mov<0x124>(v));  // row_ror:4
  if constexpr (LPR <= 8) v = f(v, dpp_mov<0x128>(v));  // row_ror:8
  if constexpr (LPR <= 16) v = rows_join(v, f);
  float lo, hi;
  halves(v, lo, hi);
  return f(lo, hi);
}

// Products of two 16-byte units, added to `sum` in fp32: 16-bit types two elements an instruction.
template <typename T>
__device__ __forceinline__ float dot(const u32x4_t& a, const u32x4_t& b, float sum) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t x = a[i], y = b[i];
    if constexpr (std::is_same<T, bf16>::value) {
      typedef __bf16 v2 __attribute__((ext_vector_type(2)));
      sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2, x), __builtin_bit_cast(v2, y), sum, false);
    } else if constexpr (std::is_same<T, f16>::value) {
      typedef _Float16 v2 __attribute__((ext_vector_type(2)));
      sum = __builtin_amdgcn_fdot2(__builtin_bit_cast(v2, x), __builtin_bit_cast(v2, y), sum, false);
    } else {
      sum = fmaf(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y), sum);
    }
  }
  return sum;
}

// What the lanes past a row's end multiply (with 0: nothing there may be infinite).
static __device__ const u32x4_t zero_unit = {0, 0, 0, 0};

constexpr int kUnroll = 4;  // loads of K (and of V) on their way in a wave

// LPR: lanes of a row (a power of two), RT: rows of the block.
template <typename T, int LPR, int RT, bool BIAS>
__global__ __launch_bounds__(256) void local_step_kernel(StepArgs a) {
  constexpr int E = 16 / sizeof(T), KPW = 64 / LPR;
  extern __shared__ float shared[];  // the bias of the rows' heads by distance back, then the waves' results
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  uint32_t pair, sub;
  if (!locate(a.grid, pair, sub)) return;
  const Shape& s = a.s;
  const uint32_t chunk = sub / a.splits, split = sub - chunk * a.splits;
  const int b = static_cast<int>(pair) / s.Hk, hk = static_cast<int>(pair) - b * s.Hk;
  const int r0 = static_cast<int>(chunk) * RT, rows = min(RT, s.R - r0);
  const int unit = lane & (LPR - 1), slot_in_wave = lane / LPR;
  const bool unit_ok = unit < s.D / E;
  const int at = unit_ok ? unit * E : 0;
  const int32_t now = a.positions[b];

  // the stream's frames in the order they are visited: the sinks' (their slots are their frames), the window's, the new
  const int sink_frames = now < 0 ? 0 : min(a.sinks, now);
  const int window_first = max(sink_frames, max(now, 0) - a.left);
  const int window_frames = now < 0 ? 0 : now - window_first;
  const int old_frames = sink_frames + window_frames;
  const int total = now < 0 ? 0 : old_frames + s.N;
  // (a window that holds frames begins behind the sinks)
  const uint32_t window_slot = window_frames > 0 ? a.by_ring.mod(static_cast<uint32_t>(window_first - a.sinks)) : 0u;

  const T* kc = static_cast<const T*>(a.k_cache) + b * a.kcs.b + hk * a.kcs.h;
  const T* vc = static_cast<const T*>(a.v_cache) + b * a.vcs.b + hk * a.vcs.h;
  const T* kn = static_cast<const T*>(a.k) + b * a.ks.b + hk * a.ks.h;
  const T* vn = static_cast<const T*>(a.v) + b * a.vs.b + hk * a.vs.h;

  const int x0 = static_cast<int>(split) * a.per_split;
  const int x1 = split + 1 == a.splits ? total : min(total, x0 + a.per_split);

  // where frame number x of the order lies
  auto locate_frame = [&](int x, const T*& kp, const T*& vp) {
    if (x < old_frames) {
      uint32_t slot = static_cast<uint32_t>(x);
      if (x >= sink_frames) {
        slot = window_slot + static_cast<uint32_t>(x - sink_frames);
        if (slot >= static_cast<uint32_t>(a.ring)) slot -= a.ring;
        slot += a.sinks;
      }
      kp = kc + slot * a.kcs.n;
      vp = vc + slot * a.vcs.n;
    } else {
      kp = kn + (x - old_frames) * a.ks.n;
      vp = vn + (x - old_frames) * a.vs.n;
    }
  };
  auto frame_of = [&](int x) { return x < sink_frames ? x : x < old_frames ? window_first + (x - sink_frames) : now + (x - old_frames); };

  u32x4_t kf[kUnroll], vf[kUnroll];
  const int step = KPW * kUnroll * waves;
  auto fetch = [&](int base) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int x = min(base + u * KPW + slot_in_wave, x1 - 1);
      const T *kp, *vp;
      locate_frame(x, kp, vp);
      kf[u] = *(unit_ok ? reinterpret_cast<const u32x4_t*>(kp + at) : &zero_unit);
      vf[u] = *(unit_ok ? reinterpret_cast<const u32x4_t*>(vp + at) : &zero_unit);
    }
  };
  const int first = x0 + wave * KPW * kUnroll;
  if (first < x1) fetch(first);

  u32x4_t q[RT];
  float o[RT][E], m[RT], l[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    m[r] = -kInf;
    l[r] = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) o[r][i] = 0.f;
    q[r] = u32x4_t{0, 0, 0, 0};
    if (r < rows && unit_ok) {
      const int row = r0 + r, n = static_cast<int>(s.by_g.div(static_cast<uint32_t>(row))), head = hk * s.G + (row - n * s.G);
      q[r] = *reinterpret_cast<const u32x4_t*>(static_cast<const T*>(a.q) + b * a.qs.b + n * a.qs.n + head * a.qs.h + at);
    }
  }

  // the new frames go into the caches: once, by the block of the first rows and frames
  if (sub == 0 && now >= 0) {
    const int units = s.D / E;
    for (int i = threadIdx.x; i < s.N * units; i += blockDim.x) {
      const int n = i / units, u = i - n * units;
      const uint32_t frame = static_cast<uint32_t>(now) + static_cast<uint32_t>(n);
      const uint32_t slot = frame < static_cast<uint32_t>(a.sinks)
                                ? frame
                                : a.sinks + a.by_ring.mod(frame - static_cast<uint32_t>(a.sinks));
      *reinterpret_cast<u32x4_t*>(static_cast<T*>(a.k_cache) + b * a.kcs.b + hk * a.kcs.h + slot * a.kcs.n + u * E) =
          *reinterpret_cast<const u32x4_t*>(kn + n * a.ks.n + u * E);
      *reinterpret_cast<u32x4_t*>(static_cast<T*>(a.v_cache) + b * a.vcs.b + hk * a.vcs.h + slot * a.vcs.n + u * E) =
          *reinterpret_cast<const u32x4_t*>(vn + n * a.vs.n + u * E);
    }
  }

  // the query of a row, and where its head's bias begins
  auto query_of = [&](int r) { return static_cast<int>(s.by_g.div(static_cast<uint32_t>(r0 + r))); };
  const int entries = a.bias.distance + 1;  // distances 0 .. back
  auto table_of = [&](int r) { return min(s.G >= RT ? r : r % s.G, min(rows, s.G) - 1) * entries; };
  if constexpr (BIAS) {
    const int heads = min(rows, s.G);
    for (int i = threadIdx.x; i < heads * entries; i += blockDim.x) {
      const int g = i / entries, back = i - g * entries;
      const int head = hk * s.G + (r0 + g) % s.G;
      shared[i] = bias_value(bias_entry(a.bias, dtype_code<T>(), s.H, head, a.bias.bucket_of[a.bias.distance - back]), kLog2e);
    }
    __syncthreads();
  }

  for (int base = first; base < x1; base += step) {
    u32x4_t kg[kUnroll], vg[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      kg[u] = kf[u];
      vg[u] = vf[u];
    }
    if (base + step < x1) fetch(base + step);
    float w[RT][kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
#pragma unroll
      for (int r = 0; r < RT; ++r) w[r][u] = lanes_sum<LPR>(dot<T>(q[r], kg[u], 0.f)) * a.scale_log2;
    }
    // what every row sees whole: sinks, or window frames past those that the later queries have left behind
    const int last = base + KPW * kUnroll;
    const bool whole = last <= min(x1, old_frames) && (base >= sink_frames + s.N - 1 || last <= sink_frames);
    if constexpr (BIAS) {
      if (whole && base >= sink_frames && now - (window_first + (last - 1 - sink_frames)) >= a.bias.distance) {
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const float far = shared[table_of(r) + a.bias.distance];
#pragma unroll
          for (int u = 0; u < kUnroll; ++u) w[r][u] += far;
        }
      } else {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          const int since = now - frame_of(base + u * KPW + slot_in_wave);
#pragma unroll
          for (int r = 0; r < RT; ++r) w[r][u] += shared[table_of(r) + min(max(since + query_of(r), 0), a.bias.distance)];
        }
      }
    }
    if (!whole) {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int x = base + u * KPW + slot_in_wave, frame = frame_of(x);
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const int back = now + query_of(r) - frame;
          w[r][u] = x < x1 && back >= 0 && (back <= a.left || frame < a.sinks) ? w[r][u] : -kInf;
        }
      }
    }
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      float top = w[r][0];
#pragma unroll
      for (int u = 1; u < kUnroll; ++u) top = fmaxf(top, w[r][u]);
      if (top > m[r]) {
        const float alpha = __builtin_amdgcn_exp2f(m[r] - top);
        m[r] = top;
        l[r] *= alpha;
#pragma unroll
        for (int i = 0; i < E; ++i) o[r][i] *= alpha;
      }
      const float ref = m[r] == -kInf ? 0.f : m[r];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        w[r][u] = __builtin_amdgcn_exp2f(w[r][u] - ref);
        l[r] += w[r][u];
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      float x[E];
      unpack<T>(vg[u], x);
#pragma unroll
      for (int r = 0; r < RT; ++r) {
#pragma unroll
        for (int i = 0; i < E; ++i) o[r][i] = fmaf(w[r][u], x[i], o[r][i]);
      }
    }
  }

  // the wave's groups, then the waves
  if constexpr (BIAS) __syncthreads();  // the bias has been read
  const int pitch = s.D + 2;
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    auto sum = [](float x, float y) { return x + y; };
    const float top = groups_join<LPR>(m[r], [](float x, float y) { return fmaxf(x, y); });
    const float f = m[r] == -kInf ? 0.f : __builtin_amdgcn_exp2f(m[r] - top);
    l[r] = groups_join<LPR>(l[r] * f, sum);
#pragma unroll
    for (int i = 0; i < E; ++i) o[r][i] = groups_join<LPR>(o[r][i] * f, sum);
    float* to = shared + (wave * RT + r) * pitch;
    if (slot_in_wave == 0 && unit_ok) {
#pragma unroll
      for (int i = 0; i < E; ++i) to[at + i] = o[r][i];
    }
    if (lane == 0) {
      to[s.D] = top;
      to[s.D + 1] = l[r];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rows * s.D; i += blockDim.x) {
    const int r = i / s.D, d = i - r * s.D;
    float top = -kInf;
    for (int w = 0; w < waves; ++w) top = fmaxf(top, shared[(w * RT + r) * pitch + s.D]);
    float sum = 0.f, x = 0.f;
    for (int w = 0; w < waves; ++w) {
      const float* from = shared + (w * RT + r) * pitch;
      const float f = from[s.D] == -kInf ? 0.f : __builtin_amdgcn_exp2f(from[s.D] - top);
      sum = fmaf(f, from[s.D + 1], sum);
      x = fmaf(f, from[d], x);
    }
    const int row = r0 + r;
    if (a.part_o) {
      const int64_t p = (static_cast<int64_t>(split) * a.grid.pairs + pair) * s.R + row;
      a.part_o[p * s.D + d] = x;
      if (d == 0) {
        a.part_m[p] = top;
        a.part_l[p] = sum;
      }
    } else {
      const int n = static_cast<int>(s.by_g.div(static_cast<uint32_t>(row))), head = hk * s.G + (row - n * s.G);
      static_cast<T*>(a.out)[((static_cast<int64_t>(b) * s.N + n) * s.H + head) * s.D + d] = from_f32<T>(sum == 0.f ? 0.f : x / sum);
    }
  }
}

// Joins the splits: a thread takes a column of a row.
template <typename T>
__global__ __launch_bounds__(256) void local_step_join_kernel(StepArgs a, uint32_t total) {
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  if (i >= total) return;
  const Shape& s = a.s;
  const uint32_t prow = i / static_cast<uint32_t>(s.D), d = i - prow * static_cast<uint32_t>(s.D);
  const int64_t rows = static_cast<int64_t>(a.grid.pairs) * s.R;
  float top = -kInf, sum = 0.f, x = 0.f;
  for (uint32_t k = 0; k < a.splits; ++k) top = fmaxf(top, a.part_m[k * rows + prow]);
  for (uint32_t k = 0; k < a.splits; ++k) {
    const float m = a.part_m[k * rows + prow], f = m == -kInf ? 0.f : __builtin_amdgcn_exp2f(m - top);
    sum = fmaf(f, a.part_l[k * rows + prow], sum);
    x = fmaf(f, a.part_o[(k * rows + prow) * s.D + d], x);
  }
  const uint32_t pair = prow / static_cast<uint32_t>(s.R);
  const int row = static_cast<int>(prow - pair * static_cast<uint32_t>(s.R));
  const int b = static_cast<int>(pair) / s.Hk, hk = static_cast<int>(pair) - b * s.Hk;
  const int n = static_cast<int>(s.by_g.div(static_cast<uint32_t>(row))), head = hk * s.G + (row - n * s.G);
  static_cast<T*>(a.out)[((static_cast<int64_t>(b) * s.N + n) * s.H + head) * s.D + d] = from_f32<T>(sum == 0.f ? 0.f : x / sum);
}

// ---------------------------------------------------------------- host

struct StepPlan {
  int lanes, rows, waves;  // of a K row, of a block, of a block
  int64_t chunks, splits, per_split;
};

// A lane group holds a row of K, a block the rows of a key head up to 8, rounded up to the next instance.  Blocks are split
// over the frames, into shares of four rounds of loads or more, where there are fewer than CUs: one stream, 8 heads of 64 on
// one key head over 60000 frames, 65 us against 1089; with 8 key heads over 4000, 20 us against 30.
StepPlan plan_step(const Shape& s, int64_t left, int64_t sinks, int dtype) {
  StepPlan p;
  const int units = s.D * static_cast<int>(dtype_size(dtype)) / 16;
  p.lanes = units <= 4 ? 4 : units <= 8 ? 8 : units <= 16 ? 16 : 32;
  p.rows = s.R == 1 ? 1 : s.R == 2 ? 2 : s.R <= 4 ? 4 : 8;
  p.chunks = (int64_t{s.R} + p.rows - 1) / p.rows;
  const int64_t frames = left + s.N + sinks, per_wave = 64 / p.lanes * kUnroll;
  p.waves = 4;
  const int64_t blocks = int64_t{s.B} * s.Hk * p.chunks, want = num_cus();
  p.splits = 1;
  if (blocks < want) p.splits = std::max<int64_t>(1, std::min((want + blocks - 1) / blocks, frames / (per_wave * p.waves * 4)));
  p.per_split = (frames + p.splits - 1) / p.splits;
  p.splits = (frames + p.per_split - 1) / p.per_split;
  return p;
}

// The rows of a [batch, positions, heads] tensor: dense, `bytes` each, where they begin and how far apart they lie.
struct RowSet {
  uintptr_t at;
  int64_t size[3], apart[3], bytes;
};

// Whether two sets of rows share a byte: whether a's row - b's row, a sum of strides times indexes, can lie within their
// bytes of each other.  The largest strides' multiples are tried first, and of each only those that the smaller ones can
// still make up for; sets that take more than 2^16 trials count as sharing one.
bool rows_meet(const RowSet& a, const RowSet& b) {
  typedef __int128 wide;
  struct Term { int64_t apart, lo, hi; } terms[6];
  int count = 0;
  auto add = [&](int64_t apart, int64_t lo, int64_t hi) {
    if (apart < 0) { apart = -apart; const int64_t t = lo; lo = -hi; hi = -t; }
    if (apart == 0 || lo == hi) return;
    int i = 0;
    while (i < count && terms[i].apart > apart) ++i;
    if (i < count && terms[i].apart == apart) {
      terms[i].lo += lo;
      terms[i].hi += hi;
      return;
    }
    for (int j = count++; j > i; --j) terms[j] = terms[j - 1];
    terms[i] = {apart, lo, hi};
  };
  for (int i = 0; i < 3; ++i) {
    if (a.size[i] == 0 || b.size[i] == 0) return false;
    add(a.apart[i], 0, a.size[i] - 1);
    add(b.apart[i], 1 - b.size[i], 0);
  }
  wide lo[7], hi[7];  // what the terms from i on can sum up to
  lo[count] = hi[count] = 0;
  for (int i = count; i-- > 0;) {
    lo[i] = lo[i + 1] + static_cast<wide>(terms[i].apart) * terms[i].lo;
    hi[i] = hi[i + 1] + static_cast<wide>(terms[i].apart) * terms[i].hi;
  }
  // the sum has to lie in (from, to), of those before i less what they have
  int64_t x[6], last[6];
  wide from[7], to[7];
  from[0] = static_cast<wide>(b.at) - a.at - a.bytes;
  to[0] = static_cast<wide>(b.at) - a.at + b.bytes;
  auto up = [](wide n, wide d) { return n >= 0 ? (n + d - 1) / d : -(-n / d); };
  auto down = [&](wide n, wide d) { return -up(-n, d); };
  auto open = [&](int i) {
    const wide first = up(from[i] + 1 - hi[i + 1], terms[i].apart), end = down(to[i] - 1 - lo[i + 1], terms[i].apart);
    x[i] = static_cast<int64_t>(first < terms[i].lo ? terms[i].lo : first > terms[i].hi ? terms[i].hi + wide{1} : first);
    last[i] = static_cast<int64_t>(end > terms[i].hi ? terms[i].hi : end < terms[i].lo ? terms[i].lo - wide{1} : end);
  };
  if (from[0] >= hi[0] || to[0] <= lo[0]) return false;
  if (count == 0) return true;
  int i = 0;
  open(0);
  for (int trials = 0; trials < 1 << 16; ++trials) {
    while (x[i] > last[i]) {
      if (--i < 0) return false;
      ++x[i];
    }
    const wide step = static_cast<wide>(terms[i].apart) * x[i];
    from[i + 1] = from[i] - step;
    to[i + 1] = to[i] - step;
    if (i + 1 == count) return true;  // (the last term's multiples are those that fit)
    open(++i);
  }
  return true;
}

size_t step_workspace(const Shape& s, const StepPlan& p) {
  if (p.splits == 1) return 0;
  const size_t rows = static_cast<size_t>(p.splits) * s.B * s.Hk * s.R;
  return align_up(rows * s.D * 4, 256) + 2 * align_up(rows * 4, 256);
}

template <typename T, int LPR, int RT>
int launch_step(const StepArgs& a, const StepPlan& p, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(grid_blocks(a.grid)));
  const size_t results = static_cast<size_t>(p.waves) * RT * (a.s.D + 2) * 4;
  if (a.bias.table) {
    const size_t table = static_cast<size_t>(std::min<int>(RT, a.s.G)) * (a.bias.distance + 1) * 4;
    local_step_kernel<T, LPR, RT, true><<<grid, 64 * p.waves, std::max(results, table), stream>>>(a);
  } else {
    local_step_kernel<T, LPR, RT, false><<<grid, 64 * p.waves, results, stream>>>(a);
  }
  return check_launch("local_step_kernel");
}

template <typename T, int LPR>
int launch_step(const StepArgs& a, const StepPlan& p, hipStream_t stream) {
  switch (p.rows) {
    case 1: return launch_step<T, LPR, 1>(a, p, stream);
    case 2: return launch_step<T, LPR, 2>(a, p, stream);
    case 4: return launch_step<T, LPR, 4>(a, p, stream);
    default: return launch_step<T, LPR, 8>(a, p, stream);
  }
}

template <typename T>
int run_step(const StepArgs& a, const StepPlan& p, hipStream_t stream) {
  int rc = PMSST_OK;
  if constexpr (sizeof(T) == 4) {
    if (p.lanes == 32) rc = launch_step<T, 32>(a, p, stream);
  }
  if (p.lanes == 4) rc = launch_step<T, 4>(a, p, stream);
  if (p.lanes == 8) rc = launch_step<T, 8>(a, p, stream);
  if (p.lanes == 16) rc = launch_step<T, 16>(a, p, stream);
  if (rc != PMSST_OK || p.splits == 1) return rc;
  const uint32_t total = a.grid.pairs * static_cast<uint32_t>(a.s.R) * a.s.D;
  local_step_join_kernel<T><<<dim3((total + 255) / 256), 256, 0, stream>>>(a, total);
  return check_launch("local_step_join_kernel");
}

}  // namespace
}  // namespace pmsst

extern "C" {

size_t pmsst_local_attention_step_workspace_size(int64_t batch, int64_t frames, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                                 int64_t left, int64_t sinks, int dtype) {
  using namespace pmsst::attn;
  LocalArgs l;
  static const int32_t some = 0;
  if (left < 0 || make_local("pmsst_local_attention_step", batch, frames, 0, heads, kv_heads, head_dim, left, 0, sinks, &some,
                             nullptr, 0, nullptr, 0, 0, 1.0, dtype, l) != PMSST_OK ||
      l.s.B == 0 || l.s.N == 0)
    return 0;
  return pmsst::step_workspace(l.s, pmsst::plan_step(l.s, left, sinks, dtype));
}

int pmsst_local_attention_step(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v,
                               const int64_t* v_strides, void* k_cache, const int64_t* k_cache_strides, void* v_cache,
                               const int64_t* v_cache_strides, const int32_t* positions, int64_t left, int64_t sinks,
                               const void* bias, int bias_dtype, const int32_t* bucket_of, int64_t buckets, int64_t max_distance,
                               void* out, int64_t batch, int64_t frames, int64_t slots, int64_t heads, int64_t kv_heads,
                               int64_t head_dim, double scale, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace pmsst;
  using namespace pmsst::attn;
  const char* what = "pmsst_local_attention_step";
  PMSST_REQUIRE(left >= 0, "%s: left must not be negative", what);
  LocalArgs l;
  int rc = make_local(what, batch, frames, slots, heads, kv_heads, head_dim, left, 0, sinks, positions, bias, bias_dtype, bucket_of,
                      buckets, max_distance, scale, dtype, l);
  if (rc != PMSST_OK) return rc;
  if (batch == 0 || frames == 0) return PMSST_OK;
  PMSST_REQUIRE(slots - sinks >= left + frames, "%s: the caches must have sinks + left + frames slots", what);
  PMSST_REQUIRE(q && k && v && k_cache && v_cache && positions && out, "%s: null pointer", what);
  StepArgs a{};
  a.s = l.s;
  a.bias = l.bias;
  if ((rc = make_strides(what, q, q_strides, frames, heads, head_dim, dtype, a.qs)) != PMSST_OK) return rc;
  if ((rc = make_strides(what, k, k_strides, frames, kv_heads, head_dim, dtype, a.ks)) != PMSST_OK) return rc;
  if ((rc = make_strides(what, v, v_strides, frames, kv_heads, head_dim, dtype, a.vs)) != PMSST_OK) return rc;
  if ((rc = make_strides(what, k_cache, k_cache_strides, slots, kv_heads, head_dim, dtype, a.kcs)) != PMSST_OK) return rc;
  if ((rc = make_strides(what, v_cache, v_cache_strides, slots, kv_heads, head_dim, dtype, a.vcs)) != PMSST_OK) return rc;
  const StepPlan p = plan_step(a.s, left, sinks, dtype);
  const size_t need = step_workspace(a.s, p);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return fail(PMSST_EWORKSPACE, "%s: workspace of %zu bytes needed, %zu given", what, need, workspace_bytes);
  PMSST_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0 || need == 0, "%s: workspace must be 16-byte aligned", what);
  PMSST_REQUIRE(k_cache != v_cache, "%s: the caches lie in one place", what);
  // the kernel reads what other blocks of it write, were the caches not apart from each other and from q, k and v
  auto rows_of = [&](const void* at, const Strides& st, int64_t positions_, int64_t heads_) {
    const int64_t size = dtype_size(dtype);
    return RowSet{reinterpret_cast<uintptr_t>(at), {batch, positions_, heads_}, {st.b * size, st.n * size, st.h * size}, head_dim * size};
  };
  const RowSet caches[2] = {rows_of(k_cache, a.kcs, slots, kv_heads), rows_of(v_cache, a.vcs, slots, kv_heads)};
  const RowSet read[3] = {rows_of(q, a.qs, frames, heads), rows_of(k, a.ks, frames, kv_heads), rows_of(v, a.vs, frames, kv_heads)};
  PMSST_REQUIRE(!rows_meet(caches[0], caches[1]), "%s: the caches share memory", what);
  for (const RowSet& cache : caches) {
    for (const RowSet& rows : read) PMSST_REQUIRE(!rows_meet(cache, rows), "%s: q, k or v lies in a cache", what);
  }
  a.q = q;
  a.k = k;
  a.v = v;
  a.k_cache = k_cache;
  a.v_cache = v_cache;
  a.positions = positions;
  a.left = static_cast<int32_t>(left);
  a.sinks = static_cast<int32_t>(sinks);
  a.ring = static_cast<int32_t>(slots - sinks);
  a.by_ring = FastDiv(static_cast<uint32_t>(a.ring));
  a.out = out;
  if (need > 0) {
    const size_t rows = static_cast<size_t>(p.splits) * a.s.B * a.s.Hk * a.s.R;
    char* at = static_cast<char*>(workspace);
    a.part_o = reinterpret_cast<float*>(at);
    at += align_up(rows * a.s.D * 4, 256);
    a.part_m = reinterpret_cast<float*>(at);
    a.part_l = reinterpret_cast<float*>(at + align_up(rows * 4, 256));
  }
  a.splits = static_cast<uint32_t>(p.splits);
  a.per_split = static_cast<int32_t>(p.per_split);
  const int64_t pairs = batch * kv_heads, per = p.chunks * p.splits;
  PMSST_REQUIRE(grid_fits(pairs, per), "%s: too many rows for one call", what);
  a.grid = make_grid(pairs, per);
  a.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case PMSST_F32: return run_step<float>(a, p, st);
    case PMSST_F16: return run_step<f16>(a, p, st);
    default: return run_step<bf16>(a, p, st);
  }
}

}  // extern "C"
