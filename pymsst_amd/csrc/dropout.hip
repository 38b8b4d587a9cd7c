// Dropout with a mask that is never stored, alone, behind a GELU, or in front of a residual sum.
//
//   forward   y  = keep * factor * act(x) (+ residual)
//   backward  dx = keep * factor * dy (* act'(x))           (the residual's gradient is dy itself)
//
// keep is drawn by philox.h from (seed, offset, element), so the backward draws it again.  GELU is the
// exact one, x Phi(x), with Phi(-a) = exp(-a^2 / 2) R(a) and R(a) = erfcx(a / sqrt 2) / 2 as t times a
// polynomial in t = 1 / (1 + c a), fitted to the least largest relative error over all a >= 0: the left
// tail keeps its digits.  The derivative Phi(x) + x phi(x) shares the exponential.
//
// A thread takes whole blocks of 8 elements (one Philox block, 16 bytes of a 16-bit type).  Bound: HBM
// (x and y, or dy, x and dx, once each): 63984 x 768 bf16 with a GELU 40 us forward (4.9 TB/s; with p = 0, without the
// random numbers, 38 to 40, so they are hidden) and 44 us backward (6.7 TB/s, x still in the last-level cache); 63984 x 192
// with a residual 12.5 us (5.9 TB/s, likewise).  The GELU in fp32: 75 us forward (5.2 TB/s), 102 backward (5.8).
#include "common.h"
#include "philox.h"

namespace pmsst {
namespace {

constexpr int kDropThreads = 256;

// Blocks of 8 elements a thread loads before it computes: 2, but 1 for the GELU forward, whose arithmetic needs the
// waves that the second block's registers cost (63984 x 768 bf16, one call after the other: 39 us, with 2 42; a residual
// sum 63984 x 192: 12.6 us, with 1 13.4).
template <int ACT, bool SECOND>
constexpr int drop_unroll() { return ACT == PMSST_ACT_GELU && !SECOND ? 1 : 2; }

constexpr int kActNone = PMSST_ACT_NONE, kActGelu = PMSST_ACT_GELU;

// R(a) / t: degree 6, relative error 7.3e-6 (a sixteenth of fp16's half step), c = 0.4; degree 9 for
// fp32, 3.4e-8 (4e-7 as evaluated), c = 0.25.
template <typename T>
__device__ __forceinline__ float gelu_tail(float a, float& gauss) {
  if constexpr (sizeof(T) == 2) {
    const float t = __builtin_amdgcn_rcpf(fmaf(0.4f, a, 1.f));
    float p = fmaf(t, 4.982240569e-02f, -1.396324573e-01f);
    p = fmaf(t, p, 5.944059876e-02f);
    p = fmaf(t, p, 7.720406742e-02f);
    p = fmaf(t, p, 1.339592469e-01f);
    p = fmaf(t, p, 1.596340519e-01f);
    p = fmaf(t, p, 1.595757447e-01f);
    gauss = __builtin_amdgcn_exp2f(a * a * -0.72134752044448f);
    return p * t * gauss;
  } else {
    const float t = 1.f / fmaf(0.25f, a, 1.f);
    float p = fmaf(t, 1.978196911e-02f, -8.087713536e-02f);
    p = fmaf(t, p, 9.559676524e-02f);
    p = fmaf(t, p, -3.171721192e-02f);
    p = fmaf(t, p, 6.369893551e-02f);
    p = fmaf(t, p, 5.897520774e-02f);
    p = fmaf(t, p, 8.160309818e-02f);
    p = fmaf(t, p, 9.346635627e-02f);
    p = fmaf(t, p, 9.973643158e-02f);
    p = fmaf(t, p, 9.973556672e-02f);
    // exp(-a^2 / 2) with the exponent's rounding errors carried: a^2 = h + l, and h times log2(e) / 2
    // (as the sum of two floats)
    const float h = a * a, l = fmaf(a, a, -h);
    const float e = h * -0.721347511f;
    const float r = fmaf(h, -0.721347511f, -e) - fmaf(h, 9.62981e-09f, l * 0.721347511f);
    const float g = __builtin_amdgcn_exp2f(e);
    gauss = fmaf(g, r * 0.693147182f, g);
    return p * t * gauss;
  }
}

// gelu(x), and its derivative where GRAD.  |x| is cut at 40, where the tail is 0 long since, so that no
// infinity meets a zero inside; x itself carries NaN and the infinities into the result.
template <typename T, bool GRAD>
__device__ __forceinline__ float gelu_of(float x) {
  float gauss;
  const float q = gelu_tail<T>(fminf(fabsf(x), 40.f), gauss);
  const float cdf = x < 0.f ? q : 1.f - q;
  if constexpr (GRAD) return fmaf(x * 0.398942280f, gauss, cdf);
  else return x * cdf;
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, int64_t at, float (&o)[8]) {
  if constexpr (sizeof(T) == 2) {
    load_pack<T, 8>(p + at, o);
  } else {
    float a[4], b[4];
    load_pack<T, 4>(p + at, a);
    load_pack<T, 4>(p + at + 4, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o[i] = a[i];
      o[i + 4] = b[i];
    }
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, int64_t at, const float (&o)[8]) {
  if constexpr (sizeof(T) == 2) {
    store_pack<T, 8>(p + at, o);
  } else {
    const float a[4] = {o[0], o[1], o[2], o[3]}, b[4] = {o[4], o[5], o[6], o[7]};
    store_pack<T, 4>(p + at, a);
    store_pack<T, 4>(p + at + 4, b);
  }
}

// v: x (forward) or dy (backward); u: the residual (forward) or x (backward, with an activation).
template <typename T, int ACT, bool SECOND, bool BACK>
__device__ __forceinline__ void drop8(float (&v)[8], const float (&u)[8], uint64_t block, const Dropout& d,
                                      const PhiloxKey& key) {
  if constexpr (ACT == kActGelu) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = BACK ? v[i] * gelu_of<T, true>(u[i]) : gelu_of<T, false>(v[i]);
  }
  if (d.limit != 0) {
    uint32_t w[4];
    philox7(key, block, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = philox_keep(w, i, d.limit) ? v[i] * d.factor : 0.f;
  }
  if constexpr (SECOND && !BACK) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += u[i];
  }
}

// VEC: every pointer is 16-byte aligned.  The last block of 8 may be cut; without VEC (views that start
// between 16 bytes) every block goes element by element.  out may be x or second: a thread reads what it
// writes before it writes it.
template <typename T, int ACT, bool SECOND, bool BACK, bool VEC>
__global__ __launch_bounds__(kDropThreads) void dropout_kernel(const T* x, const T* second, T* out, int64_t n, Dropout d) {
  constexpr int kDropUnroll = drop_unroll<ACT, SECOND>();
  const int64_t g0 = static_cast<int64_t>(blockIdx.x) * (kDropThreads * kDropUnroll) + threadIdx.x;
  const int64_t whole = n / 8;
  PhiloxKey key{};
  if (d.limit != 0) key = philox_key(d.rng);
  float v[kDropUnroll][8], u[kDropUnroll][8];
  if (VEC && g0 + (kDropUnroll - 1) * kDropThreads < whole) {
#pragma unroll
    for (int k = 0; k < kDropUnroll; ++k) {
      const int64_t at = 8 * (g0 + k * kDropThreads);
      load8(x, at, v[k]);
      if constexpr (SECOND) load8(second, at, u[k]);
    }
#pragma unroll
    for (int k = 0; k < kDropUnroll; ++k) {
      drop8<T, ACT, SECOND, BACK>(v[k], u[k], static_cast<uint64_t>(g0 + k * kDropThreads), d, key);
      store8(out, 8 * (g0 + k * kDropThreads), v[k]);
    }
    return;
  }
  for (int k = 0; k < kDropUnroll; ++k) {
    const int64_t g = g0 + k * kDropThreads;
    if (8 * g >= n) return;
    const int count = n - 8 * g < 8 ? static_cast<int>(n - 8 * g) : 8;
    if (VEC && count == 8) {
      load8(x, 8 * g, v[0]);
      if constexpr (SECOND) load8(second, 8 * g, u[0]);
      drop8<T, ACT, SECOND, BACK>(v[0], u[0], static_cast<uint64_t>(g), d, key);
      store8(out, 8 * g, v[0]);
      continue;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[0][i] = i < count ? to_f32(x[8 * g + i]) : 0.f;
      u[0][i] = SECOND && i < count ? to_f32(second[8 * g + i]) : 0.f;
    }
    drop8<T, ACT, SECOND, BACK>(v[0], u[0], static_cast<uint64_t>(g), d, key);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i < count) out[8 * g + i] = from_f32<T>(v[0][i]);
    }
  }
}

template <typename T, int ACT, bool SECOND, bool BACK>
int launch(const void* x, const void* second, void* out, int64_t n, const Dropout& d, hipStream_t stream) {
  const int64_t per_block = int64_t{8} * kDropThreads * drop_unroll<ACT, SECOND>();
  const int64_t blocks = (n + per_block - 1) / per_block;
  PMSST_REQUIRE(blocks * kDropThreads < (int64_t{1} << 32), "dropout: %lld elements are too many for one call",
                static_cast<long long>(n));
  const bool vec = ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(second) |
                     reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  const T* xp = static_cast<const T*>(x);
  const T* sp = static_cast<const T*>(second);
  T* op = static_cast<T*>(out);
  const dim3 grid(static_cast<uint32_t>(blocks));
  if (vec) dropout_kernel<T, ACT, SECOND, BACK, true><<<grid, kDropThreads, 0, stream>>>(xp, sp, op, n, d);
  else dropout_kernel<T, ACT, SECOND, BACK, false><<<grid, kDropThreads, 0, stream>>>(xp, sp, op, n, d);
  return check_launch("dropout_kernel");
}

template <typename T>
int route(const void* x, const void* second, void* out, int64_t n, const Dropout& d, bool gelu, bool back,
          hipStream_t stream) {
  if (back) {
    if (gelu) return launch<T, kActGelu, true, true>(x, second, out, n, d, stream);
    return launch<T, kActNone, false, true>(x, nullptr, out, n, d, stream);
  }
  if (gelu && second) return launch<T, kActGelu, true, false>(x, second, out, n, d, stream);
  if (gelu) return launch<T, kActGelu, false, false>(x, nullptr, out, n, d, stream);
  if (second) return launch<T, kActNone, true, false>(x, second, out, n, d, stream);
  return launch<T, kActNone, false, false>(x, nullptr, out, n, d, stream);
}

int run(const char* what, const void* x, const void* second, void* out, int64_t n, double p, const int64_t* rng,
        int activation, int dtype, bool back, void* stream) {
  if (!dtype_ok(dtype)) return fail(PMSST_EDTYPE, "%s: unsupported dtype %d", what, dtype);
  PMSST_REQUIRE(n >= 0, "%s: negative element count", what);
  PMSST_REQUIRE(p >= 0.0 && p < 1.0, "%s: the probability must lie in [0, 1)", what);
  PMSST_REQUIRE(activation == PMSST_ACT_NONE || activation == PMSST_ACT_GELU, "%s: unsupported activation %d", what,
                activation);
  if (n == 0) return PMSST_OK;
  const bool gelu = activation == PMSST_ACT_GELU;
  PMSST_REQUIRE(x && out && (!back || !gelu || second), "%s: null pointer", what);
  const Dropout d = make_dropout(p, rng);
  PMSST_REQUIRE(rng || d.limit == 0, "%s: null pointer (rng)", what);
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case PMSST_F32: return route<float>(x, second, out, n, d, gelu, back, s);
    case PMSST_F16: return route<f16>(x, second, out, n, d, gelu, back, s);
    default: return route<bf16>(x, second, out, n, d, gelu, back, s);
  }
}

}  // namespace
}  // namespace pmsst

extern "C" {

int pmsst_dropout_forward(const void* x, const void* residual, void* out, int64_t n, double p, const int64_t* rng,
                          int activation, int dtype, void* stream) {
  return pmsst::run("pmsst_dropout_forward", x, residual, out, n, p, rng, activation, dtype, false, stream);
}

int pmsst_dropout_backward(const void* grad_out, const void* x, void* grad_x, int64_t n, double p, const int64_t* rng,
                           int activation, int dtype, void* stream) {
  return pmsst::run("pmsst_dropout_backward", grad_out, x, grad_x, n, p, rng, activation, dtype, true, stream);
}

}  // extern "C"
