// Pieces that the backward kernels of the cross attention and of the local attention share
// (cross_attention_bwd.hip, local_attention_bwd.hip): the bounds that fp16's powers of two come from.
#pragma once

#include "attention.h"

namespace pmsst {
namespace attn {

constexpr int kParts = 16;
constexpr uint32_t kBoundPairs = 1u << 18;  // pairs of a grid row of attn_bound_kernel: 2^30 work-items

// What stands for dO past the last row: these rows have no weight, but 0 times the last one's infinities is none.
static __device__ const u32x4_t zero_row[32] = {};

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

// ---------------------------------------------------------------- fp16 bounds

// Args: the backward's arguments (q, k, v, dout with their strides, the key mask, the shape, vmax and l1).
template <typename T, typename Args>
__global__ __launch_bounds__(256) void attn_bound_kernel(Args a) {
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

// Its launch, over `pairs` (batch row, key head).
template <typename T, typename Args>
int launch_bound(const Args& a, int64_t pairs, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(std::min<int64_t>(pairs, kBoundPairs) * kParts),
                  static_cast<uint32_t>((pairs + kBoundPairs - 1) / kBoundPairs));
  attn_bound_kernel<T><<<grid, 256, 0, stream>>>(a);
  return check_launch("attn_bound_kernel");
}

}  // namespace attn
}  // namespace pmsst
