// Shared by the int8 kernels for few rows and the W8A8 layer.
#pragma once

#include "internal.cuh"

#include <math.h>

namespace mtp {

// D[16 x 8] += A[16 x 32] . B[32 x 8], int8 with int32 sums.
__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <typename T>
__device__ __forceinline__ T out_cast(float v);
template <>
__device__ __forceinline__ float out_cast(float v) { return v; }
template <>
__device__ __forceinline__ __half out_cast(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 out_cast(float v) { return __float2bfloat16_rn(v); }

// One warp's top-k of a token: the operations of router_token (route.cuh), so
// the same ids and weights where the logits are numbers, with each round's
// maximum and its lowest index as warp reductions over integers that order like
// the logits. NaN logits are chosen last. A token with one has NaN weights and,
// unlike there, always ids of experts, so that its result is NaN.
template <int VPT>
__device__ __forceinline__ void route_token(const float* __restrict__ row, int E, int k, int renorm, float* w_out,
                                            int* id_out) {
  const int lane = threadIdx.x & 31;
  float v[VPT], mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    v[i] = lane + 32 * i < E ? row[lane + 32 * i] : -INFINITY;
    mx = fmaxf(mx, v[i]);
  }
  mx = warp_max(mx);
  float ex[VPT], s = 0.f;
  uint32_t key[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    ex[i] = lane + 32 * i < E ? expf(v[i] - mx) : 0.f;
    s += ex[i];
    const uint32_t bits = __float_as_uint(v[i] == 0.f ? 0.f : v[i]);  // -0 ties with 0
    key[i] = lane + 32 * i >= E || v[i] != v[i] ? 0u : bits >> 31 ? ~bits : bits | 0x80000000u;
  }
  s = warp_sum(s);
  float my_w = 0.f, wsum = 0.f;
  int my_id = 0;
  for (int j = 0; j < k; ++j) {
    uint32_t best = 0;
    int at = 0;
#pragma unroll
    for (int i = VPT - 1; i >= 0; --i)
      if (key[i] >= best) best = key[i], at = i;
    const uint32_t top = __reduce_max_sync(kFullMask, best);
    const int id = __reduce_min_sync(kFullMask, best == top ? static_cast<unsigned>(lane + 32 * at) : 0xffffu);
    float p = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (lane + 32 * i == id) {
        key[i] = 0;
        p = ex[i] / s;
      }
    p = __shfl_sync(kFullMask, p, id & 31);
    wsum += p;
    if (lane == j) {
      my_w = p;
      my_id = id;
    }
  }
  if (renorm) my_w = my_w / fmaxf(wsum, 1e-20f);
  *w_out = my_w;
  *id_out = my_id;
}

}  // namespace mtp
