// Shared by the kernels that move and reduce rows: values of a row as fp32 and
// back, and launches.
#pragma once

#include "internal.cuh"

#include <string.h>

namespace mtp {

// N values of a row as fp32 and back, rounded to nearest even. Two 16-bit values
// at a time: that is one instruction a value on the way in and one for both on
// the way out (one value at a time, the conversions run at 16 a cycle and SM,
// below what HBM delivers).
template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};
template <int N>
__device__ __forceinline__ void to_floats(const Vec<float, N>& x, float* f) {
#pragma unroll
  for (int n = 0; n < N; ++n) f[n] = x.v[n];
}
template <int N>
__device__ __forceinline__ void to_floats(const Vec<__half, N>& x, float* f) {
#pragma unroll
  for (int n = 0; n + 1 < N; n += 2) {
    const float2 v = __half22float2(__halves2half2(x.v[n], x.v[n + 1]));
    f[n] = v.x;
    f[n + 1] = v.y;
  }
  if (N % 2) f[N - 1] = __half2float(x.v[N - 1]);
}
template <int N>
__device__ __forceinline__ void to_floats(const Vec<__nv_bfloat16, N>& x, float* f) {
#pragma unroll
  for (int n = 0; n + 1 < N; n += 2) {
    const __nv_bfloat162 h = __halves2bfloat162(x.v[n], x.v[n + 1]);
    uint32_t bits;
    memcpy(&bits, &h, 4);
    f[n] = __uint_as_float(bits << 16);
    f[n + 1] = __uint_as_float(bits & 0xffff0000u);
  }
  if (N % 2) f[N - 1] = __bfloat162float(x.v[N - 1]);
}
template <int N>
__device__ __forceinline__ void from_floats(const float* f, Vec<float, N>& x) {
#pragma unroll
  for (int n = 0; n < N; ++n) x.v[n] = f[n];
}
template <int N>
__device__ __forceinline__ void from_floats(const float* f, Vec<__half, N>& x) {
#pragma unroll
  for (int n = 0; n + 1 < N; n += 2) {
    const __half2 h = __floats2half2_rn(f[n], f[n + 1]);
    memcpy(&x.v[n], &h, 4);
  }
  if (N % 2) x.v[N - 1] = __float2half_rn(f[N - 1]);
}
template <int N>
__device__ __forceinline__ void from_floats(const float* f, Vec<__nv_bfloat16, N>& x) {
#pragma unroll
  for (int n = 0; n + 1 < N; n += 2) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(f[n], f[n + 1]);
    memcpy(&x.v[n], &h, 4);
  }
  if (N % 2) x.v[N - 1] = __float2bfloat16_rn(f[N - 1]);
}

// Threads of a row (a power of two in [least, 256]) and rows of a CTA.
inline dim3 row_block(int64_t vectors, int least) {
  int x = least;
  while (x < vectors && x < 256) x *= 2;
  return dim3(x, 256 / x);
}

template <typename F, typename... A>
int launch(F* kernel, dim3 grid, dim3 block, size_t smem, cudaStream_t st, A... args) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, args...) != cudaSuccess) {
    cudaGetLastError();
    return MTP_ERR_LAUNCH;
  }
  return MTP_OK;
}

}  // namespace mtp
