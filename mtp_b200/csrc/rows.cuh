// Shared by the kernels that move and reduce rows: values of a row as fp32 and
// back, and launches.
#pragma once

#include "internal.cuh"

namespace mtp {

// N values of a row as fp32 and back. Conversions to 16 bits go in pairs: one
// at a time they run at 16 a cycle and SM, below what HBM delivers.
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
  for (int n = 0; n < N; ++n) f[n] = __half2float(x.v[n]);
}
template <int N>
__device__ __forceinline__ void to_floats(const Vec<__nv_bfloat16, N>& x, float* f) {
#pragma unroll
  for (int n = 0; n < N; ++n) f[n] = __bfloat162float(x.v[n]);
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
    x.v[n] = __low2half(h);
    x.v[n + 1] = __high2half(h);
  }
  if (N % 2) x.v[N - 1] = __float2half_rn(f[N - 1]);
}
template <int N>
__device__ __forceinline__ void from_floats(const float* f, Vec<__nv_bfloat16, N>& x) {
#pragma unroll
  for (int n = 0; n + 1 < N; n += 2) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(f[n], f[n + 1]);
    x.v[n] = __low2bfloat16(h);
    x.v[n + 1] = __high2bfloat16(h);
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
