// Rows quantised to int8 with one scale each:
//   scale = max|x| / 127,  q = round(x * (127 / max|x|)), half to even.
// The codes are exactly what these fp32 operations give (one division per
// row, one product per element). A row of zeros has scale 0 and codes 0. A
// row with an infinity or a NaN has that as its scale and codes 0, so every
// product with it is NaN rather than a number. Rows below 2^-64 are scaled by
// 2^64 first, where 127 / max|x| would overflow.
//
// HBM-bound: a row is read once into registers (up to kUnits units of 8
// elements per thread), its maximum is a warp or CTA reduction, and the codes
// are written 8 bytes at a time. Longer rows read the rest a second time.
#include "quantize.cuh"

#include <algorithm>

namespace mtp {
namespace {

constexpr int kUnits = 8;

// A row per warp (CTA false) or per CTA of 256 threads.
template <typename T, bool WIDE, bool CTA>
__global__ void __launch_bounds__(256) quantize_kernel(const T* __restrict__ x, int64_t x_stride, int M, int K,
                                                       int8_t* __restrict__ q, int64_t q_stride,
                                                       float* __restrict__ scale) {
  __shared__ uint32_t red[8];
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t m = CTA ? static_cast<int64_t>(blockIdx.x) : static_cast<int64_t>(blockIdx.x) * 8 + warp;
  if (m >= M) return;
  const int first = (CTA ? threadIdx.x : lane) * 8;
  constexpr int kStep = (CTA ? 256 : 32) * 8;
  const T* row = x + m * x_stride;
  int8_t* out = q + m * q_stride;
  float v[kUnits][8];
  uint32_t most = 0;
#pragma unroll
  for (int u = 0; u < kUnits; ++u)
    if (first + u * kStep < K) load_unit<T, WIDE>(row, first + u * kStep, K, v[u]);
#pragma unroll
  for (int u = 0; u < kUnits; ++u)
    if (first + u * kStep < K) most = max(most, magnitude(v[u]));
  for (int c = first + kUnits * kStep; c < K; c += kStep) {
    float t[8];
    load_unit<T, WIDE>(row, c, K, t);
    most = max(most, magnitude(t));
  }
  most = __reduce_max_sync(kFullMask, most);
  if (CTA) {
    if (lane == 0) red[warp] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) most = max(most, red[w]);
  }
  const RowScale r = row_scale(most);
  if (first == 0) scale[m] = __fdiv_rn(__uint_as_float(most), 127.f);
#pragma unroll
  for (int u = 0; u < kUnits; ++u)
    if (first + u * kStep < K) store_unit<WIDE>(out, first + u * kStep, K, v[u], r);
  for (int c = first + kUnits * kStep; c < K; c += kStep) {
    float t[8];
    load_unit<T, WIDE>(row, c, K, t);
    store_unit<WIDE>(out, c, K, t, r);
  }
}

template <typename T>
int run(const void* x, int64_t x_stride, int M, int K, int8_t* q, int64_t q_stride, float* scale, cudaStream_t st) {
  const bool wide = aligned(x, 16) && x_stride * sizeof(T) % 16 == 0 && K % 8 == 0 && aligned(q, 8) && q_stride % 8 == 0;
  // A warp per row where the row fits its registers and there are rows for
  // every warp; a CTA per row where rows are long or few.
  const bool cta = K > kUnits * 32 * 8 || M < 148 * 8;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(cta ? M : (M + 7) / 8);
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  auto* kernel = wide ? (cta ? quantize_kernel<T, true, true> : quantize_kernel<T, true, false>)
                      : (cta ? quantize_kernel<T, false, true> : quantize_kernel<T, false, false>);
  if (cudaLaunchKernelEx(&cfg, kernel, static_cast<const T*>(x), x_stride, M, K, q, q_stride, scale) != cudaSuccess) {
    cudaGetLastError();
    return MTP_ERR_LAUNCH;
  }
  return MTP_OK;
}

}  // namespace

int launch_quantize_int8(const void* x, int64_t x_stride, int dtype, int M, int K, int8_t* q, int64_t q_stride,
                         float* scale, cudaStream_t st) {
  switch (dtype) {
    case MTP_DTYPE_BF16: return run<__nv_bfloat16>(x, x_stride, M, K, q, q_stride, scale, st);
    case MTP_DTYPE_FP16: return run<__half>(x, x_stride, M, K, q, q_stride, scale, st);
    default: return run<float>(x, x_stride, M, K, q, q_stride, scale, st);
  }
}

}  // namespace mtp
