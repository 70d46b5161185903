// Layer norm and its gradients.
//
// forward:  mean and variance of a row's H values (the variance from the
//           centred values, so an offset costs no digits), rstd = 1 / sqrt(var +
//           eps), y = (x - mean) rstd w + b.
// gradient: with xhat = (x - mean) rstd and wg = w g,
//           dx = rstd (wg - mean(wg) - xhat mean(wg xhat)),
//           dw = sum over the rows of g xhat, db = sum of g.
//
// All sums in fp32 in a fixed order; results are rounded once.
#include "rows.cuh"

#include <math.h>

#include <algorithm>

namespace mtp {
namespace {

constexpr int kThreads = 256;

// The sums of two values over the CTA, for all threads.
__device__ __forceinline__ float2 block_sum(float2 v, float2* tmp) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  v.x = warp_sum(v.x);
  v.y = warp_sum(v.y);
  __syncthreads();  // tmp of the sum before is read
  if (lane == 0) tmp[warp] = v;
  __syncthreads();
  v = tmp[0];
  for (int w = 1; w < warps; ++w) {
    v.x += tmp[w].x;
    v.y += tmp[w].y;
  }
  return v;
}

template <typename T>
__device__ __forceinline__ float value(const void* p, int64_t i) {
  Vec<T, 1> v = static_cast<const Vec<T, 1>*>(p)[i];
  float f;
  to_floats(v, &f);
  return f;
}
template <typename T>
__device__ __forceinline__ void store(void* p, int64_t i, float f) {
  Vec<T, 1> v;
  from_floats(&f, v);
  static_cast<Vec<T, 1>*>(p)[i] = v;
}

template <typename T, typename P>
__global__ void __launch_bounds__(kThreads) norm_kernel(const NormArgs a) {
  __shared__ float2 tmp[kThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  for (int t = blockIdx.x; t < a.M; t += gridDim.x) {
    const int64_t x = t * a.stride, y = static_cast<int64_t>(t) * a.H;
    float s = 0.f;
    for (int c = threadIdx.x; c < a.H; c += kThreads) s += value<T>(a.x, x + c);
    const float mean = block_sum(make_float2(s, 0.f), tmp).x / a.H;
    s = 0.f;
    for (int c = threadIdx.x; c < a.H; c += kThreads) {
      const float d = value<T>(a.x, x + c) - mean;
      s = fmaf(d, d, s);
    }
    const float rstd = 1.f / sqrtf(block_sum(make_float2(s, 0.f), tmp).x / a.H + a.eps);
    for (int c = threadIdx.x; c < a.H; c += kThreads) {
      const float w = a.weight ? value<P>(a.weight, c) : 1.f, b = a.bias ? value<P>(a.bias, c) : 0.f;
      store<T>(a.y, y + c, fmaf((value<T>(a.x, x + c) - mean) * rstd, w, b));
    }
    if (a.stats && threadIdx.x == 0) {
      a.stats[2ll * t] = mean;
      a.stats[2ll * t + 1] = rstd;
    }
  }
}

template <typename T, typename P>
__global__ void __launch_bounds__(kThreads) norm_rows_backward_kernel(const NormArgs a) {
  __shared__ float2 tmp[kThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  for (int t = blockIdx.x; t < a.M; t += gridDim.x) {
    const int64_t x = t * a.stride, y = static_cast<int64_t>(t) * a.H;
    const float mean = a.stats[2ll * t], rstd = a.stats[2ll * t + 1];
    float2 s = {0.f, 0.f};
    for (int c = threadIdx.x; c < a.H; c += kThreads) {
      const float wg = (a.weight ? value<P>(a.weight, c) : 1.f) * value<T>(a.grad, y + c);
      s.x += wg;
      s.y = fmaf(wg, (value<T>(a.x, x + c) - mean) * rstd, s.y);
    }
    s = block_sum(s, tmp);
    s.x /= a.H;
    s.y /= a.H;
    for (int c = threadIdx.x; c < a.H; c += kThreads) {
      const float wg = (a.weight ? value<P>(a.weight, c) : 1.f) * value<T>(a.grad, y + c);
      const float xhat = (value<T>(a.x, x + c) - mean) * rstd;
      store<T>(a.grad_x, y + c, rstd * (wg - s.x - xhat * s.y));
    }
  }
}

// CTA (x, p): kThreads columns, the rows p, p + gridDim.y, ...
template <typename T>
__global__ void __launch_bounds__(kThreads) norm_columns_kernel(const NormArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= a.H) return;
  float dw = 0.f, db = 0.f;
  for (int t = blockIdx.y; t < a.M; t += gridDim.y) {
    const float g = value<T>(a.grad, static_cast<int64_t>(t) * a.H + c);
    dw = fmaf(g, (value<T>(a.x, t * a.stride + c) - a.stats[2ll * t]) * a.stats[2ll * t + 1], dw);
    db += g;
  }
  float* part = a.parts + 2ll * blockIdx.y * a.H;
  part[c] = dw;
  part[a.H + c] = db;
}

// The parts' sums: 32 columns a CTA, a warp for every eighth part.
template <typename P>
__global__ void __launch_bounds__(kThreads) norm_finish_kernel(const NormArgs a, int parts) {
  __shared__ float2 tmp[8][32];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float2 s = {0.f, 0.f};
  if (c < a.H)
#pragma unroll 4
    for (int p = warp; p < parts; p += 8) {
      s.x += a.parts[2ll * p * a.H + c];
      s.y += a.parts[(2ll * p + 1) * a.H + c];
    }
  tmp[warp][lane] = s;
  __syncthreads();
  if (warp > 0 || c >= a.H) return;
  for (int w = 1; w < 8; ++w) {
    s.x += tmp[w][lane].x;
    s.y += tmp[w][lane].y;
  }
  if (a.grad_weight) store<P>(a.grad_weight, c, s.x);
  if (a.grad_bias) store<P>(a.grad_bias, c, s.y);
}

template <typename T, typename P>
int run(const NormArgs& a, bool backward, cudaStream_t st) {
  if (!backward)
    return a.M ? launch(norm_kernel<T, P>, dim3(std::min(a.M, 1 << 20)), dim3(kThreads), 0, st, a) : MTP_OK;
  if (a.grad_x && a.M) {
    const int rc = launch(norm_rows_backward_kernel<T, P>, dim3(std::min(a.M, 1 << 20)), dim3(kThreads), 0, st, a);
    if (rc != MTP_OK) return rc;
  }
  if (!a.grad_weight && !a.grad_bias) return MTP_OK;
  const int parts = static_cast<int>(layer_norm_parts(a.M, a.H));
  if (parts) {
    const int rc = launch(norm_columns_kernel<T>, dim3((a.H + kThreads - 1) / kThreads, parts), dim3(kThreads), 0, st, a);
    if (rc != MTP_OK) return rc;
  }
  return launch(norm_finish_kernel<P>, dim3((a.H + 31) / 32), dim3(kThreads), 0, st, a, parts);
}

template <typename T>
int run(const NormArgs& a, bool backward, cudaStream_t st) {
  return a.param_fp32 ? run<T, float>(a, backward, st) : run<T, T>(a, backward, st);
}

int run(const NormArgs& a, int dtype, bool backward, cudaStream_t st) {
  switch (dtype) {
    case MTP_DTYPE_BF16: return run<__nv_bfloat16>(a, backward, st);
    case MTP_DTYPE_FP16: return run<__half>(a, backward, st);
    default: return run<float, float>(a, backward, st);
  }
}

}  // namespace

int64_t layer_norm_parts(int M, int H) { return std::min(M, 64); }
int launch_layer_norm(const NormArgs& a, int dtype, cudaStream_t st) { return run(a, dtype, false, st); }
int launch_layer_norm_backward(const NormArgs& a, int dtype, cudaStream_t st) { return run(a, dtype, true, st); }

}  // namespace mtp
