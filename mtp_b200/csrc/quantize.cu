// Rows quantised to int8 with one scale each:
//   scale = max|x| / 127,  q = round(x * (127 / max|x|)), half to even.
// The codes are exactly what these fp32 operations give (one division per
// row, one product per element). A row of zeros has scale 0 and codes 0. A
// row with an infinity or a NaN has that as its scale and codes 0, so every
// product with it is NaN rather than a number. Rows below 2^-64 are scaled by
// 2^64 first, where 127 / max|x| would overflow.
//
// HBM-bound: a row is read once into registers (as it is stored, up to kUnits
// pieces of 16 bytes a thread), its maximum is a warp or CTA reduction, and the
// codes are written 8 (fp32: 4) bytes a thread. Longer rows read the rest a
// second time. 8192 x 2048 bf16 took 18.7 us with the row kept as fp32 (fewer
// warps resident) and a conversion per code.
#include "quantize.cuh"
#include "w8a8_common.cuh"

#include <algorithm>
#include <type_traits>

namespace mtp {
namespace {

constexpr int kUnits = 8;

// N elements in 16 bytes, as they are stored.
template <typename T>
struct Piece {
  static constexpr int N = 16 / sizeof(T);
  uint4 raw;
  __device__ __forceinline__ void load(const T* p) { raw = __ldcs(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void floats(float* v) const {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (sizeof(T) == 4) {
        v[i] = __uint_as_float(w[i]);
      } else if (std::is_same<T, __half>::value) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      } else {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  }
  __device__ __forceinline__ uint32_t magnitude() const {
    float v[N];
    floats(v);
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    return m;
  }
  __device__ __forceinline__ void store(int8_t* q, RowScale r) const {
    float v[N];
    floats(v);
    uint32_t w[2];
    codes_of<N>(v, r, w);
    if (N == 8)
      *reinterpret_cast<uint2*>(q) = make_uint2(w[0], w[1]);
    else
      *reinterpret_cast<uint32_t*>(q) = w[0];
  }
};

__device__ __forceinline__ uint32_t cta_max(uint32_t most, uint32_t* red) {
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) most = max(most, red[w]);
  return most;
}

// WPR warps a row, 8 / WPR rows a CTA of 256 threads; rows and codes aligned.
template <typename T, int WPR>
__device__ __forceinline__ void quantize_rows(int block, const T* __restrict__ x, int64_t x_stride, int M, int K,
                                              int8_t* __restrict__ q, int64_t q_stride, float* __restrict__ scale) {
  using P = Piece<T>;
  __shared__ uint32_t red[8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t m = static_cast<int64_t>(block) * (8 / WPR) + warp / WPR;
  const int k = m < M ? K : 0;
  const int first = (warp % WPR * 32 + lane) * P::N;
  constexpr int kStep = WPR * 32 * P::N;
  const T* row = x + m * x_stride;
  int8_t* out = q + m * q_stride;
  P v[kUnits];
  uint32_t most = 0;
#pragma unroll
  for (int u = 0; u < kUnits; ++u)
    if (first + u * kStep < k) v[u].load(row + first + u * kStep);
#pragma unroll
  for (int u = 0; u < kUnits; ++u)
    if (first + u * kStep < k) most = max(most, v[u].magnitude());
  P t;
  for (int c = first + kUnits * kStep; c < k; c += kStep) {
    t.load(row + c);
    most = max(most, t.magnitude());
  }
  most = __reduce_max_sync(kFullMask, most);
  if (WPR > 1) {
    if (lane == 0) red[warp] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WPR; ++w) most = max(most, red[warp / WPR * WPR + w]);
  }
  const RowScale r = row_scale(most);
  if (first == 0 && m < M) scale[m] = __fdiv_rn(__uint_as_float(most), 127.f);
#pragma unroll
  for (int u = 0; u < kUnits; ++u)
    if (first + u * kStep < k) v[u].store(out + first + u * kStep, r);
  for (int c = first + kUnits * kStep; c < k; c += kStep) {
    t.load(row + c);
    t.store(out + c, r);
  }
}

template <typename T, int WPR>
__global__ void __launch_bounds__(256) quantize_kernel(const T* __restrict__ x, int64_t x_stride, int M, int K,
                                                       int8_t* __restrict__ q, int64_t q_stride,
                                                       float* __restrict__ scale) {
  pdl_launch_dependents();
  pdl_wait();
  quantize_rows<T, WPR>(blockIdx.x, x, x_stride, M, K, q, q_stride, scale);
}

// Any alignment: a row per CTA, read twice.
template <typename T>
__device__ __forceinline__ void quantize_any(int64_t m, const T* __restrict__ x, int64_t x_stride, int K,
                                             int8_t* __restrict__ q, int64_t q_stride, float* __restrict__ scale) {
  __shared__ uint32_t red[8];
  const T* row = x + m * x_stride;
  uint32_t most = 0;
  for (int c = threadIdx.x; c < K; c += 256) most = max(most, __float_as_uint(one(row + c)) & 0x7fffffffu);
  most = cta_max(__reduce_max_sync(kFullMask, most), red);
  const RowScale r = row_scale(most);
  if (threadIdx.x == 0) scale[m] = __fdiv_rn(__uint_as_float(most), 127.f);
  for (int c = threadIdx.x; c < K; c += 256) {
    float v[4] = {one(row + c), 0.f, 0.f, 0.f};
    uint32_t w;
    codes_of<4>(v, r, &w);
    q[m * q_stride + c] = static_cast<int8_t>(w);
  }
}

// The rows of a layer quantised and its tokens routed, which do not depend on
// each other, in one launch: the first CTAs route 8 tokens each (a warp a
// token), the others quantise (WPR 0: rows of any alignment).
template <typename T, int WPR, int VPT>
__global__ void __launch_bounds__(256) route_quantize_kernel(const T* __restrict__ x, int M, int K,
                                                             int8_t* __restrict__ q, int64_t q_stride,
                                                             float* __restrict__ scale, const float* __restrict__ logits,
                                                             int E, int k, int renorm, float* __restrict__ weights,
                                                             int32_t* __restrict__ ids) {
  pdl_launch_dependents();
  pdl_wait();
  const int routing = (M + 7) / 8;
  if (static_cast<int>(blockIdx.x) >= routing) {
    if constexpr (WPR == 0)
      quantize_any(blockIdx.x - routing, x, K, K, q, q_stride, scale);
    else
      quantize_rows<T, WPR>(blockIdx.x - routing, x, K, M, K, q, q_stride, scale);
    return;
  }
  const int t = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (t >= M) return;
  float w;
  int id;
  route_token<VPT>(logits + static_cast<int64_t>(t) * E, E, k, renorm, &w, &id);
  if (lane < k) {
    weights[static_cast<int64_t>(t) * k + lane] = w;
    ids[static_cast<int64_t>(t) * k + lane] = id;
  }
}

template <typename T>
__global__ void __launch_bounds__(256) quantize_any_kernel(const T* __restrict__ x, int64_t x_stride, int K,
                                                           int8_t* __restrict__ q, int64_t q_stride,
                                                           float* __restrict__ scale) {
  pdl_launch_dependents();
  pdl_wait();
  quantize_any(blockIdx.x, x, x_stride, K, q, q_stride, scale);
}

// Padded copies by the warps of `blocks` CTAs, 16 bytes a lane: five aligned
// words that hold them wherever the row starts (none past the last row's end,
// none without a byte of the row), shifted into place.
__device__ __forceinline__ void pad_rows(const PadJob& j, int block, int blocks) {
  const int lane = threadIdx.x & 31;
  for (int64_t r = static_cast<int64_t>(block) * 8 + (threadIdx.x >> 5); r < j.rows;
       r += static_cast<int64_t>(blocks) * 8) {
    const int8_t* row = j.src + r * j.stride;
    for (int c = lane * 16; c < j.dst_stride; c += 512) {
      const uintptr_t at = reinterpret_cast<uintptr_t>(row + c);
      const uint32_t* word = reinterpret_cast<const uint32_t*>(at & ~static_cast<uintptr_t>(3));
      const uint32_t* end = reinterpret_cast<const uint32_t*>(row + j.K);
      const int shift = 8 * static_cast<int>(at & 3);
      uint32_t w[5], o[4];
#pragma unroll
      for (int i = 0; i < 5; ++i) w[i] = c < j.K && word + i < end && (i < 4 || shift) ? word[i] : 0u;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        o[i] = __funnelshift_r(w[i], w[i + 1], shift);
        const int left = j.K - c - 4 * i;  // bytes of the row in this word
        if (left < 4) o[i] = left > 0 ? o[i] & (0xffffffffu >> (32 - 8 * left)) : 0u;
      }
      *reinterpret_cast<uint4*>(j.dst + r * j.dst_stride + c) = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
}

__global__ void __launch_bounds__(256) pad_rows_kernel(const __grid_constant__ PadJob a, int blocks_a,
                                                       const __grid_constant__ PadJob b) {
  pdl_launch_dependents();
  pdl_wait();
  if (static_cast<int>(blockIdx.x) < blocks_a)
    pad_rows(a, blockIdx.x, blocks_a);
  else
    pad_rows(b, blockIdx.x - blocks_a, gridDim.x - blocks_a);
}

// The first M CTAs quantise a row each, the others pad.
template <typename T>
__global__ void __launch_bounds__(256) quantize_and_pad_kernel(const T* __restrict__ x, int64_t x_stride, int M, int K,
                                                               int8_t* __restrict__ q, int64_t q_stride,
                                                               float* __restrict__ scale, int wide,
                                                               const __grid_constant__ PadJob pad) {
  pdl_launch_dependents();
  pdl_wait();
  if (static_cast<int>(blockIdx.x) >= M)
    pad_rows(pad, blockIdx.x - M, gridDim.x - M);
  else if (wide)
    quantize_rows<T, 8>(blockIdx.x, x, x_stride, M, K, q, q_stride, scale);
  else
    quantize_any(blockIdx.x, x, x_stride, K, q, q_stride, scale);
}

int pad_blocks(const PadJob& j) { return static_cast<int>(std::min<int64_t>((j.rows + 7) / 8, 148 * 8)); }

template <typename F, typename... A>
int launch(F* kernel, int64_t grid, cudaStream_t st, A... args) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, args...) != cudaSuccess) {
    cudaGetLastError();
    return MTP_ERR_LAUNCH;
  }
  return MTP_OK;
}

template <typename T>
bool wide_rows(const void* x, int64_t x_stride, int K, const void* q, int64_t q_stride) {
  constexpr int N = Piece<T>::N;
  return aligned(x, 16) && x_stride * sizeof(T) % 16 == 0 && K % N == 0 && aligned(q, N) && q_stride % N == 0;
}

// Warps of a row: as few as hold it in their registers, so that a warp has as
// many loads in flight as it can, but a CTA for each row where rows are few.
template <typename T>
int warps_per_row(int M, int K) {
  int wpr = M < 148 * 8 ? 8 : 1;
  while (wpr < 8 && K > kUnits * 32 * Piece<T>::N * wpr) wpr *= 2;
  return wpr;
}

template <typename T, int WPR, int VPT>
int run_routed(const void* x, int M, int K, int8_t* q, int64_t q_stride, float* scale, const float* logits, int E, int k,
               int renorm, float* weights, int32_t* ids, cudaStream_t st) {
  const int64_t rows = WPR ? (static_cast<int64_t>(M) * WPR + 7) / 8 : M;
  return launch(route_quantize_kernel<T, WPR, VPT>, (M + 7) / 8 + rows, st, static_cast<const T*>(x), M, K, q,
                q_stride, scale, logits, E, k, renorm, weights, ids);
}

template <typename T, int WPR>
int by_experts(const void* x, int M, int K, int8_t* q, int64_t q_stride, float* scale, const float* logits, int E, int k,
               int renorm, float* weights, int32_t* ids, cudaStream_t st) {
  return E <= 256 ? run_routed<T, WPR, 8>(x, M, K, q, q_stride, scale, logits, E, k, renorm, weights, ids, st)
                  : run_routed<T, WPR, 32>(x, M, K, q, q_stride, scale, logits, E, k, renorm, weights, ids, st);
}

template <typename T>
int route_and_quantize(const void* x, int M, int K, int8_t* q, int64_t q_stride, float* scale,
                       const float* logits, int E, int k, int renorm, float* weights, int32_t* ids, cudaStream_t st) {
  if (!wide_rows<T>(x, K, K, q, q_stride))
    return by_experts<T, 0>(x, M, K, q, q_stride, scale, logits, E, k, renorm, weights, ids, st);
  return warps_per_row<T>(M, K) == 1
             ? by_experts<T, 1>(x, M, K, q, q_stride, scale, logits, E, k, renorm, weights, ids, st)
             : by_experts<T, 8>(x, M, K, q, q_stride, scale, logits, E, k, renorm, weights, ids, st);
}

template <typename T>
int run(const void* x, int64_t x_stride, int M, int K, int8_t* q, int64_t q_stride, float* scale, cudaStream_t st) {
  const bool wide = wide_rows<T>(x, x_stride, K, q, q_stride);
  const int wpr = warps_per_row<T>(M, K);
  const T* p = static_cast<const T*>(x);
  if (!wide) return launch(quantize_any_kernel<T>, M, st, p, x_stride, K, q, q_stride, scale);
  auto* kernel = wpr == 1   ? quantize_kernel<T, 1>
                 : wpr == 2 ? quantize_kernel<T, 2>
                 : wpr == 4 ? quantize_kernel<T, 4>
                            : quantize_kernel<T, 8>;
  return launch(kernel, (static_cast<int64_t>(M) * wpr + 7) / 8, st, p, x_stride, M, K, q, q_stride, scale);
}

template <typename T>
int run_padded(const void* x, int64_t x_stride, int M, int K, int8_t* q, int64_t q_stride, float* scale,
               const PadJob& pad, cudaStream_t st) {
  return launch(quantize_and_pad_kernel<T>, static_cast<int64_t>(M) + pad_blocks(pad), st, static_cast<const T*>(x),
                x_stride, M, K, q, q_stride, scale, wide_rows<T>(x, x_stride, K, q, q_stride) ? 1 : 0, pad);
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

int launch_route_quantize(const void* x, int dtype, int M, int K, int8_t* q, int64_t q_stride, float* scale,
                          const float* logits, int E, int k, int renorm, float* weights, int32_t* ids,
                          cudaStream_t st) {
  switch (dtype) {
    case MTP_DTYPE_BF16:
      return route_and_quantize<__nv_bfloat16>(x, M, K, q, q_stride, scale, logits, E, k, renorm, weights, ids, st);
    case MTP_DTYPE_FP16:
      return route_and_quantize<__half>(x, M, K, q, q_stride, scale, logits, E, k, renorm, weights, ids, st);
    default:
      return route_and_quantize<float>(x, M, K, q, q_stride, scale, logits, E, k, renorm, weights, ids, st);
  }
}

int launch_pad_rows(const PadJob& a, const PadJob& b, cudaStream_t st) {
  const int blocks = pad_blocks(a) + pad_blocks(b);
  return blocks ? launch(pad_rows_kernel, blocks, st, a, pad_blocks(a), b) : MTP_OK;
}

int launch_quantize_and_pad(const void* x, int64_t x_stride, int dtype, int M, int K, int8_t* q, int64_t q_stride,
                            float* scale, const PadJob& pad, cudaStream_t st) {
  // one launch where there are few rows; many are worth their own kernel
  if (!pad.rows || M >= 148 * 8) {
    const int rc = launch_pad_rows(pad, PadJob{}, st);
    return rc != MTP_OK ? rc : launch_quantize_int8(x, x_stride, dtype, M, K, q, q_stride, scale, st);
  }
  switch (dtype) {
    case MTP_DTYPE_BF16: return run_padded<__nv_bfloat16>(x, x_stride, M, K, q, q_stride, scale, pad, st);
    case MTP_DTYPE_FP16: return run_padded<__half>(x, x_stride, M, K, q, q_stride, scale, pad, st);
    default: return run_padded<float>(x, x_stride, M, K, q, q_stride, scale, pad, st);
  }
}

}  // namespace mtp
