// int8 products of at most 8 rows with one weight matrix (decode): every weight
// is used a few times at most, so the work is to stream the weights and the
// latency of a call. A tensor-core tile with its ring, barriers and tensor
// memory takes 4 us before its first result; here the weights go straight from
// global memory into the registers of mma.m16n8k32 (16 channels x 32 of K
// against 8 rows): each lane loads 16 bytes of K of two channels and of one row,
// and since both operands are cut the same way, which of the product's 32
// positions of K a byte takes does not matter.
//
// A unit is 16 output channels. ks warps of a CTA share a unit, each taking every
// ks-th 128 bytes of K; their int32 sums meet in shared memory (exact, so the
// order does not matter). All of a warp's loads of a round (kSteps x 128 of K)
// are in flight together, and the next unit's are issued before the last one's
// results are written.
//
// QUANT: the rows come as bf16, fp16 or fp32 and every CTA quantises them itself
// into shared memory, while its first weights are on their way: a second launch
// for so few rows costs more than quantising them again in every CTA. One row of
// 2048 to 1024 channels takes 3.8 us, the two kernels of the tile path 8.0; both
// are latency (2 MB of weights are 0.3 us of HBM). 8192 x 8192 at one row 17 us,
// 3.9 TB/s.
#include "quantize.cuh"
#include "w8a8_common.cuh"

#include <algorithm>

namespace mtp {
namespace {

constexpr int kSWarps = 8;
constexpr int kSThreads = kSWarps * 32;
constexpr int kSRows = 8;
constexpr int kSteps = 2;              // 128 bytes of K in flight per round and warp
constexpr int kSRowBytes = 48 * 1024;  // QUANT: most bytes of quantised rows

struct StreamArgs {
  const int8_t* a;      // codes, rows a_stride apart (not QUANT)
  int64_t a_stride;
  const int8_t* b;      // weights, rows b_stride apart
  int64_t b_stride;
  int kp;               // K in whole 16-byte pieces
  int ks, strips;       // warps of a unit, units
  const void* x;        // QUANT: rows x_stride elements apart
  int64_t x_stride;
  int x_dtype, x_wide;
  int pitch;            // QUANT: bytes between quantised rows
};

// Rows quantised into shared memory by the whole CTA, warps_per_row warps a row.
template <typename X, bool WIDE>
__device__ void quantise_rows(const StreamArgs& p, int M, int K, uint8_t* codes, float* scales, uint32_t* most) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per_row = M == 1 ? 8 : M == 2 ? 4 : M <= 4 ? 2 : 1;
  const int first = ((warp % per_row) * 32 + lane) * 8, step = per_row * 256;
  for (int m = warp / per_row; m < M; m += kSWarps / per_row) {
    const X* row = static_cast<const X*>(p.x) + m * p.x_stride;
    uint32_t mx = 0;
    for (int c = first; c < K; c += step) {
      float v[8];
      load_unit<X, WIDE>(row, c, K, v);
      mx = max(mx, magnitude(v));
    }
    mx = __reduce_max_sync(kFullMask, mx);
    if (lane == 0) atomicMax(most + m, mx);
  }
  __syncthreads();
  for (int m = warp / per_row; m < M; m += kSWarps / per_row) {
    const X* row = static_cast<const X*>(p.x) + m * p.x_stride;
    const RowScale r = row_scale(most[m]);
    if (first == 0) scales[m] = __fdiv_rn(__uint_as_float(most[m]), 127.f);
    for (int c = first; c < p.kp; c += step) {
      float v[8];
      if (c < K)
        load_unit<X, WIDE>(row, c, K, v);
      else
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.f;
      store_unit(reinterpret_cast<int8_t*>(codes + m * p.pitch + c), v, r);
    }
  }
  __syncthreads();
}

template <bool QUANT, typename T>
__global__ void __launch_bounds__(kSThreads, 2) stream_kernel(const __grid_constant__ Int8Args a,
                                                              const __grid_constant__ StreamArgs p) {
  extern __shared__ __align__(16) uint8_t codes[];
  __shared__ int red[2][kSWarps][4][32];
  __shared__ float scales[kSRows];
  __shared__ uint32_t most[kSRows];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, q = lane & 3;
  if (QUANT && threadIdx.x < kSRows) most[threadIdx.x] = 0;
  if (QUANT) __syncthreads();
  pdl_launch_dependents();
  pdl_wait();
  T* out = static_cast<T*>(a.out);
  const int ks = p.ks, team = warp / ks, part = warp % ks, teams = kSWarps / ks;
  const int steps = (p.kp + 127) / 128, rounds = (steps + kSteps * ks - 1) / (kSteps * ks);

  // the weights of this lane's two channels (g and g + 8 of the unit's 16), and
  // its row's codes
  uint4 wa[kSteps][4], xa[QUANT ? 1 : kSteps][2];
  const uint4 none = make_uint4(0, 0, 0, 0);
  float sb[2], bias[2], sa[2];
  auto load = [&](int unit, int round) {
    const int ch = unit * 16 + g;
    const int8_t* w0 = p.b + min(ch, a.N - 1) * p.b_stride + q * 16;
    const int8_t* w1 = p.b + min(ch + 8, a.N - 1) * p.b_stride + q * 16;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int k0 = ((round * kSteps + i) * ks + part) * 128;
      const bool in0 = k0 + q * 16 < p.kp, in1 = k0 + 64 + q * 16 < p.kp;
      wa[i][0] = in0 ? ldg_stream16(w0 + k0) : none;
      wa[i][1] = in1 ? ldg_stream16(w0 + k0 + 64) : none;
      wa[i][2] = in0 ? ldg_stream16(w1 + k0) : none;
      wa[i][3] = in1 ? ldg_stream16(w1 + k0 + 64) : none;
      if (!QUANT) {
        const int8_t* x = p.a + g * p.a_stride + q * 16 + k0;
        xa[i][0] = g < a.P && in0 ? __ldg(reinterpret_cast<const uint4*>(x)) : none;
        xa[i][1] = g < a.P && in1 ? __ldg(reinterpret_cast<const uint4*>(x + 64)) : none;
      }
    }
  };
  float next_sb[2], next_bias[2];
  auto load_scales = [&](int unit) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int ch = min(unit * 16 + g + 8 * h, a.N - 1);
      next_sb[h] = a.b_scale[ch];
      next_bias[h] = a.bias ? a.bias[ch] : 0.f;
    }
  };

  int unit = blockIdx.x * teams + team;
  const int stride = gridDim.x * teams;
  if (unit < p.strips) {
    load(unit, 0);
    load_scales(unit);
  }
  if (QUANT) {
    if (p.x_dtype == MTP_DTYPE_BF16)
      p.x_wide ? quantise_rows<__nv_bfloat16, true>(p, a.P, a.K, codes, scales, most)
               : quantise_rows<__nv_bfloat16, false>(p, a.P, a.K, codes, scales, most);
    else if (p.x_dtype == MTP_DTYPE_FP16)
      p.x_wide ? quantise_rows<__half, true>(p, a.P, a.K, codes, scales, most)
               : quantise_rows<__half, false>(p, a.P, a.K, codes, scales, most);
    else
      p.x_wide ? quantise_rows<float, true>(p, a.P, a.K, codes, scales, most)
               : quantise_rows<float, false>(p, a.P, a.K, codes, scales, most);
  }
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int r = 2 * q + t;
    sa[t] = r >= a.P ? 0.f : QUANT ? scales[r] : a.a_scale[r];
  }
  int buf = 0;
  for (; unit < p.strips; unit += stride) {
    int acc[4] = {0, 0, 0, 0};
#pragma unroll
    for (int h = 0; h < 2; ++h) sb[h] = next_sb[h], bias[h] = next_bias[h];
    for (int round = 0; round < rounds; ++round) {
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint4 x = none;
          if (QUANT) {
            const int k = ((round * kSteps + s) * ks + part) * 128 + h * 64 + q * 16;
            if (g < a.P && k < p.kp) x = lds128(smem_u32(codes + g * p.pitch + k));
          } else {
            x = xa[s][h];
          }
          const uint4 w0 = wa[s][h], w1 = wa[s][2 + h];
          mma_s8(acc, w0.x, w1.x, w0.y, w1.y, x.x, x.y);
          mma_s8(acc, w0.z, w1.z, w0.w, w1.w, x.z, x.w);
        }
      if (round + 1 < rounds) {
        load(unit, round + 1);
      } else if (unit + stride < p.strips) {
        load(unit + stride, 0);
        load_scales(unit + stride);
      }
    }
    // the sums of the team's warps; then each warp writes its share of the results
    if (ks > 1) {
#pragma unroll
      for (int r = 0; r < 4; ++r) red[buf][warp][r][lane] = acc[r];
      named_bar_sync(1 + team, 32 * ks);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (r % ks != part) continue;
      int v = acc[r];
      if (ks > 1) {
        v = 0;
        for (int w = 0; w < ks; ++w) v += red[buf][team * ks + w][r][lane];
      }
      const int row = 2 * q + (r & 1), h = r >> 1, ch = unit * 16 + g + 8 * h;
      if (row < a.P && ch < a.N)
        out[static_cast<int64_t>(row) * a.N + ch] = out_cast<T>(fmaf(__int2float_rn(v) * sa[r & 1], sb[h], bias[h]));
    }
    buf ^= 1;  // its readers are past the next unit's barrier before it is written again
  }
}

template <bool QUANT, typename T>
int run(const Int8Args& a, StreamArgs p, cudaStream_t st) {
  auto* kernel = stream_kernel<QUANT, T>;
  const int sms = device_sm_count();
  if (!sms) return MTP_ERR_CUDA;
  static DeviceRecord record;
  const int rc = allow_shared(record, kernel, kSRowBytes);
  if (rc != MTP_OK) return rc;
  p.kp = (a.K + 15) / 16 * 16;
  p.strips = (a.N + 15) / 16;
  // Warps of a unit: as many as it takes to give every warp of the GPU work.
  const int steps = (p.kp + 127) / 128;
  p.ks = 1;
  while (p.ks < kSWarps && p.ks < steps && static_cast<int64_t>(p.strips) * p.ks < 2ll * sms * kSWarps) p.ks *= 2;
  const int ctas = (p.strips * p.ks + kSWarps - 1) / kSWarps;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(std::min(ctas, 2 * sms));
  cfg.blockDim = dim3(kSThreads);
  cfg.dynamicSmemBytes = QUANT ? static_cast<size_t>(a.P) * p.pitch : 0;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, a, p) != cudaSuccess) {
    cudaGetLastError();
    return MTP_ERR_LAUNCH;
  }
  return MTP_OK;
}

template <bool QUANT>
int by_out(const Int8Args& a, const StreamArgs& p, int out_dtype, cudaStream_t st) {
  switch (out_dtype) {
    case MTP_DTYPE_BF16: return run<QUANT, __nv_bfloat16>(a, p, st);
    case MTP_DTYPE_FP16: return run<QUANT, __half>(a, p, st);
    default: return run<QUANT, float>(a, p, st);
  }
}

// Quantised rows half a bank row apart: the eight rows that a load of shared
// memory touches fall on different banks.
int row_pitch(int K) { return (K + 127) / 128 * 128 + 64; }

}  // namespace

bool int8_stream_takes(int rows) { return rows <= kSRows; }

bool int8_stream_quantises(int rows, int K) {
  return rows <= kSRows && static_cast<int64_t>(rows) * row_pitch(K) <= kSRowBytes;
}

int launch_int8_stream(Int8Args a, int out_dtype, const void* ap, int64_t a_stride, const void* bp, int64_t b_stride,
                       cudaStream_t st) {
  StreamArgs p = {};
  p.a = static_cast<const int8_t*>(ap);
  p.a_stride = a_stride;
  p.b = static_cast<const int8_t*>(bp);
  p.b_stride = b_stride;
  return by_out<false>(a, p, out_dtype, st);
}

int launch_int8_stream_quantise(Int8Args a, int out_dtype, const void* x, int64_t x_stride, int x_dtype, const void* bp,
                                int64_t b_stride, cudaStream_t st) {
  StreamArgs p = {};
  p.b = static_cast<const int8_t*>(bp);
  p.b_stride = b_stride;
  p.x = x;
  p.x_stride = x_stride;
  p.x_dtype = x_dtype;
  const int64_t size = x_dtype == MTP_DTYPE_FP32 ? 4 : 2;
  p.x_wide = aligned(x, 16) && a.K % 8 == 0 && (a.P == 1 || x_stride * size % 16 == 0);
  p.pitch = row_pitch(a.K);
  return by_out<true>(a, p, out_dtype, st);
}

}  // namespace mtp
