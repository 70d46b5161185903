// Products of int8 rows and int8 weights with one scale per row and one per
// output channel, for one weight matrix or one per group of rows:
//   out[m, n] = (sum_k a[m, k] * b[g(m), n, k]) * sa[m] * sb[g(m), n] (+ bias[n])
// and, gated, out[m, i] = silu(z[m, i]) * z[m, I + i] of that z, I = N / 2.
// The sum is exact in int32 (K < 2^17); the scales are applied in fp32 and the
// result is rounded once.
//
// tile_kernel: persistent, warp-specialised, one CTA per SM. A tile is 128
// output channels (the MMA's M) x up to NT rows of one group (its N, rounded
// up to 16 for a group's last tile, so a ragged group costs what it has).
//   warp 8    producer: per stage (128 of K) one TMA box of weights and the
//             boxes of rows that the tile has, 128-byte swizzle; columns past
//             K and rows past the end arrive as zeros;
//   warp 9    one thread issues tcgen05.mma kind::i8 (K = 32) into one of two
//             accumulators of NT columns in tensor memory;
//   warps 0-7 epilogue: tensor memory -> scales -> output, while the next
//             tile's products run.
// Gated tiles hold 16 gate channels, then their 16 up channels, four times,
// so that a gate and its up value lie 16 lanes apart in one warp.
#include "internal.cuh"

#include <cuda.h>

#include <algorithm>

namespace mtp {
namespace {

constexpr int kTK = 128;            // K of a stage: one 128-byte swizzle row of int8
constexpr int kTM = 128;            // channels of a tile
constexpr int kTEpiWarps = 8;
constexpr int kTThreads = (kTEpiWarps + 2) * 32;
constexpr int kTMaxGroups = 1024;
constexpr uint32_t kTWBytes = kTM * kTK;
constexpr uint64_t kTTimeoutNs = 2000000000ull;
constexpr uint32_t kTIdesc = (2u << 4) | (1u << 7) | (1u << 10) | (8u << 24);  // D s32, A and B s8, M = 128

// Ring of a tile of NT rows.
template <int NT>
struct Ring {
  static constexpr int kStages = NT == 256 ? 4 : NT == 128 ? 6 : 8;
  static constexpr int kBox = NT < 64 ? NT : 64;  // rows of one TMA box
  static constexpr uint32_t kBytes = kTWBytes + NT * kTK;
};

struct alignas(8) TileCtrl {
  uint64_t full[8], empty[8];  // stage landed / consumed
  uint64_t dfull[2], dempty[2];  // accumulator complete / read
  uint32_t tmem;
  int routed;                  // rows before offsets[E]
  int pre[kTMaxGroups + 1];    // row tiles before each group
};
constexpr uint32_t kTCtrl = 6144;  // control block at the end of the stages
static_assert(sizeof(TileCtrl) <= kTCtrl, "control block");

template <int NT>
constexpr size_t tile_smem() {
  return 1024 + static_cast<size_t>(Ring<NT>::kStages) * Ring<NT>::kBytes + kTCtrl;
}
static_assert(tile_smem<256>() <= 227 * 1024 && tile_smem<128>() <= 227 * 1024 && tile_smem<64>() <= 227 * 1024,
              "shared memory");

__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          dst),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}

// D[tmem] (+)= A[smem] x B[smem]^T, kind::i8
__device__ __forceinline__ void umma_i8_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}

// K-major operand in the 128-byte swizzle: 8-row groups of 1024 bytes.
__device__ __forceinline__ uint64_t desc_swizzle128(uint32_t addr) {
  return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (1ull << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}

// A wait of at most kTTimeoutNs. After one that ran out (recorded in the
// caller's status) this thread's waits only look once, so the kernel runs to
// its end.
struct Waits {
  int32_t* status;
  bool out = false;
  __device__ __forceinline__ explicit Waits(const Int8Args& a) : status(a.status) {}
  __device__ __forceinline__ void operator()(uint32_t bar, uint32_t parity) {
    if (mbar_try_wait(bar, parity) || out) return;
    if (!mbar_wait(bar, parity, global_timer_ns() + kTTimeoutNs)) {
      out = true;
      if (status) atomicOr(status, 1);
    }
  }
};

// One tile of the walk: group, first row, rows, channel tile.
struct Tile {
  int e, row, n, ct;
};

template <int NT>
__device__ __forceinline__ Tile tile_at(const Int8Args& a, const TileCtrl& cb, int t, int& e) {
  Tile r;
  const int blk = t / a.ctiles;
  r.ct = t - blk * a.ctiles;
  // first group whose tiles end past blk; tiles ascend, so the last one's
  // group is a lower bound
  int lo = e, hi = a.E - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (cb.pre[mid + 1] > blk)
      hi = mid;
    else
      lo = mid + 1;
  }
  e = lo;
  r.e = lo;
  int first = 0, last = a.P;
  if (a.offsets) {
    first = min(max(a.offsets[lo], 0), a.P);
    last = min(max(a.offsets[lo + 1], 0), a.P);
  }
  r.row = first + (blk - cb.pre[lo]) * NT;
  r.n = min(NT, last - r.row);
  return r;
}

template <typename T>
__device__ __forceinline__ T out_cast(float v);
template <>
__device__ __forceinline__ float out_cast(float v) { return v; }
template <>
__device__ __forceinline__ __half out_cast(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 out_cast(float v) { return __float2bfloat16_rn(v); }

template <int NT, bool GATED>
__device__ void tile_producer(const CUtensorMap* ta, const CUtensorMap* tb, const Int8Args& a, TileCtrl& cb,
                              uint32_t stages, int ntiles) {
  constexpr int S = Ring<NT>::kStages, BOX = Ring<NT>::kBox;
  const int nk = (a.K + kTK - 1) / kTK;
  Waits wait(a);
  int st = 0, e = 0;
  uint32_t ph = 0;
  int64_t issued = 0;
  for (int t = blockIdx.x; t < ntiles; t += gridDim.x) {
    const Tile w = tile_at<NT>(a, cb, t, e);
    const int boxes = (w.n + BOX - 1) / BOX;
    for (int s = 0; s < nk; ++s) {
      wait(smem_u32(&cb.empty[st]), ph ^ 1u);
      const uint32_t sb = stages + st * Ring<NT>::kBytes, bar = smem_u32(&cb.full[st]);
      mbar_arrive_expect_tx(bar, kTWBytes + boxes * (BOX * kTK));
      if (GATED) {
        const int g0 = w.e * a.N + w.ct * 64, u0 = g0 + a.N / 2;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          tma_2d(sb + q * 4096, tb, s * kTK, g0 + 16 * q, bar);
          tma_2d(sb + q * 4096 + 2048, tb, s * kTK, u0 + 16 * q, bar);
        }
      } else {
        tma_2d(sb, tb, s * kTK, w.e * a.N + w.ct * kTM, bar);
      }
      for (int q = 0; q < boxes; ++q) tma_2d(sb + kTWBytes + q * (BOX * kTK), ta, s * kTK, w.row + q * BOX, bar);
      ++issued;
      if (++st == S) {
        st = 0;
        ph ^= 1u;
      }
    }
  }
  // no copy may still be writing shared memory when the CTA exits
  wait.out = false;
  for (int64_t j = issued - 1; j >= 0 && j >= issued - S; --j)
    wait(smem_u32(&cb.full[j % S]), static_cast<uint32_t>((j / S) & 1));
}

template <int NT>
__device__ void tile_mma(const Int8Args& a, TileCtrl& cb, uint32_t stages, uint32_t tmem, int ntiles) {
  constexpr int S = Ring<NT>::kStages;
  const int nk = (a.K + kTK - 1) / kTK;
  Waits wait(a);
  int st = 0, db = 0, e = 0;
  uint32_t ph = 0, dph = 0;
  for (int t = blockIdx.x; t < ntiles; t += gridDim.x) {
    const Tile w = tile_at<NT>(a, cb, t, e);
    const uint32_t idesc = kTIdesc | (static_cast<uint32_t>((w.n + 15) >> 4) << 18);
    wait(smem_u32(&cb.dempty[db]), dph ^ 1u);
    tc_fence_after();
    const uint32_t d = tmem + db * NT;
    for (int s = 0; s < nk; ++s) {
      wait(smem_u32(&cb.full[st]), ph);
      tc_fence_after();
      const uint64_t wd = desc_swizzle128(stages + st * Ring<NT>::kBytes);
      const uint64_t xd = desc_swizzle128(stages + st * Ring<NT>::kBytes + kTWBytes);
#pragma unroll
      for (int j = 0; j < kTK / 32; ++j) umma_i8_ss(d, wd + 2 * j, xd + 2 * j, idesc, (s | j) != 0);
      umma_commit(smem_u32(&cb.empty[st]));
      if (++st == S) {
        st = 0;
        ph ^= 1u;
      }
    }
    umma_commit(smem_u32(&cb.dfull[db]));
    if (++db == 2) {
      db = 0;
      dph ^= 1u;
    }
  }
}

// Rows behind the last group's are zero: the bytes [from, to) of the output,
// shared out over all epilogue threads of the grid.
__device__ __forceinline__ void zero_tail(uint8_t* from, uint8_t* to) {
  const int64_t tid = static_cast<int64_t>(blockIdx.x) * (kTEpiWarps * 32) + threadIdx.x;
  const int64_t all = static_cast<int64_t>(gridDim.x) * (kTEpiWarps * 32);
  uint8_t* lo = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(from) + 15) & ~static_cast<uintptr_t>(15));
  uint8_t* hi = reinterpret_cast<uint8_t*>(reinterpret_cast<uintptr_t>(to) & ~static_cast<uintptr_t>(15));
  if (lo >= hi) {
    for (int64_t i = tid; i < to - from; i += all) from[i] = 0;
    return;
  }
  for (int64_t i = tid; i < (hi - lo) / 16; i += all) reinterpret_cast<uint4*>(lo)[i] = make_uint4(0, 0, 0, 0);
  if (tid < lo - from) from[tid] = 0;
  if (tid < to - hi) hi[tid] = 0;
}

template <int NT, bool GATED, typename T>
__device__ void tile_epilogue(const Int8Args& a, TileCtrl& cb, uint32_t tmem, int ntiles) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int quad = warp & 3, half = warp >> 2;
  const int width = GATED ? a.N / 2 : a.N;  // columns of the output
  T* out = static_cast<T*>(a.out);
  if (cb.routed < a.P)
    zero_tail(reinterpret_cast<uint8_t*>(out + static_cast<int64_t>(cb.routed) * width),
              reinterpret_cast<uint8_t*>(out + static_cast<int64_t>(a.P) * width));
  Waits wait(a);
  int db = 0, e = 0;
  uint32_t dph = 0;
  for (int t = blockIdx.x; t < ntiles; t += gridDim.x) {
    const Tile w = tile_at<NT>(a, cb, t, e);
    // this lane's output channel and the row of b behind its accumulator lane
    const int ch = GATED ? w.ct * 64 + 16 * quad + (lane & 15) : w.ct * kTM + 32 * quad + lane;
    const bool valid = ch < width;
    const int brow = GATED && lane >= 16 ? a.N / 2 + ch : ch;
    const float sb = valid ? a.b_scale[static_cast<int64_t>(w.e) * a.N + brow] : 0.f;
    const float bias = valid && a.bias ? a.bias[ch] : 0.f;
    wait(smem_u32(&cb.dfull[db]), dph);
    tc_fence_after();
    const uint32_t dt = tmem + (static_cast<uint32_t>(32 * quad) << 16) + db * NT;
    for (int c = 16 * half; c < w.n; c += 32) {
      const int mine = c + (lane & 15);
      const float sa = mine < w.n ? a.a_scale[w.row + mine] : 0.f;
      uint32_t v[16];
      tmem_ld16(dt + c, v);
      tmem_wait_ld();
      T* o = out + static_cast<int64_t>(w.row + c) * width + ch;
      if (GATED) {
        // two rows at a time: the low lanes take the first, the high lanes the second
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
          const float z0 = __int2float_rn(static_cast<int>(v[j])) * __shfl_sync(kFullMask, sa, j) * sb;
          const float z1 = __int2float_rn(static_cast<int>(v[j + 1])) * __shfl_sync(kFullMask, sa, j + 1) * sb;
          const float got = __shfl_xor_sync(kFullMask, lane < 16 ? z1 : z0, 16);
          const float h = lane < 16 ? silu_fast(z0) * got : silu_fast(got) * z1;
          const int r = j + (lane >> 4);
          if (valid && c + r < w.n) o[static_cast<int64_t>(r) * width] = out_cast<T>(h);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float z = __int2float_rn(static_cast<int>(v[j])) * __shfl_sync(kFullMask, sa, j) * sb + bias;
          if (valid && c + j < w.n) o[static_cast<int64_t>(j) * width] = out_cast<T>(z);
        }
      }
    }
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&cb.dempty[db]));
    if (++db == 2) {
      db = 0;
      dph ^= 1u;
    }
  }
}

template <int NT, bool GATED, typename T>
__global__ void __launch_bounds__(kTThreads, 1) tile_kernel(const __grid_constant__ CUtensorMap ta,
                                                            const __grid_constant__ CUtensorMap tb, const Int8Args a) {
  extern __shared__ uint8_t smem_raw[];
  constexpr int S = Ring<NT>::kStages;
  const uint32_t stages = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* aligned = smem_raw + (stages - smem_u32(smem_raw));
  TileCtrl& cb = *reinterpret_cast<TileCtrl*>(aligned + S * Ring<NT>::kBytes);
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(smem_u32(&cb.full[i]), 1);
      mbar_init(smem_u32(&cb.empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&cb.dfull[i]), 1);
      mbar_init(smem_u32(&cb.dempty[i]), kTEpiWarps);
    }
    fence_mbar_init();
  }
  if (warp == kTEpiWarps + 1) {
    tmem_alloc(smem_u32(&cb.tmem), 2 * NT);
    tmem_relinquish();
  }
  pdl_launch_dependents();
  pdl_wait();
  // row tiles of every group, then their running sum
  for (int e = threadIdx.x; e < a.E; e += kTThreads) {
    int n = a.P;
    if (a.offsets) n = min(max(a.offsets[e + 1], 0), a.P) - min(max(a.offsets[e], 0), a.P);
    cb.pre[e + 1] = (max(n, 0) + NT - 1) / NT;
  }
  __syncthreads();
  if (warp == 0) {
    const int lane = threadIdx.x;
    int run = 0;
    for (int e0 = 0; e0 < a.E; e0 += 32) {
      int x = e0 + lane < a.E ? cb.pre[e0 + lane + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(kFullMask, x, o);
        if (lane >= o) x += y;
      }
      if (e0 + lane < a.E) cb.pre[e0 + lane + 1] = run + x;
      run += __shfl_sync(kFullMask, x, 31);
    }
    if (lane == 0) {
      cb.pre[0] = 0;
      cb.routed = a.offsets ? min(max(a.offsets[a.E], 0), a.P) : a.P;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = cb.tmem;
  const int ntiles = cb.pre[a.E] * a.ctiles;
  if (warp == kTEpiWarps) {
    if ((threadIdx.x & 31) == 0) tile_producer<NT, GATED>(&ta, &tb, a, cb, stages, ntiles);
  } else if (warp == kTEpiWarps + 1) {
    if ((threadIdx.x & 31) == 0) tile_mma<NT>(a, cb, stages, tmem, ntiles);
  } else {
    tile_epilogue<NT, GATED, T>(a, cb, tmem, ntiles);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == kTEpiWarps + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 2 * NT);
  }
}

// ---------------------------------------------------------------------------
// rows into a layout that TMA takes (16-byte aligned base and stride)
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(256) pad_rows_kernel(const int8_t* __restrict__ src, int64_t stride, int64_t rows,
                                                       int K, int8_t* __restrict__ dst, int64_t dst_stride) {
  pdl_launch_dependents();
  pdl_wait();
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); r < rows;
       r += static_cast<int64_t>(gridDim.x) * 8)
    for (int c = (threadIdx.x & 31) * 4; c < K; c += 128) {
      uint32_t w = 0;
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (c + q < K) w |= static_cast<uint32_t>(static_cast<uint8_t>(src[r * stride + c + q])) << (8 * q);
      *reinterpret_cast<uint32_t*>(dst + r * dst_stride + c) = w;
    }
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

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_fn() {
  static EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      p = nullptr;
    }
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
}

// [rows, K] int8 with a row stride, in boxes of box_rows x 128 bytes.
int encode_rows(CUtensorMap* map, const void* base, int64_t rows, int K, int64_t stride, int box_rows) {
  EncodeTiled fn = encode_fn();
  if (!fn) return MTP_ERR_CUDA;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(K), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride)};
  const cuuint32_t box[2] = {kTK, static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t step[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, step,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? MTP_OK
             : MTP_ERR_CUDA;
}

int device_sms() {
  static int sms[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  if (!sms[dev]) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    sms[dev] = n;
  }
  return sms[dev];
}

template <int NT, bool GATED, typename T>
int run_tiles(Int8Args& a, const void* ap, int64_t a_stride, const void* bp, int64_t b_stride, int sms,
              cudaStream_t st) {
  auto* kernel = tile_kernel<NT, GATED, T>;
  constexpr size_t smem = tile_smem<NT>();
  static int configured_device = -1;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return MTP_ERR_CUDA;
  if (configured_device != dev) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) !=
        cudaSuccess)
      return MTP_ERR_CUDA;
    configured_device = dev;
  }
  CUtensorMap ta, tb;
  int rc = encode_rows(&ta, ap, a.P, a.K, a_stride, Ring<NT>::kBox);
  if (rc == MTP_OK) rc = encode_rows(&tb, bp, static_cast<int64_t>(a.E) * a.N, a.K, b_stride, GATED ? 16 : kTM);
  if (rc != MTP_OK) return rc;
  a.ctiles = GATED ? (a.N / 2 + 63) / 64 : (a.N + kTM - 1) / kTM;
  // row tiles: at most one partial one per group that has rows
  const int64_t blocks = a.P / NT + std::min(a.P, a.E);
  const int64_t grid = std::min<int64_t>(sms, std::max<int64_t>(blocks * a.ctiles, 1));
  return launch(kernel, dim3(static_cast<unsigned>(grid)), dim3(kTThreads), smem, st, ta, tb, a);
}

template <int NT, bool GATED>
int by_out(Int8Args& a, int out_dtype, const void* ap, int64_t as, const void* bp, int64_t bs, int sms,
           cudaStream_t st) {
  switch (out_dtype) {
    case MTP_DTYPE_BF16: return run_tiles<NT, GATED, __nv_bfloat16>(a, ap, as, bp, bs, sms, st);
    case MTP_DTYPE_FP16: return run_tiles<NT, GATED, __half>(a, ap, as, bp, bs, sms, st);
    default: return run_tiles<NT, GATED, float>(a, ap, as, bp, bs, sms, st);
  }
}

template <bool GATED>
int by_rows(Int8Args& a, int nt, int out_dtype, const void* ap, int64_t as, const void* bp, int64_t bs, int sms,
            cudaStream_t st) {
  if (nt == 256) return by_out<256, GATED>(a, out_dtype, ap, as, bp, bs, sms, st);
  if (nt == 128) return by_out<128, GATED>(a, out_dtype, ap, as, bp, bs, sms, st);
  if (nt == 64) return by_out<64, GATED>(a, out_dtype, ap, as, bp, bs, sms, st);
  return by_out<32, GATED>(a, out_dtype, ap, as, bp, bs, sms, st);
}

}  // namespace

bool tma_rows_ok(const void* base, int64_t stride) { return aligned(base, 16) && stride % 16 == 0; }

int launch_pad_rows(const void* src, int64_t stride, int64_t rows, int K, void* dst, int64_t dst_stride,
                    cudaStream_t st) {
  const int64_t grid = std::min<int64_t>((rows + 7) / 8, 148 * 16);
  return launch(pad_rows_kernel, dim3(static_cast<unsigned>(grid)), dim3(256), 0, st, static_cast<const int8_t*>(src),
                stride, rows, K, static_cast<int8_t*>(dst), dst_stride);
}

int launch_int8_matmul(Int8Args a, bool gated, int out_dtype, const void* ap, int64_t a_stride, const void* bp,
                       int64_t b_stride, cudaStream_t st) {
  const int sms = device_sms();
  if (!sms) return MTP_ERR_CUDA;
  // Rows of a tile: enough for the average group, fewer while the tiles do not
  // fill the SMs.
  const int per_group = (a.P + a.E - 1) / a.E;
  int nt = per_group <= 24 ? 32 : per_group <= 48 ? 64 : per_group <= 96 ? 128 : 256;
  const int64_t ct = gated ? (a.N / 2 + 63) / 64 : (a.N + kTM - 1) / kTM;
  while (nt > 32 && ct * ((per_group + nt - 1) / nt) * std::min(a.P, a.E) < sms) nt /= 2;
  return gated ? by_rows<true>(a, nt, out_dtype, ap, a_stride, bp, b_stride, sms, st)
               : by_rows<false>(a, nt, out_dtype, ap, a_stride, bp, b_stride, sms, st);
}

}  // namespace mtp
