// Layer norm and its gradients.
//
// forward:  mean and variance of a row's H values (the variance from the
//           centred values, so an offset costs no digits), rstd = 1 / sqrt(var +
//           eps), y = (x - mean) rstd w + b.
// gradient: with xhat = (x - mean) rstd and wg = w g,
//           dx = rstd (wg - mean(wg) - xhat mean(wg xhat)),
//           dw = sum over the rows of g xhat, db = sum of g.
//
// All sums in fp32, in an order that sizes and memory layout fix; results are
// rounded once. In the ring 1 / sqrt is rsqrtf, within 2 units in the last place,
// and sums go warp by warp: the bits of a row may differ between calls of up to 296
// rows, which norm_row_kernel takes, and of more.
//
// The bytes are x in and y out; for the gradients x and grad in and dx out. What
// keeps the kernels from HBM's rate is the work per row between its two sums
// (16384 x 8192 bf16: 14 and 24 instructions a value, one barrier a row):
//   8192 x 2048 bf16:  19 us forward, 36 backward (bytes alone 10 and 15)
//   16384 x 8192 bf16: 113 us and 182 us (82 and 123: 4.7 and 4.4 TB/s)
//   16384 x 4096 fp32: 96 us and 129 us (82 and 123: 5.6 and 6.2 TB/s)
//   20000 x 5001 bf16: 147 us and 371 us (61 and 92: values one by one)
//   one row of 2048: 2.5 us, 6.4 us
// Rows that the ring has no room for (two stages of whole rows and the parameters:
// forward up to 16384 values of 16 bits and 14336 of fp32, the gradients, with x
// and grad in it, 16384 and 11264) take norm_row_kernel forward, up to its 8192
// vectors, and otherwise plain kernels that read a row three times, a value a load:
//   4096 x 12288 fp32: 92 us (ring) and 305 us (62 and 92)
//   4096 x 16384 fp32: 146 us and 475 us (82 and 123)
//   8192 x 20480 bf16: 314 us and 818 us (103 and 154)
//   8192 x 32769 bf16: 790 us and 1634 us (164 and 246)
// Taken one after the other, 16384 x 8192 bf16 there and back: rows read three
// times and columns by a kernel of their own 197 + 681 us; one pass, rows in
// registers 176 + 463; a ring of bulk copies with one value a load 188 + 307, with
// 16 bytes a load and two fp32 operations an instruction 128 + 175; two rows a
// barrier, parameters in registers 113 + 177.
#include "rows.cuh"

#include <math.h>

#include <algorithm>

namespace mtp {
namespace {

constexpr int kThreads = 256;
constexpr int kPlainCtas = 32768;    // most of the plain kernels, whose 32-bit row index steps past the last row by as many
constexpr int kSms = 148;
constexpr int kRowThreads = 1024;    // most threads of a row in norm_row_kernel
constexpr int kGroupThreads = 512;   // of a CTA of the ring kernels: 128 registers each
constexpr int kGroupWarps = kGroupThreads / 32;
constexpr int kRing = 224 * 1024;    // bytes of rows in flight and parameters of such a CTA
constexpr int kStages = 4;
constexpr uint64_t kTimeoutNs = 2000000000ull;

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

template <typename P, int N>
__device__ __forceinline__ void params(const void* p, int c, float* f) {
  constexpr int kPiece = N * sizeof(P) <= 16 ? N : 16 / sizeof(P);
#pragma unroll
  for (int n = 0; n < N; n += kPiece) {
    const Vec<P, kPiece> x = *reinterpret_cast<const Vec<P, kPiece>*>(static_cast<const P*>(p) + c + n);
    to_floats(x, f + n);
  }
}
// N parameters from index c on, `otherwise` without any.
template <typename T, int N>
__device__ __forceinline__ void params(const void* p, bool fp32, int c, float otherwise, float* f) {
  if (!p) {
#pragma unroll
    for (int n = 0; n < N; ++n) f[n] = otherwise;
  } else if (fp32) {
    params<float, N>(p, c, f);
  } else {
    params<T, N>(p, c, f);
  }
}

// ---------------------------------------------------------------------------
// forward of a few rows: a row in the registers of blockDim.x threads
// ---------------------------------------------------------------------------
// (and of rows wider than the ring's 16384 values of 16 bits or 14336 of fp32, up
// to 8192 vectors). One row of 2048 bf16: 2.5 us; for 8192 of them it takes 39 us,
// the ring 19.
template <typename T, int N, int NV>
__global__ void __launch_bounds__(kRowThreads, 1) norm_row_kernel(const NormArgs a) {
  using V = Vec<T, N>;
  __shared__ float2 tmp[kRowThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int64_t t = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + t * a.stride;
  V v[NV];
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (threadIdx.x + i * blockDim.x) * N;
    if (c < a.H) v[i] = *reinterpret_cast<const V*>(x + c);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float f[N];
    to_floats(v[i], f);
    if ((threadIdx.x + i * blockDim.x) * N < a.H)
#pragma unroll
      for (int n = 0; n < N; ++n) s += f[n];
  }
  const float mean = block_sum(make_float2(s, 0.f), tmp).x / a.H;
  s = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float f[N];
    to_floats(v[i], f);
    if ((threadIdx.x + i * blockDim.x) * N < a.H)
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const float d = f[n] - mean;
        s = fmaf(d, d, s);
      }
  }
  const float rstd = 1.f / sqrtf(block_sum(make_float2(s, 0.f), tmp).x / a.H + a.eps);
  T* y = static_cast<T*>(a.y) + t * a.H;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (threadIdx.x + i * blockDim.x) * N;
    if (c >= a.H) break;
    float f[N], w[N], b[N];
    params<T, N>(a.weight, a.param_fp32, c, 1.f, w);
    params<T, N>(a.bias, a.param_fp32, c, 0.f, b);
    to_floats(v[i], f);
#pragma unroll
    for (int n = 0; n < N; ++n) f[n] = fmaf((f[n] - mean) * rstd, w[n], b[n]);
    V o;
    from_floats(f, o);
    *reinterpret_cast<V*>(y + c) = o;
  }
  if (a.stats && threadIdx.x == 0) *reinterpret_cast<float2*>(a.stats + 2 * t) = make_float2(mean, rstd);
}

// ---------------------------------------------------------------------------
// many rows: through a ring of bulk copies
// ---------------------------------------------------------------------------
// A CTA's threads form groups of `lanes` (whole warps). A group takes a block of
// `batch` rows after another, and each thread has the same E columns of all of
// them, so that parameters and, for the gradient, the sums over the rows stay in
// its registers. The rows come by bulk copies into a ring of the group's own:
// the bytes in flight depend neither on registers nor on the barrier that a row
// takes (one: a row's sums of all warps go through shared memory, in two buffers
// in turn). A copy begins and ends on 16 bytes, so the units around a block's
// ends come too; where those reach over the tensor's ends their values are
// stored by the thread that issues the copy instead.
struct NormPlan {
  int lanes, groups, batch, stages, blocks, ctas;
  uint32_t row_pitch, stage_bytes;  // in the ring; row_pitch 0: rows follow one another as in memory
  uint32_t ring_bytes, columns;     // the parameters lie behind the ring, `columns` apart
};

// Rows of one tensor as the ring holds them; ALIGNED: they start on 16 bytes.
template <typename T, bool ALIGNED>
struct Rows {
  const T* base;
  int64_t stride;  // elements
  int M, H;
  uint32_t pitch;

  __device__ __forceinline__ const T* row(int64_t t) const { return base + t * stride; }
  // Bytes of a block's rows in front of which the copies begin.
  __device__ __forceinline__ uint32_t lead(const T* p) const {
    return ALIGNED ? 0 : static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p) & 15);
  }
  // Where row t0 + r of the block that begins with t0 lies.
  __device__ __forceinline__ uint32_t offset(int64_t t0, int r) const {
    return pitch ? r * pitch + lead(row(t0 + r)) : lead(row(t0)) + r * H * static_cast<uint32_t>(sizeof(T));
  }
  // The copies of values [p, p + n) to `to`: their bytes, and with ISSUE the
  // copies themselves. The values outside them are stored without.
  template <bool ISSUE>
  __device__ __forceinline__ uint32_t span(const T* p, int n, uint8_t* to, uint32_t bar) const {
    if (ALIGNED) {
      if (ISSUE) bulk_g2s(smem_u32(to), p, n * sizeof(T), bar);
      return n * sizeof(T);
    }
    const uintptr_t begin = reinterpret_cast<uintptr_t>(p), end = reinterpret_cast<uintptr_t>(p + n);
    const uintptr_t zero = begin & ~static_cast<uintptr_t>(15);
    uintptr_t from = zero, past = (end + 15) & ~static_cast<uintptr_t>(15);
    if (from < reinterpret_cast<uintptr_t>(base)) from += 16;
    if (past > reinterpret_cast<uintptr_t>(row(M - 1) + H)) past -= 16;
    if (from > past) from = past = zero;
    if (ISSUE) {
      if (past > from)
        bulk_g2s(smem_u32(to + (from - zero)), reinterpret_cast<const void*>(from), static_cast<uint32_t>(past - from), bar);
    } else {
      for (uintptr_t q = begin; q < end && q < from; q += sizeof(T))
        *reinterpret_cast<T*>(to + (q - zero)) = *reinterpret_cast<const T*>(q);
      for (uintptr_t q = past > begin ? past : begin; q < end; q += sizeof(T))
        *reinterpret_cast<T*>(to + (q - zero)) = *reinterpret_cast<const T*>(q);
    }
    return static_cast<uint32_t>(past - from);
  }
  template <bool ISSUE>
  __device__ __forceinline__ uint32_t block(int64_t t0, int rows, uint8_t* to, uint32_t bar) const {
    if (!pitch) return span<ISSUE>(row(t0), rows * H, to, bar);
    uint32_t bytes = 0;
    for (int r = 0; r < rows; ++r) bytes += span<ISSUE>(row(t0 + r), H, to + r * pitch, bar);
    return bytes;
  }
};

// The group's place, its ring and the walk over its blocks.
struct Walk {
  uint64_t (*full)[kStages];
  uint8_t* ring;
  int group, at, first, step, s;
  uint32_t phase;
  // NaN once a wait of this thread ran out. It joins the thread's part of a row's sums, so that all of the row is NaN
  // whichever thread it was, and the rows behind it. The thread that issues copies then issues no more: a barrier whose
  // phase may not be over takes no arrival, and what the others wait for runs out too.
  float poison;

  __device__ __forceinline__ uint32_t bar(int q) const { return smem_u32(&full[group][q]); }
  __device__ __forceinline__ void begin(const NormPlan& p, uint64_t (*bars)[kStages], uint8_t* smem, int parts) {
    full = bars;
    group = threadIdx.x / p.lanes;
    at = threadIdx.x - group * p.lanes;
    ring = smem + static_cast<size_t>(group) * p.stages * parts * p.stage_bytes;
    first = blockIdx.x + p.ctas * group;
    step = p.ctas * p.groups;
    s = 0;
    phase = 0;
    poison = 0.f;
    if (at == 0)
      for (int q = 0; q < p.stages; ++q) mbar_init(bar(q), 1);
    fence_mbar_init();
    __syncthreads();
    pdl_launch_dependents();
    pdl_wait();
  }
  __device__ __forceinline__ void wait() {
    if (!mbar_try_wait(bar(s), phase) && (poison != 0.f || !mbar_wait(bar(s), phase, global_timer_ns() + kTimeoutNs)))
      poison = __int_as_float(0x7fffffff);
  }
  __device__ __forceinline__ void advance(const NormPlan& p) {
    if (++s == p.stages) {
      s = 0;
      phase ^= 1u;
    }
  }
  // After a wait that ran out, copies may still be on their way into this CTA.
  __device__ __forceinline__ void drain(const NormPlan& p) {
    if (poison == 0.f) return;
    for (int q = 0; q < p.stages; ++q)
      for (uint32_t x = 0; x < 2; ++x)
        if (!mbar_try_wait(bar(q), x)) mbar_wait(bar(q), x, global_timer_ns() + kTimeoutNs / 16);
  }
};

__device__ __forceinline__ int rows_of(const NormArgs& a, const NormPlan& p, int block) {
  return min(p.batch, a.M - block * p.batch);
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n.reg .b64 a, b, c, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmov.b64 c, {%6, %7};\n"
      "fma.rn.f32x2 d, a, b, c;\nmov.b64 {%0, %1}, d;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n.reg .b64 a, b, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nadd.rn.f32x2 d, a, b;\nmov.b64 {%0, %1}, d;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n.reg .b64 a, b, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmul.rn.f32x2 d, a, b;\nmov.b64 {%0, %1}, d;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// s / n with n's reciprocal at hand: one correction makes a quotient that is a
// number of fp32 exact, so that constant rows have no variance.
__device__ __forceinline__ float quotient(float s, float n, float inv) {
  const float q = s * inv;
  return fmaf(fmaf(-q, n, s), inv, q);
}

// The sums of two values over the warp at once, the first in the lower half of
// the lanes, the second in the upper.
__device__ __forceinline__ float half_sums(float p, float q) {
  const bool upper = threadIdx.x & 16;
  float s = (upper ? q : p) + __shfl_xor_sync(kFullMask, upper ? p : q, 16);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) s += __shfl_xor_sync(kFullMask, s, o);
  return s;
}

// The columns of a thread: kVectors vectors of kWidth values as pairs. Vectors
// of one value hold two columns that are `lanes` apart.
template <typename T, int N, int E>
struct Columns {
  static constexpr int kWidth = N == 1 ? 2 : N, kPairs = kWidth / 2, kVectors = E / kWidth;
  int at, lanes, H;

  __device__ __forceinline__ int column(int i, int n = 0) const {
    return N == 1 ? at + (2 * i + n) * lanes : (at + i * lanes) * N + n;
  }
  __device__ __forceinline__ bool has(int i, int n = 0) const { return N == 1 ? column(i, n) < H : column(i) < H; }
  // A row's values; where the thread has no column, zeros or others of the row (without a branch).
  __device__ __forceinline__ void read(const uint8_t* row, int i, float2 (&v)[kPairs]) const {
    float* f = reinterpret_cast<float*>(v);
    if (N == 1) {
#pragma unroll
      for (int n = 0; n < 2; ++n) f[n] = has(i, n) ? value<T>(row, column(i, n)) : 0.f;
    } else {
      const Vec<T, N> x = *reinterpret_cast<const Vec<T, N>*>(row + min(column(i), H - N) * sizeof(T));  // one load
      to_floats(x, f);
    }
  }
  // Other values where the thread has no column.
  __device__ __forceinline__ void fill(float2 (&v)[kVectors][kPairs], float other) const {
#pragma unroll
    for (int i = 0; i < kVectors; ++i)
#pragma unroll
      for (int n = 0; n < kWidth; ++n)
        if (!has(i, n)) reinterpret_cast<float*>(v[i])[n] = other;
  }
  // Parameters that the CTA keeps in shared memory: zeros for columns that the row has not, so that
  // what read() gives there adds nothing to a row's sums.
  __device__ __forceinline__ void kept(const float* p, int i, float2 (&v)[kPairs]) const {
    float* f = reinterpret_cast<float*>(v);
    if (N == 1) {
#pragma unroll
      for (int n = 0; n < 2; ++n) f[n] = p[column(i, n)];
    } else {
      constexpr int kPiece = N < 4 ? N : 4;
#pragma unroll
      for (int n = 0; n < N; n += kPiece) {
        const Vec<float, kPiece> x = *reinterpret_cast<const Vec<float, kPiece>*>(p + column(i) + n);
        to_floats(x, f + n);
      }
    }
  }
  __device__ __forceinline__ void write(T* row, int i, const float2 (&v)[kPairs]) const {
    const float* f = reinterpret_cast<const float*>(v);
    if (N == 1) {
#pragma unroll
      for (int n = 0; n < 2; ++n)
        if (has(i, n)) store<T>(row, column(i, n), f[n]);
    } else if (has(i)) {
      Vec<T, N> o;
      from_floats(f, o);
      *reinterpret_cast<Vec<T, N>*>(row + column(i)) = o;
    }
  }
};

// Parameters into shared memory as fp32, zeros behind the last column.
template <typename T>
__device__ __forceinline__ void keep_params(const void* p, const NormArgs& a, int columns, float otherwise, float* kept) {
  for (int c = threadIdx.x; c < columns; c += blockDim.x)
    kept[c] = c >= a.H ? 0.f : !p ? otherwise : a.param_fp32 ? static_cast<const float*>(p)[c] : value<T>(p, c);
}

// R rows of a block at a time: their sums take the same barrier.
template <typename T, int N, int E, int R>
__global__ void __launch_bounds__(kGroupThreads, 1) norm_ring_kernel(const NormArgs a, const NormPlan plan) {
  using C = Columns<T, N, E>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t full[kGroupWarps][kStages];
  __shared__ float red[2][R][2][kGroupWarps];  // [parity][row]: sum, squares around the warp's mean [warp of the CTA]
  float* weight = reinterpret_cast<float*>(smem + plan.ring_bytes);
  float* bias = weight + plan.columns;
  Walk g;
  g.begin(plan, full, smem, 1);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = plan.lanes >> 5, first_warp = g.group * warps;
  const C cols = {g.at, plan.lanes, a.H};
  const Rows<T, N * sizeof(T) == 16> x = {static_cast<const T*>(a.x), a.stride, a.M, a.H, plan.row_pitch};
  auto issue = [&](int block, int q) {
    const int64_t t0 = static_cast<int64_t>(block) * plan.batch;
    const int rows = rows_of(a, plan, block);
    uint8_t* to = g.ring + static_cast<size_t>(q) * plan.stage_bytes;
    mbar_arrive_expect_tx(g.bar(q), x.template block<false>(t0, rows, to, 0));
    x.template block<true>(t0, rows, to, g.bar(q));
  };
  if (g.at == 0)
    for (int q = 0; q < plan.stages && g.first + q * g.step < plan.blocks; ++q) issue(g.first + q * g.step, q);
  keep_params<T>(a.weight, a, plan.columns, 1.f, weight);
  keep_params<T>(a.bias, a, plan.columns, 0.f, bias);
  __syncthreads();
  // columns of this thread, of its warp, and of the group's warp (lane % 16)
  int mine = 0;
#pragma unroll
  for (int i = 0; i < C::kVectors; ++i)
#pragma unroll
    for (int n = 0; n < C::kWidth; ++n) mine += cols.has(i, n);
  const float columns = __reduce_add_sync(kFullMask, mine);
  const float inv_columns = columns > 0.f ? 1.f / columns : 0.f;
  if (lane == 0) red[0][0][0][warp] = columns;
  __syncthreads();
  const float others = (lane & 15) < warps ? red[0][0][0][first_warp + (lane & 15)] : 0.f;
  const float inv_others = others > 0.f ? 1.f / others : 0.f;
  __syncthreads();
  // Up to 16 columns a thread keeps their parameters in registers.
  constexpr bool kKeep = E <= 16;
  float2 w[kKeep ? C::kVectors : 1][C::kPairs], b[kKeep ? C::kVectors : 1][C::kPairs];
  if (kKeep)
#pragma unroll
    for (int i = 0; i < C::kVectors; ++i) {
      cols.kept(weight, i, w[i]);
      cols.kept(bias, i, b[i]);
    }
  const float inv = 1.f / a.H;
  // With two rows the lower half of the lanes adds up the first's sums, the upper the second's.
  const int half = R == 2 ? lane >> 4 : 0;
  int parity = 0;
  for (int block = g.first; block < plan.blocks; block += g.step) {
    g.wait();
    const int rows = rows_of(a, plan, block);
    const int64_t t0 = static_cast<int64_t>(block) * plan.batch;
    const uint8_t* stage = g.ring + static_cast<size_t>(g.s) * plan.stage_bytes;
    for (int r0 = 0; r0 < rows; r0 += R) {
      float2 v[R][C::kVectors][C::kPairs];
      float sum[R], centre[R], squares[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const uint8_t* row = stage + x.offset(t0, min(r0 + r, rows - 1));
        float2 s = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < C::kVectors; ++i) cols.read(row, i, v[r][i]);
        if (mine < E) cols.fill(v[r], 0.f);
#pragma unroll
        for (int i = 0; i < C::kVectors; ++i)
#pragma unroll
          for (int e = 0; e < C::kPairs; ++e) s = add2(s, v[r][i][e]);
        sum[r] = s.x + s.y + g.poison;
      }
      // this lane's row (half): the warp's sum
      const float my_sum = R == 2 ? half_sums(sum[0], sum[R - 1]) : warp_sum(sum[0]);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        centre[r] = quotient(R == 2 ? __shfl_sync(kFullMask, my_sum, 16 * r) : my_sum, columns, inv_columns);
        if (mine < E) cols.fill(v[r], centre[r]);  // no square
        float2 s = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < C::kVectors; ++i)
#pragma unroll
          for (int e = 0; e < C::kPairs; ++e) {
            const float2 d = add2(v[r][i][e], both(-centre[r]));
            s = fma2(d, d, s);
          }
        squares[r] = s.x + s.y;
      }
      float my_squares = R == 2 ? half_sums(squares[0], squares[R - 1]) : warp_sum(squares[0]);
      float my_mean = quotient(my_sum, a.H, inv);
      if (warps > 1) {
        if ((lane & 15) == 0 && half == lane >> 4) {
          red[parity][half][0][warp] = my_sum;
          red[parity][half][1][warp] = my_squares;
        }
        named_bar_sync(1 + g.group, plan.lanes);  // barrier 0 is the whole CTA's
        const bool in = (lane & 15) < warps;
        const float s = in ? red[parity][half][0][first_warp + (lane & 15)] : 0.f;
        my_squares = in ? red[parity][half][1][first_warp + (lane & 15)] : 0.f;
        my_mean = s;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) my_mean += __shfl_xor_sync(kFullMask, my_mean, o);
        my_mean = quotient(my_mean, a.H, inv);
        // squares around the row's mean: those around a warp's, and its distance
        const float d = quotient(s, others, inv_others) - my_mean;
        my_squares = fmaf(others * d, d, my_squares);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) my_squares += __shfl_xor_sync(kFullMask, my_squares, o);
        parity ^= 1;
      } else {
        __syncwarp();
      }
      if (r0 + R >= rows) {  // every thread has its values of the last row
        const int ahead = block + plan.stages * g.step;
        if (g.at == 0 && ahead < plan.blocks && g.poison == 0.f) issue(ahead, g.s);
        g.advance(plan);
      }
      const float my_rstd = rsqrtf(fmaf(my_squares, inv, a.eps));
      if (a.stats && (g.at & ~16) == 0 && half == g.at >> 4 && r0 + half < rows)
        *reinterpret_cast<float2*>(a.stats + 2 * (t0 + r0 + half)) = make_float2(my_mean, my_rstd);
      float rstd[R], mean[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        rstd[r] = R == 2 ? __shfl_sync(kFullMask, my_rstd, 16 * r) : my_rstd;
        mean[r] = R == 2 ? __shfl_sync(kFullMask, my_mean, 16 * r) : my_mean;
      }
      T* out = static_cast<T*>(a.y) + (t0 + r0) * a.H;
#pragma unroll
      for (int i = 0; i < C::kVectors; ++i) {
        if (!kKeep) {
          cols.kept(weight, i, w[0]);
          cols.kept(bias, i, b[0]);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
          for (int e = 0; e < C::kPairs; ++e)
            v[r][i][e] = fma2(mul2(add2(v[r][i][e], both(-mean[r])), both(rstd[r])), w[kKeep ? i : 0][e], b[kKeep ? i : 0][e]);
          if (r0 + r < rows) cols.write(out + r * static_cast<int64_t>(a.H), i, v[r][i]);
        }
      }
    }
  }
  g.drain(plan);
}

template <typename T, int N, int E>
__global__ void __launch_bounds__(kGroupThreads, 1) norm_backward_kernel(const NormArgs a, const NormPlan plan) {
  using C = Columns<T, N, E>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t full[kGroupWarps][kStages];
  __shared__ float red[2][2][kGroupWarps];  // [parity][sum][warp of the CTA]
  float* weight = reinterpret_cast<float*>(smem + plan.ring_bytes);
  Walk g;
  g.begin(plan, full, smem, 2);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = plan.lanes >> 5, first_warp = g.group * warps;
  const C cols = {g.at, plan.lanes, a.H};
  const Rows<T, N * sizeof(T) == 16> x = {static_cast<const T*>(a.x), a.stride, a.M, a.H, plan.row_pitch};
  const Rows<T, N * sizeof(T) == 16> grad = {static_cast<const T*>(a.grad), a.H, a.M, a.H, 0};
  auto issue = [&](int block, int q) {
    const int64_t t0 = static_cast<int64_t>(block) * plan.batch;
    const int rows = rows_of(a, plan, block);
    uint8_t* to = g.ring + static_cast<size_t>(q) * 2 * plan.stage_bytes;
    const uint32_t bytes = x.template block<false>(t0, rows, to, 0) + grad.template block<false>(t0, rows, to + plan.stage_bytes, 0);
    mbar_arrive_expect_tx(g.bar(q), bytes);
    x.template block<true>(t0, rows, to, g.bar(q));
    grad.template block<true>(t0, rows, to + plan.stage_bytes, g.bar(q));
  };
  if (g.at == 0)
    for (int q = 0; q < plan.stages && g.first + q * g.step < plan.blocks; ++q) issue(g.first + q * g.step, q);
  keep_params<T>(a.weight, a, plan.columns, 1.f, weight);
  __syncthreads();
  // Up to 16 columns a thread keeps the weight and, over the barrier, xhat and
  // weight * grad; with more it takes them once more from shared memory.
  constexpr bool kKeep = E <= 16;
  constexpr int kPairs = C::kPairs, kVectors = C::kVectors;
  float2 dw[kVectors][kPairs], db[kVectors][kPairs];
  float2 xhat[kKeep ? kVectors : 1][kPairs], wg[kKeep ? kVectors : 1][kPairs], w[kKeep ? kVectors : 1][kPairs];
  if (kKeep)
#pragma unroll
    for (int i = 0; i < kVectors; ++i) cols.kept(weight, i, w[i]);
#pragma unroll
  for (int i = 0; i < kVectors; ++i)
#pragma unroll
    for (int e = 0; e < kPairs; ++e) dw[i][e] = db[i][e] = make_float2(0.f, 0.f);
  const float inv = 1.f / a.H;
  int parity = 0;
  auto stat = [&](int64_t t) { return *reinterpret_cast<const float2*>(a.stats + 2 * t); };
  float2 st = {0.f, 0.f};
  if (g.first < plan.blocks) st = stat(static_cast<int64_t>(g.first) * plan.batch);
  for (int block = g.first; block < plan.blocks; block += g.step) {
    g.wait();
    const int rows = rows_of(a, plan, block);
    const int64_t t0 = static_cast<int64_t>(block) * plan.batch;
    const uint8_t* stage = g.ring + static_cast<size_t>(g.s) * 2 * plan.stage_bytes;
    for (int r = 0; r < rows; ++r) {
      const float rstd = st.y + g.poison, mean = st.x;
      const int64_t next = r + 1 < rows ? t0 + r + 1 : static_cast<int64_t>(block + g.step) * plan.batch;
      if (next < a.M) st = stat(next);
      const uint8_t* xs = stage + x.offset(t0, r);
      const uint8_t* gs = stage + plan.stage_bytes + grad.offset(t0, r);
      // xhat and grad of vector i (and, where it is not kept, its weight)
      auto values = [&](int i, float2 (&xh)[kPairs], float2 (&gr)[kPairs]) {
        cols.read(xs, i, xh);
        cols.read(gs, i, gr);
        if (!kKeep) cols.kept(weight, i, w[0]);
#pragma unroll
        for (int e = 0; e < kPairs; ++e) xh[e] = mul2(add2(xh[e], both(-mean)), both(rstd));
      };
      float2 s1 = {0.f, 0.f}, s2 = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < kVectors; ++i) {
        float2 (&xh)[kPairs] = xhat[kKeep ? i : 0];
        float2 (&gr)[kPairs] = wg[kKeep ? i : 0];
        values(i, xh, gr);
#pragma unroll
        for (int e = 0; e < kPairs; ++e) {
          dw[i][e] = fma2(gr[e], xh[e], dw[i][e]);
          db[i][e] = add2(db[i][e], gr[e]);
          gr[e] = mul2(gr[e], w[kKeep ? i : 0][e]);
          s1 = add2(s1, gr[e]);
          s2 = fma2(gr[e], xh[e], s2);
        }
      }
      float p = half_sums(s1.x + s1.y, s2.x + s2.y);
      if (warps > 1) {
        if ((lane & 15) == 0) red[parity][lane >> 4][warp] = p;
        named_bar_sync(1 + g.group, plan.lanes);  // barrier 0 is the whole CTA's
        p = (lane & 15) < warps ? red[parity][lane >> 4][first_warp + (lane & 15)] : 0.f;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) p += __shfl_xor_sync(kFullMask, p, o);
        parity ^= 1;
      }
      const float m1 = __shfl_sync(kFullMask, p, 0) * inv, m2 = __shfl_sync(kFullMask, p, 16) * inv;
      auto refill = [&] {
        const int ahead = block + plan.stages * g.step;
        if (g.at == 0 && ahead < plan.blocks && g.poison == 0.f) issue(ahead, g.s);
        g.advance(plan);
      };
      if (kKeep && r == rows - 1) refill();  // every thread has its values of the last row
      const float c1 = -m1 * rstd, c2 = -m2 * rstd;
      T* out = static_cast<T*>(a.grad_x) + (t0 + r) * a.H;
      if (a.grad_x)
#pragma unroll
        for (int i = 0; i < kVectors; ++i) {
          float2 (&xh)[kPairs] = xhat[kKeep ? i : 0];
          float2 (&gr)[kPairs] = wg[kKeep ? i : 0];
          if (!kKeep) {
            values(i, xh, gr);
#pragma unroll
            for (int e = 0; e < kPairs; ++e) gr[e] = mul2(gr[e], w[0][e]);
          }
          float2 dx[kPairs];
#pragma unroll
          for (int e = 0; e < kPairs; ++e) dx[e] = fma2(xh[e], both(c2), fma2(gr[e], both(rstd), both(c1)));
          cols.write(out, i, dx);
        }
      if (!kKeep && r == rows - 1) {
        if (warps > 1)
          named_bar_sync(1 + g.group, plan.lanes);
        else
          __syncwarp();
        refill();
      }
    }
  }
  g.drain(plan);
  if (!a.grad_weight && !a.grad_bias) return;
  // the groups' sums, one after the other; the rings are free
  float* total = reinterpret_cast<float*>(smem);
  for (int q = 0; q < plan.groups; ++q) {
    __syncthreads();
    if (q != g.group) continue;
#pragma unroll
    for (int i = 0; i < kVectors; ++i)
#pragma unroll
      for (int n = 0; n < C::kWidth; ++n) {
        if (!cols.has(i, n)) continue;
        const int c = cols.column(i, n);
        total[c] = (q ? total[c] : 0.f) + reinterpret_cast<const float*>(dw[i])[n] + g.poison;
        total[a.H + c] = (q ? total[a.H + c] : 0.f) + reinterpret_cast<const float*>(db[i])[n] + g.poison;
      }
  }
  __syncthreads();
  float* part = a.parts + 2ll * blockIdx.x * a.H;
  for (int c = threadIdx.x; c < 2 * a.H; c += blockDim.x) part[c] = total[c];
}

// ---------------------------------------------------------------------------
// rows of any width
// ---------------------------------------------------------------------------
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

// The widest vector that all rows and parameters allow.
template <typename T>
int vector_of(const NormArgs& a, const void* x, const void* y, const void* z) {
  constexpr int kWide = 16 / sizeof(T), kPair = 4 / sizeof(T);
  const uintptr_t rows = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(z) |
                         static_cast<uintptr_t>(a.H * static_cast<int64_t>(sizeof(T))) |
                         static_cast<uintptr_t>(a.M > 1 ? a.stride * static_cast<int64_t>(sizeof(T)) : 0);
  const uintptr_t par = reinterpret_cast<uintptr_t>(a.weight) | reinterpret_cast<uintptr_t>(a.bias);
  if ((rows & 15) == 0 && (par & 15) == 0) return kWide;
  return (rows & 3) == 0 && (par & (a.param_fp32 ? 7 : 3)) == 0 ? kPair : 1;
}

// How a ring kernel takes rows in vectors of N values and `e` columns a thread;
// false where the rows are too wide for it.
template <typename T, int N>
bool make_plan(const NormArgs& a, int e, int together, bool backward, NormPlan& p) {
  const int64_t vectors = (static_cast<int64_t>(a.H) + N - 1) / N, row = static_cast<int64_t>(a.H) * sizeof(T);
  const int64_t lanes = ((vectors + e / N - 1) / (e / N) + 31) / 32 * 32;
  const int parts = backward ? 2 : 1;
  if (lanes > 512) return false;  // at most 16 warps: half a warp adds their sums up
  p.lanes = static_cast<int>(lanes);
  p.groups = std::min(kGroupThreads / p.lanes, p.lanes == 32 ? kGroupWarps : 15);  // a named barrier each
  p.columns = static_cast<uint32_t>(p.lanes * e);  // the threads' columns, those past H too
  const int64_t kept = 4ll * p.columns * (backward ? 1 : 2);
  p.row_pitch = a.stride == a.H || a.M == 1 ? 0 : static_cast<uint32_t>(round_up(row + 15, 16));
  // blocks of about 2 KB and at least `together` rows, fewer where that leaves groups without one
  const int64_t in_ring = p.row_pitch ? p.row_pitch : row;
  p.batch = static_cast<int>(std::max<int64_t>(std::min<int64_t>(std::max<int64_t>(2048 / in_ring, together), a.M / (kSms * p.groups)), 1));
  // a lead of up to 15 bytes, and the last unit to its end
  p.stage_bytes = static_cast<uint32_t>(round_up(p.batch * in_ring + (p.row_pitch || N * sizeof(T) == 16 ? 0 : 30), 128));
  p.stages = static_cast<int>(std::min<int64_t>((kRing - kept) / p.groups / (static_cast<int64_t>(parts) * p.stage_bytes), kStages));
  if (p.stages < 2) return false;
  p.ring_bytes = static_cast<uint32_t>(p.stage_bytes * p.stages * p.groups * parts);
  if (backward) p.ring_bytes = std::max<uint32_t>(p.ring_bytes, static_cast<uint32_t>(round_up(8ll * a.H, 16)));
  if (p.ring_bytes + kept > kRing) return false;
  p.blocks = (a.M + p.batch - 1) / p.batch;
  p.ctas = std::min(p.blocks, kSms);
  return true;
}

template <typename K>
int ring_run(K* kernel, DeviceRecord& record, const NormArgs& a, const NormPlan& p, int kept, cudaStream_t st) {
  const int rc = allow_shared(record, kernel, kRing);
  return rc != MTP_OK ? rc : launch(kernel, dim3(p.ctas), dim3(p.lanes * p.groups), p.ring_bytes + 4ull * kept * p.columns, st, a, p);
}

template <typename T, int N, int E, int R>
int forward_ring(const NormArgs& a, const NormPlan& p, cudaStream_t st) {
  static DeviceRecord record;
  return ring_run(norm_ring_kernel<T, N, E, R>, record, a, p, 2, st);
}
template <typename T, int N, int E>
int backward_ring(const NormArgs& a, const NormPlan& p, cudaStream_t st) {
  static DeviceRecord record;
  return ring_run(norm_backward_kernel<T, N, E>, record, a, p, 1, st);
}

template <typename T, int N>
int forward_run(const NormArgs& a, cudaStream_t st) {
  const int64_t vectors = (static_cast<int64_t>(a.H) + N - 1) / N;
  NormPlan p;
  if (a.M > 2 * kSms) {
    // columns of a thread: few where rows are narrow, and of fp32, whose rows are twice as long
    const int e = a.H > (N == 1 ? 512 : 16 * kGroupThreads) ? 32 : a.H > (sizeof(T) == 4 ? 8 * kGroupThreads : 256) ? 16 : 8;
    if (make_plan<T, N>(a, e, 2, false, p) && p.batch > 1)
      return e == 32 ? forward_ring<T, N, 32, 2>(a, p, st) : e == 16 ? forward_ring<T, N, 16, 2>(a, p, st) : forward_ring<T, N, 8, 2>(a, p, st);
    if (make_plan<T, N>(a, e, 1, false, p))
      return e == 32 ? forward_ring<T, N, 32, 1>(a, p, st) : e == 16 ? forward_ring<T, N, 16, 1>(a, p, st) : forward_ring<T, N, 8, 1>(a, p, st);
  }
  if (vectors > 8 * kRowThreads)
    return launch(a.param_fp32 ? norm_kernel<T, float> : norm_kernel<T, T>, dim3(std::min(a.M, kPlainCtas)), dim3(kThreads), 0, st, a);
  const int lanes = static_cast<int>(std::min<int64_t>((vectors + 31) / 32 * 32, kRowThreads));
  const int nv = static_cast<int>((vectors + lanes - 1) / lanes);
  auto* kernel = nv == 1 ? norm_row_kernel<T, N, 1> : nv <= 4 ? norm_row_kernel<T, N, 4> : norm_row_kernel<T, N, 8>;
  return launch(kernel, dim3(a.M), dim3(lanes), 0, st, a);
}

// One pass over rows and columns; false where the rows are too wide for it.
template <typename T, int N>
bool backward_run(const NormArgs& a, cudaStream_t st, int& rc, int& parts) {
  NormPlan p;
  const int e = a.H <= 8 * kGroupThreads ? 8 : a.H <= 16 * kGroupThreads ? 16 : 32;
  if (!make_plan<T, N>(a, e, 1, true, p)) return false;
  parts = p.ctas;
  rc = e == 8 ? backward_ring<T, N, 8>(a, p, st) : e == 16 ? backward_ring<T, N, 16>(a, p, st) : backward_ring<T, N, 32>(a, p, st);
  return true;
}

template <typename T, typename P>
int finish_run(const NormArgs& a, int parts, cudaStream_t st) {
  return launch(norm_finish_kernel<P>, dim3((a.H + 31) / 32), dim3(kThreads), 0, st, a, parts);
}

template <typename T>
int run(const NormArgs& a, bool backward, cudaStream_t st) {
  constexpr int kWide = 16 / sizeof(T), kPair = 4 / sizeof(T);
  if (!backward) {
    const int n = vector_of<T>(a, a.x, a.y, nullptr);
    return n == kWide ? forward_run<T, kWide>(a, st) : n == 1 ? forward_run<T, 1>(a, st) : forward_run<T, kPair>(a, st);
  }
  int rc = MTP_OK, parts = 0;
  if (a.M) {
    const int n = vector_of<T>(a, a.x, a.grad, a.grad_x);
    const bool fused = n == kWide ? backward_run<T, kWide>(a, st, rc, parts)
                       : n == 1   ? backward_run<T, 1>(a, st, rc, parts)
                                  : backward_run<T, kPair>(a, st, rc, parts);
    if (!fused) {
      if (a.grad_x)
        rc = launch(a.param_fp32 ? norm_rows_backward_kernel<T, float> : norm_rows_backward_kernel<T, T>,
                    dim3(std::min(a.M, kPlainCtas)), dim3(kThreads), 0, st, a);
      parts = std::min(a.M, 64);
      if (rc == MTP_OK && (a.grad_weight || a.grad_bias))
        rc = launch(norm_columns_kernel<T>, dim3((a.H + kThreads - 1) / kThreads, parts), dim3(kThreads), 0, st, a);
    }
  }
  if (rc != MTP_OK || (!a.grad_weight && !a.grad_bias)) return rc;
  return a.param_fp32 ? finish_run<T, float>(a, parts, st) : finish_run<T, T>(a, parts, st);
}

int run(const NormArgs& a, int dtype, bool backward, cudaStream_t st) {
  switch (dtype) {
    case MTP_DTYPE_BF16: return run<__nv_bfloat16>(a, backward, st);
    case MTP_DTYPE_FP16: return run<__half>(a, backward, st);
    default: return run<float>(a, backward, st);
  }
}

}  // namespace

int64_t layer_norm_parts(int M, int H) { return std::min(M, kSms); }
int launch_layer_norm(const NormArgs& a, int dtype, cudaStream_t st) { return run(a, dtype, false, st); }
int launch_layer_norm_backward(const NormArgs& a, int dtype, cudaStream_t st) { return run(a, dtype, true, st); }

}  // namespace mtp
