// The router of a training step: top-k weights with their gradient, the pairs
// of every expert, the balance loss and the z loss.
//
// forward:  p = softmax(z[t]), ids = the k largest (ties: lowest id), w = p[ids],
//           divided by their sum if renormalised. Over the n counted tokens:
//           counts[e] = #{pairs of e}, load[e] = sum_t p[t, e],
//           balance = sum_e pull[e] load[e] with pull[e] = E counts[e] / (k n^2),
//           z_loss = sum_t lse(z[t])^2 / n.
// gradient: with gb, gz of the losses and g of the weights, a[e] = gb pull[e],
//           dz[e] = p[e] (a[e] - sum_i a[i] p[i] + gz 2/n lse)
//                   + (e = ids[j]) w[j] (g[j] - sum_i g[i] w[i])   renormalised;
//           without, g[j] is added to a[ids[j]] instead.
//           counts have no gradient.
//
// A warp takes a token, its logits stay in registers. The sums over tokens go
// warp by warp in registers, then over the warps, then over the CTAs, always in
// the same order; the counts are integers. So results do not depend on timing.
//
// The logits are read once forward and once, with the gradient written,
// backward. Forward the dependent steps of a token bound it (k rounds of maximum
// and vote, ranking in shared memory, exponentials), with 16 warps a SM to hide
// them from 257 experts on: 65536 x 512 logits fill 62 % of the issue slots and a
// quarter of HBM's rate. The gradient is near HBM's (5 TB/s there).
//   8192 x 256, top-8:  16.5 us forward (two launches), 6.3 us backward
//   65536 x 512, top-8: 89 us and 55 us (bytes alone 21 and 41)
//   32768 x 1024, top-8: 71 us and 63 us (21 and 41)
//   one token: 4.1 us and 2.3 us
// More choices, and rows whose logits are all equal, go one by one (see there):
//   8192 x 256, top-16, 20, 24 and 32: 31, 64, 97 and 124 us forward
//   8192 x 1024, top-8, 20 and 32:     28, 318 and 558 us
//   equal logits, 8192 x 256 and 65536 x 512, top-8: 42 us and 540 us
#include "rows.cuh"

#include <math.h>

#include <algorithm>

namespace mtp {
namespace {

constexpr int kFinishCtas = 8;  // one cluster
constexpr int kFinishThreads = 1024;
// Up to here one CTA does all, 4.3 us; two launches take 9.6 (64 tokens).
constexpr int kOneCtaTokens = 16;
constexpr int kSms = 148;
constexpr int kTogether = 19;  // parts of a column that a thread has in flight: all of 148

// Warps of a CTA: a token each as far as the SMs go, then what registers allow.
int loss_warps(int M, int E) {
  return M <= kOneCtaTokens ? kOneCtaTokens : std::max(4, std::min((M - 1) / kSms + 1, E <= 256 ? 32 : 16));
}

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// Whether the lane's i-th expert is one; FULL: E is 32 VPT.
template <bool FULL>
__device__ __forceinline__ bool has(const RouteLossArgs& a, int lane, int i) {
  return FULL || lane + 32 * i < a.E;
}

template <bool FULL, typename T, int VPT>
__device__ __forceinline__ void load_row(const RouteLossArgs& a, int t, int lane, float (&v)[VPT]) {
  const T* row = static_cast<const T*>(a.logits) + t * a.stride + lane;
#pragma unroll
  for (int i = 0; i < VPT; ++i) v[i] = has<FULL>(a, lane, i) ? as_float(row[32 * i]) : -INFINITY;
}

template <int VPT>
__device__ __forceinline__ float row_max(const float (&v)[VPT]) {
  float mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < VPT; ++i) mx = fmaxf(mx, v[i]);
  return warp_max(mx);
}

// exp(v) by one instruction, for v = z - max of a row. Subtracted before it is
// scaled: max log2(e) rounded by itself is a factor that the row's values share,
// but from |max| of 2e9 on one that no number of fp32 holds. v is 0 at the
// maximum. The argument is rounded twice, an error of |v| 2^-23 of the result.
__device__ __forceinline__ float fast_exp(float v) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(v * 1.44269504f));
  return e;
}

// v -> exp(v - max) (0 past the last expert); returns max and sum. The forward
// pass has the exponential of mtp_router_topk, so that both give the same bits.
// FAST: fast_exp.
template <bool FULL, bool FAST, int VPT>
__device__ __forceinline__ float2 softmax_row(const RouteLossArgs& a, int lane, float (&v)[VPT], float mx) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const float e = FAST ? fast_exp(v[i] - mx) : expf(v[i] - mx);
    v[i] = has<FULL>(a, lane, i) ? e : 0.f;
    s += v[i];
  }
  return make_float2(mx, warp_sum(s));
}

__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
  return v;
}

// pull[e] of an expert, 0 without counted tokens.
__device__ __forceinline__ float pull_of(const RouteLossArgs& a, int count, double n) {
  return n > 0 ? static_cast<float>(static_cast<double>(a.E) * count / (static_cast<double>(a.k) * n * n)) : 0.f;
}

// Integers that order like numbers do (0 below all of them, NaN below -inf).
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t bits = __float_as_uint(v == 0.f ? 0.f : v);  // -0 ties with 0
  return v != v ? 1u : bits >> 31 ? ~bits : bits | 0x80000000u;
}

// What a warp's chosen experts give: lane j has the j-th, wsum is their
// probabilities' sum in this order.
__device__ __forceinline__ void write_choice(const RouteLossArgs& a, float p, int id, float wsum, int64_t o, int* hist) {
  if (a.renorm) p = p / fmaxf(wsum, 1e-20f);
  if ((threadIdx.x & 31) < a.k) {
    a.weights[o] = p;
    a.ids[o] = id;
    atomicAdd(&hist[id], 1);
  }
}

// The k largest, one after the other: a maximum over the warp each. For the rows
// that choose() does not take: those with a NaN, without k finite logits, or with
// more than 32 candidates. Of normal logits of 256 experts the last are none for
// k = 8, 0.1 % for 16, 15 % for 20, 92 % for 24 and all for 32 (1024 experts and
// k = 20: 26 %); rows of more than 32 equal logits are too. It keeps no registers
// and reads the row again k times.
template <typename T>
__device__ __forceinline__ void choose_one_by_one(const RouteLossArgs& a, int t, float2 ms, int64_t o, int* hist) {
  const int lane = threadIdx.x & 31;
  const T* row = static_cast<const T*>(a.logits) + t * a.stride;
  uint32_t taken = 0;  // of this lane's experts
  float my_p = 0.f, wsum = 0.f;
  int my_id = 0;
#pragma unroll 1
  for (int j = 0; j < a.k; ++j) {
    uint32_t best = 0;
    int at = 0;
#pragma unroll 1
    for (int i = 0; lane + 32 * i < a.E; ++i) {
      const uint32_t key = taken >> i & 1 ? 0u : order_key(as_float(row[lane + 32 * i]));
      if (key > best) best = key, at = i;
    }
    const uint32_t top = __reduce_max_sync(kFullMask, best);
    const int id = __reduce_min_sync(kFullMask, best == top ? static_cast<unsigned>(lane + 32 * at) : 0xffffu);
    if (lane == (id & 31)) taken |= 1u << (id >> 5);
    const float p = expf(as_float(row[id]) - ms.x) / ms.y;
    wsum += p;
    if (lane == j) {
      my_p = p;
      my_id = id;
    }
  }
  write_choice(a, my_p, my_id, wsum, o, hist);
}

struct Chosen {
  struct alignas(8) {
    float z;
    int id;
  } at[32];
};

// The same with less work: the k-th largest of the lanes' own maxima is no more
// than the k-th largest of all, so that few values (the k, and those that share
// a lane with one of them) are left to rank. Gives their number, 0 where they
// are more than 32 or there is no finite one.
// 65536 tokens of 512 experts, top-8: 195 us one by one, 127 us so.
template <int VPT>
__device__ __forceinline__ int candidates(const RouteLossArgs& a, const float (&z)[VPT], float best, Chosen& c) {
  const int lane = threadIdx.x & 31;
  uint32_t mine = lane < a.E ? order_key(best) : 0u, least = 0;
  for (int j = 0; j < a.k; ++j) {
    least = __reduce_max_sync(kFullMask, mine);
    const unsigned at = __ballot_sync(kFullMask, mine == least);
    if (lane == __ffs(at) - 1) mine = 0;
  }
  // the number of that order
  const float bound = __uint_as_float(least >> 31 ? least & 0x7fffffffu : ~least);
  if (!(bound > -INFINITY)) return 0;
  int n = 0;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const bool in = z[i] >= bound;  // -inf past the last expert
    const unsigned votes = __ballot_sync(kFullMask, in);
    if (votes == 0) continue;
    const int at = n + __popc(votes & ((1u << lane) - 1u));
    if (in && at < 32) {
      c.at[at].z = z[i];
      c.at[at].id = lane + 32 * i;
    }
    n += __popc(votes);
  }
  return n <= 32 ? n : 0;
}

__device__ __forceinline__ void choose(const RouteLossArgs& a, int n, float2 ms, int64_t o, Chosen& c, int* hist) {
  const int lane = threadIdx.x & 31;
  __syncwarp();
  const auto mine = c.at[lane];  // of a lane below n
  int rank = 0;
#pragma unroll 4
  for (int x = 0; x < n; ++x) {
    const auto other = c.at[x];
    rank += other.z > mine.z || (other.z == mine.z && other.id < mine.id);
  }
  __syncwarp();
  if (lane < n && rank < a.k) {
    c.at[rank].z = expf(mine.z - ms.x) / ms.y;
    c.at[rank].id = mine.id;
  }
  __syncwarp();
  float wsum = 0.f;
  for (int j = 0; j < a.k; ++j) wsum += c.at[j].z;
  write_choice(a, c.at[lane].z, c.at[lane].id, wsum, o, hist);
  __syncwarp();
}


template <typename T, int VPT, bool FULL>
__global__ void __launch_bounds__(VPT <= 8 ? 1024 : 512, 1) route_loss_kernel(const RouteLossArgs a) {
  extern __shared__ __align__(16) float sm[];  // [warps][E] loads, then [E] counts
  __shared__ double red[32][2];
  __shared__ Chosen chosen[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
  int* hist = reinterpret_cast<int*>(sm + warps * a.E);
  for (int e = tid; e < a.E; e += blockDim.x) hist[e] = 0;
  pdl_launch_dependents();
  pdl_wait();
  __syncthreads();
  float load[VPT], squares = 0.f;
  int tokens = 0;
#pragma unroll
  for (int i = 0; i < VPT; ++i) load[i] = 0.f;
  const int step = gridDim.x * warps;
  float ahead[VPT];  // the next token's logits, on their way while this one's are ranked
  int t = blockIdx.x * warps + warp;
  if (t < a.M) load_row<FULL, T>(a, t, lane, ahead);
  for (; t < a.M; t += step) {
    const int64_t o = static_cast<int64_t>(t) * a.k + lane;
    float v[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) v[i] = ahead[i];
    if (t + step < a.M) load_row<FULL, T>(a, t + step, lane, ahead);
    if (a.mask && !a.mask[t]) {
      if (lane < a.k) {
        a.weights[o] = 0.f;
        a.ids[o] = -1;
      }
      continue;
    }
    float best = -INFINITY;  // of this lane
#pragma unroll
    for (int i = 0; i < VPT; ++i) best = fmaxf(best, v[i]);
    const int n = candidates<VPT>(a, v, best, chosen[warp]);
    const float2 ms = softmax_row<FULL, false>(a, lane, v, warp_max(best));
    if (n && ms.y < INFINITY)  // no NaN among them
      choose(a, n, ms, o, chosen[warp], hist);
    else
      choose_one_by_one<T>(a, t, ms, o, hist);
    const float inv = 1.f / ms.y;
#pragma unroll
    for (int i = 0; i < VPT; ++i) load[i] = fmaf(v[i], inv, load[i]);
    const float lse = ms.x + logf(ms.y);
    squares = fmaf(lse, lse, squares);
    ++tokens;
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i)
    if (lane + 32 * i < a.E) sm[warp * a.E + lane + 32 * i] = load[i];
  if (lane == 0) {
    red[warp][0] = squares;
    red[warp][1] = tokens;
  }
  __syncthreads();
  double squares_all = 0, n_all = 0;
  for (int w = 0; w < warps; ++w) {
    squares_all += red[w][0];
    n_all += red[w][1];
  }
  if (gridDim.x > 1) {  // route_finish_kernel sums over the CTAs
    for (int e = tid; e < a.E; e += blockDim.x) {
      float s = 0.f;
      for (int w = 0; w < warps; ++w) s += sm[w * a.E + e];
      a.part_load[static_cast<int64_t>(blockIdx.x) * a.E + e] = s;
      a.part_count[static_cast<int64_t>(blockIdx.x) * a.E + e] = hist[e];
    }
    if (tid == 0) {
      a.part_sums[2 * blockIdx.x] = squares_all;
      a.part_sums[2 * blockIdx.x + 1] = n_all;
    }
    return;
  }
  double balance = 0;
  for (int e = tid; e < a.E; e += blockDim.x) {
    float s = 0.f;
    for (int w = 0; w < warps; ++w) s += sm[w * a.E + e];
    const float pull = pull_of(a, hist[e], n_all);
    balance += static_cast<double>(pull) * s;
    a.counts[e] = hist[e];
    if (a.pull) a.pull[e] = pull;
  }
  balance = warp_sum64(balance);
  __syncthreads();
  if (lane == 0) red[warp][0] = balance;
  __syncthreads();
  if (tid == 0) {
    balance = 0;
    for (int w = 0; w < warps; ++w) balance += red[w][0];
    *a.balance = static_cast<float>(balance);
    *a.z_loss = n_all > 0 ? static_cast<float>(squares_all / n_all) : 0.f;
    if (a.pull) a.pull[a.E] = n_all > 0 ? static_cast<float>(2. / n_all) : 0.f;
  }
}

// The sums over the CTAs of route_loss_kernel: CTA r takes the experts
// [128 r, 128 r + 128), eight threads each.
__global__ void __cluster_dims__(kFinishCtas, 1, 1) __launch_bounds__(kFinishThreads, 1)
    route_finish_kernel(const RouteLossArgs a, int parts) {
  __shared__ float loads[8][128];
  __shared__ int counts[8][128];
  __shared__ double sums[32][2];
  __shared__ double balances[kFinishCtas];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = blockIdx.x;
  const int col = tid & 127, row = tid >> 7, e = rank * 128 + col;
  asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");  // this CTA runs: its shared memory may be written
  pdl_launch_dependents();
  pdl_wait();
  float load = 0.f;
  int count = 0;
  if (e < a.E)
    for (int g0 = row; g0 < parts; g0 += 8 * kTogether) {
      float l[kTogether];
      int n[kTogether];
#pragma unroll
      for (int x = 0; x < kTogether; ++x) {
        const int64_t at = static_cast<int64_t>(g0 + 8 * x) * a.E + e;
        const bool in = g0 + 8 * x < parts;
        l[x] = in ? a.part_load[at] : 0.f;
        n[x] = in ? a.part_count[at] : 0;
      }
#pragma unroll
      for (int x = 0; x < kTogether; ++x) {
        load += l[x];
        count += n[x];
      }
    }
  loads[row][col] = load;
  counts[row][col] = count;
  double squares = 0, n = 0;
  for (int g = tid; g < parts; g += kFinishThreads) {
    squares += a.part_sums[2 * g];
    n += a.part_sums[2 * g + 1];
  }
  squares = warp_sum64(squares);
  n = warp_sum64(n);
  if (lane == 0) {
    sums[warp][0] = squares;
    sums[warp][1] = n;
  }
  __syncthreads();
  squares = n = 0;
  for (int w = 0; w < 32; ++w) {
    squares += sums[w][0];
    n += sums[w][1];
  }
  double balance = 0;
  if (tid < 128 && e < a.E) {
    load = 0.f;
    count = 0;
    for (int r = 0; r < 8; ++r) {
      load += loads[r][col];
      count += counts[r][col];
    }
    const float pull = pull_of(a, count, n);
    balance = static_cast<double>(pull) * load;
    a.counts[e] = count;
    if (a.pull) a.pull[e] = pull;
  }
  __syncthreads();
  balance = warp_sum64(balance);
  if (lane == 0) sums[warp][0] = balance;
  __syncthreads();
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  if (tid == 0) {
    balance = sums[0][0] + sums[1][0] + sums[2][0] + sums[3][0];
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(remote) : "r"(smem_u32(&balances[rank])));
    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(remote), "d"(balance) : "memory");
  }
  asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
  if (rank == 0 && tid == 0) {
    balance = 0;
    for (int r = 0; r < kFinishCtas; ++r) balance += balances[r];
    *a.balance = static_cast<float>(balance);
    *a.z_loss = n > 0 ? static_cast<float>(squares / n) : 0.f;
    if (a.pull) a.pull[a.E] = n > 0 ? static_cast<float>(2. / n) : 0.f;
  }
}

template <typename T>
__device__ __forceinline__ T rounded(float v) {
  Vec<T, 1> o;
  from_floats(&v, o);
  return o.v[0];
}

template <typename T, int VPT, bool FULL>
__global__ void __launch_bounds__(256) route_backward_kernel(const RouteLossArgs a) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  pdl_launch_dependents();
  pdl_wait();
  const float gb = a.grad_balance ? *a.grad_balance : 0.f;
  const float cz = a.grad_z_loss ? *a.grad_z_loss * a.pull[a.E] : 0.f;
  float pull[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) pull[i] = a.grad_balance && has<FULL>(a, lane, i) ? gb * a.pull[lane + 32 * i] : 0.f;
  for (int t = blockIdx.x * warps + warp; t < a.M; t += gridDim.x * warps) {
    T* out = static_cast<T*>(a.grad_logits) + static_cast<int64_t>(t) * a.E;
    if (a.mask && !a.mask[t]) {
#pragma unroll
      for (int i = 0; i < VPT; ++i)
        if (has<FULL>(a, lane, i)) out[lane + 32 * i] = rounded<T>(0.f);
      continue;
    }
    float v[VPT];
    load_row<FULL, T>(a, t, lane, v);
    int id = -1;
    float g = 0.f, zj = 0.f;
    if (a.grad_weights && lane < a.k) {
      const int64_t o = static_cast<int64_t>(t) * a.k + lane;
      id = a.ids_in[o];
      g = a.grad_weights[o];
      if (id < 0 || id >= a.E) id = -1;
      if (id >= 0) zj = as_float((static_cast<const T*>(a.logits) + t * a.stride)[id]);
    }
    const float2 ms = softmax_row<FULL, true>(a, lane, v, row_max(v));
    const float inv = 1.f / ms.y;
    float mean = 0.f;  // sum_i a[i] p[i]
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      v[i] *= inv;
      mean = fmaf(pull[i], v[i], mean);
    }
    float direct = 0.f, pj = 0.f;
    if (a.grad_weights) {
      pj = id >= 0 ? fast_exp(zj - ms.x) * inv : 0.f;
      if (a.renorm) {
        const float w = pj / fmaxf(warp_sum(pj), 1e-20f);
        const float wg = id >= 0 ? w * g : 0.f;
        direct = w * (g - warp_sum(wg));
      } else {
        direct = id >= 0 ? pj * g : 0.f;
        mean += direct;
      }
    }
    mean = warp_sum(mean);
    const float shift = (a.grad_z_loss ? cz * (ms.x + logf(ms.y)) : 0.f) - mean;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (has<FULL>(a, lane, i)) out[lane + 32 * i] = rounded<T>(v[i] * (pull[i] + shift));
    if (a.grad_weights) {
      __syncwarp();  // the chosen experts' entries once more, over the row's
      if (id >= 0) out[id] = rounded<T>(fmaf(pj, (a.grad_balance ? gb * a.pull[id] : 0.f) + shift, direct));
    }
  }
}

}  // namespace

// CTAs of route_loss_kernel whose sums route_finish_kernel takes, 0: none.
int64_t route_loss_parts(int M, int E) {
  if (M <= kOneCtaTokens) return 0;
  const int warps = loss_warps(M, E);
  return std::min<int64_t>((static_cast<int64_t>(M) + warps - 1) / warps, kSms);
}

namespace {

template <typename T, int VPT, bool FULL>
int forward_run(const RouteLossArgs& a, cudaStream_t st) {
  const int threads = 32 * loss_warps(a.M, a.E), ctas = static_cast<int>(std::max<int64_t>(route_loss_parts(a.M, a.E), 1));
  const size_t smem = static_cast<size_t>(threads / 32 + 1) * a.E * sizeof(float);
  static DeviceRecord record;
  const int allowed = allow_shared(record, route_loss_kernel<T, VPT, FULL>, static_cast<size_t>(VPT <= 8 ? 33 : 17) * 32 * VPT * sizeof(float));
  if (allowed != MTP_OK) return allowed;
  const int rc = launch(route_loss_kernel<T, VPT, FULL>, dim3(ctas), dim3(threads), smem, st, a);
  if (rc != MTP_OK || ctas == 1) return rc;
  return launch(route_finish_kernel, dim3(kFinishCtas), dim3(kFinishThreads), 0, st, a, ctas);
}

template <typename T, int VPT, bool FULL>
int backward_run(const RouteLossArgs& a, cudaStream_t st) {
  return launch(route_backward_kernel<T, VPT, FULL>, dim3(std::min((a.M + 7) / 8, 8 * kSms)), dim3(256), 0, st, a);
}

template <typename T>
int run(const RouteLossArgs& a, bool backward, cudaStream_t st) {
  const int vpt = (a.E + 31) / 32;
#define MTP_RUN(n, full) (backward ? backward_run<T, n, full>(a, st) : forward_run<T, n, full>(a, st))
#define MTP_VPT(n) \
  if (vpt <= n) return a.E == 32 * n ? MTP_RUN(n, true) : MTP_RUN(n, false);
  MTP_VPT(1) MTP_VPT(2) MTP_VPT(4) MTP_VPT(8) MTP_VPT(16)
#undef MTP_VPT
  return a.E == 1024 ? MTP_RUN(32, true) : MTP_RUN(32, false);
#undef MTP_RUN
}

int run(const RouteLossArgs& a, int dtype, bool backward, cudaStream_t st) {
  switch (dtype) {
    case MTP_DTYPE_BF16: return run<__nv_bfloat16>(a, backward, st);
    case MTP_DTYPE_FP16: return run<__half>(a, backward, st);
    default: return run<float>(a, backward, st);
  }
}

}  // namespace

int launch_route_loss(const RouteLossArgs& a, int dtype, cudaStream_t st) { return run(a, dtype, false, st); }
int launch_route_loss_backward(const RouteLossArgs& a, int dtype, cudaStream_t st) { return run(a, dtype, true, st); }

}  // namespace mtp
