// Tokens sorted by expert, and back with the routing weights applied.
//
// sort:    the pairs (t, j) of a token and its j-th choice get the key
//          expert_map[topk_ids[t, j]] (or the id itself), E where that is no
//          expert of this rank. Row p(t, j) = #{pairs of a smaller key} +
//          #{earlier pairs of the same key}: a stable sort, so the result
//          does not depend on scheduling. rows[p(t, j)] = x[t]; pairs without
//          an expert come last and their rows are zero. positions holds p,
//          or ~p (negative) for a pair without an expert, so every pair knows
//          the one row that is its own. offsets[e] = #{pairs of a key < e}.
// unsort:  out[t] = sum over the routed j, ascending, of w[t, j] * rows[p(t, j)]
//          (w = 1 without weights: the gradient of the sort), in fp32, rounded
//          once.
// its gradient: grad_rows[p(t, j)] = w[t, j] * g[t], zero rows for unrouted
//          pairs, grad_w[t, j] = <g[t], rows[p(t, j)]> in fp32.
//
// All three move rows and are bound by HBM; the ranking is integer counting.
// 8192 tokens x 8 x 2048 bf16: ranks 12 us, rows copied in 46 us (6.5 TB/s),
// unsort 48.7 us (6.2 TB/s), its gradients 96 us (5.9 TB/s); one token 2.6 us.
#include "internal.cuh"
#include "route.cuh"
#include "rows.cuh"

#include <algorithm>

namespace mtp {
namespace {

constexpr int kRankCtas = 8;        // one cluster ranks all pairs of a large call
constexpr int kRankThreads = 1024;
constexpr int kRankWarps = kRankThreads / 32;
// Up to this many pairs every CTA of the copy ranks its own token's pairs by
// counting over all keys in shared memory (one launch); above, a cluster ranks
// all pairs first (8 x 2048 bf16: 384 tokens 8.5 us, 512 tokens 11.1 in one
// launch against 9.4 in two).
constexpr int kSmallPairs = 3328;  // at most 4096: 12 bits
constexpr int kSmallThreads = 256;

__device__ __forceinline__ int sort_key(const SortArgs& a, int i) {
  int id = a.ids[i];
  if (a.emap) id = id >= 0 && id < a.E_map ? a.emap[id] : -1;
  return id >= 0 && id < a.E ? id : a.E;
}

template <typename V>
__device__ __forceinline__ V zero_of() {
  V v;
  memset(&v, 0, sizeof(V));
  return v;
}

// Row t of x to its k rows (zeros where the position is negative). `lane` of
// `lanes` threads take the row's vectors in turn.
template <typename V>
__device__ __forceinline__ void copy_row(const SortArgs& a, int t, const int* pos, int lane, int lanes) {
  const V* src = reinterpret_cast<const V*>(a.x + static_cast<int64_t>(t) * a.x_stride);
  const int n = static_cast<int>(a.row_bytes / sizeof(V));
  for (int c = lane; c < n; c += lanes) {
    const V v = src[c];
    for (int j = 0; j < a.k; ++j) {
      const int p = pos[j];
      V* dst = reinterpret_cast<V*>(a.rows + static_cast<int64_t>(p >= 0 ? p : ~p) * a.row_bytes);
      dst[c] = p >= 0 ? v : zero_of<V>();
    }
  }
  if (a.row_scales)
    for (int j = lane; j < a.k; j += lanes) {
      const int p = pos[j];
      a.sorted_scales[p >= 0 ? p : ~p] = p >= 0 ? a.row_scales[t] : 0.f;
    }
}

// ---------------------------------------------------------------------------
// one launch: CTA t ranks the pairs of token t and copies its row
// ---------------------------------------------------------------------------
template <typename V>
__global__ void __launch_bounds__(kSmallThreads) sort_small_kernel(const SortArgs a) {
  // key << 12 | pair of every pair, so that one comparison orders both, up to a
  // multiple of 128 with values above all; then the token's k positions
  extern __shared__ __align__(16) int keys[];
  const int padded = (a.numel + 127) / 128 * 128;
  int* pos = keys + padded;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
  pdl_launch_dependents();
  pdl_wait();
  for (int i = tid; i < padded; i += blockDim.x) keys[i] = i < a.numel ? sort_key(a, i) << 12 | i : INT_MAX;
  __syncthreads();
  auto below = [&](int bound) {  // pairs below bound, by a warp
    int n = 0;
    for (int q = 4 * lane; q < padded; q += 128) {
      const int4 v = *reinterpret_cast<const int4*>(keys + q);
      n += v.x < bound;
      n += v.y < bound;
      n += v.z < bound;
      n += v.w < bound;
    }
    return __reduce_add_sync(kFullMask, n);
  };
  const int t = blockIdx.x;
  if (t < a.M) {
    for (int j = warp; j < a.k; j += warps) {
      const int i = t * a.k + j, before = below(keys[i]);
      if (lane == 0) {
        const int p = keys[i] >> 12 < a.E ? before : ~before;
        pos[j] = p;
        a.positions[i] = p;
      }
    }
  }
  // offsets: entry e belongs to CTA e % gridDim; a thread each where the CTA
  // has many, a warp each where it has few
  const int mine = (a.E + 1 - t + gridDim.x - 1) / static_cast<int>(gridDim.x);
  if (mine > 2 * warps || a.numel <= 64) {
    for (int e = t + tid * gridDim.x; e <= a.E; e += blockDim.x * gridDim.x) {
      int before = 0;
      for (int q = 0; q < a.numel; ++q) before += keys[q] < e << 12 ? 1 : 0;
      a.offsets[e] = before;
    }
  } else {
    for (int e = t + warp * gridDim.x; e <= a.E; e += warps * gridDim.x) {
      const int before = below(e << 12);
      if (lane == 0) a.offsets[e] = before;
    }
  }
  __syncthreads();
  if (t < a.M) copy_row<V>(a, t, pos, tid, blockDim.x);
}

// ---------------------------------------------------------------------------
// large calls: ranks from one cluster, then the copy
// ---------------------------------------------------------------------------
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ int ld_cluster(uint32_t local, int cta) {
  uint32_t remote;
  int v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(cta));
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(remote));
  return v;
}

// The lanes whose key (below 2^bits) is this lane's: a vote per bit. match.any
// gives the same at about 200 cycles a warp, which made it most of this kernel.
__device__ __forceinline__ unsigned same_key(int key, int bits) {
  unsigned same = kFullMask;
#pragma unroll
  for (int b = 0; b < 11; ++b) {  // keys go up to 1025
    if (b >= bits) break;
    const bool one = (key & (1 << b)) != 0;
    const unsigned votes = __ballot_sync(kFullMask, one);
    same &= one ? votes : ~votes;
  }
  return same;
}

// Keys of a CTA that stay in shared memory between its two walks.
constexpr int kRankKeep = 16384;

inline size_t rank_smem(int E) {
  return (static_cast<size_t>(kRankWarps + 2) * (E + 1) + kRankKeep) * sizeof(int);
}

// Every warp of the cluster takes one contiguous range of the pairs and walks
// it twice: first it counts its pairs of every key, then, with the counts of
// the ranges before its own summed (over the warps of the CTA in shared memory,
// over the CTAs through distributed shared memory), it numbers them. The loops
// stay rolled: a launch this short runs each instruction from a cold cache, and
// unrolling them by 16 made the first walk 7000 cycles longer.
__global__ void __cluster_dims__(kRankCtas, 1, 1) __launch_bounds__(kRankThreads, 1) sort_rank_kernel(const SortArgs a) {
  extern __shared__ int sm[];
  __shared__ int scan_tmp[32];
  const int bins = a.E + 1;
  int* wcnt = sm;                       // [warps][bins]
  int* tot = sm + kRankWarps * bins;    // [bins] this CTA's pairs of every key
  int* base = tot + bins;               // [bins] first row of this CTA's pairs of a key
  int* kept = base + bins;              // [kRankKeep] key | rank in its round << 16 | equal keys << 24
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, cta = blockIdx.x;
  for (int x = tid; x < kRankWarps * bins; x += kRankThreads) wcnt[x] = 0;
  pdl_launch_dependents();
  pdl_wait();
  __syncthreads();
  const int64_t parts = kRankCtas * kRankWarps;
  const int64_t span = (a.numel + parts * 32 - 1) / (parts * 32) * 32;
  const int64_t begin = (static_cast<int64_t>(cta) * kRankWarps + warp) * span;
  const int64_t end = min(begin + span, static_cast<int64_t>(a.numel));
  int* mine = wcnt + warp * bins;
  const int bits = 32 - __clz(bins);
  const bool keep = span * kRankWarps <= kRankKeep;
  if (keep) {
    const int64_t first = static_cast<int64_t>(cta) * kRankWarps * span;
#pragma unroll 4
    for (int x = tid; x < span * kRankWarps; x += kRankThreads)
      kept[x] = first + x < a.numel ? sort_key(a, static_cast<int>(first + x)) : bins;
    __syncthreads();
  }
  int* own = kept + warp * static_cast<int>(keep ? span : 0) + lane;
  // this lane's pair of round r: its key, rank among the round's equal keys, and their number
  auto ranked = [&](int r) {
    const int64_t i = begin + r * 32 + lane;
    const int key = keep ? own[r * 32] : i < end ? sort_key(a, static_cast<int>(i)) : bins;
    const unsigned same = same_key(key, bits);
    return key | __popc(same & ((1u << lane) - 1u)) << 16 | __popc(same) << 24;
  };
  const int rounds = static_cast<int>((max(end - begin, static_cast<int64_t>(0)) + 31) / 32);
#pragma unroll 1
  for (int r = 0; r < rounds; ++r) {
    const int x = ranked(r), k = x & 0xffff;
    if (keep) own[r * 32] = x;
    if (k < bins && (x >> 16 & 0xff) == 0) mine[k] += x >> 24;
    __syncwarp();
  }
  __syncthreads();
  for (int b = tid; b < bins; b += kRankThreads) {
    int v[kRankWarps], run = 0;
#pragma unroll
    for (int w = 0; w < kRankWarps; ++w) v[w] = wcnt[w * bins + b];
#pragma unroll
    for (int w = 0; w < kRankWarps; ++w) {
      wcnt[w * bins + b] = run;
      run += v[w];
    }
    tot[b] = run;
  }
  cluster_sync_all();
  int all = 0, before = 0;
  if (tid < a.E) {
    int v[kRankCtas];
#pragma unroll
    for (int r = 0; r < kRankCtas; ++r) v[r] = ld_cluster(smem_u32(tot + tid), r);
#pragma unroll
    for (int r = 0; r < kRankCtas; ++r) {
      before += r < cta ? v[r] : 0;
      all += v[r];
    }
  }
  int routed;
  const int off = block_exclusive_scan(all, &routed, scan_tmp);
  if (tid < a.E) {
    base[tid] = off + before;
    if (cta == 0) a.offsets[tid] = off;
  }
  if (tid == 0) {
    if (cta == 0) a.offsets[a.E] = routed;
    int unrouted = 0;
    for (int r = 0; r < cta; ++r) unrouted += ld_cluster(smem_u32(tot + a.E), r);
    base[a.E] = routed + unrouted;
  }
  cluster_sync_all();  // also: no CTA leaves while another reads its counts
#pragma unroll 1
  for (int r = 0; r < rounds; ++r) {
    const int x = keep ? own[r * 32] : ranked(r), k = x & 0xffff, rank = x >> 16 & 0xff;
    int p = 0;
    if (k < bins) p = base[k] + mine[k] + rank;
    __syncwarp();
    if (k < bins) {
      a.positions[begin + r * 32 + lane] = k < a.E ? p : ~p;
      if (rank == 0) mine[k] += x >> 24;
    }
    __syncwarp();
  }
}

// blockDim (lanes of a row, tokens of a CTA)
template <typename V>
__global__ void __launch_bounds__(256) sort_copy_kernel(const SortArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int64_t t = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  if (t >= a.M) return;
  copy_row<V>(a, static_cast<int>(t), a.positions + t * a.k, threadIdx.x, blockDim.x);
}

// ---------------------------------------------------------------------------
// unsort
// ---------------------------------------------------------------------------
constexpr int kSlots = 8;  // slots whose rows a thread has in flight together

// T: the rows' type, O: the result's.
template <typename T, typename O, int N>
__global__ void __launch_bounds__(256) unsort_kernel(const UnsortArgs a) {
  using V = Vec<T, N>;
  // The next kernel only after the wait: launched before it, its CTAs (and those
  // of the kernels behind it) take their places while the producer of the rows
  // still runs. The W8A8 layer of 16 tokens 71.2 -> 66.6 us, sort and unsort of
  // 64 tokens x 8 x 2048 bf16 7.4 -> 5.2 (unsort alone, 256 tokens: 2.4 -> 2.6).
  pdl_wait();
  pdl_launch_dependents();
  const int64_t t = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  if (t >= a.M) return;
  const int32_t* pos = a.positions + t * a.k;
  const float* wt = a.weights ? a.weights + t * a.k : nullptr;
  const T* rows = static_cast<const T*>(a.rows);
  O* out = static_cast<O*>(a.out) + t * a.H;
  for (int c = (blockIdx.y * blockDim.x + threadIdx.x) * N; c < a.H; c += gridDim.y * blockDim.x * N) {
    float acc[N];
#pragma unroll
    for (int n = 0; n < N; ++n) acc[n] = 0.f;
    for (int j0 = 0; j0 < a.k; j0 += kSlots) {
      V v[kSlots];
      float w[kSlots];
      bool here[kSlots];
#pragma unroll
      for (int j = 0; j < kSlots; ++j) {
        const int p = j0 + j < a.k ? pos[j0 + j] : -1;
        here[j] = p >= 0 && p < a.num_rows;
        w[j] = here[j] && wt ? wt[j0 + j] : 1.f;
        if (here[j]) v[j] = *reinterpret_cast<const V*>(rows + static_cast<int64_t>(p) * a.H + c);
      }
#pragma unroll
      for (int j = 0; j < kSlots; ++j)
        if (here[j]) {
          float f[N];
          to_floats(v[j], f);
#pragma unroll
          for (int n = 0; n < N; ++n) acc[n] = fmaf(w[j], f[n], acc[n]);
        }
    }
    Vec<O, N> o;
    from_floats(acc, o);
    *reinterpret_cast<Vec<O, N>*>(out + c) = o;
  }
}

// blockDim.x is a multiple of 32: the lanes of a token are whole warps.
template <typename T, int N>
__global__ void __launch_bounds__(256) unsort_backward_kernel(const UnsortArgs a) {
  using V = Vec<T, N>;
  __shared__ float red[8][kSlots];
  pdl_launch_dependents();
  pdl_wait();
  const int64_t t = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  const bool in = t < a.M;
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int32_t* pos = a.positions + t * a.k;
  const float* wt = a.weights ? a.weights + t * a.k : nullptr;
  const T* g = static_cast<const T*>(a.grad) + t * a.H;
  const T* rows = static_cast<const T*>(a.rows);
  T* grows = static_cast<T*>(a.grad_rows);
  for (int j0 = 0; j0 < a.k; j0 += kSlots) {
    float dot[kSlots], w[kSlots];
    int p[kSlots];
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      dot[j] = 0.f;
      const bool slot = in && j0 + j < a.k;
      p[j] = slot ? pos[j0 + j] : INT_MIN;  // ~INT_MIN is past every row
      w[j] = slot && wt && p[j] >= 0 ? wt[j0 + j] : 1.f;
    }
    if (in)
      for (int c = threadIdx.x * N; c < a.H; c += blockDim.x * N) {
        float gf[N];
        to_floats(*reinterpret_cast<const V*>(g + c), gf);
        V v[kSlots];
        if (a.grad_weights) {
#pragma unroll
          for (int j = 0; j < kSlots; ++j)
            if (p[j] >= 0 && p[j] < a.num_rows)
              v[j] = *reinterpret_cast<const V*>(rows + static_cast<int64_t>(p[j]) * a.H + c);
#pragma unroll
          for (int j = 0; j < kSlots; ++j)
            if (p[j] >= 0 && p[j] < a.num_rows) {
              float f[N];
              to_floats(v[j], f);
#pragma unroll
              for (int n = 0; n < N; ++n) dot[j] = fmaf(gf[n], f[n], dot[j]);
            }
        }
        if (grows)
#pragma unroll
          for (int j = 0; j < kSlots; ++j) {
            const int r = p[j] >= 0 ? p[j] : ~p[j];
            if (r >= a.num_rows) continue;
            float f[N];
#pragma unroll
            for (int n = 0; n < N; ++n) f[n] = p[j] >= 0 ? w[j] * gf[n] : 0.f;
            V o;
            from_floats(f, o);
            *reinterpret_cast<V*>(grows + static_cast<int64_t>(r) * a.H + c) = o;
          }
      }
    if (a.grad_weights) {
#pragma unroll
      for (int j = 0; j < kSlots; ++j) dot[j] = warp_sum(dot[j]);
      if (lane == 0)
#pragma unroll
        for (int j = 0; j < kSlots; ++j) red[threadIdx.y * warps + warp][j] = dot[j];
      __syncthreads();
      if (in && threadIdx.x < kSlots && j0 + static_cast<int>(threadIdx.x) < a.k) {
        float s = 0.f;
        for (int x = 0; x < warps; ++x) s += red[threadIdx.y * warps + x][threadIdx.x];
        a.grad_weights[t * a.k + j0 + threadIdx.x] = s;
      }
      __syncthreads();
    }
  }
}

// ---------------------------------------------------------------------------
// unsort of large calls: the rows come by bulk copies
// ---------------------------------------------------------------------------
// Every warp runs a ring of its own in shared memory: a slot holds one segment
// (32 * NP pieces of 16 bytes) of a token's k rows, for the gradient also of g.
// Lane j finds pair j's row and issues its copy, a slot's meta data keeps row
// and weight until the segment is summed. So the bytes in flight (about 190 KB
// per SM) depend neither on registers nor on how long a row's position took;
// with plain loads 8192 tokens x 8 x 2048 bf16 took 76 us forward and 222 us
// backward.
constexpr int kBulkWarps = 8;
constexpr int kBulkRing = 24 * 1024;  // bytes of a warp's ring
constexpr int kBulkSlots = 8;
constexpr uint64_t kBulkTimeoutNs = 2000000000ull;

struct BulkCtrl {
  uint64_t full[kBulkWarps][kBulkSlots];
  int pos[kBulkWarps][kBulkSlots][32];
  float weight[kBulkWarps][kBulkSlots][32];
};
constexpr size_t kBulkSmem = kBulkWarps * kBulkRing + sizeof(BulkCtrl);

// The timer is read only where the bytes are not there yet (a read takes longer
// than many waits).
__device__ __forceinline__ bool bulk_wait(uint32_t bar, uint32_t parity, bool patient) {
  if (mbar_try_wait(bar, parity)) return true;
  return patient && mbar_wait(bar, parity, global_timer_ns() + kBulkTimeoutNs);
}

template <typename T, typename O, int NP, bool BACKWARD>
__global__ void __launch_bounds__(kBulkWarps * 32, 1) unsort_bulk_kernel(const UnsortArgs a, int slots) {
  constexpr int N = 16 / sizeof(T);
  constexpr int kSeg = NP * 512;  // bytes
  using V = Vec<T, N>;
  extern __shared__ __align__(128) uint8_t smem[];
  BulkCtrl& cb = *reinterpret_cast<BulkCtrl*>(smem + kBulkWarps * kBulkRing);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* ring = smem + warp * kBulkRing;
  const int row_bytes = a.H * static_cast<int>(sizeof(T));
  const int segs = (row_bytes + kSeg - 1) / kSeg;
  const int slot_bytes = (a.k + (BACKWARD ? 1 : 0)) * kSeg;
  if (lane < slots) mbar_init(smem_u32(&cb.full[warp][lane]), 1);
  fence_mbar_init();
  __syncwarp();
  pdl_launch_dependents();
  pdl_wait();
  const int warps = gridDim.x * kBulkWarps, first = blockIdx.x * kBulkWarps + warp;
  // Tasks: forward every segment on its own, backward a token's segments one
  // after the other (its dot products stay with the warp).
  struct Task {
    int t, seg;
  };
  const int dt = BACKWARD ? warps : warps / segs, ds = BACKWARD ? 0 : warps % segs;
  auto advance = [&](Task& q) {
    if (BACKWARD) {
      if (++q.seg == segs) {
        q.seg = 0;
        q.t += dt;
      }
    } else {
      q.t += dt;
      q.seg += ds;
      if (q.seg >= segs) {
        q.seg -= segs;
        ++q.t;
      }
    }
  };
  Task use = BACKWARD ? Task{first, 0} : Task{first / segs, first % segs};
  Task fetch = use;
  const uint8_t* rows = static_cast<const uint8_t*>(a.rows);
  const uint8_t* grad = static_cast<const uint8_t*>(a.grad);
  int pos = -1;
  float weight = 0.f;
  auto load_meta = [&] {  // of the task that is fetched next
    pos = -1;
    weight = 1.f;
    if (fetch.t < a.M && lane < a.k) {
      const int64_t i = static_cast<int64_t>(fetch.t) * a.k + lane;
      pos = a.positions[i];
      if (a.weights) weight = a.weights[i];
    }
  };
  auto issue = [&](int s) {
    const int at = fetch.seg * kSeg, bytes = min(kSeg, row_bytes - at);
    const bool here = lane < a.k && pos >= 0 && pos < a.num_rows;
    const bool rows_too = !BACKWARD || a.grad_weights != nullptr;
    const uint32_t bar = smem_u32(&cb.full[warp][s]);
    cb.pos[warp][s][lane] = pos;
    cb.weight[warp][s][lane] = weight;
    const int copies = (rows_too ? __popc(__ballot_sync(kFullMask, here)) : 0) + (BACKWARD ? 1 : 0);
    if (lane == 0) mbar_arrive_expect_tx(bar, copies * bytes);
    __syncwarp();
    const uint32_t dst = smem_u32(ring + s * slot_bytes);
    if (rows_too && here)
      bulk_g2s(dst + lane * kSeg, rows + static_cast<int64_t>(pos) * row_bytes + at, bytes, bar);
    if (BACKWARD && lane == 31)
      bulk_g2s(dst + a.k * kSeg, grad + static_cast<int64_t>(fetch.t) * row_bytes + at, bytes, bar);
    advance(fetch);
    load_meta();
  };
  load_meta();
  int filled = 0;
  for (; filled < slots && fetch.t < a.M; ++filled) issue(filled);
  int s = 0;
  uint32_t ph = 0;
  float dot = 0.f;
  float poison = 0.f;  // NaN once a wait ran out: the results from there on say so
  while (use.t < a.M) {
    if (!bulk_wait(smem_u32(&cb.full[warp][s]), ph, poison == 0.f)) poison = __int_as_float(0x7fffffff);
    const uint8_t* slot = ring + s * slot_bytes;
    const int at = use.seg * kSeg, bytes = min(kSeg, row_bytes - at);
    const int* ps = cb.pos[warp][s];
    const float* ws = cb.weight[warp][s];
    if (!BACKWARD) {
      float acc[NP][N];
#pragma unroll
      for (int q = 0; q < NP; ++q)
#pragma unroll
        for (int n = 0; n < N; ++n) acc[q][n] = poison;
#pragma unroll 4
      for (int j = 0; j < a.k; ++j) {
        const int p = ps[j];
        if (p < 0 || p >= a.num_rows) continue;
        const float w = ws[j];
#pragma unroll
        for (int q = 0; q < NP; ++q) {
          float f[N];
          to_floats(*reinterpret_cast<const V*>(slot + j * kSeg + (q * 32 + lane) * 16), f);
#pragma unroll
          for (int n = 0; n < N; ++n) acc[q][n] = fmaf(w, f[n], acc[q][n]);
        }
      }
      O* out = static_cast<O*>(a.out) + static_cast<int64_t>(use.t) * a.H + at / static_cast<int>(sizeof(T));
#pragma unroll
      for (int q = 0; q < NP; ++q) {
        Vec<O, N> o;
        from_floats(acc[q], o);
        if ((q * 32 + lane) * 16 < bytes) *reinterpret_cast<Vec<O, N>*>(out + (q * 32 + lane) * N) = o;
      }
    } else {
      float g[NP][N];
      bool in[NP];
#pragma unroll
      for (int q = 0; q < NP; ++q) {
        in[q] = (q * 32 + lane) * 16 < bytes;
        to_floats(*reinterpret_cast<const V*>(slot + a.k * kSeg + (q * 32 + lane) * 16), g[q]);
#pragma unroll
        for (int n = 0; n < N; ++n) g[q][n] += poison;
      }
      // eight pairs together: their dot products are reduced as one
#pragma unroll 1
      for (int j0 = 0; j0 < a.k; j0 += 8) {
        float d[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          d[x] = 0.f;
          const int j = j0 + x, p = j < a.k ? ps[j] : INT_MIN, r = p >= 0 ? p : ~p;
          if (r >= a.num_rows) continue;
          const float w = ws[j];
          if (a.grad_weights && p >= 0)
#pragma unroll
            for (int q = 0; q < NP; ++q) {
              float f[N];
              to_floats(*reinterpret_cast<const V*>(slot + j * kSeg + (q * 32 + lane) * 16), f);
#pragma unroll
              for (int n = 0; n < N; ++n) d[x] = in[q] ? fmaf(g[q][n], f[n], d[x]) : d[x];
            }
          if (a.grad_rows) {
            uint8_t* out = static_cast<uint8_t*>(a.grad_rows) + static_cast<int64_t>(r) * row_bytes + at;
#pragma unroll
            for (int q = 0; q < NP; ++q) {
              float f[N];
#pragma unroll
              for (int n = 0; n < N; ++n) f[n] = p >= 0 ? w * g[q][n] : 0.f;
              V o;
              from_floats(f, o);
              if (in[q]) *reinterpret_cast<V*>(out + (q * 32 + lane) * 16) = o;
            }
          }
        }
        if (a.grad_weights) {
          // halve the values and the lanes that hold each, then sum over the last four lanes:
          // lane bits 4, 3, 2 number the value that a lane ends with
#pragma unroll
          for (int half = 4; half > 0; half /= 2) {
            const bool upper = lane & (4 * half);
#pragma unroll
            for (int x = 0; x < half; ++x) {
              const float give = upper ? d[x] : d[x + half], keep = upper ? d[x + half] : d[x];
              d[x] = keep + __shfl_xor_sync(kFullMask, give, 4 * half);
            }
          }
          d[0] += __shfl_xor_sync(kFullMask, d[0], 2);
          d[0] += __shfl_xor_sync(kFullMask, d[0], 1);
          // lane j keeps pair j's sum
          const float mine = __shfl_sync(kFullMask, d[0], 4 * (lane & 7));
          if (lane >> 3 == j0 >> 3) dot += mine;
        }
      }
      if (use.seg == segs - 1) {
        if (a.grad_weights && lane < a.k) a.grad_weights[static_cast<int64_t>(use.t) * a.k + lane] = dot;
        dot = 0.f;
      }
    }
    __syncwarp();  // the slot is read
    if (fetch.t < a.M) issue(s);
    advance(use);
    if (++s == slots) {
      s = 0;
      ph ^= 1u;
    }
  }
  // after a wait that ran out, copies may still be on their way into this CTA
  if (poison != 0.f)
    for (int x = 0; x < filled; ++x, s = s + 1 == slots ? 0 : s + 1) {
      mbar_wait(smem_u32(&cb.full[warp][s]), ph ^ 1u, global_timer_ns() + kBulkTimeoutNs);
      if (s + 1 == slots) ph ^= 1u;
    }
}

template <typename V>
int sort_run(const SortArgs& a, cudaStream_t st) {
  if (a.numel <= kSmallPairs)
    return launch(sort_small_kernel<V>, dim3(std::max(a.M, 1)), dim3(kSmallThreads),
                  static_cast<size_t>((a.numel + 127) / 128 * 128 + a.k) * sizeof(int), st, a);
  static DeviceRecord record;
  int rc = allow_shared(record, sort_rank_kernel, rank_smem(1024));
  if (rc != MTP_OK) return rc;
  rc = launch(sort_rank_kernel, dim3(kRankCtas), dim3(kRankThreads), rank_smem(a.E), st, a);
  if (rc != MTP_OK) return rc;
  const dim3 block = row_block(a.row_bytes / static_cast<int64_t>(sizeof(V)), 8);
  return launch(sort_copy_kernel<V>, dim3((a.M + block.y - 1) / block.y), block, 0, st, a);
}

template <typename T, typename O, int NP, bool BACKWARD>
int bulk_run(const UnsortArgs& a, int slots, int sms, cudaStream_t st) {
  auto* kernel = unsort_bulk_kernel<T, O, NP, BACKWARD>;
  static DeviceRecord record;
  const int rc = allow_shared(record, kernel, kBulkSmem);
  return rc != MTP_OK ? rc : launch(kernel, dim3(sms), dim3(kBulkWarps * 32), kBulkSmem, st, a, slots);
}

// The widest vector that every row start and length allows.
template <typename T>
int unsort_vector(const UnsortArgs& a) {
  constexpr int kWide = 16 / sizeof(T), kPair = 4 / sizeof(T);
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a.rows) | reinterpret_cast<uintptr_t>(a.out) |
                         reinterpret_cast<uintptr_t>(a.grad) | reinterpret_cast<uintptr_t>(a.grad_rows) |
                         static_cast<uintptr_t>(static_cast<int64_t>(a.H) * sizeof(T));
  return (bits & 15) == 0 ? kWide : (bits & 3) == 0 ? kPair : 1;
}

// Bulk copies where rows are wide (512 bytes: a segment) and there is enough
// to fill the rings; a small call is done before that (backward of 8 x 2048
// bf16: 512 tokens 11 us against 13 by bulk copies, 1024 tokens 28 against 17).
// Returns whether this call is one, with its launch status in rc.
template <typename T, typename O, bool BACKWARD>
bool unsort_bulk(const UnsortArgs& a, cudaStream_t st, int& rc) {
  const int64_t row_bytes = static_cast<int64_t>(a.H) * sizeof(T);
  const int parts = a.k + (BACKWARD ? 1 : 0);
  if (row_bytes < 512 || row_bytes >= (1 << 30) || 2 * parts * 512 > kBulkRing) return false;
  // the widest segment of which a ring holds two tasks
  int seg = 2048;
  while (seg > 512 && (2 * parts * seg > kBulkRing || row_bytes < seg)) seg /= 2;
  const int sms = device_sm_count();
  if (!sms) {
    rc = MTP_ERR_CUDA;
    return true;
  }
  const int64_t tasks = a.M * (BACKWARD ? 1 : (row_bytes + seg - 1) / seg);
  if (tasks < (BACKWARD ? 4ll : 16ll) * sms) return false;
  const int slots = std::min(kBulkSlots, kBulkRing / (parts * seg));
  rc = seg == 2048   ? bulk_run<T, O, 4, BACKWARD>(a, slots, sms, st)
       : seg == 1024 ? bulk_run<T, O, 2, BACKWARD>(a, slots, sms, st)
                     : bulk_run<T, O, 1, BACKWARD>(a, slots, sms, st);
  return true;
}

// Three kernels for the vectors that unsort_vector gives; several CTAs a row
// (grid.y) where the kernel takes them.
template <typename F>
int launch_rows(const UnsortArgs& a, int n, int wide_n, int least, bool split, F* wide, F* pair, F* one,
                cudaStream_t st) {
  const int64_t vectors = (a.H + n - 1) / n;
  const dim3 block = row_block(vectors, least);
  dim3 grid((a.M + block.y - 1) / block.y);
  // Few rows wider than a CTA are latency: 16 rows of 2048 fp32 x 8 take 7.8 us in one CTA each, 4.8 in two.
  if (split && grid.x <= 148) grid.y = static_cast<unsigned>(std::min<int64_t>((vectors + block.x - 1) / block.x, 16));
  return launch(n == wide_n ? wide : n == 1 ? one : pair, grid, block, 0, st, a);
}

template <typename T, typename O>
int unsort_forward(const UnsortArgs& a, cudaStream_t st) {
  constexpr int kWide = 16 / sizeof(T), kPair = 4 / sizeof(T);
  const int n = unsort_vector<T>(a);
  int rc;
  if (n == kWide && unsort_bulk<T, O, false>(a, st, rc)) return rc;
  return launch_rows(a, n, kWide, 8, true, unsort_kernel<T, O, kWide>, unsort_kernel<T, O, kPair>, unsort_kernel<T, O, 1>, st);
}

template <typename T>
int unsort_backward(const UnsortArgs& a, cudaStream_t st) {
  constexpr int kWide = 16 / sizeof(T), kPair = 4 / sizeof(T);
  const int n = unsort_vector<T>(a);
  int rc;
  if (n == kWide && unsort_bulk<T, T, true>(a, st, rc)) return rc;
  return launch_rows(a, n, kWide, 32, false, unsort_backward_kernel<T, kWide>, unsort_backward_kernel<T, kPair>,
                     unsort_backward_kernel<T, 1>, st);
}

}  // namespace

int launch_sort_tokens(const SortArgs& a, cudaStream_t st) {
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.rows) |
                         static_cast<uintptr_t>(a.row_bytes) | static_cast<uintptr_t>(a.x_stride);
  if ((bits & 15) == 0) return sort_run<uint4>(a, st);
  if ((bits & 7) == 0) return sort_run<uint2>(a, st);
  if ((bits & 3) == 0) return sort_run<uint32_t>(a, st);
  if ((bits & 1) == 0) return sort_run<uint16_t>(a, st);
  return sort_run<uint8_t>(a, st);
}

int launch_unsort_tokens(const UnsortArgs& a, int dtype, cudaStream_t st) {
  switch (dtype) {
    case MTP_DTYPE_BF16: return unsort_forward<__nv_bfloat16, __nv_bfloat16>(a, st);
    case MTP_DTYPE_FP16: return unsort_forward<__half, __half>(a, st);
    default: return unsort_forward<float, float>(a, st);
  }
}

int launch_unsort_fp32_rows(const UnsortArgs& a, int out_dtype, cudaStream_t st) {
  switch (out_dtype) {
    case MTP_DTYPE_BF16: return unsort_forward<float, __nv_bfloat16>(a, st);
    case MTP_DTYPE_FP16: return unsort_forward<float, __half>(a, st);
    default: return unsort_forward<float, float>(a, st);
  }
}

int launch_unsort_backward(const UnsortArgs& a, int dtype, cudaStream_t st) {
  switch (dtype) {
    case MTP_DTYPE_BF16: return unsort_backward<__nv_bfloat16>(a, st);
    case MTP_DTYPE_FP16: return unsort_backward<__half>(a, st);
    default: return unsort_backward<float>(a, st);
  }
}

}  // namespace mtp
