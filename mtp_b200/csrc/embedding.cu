// Rows of a table by token ids, scaled, and the table's gradient.
//
// forward:  out[t] = scale * table[id[t]], zeros for an id outside [0, V).
// gradient: grad_table[v] = scale * sum over the tokens t of v, ascending, of
//           grad[t], in fp32, rounded once; zeros for rows without a token.
//
// The gradient sorts the tokens by id first, so that no sum depends on timing:
// 1. embed_sort_kernel: a CTA takes a slice of the table's rows, finds the
//    tokens of that slice among all, sorts them (stable) and writes zeros to
//    the rows that have none. Where a slice's tokens go needs no word from the
//    other CTAs: the tokens of smaller ids are counted on the way.
// 2. embed_sum_kernel: a warp takes a chunk of the sorted tokens and a slice of
//    the columns and sums row after row. So the work is even however uneven the
//    rows' tokens are. Rows that lie inside a chunk are written, the others'
//    sums go to `parts`: [chunk][0] of the row that reaches in from the chunk
//    before, [chunk][1] of one that begins in the chunk and reaches out.
// 3. embed_join_kernel: sums the parts of each row that reaches over chunks.
//
// Rows that come in and go out bound the forward pass, the table's rows and the
// tokens' gradients the backward pass:
//   8192 tokens of 131072 x 2048 bf16: 10.3 us and 111 us (bytes alone 7.6 and
//     87: 537 MB of zeros are written at 6.1 TB/s, then the sums take 19 us)
//   61441 tokens of 50021 x 1000 bf16: 30 us and 77 us (23 and 34)
//   65536 tokens of 5000 x 2048 bf16:  54 us and 92 us (44 and 44)
//   8192 tokens of 40 x 2048 fp32:     15 us and 34 us (10 and 10)
// What is left over the bytes is three launches in a row, the slice with the most
// tokens (its CTA sorts longest), and rows that reach over chunks.
#include "rows.cuh"

#include <algorithm>

namespace mtp {
namespace {

constexpr int kSms = 148;
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSliceRows = 1 << 17;   // rows that a CTA takes at once: bits in shared memory
constexpr int kCounted = 512;         // tokens of a slice that are sorted by counting
constexpr int kDigitBits = 6;         // of a round of the radix sort
constexpr int kBatch = 4;             // times four ids that a lane has in flight
constexpr int kKept = 256;            // tokens of a warp's range that it keeps while it counts them
constexpr int kListed = 8192;         // tokens of a slice that are sorted in shared memory
constexpr int kJoinThreads = 512;

template <typename ID>
__device__ __forceinline__ ID id_at(const EmbedArgs& a, int i) {
  return static_cast<const ID*>(a.ids)[i];
}
template <typename ID>
struct alignas(16) Four {
  ID id[4];
};
// An id as a number without sign: negative ones lie behind all rows.
__device__ __forceinline__ uint32_t unsigned_id(int32_t id) { return static_cast<uint32_t>(id); }
__device__ __forceinline__ uint64_t unsigned_id(int64_t id) { return static_cast<uint64_t>(id); }

// ---------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------
constexpr int kVectors = 4;  // of a row that a thread has in flight

template <typename ID, typename T, int N>
__global__ void __launch_bounds__(256) embed_kernel(const EmbedArgs a) {
  using V = Vec<T, N>;
  pdl_launch_dependents();
  pdl_wait();
  const int64_t t = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  if (t >= a.N) return;
  const int64_t id = id_at<ID>(a, static_cast<int>(t));
  const bool here = id >= 0 && id < a.V;
  const T* row = static_cast<const T*>(a.table) + (here ? id : 0) * a.H;
  T* out = static_cast<T*>(a.out) + t * a.H;
  const int step = blockDim.x * N;
  for (int64_t c0 = threadIdx.x * N; c0 < a.H; c0 += kVectors * step) {
    V v[kVectors];
#pragma unroll
    for (int i = 0; i < kVectors; ++i)
      if (here && c0 + i * step < a.H) v[i] = *reinterpret_cast<const V*>(row + c0 + i * step);
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      if (c0 + i * step >= a.H) break;
      float f[N];
#pragma unroll
      for (int n = 0; n < N; ++n) f[n] = 0.f;
      if (here) {
        to_floats(v[i], f);
#pragma unroll
        for (int n = 0; n < N; ++n) f[n] *= a.scale;
      }
      V o;
      from_floats(f, o);
      *reinterpret_cast<V*>(out + c0 + i * step) = o;
    }
  }
}

// ---------------------------------------------------------------------------
// gradient: the sort
// ---------------------------------------------------------------------------
struct SortShared {
  uint32_t present[kSliceRows / 32];
  int count[kSortWarps][1 << kDigitBits];
  int start[1 << kDigitBits];
  __align__(16) uint32_t key[kCounted];  // row << 9 | number in the slice
  int token[kCounted];
  int warp_in[kSortWarps], warp_below[kSortWarps];
  int list[2][2][kListed];  // two lists of keys and tokens; the second keeps the warps' tokens before that
};
static_assert(kSortWarps * kKept <= kListed, "the second list holds what the warps keep");

// One stable round of the radix sort: entries [0, n) of (key, token) by `bits`
// bits of key - lo from `shift` on.
__device__ void radix_round(SortShared& s, const int32_t* key, const int32_t* token, int32_t* key_out,
                            int32_t* token_out, int n, int lo, int shift, int bits) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, bins = 1 << bits;
  for (int x = tid; x < kSortWarps * bins; x += kSortThreads) s.count[x / bins][x % bins] = 0;
  __syncthreads();
  const int span = ((n + kSortWarps - 1) / kSortWarps + 31) / 32 * 32;
  const int begin = min(warp * span, n), end = min(begin + span, n);
  auto ranked = [&](int i, int& digit, int& rank) {  // and how many of the round have this digit
    digit = i < end ? (key[i] - lo) >> shift & (bins - 1) : bins;
    unsigned same = kFullMask;
    for (int b = 0; b <= bits; ++b) {
      const bool one = digit >> b & 1;
      const unsigned votes = __ballot_sync(kFullMask, one);
      same &= one ? votes : ~votes;
    }
    rank = __popc(same & ((1u << lane) - 1u));
    return __popc(same);
  };
  for (int i = begin; i < end; i += 32) {
    int digit, rank;
    const int equal = ranked(i + lane, digit, rank);
    if (digit < bins && rank == 0) s.count[warp][digit] += equal;
    __syncwarp();
  }
  __syncthreads();
  if (tid < bins) {
    int run = 0;
    for (int w = 0; w < kSortWarps; ++w) {
      const int v = s.count[w][tid];
      s.count[w][tid] = run;
      run += v;
    }
    s.start[tid] = run;
  }
  __syncthreads();
  if (warp == 0) {  // the digits' first places
    int run = 0;
    for (int b0 = 0; b0 < bins; b0 += 32) {
      const int v = b0 + lane < bins ? s.start[b0 + lane] : 0;
      int sum = v;
      for (int o = 1; o < 32; o *= 2) {
        const int x = __shfl_up_sync(kFullMask, sum, o);
        if (lane >= o) sum += x;
      }
      if (b0 + lane < bins) s.start[b0 + lane] = run + sum - v;
      run += __shfl_sync(kFullMask, sum, 31);
    }
  }
  __syncthreads();
  for (int i = begin; i < end; i += 32) {
    int digit, rank;
    const int equal = ranked(i + lane, digit, rank);
    int p = 0;
    if (digit < bins) p = s.start[digit] + s.count[warp][digit] + rank;
    __syncwarp();
    if (digit < bins) {
      key_out[p] = key[i + lane];
      token_out[p] = token[i + lane];
      if (rank == 0) s.count[warp][digit] += equal;
    }
    __syncwarp();
  }
  __syncthreads();
}

template <typename ID, typename V>
__global__ void __launch_bounds__(kSortThreads, 1) embed_sort_kernel(const EmbedArgs a, int rows, int64_t row_vectors) {
  extern __shared__ __align__(16) uint8_t smem[];
  SortShared& s = *reinterpret_cast<SortShared*>(smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_launch_dependents();
  pdl_wait();
  if (blockIdx.x == 0 && tid == 0) a.valid[1] = 0;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * rows, last = min(first + rows, static_cast<int64_t>(a.V));
  const int span = ((a.N + kSortWarps - 1) / kSortWarps + 127) / 128 * 128;
  const bool aligned_ids = (reinterpret_cast<uintptr_t>(a.ids) & 15) == 0;
  const int64_t begin64 = static_cast<int64_t>(warp) * span;
  const int begin = static_cast<int>(min(begin64, static_cast<int64_t>(a.N)));
  const int end = static_cast<int>(min(begin64 + span, static_cast<int64_t>(a.N)));
  for (int64_t lo64 = first; lo64 < last; lo64 += kSliceRows) {
    const int lo = static_cast<int>(lo64), have = static_cast<int>(min(static_cast<int64_t>(kSliceRows), last - lo64));
    for (int x = tid; x < (have + 31) / 32; x += kSortThreads) s.present[x] = 0;
    __syncthreads();
    int in = 0, below = 0;
    // A lane takes four ids that follow one another, the warp 128 in order. fn(position of
    // the lane's first match among those so far, i, their rows, which of the four match)
    // where the warp has any; most slices have none of most 128.
    auto walk = [&](bool count, auto fn) {
      int seen = 0;
      for (int i0 = begin; i0 < end; i0 += 128 * kBatch) {
        ID id[kBatch][4];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int i = i0 + 128 * u + 4 * lane;
          if (aligned_ids && i + 4 <= end) {
            const Four<ID> four = *reinterpret_cast<const Four<ID>*>(static_cast<const ID*>(a.ids) + i);
#pragma unroll
            for (int x = 0; x < 4; ++x) id[u][x] = four.id[x];
          } else {
#pragma unroll
            for (int x = 0; x < 4; ++x) id[u][x] = i + x < end ? id_at<ID>(a, i + x) : ID(-1);
          }
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          unsigned match = 0;
          int row[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const auto v = unsigned_id(id[u][x]);
            using U = decltype(unsigned_id(id[u][x]));
            if (count) below += v < static_cast<U>(lo);
            const U r = v - static_cast<U>(lo);
            row[x] = static_cast<int>(r);
            match |= (r < static_cast<U>(have) ? 1u : 0u) << x;
          }
          if (!__any_sync(kFullMask, match)) continue;
          const int mine = __popc(match);
          const unsigned under = (1u << lane) - 1u, b0 = __ballot_sync(kFullMask, mine & 1),
                         b1 = __ballot_sync(kFullMask, mine & 2), b2 = __ballot_sync(kFullMask, mine & 4);
          fn(seen + __popc(b0 & under) + 2 * __popc(b1 & under) + 4 * __popc(b2 & under), i0 + 128 * u + 4 * lane, row, match);
          seen += __popc(b0) + 2 * __popc(b1) + 4 * __popc(b2);
        }
      }
      return seen;
    };
    in = walk(true, [&](int p, int i, const int (&row)[4], unsigned match) {
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        if (!(match >> x & 1)) continue;
        const uint32_t bit = 1u << (row[x] & 31);
        if (!(*static_cast<volatile uint32_t*>(&s.present[row[x] >> 5]) & bit)) atomicOr(&s.present[row[x] >> 5], bit);
        if (p < kKept) {
          s.list[1][0][warp * kKept + p] = row[x];
          s.list[1][1][warp * kKept + p] = i + x;
        }
        ++p;
      }
    });
    below = __reduce_add_sync(kFullMask, below);
    if (lane == 0) {
      s.warp_in[warp] = in;
      s.warp_below[warp] = below;
    }
    __syncthreads();
    int base = 0, n = 0, at = 0;
    for (int w = 0; w < kSortWarps; ++w) {
      at += w < warp ? s.warp_in[w] : 0;
      n += s.warp_in[w];
      base += s.warp_below[w];
    }
    if (tid == 0 && lo64 + have == a.V) a.valid[0] = base + n;
    // Many tokens are sorted in shared memory, too many between the halves of keys and order;
    // the last round writes the first half.
    const int bits = have > 1 ? 32 - __clz(have - 1) : 0;
    const int rounds = n <= kCounted ? 0 : (bits + kDigitBits - 1) / kDigitBits;
    int32_t* key = a.keys + base;
    int32_t* token = a.order + base;
    if (n > 0) {
      const bool counted = n <= kCounted, listed = n <= kListed;
      // keys and tokens before round r
      auto keys_of = [&](int r) { return r == rounds ? key : listed ? s.list[r & 1][0] : key + ((rounds - r) & 1 ? a.N : 0); };
      auto tokens_of = [&](int r) { return r == rounds ? token : listed ? s.list[r & 1][1] : token + ((rounds - r) & 1 ? a.N : 0); };
      int32_t* key_to = keys_of(0);
      int32_t* token_to = tokens_of(0);
      auto put = [&](int p, int row, int t) {
        if (counted) {
          s.key[p] = static_cast<uint32_t>(row) << 9 | p;
          s.token[p] = t;
        } else {
          key_to[p] = lo + row;
          token_to[p] = t;
        }
      };
      if (in <= kKept) {
        for (int x = lane; x < in; x += 32) put(at + x, s.list[1][0][warp * kKept + x], s.list[1][1][warp * kKept + x]);
      } else {
        walk(false, [&](int p, int i, const int (&row)[4], unsigned match) {
#pragma unroll
          for (int x = 0; x < 4; ++x)
            if (match >> x & 1) put(at + p++, row[x], i + x);
        });
      }
      if (counted)
        for (int x = n + tid; x < (n + 3) / 4 * 4; x += kSortThreads) s.key[x] = 0xffffffffu;
      __syncthreads();
      if (counted && tid < n) {
        const uint32_t k = s.key[tid];
        int p = 0;
        for (int x = 0; x < n; x += 4) {
          const uint4 v = *reinterpret_cast<const uint4*>(s.key + x);
          p += (v.x < k) + (v.y < k) + (v.z < k) + (v.w < k);
        }
        key[p] = lo + static_cast<int>(k >> 9);
        token[p] = s.token[tid];
      }
      const int each = rounds ? (bits + rounds - 1) / rounds : 0;
      for (int r = 0; r < rounds; ++r)
        radix_round(s, keys_of(r), tokens_of(r), keys_of(r + 1), tokens_of(r + 1), n, lo, r * each, min(each, bits - r * each));
    }
    // zeros to the rows without a token: a warp a row
    V zero;
    memset(&zero, 0, sizeof(V));
    for (int row = warp; row < have; row += kSortWarps) {
      if (s.present[row >> 5] >> (row & 31) & 1) continue;
      V* out = static_cast<V*>(a.grad_table) + (lo64 + row) * row_vectors;
      for (int64_t c = lane; c < row_vectors; c += 32) out[c] = zero;
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// gradient: the sums
// ---------------------------------------------------------------------------
constexpr int kAhead = 8;  // tokens whose rows a thread has in flight

// A row that reaches over one border of chunks with fewer than kWhole tokens
// behind it is summed whole by the item in whose chunk it begins; so most rows
// need no parts. Chunks have at least kWhole tokens.
constexpr int kWhole = 32;

// blockDim (lanes of an item, items): an item is a chunk of the sorted tokens
// and as many columns as its lanes hold.
template <typename T, int N>
__global__ void __launch_bounds__(256, 4) embed_sum_kernel(const EmbedArgs a, int slices) {
  using V = Vec<T, N>;
  pdl_launch_dependents();
  pdl_wait();
  const int64_t item = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  const int chunk = static_cast<int>(item / slices), slice = static_cast<int>(item % slices);
  const int valid = a.valid[0];
  const int64_t begin64 = static_cast<int64_t>(chunk) * a.chunk;
  if (begin64 >= valid) return;
  int begin = static_cast<int>(begin64), end = static_cast<int>(min(begin64 + a.chunk, static_cast<int64_t>(valid)));
  // the item's lanes count the keys equal to `key` among the kWhole from position i on
  const unsigned lanes = (blockDim.x == 32 ? kFullMask : (1u << blockDim.x) - 1u) << ((threadIdx.y * blockDim.x) & 31);
  auto run = [&](int i, int key) {
    int n = 0;
    for (int x = threadIdx.x; x < kWhole; x += blockDim.x)
      n += static_cast<int64_t>(i) + x < valid && a.keys[static_cast<int64_t>(i) + x] == key;
    return __reduce_add_sync(lanes, n);
  };
  int row = a.keys[begin];
  const int last = a.keys[end - 1];
  int head = begin > 0 && a.keys[begin - 1] == row ? row : -1;  // a row that reaches in
  int tail = end < valid && a.keys[end] == last ? last : -1;    // or out
  bool owner = false;
  if (head >= 0) {
    const int n = run(begin, row);
    if (n < kWhole && !(begin > a.chunk && a.keys[begin - a.chunk - 1] == row)) {  // whole, by the item before
      begin += n;
      head = -1;
      if (begin >= end) return;
      row = a.keys[begin];
    }
  }
  if (tail >= 0 && head != tail) {
    const int n = run(end, last);
    if (n < kWhole) {
      end += n;
      tail = -1;
    } else {
      owner = true;
    }
  }
  if (owner && slice == 0 && threadIdx.x == 0) a.owners[atomicAdd(a.valid + 1, 1)] = chunk;
  const int64_t c = (static_cast<int64_t>(slice) * blockDim.x + threadIdx.x) * N;
  if (c >= a.H) return;
  const T* grad = static_cast<const T*>(a.grad) + c;
  float acc[N];
#pragma unroll
  for (int n = 0; n < N; ++n) acc[n] = 0.f;
  auto write = [&] {  // the row's sum
    const bool in = row == head, out = row == tail;
    if (in || out) {
      float* part = a.parts + (2ll * chunk + (in ? 0 : 1)) * a.H + c;
#pragma unroll
      for (int n = 0; n < N; ++n) part[n] = acc[n];
    } else {
#pragma unroll
      for (int n = 0; n < N; ++n) acc[n] *= a.scale;
      V o;
      from_floats(acc, o);
      *reinterpret_cast<V*>(static_cast<T*>(a.grad_table) + static_cast<int64_t>(row) * a.H + c) = o;
    }
#pragma unroll
    for (int n = 0; n < N; ++n) acc[n] = 0.f;
  };
  for (int i0 = begin; i0 < end; i0 += kAhead) {
    V v[kAhead];
    int key[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = min(i0 + u, end - 1);
      key[u] = a.keys[i];
      v[u] = *reinterpret_cast<const V*>(grad + static_cast<int64_t>(a.order[i]) * a.H);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (i0 + u >= end) break;
      if (key[u] != row) {
        write();
        row = key[u];
      }
      float f[N];
      to_floats(v[u], f);
#pragma unroll
      for (int n = 0; n < N; ++n) acc[n] += f[n];
    }
  }
  write();
}

// A CTA takes a row that reaches over chunks and `lanes` * N of its columns; its
// groups of `lanes` threads share the chunks out evenly and in order.
template <typename T, int N>
__global__ void __launch_bounds__(kJoinThreads) embed_join_kernel(const EmbedArgs a, int lanes) {
  __shared__ Vec<float, N> sums[kJoinThreads];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, group = threadIdx.x / lanes, groups = kJoinThreads / lanes;
  const int valid = a.valid[0], owners = a.valid[1];
  const int blocks = (a.H + lanes * N - 1) / (lanes * N);
  for (int64_t item = blockIdx.x; item < static_cast<int64_t>(owners) * blocks; item += gridDim.x) {
    const int chunk = a.owners[item / blocks];
    const int64_t c = (item % blocks * lanes + threadIdx.x % lanes) * N;
    const int row = a.keys[(chunk + 1ll) * a.chunk];
    // chunks that the row reaches into: a search among the chunks' first keys, 32 at a time
    int more = 1;
    for (int64_t left = (valid - 1) / a.chunk - chunk; more < left;) {  // the row has `more`, at most `left`
      const int64_t stride = (left - more + 31) / 32;
      const int64_t q = min(more + stride * (lane + 1), left);
      const unsigned votes = __ballot_sync(kFullMask, a.keys[(chunk + q) * a.chunk] == row);
      const int n = __popc(votes);  // the first n of them are the row's
      if (n == 32) {
        more = static_cast<int>(left);
      } else {
        left = min(more + stride * (n + 1), left) - 1;
        more = static_cast<int>(min(more + stride * n, left));
      }
    }
    const int each = (more + groups) / groups;  // of more + 1 parts
    const int from = group * each, to = min(from + each, more + 1);
    Vec<float, N> s = {};
    if (c < a.H)
#pragma unroll 8
      for (int p = from; p < to; ++p) {
        const Vec<float, N> v = *reinterpret_cast<const Vec<float, N>*>(a.parts + (2ll * (chunk + p) + (p == 0 ? 1 : 0)) * a.H + c);
#pragma unroll
        for (int n = 0; n < N; ++n) s.v[n] += v.v[n];
      }
    sums[threadIdx.x] = s;
    __syncthreads();
    if (group == 0 && c < a.H) {
      float f[N];
#pragma unroll
      for (int n = 0; n < N; ++n) f[n] = 0.f;
#pragma unroll 8
      for (int w = 0; w < (more + each) / each; ++w) {  // the groups that have parts
        const Vec<float, N> v = sums[w * lanes + threadIdx.x];
#pragma unroll
        for (int n = 0; n < N; ++n) f[n] += v.v[n];
      }
      T* out = static_cast<T*>(a.grad_table) + static_cast<int64_t>(row) * a.H + c;
#pragma unroll
      for (int n = 0; n < N; ++n) f[n] *= a.scale;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        Vec<T, 1> o;
        from_floats(f + n, o);
        reinterpret_cast<Vec<T, 1>*>(out)[n] = o;
      }
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
// The widest vector that the rows of both tensors allow.
template <typename T>
int vector_of(const void* x, const void* y, int H) {
  constexpr int kWide = 16 / sizeof(T), kPair = 4 / sizeof(T);
  const uintptr_t bits = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y) |
                         static_cast<uintptr_t>(static_cast<int64_t>(H) * sizeof(T));
  return (bits & 15) == 0 ? kWide : (bits & 3) == 0 ? kPair : 1;
}

template <typename ID, typename T, int N>
int forward_run(const EmbedArgs& a, cudaStream_t st) {
  // a few tokens take all lanes at once
  const int64_t vectors = (a.H + N - 1) / N;
  const dim3 block = row_block(a.N > 2 * kSms ? (vectors + kVectors - 1) / kVectors : vectors, 8);
  return launch(embed_kernel<ID, T, N>, dim3((a.N + block.y - 1) / block.y), block, 0, st, a);
}

template <typename ID, typename V>
int sort_run(const EmbedArgs& a, int64_t row_bytes, cudaStream_t st) {
  static DeviceRecord record;
  auto* kernel = embed_sort_kernel<ID, V>;
  const int rc = allow_shared(record, kernel, sizeof(SortShared));
  if (rc != MTP_OK) return rc;
  const int rows = (a.V - 1) / kSms + 1;
  return launch(kernel, dim3((a.V - 1) / rows + 1), dim3(kSortThreads), sizeof(SortShared), st, a, rows,
                row_bytes / static_cast<int64_t>(sizeof(V)));
}

template <typename ID>
int sort_run(const EmbedArgs& a, int64_t row_bytes, cudaStream_t st) {
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a.grad_table) | static_cast<uintptr_t>(row_bytes);
  if ((bits & 15) == 0) return sort_run<ID, uint4>(a, row_bytes, st);
  if ((bits & 3) == 0) return sort_run<ID, uint32_t>(a, row_bytes, st);
  return sort_run<ID, uint16_t>(a, row_bytes, st);
}

template <typename T, int N>
int sum_run(const EmbedArgs& a, cudaStream_t st) {
  const int64_t vectors = a.H / N, chunks = (static_cast<int64_t>(a.N) + a.chunk - 1) / a.chunk;
  int lanes = 4;
  while (lanes < vectors && lanes < 32) lanes *= 2;
  const int64_t slices = (vectors + lanes - 1) / lanes, items = chunks * slices;
  const int per = 256 / lanes;
  if ((items + per - 1) / per > 0x7fffffff) return MTP_ERR_SHAPE;
  int rc = launch(embed_sum_kernel<T, N>, dim3(static_cast<unsigned>((items + per - 1) / per)), dim3(lanes, per), 0, st,
                  a, static_cast<int>(slices));
  if (rc != MTP_OK || chunks == 1) return rc;
  const int columns = a.H % 4 ? 1 : 4;
  int join_lanes = 4;
  while (join_lanes * columns < a.H && join_lanes < 32) join_lanes *= 2;
  return launch(columns == 1 ? embed_join_kernel<T, 1> : embed_join_kernel<T, 4>, dim3(4 * kSms), dim3(kJoinThreads), 0, st, a,
                join_lanes);
}

template <typename T>
int run(const EmbedArgs& a, bool backward, cudaStream_t st) {
  constexpr int kWide = 16 / sizeof(T), kPair = 4 / sizeof(T);
  if (!backward) {
    const int n = vector_of<T>(a.table, a.out, a.H);
    if (a.wide_ids)
      return n == kWide ? forward_run<int64_t, T, kWide>(a, st)
             : n == 1   ? forward_run<int64_t, T, 1>(a, st)
                        : forward_run<int64_t, T, kPair>(a, st);
    return n == kWide ? forward_run<int32_t, T, kWide>(a, st)
           : n == 1   ? forward_run<int32_t, T, 1>(a, st)
                      : forward_run<int32_t, T, kPair>(a, st);
  }
  const int64_t row_bytes = static_cast<int64_t>(a.H) * sizeof(T);
  const int rc = a.wide_ids ? sort_run<int64_t>(a, row_bytes, st) : sort_run<int32_t>(a, row_bytes, st);
  if (rc != MTP_OK || a.N == 0) return rc;
  const int n = vector_of<T>(a.grad, a.grad_table, a.H);
  return n == kWide ? sum_run<T, kWide>(a, st) : n == 1 ? sum_run<T, 1>(a, st) : sum_run<T, kPair>(a, st);
}

int run(const EmbedArgs& a, int dtype, bool backward, cudaStream_t st) {
  switch (dtype) {
    case MTP_DTYPE_BF16: return run<__nv_bfloat16>(a, backward, st);
    case MTP_DTYPE_FP16: return run<__half>(a, backward, st);
    default: return run<float>(a, backward, st);
  }
}

}  // namespace

EmbedWs embed_workspace(int N, int H, int dtype) {
  EmbedWs w;
  // chunks so long that the items (a warp for 512 bytes of a row) fill the GPU once
  const int64_t slices = (static_cast<int64_t>(H) * (dtype == MTP_DTYPE_FP32 ? 4 : 2) + 511) / 512;
  w.chunk = 32;  // at least embed_sum_kernel's kWhole
  while (w.chunk < 256 && static_cast<int64_t>(N) * slices > 32ll * kSms * w.chunk) w.chunk *= 2;
  const int64_t chunks = (static_cast<int64_t>(N) + w.chunk - 1) / w.chunk;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at = round_up(at + bytes, 256);
    return o;
  };
  w.valid = take(8);
  w.owners = take(4 * chunks);
  w.keys = take(8ll * N);
  w.order = take(8ll * N);
  w.parts = take(chunks > 1 ? 8 * chunks * H : 0);
  w.total = at;
  return w;
}
int launch_embed(const EmbedArgs& a, int dtype, cudaStream_t st) { return run(a, dtype, false, st); }
int launch_embed_backward(const EmbedArgs& a, int dtype, cudaStream_t st) { return run(a, dtype, true, st); }

}  // namespace mtp
