// Shared by the int8 product kernels: the row blocks of ragged groups.
#pragma once

#include "internal.cuh"

namespace mtp {

constexpr int kMaxGroups = 1024;
constexpr int kBlockTable = 1024;  // row blocks whose group is looked up once per CTA

struct RowBlock {
  int row, n, e;  // first row, rows, group
};

// The rows of every group cut into blocks, in shared memory.
struct RowBlocks {
  int routed;                  // rows before offsets[E]
  int pre[kMaxGroups + 1];     // blocks before each group
  int first[kMaxGroups + 1];   // first row of each group
  uint16_t rows[kMaxGroups];   // rows of a block of each group
  int2 table[kBlockTable];     // the first blocks: row, rows | group << 16

  // Without the table: the group is the first whose blocks end past blk.
  __device__ __forceinline__ int2 find(int blk, int groups) const {
    int e = 0, hi = groups - 1;
    while (e < hi) {
      const int mid = (e + hi) >> 1;
      if (pre[mid + 1] > blk)
        hi = mid;
      else
        e = mid + 1;
    }
    const int row = first[e] + (blk - pre[e]) * rows[e];
    return make_int2(row, min(static_cast<int>(rows[e]), first[e + 1] - row) | e << 16);
  }
  __device__ __forceinline__ RowBlock at(int blk, int groups) const {
    const int2 b = blk < kBlockTable ? table[blk] : find(blk, groups);
    return {b.x, b.y & 0xffff, b.y >> 16};
  }
};

// By all `threads` threads of the CTA; blocks of at most `most` rows: an even
// share of the group's, so that its last block has no mere rest, in multiples
// of `unit`. Offsets outside the rows are clamped. Ends with the table written
// but not yet synchronised.
__device__ __forceinline__ void build_row_blocks(const Int8Args& a, RowBlocks& b, int most, int unit, int threads) {
  for (int e = threadIdx.x; e <= a.E; e += threads) {
    const int lo = a.offsets ? min(max(a.offsets[e], 0), a.P) : e * a.P;
    b.first[e] = lo;
    if (e == a.E) {
      b.routed = lo;
      break;
    }
    const int hi = a.offsets ? min(max(a.offsets[e + 1], 0), a.P) : a.P;
    const int n = max(hi - lo, 0), blocks = (n + most - 1) / most;
    const int share = blocks > 0 ? ((n + blocks - 1) / blocks + unit - 1) / unit * unit : most;
    b.rows[e] = static_cast<uint16_t>(share);
    b.pre[e + 1] = (n + share - 1) / share;
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int run = 0;
    for (int e0 = 0; e0 < a.E; e0 += 32) {
      int x = e0 + lane < a.E ? b.pre[e0 + lane + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(kFullMask, x, o);
        if (lane >= o) x += y;
      }
      if (e0 + lane < a.E) b.pre[e0 + lane + 1] = run + x;
      run += __shfl_sync(kFullMask, x, 31);
    }
    if (lane == 0) b.pre[0] = 0;
  }
  __syncthreads();
  for (int x = threadIdx.x; x < min(b.pre[a.E], kBlockTable); x += threads) b.table[x] = b.find(x, a.E);
}

// Rows of no group are zero: the bytes [from, to) of the output,
// shared out over the first `threads` threads of every CTA.
__device__ __forceinline__ void zero_rows(uint8_t* from, uint8_t* to, int threads) {
  const int64_t tid = static_cast<int64_t>(blockIdx.x) * threads + threadIdx.x;
  const int64_t all = static_cast<int64_t>(gridDim.x) * threads;
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

}  // namespace mtp
