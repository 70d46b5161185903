// Products of int8 rows and int8 weights with one scale per row and one per
// output channel, for one weight matrix or one per group of rows:
//   out[m, n] = (sum_k a[m, k] * b[g(m), n, k]) * sa[m] * sb[g(m), n] (+ bias[n])
// and, gated, out[m, i] = silu(z[m, i]) * z[m, I + i] of that z, I = N / 2.
// The sum is exact in int32 (K < 2^17); the scales are applied in fp32 and the
// result is rounded once.
//
// tile_kernel: persistent, warp-specialised, one CTA per SM. A CTA's tile is
// 128 output channels (the MMA's M) x up to NT rows of one group (its N): a
// group's rows are shared out evenly over its tiles in multiples of 16 or 32, so
// a ragged group costs what it has.
//   warp 8    producer: per stage (128 of K) one TMA box of weights and one of
//             rows (a few of 32 where the tile has few), 128-byte swizzle;
//             columns past K and rows past the end arrive as zeros. Few large
//             boxes: with boxes of 32 rows throughout, 8192^2 x 2048 took 113 us
//             against 102;
//   warp 9    one thread issues tcgen05.mma kind::i8 (K = 32) into one of two
//             accumulators of NT columns in tensor memory;
//   warps 0-7 epilogue: each warp takes its 32 channels of every other 32 rows on
//             its own: tensor memory -> scales -> its own staging rows
//             in shared memory -> 16 bytes a thread to the output, while the
//             next tile's products run and the next scales are on their way.
// PAIR: two CTAs of a cluster take 256 channels together (cta_group::2): each
// holds its 128 channels and half of the rows, so per product a CTA loads 2/3
// of what it loads alone. Gated tiles hold 16 gate channels, then their 16 up
// channels, four times, so that a gate and its up value lie 16 lanes apart in
// one warp.
//
// Many rows a group: bound by the tensor cores and the power cap (8192 x 8192 x
// 2048 in 92.8 us in a burst, 2960 TOP/s with the tensor pipe 79 % active).
// Fewer: by HBM (1024 x 2048 weights of 256 experts: 512 rows 68.7 us, 438 MB
// read and written, 6.4 TB/s; 16384 rows gated to fp32 98 us, 605 MB, 6.2 TB/s;
// 65536 rows 152 us, 5.3 TB/s).
#include "int8_common.cuh"

#include <cuda.h>

#include <algorithm>
#include <cmath>

namespace mtp {
namespace {

constexpr int kTK = 128;            // K of a stage: one 128-byte swizzle row of int8
constexpr int kTM = 128;            // channels of a CTA's tile
constexpr int kTEpiWarps = 8;       // two for each quarter of the tensor-memory lanes
constexpr int kTParts = kTEpiWarps / 4;
constexpr int kTThreads = (kTEpiWarps + 2) * 32;
constexpr int kTBox = 32;           // rows of a small TMA box
constexpr uint32_t kTWBytes = kTM * kTK;
constexpr uint32_t kTStagingBytes = 2048;  // one chunk of output rows of an epilogue warp
constexpr uint64_t kTTimeoutNs = 2000000000ull;
constexpr uint32_t kTIdesc = (2u << 4) | (1u << 7) | (1u << 10);  // D s32, A and B s8

// Ring of a tile of NT rows; a CTA of a pair holds half of them.
template <int NT, bool PAIR>
struct Ring {
  static constexpr int kRows = PAIR ? NT / 2 : NT;
  static constexpr int kStages = kRows >= 128 ? 5 : kRows == 64 ? 7 : 8;
  static constexpr uint32_t kBytes = kTWBytes + kRows * kTK;
};

struct alignas(16) TileCtrl {
  uint64_t full[8], empty[8];     // stage landed / consumed
  uint64_t dfull[2], dempty[2];   // accumulator complete / read
  uint32_t tmem;
  alignas(16) float sa[kTEpiWarps][32];  // row scales of a warp's chunk
  RowBlocks rows;
};
constexpr uint32_t kTCtrl = 20480;
static_assert(sizeof(TileCtrl) <= kTCtrl, "control block");

template <int NT, bool PAIR>
constexpr size_t tile_smem() {
  return 1024 + static_cast<size_t>(Ring<NT, PAIR>::kStages) * Ring<NT, PAIR>::kBytes + kTEpiWarps * kTStagingBytes + kTCtrl;
}
static_assert(tile_smem<256, true>() <= 227 * 1024 && tile_smem<128, true>() <= 227 * 1024 &&
                  tile_smem<64, false>() <= 227 * 1024 && tile_smem<32, false>() <= 227 * 1024,
              "shared memory");

template <bool PAIR>
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  if (PAIR)
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
        "%3}], [%4];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}

template <bool PAIR>
__device__ __forceinline__ void tma_5d(uint32_t dst, const CUtensorMap* map, int x, int block, int group, uint32_t bar) {
  if (PAIR)
    asm volatile(
        "cp.async.bulk.tensor.5d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
        "%3, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(map), "r"(x), "r"(0), "r"(block), "r"(group), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %3, %4, "
        "%5}], [%6];" ::"r"(dst),
        "l"(map), "r"(x), "r"(0), "r"(block), "r"(group), "r"(bar)
        : "memory");
}

// D[tmem] (+)= A[smem] x B[smem]^T, kind::i8
template <bool PAIR>
__device__ __forceinline__ void umma_i8_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  if (PAIR)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}

// Arrive on this barrier (of both CTAs of a pair) when the products issued so far are done.
template <bool PAIR>
__device__ __forceinline__ void tile_commit(uint32_t bar) {
  if (PAIR)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"(static_cast<uint16_t>(3))
        : "memory");
  else
    umma_commit(bar);
}

template <bool PAIR>
__device__ __forceinline__ void tile_tmem_alloc(uint32_t dst, uint32_t cols) {
  if (PAIR) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    tmem_alloc(dst, cols);
    tmem_relinquish();
  }
}
template <bool PAIR>
__device__ __forceinline__ void tile_tmem_free(uint32_t addr, uint32_t cols) {
  if (PAIR)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
  else
    tmem_dealloc(addr, cols);
}

__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The same shared-memory address in the pair's first CTA.
__device__ __forceinline__ uint32_t in_leader(uint32_t addr) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}
// Relaxed: a release would wait for the thread's output stores (1000 cycles or
// more), and what the arrival reports, reads of tensor memory, has completed.
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait_cluster(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n.reg .pred p;\nmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, "
      "p;\n}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}

// 32 consecutive 32-bit columns of this thread's lane.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_chunk(uint32_t taddr, uint32_t (&r)[32]) { tmem_ld32(taddr, r); }
__device__ __forceinline__ void tmem_ld_chunk(uint32_t taddr, uint32_t (&r)[16]) { tmem_ld16(taddr, r); }

// K-major operand in the 128-byte swizzle: 8-row groups of 1024 bytes.
__device__ __forceinline__ uint64_t desc_swizzle128(uint32_t addr) {
  return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (1ull << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}

// One lane of a converged warp. The producer and MMA warps run their loops
// with all lanes, so that addresses and descriptors stay in uniform registers,
// and let the elected lane issue: with the whole loop inside one lane's branch
// a stage took its thread 400 cycles, nearly as long as its products.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(p));
  return p != 0;
}

template <bool CLUSTER>
__device__ __forceinline__ bool mbar_done(uint32_t bar, uint32_t parity) {
  return CLUSTER ? mbar_try_wait_cluster(bar, parity) : mbar_try_wait(bar, parity);
}
template <bool CLUSTER>
__device__ __noinline__ bool mbar_wait_long(uint32_t bar, uint32_t parity) {
  const uint64_t deadline = global_timer_ns() + kTTimeoutNs;
  do {
    if (mbar_done<CLUSTER>(bar, parity)) return true;
  } while (global_timer_ns() < deadline);
  return false;
}

// A wait of at most kTTimeoutNs. After one that ran out (recorded in the
// caller's status) this thread's waits only look once, so the kernel runs to
// its end.
struct Waits {
  int32_t* status;
  bool out = false;
  __device__ __forceinline__ explicit Waits(const Int8Args& a) : status(a.status) {}
  template <bool CLUSTER = false>  // CLUSTER: arrivals of the other CTA of the pair
  __device__ __forceinline__ void on(uint32_t bar, uint32_t parity) {
    if (mbar_done<CLUSTER>(bar, parity) || out) return;
    if (!mbar_wait_long<CLUSTER>(bar, parity)) {
      out = true;
      if (status) atomicOr(status, 1);
    }
  }
};

// One tile of the walk: group, first row, rows, channel tile of this CTA.
struct Tile {
  int e, row, n, ct;
};

// The tiles of a CTA: channel tiles of a row tile next to each other, so that
// the CTAs of a moment share rows and weights in L2. Stepped without a
// division: what every role does per tile is on its critical path.
template <int NT, bool PAIR>
struct Walk {
  const RowBlocks& rb;
  int groups, ctiles, blocks, blk, ct, dblk, dct, rank;
  __device__ __forceinline__ Walk(const Int8Args& a, const TileCtrl& c)
      : rb(c.rows), groups(a.E), ctiles(a.ctiles), blocks(c.rows.pre[a.E]) {
    rank = PAIR ? static_cast<int>(cta_rank()) : 0;
    const int t = PAIR ? blockIdx.x / 2 : blockIdx.x, step = PAIR ? gridDim.x / 2 : gridDim.x;
    blk = t / ctiles;
    ct = t - blk * ctiles;
    dblk = step / ctiles;
    dct = step - dblk * ctiles;
  }
  __device__ __forceinline__ bool next(Tile& r) {
    if (blk >= blocks) return false;
    const RowBlock b = rb.at(blk, groups);
    r.row = b.row;
    r.n = b.n;
    r.e = b.e;
    r.ct = PAIR ? 2 * ct + rank : ct;
    blk += dblk;
    ct += dct;
    if (ct >= ctiles) {
      ct -= ctiles;
      ++blk;
    }
    return true;
  }
};

// Two values of neighbouring rows at p and p + pitch bytes. Conversions to 16
// bits go in pairs: one at a time they run at 16 a cycle and SM, which alone
// would take as long as a tile's products.
__device__ __forceinline__ void put2(uint8_t* p, int pitch, float a, float b, float) {
  *reinterpret_cast<float*>(p) = a;
  *reinterpret_cast<float*>(p + pitch) = b;
}
__device__ __forceinline__ void put2(uint8_t* p, int pitch, float a, float b, __half) {
  const __half2 v = __floats2half2_rn(a, b);
  *reinterpret_cast<__half*>(p) = __low2half(v);
  *reinterpret_cast<__half*>(p + pitch) = __high2half(v);
}
__device__ __forceinline__ void put2(uint8_t* p, int pitch, float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  *reinterpret_cast<__nv_bfloat16*>(p) = __low2bfloat16(v);
  *reinterpret_cast<__nv_bfloat16*>(p + pitch) = __high2bfloat16(v);
}

// Tensor maps: rows of a in boxes of a ring's rows and of kTBox, weights.
struct Maps {
  CUtensorMap rows, few, weights;
  int blocks;  // gated: 16-channel blocks of gate and up in one box of the weights' map
};

template <int NT, bool PAIR, bool GATED>
__device__ void tile_producer(const Maps& m, const Int8Args& a, TileCtrl& cb, uint32_t stages) {
  using R = Ring<NT, PAIR>;
  const int nk = (a.K + kTK - 1) / kTK;
  Waits wait(a);
  Walk<NT, PAIR> walk(a, cb);
  int st = 0;
  uint32_t ph = 0;
  int64_t issued = 0;
  Tile w;
  while (walk.next(w)) {
    // rows of this CTA: all of the tile's, or this rank's half of the MMA's N
    const int rows = PAIR ? (w.n + 31) / 32 * 16 : w.n;
    const int row = w.row + (PAIR ? walk.rank * rows : 0);
    const int boxes = 2 * rows > R::kRows ? 0 : (rows + kTBox - 1) / kTBox;  // 0: one large box
    const uint32_t bytes = kTWBytes + (boxes ? boxes * kTBox : R::kRows) * kTK;
    const int ch = GATED ? w.e * a.N + w.ct * 64 : w.e * a.N + w.ct * kTM;
    for (int s = 0; s < nk; ++s) {
      wait.on(smem_u32(&cb.empty[st]), ph ^ 1u);
      const uint32_t sb = stages + st * R::kBytes;
      uint32_t bar = smem_u32(&cb.full[st]);
      if (elect_one()) {
        if (PAIR) {
          // both CTAs' bytes arrive on the first one's barrier
          if (walk.rank == 0) mbar_arrive_expect_tx(bar, 2 * bytes);
          bar = in_leader(bar);
        } else {
          mbar_arrive_expect_tx(bar, bytes);
        }
        if (!GATED) {
          tma_2d<PAIR>(sb, &m.weights, s * kTK, ch, bar);
        } else if (m.blocks) {
          tma_5d<PAIR>(sb, &m.weights, s * kTK, w.ct * 4, w.e, bar);
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            tma_2d<PAIR>(sb + q * 4096, &m.weights, s * kTK, ch + 16 * q, bar);
            tma_2d<PAIR>(sb + q * 4096 + 2048, &m.weights, s * kTK, ch + a.N / 2 + 16 * q, bar);
          }
        }
        if (!boxes) tma_2d<PAIR>(sb + kTWBytes, &m.rows, s * kTK, row, bar);
        for (int q = 0; q < boxes; ++q)
          tma_2d<PAIR>(sb + kTWBytes + q * (kTBox * kTK), &m.few, s * kTK, row + q * kTBox, bar);
      }
      __syncwarp();
      ++issued;
      if (++st == R::kStages) {
        st = 0;
        ph ^= 1u;
      }
    }
  }
  // No copy may still be writing shared memory when the CTA exits: stage j's
  // products (whose completion both CTAs of a pair see) came after its bytes.
  wait.out = false;
  for (int64_t j = issued - 1; j >= 0 && j >= issued - R::kStages; --j)
    wait.on(smem_u32(&cb.empty[j % R::kStages]), static_cast<uint32_t>((j / R::kStages) & 1));
}

template <int NT, bool PAIR>
__device__ void tile_mma(const Int8Args& a, TileCtrl& cb, uint32_t stages, uint32_t tmem) {
  using R = Ring<NT, PAIR>;
  const int nk = (a.K + kTK - 1) / kTK;
  Waits wait(a);
  Walk<NT, PAIR> walk(a, cb);
  int st = 0, db = 0;
  uint32_t ph = 0, dph = 0;
  Tile w;
  while (walk.next(w)) {
    const uint32_t n = PAIR ? (w.n + 31) / 32 * 32 : (w.n + 15) / 16 * 16;
    const uint32_t idesc = kTIdesc | (n >> 3 << 17) | ((PAIR ? 16u : 8u) << 24);
    wait.template on<PAIR>(smem_u32(&cb.dempty[db]), dph ^ 1u);
    tc_fence_after();
    const uint32_t d = tmem + db * NT;
    for (int s = 0; s < nk; ++s) {
      wait.on(smem_u32(&cb.full[st]), ph);
      tc_fence_after();
      const uint64_t wd = desc_swizzle128(stages + st * R::kBytes);
      const uint64_t xd = desc_swizzle128(stages + st * R::kBytes + kTWBytes);
      if (elect_one()) {
#pragma unroll
        for (int j = 0; j < kTK / 32; ++j) umma_i8_ss<PAIR>(d, wd + 2 * j, xd + 2 * j, idesc, (s | j) != 0);
        tile_commit<PAIR>(smem_u32(&cb.empty[st]));
      }
      __syncwarp();
      if (++st == R::kStages) {
        st = 0;
        ph ^= 1u;
      }
    }
    if (elect_one()) tile_commit<PAIR>(smem_u32(&cb.dfull[db]));
    __syncwarp();
    if (++db == 2) {
      db = 0;
      dph ^= 1u;
    }
  }
}

template <int NT, bool PAIR, bool GATED, typename T>
__device__ void tile_epilogue(const Int8Args& a, TileCtrl& cb, uint8_t* staging, uint32_t tmem) {
  constexpr int kChannels = GATED ? 16 : 32;                // output channels of a warp
  constexpr int kRow = kChannels * sizeof(T);               // bytes of a staged row
  constexpr int kChunk = 64 / sizeof(T);                    // rows staged together
  constexpr int kUnits = (NT + 32 * kTParts - 1) / (32 * kTParts);  // units of 32 rows of a warp in a tile
  constexpr int kPieces = kRow / 16;
  static_assert(kChunk * kRow <= static_cast<int>(kTStagingBytes), "staging");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int quad = warp & 3, part = warp >> 2;
  const int width = GATED ? a.N / 2 : a.N;  // columns of the output
  T* out = static_cast<T*>(a.out);
  if (cb.rows.first[0] > 0)
    zero_rows(reinterpret_cast<uint8_t*>(out),
              reinterpret_cast<uint8_t*>(out + static_cast<int64_t>(cb.rows.first[0]) * width), kTEpiWarps * 32);
  if (cb.rows.routed < a.P)
    zero_rows(reinterpret_cast<uint8_t*>(out + static_cast<int64_t>(cb.rows.routed) * width),
              reinterpret_cast<uint8_t*>(out + static_cast<int64_t>(a.P) * width), kTEpiWarps * 32);
  const int64_t pitch = static_cast<int64_t>(width) * sizeof(T);
  const bool wide = pitch % 16 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  uint8_t* sw = staging + warp * kTStagingBytes;
  float* sas = cb.sa[warp];
  const uint32_t dbar = PAIR ? in_leader(smem_u32(&cb.dempty[0])) : smem_u32(&cb.dempty[0]);
  const int local = GATED ? lane & 15 : lane;  // channel of the warp's
  // scales of a tile: this lane's channel (gated: of its gate or up row) and its row of each of the warp's units
  struct Scales {
    float sb, bias, sa[kUnits];
  };
  auto first_channel = [&](const Tile& w) { return w.ct * 4 * kChannels + quad * kChannels; };
  auto load = [&](const Tile& w) {
    const int ch = first_channel(w) + local;
    const bool in = ch < width;
    Scales r;
    r.sb = in ? a.b_scale[static_cast<int64_t>(w.e) * a.N + ch + (GATED && lane >= 16 ? a.N / 2 : 0)] : 0.f;
    r.bias = in && a.bias ? a.bias[ch] : 0.f;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int row = 32 * (part + kTParts * u) + lane;
      r.sa[u] = row < w.n ? a.a_scale[w.row + row] : 0.f;
    }
    return r;
  };
  Waits wait(a);
  Walk<NT, PAIR> walk(a, cb);
  int db = 0;
  uint32_t dph = 0;
  Tile w, after;
  bool more = walk.next(w);
  Scales sc = {}, nsc = {};
  if (more) sc = load(w);
  while (more) {
    more = walk.next(after);
    if (more) nsc = load(after);  // on its way during this tile
    wait.on(smem_u32(&cb.dfull[db]), dph);
    tc_fence_after();
    const uint32_t dt = tmem + (static_cast<uint32_t>(32 * quad) << 16) + db * NT;
    const int ch0 = first_channel(w);
    const int row_bytes = min(kChannels, width - ch0) * static_cast<int>(sizeof(T));
    // The accumulator is free when a warp has read its last rows of it.
    auto release = [&] {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (PAIR)
          mbar_arrive_cluster(dbar + 8 * db);
        else
          mbar_arrive(dbar + 8 * db);
      }
    };
    if (32 * part >= w.n) release();
#pragma unroll 1
    for (int c = 32 * part; c < w.n;) {
      sas[lane] = sc.sa[0];
#pragma unroll
      for (int x = 0; x + 1 < kUnits; ++x) sc.sa[x] = sc.sa[x + 1];
      const int unit = c;
      c += 32 * kTParts;
#pragma unroll
      for (int h = 0; h < 32; h += kChunk) {
        if (unit + h >= w.n) break;
        uint32_t v[kChunk];
        tmem_ld_chunk(dt + unit + h, v);
        __syncwarp();  // the scales are there, and the last chunk's staged rows are read
        tmem_wait_ld();
        if (c >= w.n && (h + kChunk == 32 || unit + h + kChunk >= w.n)) release();
        if (GATED) {
          // two rows at a time: the low lanes take the first, the high lanes the second
          uint8_t* at = sw + local * sizeof(T) + (lane >> 4) * kRow;
#pragma unroll
          for (int j = 0; j < kChunk; j += 4) {
            const float4 s4 = *reinterpret_cast<const float4*>(sas + h + j);
            const float s[4] = {s4.x, s4.y, s4.z, s4.w};
            float o[2];
#pragma unroll
            for (int q = 0; q < 4; q += 2) {
              const float z0 = __int2float_rn(static_cast<int>(v[j + q])) * s[q] * sc.sb;
              const float z1 = __int2float_rn(static_cast<int>(v[j + q + 1])) * s[q + 1] * sc.sb;
              const float got = __shfl_xor_sync(kFullMask, lane < 16 ? z1 : z0, 16);
              const float gate = lane < 16 ? z0 : got, up = lane < 16 ? got : z1;
              o[q / 2] = (sizeof(T) == 4 ? silu_fp32(gate) : silu_fast(gate)) * up;
            }
            put2(at + j * kRow, 2 * kRow, o[0], o[1], T());
          }
        } else {
          uint8_t* at = sw + local * sizeof(T);
#pragma unroll
          for (int j = 0; j < kChunk; j += 4) {
            const float4 s4 = *reinterpret_cast<const float4*>(sas + h + j);
            const float s[4] = {s4.x, s4.y, s4.z, s4.w};
            float z[4];
#pragma unroll
            for (int q = 0; q < 4; ++q)
              z[q] = fmaf(__int2float_rn(static_cast<int>(v[j + q])) * s[q], sc.sb, sc.bias);
            put2(at + j * kRow, kRow, z[0], z[1], T());
            put2(at + (j + 2) * kRow, kRow, z[2], z[3], T());
          }
        }
        __syncwarp();  // the rows are staged, and the scales are read
        const int rows = min(kChunk, w.n - unit - h);
        uint8_t* o = reinterpret_cast<uint8_t*>(out) + (w.row + unit + h) * pitch + static_cast<int64_t>(ch0) * sizeof(T);
        if (wide) {
#pragma unroll
          for (int i = 0; i < kChunk * kPieces / 32; ++i) {
            const int x = lane + 32 * i, r = x / kPieces, piece = x % kPieces;
            if (r < rows && piece * 16 < row_bytes)
              *reinterpret_cast<uint4*>(o + r * pitch + piece * 16) = lds128(smem_u32(sw + r * kRow + piece * 16));
          }
        } else {
          for (int x = lane; x < kChunk * kChannels; x += 32) {
            const int r = x / kChannels, q = x % kChannels * static_cast<int>(sizeof(T));
            if (r < rows && q < row_bytes)
              *reinterpret_cast<T*>(o + r * pitch + q) = *reinterpret_cast<const T*>(sw + r * kRow + q);
          }
        }
      }
    }
    if (++db == 2) {
      db = 0;
      dph ^= 1u;
    }
    w = after;
    sc = nsc;
  }
}

template <int NT, bool PAIR, bool GATED, typename T>
__global__ void __launch_bounds__(kTThreads, 1) tile_kernel(const __grid_constant__ Maps maps,
                                                            const __grid_constant__ Int8Args a) {
  extern __shared__ uint8_t smem_raw[];
  using R = Ring<NT, PAIR>;
  const uint32_t stages = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* aligned = smem_raw + (stages - smem_u32(smem_raw));
  uint8_t* staging = aligned + R::kStages * R::kBytes;
  TileCtrl& cb = *reinterpret_cast<TileCtrl*>(staging + kTEpiWarps * kTStagingBytes);
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    for (int i = 0; i < R::kStages; ++i) {
      mbar_init(smem_u32(&cb.full[i]), 1);
      mbar_init(smem_u32(&cb.empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&cb.dfull[i]), 1);
      mbar_init(smem_u32(&cb.dempty[i]), PAIR ? 2 * kTEpiWarps : kTEpiWarps);
    }
    fence_mbar_init();
  }
  if (warp == kTEpiWarps + 1) tile_tmem_alloc<PAIR>(smem_u32(&cb.tmem), 2 * NT);
  pdl_launch_dependents();
  pdl_wait();
  build_row_blocks(a, cb.rows, NT, PAIR ? 32 : 16, kTThreads);
  tc_fence_before();
  if (PAIR) cluster_sync();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = cb.tmem;
  if (warp == kTEpiWarps) {
    tile_producer<NT, PAIR, GATED>(maps, a, cb, stages);
  } else if (warp == kTEpiWarps + 1) {
    if (!PAIR || cta_rank() == 0) tile_mma<NT, PAIR>(a, cb, stages, tmem);
  } else {
    tile_epilogue<NT, PAIR, GATED, T>(a, cb, staging, tmem);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync();  // the other CTA's barriers and tensor memory are in use until here
  if (warp == kTEpiWarps + 1) {
    tc_fence_after();
    tile_tmem_free<PAIR>(tmem, 2 * NT);
  }
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

int encode(CUtensorMap* map, int rank, const void* base, const cuuint64_t* dims, const cuuint64_t* strides,
           const cuuint32_t* box) {
  EncodeTiled fn = encode_fn();
  const cuuint32_t step[5] = {1, 1, 1, 1, 1};
  return fn && fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, rank, const_cast<void*>(base), dims, strides, box, step,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? MTP_OK
             : MTP_ERR_CUDA;
}

// [rows, K] int8 with a row stride, in boxes of box_rows x 128 bytes.
int encode_rows(CUtensorMap* map, const void* base, int64_t rows, int K, int64_t stride, int box_rows) {
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(K), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride)};
  const cuuint32_t box[2] = {kTK, static_cast<cuuint32_t>(box_rows)};
  return encode(map, 2, base, dims, strides, box);
}

// [E, 2, I, K] gate and up rows in one box of four blocks of 16 gate channels
// and their 16 up channels. I a multiple of 16.
int encode_gated(CUtensorMap* map, const void* base, int E, int I, int K, int64_t stride) {
  const cuuint64_t dims[5] = {static_cast<cuuint64_t>(K), 16, 2, static_cast<cuuint64_t>(I / 16),
                              static_cast<cuuint64_t>(E)};
  const cuuint64_t s = static_cast<cuuint64_t>(stride);
  const cuuint64_t strides[4] = {s, s * I, s * 16, s * 2 * I};
  const cuuint32_t box[5] = {kTK, 16, 2, 4, 1};
  return encode(map, 5, base, dims, strides, box);
}

// Clusters of two CTAs that the device holds at once.
template <typename F>
int pair_slots(F* kernel, size_t smem, int sms) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(sms / 2 * 2);
  cfg.blockDim = dim3(kTThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  return n;
}

template <int NT, bool PAIR, bool GATED, typename T>
int run_tiles(Int8Args& a, const void* ap, int64_t a_stride, const void* bp, int64_t b_stride, int sms,
              cudaStream_t st) {
  auto* kernel = tile_kernel<NT, PAIR, GATED, T>;
  constexpr size_t smem = tile_smem<NT, PAIR>();
  static DeviceRecord record;
  int rc = allow_shared(record, kernel, smem);
  if (rc != MTP_OK) return rc;
  int slots = sms;
  if (PAIR) {
    static int pairs[64] = {};  // by device, 0 before the first call
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return MTP_ERR_CUDA;
    if (!pairs[dev]) pairs[dev] = pair_slots(kernel, smem, sms);
    slots = pairs[dev];
    if (slots < 1) return MTP_ERR_CUDA;
  }
  Maps maps;
  maps.blocks = GATED && a.N % 32 == 0;
  rc = encode_rows(&maps.rows, ap, a.P, a.K, a_stride, Ring<NT, PAIR>::kRows);
  if (rc == MTP_OK) rc = encode_rows(&maps.few, ap, a.P, a.K, a_stride, kTBox);
  if (rc == MTP_OK)
    rc = maps.blocks ? encode_gated(&maps.weights, bp, a.E, a.N / 2, a.K, b_stride)
                     : encode_rows(&maps.weights, bp, static_cast<int64_t>(a.E) * a.N, a.K, b_stride, GATED ? 16 : kTM);
  if (rc != MTP_OK) return rc;
  const int channels = (GATED ? 64 : kTM) * (PAIR ? 2 : 1), width = GATED ? a.N / 2 : a.N;
  a.ctiles = (width + channels - 1) / channels;
  // row tiles: at most one that is not full per group that has rows, and the
  // even shares add none
  const int64_t blocks = a.P / NT + std::min(a.P, a.E);
  const int64_t grid = std::min<int64_t>(slots, std::max<int64_t>(blocks * a.ctiles, 1)) * (PAIR ? 2 : 1);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(kTThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = PAIR ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, kernel, maps, a) != cudaSuccess) {
    cudaGetLastError();
    return MTP_ERR_LAUNCH;
  }
  return MTP_OK;
}

template <int NT, bool PAIR, bool GATED>
int by_out(Int8Args& a, int out_dtype, const void* ap, int64_t as, const void* bp, int64_t bs, int sms,
           cudaStream_t st) {
  switch (out_dtype) {
    case MTP_DTYPE_BF16: return run_tiles<NT, PAIR, GATED, __nv_bfloat16>(a, ap, as, bp, bs, sms, st);
    case MTP_DTYPE_FP16: return run_tiles<NT, PAIR, GATED, __half>(a, ap, as, bp, bs, sms, st);
    default: return run_tiles<NT, PAIR, GATED, float>(a, ap, as, bp, bs, sms, st);
  }
}

template <bool GATED>
int by_rows(Int8Args& a, int nt, int out_dtype, const void* ap, int64_t as, const void* bp, int64_t bs, int sms,
            cudaStream_t st) {
  if (nt == 256) return by_out<256, true, GATED>(a, out_dtype, ap, as, bp, bs, sms, st);
  if (nt == 128) return by_out<128, true, GATED>(a, out_dtype, ap, as, bp, bs, sms, st);
  if (nt == 64) return by_out<64, false, GATED>(a, out_dtype, ap, as, bp, bs, sms, st);
  return by_out<32, false, GATED>(a, out_dtype, ap, as, bp, bs, sms, st);
}

}  // namespace

bool tma_rows_ok(const void* base, int64_t stride) { return aligned(base, 16) && stride % 16 == 0; }

int launch_int8_matmul(Int8Args a, bool gated, int out_dtype, const void* ap, int64_t a_stride, bool a_padded,
                       const void* bp, int64_t b_stride, cudaStream_t st) {
  const int sms = device_sm_count();
  if (!sms) return MTP_ERR_CUDA;
  if (!a.offsets && !gated && int8_stream_takes(a.P) && (a.K % 16 == 0 || a_padded))
    return launch_int8_stream(a, out_dtype, ap, a_stride, bp, b_stride, st);
  // Rows of a tile: the choice of the least time, rounds of tiles over the SMs
  // times the time of a stage. A stage takes about 0.21, 0.22, 0.235 and 0.35 us
  // with 32, 64, 128 (CTA pair) and 256 (pair) rows: most of it is issue and
  // latency until there are 256. So more, smaller tiles only pay while they fit
  // into one round: 256 x 4096 x 8192 takes 27.9 us with tiles of 32 rows (two
  // rounds), 16.9 with 64, 17.5 with 128, 24.9 with 256; 512 x 4096 x 2048 16.5,
  // 10.6, 8.4 and 11.3. Groups differ in size, so on average half a tile of
  // each is empty: 64 rows a group want 128 (98.3 us; 64: 105.3).
  const int width = gated ? a.N / 2 : a.N;
  const double per_group = static_cast<double>(a.P) / a.E, used = std::min(a.P, a.E);
  int nt = 0;
  double best = 0;
  for (int rows = 32, i = 0; rows <= 256; rows *= 2, ++i) {
    constexpr double kStage[4] = {0.21, 0.22, 0.235, 0.35};
    const int pair = rows >= 128 ? 2 : 1, channels = (gated ? 64 : kTM) * pair;
    const double tiles = a.offsets ? used * std::max(1.0, per_group / rows + 0.5) : (a.P + rows - 1) / rows;
    const double ctas = tiles * ((width + channels - 1) / channels) * pair;
    const double time = std::ceil(ctas / sms) * kStage[i];
    if (!nt || time < best) nt = rows, best = time;
  }
  return gated ? by_rows<true>(a, nt, out_dtype, ap, a_stride, bp, b_stride, sms, st)
               : by_rows<false>(a, nt, out_dtype, ap, a_stride, bp, b_stride, sms, st);
}

}  // namespace mtp
