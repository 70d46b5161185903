// The W8A8 MoE layer for a few tokens (decode) in two launches.
//
// What the separate kernels of a layer cost at one token is launches and waits,
// not work: seven of them take 26 us (31 with their launches) for 25 MB of
// weights, 4 us of HBM. Here, one CTA per SM in both:
//   up    every CTA routes all tokens (a warp each) while its other warps quantise
//         their rows into shared memory, and lists the pairs of each expert: the
//         same in every CTA, so nothing has to be exchanged; then its share of the
//         gate_up units (8 gate + 8 up channels of one expert's up to 8 pairs)
//         gives h = silu(gate) * up in fp32. The first CTA leaves the lists.
//   down  each CTA quantises the h rows of the experts it works on while its first
//         weights are on their way, and takes its share of the down units (16
//         channels), y in fp32. The last unit of a strip of channels to finish
//         sums it: out[t] = sum over the token's pairs, in order, of weight * y.
// (One launch with grid barriers between these phases took 19.3 us a call, the
// two take 17: a barrier over 148 SMs costs more than the end of a kernel.)
// A unit's product is streamed as in int8_stream.cu: 16 bytes of K a lane from
// global memory into mma.m16n8k32, ks warps a unit, int32 sums through shared
// memory. A CTA's units are one range of (block, strip), so it touches few
// experts' rows.
#include "quantize.cuh"
#include "w8a8_common.cuh"

#include <algorithm>

namespace mtp {
namespace {

constexpr int kDWarps = 16;
constexpr int kDThreads = kDWarps * 32;
constexpr int kDTokens = 8;
constexpr int kDPairs = 256;          // tokens * top_k
constexpr int kDSteps = 4;            // 128 bytes of K in flight per round and warp
constexpr int kDRows = 16;            // rows of h quantised together (two blocks)

constexpr int kDCodes = 96 * 1024;    // most bytes of quantised rows

// The pairs, and their blocks of up to 8 of one expert.
struct DecodeLists {
  int blocks;
  int expert[kDPairs];                // of each pair, -1 without one
  float weight[kDPairs];
  int block_expert[kDPairs];
  int block_pair[kDPairs][8];         // -1 past the end of a block
};
struct DecodeShared {
  DecodeLists l;
  int rank[kDPairs];                  // of a pair among those of its expert
  int block[kDPairs];                 // of a pair that starts one
  float scale[kDRows];                // of the quantised rows
  uint32_t most[kDRows];
  int red[2][kDWarps][4][32];
  int last[kDWarps];                  // whether a team finished its strip
};

// Quantised rows half a bank row apart: the eight rows that a load of shared
// memory touches fall on different banks.
__host__ __device__ constexpr int decode_pitch(int K) { return (K + 127) / 128 * 128 + 64; }

// Up to kDRows rows of K elements into codes by `warps` warps of which this is
// number w (named barrier 15 joins them); row(m) is the m-th.
template <typename X, typename F>
__device__ __forceinline__ void quantise_into(F row, int rows, int K, uint8_t* codes, int pitch, DecodeShared& d, int w,
                                              int warps) {
  const int lane = threadIdx.x & 31;
  if (w == 0 && lane < kDRows) d.most[lane] = 0;
  named_bar_sync(15, 32 * warps);
  int per_row = warps;
  while (per_row > 1 && per_row * rows > warps) per_row /= 2;
  const int first = ((w % per_row) * 32 + lane) * 8, step = per_row * 256;
  const int m = w / per_row;
  const X* src = m < rows ? row(m) : nullptr;
  uint32_t mx = 0;
  float keep[8];
  if (src) {
    for (int c = first; c < K; c += step) {
      float v[8];
      load_unit<X, true>(src, c, K, v);
      mx = max(mx, magnitude(v));
      if (c == first)
#pragma unroll
        for (int i = 0; i < 8; ++i) keep[i] = v[i];
    }
    mx = __reduce_max_sync(kFullMask, mx);
    if (lane == 0) atomicMax(&d.most[m], mx);
  }
  named_bar_sync(15, 32 * warps);
  if (src) {
    const uint32_t most = d.most[m];
    const RowScale r = row_scale(most);
    if (first == 0) d.scale[m] = __fdiv_rn(__uint_as_float(most), 127.f);
    for (int c = first; c < K; c += step) {
      float v[8];
      if (c == first)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = keep[i];
      else
        load_unit<X, true>(src, c, K, v);
      store_unit(reinterpret_cast<int8_t*>(codes + m * pitch + c), v, r);
    }
  }
}

// Experts and weights of the pairs, by warp w of kDTokens.
template <int VPT>
__device__ __forceinline__ void decode_route(const DecodeArgs& a, DecodeShared& d, int w) {
  const int lane = threadIdx.x & 31;
  if (w >= a.M) return;
  float weight = 0.f;
  int id = -1;
  if (a.logits) {
    route_token<VPT>(a.logits + static_cast<int64_t>(w) * a.E, a.E, a.k, a.renorm, &weight, &id);
  } else if (lane < a.k) {
    id = a.topk_ids[w * a.k + lane];
    weight = a.topk_weights[w * a.k + lane];
    if (a.emap) id = id >= 0 && id < a.E_map ? a.emap[id] : -1;
  }
  if (lane < a.k) {
    d.l.expert[w * a.k + lane] = id >= 0 && id < a.E ? id : -1;
    d.l.weight[w * a.k + lane] = weight;
  }
}

// Blocks of up to 8 pairs of one expert, in the order of their first pairs.
__device__ __forceinline__ void decode_lists(const DecodeArgs& a, DecodeShared& d) {
  const int pairs = a.M * a.k, i = threadIdx.x;
  for (int x = i; x < pairs * 8; x += kDThreads) d.l.block_pair[x / 8][x % 8] = -1;
  __syncthreads();  // (also: the pairs' experts are there)
  if (pairs <= 32) {
    if (i < 32) {
      const int e = i < pairs ? d.l.expert[i] : -1;
      const unsigned same = __match_any_sync(kFullMask, e);
      const int rank = __popc(same & ((1u << i) - 1u));
      const unsigned starts = __ballot_sync(kFullMask, e >= 0 && rank % 8 == 0);
      // the last starting pair of this expert up to this one
      const unsigned mine = same & starts & (0xffffffffu >> (31 - i));
      const int first = mine ? 31 - __clz(mine) : 0;
      const int b = __popc(starts & ((1u << first) - 1u));
      if (e >= 0) {
        d.l.block_pair[b][rank % 8] = i;
        d.l.block_expert[b] = e;
      }
      if (i == 0) d.l.blocks = __popc(starts);
    }
    __syncthreads();
    return;
  }
  if (i < pairs) {
    int r = 0;
    for (int j = 0; j < i; ++j) r += d.l.expert[j] == d.l.expert[i] ? 1 : 0;
    d.rank[i] = r;
  }
  __syncthreads();
  auto starts = [&](int j) { return d.l.expert[j] >= 0 && d.rank[j] % 8 == 0; };
  if (i < pairs && starts(i)) {
    int b = 0;
    for (int j = 0; j < i; ++j) b += starts(j) ? 1 : 0;
    d.block[i] = b;
    d.l.block_expert[b] = d.l.expert[i];
  }
  if (i == kDThreads - 1) {
    int b = 0;
    for (int j = 0; j < pairs; ++j) b += starts(j) ? 1 : 0;
    d.l.blocks = b;
  }
  __syncthreads();
  if (i < pairs && d.l.expert[i] >= 0) {
    int s = i;  // the pair that starts this one's block
    while (d.l.expert[s] != d.l.expert[i] || d.rank[s] != d.rank[i] / 8 * 8) --s;
    d.l.block_pair[d.block[s]][d.rank[i] % 8] = i;
  }
  __syncthreads();
}

// This CTA's range of the units (block, strip) of a phase.
struct Range {
  int lo, hi, strips, ks, rounds;
  __device__ __forceinline__ Range(int blocks, int strips_, int K) : strips(strips_) {
    const int64_t units = static_cast<int64_t>(blocks) * strips;
    lo = static_cast<int>(units * blockIdx.x / gridDim.x);
    hi = static_cast<int>(units * (blockIdx.x + 1) / gridDim.x);
    const int steps = (K + 127) / 128;
    ks = 1;  // warps of a unit: as many as the range leaves
    while (ks < kDWarps && 2 * ks <= steps && 2 * ks * (hi - lo) <= kDWarps) ks *= 2;
    rounds = (steps + kDSteps * ks - 1) / (kDSteps * ks);
  }
};

struct Weights {
  uint4 v[kDSteps][4];
};

// The weights of a unit's round: this lane's two rows (gated: a gate and its up
// row; else channels 8 apart), clamped to the expert's.
template <bool GATED>
__device__ __forceinline__ void load_weights(Weights& w, const int8_t* b, int e, int N, int K, int strip, int round,
                                             int ks, int part) {
  const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int c0 = GATED ? min(strip * 8 + g, N / 2 - 1) : min(strip * 16 + g, N - 1);
  const int c1 = GATED ? N / 2 + c0 : min(strip * 16 + g + 8, N - 1);
  const int8_t* base = b + static_cast<int64_t>(e) * N * K + q * 16;
  const int8_t* p0 = base + static_cast<int64_t>(c0) * K;
  const int8_t* p1 = base + static_cast<int64_t>(c1) * K;
  const uint4 none = make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int i = 0; i < kDSteps; ++i) {
    const int k0 = ((round * kDSteps + i) * ks + part) * 128;
    const bool in0 = k0 + q * 16 < K, in1 = k0 + 64 + q * 16 < K;
    w.v[i][0] = in0 ? ldg_stream16(p0 + k0) : none;
    w.v[i][1] = in1 ? ldg_stream16(p0 + k0 + 64) : none;
    w.v[i][2] = in0 ? ldg_stream16(p1 + k0) : none;
    w.v[i][3] = in1 ? ldg_stream16(p1 + k0 + 64) : none;
  }
}

// A team has written y of strip s for its block: the last of the strip's blocks
// to get here has all of them to sum, in the order of the token's pairs.
template <typename T>
__device__ __forceinline__ void decode_finish(const DecodeArgs& a, DecodeShared& d, int s, const Range& r) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, team = warp / r.ks, part = warp % r.ks;
  auto together = [&] {
    if (r.ks > 1)
      named_bar_sync(1 + team, 32 * r.ks);
    else
      __syncwarp();
  };
  together();
  // releases what the team wrote and, for the last, acquires what the others did
  if (part == 0 && lane == 0) d.last[team] = atom_acq_rel_gpu_add(a.done + s, 1) == d.l.blocks - 1;
  together();
  if (!d.last[team]) return;
  T* out = static_cast<T*>(a.out);
  for (int x = part * 32 + lane; x < a.M * 16; x += 32 * r.ks) {
    const int t = x / 16, c = s * 16 + x % 16;
    if (c >= a.H) continue;
    float acc = 0.f;
#pragma unroll 8
    for (int j = 0; j < a.k; ++j) {
      const int p = t * a.k + j;
      if (d.l.expert[p] >= 0) acc = fmaf(d.l.weight[p], __ldcg(a.y + static_cast<int64_t>(p) * a.H + c), acc);
    }
    out[static_cast<int64_t>(t) * a.H + c] = out_cast<T>(acc);
  }
}

// Units lo .. hi of one phase, team by team. Gated: rows are the tokens' codes,
// the result h; else the codes of the rows of blocks first, first + 1 (8 rows
// each), the result y. The first unit's weights may already be in w.
template <bool GATED, typename T>
__device__ __forceinline__ void decode_units(const DecodeArgs& a, DecodeShared& d, const Range& r, int lo, int hi,
                                             int first, Weights& w, bool loaded, const uint8_t* codes, int& buf) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int N = GATED ? 2 * a.I : a.H, K = GATED ? a.H : a.I;
  const int8_t* b = GATED ? a.w13 : a.w2;
  const float* bs = GATED ? a.s13 : a.s2;
  const int pitch = decode_pitch(K), width = GATED ? a.I : a.H;
  const int ks = r.ks, team = warp / ks, part = warp % ks, teams = kDWarps / ks;
  int u = lo + team;
  if (!loaded && u < hi) load_weights<GATED>(w, b, d.l.block_expert[u / r.strips], N, K, u % r.strips, 0, ks, part);
  for (; u < hi; u += teams) {
    const int blk = u / r.strips, s = u - blk * r.strips, e = d.l.block_expert[blk];
    const int mine = d.l.block_pair[blk][g];  // the pair whose row this lane feeds
    const uint8_t* xrow = codes + (GATED ? max(mine, 0) / a.k : 8 * (blk - first) + g) * pitch;
    const int ch0 = GATED ? s * 8 + g : s * 16 + g, c1 = GATED ? a.I + ch0 : ch0 + 8;
    const float sb0 = bs[static_cast<int64_t>(e) * N + min(ch0, N - 1)];
    const float sb1 = bs[static_cast<int64_t>(e) * N + min(c1, N - 1)];
    int acc[4] = {0, 0, 0, 0};
    for (int round = 0; round < r.rounds; ++round) {
#pragma unroll
      for (int i = 0; i < kDSteps; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int k = ((round * kDSteps + i) * ks + part) * 128 + h * 64 + q * 16;
          uint4 x = make_uint4(0, 0, 0, 0);
          if (mine >= 0 && k < K) x = lds128(smem_u32(xrow + k));
          const uint4 w0 = w.v[i][h], w1 = w.v[i][2 + h];
          mma_s8(acc, w0.x, w1.x, w0.y, w1.y, x.x, x.y);
          mma_s8(acc, w0.z, w1.z, w0.w, w1.w, x.z, x.w);
        }
      if (round + 1 < r.rounds) {
        load_weights<GATED>(w, b, e, N, K, s, round + 1, ks, part);
      } else if (u + teams < hi) {
        const int n = u + teams, nblk = n / r.strips;
        load_weights<GATED>(w, b, d.l.block_expert[nblk], N, K, n - nblk * r.strips, 0, ks, part);
      }
    }
    if (ks > 1) {
#pragma unroll
      for (int x = 0; x < 4; ++x) d.red[buf][warp][x][lane] = acc[x];
      named_bar_sync(1 + team, 32 * ks);
    }
    auto sum = [&](int x) {
      if (ks == 1) return acc[x];
      int v = 0;
      for (int y = 0; y < ks; ++y) v += d.red[buf][team * ks + y][x][lane];
      return v;
    };
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int col = 2 * q + t, pair = d.l.block_pair[blk][col];
      if (pair < 0) continue;
      if (GATED) {
        if (t % ks != part || ch0 >= width) continue;
        const float sa = d.scale[pair / a.k];
        const float gate = __int2float_rn(sum(t)) * sa * sb0, up = __int2float_rn(sum(2 + t)) * sa * sb1;
        a.h[static_cast<int64_t>(pair) * a.I + ch0] = silu_fp32(gate) * up;
      } else {
        const float sa = d.scale[8 * (blk - first) + col];
        float* o = a.y + static_cast<int64_t>(pair) * a.H;
        if (2 * t % ks == part && ch0 < width) o[ch0] = __int2float_rn(sum(t)) * sa * sb0;
        if ((2 * t + 1) % ks == part && c1 < width) o[c1] = __int2float_rn(sum(2 + t)) * sa * sb1;
      }
    }
    buf ^= 1;  // its readers are past the next unit's barrier before it is written again
    if (!GATED) decode_finish<T>(a, d, s, r);
  }
}

template <int VPT, typename T>
__global__ void __launch_bounds__(kDThreads, 1) decode_up_kernel(const __grid_constant__ DecodeArgs a) {
  extern __shared__ __align__(16) uint8_t codes[];
  __shared__ DecodeShared d;
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5;
  if (warp < kDTokens)
    decode_route<VPT>(a, d, warp);
  else
    quantise_into<T>([&](int m) { return static_cast<const T*>(a.x) + static_cast<int64_t>(m) * a.H; }, a.M, a.H,
                     codes, decode_pitch(a.H), d, warp - kDTokens, kDWarps - kDTokens);
  decode_lists(a, d);
  Weights w;
  int buf = 0;
  const Range up(d.l.blocks, (a.I + 7) / 8, a.H);
  decode_units<true, T>(a, d, up, up.lo, up.hi, 0, w, false, codes, buf);
  // what the down kernel needs, by the last CTA (whose range is never the longer one)
  if (blockIdx.x == gridDim.x - 1) {
    const int pairs = a.M * a.k, i = threadIdx.x;
    DecodeLists& o = *static_cast<DecodeLists*>(a.lists);
    if (i < pairs) {
      o.expert[i] = d.l.expert[i];
      o.weight[i] = d.l.weight[i];
      o.block_expert[i] = i < d.l.blocks ? d.l.block_expert[i] : 0;
    }
    for (int x = i; x < pairs * 8; x += kDThreads) o.block_pair[x / 8][x % 8] = d.l.block_pair[x / 8][x % 8];
    if (i == 0) o.blocks = d.l.blocks;
    for (int x = i; x < (a.H + 15) / 16; x += kDThreads) a.done[x] = 0;
  }
}

template <typename T>
__global__ void __launch_bounds__(kDThreads, 1) decode_down_kernel(const __grid_constant__ DecodeArgs a) {
  extern __shared__ __align__(16) uint8_t codes[];
  __shared__ DecodeShared d;
  const int warp = threadIdx.x >> 5, pairs = a.M * a.k, i = threadIdx.x;
  pdl_launch_dependents();
  pdl_wait();
  const DecodeLists& o = *static_cast<const DecodeLists*>(a.lists);
  if (i < pairs) {
    d.l.expert[i] = o.expert[i];
    d.l.weight[i] = o.weight[i];
    d.l.block_expert[i] = o.block_expert[i];
  }
  for (int x = i; x < pairs * 8; x += kDThreads) d.l.block_pair[x / 8][x % 8] = o.block_pair[x / 8][x % 8];
  if (i == kDThreads - 1) d.l.blocks = o.blocks;
  __syncthreads();
  if (d.l.blocks == 0) {  // no pair has an expert
    T* out = static_cast<T*>(a.out);
    for (int x = blockIdx.x * kDThreads + i; x < a.M * a.H; x += gridDim.x * kDThreads) out[x] = out_cast<T>(0.f);
    return;
  }
  Weights w;
  int buf = 0;
  const Range r(d.l.blocks, (a.H + 15) / 16, a.I);
  // two blocks at a time: their rows of h quantised, then their units
  for (int lo = r.lo; lo < r.hi;) {
    const int first = lo / r.strips, hi = min(r.hi, (first + 2) * r.strips);
    const int u = lo + warp / r.ks, blk = u / r.strips;
    if (u < hi)
      load_weights<false>(w, a.w2, d.l.block_expert[blk], a.H, a.I, u - blk * r.strips, 0, r.ks, warp % r.ks);
    const int rows = 8 * ((hi - 1) / r.strips - first) + 8;
    quantise_into<float>(
        [&](int m) {
          const int pair = d.l.block_pair[first + m / 8][m % 8];
          return pair >= 0 ? a.h + static_cast<int64_t>(pair) * a.I : static_cast<const float*>(nullptr);
        },
        rows, a.I, codes, decode_pitch(a.I), d, warp, kDWarps);
    __syncthreads();
    decode_units<false, T>(a, d, r, lo, hi, first, w, true, codes, buf);
    lo = hi;
    __syncthreads();  // the codes are read
  }
}

int launch(void (*kernel)(DecodeArgs), const DecodeArgs& a, int sms, size_t smem, cudaStream_t st) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(sms);
  cfg.blockDim = dim3(kDThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, a) != cudaSuccess) {
    cudaGetLastError();
    return MTP_ERR_LAUNCH;
  }
  return MTP_OK;
}

template <int VPT, typename T>
int run(const DecodeArgs& a, cudaStream_t st) {
  const int sms = device_sm_count();
  if (!sms) return MTP_ERR_CUDA;
  static DeviceRecord up, down;
  int rc = allow_shared(up, decode_up_kernel<VPT, T>, kDCodes);
  if (rc == MTP_OK) rc = allow_shared(down, decode_down_kernel<T>, kDCodes);
  if (rc != MTP_OK) return rc;
  rc = launch(decode_up_kernel<VPT, T>, a, sms, static_cast<size_t>(a.M) * decode_pitch(a.H), st);
  return rc != MTP_OK ? rc : launch(decode_down_kernel<T>, a, sms, kDRows * decode_pitch(a.I), st);
}

template <typename T>
int by_experts(const DecodeArgs& a, cudaStream_t st) {
  return a.E <= 256 ? run<8, T>(a, st) : run<32, T>(a, st);
}

}  // namespace

int64_t w8a8_decode_list_bytes() { return sizeof(DecodeLists); }

// Up to 100 MB of weights: beyond, streaming them at HBM's rate matters more than
// launches, and the tile kernels do that better. These kernels against those, us a
// call in a graph over four layers' weights: 2048 x 512, top-8 of 256, 1 token 17.1
// against 25.9, 4 tokens (96 MB at most) 30.2 and 35.2, 5 tokens 36.5 and 38.1, 6
// tokens 47.1 and 42.8; 2048 x 768, top-8 of 128, 2 tokens (72 MB) 25.7 and 32.3,
// 4 tokens (144 MB) 42.0 and 42.0, 5 tokens 47.0 and 45.0.
bool w8a8_decode_takes(int M, int H, int I, int E, int k) {
  return M <= kDTokens && std::min<int64_t>(static_cast<int64_t>(M) * k, E) * 3 * H * I <= (100ll << 20) && M * k <= kDPairs && H % 16 == 0 && I % 16 == 0 &&
         static_cast<int64_t>(M) * decode_pitch(H) <= kDCodes && static_cast<int64_t>(kDRows) * decode_pitch(I) <= kDCodes;
}

int launch_w8a8_decode(const DecodeArgs& a, int dtype, cudaStream_t st) {
  switch (dtype) {
    case MTP_DTYPE_BF16: return by_experts<__nv_bfloat16>(a, st);
    case MTP_DTYPE_FP16: return by_experts<__half>(a, st);
    default: return by_experts<float>(a, st);
  }
}

}  // namespace mtp
