// Declarations shared between the .cu files of libmtp_b200 (not part of the ABI).
#pragma once

#include "common.cuh"

namespace mtp {

// Work segment: kWsBlocks token block(s) of one expert (or of the shared
// expert), written by the route kernel and copied into shared memory by the
// fused kernel. 12 ints = 48 bytes (16-byte multiple). One block per segment
// lets every unit of a segment reuse the same operand rows.
constexpr int kWsBlocks = 1;
constexpr int kWsInts = 4 + 8 * kWsBlocks;
//   [0..1] expert blob address (0 = missing), [2] block count,
//   [3] flags (bit 0 shared expert, bit 1 blob in host memory),
//   [4..] pair ids (row of h / y), -1 for padding.

// One quantised x row: H high-digit bytes, H low-digit bytes, the per-group sums
// of the 16-bit values (int32, room for groups of 64), the row scale (fp32)
// and padding to 16 bytes. The meta travels with the row in one bulk copy.
__host__ __device__ constexpr uint32_t xq_row_bytes(int H) {
  return 2u * static_cast<uint32_t>(H) + static_cast<uint32_t>(H) / 16u + 16u;
}

// Device-side arguments of the fused layer kernel (moe_fused.cu).
struct FusedArgs {
  int M, H, I, E, k, numel, zero_mode, has_shared, G, renorm, max_ws;
  const uint16_t* x;
  const float* logits;       // [M, E] or NULL (topk_w / topk_ids given)
  const uint16_t* gate_w;    // [H] shared-expert gate or NULL
  float* topk_w;             // [M*k] written when logits != NULL
  int32_t* topk_ids;         // [M*k] local ids (written when logits != NULL or emap != NULL)
  const int32_t* topk_ids_in;  // [M*k] the caller's ids (global when emap != NULL)
  const int32_t* emap;       // [E_map] global -> local expert or -1; NULL: ids are local
  int E_map;
  int sh_begin, sh_end;      // rows that get the shared expert
  int32_t* wseg;             // [max_ws][kWsInts] spill area for large ranges
  MtpExpertLayout L;
  const uint8_t* blobs;
  int64_t expert_bytes;
  const int32_t* slot_table;
  const uint8_t* host_blobs;
  const uint8_t* shared_blob;
  float* gate;               // [M] sigmoid(x . w_g)
  uint8_t* xq;               // [M][xq_row_bytes(H)] quantised x rows, see xq_row_bytes
  int32_t* bar;              // [8] grid-barrier count, (unused),       \ zero before the first
                             //     CTAs done, dirty flag, timeouts seen |
  int32_t* cnt;              // [E] pairs per expert                    |  call; every call
  int32_t* seg_done;         // [max_ws] W1 units published per segment /  leaves them zero
  int32_t* lists;            // [E][M] pair ids per expert
  float* gu;                 // [numel + M][2I + 4] fp32 W1 sums per pair: gate | up, combine weight
  float* ybuf;
  uint16_t* out;
  float* out_f32;
  int32_t* status;
  int32_t* demand_log;
  int stages, sk;             // weight stages in the ring, K per stage
  uint32_t stage_bytes;
  uint32_t xbuf_bytes;
};

// Fixed counter regions of the layer workspace (see capi.cu layer_ws).
constexpr int kMaxExpertsWs = 1024;
constexpr int kMaxWorkSegments = 32768;

int launch_router_topk(const float* logits, int M, int E, int k, int renorm, float* w,
                       int32_t* ids, int32_t* tei, cudaStream_t st);
int launch_moe_align(const int32_t* ids, int numel, int E, int BM, const int32_t* emap,
                     int ignore_invalid, int cap, int max_blocks, int max_seg, int32_t* sorted,
                     int32_t* eids, int32_t* ntpp, int32_t* segs, int32_t* nseg, cudaStream_t st);
int expert_layout(int hidden, int inter, int G, MtpExpertLayout* out);
int repack_gptq(const int32_t* w13q, const int32_t* w13z, const uint16_t* w13s, const int32_t* w2q,
                const int32_t* w2z, const uint16_t* w2s, int E, int H, int I, int G, uint8_t* out,
                cudaStream_t st);
int gptq_dequant(const int32_t* q, const int32_t* z, const uint16_t* s, const int32_t* gidx, int K,
                 int N, int G, int zero_mode, float* out, cudaStream_t st);

int predictor_pack(const uint16_t* w, int rows, int cols, uint16_t* out, cudaStream_t st);
// K-splits of the predictor's linears are at most this (workspace sizing).
constexpr int kMaxPredictorKs = 8;
int predictor_run(const uint16_t* h, int M, int H, const uint16_t* w1p, const uint16_t* b1, int width,
                  const uint16_t* w2p, const uint16_t* b2, int F, int E, int k, float* logits, int32_t* ids,
                  float* part1, float* part2, cudaStream_t st);
int predictor_hr_run(const uint16_t* h, const int32_t* layer_ids, int M, int H, const uint16_t* w1p,
                     const uint16_t* b1, int width, const uint16_t* ln_w, const uint16_t* ln_b, float eps,
                     const uint16_t* layer_emb, int num_layers, const uint16_t* delta_emb, int F,
                     const uint16_t* wcp, const uint16_t* bc, int E, int k, float* logits, int32_t* ids, float* part1,
                     uint16_t* ctx, float* part2, cudaStream_t st);

bool fused_supported(int H, int I, int G);
int fused_max_work_segments(int M, int max_seg, int max_blocks);
int launch_moe_fused(const FusedArgs& a, cudaStream_t st);

// Prefill path (moe_prefill.cu): pairs per expert in blocks of 128.
struct PrefillArgs {
  int M, H, I, E, k, kx, numel_x, G, zero_mode, has_shared;
  int cap, max_blocks;         // sorted capacity and blocks (align sizes for 128-pair blocks)
  const uint16_t* x;           // [M, H] bf16
  const uint16_t* gate_w;      // [H] bf16 shared-expert gate or NULL
  const float* topk_w;         // [M, k]
  const int32_t* topk_ids;     // [M, k] (global ids when emap != NULL)
  const int32_t* emap;         // [E_map] global -> local expert or -1; NULL: ids are local
  int E_map;
  int sh_begin, sh_end;        // rows that get the shared expert
  int32_t* ids_x;              // [M, kx] pairs extended by the shared expert (id E)
  float* w_x;                  // [M, kx] pair weights (sigmoid gate for the shared expert)
  int32_t* inv;                // [M, kx] sorted position of each pair, -1 if not routed
  int32_t* sorted;             // [cap] align output
  int32_t* eids;               // [max_blocks] expert per block (E = shared)
  int32_t* ntpp;               // [1] positions used
  int32_t* pos_tok;            // [cap] token of each position, -1 for padding
  float* pos_w;                // [cap] weight of each position
  int32_t* blk_n;              // [max_blocks] valid columns rounded up to 16 (MMA N)
  int32_t* hist;               // [chunks][E (+1)] align: per-chunk counts, then offsets
  int32_t* ebase;              // [E (+1)] align: first position of each expert
  uint8_t* xg;                 // [max_blocks] blocks of x rows in the B-operand layout
  uint8_t* hg;                 // [max_blocks] blocks of h rows in the B-operand layout
  uint16_t* y;                 // [cap, H] bf16 W2 output times the pair weight
  MtpExpertLayout L;
  const uint8_t* blobs;
  int64_t expert_bytes;
  const uint8_t* shared_blob;
  uint16_t* out;
  float* out_f32;
  int32_t* status;
};

struct PrefillWs {
  int64_t cap, max_blocks, nchunks;
  int64_t tw, tid, ids_x, w_x, inv, sorted, eids, ntpp, pos_tok, pos_w, blk_n, hist, ebase, status, xg, hg, y, total;
};

PrefillWs prefill_ws(int M, int E, int k, int H, int I, int has_shared);
int launch_moe_prefill(PrefillArgs& a, int renorm, const float* logits, cudaStream_t st);

// SMs of the current device (0 when it cannot be asked).
inline int device_sm_count() {
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

// Lets a kernel use `bytes` of dynamic shared memory, once per device; `done` is
// the caller's record (static, one per kernel). Setting it twice does no harm.
struct DeviceRecord {
  bool done[64];
};
template <typename F>
int allow_shared(DeviceRecord& r, F* kernel, size_t bytes) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return MTP_ERR_CUDA;
  if (!r.done[dev]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)) !=
        cudaSuccess) {
      cudaGetLastError();
      return MTP_ERR_CUDA;
    }
    r.done[dev] = true;
  }
  return MTP_OK;
}

// Token sort and unsort (token_sort.cu). Strides and row sizes in bytes.
struct SortArgs {
  int M, k, E, E_map, numel;
  int64_t x_stride, row_bytes;  // row_bytes 0: positions and offsets only
  const uint8_t* x;
  const int32_t* ids;          // [M, k]
  const int32_t* emap;         // [E_map] or NULL
  const float* row_scales;     // [M] or NULL
  uint8_t* rows;               // [M * k] rows
  float* sorted_scales;        // [M * k] with row_scales
  int32_t* positions;          // [M, k]
  int32_t* offsets;            // [E + 1]
};
struct UnsortArgs {
  int M, k, H;
  int64_t num_rows;
  const void* rows;            // [num_rows, H]
  const int32_t* positions;    // [M, k]
  const float* weights;        // [M, k] or NULL (= 1)
  void* out;                   // forward: [M, H]
  const void* grad;            // backward: [M, H]
  void* grad_rows;             // [num_rows, H] or NULL
  float* grad_weights;         // [M, k] or NULL
};
int launch_sort_tokens(const SortArgs& a, cudaStream_t st);
int launch_unsort_tokens(const UnsortArgs& a, int dtype, cudaStream_t st);
int launch_unsort_fp32_rows(const UnsortArgs& a, int out_dtype, cudaStream_t st);  // rows fp32, out of out_dtype
int launch_unsort_backward(const UnsortArgs& a, int dtype, cudaStream_t st);

// The router with its losses (route_loss.cu).
struct RouteLossArgs {
  int M, E, k, renorm;
  int64_t stride;              // elements between the rows of logits
  const void* logits;          // [M, E]
  const uint8_t* mask;         // [M] or NULL: tokens that count
  float* weights;              // [M, k]
  int32_t* ids;                // [M, k]
  int32_t* counts;             // [E]
  float* balance;
  float* z_loss;
  float* pull;                 // [E + 1] for the gradient (or NULL): E counts[e] / (k n^2), then 2 / n
  float* part_load;            // [parts, E]
  int32_t* part_count;         // [parts, E]
  double* part_sums;           // [parts, 2]: lse^2, tokens
  const int32_t* ids_in;       // backward: [M, k]
  const float* grad_weights;   // [M, k] or NULL
  const float* grad_balance;   // [1] or NULL
  const float* grad_z_loss;    // [1] or NULL
  void* grad_logits;           // [M, E]
};
int64_t route_loss_parts(int M, int E);
int launch_route_loss(const RouteLossArgs& a, int dtype, cudaStream_t st);
int launch_route_loss_backward(const RouteLossArgs& a, int dtype, cudaStream_t st);

// Layer norm (layer_norm.cu). param_fp32: weight, bias and their gradients are fp32, else of the rows' type.
struct NormArgs {
  int M, H;
  bool param_fp32;
  float eps;
  int64_t stride;              // elements between the rows of x
  const void* x;               // [M, H]
  const void* weight;          // [H] or NULL (= 1)
  const void* bias;            // [H] or NULL (= 0)
  void* y;                     // [M, H]
  float* stats;                // [M, 2] mean, 1 / sqrt(var + eps); forward: or NULL
  const void* grad;            // [M, H]
  void* grad_x;                // [M, H] or NULL
  void* grad_weight;           // [H] or NULL
  void* grad_bias;             // [H] or NULL
  float* parts;                // [layer_norm_parts, 2, H]
};
int64_t layer_norm_parts(int M, int H);
int launch_layer_norm(const NormArgs& a, int dtype, cudaStream_t st);
int launch_layer_norm_backward(const NormArgs& a, int dtype, cudaStream_t st);

// Embedding (embedding.cu).
struct EmbedArgs {
  int N, V, H;
  bool wide_ids;               // int64 ids, else int32
  float scale;
  const void* ids;             // [N]
  const void* table;           // [V, H]
  void* out;                   // [N, H]
  const void* grad;            // [N, H]
  void* grad_table;            // [V, H]
  int chunk;                   // sorted tokens that a warp sums, and what embed_workspace lays out:
  int32_t* valid;              // [2] tokens whose id is a row; entries of owners
  int32_t* owners;             // [chunks] chunks in which a row begins that reaches over chunks
  int32_t* keys;               // [2][N] their ids in order, and a buffer
  int32_t* order;              // [2][N] their tokens
  float* parts;                // [chunks][2][H] sums of rows that reach over chunks
};
struct EmbedWs {
  int chunk;
  int64_t valid, owners, keys, order, parts, total;
};
EmbedWs embed_workspace(int N, int H, int dtype);
int launch_embed(const EmbedArgs& a, int dtype, cudaStream_t st);
int launch_embed_backward(const EmbedArgs& a, int dtype, cudaStream_t st);

// Rows to int8 (quantize.cu); strides in elements.
int launch_quantize_int8(const void* x, int64_t x_stride, int dtype, int M, int K, int8_t* q, int64_t q_stride,
                         float* scale, cudaStream_t st);

// Contiguous rows to int8 and their tokens' top-k (route_token).
int launch_route_quantize(const void* x, int dtype, int M, int K, int8_t* q, int64_t q_stride, float* scale,
                          const float* logits, int E, int k, int renorm, float* weights, int32_t* ids,
                          cudaStream_t st);

// int8 products (int8_matmul.cu).
struct Int8Args {
  int P, N, K, E;              // rows, rows of b per group, K, groups
  int ctiles;                  // channel tiles (set by the launcher)
  const float* a_scale;        // [P]
  const float* b_scale;        // [E, N]
  const float* bias;           // [N] or NULL
  const int32_t* offsets;      // [E + 1] or NULL (one group of all rows)
  void* out;                   // [P, N] or, gated, [P, N / 2]
  int32_t* status;             // [1] or NULL: bit 0 set when a wait ran out
};
bool tma_rows_ok(const void* base, int64_t stride);
// Rows into a layout that TMA and 16-byte loads take (quantize.cu): zeros from K
// to dst_stride, a multiple of 16. rows 0: nothing.
struct PadJob {
  const int8_t* src;
  int64_t stride, rows;
  int K;
  int8_t* dst;
  int64_t dst_stride;
};
int launch_pad_rows(const PadJob& a, const PadJob& b, cudaStream_t st);
// Rows to int8 as launch_quantize_int8, and other rows padded.
int launch_quantize_and_pad(const void* x, int64_t x_stride, int dtype, int M, int K, int8_t* q, int64_t q_stride,
                            float* scale, const PadJob& pad, cudaStream_t st);
// a_padded: ap is a workspace whose rows may be read up to a multiple of 16.
int launch_int8_matmul(Int8Args a, bool gated, int out_dtype, const void* ap, int64_t a_stride, bool a_padded,
                       const void* bp, int64_t b_stride, cudaStream_t st);
// A few rows of one group (int8_stream.cu), given as codes or quantised in the
// same kernel.
bool int8_stream_takes(int rows);
int launch_int8_stream(Int8Args a, int out_dtype, const void* ap, int64_t a_stride, const void* bp, int64_t b_stride,
                       cudaStream_t st);
bool int8_stream_quantises(int rows, int K);
int launch_int8_stream_quantise(Int8Args a, int out_dtype, const void* x, int64_t x_stride, int x_dtype, const void* bp,
                                int64_t b_stride, cudaStream_t st);

// The W8A8 layer of a few tokens (w8a8_decode.cu). Rows and
// weights start on 16 bytes.
struct DecodeArgs {
  int M, H, I, E, k, renorm, E_map;
  const void* x;               // [M, H]
  const float* logits;         // [M, E] or NULL
  const float* topk_weights;   // [M, k] without logits
  const int32_t* topk_ids;
  const int32_t* emap;         // [E_map] or NULL
  const int8_t* w13;           // [E, 2I, H]
  const float* s13;
  const int8_t* w2;            // [E, H, I]
  const float* s2;
  float* h;                    // [M * k, I]
  float* y;                    // [M * k, H]
  void* out;                   // [M, H]
  void* lists;                 // w8a8_decode_list_bytes
  int32_t* done;               // [H / 16] blocks whose strip of y is written
};
int64_t w8a8_decode_list_bytes();
bool w8a8_decode_takes(int M, int H, int I, int E, int k);
int launch_w8a8_decode(const DecodeArgs& a, int dtype, cudaStream_t st);

}  // namespace mtp
