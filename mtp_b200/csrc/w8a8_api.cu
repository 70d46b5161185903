// extern "C" entry points of the token sort and the int8 (W8A8) products:
// argument checks, workspace carving, launch order. Nothing throws.
#include "internal.cuh"

using namespace mtp;

namespace {

bool float_dtype(int d) { return d == MTP_DTYPE_BF16 || d == MTP_DTYPE_FP16 || d == MTP_DTYPE_FP32; }
int64_t dtype_bytes(int d) { return d == MTP_DTYPE_FP32 ? 4 : d == MTP_DTYPE_INT8 ? 1 : 2; }

struct Carver {
  int64_t at = 0;
  int64_t take(int64_t bytes) {
    const int64_t o = at;
    at = round_up(at + bytes, 256);
    return o;
  }
};

constexpr int kMaxK = 131071;  // 128 * 128 * k stays below 2^31
// Rows, columns, pairs and channels of a call: the kernels index them in 32
// bits, and their loops step past the last one by up to 32768.
constexpr int64_t kMaxExtent = 0x7fffffffll - 0xffff;
bool extent(int64_t n) { return n >= 0 && n <= kMaxExtent; }

struct MatmulWs {
  int64_t codes, scales, b, total;  // -1: not needed
  int64_t kp;
  bool fused;  // quantised by the product kernel
};

int matmul_shapes(const MtpInt8MatmulArgs& a) {
  if (!extent(a.rows) || a.n < 1 || a.k < 1 || a.k > kMaxK) return MTP_ERR_SHAPE;
  if (a.num_groups < 1 || a.num_groups > 1024 || (!a.offsets && a.num_groups != 1)) return MTP_ERR_SHAPE;
  if (!extent(static_cast<int64_t>(a.num_groups) * a.n) || a.a_stride < (a.rows > 1 ? a.k : 0))
    return MTP_ERR_SHAPE;
  if ((a.a_dtype != MTP_DTYPE_INT8 && !float_dtype(a.a_dtype)) || !float_dtype(a.out_dtype)) return MTP_ERR_ARG;
  if (a.activation != MTP_ACT_NONE && a.activation != MTP_ACT_SILU_MUL) return MTP_ERR_ARG;
  if (a.activation == MTP_ACT_SILU_MUL && (a.n % 2 || a.bias)) return MTP_ERR_SHAPE;
  return MTP_OK;
}

MatmulWs matmul_ws(const MtpInt8MatmulArgs& a) {
  MatmulWs w;
  Carver c;
  w.kp = round_up(a.k, 16);
  w.codes = w.scales = w.b = -1;
  const bool quantise = a.a_dtype != MTP_DTYPE_INT8;
  w.fused = quantise && !a.offsets && a.activation == MTP_ACT_NONE && int8_stream_quantises(a.rows, a.k);
  if (!w.fused && (quantise || !tma_rows_ok(a.a, a.rows > 1 ? a.a_stride : 0))) w.codes = c.take(w.kp * a.rows);
  if (!w.fused && quantise) w.scales = c.take(4ll * a.rows);
  if (!tma_rows_ok(a.b, a.k)) w.b = c.take(w.kp * a.num_groups * a.n);
  w.total = c.at;
  return w;
}

}  // namespace

extern "C" {

int mtp_sort_tokens(const void* x, int64_t x_stride, int32_t dtype, int32_t M, int32_t H, const int32_t* topk_ids,
                    int32_t k, int32_t num_experts, const int32_t* expert_map, int32_t global_num_experts,
                    const float* row_scales, void* rows, float* sorted_scales, int32_t* positions, int32_t* offsets,
                    void* stream) {
  if (!offsets || (M > 0 && (!topk_ids || !positions)) || (x && M > 0 && !rows) || (row_scales && !sorted_scales))
    return MTP_ERR_NULL;
  if (M < 0 || !extent(H) || k < 1 || k > 32 || num_experts < 1 || num_experts > 1024 ||
      !extent(static_cast<int64_t>(M) * k) || (expert_map && global_num_experts < 1) || (x && x_stride < 0))
    return MTP_ERR_SHAPE;
  if (!float_dtype(dtype) && dtype != MTP_DTYPE_INT8) return MTP_ERR_ARG;
  const int64_t size = dtype_bytes(dtype);
  if ((x && !aligned(x, size)) || (rows && !aligned(rows, size))) return MTP_ERR_ALIGN;
  SortArgs a = {};
  a.M = M;
  a.k = k;
  a.E = num_experts;
  a.E_map = global_num_experts;
  a.numel = M * k;
  a.x_stride = x_stride * size;
  a.row_bytes = x ? H * size : 0;
  a.x = static_cast<const uint8_t*>(x);
  a.ids = topk_ids;
  a.emap = expert_map;
  a.row_scales = row_scales;
  a.rows = static_cast<uint8_t*>(rows);
  a.sorted_scales = sorted_scales;
  a.positions = positions;
  a.offsets = offsets;
  return launch_sort_tokens(a, static_cast<cudaStream_t>(stream));
}

static int unsort_shapes(int64_t num_rows, int32_t dtype, int32_t M, int32_t k, int32_t H) {
  if (M < 0 || !extent(H) || k < 1 || k > 32 || !extent(num_rows) || !extent(static_cast<int64_t>(M) * k))
    return MTP_ERR_SHAPE;
  return float_dtype(dtype) ? MTP_OK : MTP_ERR_ARG;
}

int mtp_unsort_tokens(const void* rows, int64_t num_rows, int32_t dtype, const int32_t* positions,
                      const float* weights, int32_t M, int32_t k, int32_t H, void* out, void* stream) {
  const int rc = unsort_shapes(num_rows, dtype, M, k, H);
  if (rc != MTP_OK) return rc;
  if (M == 0 || H == 0) return MTP_OK;
  if (!positions || !out || (!rows && num_rows > 0)) return MTP_ERR_NULL;
  if (!aligned(rows, dtype_bytes(dtype)) || !aligned(out, dtype_bytes(dtype))) return MTP_ERR_ALIGN;
  UnsortArgs a = {};
  a.M = M;
  a.k = k;
  a.H = H;
  a.num_rows = num_rows;
  a.rows = rows;
  a.positions = positions;
  a.weights = weights;
  a.out = out;
  return launch_unsort_tokens(a, dtype, static_cast<cudaStream_t>(stream));
}

int mtp_unsort_tokens_backward(const void* grad, const void* rows, int64_t num_rows, int32_t dtype,
                               const int32_t* positions, const float* weights, int32_t M, int32_t k, int32_t H,
                               void* grad_rows, float* grad_weights, void* stream) {
  const int rc = unsort_shapes(num_rows, dtype, M, k, H);
  if (rc != MTP_OK) return rc;
  if (M == 0 || (!grad_rows && !grad_weights)) return MTP_OK;
  if (!positions || (!grad && H > 0) || (grad_weights && !rows && H > 0 && num_rows > 0)) return MTP_ERR_NULL;
  const int64_t size = dtype_bytes(dtype);
  if (!aligned(rows, size) || !aligned(grad, size) || !aligned(grad_rows, size)) return MTP_ERR_ALIGN;
  UnsortArgs a = {};
  a.M = M;
  a.k = k;
  a.H = H;
  a.num_rows = num_rows;
  a.rows = rows;
  a.positions = positions;
  a.weights = weights;
  a.grad = grad;
  a.grad_rows = grad_rows;
  a.grad_weights = grad_weights;
  return launch_unsort_backward(a, dtype, static_cast<cudaStream_t>(stream));
}

int mtp_quantize_int8(const void* x, int64_t x_stride, int32_t dtype, int32_t M, int32_t K, int8_t* q,
                      int64_t q_stride, float* scale, void* stream) {
  if (!extent(M) || K < 1 || !extent(K) || x_stride < 0 || q_stride < (M > 1 ? K : 0)) return MTP_ERR_SHAPE;
  if (!float_dtype(dtype)) return MTP_ERR_ARG;
  if (M == 0) return MTP_OK;
  if (!x || !q || !scale) return MTP_ERR_NULL;
  if (!aligned(x, dtype_bytes(dtype))) return MTP_ERR_ALIGN;
  return launch_quantize_int8(x, x_stride, dtype, M, K, q, q_stride, scale, static_cast<cudaStream_t>(stream));
}

int mtp_int8_matmul_workspace_size(const MtpInt8MatmulArgs* args, int64_t* bytes) {
  if (!args || !bytes) return MTP_ERR_NULL;
  const int rc = matmul_shapes(*args);
  if (rc != MTP_OK) return rc;
  *bytes = matmul_ws(*args).total;
  return MTP_OK;
}

int mtp_int8_matmul(const MtpInt8MatmulArgs* args, void* stream) {
  if (!args) return MTP_ERR_NULL;
  const MtpInt8MatmulArgs& p = *args;
  int rc = matmul_shapes(p);
  if (rc != MTP_OK) return rc;
  if (p.rows == 0) return MTP_OK;
  const bool quantise = p.a_dtype != MTP_DTYPE_INT8;
  if (!p.a || !p.b || !p.b_scale || !p.out || (!quantise && !p.a_scale)) return MTP_ERR_NULL;
  if (!aligned(p.a, dtype_bytes(p.a_dtype)) || !aligned(p.out, dtype_bytes(p.out_dtype)) ||
      (p.workspace && !aligned(p.workspace, 256)))
    return MTP_ERR_ALIGN;
  const MatmulWs w = matmul_ws(p);
  if (w.total > 0 && !p.workspace) return MTP_ERR_NULL;
  if (p.workspace_bytes < w.total) return MTP_ERR_WORKSPACE;
  uint8_t* ws = static_cast<uint8_t*>(p.workspace);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const void* ap = p.a;
  const void* bp = p.b;
  int64_t a_stride = p.rows > 1 ? p.a_stride : w.kp, b_stride = p.k;
  const float* a_scale = p.a_scale;
  PadJob pad_a = {}, pad_b = {};
  if (w.b >= 0) {
    pad_b = {p.b, p.k, static_cast<int64_t>(p.num_groups) * p.n, p.k, reinterpret_cast<int8_t*>(ws + w.b), w.kp};
    bp = ws + w.b;
    b_stride = w.kp;
  }
  if (w.codes >= 0) {
    int8_t* codes = reinterpret_cast<int8_t*>(ws + w.codes);
    if (quantise) {
      float* scales = reinterpret_cast<float*>(ws + w.scales);
      rc = launch_quantize_and_pad(p.a, p.a_stride, p.a_dtype, p.rows, p.k, codes, w.kp, scales, pad_b, st);
      if (rc != MTP_OK) return rc;
      pad_b.rows = 0;
      a_scale = scales;
    } else {
      pad_a = {static_cast<const int8_t*>(p.a), a_stride, p.rows, p.k, codes, w.kp};
    }
    ap = codes;
    a_stride = w.kp;
  }
  rc = launch_pad_rows(pad_a, pad_b, st);
  if (rc != MTP_OK) return rc;
  Int8Args a = {};
  a.P = p.rows;
  a.N = p.n;
  a.K = p.k;
  a.E = p.num_groups;
  a.a_scale = a_scale;
  a.b_scale = p.b_scale;
  a.bias = p.bias;
  a.offsets = p.offsets;
  a.out = p.out;
  a.status = p.status;
  if (w.fused) return launch_int8_stream_quantise(a, p.out_dtype, p.a, p.a_stride, p.a_dtype, bp, b_stride, st);
  return launch_int8_matmul(a, p.activation == MTP_ACT_SILU_MUL, p.out_dtype, ap, a_stride, w.codes >= 0, bp, b_stride,
                            st);
}

}  // extern "C"

namespace {

struct LayerWs8 {
  int64_t tw, tid, xq, xs, rows, rs, positions, offsets, h, hq, hs, y, w13, w2, lists, done, total;
  int64_t hp, ip;
  bool decode;  // the kernels for a few tokens
};

int layer_shapes(const MtpW8A8LayerArgs& a) {
  if (a.num_tokens < 0 || a.hidden < 1 || a.hidden > kMaxK || a.inter < 1 || a.inter > kMaxK / 2 || a.num_experts < 1 ||
      a.num_experts > 1024 || a.top_k < 1 || a.top_k > 32)
    return MTP_ERR_SHAPE;
  if (a.router_logits && a.top_k > a.num_experts) return MTP_ERR_SHAPE;
  if (!extent(static_cast<int64_t>(a.num_tokens) * a.top_k) || !extent(static_cast<int64_t>(a.num_experts) * 2 * a.inter) ||
      !extent(static_cast<int64_t>(a.num_experts) * a.hidden))
    return MTP_ERR_SHAPE;
  if (a.expert_map) {
    if (a.router_logits) return MTP_ERR_ARG;
    if (a.global_num_experts < 1) return MTP_ERR_SHAPE;
  }
  return float_dtype(a.dtype) ? MTP_OK : MTP_ERR_ARG;
}

LayerWs8 layer_ws8(const MtpW8A8LayerArgs& a) {
  LayerWs8 w = {};
  Carver c;
  const int64_t m = a.num_tokens, p = m * a.top_k;
  w.hp = round_up(a.hidden, 16);
  w.ip = round_up(a.inter, 16);
  w.decode = w8a8_decode_takes(a.num_tokens, a.hidden, a.inter, a.num_experts, a.top_k) && aligned(a.hidden_states, 16) &&
             tma_rows_ok(a.w13, a.hidden) && tma_rows_ok(a.w2, a.inter);
  if (w.decode) {
    w.h = c.take(4 * p * a.inter);
    w.y = c.take(4 * p * a.hidden);
    w.lists = c.take(w8a8_decode_list_bytes());
    w.done = c.take(4ll * (a.hidden / 16));
    w.total = c.at;
    return w;
  }
  w.tw = c.take(a.router_logits ? 4 * p : 0);
  w.tid = c.take(a.router_logits ? 4 * p : 0);
  w.xq = c.take(m * w.hp);
  w.xs = c.take(4 * m);
  w.rows = c.take(p * w.hp);
  w.rs = c.take(4 * p);
  w.positions = c.take(4 * p);
  w.offsets = c.take(4ll * (a.num_experts + 1));
  w.h = c.take(4 * p * a.inter);
  w.hq = c.take(p * w.ip);
  w.hs = c.take(4 * p);
  w.y = c.take(4 * p * a.hidden);
  w.w13 = tma_rows_ok(a.w13, a.hidden) ? -1 : c.take(2ll * a.num_experts * a.inter * w.hp);
  w.w2 = tma_rows_ok(a.w2, a.inter) ? -1 : c.take(static_cast<int64_t>(a.num_experts) * a.hidden * w.ip);
  w.total = c.at;
  return w;
}

}  // namespace

extern "C" {

int mtp_w8a8_moe_layer_workspace_size(const MtpW8A8LayerArgs* args, int64_t* bytes) {
  if (!args || !bytes) return MTP_ERR_NULL;
  const int rc = layer_shapes(*args);
  if (rc != MTP_OK) return rc;
  *bytes = layer_ws8(*args).total;
  return MTP_OK;
}

int mtp_w8a8_moe_layer(const MtpW8A8LayerArgs* args, void* stream) {
  if (!args) return MTP_ERR_NULL;
  const MtpW8A8LayerArgs& p = *args;
  int rc = layer_shapes(p);
  if (rc != MTP_OK) return rc;
  if (p.num_tokens == 0) return MTP_OK;
  if (!p.hidden_states || !p.w13 || !p.w13_scale || !p.w2 || !p.w2_scale || !p.out || !p.workspace ||
      (!p.router_logits && (!p.topk_weights || !p.topk_ids)))
    return MTP_ERR_NULL;
  const int64_t size = dtype_bytes(p.dtype);
  if (!aligned(p.hidden_states, size) || !aligned(p.out, size) || !aligned(p.workspace, 256)) return MTP_ERR_ALIGN;
  const LayerWs8 w = layer_ws8(p);
  if (p.workspace_bytes < w.total) return MTP_ERR_WORKSPACE;
  uint8_t* ws = static_cast<uint8_t*>(p.workspace);
  auto f32 = [&](int64_t o) { return reinterpret_cast<float*>(ws + o); };
  auto i32 = [&](int64_t o) { return reinterpret_cast<int32_t*>(ws + o); };
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int M = p.num_tokens, H = p.hidden, I = p.inter, E = p.num_experts, k = p.top_k;
  const int P = M * k;

  if (w.decode) {
    DecodeArgs d = {};
    d.M = M;
    d.H = H;
    d.I = I;
    d.E = E;
    d.k = k;
    d.renorm = p.renormalize ? 1 : 0;
    d.E_map = p.global_num_experts;
    d.x = p.hidden_states;
    d.logits = p.router_logits;
    d.topk_weights = p.topk_weights;
    d.topk_ids = p.topk_ids;
    d.emap = p.expert_map;
    d.w13 = p.w13;
    d.s13 = p.w13_scale;
    d.w2 = p.w2;
    d.s2 = p.w2_scale;
    d.h = f32(w.h);
    d.y = f32(w.y);
    d.out = p.out;
    d.lists = ws + w.lists;
    d.done = i32(w.done);
    return launch_w8a8_decode(d, p.dtype, st);
  }

  const float* weights = p.topk_weights;
  const int32_t* ids = p.topk_ids;
  int8_t* xq = reinterpret_cast<int8_t*>(ws + w.xq);
  if (p.router_logits) {
    rc = launch_route_quantize(p.hidden_states, p.dtype, M, H, xq, w.hp, f32(w.xs), p.router_logits, E, k,
                               p.renormalize ? 1 : 0, f32(w.tw), i32(w.tid), st);
    weights = f32(w.tw);
    ids = i32(w.tid);
  } else {
    rc = launch_quantize_int8(p.hidden_states, H, p.dtype, M, H, xq, w.hp, f32(w.xs), st);
  }
  if (rc != MTP_OK) return rc;

  SortArgs s = {};
  s.M = M;
  s.k = k;
  s.E = E;
  s.E_map = p.global_num_experts;
  s.numel = P;
  s.x_stride = s.row_bytes = w.hp;
  s.x = ws + w.xq;
  s.ids = ids;
  s.emap = p.expert_map;
  s.row_scales = f32(w.xs);
  s.rows = ws + w.rows;
  s.sorted_scales = f32(w.rs);
  s.positions = i32(w.positions);
  s.offsets = i32(w.offsets);
  rc = launch_sort_tokens(s, st);
  if (rc != MTP_OK) return rc;

  const void* w13 = p.w13;
  const void* w2 = p.w2;
  int64_t w13_stride = H, w2_stride = I;
  PadJob pad13 = {}, pad2 = {};
  if (w.w13 >= 0) {
    pad13 = {p.w13, H, 2ll * E * I, H, reinterpret_cast<int8_t*>(ws + w.w13), w.hp};
    w13 = ws + w.w13;
    w13_stride = w.hp;
  }
  if (w.w2 >= 0) {
    pad2 = {p.w2, I, static_cast<int64_t>(E) * H, I, reinterpret_cast<int8_t*>(ws + w.w2), w.ip};
    w2 = ws + w.w2;
    w2_stride = w.ip;
  }
  rc = launch_pad_rows(pad13, pad2, st);
  if (rc != MTP_OK) return rc;

  Int8Args g = {};
  g.P = P;
  g.N = 2 * I;
  g.K = H;
  g.E = E;
  g.a_scale = f32(w.rs);
  g.b_scale = p.w13_scale;
  g.offsets = i32(w.offsets);
  g.out = f32(w.h);
  g.status = p.status;
  rc = launch_int8_matmul(g, true, MTP_DTYPE_FP32, ws + w.rows, w.hp, true, w13, w13_stride, st);
  if (rc != MTP_OK) return rc;
  rc = launch_quantize_int8(f32(w.h), I, MTP_DTYPE_FP32, P, I, reinterpret_cast<int8_t*>(ws + w.hq), w.ip, f32(w.hs),
                            st);
  if (rc != MTP_OK) return rc;
  g.N = H;
  g.K = I;
  g.a_scale = f32(w.hs);
  g.b_scale = p.w2_scale;
  g.out = ws + w.y;
  // y in fp32, as the few-token kernels hold it: an fp16 pair may pass 65504 where the weighted sum does
  // not, and a token's result does not depend on the others of its call
  rc = launch_int8_matmul(g, false, MTP_DTYPE_FP32, ws + w.hq, w.ip, true, w2, w2_stride, st);
  if (rc != MTP_OK) return rc;

  UnsortArgs u = {};
  u.M = M;
  u.k = k;
  u.H = H;
  u.num_rows = P;
  u.rows = ws + w.y;
  u.positions = i32(w.positions);
  u.weights = weights;
  u.out = p.out;
  return launch_unsort_fp32_rows(u, p.dtype, st);
}

}  // extern "C"
