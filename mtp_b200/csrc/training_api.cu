// extern "C" entry points of a training step's operators (router with losses,
// layer norm, embedding): argument checks, workspace carving. Nothing throws.
#include "internal.cuh"

using namespace mtp;

namespace {

bool float_dtype(int d) { return d == MTP_DTYPE_BF16 || d == MTP_DTYPE_FP16 || d == MTP_DTYPE_FP32; }
int64_t dtype_bytes(int d) { return d == MTP_DTYPE_FP32 ? 4 : 2; }
// Rows, columns and tokens of a call: the kernels index them in 32 bits, and
// their loops step past the last one by up to 32768.
bool extent(int64_t n) { return n >= 0 && n <= 0x7fffffffll - 0xffff; }

struct RouteWs {
  int64_t load, count, sums, total;
};
RouteWs route_ws(int M, int E) {
  const int64_t parts = route_loss_parts(M, E);
  RouteWs w;
  w.load = 0;
  w.count = round_up(4 * parts * E, 256);
  w.sums = 2 * w.count;
  w.total = w.sums + 16 * parts;
  return w;
}

int route_shapes(int64_t stride, int32_t dtype, int32_t M, int32_t E, int32_t k) {
  if (E < 1 || E > 1024 || k < 1 || k > 32 || k > E || M < 0 || !extent(static_cast<int64_t>(M) * k) ||
      stride < (M > 1 ? E : 0))
    return MTP_ERR_SHAPE;
  return float_dtype(dtype) ? MTP_OK : MTP_ERR_ARG;
}

int norm_shapes(int64_t stride, int32_t dtype, int32_t M, int32_t H, int32_t param_dtype) {
  if (!extent(M) || H < 1 || !extent(H) || stride < (M > 1 ? H : 0)) return MTP_ERR_SHAPE;
  return float_dtype(dtype) && (param_dtype == dtype || param_dtype == MTP_DTYPE_FP32) ? MTP_OK : MTP_ERR_ARG;
}

int embed_shapes(int32_t id_bytes, int32_t N, int32_t dtype, int32_t V, int32_t H) {
  if (!extent(N) || V < 1 || !extent(V) || H < 1 || !extent(H)) return MTP_ERR_SHAPE;
  return float_dtype(dtype) && (id_bytes == 4 || id_bytes == 8) ? MTP_OK : MTP_ERR_ARG;
}

}  // namespace

extern "C" {

int mtp_route_tokens_workspace_size(int32_t M, int32_t num_experts, int64_t* bytes) {
  if (!bytes) return MTP_ERR_NULL;
  if (!extent(M) || num_experts < 1 || num_experts > 1024) return MTP_ERR_SHAPE;
  *bytes = route_ws(M, num_experts).total;
  return MTP_OK;
}

int mtp_route_tokens(const void* logits, int64_t logits_stride, int32_t dtype, int32_t M, int32_t num_experts,
                     int32_t k, int32_t renormalize, const uint8_t* token_mask, float* weights, int32_t* ids,
                     int32_t* counts, float* balance_loss, float* z_loss, float* pull, void* workspace,
                     int64_t workspace_bytes, void* stream) {
  const int rc = route_shapes(logits_stride, dtype, M, num_experts, k);
  if (rc != MTP_OK) return rc;
  if (!counts || !balance_loss || !z_loss || (M > 0 && (!logits || !weights || !ids))) return MTP_ERR_NULL;
  if (!aligned(logits, dtype_bytes(dtype))) return MTP_ERR_ALIGN;
  const RouteWs w = route_ws(M, num_experts);
  if (w.total > 0 && !workspace) return MTP_ERR_NULL;
  if (workspace_bytes < w.total) return MTP_ERR_WORKSPACE;
  if (!aligned(workspace, 256)) return MTP_ERR_ALIGN;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  RouteLossArgs a = {};
  a.M = M;
  a.E = num_experts;
  a.k = k;
  a.renorm = renormalize;
  a.stride = logits_stride;
  a.logits = logits;
  a.mask = token_mask;
  a.weights = weights;
  a.ids = ids;
  a.counts = counts;
  a.balance = balance_loss;
  a.z_loss = z_loss;
  a.pull = pull;
  a.part_load = reinterpret_cast<float*>(ws + w.load);
  a.part_count = reinterpret_cast<int32_t*>(ws + w.count);
  a.part_sums = reinterpret_cast<double*>(ws + w.sums);
  return launch_route_loss(a, dtype, static_cast<cudaStream_t>(stream));
}

int mtp_route_tokens_backward(const void* logits, int64_t logits_stride, int32_t dtype, int32_t M,
                              int32_t num_experts, int32_t k, int32_t renormalize, const uint8_t* token_mask,
                              const int32_t* ids, const float* pull, const float* grad_weights,
                              const float* grad_balance_loss, const float* grad_z_loss, void* grad_logits,
                              void* stream) {
  const int rc = route_shapes(logits_stride, dtype, M, num_experts, k);
  if (rc != MTP_OK) return rc;
  if (M == 0) return MTP_OK;
  if (!logits || !grad_logits || (grad_weights && !ids) || ((grad_balance_loss || grad_z_loss) && !pull))
    return MTP_ERR_NULL;
  if (!aligned(logits, dtype_bytes(dtype)) || !aligned(grad_logits, dtype_bytes(dtype))) return MTP_ERR_ALIGN;
  RouteLossArgs a = {};
  a.M = M;
  a.E = num_experts;
  a.k = k;
  a.renorm = renormalize;
  a.stride = logits_stride;
  a.logits = logits;
  a.mask = token_mask;
  a.pull = const_cast<float*>(pull);
  a.ids_in = ids;
  a.grad_weights = grad_weights;
  a.grad_balance = grad_balance_loss;
  a.grad_z_loss = grad_z_loss;
  a.grad_logits = grad_logits;
  return launch_route_loss_backward(a, dtype, static_cast<cudaStream_t>(stream));
}

int mtp_layer_norm(const void* x, int64_t x_stride, int32_t dtype, int32_t M, int32_t H, const void* weight,
                   const void* bias, int32_t param_dtype, float eps, void* y, float* stats, void* stream) {
  const int rc = norm_shapes(x_stride, dtype, M, H, param_dtype);
  if (rc != MTP_OK) return rc;
  if (!(eps >= 0.f)) return MTP_ERR_ARG;
  if (M == 0) return MTP_OK;
  if (!x || !y) return MTP_ERR_NULL;
  const int64_t size = dtype_bytes(dtype), psize = dtype_bytes(param_dtype);
  if (!aligned(x, size) || !aligned(y, size) || !aligned(weight, psize) || !aligned(bias, psize) || !aligned(stats, 8))
    return MTP_ERR_ALIGN;
  NormArgs a = {};
  a.M = M;
  a.H = H;
  a.param_fp32 = param_dtype == MTP_DTYPE_FP32;
  a.eps = eps;
  a.stride = x_stride;
  a.x = x;
  a.weight = weight;
  a.bias = bias;
  a.y = y;
  a.stats = stats;
  return launch_layer_norm(a, dtype, static_cast<cudaStream_t>(stream));
}

int mtp_layer_norm_backward_workspace_size(int32_t M, int32_t H, int64_t* bytes) {
  if (!bytes) return MTP_ERR_NULL;
  if (!extent(M) || H < 1 || !extent(H)) return MTP_ERR_SHAPE;
  *bytes = 8 * layer_norm_parts(M, H) * H;
  return MTP_OK;
}

int mtp_layer_norm_backward(const void* grad, const void* x, int64_t x_stride, int32_t dtype, int32_t M, int32_t H,
                            const void* weight, int32_t param_dtype, const float* stats, void* grad_x,
                            void* grad_weight, void* grad_bias, void* workspace, int64_t workspace_bytes,
                            void* stream) {
  const int rc = norm_shapes(x_stride, dtype, M, H, param_dtype);
  if (rc != MTP_OK) return rc;
  if (!grad_x && !grad_weight && !grad_bias) return MTP_OK;
  if (M > 0 && (!grad || !x || !stats)) return MTP_ERR_NULL;
  const int64_t size = dtype_bytes(dtype), psize = dtype_bytes(param_dtype);
  if (!aligned(grad, size) || !aligned(x, size) || !aligned(grad_x, size) || !aligned(weight, psize) ||
      !aligned(grad_weight, psize) || !aligned(grad_bias, psize) || !aligned(stats, 8))
    return MTP_ERR_ALIGN;
  if (grad_weight || grad_bias) {
    const int64_t need = 8 * layer_norm_parts(M, H) * H;
    if (need > 0 && !workspace) return MTP_ERR_NULL;
    if (workspace_bytes < need) return MTP_ERR_WORKSPACE;
    if (!aligned(workspace, 256)) return MTP_ERR_ALIGN;
  }
  NormArgs a = {};
  a.M = M;
  a.H = H;
  a.param_fp32 = param_dtype == MTP_DTYPE_FP32;
  a.stride = x_stride;
  a.x = x;
  a.weight = weight;
  a.stats = const_cast<float*>(stats);
  a.grad = grad;
  a.grad_x = grad_x;
  a.grad_weight = grad_weight;
  a.grad_bias = grad_bias;
  a.parts = static_cast<float*>(workspace);
  return launch_layer_norm_backward(a, dtype, static_cast<cudaStream_t>(stream));
}

int mtp_embed_tokens(const void* ids, int32_t id_bytes, int32_t N, const void* table, int32_t dtype, int32_t V,
                     int32_t H, float scale, void* out, void* stream) {
  const int rc = embed_shapes(id_bytes, N, dtype, V, H);
  if (rc != MTP_OK) return rc;
  if (N == 0) return MTP_OK;
  if (!ids || !table || !out) return MTP_ERR_NULL;
  const int64_t size = dtype_bytes(dtype);
  if (!aligned(ids, id_bytes) || !aligned(table, size) || !aligned(out, size)) return MTP_ERR_ALIGN;
  EmbedArgs a = {};
  a.N = N;
  a.V = V;
  a.H = H;
  a.wide_ids = id_bytes == 8;
  a.scale = scale;
  a.ids = ids;
  a.table = table;
  a.out = out;
  return launch_embed(a, dtype, static_cast<cudaStream_t>(stream));
}

int mtp_embed_tokens_backward_workspace_size(int32_t N, int32_t H, int32_t dtype, int64_t* bytes) {
  if (!bytes) return MTP_ERR_NULL;
  const int rc = embed_shapes(4, N, dtype, 1, H);
  if (rc != MTP_OK) return rc;
  *bytes = embed_workspace(N, H, dtype).total;
  return MTP_OK;
}

int mtp_embed_tokens_backward(const void* ids, int32_t id_bytes, int32_t N, const void* grad, int32_t dtype,
                              int32_t V, int32_t H, float scale, void* grad_table, void* workspace,
                              int64_t workspace_bytes, void* stream) {
  const int rc = embed_shapes(id_bytes, N, dtype, V, H);
  if (rc != MTP_OK) return rc;
  if (!grad_table || (N > 0 && (!ids || !grad)) || !workspace) return MTP_ERR_NULL;
  const int64_t size = dtype_bytes(dtype);
  if (!aligned(ids, id_bytes) || !aligned(grad, size) || !aligned(grad_table, size) || !aligned(workspace, 256))
    return MTP_ERR_ALIGN;
  const EmbedWs w = embed_workspace(N, H, dtype);
  if (workspace_bytes < w.total) return MTP_ERR_WORKSPACE;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  EmbedArgs a = {};
  a.N = N;
  a.V = V;
  a.H = H;
  a.wide_ids = id_bytes == 8;
  a.scale = scale;
  a.ids = ids;
  a.grad = grad;
  a.grad_table = grad_table;
  a.chunk = w.chunk;
  a.valid = reinterpret_cast<int32_t*>(ws + w.valid);
  a.owners = reinterpret_cast<int32_t*>(ws + w.owners);
  a.keys = reinterpret_cast<int32_t*>(ws + w.keys);
  a.order = reinterpret_cast<int32_t*>(ws + w.order);
  a.parts = reinterpret_cast<float*>(ws + w.parts);
  return launch_embed_backward(a, dtype, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
