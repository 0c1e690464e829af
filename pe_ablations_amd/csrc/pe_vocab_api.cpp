// C-ABI entry points over the vocabulary (declared in include/pe_vocab.h).  Host code only: checks the
// arguments, carves the caller's workspace and enqueues the kernels on the caller's stream.
#include <hip/hip_runtime.h>
#include <string.h>

#include "pe_internal.h"
#include "pe_vocab.h"

namespace {

bool float_dtype(int d) { return d == PE_DTYPE_BF16 || d == PE_DTYPE_FP32 || d == PE_DTYPE_FP16; }
int elem_size(int d) { return d == PE_DTYPE_FP32 ? 4 : 2; }
bool id_size(int b) { return b == 4 || b == 8; }
bool aligned(const void* p, int bytes) { return (uintptr_t)p % (uintptr_t)bytes == 0; }

int embed_check(const void* ids, int32_t id_bytes, int64_t n, const void* x, int32_t dtype, int64_t vocab, int32_t dim,
                int64_t x_rs, const void* y, int64_t y_rs) {
  if (n < 0 || n > 0x7fffffff || vocab <= 0 || vocab > 0x7ffffffe || dim <= 0) return PE_ERR_SHAPE;
  if (!float_dtype(dtype) || !id_size(id_bytes)) return PE_ERR_MODE;
  if (x_rs < dim || y_rs < dim) return PE_ERR_STRIDE;
  if (!aligned(ids, id_bytes) || !aligned(x, elem_size(dtype)) || !aligned(y, elem_size(dtype))) return PE_ERR_STRIDE;
  return PE_OK;
}

// the teacher's rows: ids and probabilities of K + 1 places, two sums
int64_t teacher_floats(const pe_loss_params* p) { return p->soft_weight > 0.f ? p->rows * (2 * (int64_t)p->top_k + 4) : 0; }
void set_teacher(pe::LossArgs& a, float* at) {
  a.place = (int32_t*)at;
  a.prob = at + a.rows * (a.K + 1);
  a.tsum = a.prob + a.rows * (a.K + 1);
}

pe::LossArgs loss_args(const pe_loss_params* p, const void* z, const void* labels, const void* tid, const void* tlog) {
  pe::LossArgs a;
  memset(&a, 0, sizeof(a));
  a.z = z; a.z_rs = p->row_stride;
  a.dz_rs = p->grad_row_stride;
  a.labels = labels; a.label_bytes = p->label_bytes; a.shift = p->shift; a.ignore = p->ignore_index;
  a.tid = tid; a.tid_rs = p->teacher_id_stride; a.tid_bytes = p->teacher_id_bytes;
  a.tlog = tlog; a.tlog_rs = p->teacher_row_stride; a.tlog_dtype = p->teacher_dtype;
  a.rows = p->rows; a.V = p->vocab; a.K = p->top_k; a.reduction = p->reduction;
  a.hw = p->hard_weight; a.sw = p->soft_weight; a.T = p->temperature; a.factor = p->grad_factor;
  return a;
}

int loss_inputs(const pe_loss_params* p, const void* z, const void* labels, const void* tid, const void* tlog) {
  const int rc = pe_loss_check(p);
  if (rc) return rc;
  if (p->rows == 0) return PE_OK;
  if (!z || (!labels && p->hard_weight != 0.f) || (p->top_k && (!tid || !tlog))) return PE_ERR_NULL;
  if (!aligned(z, elem_size(p->dtype)) || !aligned(labels, p->label_bytes)) return PE_ERR_STRIDE;
  if (p->top_k && (!aligned(tid, p->teacher_id_bytes) || !aligned(tlog, elem_size(p->teacher_dtype)))) return PE_ERR_STRIDE;
  return PE_OK;
}

}  // namespace

extern "C" {

int pe_embed_fwd(const void* ids, int32_t id_bytes, int64_t n, const void* weight, int32_t dtype, int64_t vocab,
                 int32_t dim, int64_t weight_row_stride, float scale, void* out, int64_t out_row_stride, void* stream) {
  int rc = embed_check(ids, id_bytes, n, weight, dtype, vocab, dim, weight_row_stride, out, out_row_stride);
  if (rc) return rc;
  if (n == 0) return PE_OK;
  if (!ids || !weight || !out) return PE_ERR_NULL;
  if ((rc = pe::device_ready())) return rc;
  pe::EmbedArgs a;
  memset(&a, 0, sizeof(a));
  a.ids = ids; a.id_bytes = id_bytes; a.n = n;
  a.x = weight; a.x_rs = weight_row_stride;
  a.y = out; a.y_rs = out_row_stride;
  a.V = vocab; a.H = dim; a.scale = scale;
  return pe::launch_embed_fwd(dtype, a, (hipStream_t)stream);
}

size_t pe_embed_bwd_workspace_bytes(int64_t n, int64_t vocab, int32_t dim) {
  if (n < 0 || n > (1 << 24) || vocab <= 0 || vocab > 0x7ffffffe || dim <= 0) return 0;
  return (size_t)pe::embed_bwd_workspace(n, vocab, dim);
}

int pe_embed_bwd(const void* ids, int32_t id_bytes, int64_t n, const void* dy, int32_t dtype, int64_t dy_row_stride,
                 int64_t vocab, int32_t dim, float scale, int64_t padding_idx, void* dweight,
                 int64_t dweight_row_stride, void* workspace, size_t ws_bytes, void* stream) {
  int rc = embed_check(ids, id_bytes, n, dy, dtype, vocab, dim, dy_row_stride, dweight, dweight_row_stride);
  if (rc) return rc;
  if (n > (1 << 24) || padding_idx < -1 || padding_idx >= vocab) return PE_ERR_SHAPE;
  if (!dweight || (n && (!ids || !dy))) return PE_ERR_NULL;
  const size_t need = pe_embed_bwd_workspace_bytes(n, vocab, dim);
  if (need && (!workspace || !aligned(workspace, 16) || ws_bytes < need)) return PE_ERR_WORKSPACE;
  if ((rc = pe::device_ready())) return rc;
  pe::EmbedArgs a;
  memset(&a, 0, sizeof(a));
  a.ids = ids; a.id_bytes = id_bytes; a.n = n;
  a.x = dy; a.x_rs = dy_row_stride;
  a.y = dweight; a.y_rs = dweight_row_stride;
  a.V = vocab; a.H = dim; a.scale = scale; a.pad = padding_idx;
  return pe::launch_embed_bwd(dtype, a, workspace, (hipStream_t)stream);
}

int pe_loss_check(const pe_loss_params* p) {
  if (!p) return PE_ERR_NULL;
  if (p->rows < 0 || p->rows > 0x7fffffff || p->vocab <= 0 || p->vocab > (1 << 28) || p->shift < 0 || p->top_k < 0 || p->top_k > PE_LOSS_MAX_TOP_K)
    return PE_ERR_SHAPE;
  if (p->shift && p->rows % p->shift) return PE_ERR_SHAPE;
  if (!float_dtype(p->dtype) || !id_size(p->label_bytes) || p->reduction < PE_LOSS_NONE || p->reduction > PE_LOSS_MEAN)
    return PE_ERR_MODE;
  if (p->top_k && (!float_dtype(p->teacher_dtype) || !id_size(p->teacher_id_bytes))) return PE_ERR_MODE;
  // the negated forms refuse NaN as well
  if (!(p->hard_weight >= 0.f) || !(p->soft_weight >= 0.f) || !(p->hard_weight + p->soft_weight > 0.f)) return PE_ERR_MODE;
  if (!(p->hard_weight <= 3e38f) || !(p->soft_weight <= 3e38f)) return PE_ERR_MODE;
  if (p->soft_weight > 0.f && (!p->top_k || !(p->temperature > 0.f) || !(p->temperature <= 3e38f))) return PE_ERR_MODE;
  if (p->row_stride < p->vocab || p->grad_row_stride < p->vocab) return PE_ERR_STRIDE;
  if (p->top_k && (p->teacher_id_stride < p->top_k || p->teacher_row_stride < p->top_k)) return PE_ERR_STRIDE;
  return PE_OK;
}

size_t pe_loss_workspace_bytes(const pe_loss_params* p) {
  // the row losses, the number of rows that count, the teacher's rows
  return pe_loss_check(p) ? 0 : (size_t)(p->rows + 1 + teacher_floats(p)) * 4;
}

int64_t pe_loss_stats_floats(const pe_loss_params* p) { return pe_loss_check(p) ? 0 : 3 * p->rows + 1 + teacher_floats(p); }

int pe_loss_fwd(const pe_loss_params* p, const void* logits, const void* labels, const void* teacher_ids,
                const void* teacher_logits, float* loss, float* stats, void* workspace, size_t ws_bytes, void* stream) {
  int rc = loss_inputs(p, logits, labels, teacher_ids, teacher_logits);
  if (rc) return rc;
  if (p->rows == 0 && p->reduction == PE_LOSS_NONE) return PE_OK;
  if (!loss) return PE_ERR_NULL;
  if (!aligned(loss, 4) || !aligned(stats, 4)) return PE_ERR_STRIDE;
  if (!workspace || !aligned(workspace, 4) || ws_bytes < pe_loss_workspace_bytes(p)) return PE_ERR_WORKSPACE;
  if ((rc = pe::device_ready())) return rc;
  pe::LossArgs a = loss_args(p, logits, labels, teacher_ids, teacher_logits);
  const bool whole = p->reduction != PE_LOSS_NONE;
  a.row_loss = whole ? (float*)workspace : loss;
  a.stats = stats;
  set_teacher(a, stats ? stats + 3 * p->rows + 1 : (float*)workspace + p->rows + 1);
  if ((rc = pe::launch_loss_prepare(a, nullptr, (hipStream_t)stream))) return rc;
  if ((rc = pe::launch_loss(p->dtype, pe::LOSS_FWD, a, (hipStream_t)stream)) || !whole) return rc;
  return pe::launch_loss_reduce(a, loss, stats ? stats + 3 * p->rows : (float*)workspace + p->rows, true, (hipStream_t)stream);
}

int pe_loss_bwd(const pe_loss_params* p, const void* logits, const void* labels, const void* teacher_ids,
                const void* teacher_logits, const float* stats, const float* dloss, void* dlogits, void* stream) {
  int rc = loss_inputs(p, logits, labels, teacher_ids, teacher_logits);
  if (rc) return rc;
  if (p->rows == 0) return PE_OK;
  if (!stats || !dloss || !dlogits) return PE_ERR_NULL;
  if (!aligned(dlogits, elem_size(p->dtype)) || !aligned(stats, 4) || !aligned(dloss, 4)) return PE_ERR_STRIDE;
  if ((rc = pe::device_ready())) return rc;
  pe::LossArgs a = loss_args(p, logits, labels, teacher_ids, teacher_logits);
  a.dz = dlogits;
  a.stats = const_cast<float*>(stats);
  set_teacher(a, a.stats + 3 * p->rows + 1);
  a.dloss = dloss;
  a.count = p->reduction == PE_LOSS_MEAN ? stats + 3 * p->rows : nullptr;
  return pe::launch_loss(p->dtype, pe::LOSS_BWD, a, (hipStream_t)stream);
}

int pe_loss_step(const pe_loss_params* p, const void* logits, const void* labels, const void* teacher_ids,
                 const void* teacher_logits, const float* grad_scale, float* loss, void* dlogits, void* workspace,
                 size_t ws_bytes, void* stream) {
  int rc = loss_inputs(p, logits, labels, teacher_ids, teacher_logits);
  if (rc) return rc;
  if (p->reduction == PE_LOSS_NONE) return PE_ERR_MODE;
  if (!loss || (p->rows && !dlogits)) return PE_ERR_NULL;
  if (!aligned(dlogits, elem_size(p->dtype)) || !aligned(loss, 4) || !aligned(grad_scale, 4)) return PE_ERR_STRIDE;
  if (!workspace || !aligned(workspace, 4) || ws_bytes < pe_loss_workspace_bytes(p)) return PE_ERR_WORKSPACE;
  if ((rc = pe::device_ready())) return rc;
  pe::LossArgs a = loss_args(p, logits, labels, teacher_ids, teacher_logits);
  a.dz = dlogits;
  a.row_loss = (float*)workspace;
  a.dloss = grad_scale;
  set_teacher(a, (float*)workspace + p->rows + 1);
  float* count = p->reduction == PE_LOSS_MEAN ? (float*)workspace + p->rows : nullptr;
  if ((rc = pe::launch_loss_prepare(a, count, (hipStream_t)stream))) return rc;
  a.count = count;
  if ((rc = pe::launch_loss(p->dtype, pe::LOSS_STEP, a, (hipStream_t)stream))) return rc;
  return pe::launch_loss_reduce(a, loss, count, false, (hipStream_t)stream);
}

}  // extern "C"
