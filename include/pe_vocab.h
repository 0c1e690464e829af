/*
 * pe_vocab.h -- C ABI of the library's operators over the vocabulary (libpe_attn.so, gfx950): the scaled
 * token embedding with its gradient, and the losses over the logits, next-token cross entropy and
 * distillation from a teacher's top logits, with theirs.
 *
 * Conventions, element types (PE_DTYPE_*) and error codes are those of pe_attn.h: plain C types, device
 * pointers, element strides, a hipStream_t passed as void*.  Nothing is allocated, freed or synchronised, no
 * pointer is kept, and calls on buffers of their own may overlap.  Functions return 0 or a negative PE_ERR_*.
 * Every sum runs in a fixed order, in 32 bits or more: a call repeated on the same inputs gives the same bits.
 *
 * What they replace (shyampathak22/pe_ablations): pe_embed_* nn.Embedding of TokenEmbedding
 * (src/model/embeddings.py:7-34) and its autograd; pe_loss_* the shifted copy of the logits and F.cross_entropy
 * of Transformer.forward (src/model/transformer.py:357-364) and their autograd.
 */
#ifndef PE_VOCAB_H
#define PE_VOCAB_H

#include "pe_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Embedding lookup: out[t] = weight[ids[t]] * scale for t < n, the product in fp32 and rounded once to the
 * tensors' type (PE_DTYPE_*, one for weight and out).  ids: n contiguous integers of id_bytes (4 or 8).  Rows have
 * dim elements of unit stride.  An id outside [0, vocab) gives a row of NaN. */
int pe_embed_fwd(const void* ids, int32_t id_bytes, int64_t n, const void* weight, int32_t dtype, int64_t vocab,
                 int32_t dim, int64_t weight_row_stride, float scale, void* out, int64_t out_row_stride, void* stream);

/* Its weight gradient: dweight[v] = scale * sum of dy[t] over the t with ids[t] == v, in increasing t, for every v
 * of the vocabulary (0 where no token has it, and for v == padding_idx; pass -1 for none).  ids outside
 * [0, vocab) add nothing.  The workspace holds the tokens sorted by id; up to 4096 tokens need none (0 bytes, NULL).
 * n <= 2^24. */
size_t pe_embed_bwd_workspace_bytes(int64_t n, int64_t vocab, int32_t dim);
int pe_embed_bwd(const void* ids, int32_t id_bytes, int64_t n, const void* dy, int32_t dtype, int64_t dy_row_stride,
                 int64_t vocab, int32_t dim, float scale, int64_t padding_idx, void* dweight,
                 int64_t dweight_row_stride, void* workspace, size_t ws_bytes, void* stream);

/* how row losses are put together */
enum { PE_LOSS_NONE = 0, PE_LOSS_SUM = 1, PE_LOSS_MEAN = 2 };

#define PE_LOSS_MAX_TOP_K 1024

/* A loss over (rows, vocab) logits z.  Row r has the label y = labels[r], or with shift = S > 0 (rows in
 * sequences of S) labels[r + 1], and none in the last row of each sequence.  A row without a label, or with
 * ignore_index, does not count: its loss and gradient are 0 and its logits are not read.  With labels NULL every row
 * counts (hard_weight must be 0 then).  The teacher gives top_k pairs (id, logit) a row; pairs whose id is outside
 * [0, vocab) or whose logit is -inf are absent, and an id may come twice (its probabilities add up).  With
 * p = softmax(teacher logits / T) over the pairs present and q_T = softmax(z / T):
 *     hard = -log softmax(z)_y          soft = T^2 sum_k p_k (log p_k - log q_T[id_k])     (0 if none is present)
 *     row  = hard_weight * hard + soft_weight * soft
 * PE_LOSS_MEAN divides the sum by the number of rows that count (none: NaN).  A label outside [0, vocab) that is
 * not ignore_index makes its row's loss and gradient NaN. */
typedef struct {
  int64_t rows;
  int64_t row_stride;        /* elements between rows of the logits (unit stride inside) */
  int64_t grad_row_stride;   /* the same for the gradient */
  int64_t shift;             /* 0, or the length of a sequence of rows */
  int64_t ignore_index;
  int64_t teacher_id_stride; /* elements between rows of the teacher's ids / logits */
  int64_t teacher_row_stride;
  int32_t vocab;             /* at most 2^28 */
  int32_t dtype;             /* PE_DTYPE_* of logits and gradient */
  int32_t label_bytes;       /* 4 or 8 */
  int32_t reduction;         /* PE_LOSS_* */
  int32_t top_k;             /* 0 = no teacher, at most PE_LOSS_MAX_TOP_K */
  int32_t teacher_dtype;     /* PE_DTYPE_* of the teacher's logits */
  int32_t teacher_id_bytes;  /* 4 or 8 */
  float hard_weight, soft_weight, temperature;
  float grad_factor;         /* host factor on the gradient (1 = none) */
  int32_t reserved;          /* 0 */
} pe_loss_params;

/* Host-only validation (no device work). */
int pe_loss_check(const pe_loss_params* p);

/* Forward: loss (rows floats for PE_LOSS_NONE, else one).  stats (pe_loss_stats_floats floats, or NULL when no
 * backward follows) keeps what pe_loss_bwd needs of each row: the maximum, the two sums, and the teacher's
 * probabilities, which the backward does not form again (its teacher_ids and teacher_logits are not read). */
size_t pe_loss_workspace_bytes(const pe_loss_params* p);
int64_t pe_loss_stats_floats(const pe_loss_params* p);
int pe_loss_fwd(const pe_loss_params* p, const void* logits, const void* labels, const void* teacher_ids,
                const void* teacher_logits, float* loss, float* stats, void* workspace, size_t ws_bytes, void* stream);

/* Backward: dlogits (rows, vocab) for the loss's gradient dloss (device: rows floats for PE_LOSS_NONE, else one),
 *     dz_j = c (hard_weight (q_j - [j = y]) + soft_weight T (q_T,j - sum_{k: id_k = j} p_k)),
 * c = grad_factor * dloss, over the number of rows that count for PE_LOSS_MEAN.  stats as pe_loss_fwd wrote it for
 * the same arguments.  dlogits must not overlap the logits. */
int pe_loss_bwd(const pe_loss_params* p, const void* logits, const void* labels, const void* teacher_ids,
                const void* teacher_logits, const float* stats, const float* dloss, void* dlogits, void* stream);

/* Both in one pass over the logits: loss and dlogits, the latter times the device scalar grad_scale (NULL = 1) and
 * grad_factor.  PE_LOSS_SUM or PE_LOSS_MEAN. */
int pe_loss_step(const pe_loss_params* p, const void* logits, const void* labels, const void* teacher_ids,
                 const void* teacher_logits, const float* grad_scale, float* loss, void* dlogits, void* workspace,
                 size_t ws_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* PE_VOCAB_H */
