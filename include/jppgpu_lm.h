/*
 * jppgpu_lm -- the operators of a re-ranking language model, to train one and to score with one.
 *
 * The analysis path scores with the recurrent language model of a model file (jppgpu.h: rnn_*): a row of the embedding
 * table a word, a recurrence over the words of a path, the noise-contrastive score of the word that follows.  These entry
 * points are that chain's three operators on the caller's own tensors, with their gradients, for a model of the caller's
 * own beside it -- one that a host scorer (jppgpu_analyze_batch_scored) asks for its scores.  The recurrence is a gated
 * linear one: it is a scan, so it runs in parallel along the words too, and so does its gradient.
 *
 * Every pointer is a DEVICE pointer; the calls enqueue on `stream` (a hipStream_t, may be NULL) of `device` and return
 * without waiting.  They allocate nothing, keep nothing from one call for the next and may be captured into a graph.
 * Threads may call at once; the caller owns the workspaces, and two calls that may run at once need two.  Results do not
 * depend on timing: the same inputs give the same bits.
 *
 * Matrices are rows with a stride (in elements, at least the row length, below 2^32) and contiguous columns, of 32-bit floats, bfloat16
 * or IEEE half.  Sums, states and softplus are held in 32 bits, an output is rounded once.  Outputs must not overlap inputs
 * or each other.  Word ids are int32 or int64; one outside [0, vocab) names no word.
 *
 * A packed batch: `rows` rows and n + 1 int32 offsets, sentence i in rows offsets[i] .. offsets[i + 1] - 1 (none: an empty
 * sentence).  The offsets must not fall; they are on the device and are not checked (offsets that fall or leave
 * 0 .. rows give unspecified values in the outputs' own rows, never an access outside them).  Rows before offsets[0] and
 * from offsets[n] on belong to no sentence: outputs leave them as they were, or clear them (JPPGPU_LM_CLEAR_REST).
 *
 * Return codes and messages: jppgpu.h (JPPGPU_OK, JPPGPU_INVALID_PARAMETER, ..., jppgpu_last_error).  A refused call has
 * enqueued nothing.
 */
#ifndef JPPGPU_LM_H
#define JPPGPU_LM_H

#include "jppgpu.h"

#ifdef __cplusplus
extern "C" {
#endif

/* element types */
enum { JPPGPU_LM_F32 = 0, JPPGPU_LM_BF16 = 1, JPPGPU_LM_F16 = 2 };
/* or'ed to the type of a packed batch's result (h, dgate, dx): its rows that belong to no sentence are set to zero */
enum { JPPGPU_LM_CLEAR_REST = 0x100 };

typedef struct {
  void* data;       /* first element; may be NULL where the matrix has no rows, or where it is optional */
  int64_t stride;   /* elements from one row to the next */
  int32_t type;     /* JPPGPU_LM_F32, _BF16 or _F16 */
  int32_t reserved; /* 0 */
} jppgpu_lm_matrix;

typedef struct {
  const void* data; /* int32 or int64 ids, contiguous */
  int32_t bytes;    /* 4 or 8 */
  int32_t reserved; /* 0 */
} jppgpu_lm_ids;

/* out[t][:] = scale * table[ids[t]][:] for t < n; an id that names no word gives a row of zeros.  table: vocab x dim; out:
 * n x dim, of the table's type, or 16-bit from a 32-bit table. */
int jppgpu_lm_embed(const jppgpu_lm_matrix* table, int64_t vocab, int64_t dim, const jppgpu_lm_ids* ids, int64_t n, float scale,
                    const jppgpu_lm_matrix* out, int32_t device, void* stream);

/* The gradient of the table: grad[v][:] = scale * sum over t with ids[t] = v of dy[t][:]; rows that no token names are zero.
 * The tokens of a word are summed in ascending order in parts, and the parts in order; where a part ends follows from the sizes
 * and from all ids, so the same inputs give the same bits, but other ids elsewhere may round a word's sum differently.
 * grad: vocab x dim, 32-bit, written whole.  dy: n x dim.  n < 2^31. */
int jppgpu_lm_embed_grad_workspace(int64_t n, int64_t vocab, int64_t dim, uint64_t* bytes);
int jppgpu_lm_embed_grad(const jppgpu_lm_matrix* dy, const jppgpu_lm_ids* ids, int64_t n, int64_t vocab, int64_t dim, float scale,
                         const jppgpu_lm_matrix* grad, void* workspace, uint64_t workspace_bytes, int32_t device, void* stream);

/* The gated linear recurrence.  For the rows of a sentence in order, a = sigmoid(gate):
 *     h_t = a_t h_(t-1) + (1 - a_t) x_t,   h_(-1) = the sentence's row of `state` (NULL data: zero)
 * last[i] = the state behind sentence i (its initial state if it is empty).  gate, x, h: rows x dim of one type; state,
 * last: n x dim, 32-bit; last may have NULL data.  One row a sentence (offsets 0, 1, 2, ...) is the serving form: a step
 * of n sentences.
 * max_len: the length of the longest sentence as far as the caller knows it, 0 for "unknown": it decides how the work is
 * split (and with it the rounding of the last bits), not what is computed.
 * saved: NULL, or jppgpu_lm_scan_saved(rows) x dim 32-bit floats, contiguous, which jppgpu_lm_scan_grad takes: the state in
 * front of every 8th row. */
int64_t jppgpu_lm_scan_saved(int64_t rows);
int jppgpu_lm_scan_workspace(int64_t rows, int64_t n, int64_t dim, int64_t max_len, uint64_t* bytes);
int jppgpu_lm_scan(const jppgpu_lm_matrix* gate, const jppgpu_lm_matrix* x, const int32_t* offsets, int64_t n, int64_t rows,
                   int64_t dim, int64_t max_len, const jppgpu_lm_matrix* state, const jppgpu_lm_matrix* h,
                   const jppgpu_lm_matrix* last, float* saved, void* workspace, uint64_t workspace_bytes, int32_t device,
                   void* stream);
/* Its gradient: dh (rows x dim, the type of x) and dlast (n x dim, 32-bit, may have NULL data) are the gradients of h and
 * last; dgate, dx (rows x dim, the type of x) and dstate (n x dim, 32-bit, may have NULL data) those of the inputs.  gate,
 * x, offsets and state as in the forward call that made `saved`. */
int jppgpu_lm_scan_grad(const jppgpu_lm_matrix* gate, const jppgpu_lm_matrix* x, const int32_t* offsets, int64_t n, int64_t rows,
                        int64_t dim, int64_t max_len, const jppgpu_lm_matrix* state, const float* saved,
                        const jppgpu_lm_matrix* dh, const jppgpu_lm_matrix* dlast, const jppgpu_lm_matrix* dgate,
                        const jppgpu_lm_matrix* dx, const jppgpu_lm_matrix* dstate, void* workspace, uint64_t workspace_bytes,
                        int32_t device, void* stream);

/* scores[t * cands + k] = <h_t, table[ids[t * cands + k]]> - constant, -infinity where the id names no word: the
 * re-ranker's score without its maximum-entropy part.  h: n x dim, table: vocab x dim, of one type. */
int jppgpu_lm_nce_score(const jppgpu_lm_matrix* h, const jppgpu_lm_matrix* table, int64_t vocab, int64_t dim,
                        const jppgpu_lm_ids* ids, int64_t n, int64_t cands, float constant, float* scores, int32_t device,
                        void* stream);

/* The noise-contrastive loss of n tokens with its gradients.  ids[t * cands] is the word that follows token t, the other
 * cands - 1 ids are words drawn from the noise; log_noise[v] = ln((cands - 1) p_noise(v)).
 *     z_k = <h_t, table[c_k]> - constant - log_noise[c_k]
 *     loss[t] = weight[t] * (softplus(-z_0) + sum over k > 0 of softplus(z_k))     (weight NULL: 1)
 * dh = d(sum of loss)/dh (n x dim, the type of h), dtable = d(sum of loss)/dtable (vocab x dim, 32-bit, written whole, summed
 * like jppgpu_lm_embed_grad).  A token without a following word (ids[t * cands] names none) has loss zero and no gradient,
 * whatever its row of h holds; a noise id that names no word is left out of the sum.  dh and dtable may have NULL data, both
 * or either: not wanted.  n * cands < 2^31.  The workspace is needed where either is wanted. */
int jppgpu_lm_nce_loss_workspace(int64_t n, int64_t cands, int64_t vocab, int64_t dim, uint64_t* bytes);
int jppgpu_lm_nce_loss(const jppgpu_lm_matrix* h, const jppgpu_lm_matrix* table, int64_t vocab, int64_t dim,
                       const jppgpu_lm_ids* ids, int64_t n, int64_t cands, const float* log_noise, float constant,
                       const float* weight, float* loss, const jppgpu_lm_matrix* dh, const jppgpu_lm_matrix* dtable,
                       void* workspace, uint64_t workspace_bytes, int32_t device, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* JPPGPU_LM_H */
