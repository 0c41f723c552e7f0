/*
 * pcp_score.h — scores of given tokens: log-probs, entropy and the top alternatives of
 * rows of logits, and the gradient of any function of the log-probs and entropies.
 *
 * The reference scores its rollouts inside the training graph alone, by the log-softmax and
 * gather of tools/export_qwen_forward.py:154-156, and has no counterpart of the entropy, the
 * alternatives or a gradient other than its loss's. They stand beside the loss head of
 * pcp_grpo.h and share its token arrays, masks, flags, status codes and context: what a
 * rollout's server reports with each token, and the entropy bonus that is added to the
 * loss head's dlogits.
 *
 * All pointers are device (HBM) addresses. Calls are synchronous unless PCP_FLAG_ASYNC
 * is set; then they only enqueue kernels once the context's work buffer has grown, and
 * can be captured in a HIP graph. A call under capture that would need a larger work
 * buffer fails with PCP_ERR_INVALID_ARG before any work: make one uncaptured call of the
 * same sizes first (pcp_score_bwd needs none). Calls on one context share its work buffer
 * and run in stream order; calls (and replayed graphs) that may overlap need separate
 * contexts. A captured call's work buffer stays where it is when a later call needs a larger
 * one, until pcp_release_workspace or pcp_destroy, after which its graph must not be
 * replayed. The calling thread's current device is the same after a call as before it.
 */
#ifndef PCP_SCORE_H
#define PCP_SCORE_H

#include <stdint.h>

#include "pcp_grpo.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Most alternatives per row, and the largest vocabulary of both entry points. */
#define PCP_SCORE_TOP_MAX 256
#define PCP_SCORE_MAX_VOCAB (1 << 24)

/*
 * Row (s, t), t < rows, is the V logits x from element s * seq_stride + t * row_stride on,
 * and scores the token ids[i] with weight mask[i], i = s * tok_seq_stride + tok_offset + t.
 * With z = x / temperature, m = max x and log_sum = log sum_v exp((x_v - m) / temperature):
 *   logp    = (x_id - m) / temperature - log_sum
 *   entropy = -sum_v p_v log p_v,  log p_v = (x_v - m) / temperature - log_sum
 *   row_max = m
 *   top     = the k largest logits by falling logit, equal ones by rising id, as log p and id
 * each at index i (top_*: i * k + rank). Rows whose token weighs 0 or is PCP_IGNORE_INDEX
 * have zero outputs and alternatives with the id PCP_IGNORE_INDEX; entries that no row
 * addresses are not written. Tokens of probability 0 add nothing to the entropy. No log-prob is
 * above 0, no entropy and no log_sum below 0 (of rows that are not reported). -0 counts as 0;
 * NaN ranks below every number. A finite mask of any size (-1e30, a type's lowest value)
 * is a logit like any other.
 *
 * Reported after the call (or by pcp_sync): a token id outside [0, V) on a row with weight
 * (PCP_ERR_TOKEN_RANGE; the row counts as one without weight), and a row whose row_max or log_sum is not finite
 * (a NaN or +Inf logit, nothing above -Inf: PCP_ERR_NONFINITE; its outputs are written and mean nothing).
 * Rows are summed in a fixed order: the same call gives the same bits, but calls with other row
 * counts may deal a row to other numbers of workgroups.
 */
typedef struct pcp_score_args {
  int64_t n_seq;            /* S                                                          */
  int64_t rows;             /* token-carrying rows per sequence                           */
  int64_t vocab;            /* V, 1 .. PCP_SCORE_MAX_VOCAB                                */
  int64_t row_stride;       /* elements between rows, >= V; 0 => V                        */
  int64_t seq_stride;       /* elements between sequences, >= V; 0 => rows * row_stride   */
  int64_t tok_seq_stride;   /* elements between sequences in token arrays; 0 => rows      */
  int64_t tok_offset;       /* token index of row t is tok_offset + t                     */

  int32_t k;                /* alternatives per row, 0 .. min(V, PCP_SCORE_TOP_MAX)       */
  int32_t logits_dtype;     /* PCP_BF16 | PCP_F16 | PCP_F32                               */
  int32_t ids_dtype;        /* PCP_I64 | PCP_I32                                          */
  int32_t mask_dtype;       /* PCP_F32 | PCP_BOOL (u8); ignored when mask == NULL         */
  int32_t top_ids_dtype;    /* PCP_I32 | PCP_I64                                          */
  float temperature;        /* > 0, finite                                                */

  const void* logits;       /* rows at any element                                        */
  const void* ids;          /* tokens; NULL => no row has one (logp must be NULL)         */
  const void* mask;         /* token weights (0: row left out); NULL => all ones          */

  float* logp;              /* per-token outputs, each optional                           */
  float* entropy;
  float* row_max;
  float* log_sum;
  float* top_logp;          /* [n_seq * tok_seq_stride, k]; needed with k > 0             */
  void* top_ids;            /* the same                                                   */

  uint32_t flags;           /* PCP_FLAG_ASYNC                                             */
  void* stream;             /* hipStream_t; NULL => the default stream                    */
} pcp_score_args;

/* Defaults: strides, offset and k 0, bf16 logits, i64 ids, f32 mask, i32 top ids, temperature 1. */
void pcp_score_args_init(pcp_score_args* a);
int pcp_score_fwd(pcp_ctx* ctx, const pcp_score_args* a);

/*
 * The gradient of a function f of the rows' logp and entropy, given d f / d logp and
 * d f / d entropy and the forward's row_max, log_sum and entropy of the same rows:
 *   dz_v = dlogp (1[v = id] - p_v) - dentropy p_v (log p_v + entropy),   dlogits_v = dz_v / temperature
 * Row (s, t), t < logit_rows, of dlogits begins at element s * dseq_stride + t * drow_stride.
 * Rows t >= rows, rows whose token weighs 0 or is PCP_IGNORE_INDEX and rows whose two gradients
 * are both 0 are not read: their dlogits are 0. With accumulate the gradient is added to what
 * dlogits hold, in f32 and rounded once, and those rows stay as they are. dlogits may be the
 * logits themselves (their element type, address and strides); other overlaps are refused.
 *
 * Reported after the call (or by pcp_sync): a token id outside [0, V) on a row with weight
 * (PCP_ERR_TOKEN_RANGE; the row counts as one without weight), and a row_max, log_sum, entropy
 * or gradient that is not finite on a row that is read (PCP_ERR_NONFINITE; its dlogits hold NaN).
 * An element's bits depend on its row alone.
 */
typedef struct pcp_score_bwd_args {
  int64_t n_seq;            /* S                                                          */
  int64_t rows;             /* token-carrying rows per sequence                           */
  int64_t logit_rows;       /* dlogits rows per sequence, >= rows; 0 => rows              */
  int64_t vocab;            /* V, 1 .. PCP_SCORE_MAX_VOCAB                                */
  int64_t row_stride;       /* elements between logits rows, >= V; 0 => V                 */
  int64_t seq_stride;       /* elements between sequences, >= V; 0 => logit_rows * row_stride */
  int64_t drow_stride;      /* the same of dlogits; their rows may not overlap            */
  int64_t dseq_stride;
  int64_t tok_seq_stride;   /* elements between sequences in token arrays; 0 => rows      */
  int64_t tok_offset;       /* token index of row t is tok_offset + t                     */

  int32_t logits_dtype;     /* PCP_BF16 | PCP_F16 | PCP_F32                               */
  int32_t dlogits_dtype;    /* logits_dtype or PCP_F32                                    */
  int32_t ids_dtype;        /* PCP_I64 | PCP_I32                                          */
  int32_t mask_dtype;       /* PCP_F32 | PCP_BOOL (u8); ignored when mask == NULL         */
  int32_t accumulate;       /* 0: dlogits are written, 1: added to                        */
  float temperature;        /* that of the forward                                        */

  const void* logits;
  const void* ids;          /* NULL => no row has a token (dlogp must be NULL)            */
  const void* mask;         /* NULL => all ones                                           */
  const float* row_max;     /* of the forward, token arrays as there                      */
  const float* log_sum;
  const float* entropy;     /* needed with dentropy                                       */
  const float* dlogp;       /* token arrays; NULL => 0                                    */
  const float* dentropy;

  void* dlogits;

  uint32_t flags;           /* PCP_FLAG_ASYNC                                             */
  void* stream;             /* hipStream_t; NULL => the default stream                    */
} pcp_score_bwd_args;

/* Defaults: strides, offset and logit_rows 0, bf16 / bf16 / i64 / f32, no accumulation, temperature 1. */
void pcp_score_bwd_args_init(pcp_score_bwd_args* a);
int pcp_score_bwd(pcp_ctx* ctx, const pcp_score_bwd_args* a);

#ifdef __cplusplus
}
#endif

#endif /* PCP_SCORE_H */
