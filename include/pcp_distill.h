/*
 * pcp_distill.h — learning from another model's distribution: the top logits of rows
 * (what a teacher hands on) and the distillation loss on them with its gradient.
 *
 * The reference trains its policy by GRPO alone (src/nodes/controllers/rl_shepherd.zig:460-687)
 * and has no counterpart of either. They stand beside the loss head of pcp_grpo.h and
 * share its row layout, masks, aggregation, flags, status codes and context: a smaller
 * policy, or the draft model whose tokens pcp_verify_drafts checks, learns from the
 * policy's or a teacher's rows.
 *
 * All pointers are device (HBM) addresses. Calls are synchronous unless PCP_FLAG_ASYNC
 * is set; then they only enqueue kernels once the context's work buffer has grown, and
 * can be captured in a HIP graph. A call under capture that would need a larger work
 * buffer fails with PCP_ERR_INVALID_ARG before any work: make one uncaptured call of the
 * same sizes first. Calls on one context share its work buffer and run in stream order;
 * calls (and replayed graphs) that may overlap need separate contexts. A captured call's
 * work buffer stays where it is when a later call needs a larger one, until
 * pcp_release_workspace or pcp_destroy, after which its graph must not be replayed. The
 * calling thread's current device is the same after a call as before it.
 */
#ifndef PCP_DISTILL_H
#define PCP_DISTILL_H

#include <stdint.h>

#include "pcp_grpo.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Most entries per row, and the largest vocabulary of both entry points. */
#define PCP_TOP_LOGITS_MAX 256
#define PCP_DISTILL_MAX_VOCAB (1 << 24)

/* The k largest logits of each row with their ids, by falling logit, equal logits by
 * rising id, and the row's log-sum-exp  lse = log sum_v exp(logit_v / temperature).
 * -0 counts as 0 and is handed on as 0. NaN ranks below every number; a row whose
 * log-sum-exp is not finite as an f32 (a NaN or +Inf logit, nothing above -Inf, or a
 * largest logit that leaves f32's range divided by the temperature) is reported as
 * PCP_ERR_NONFINITE after the call, with its outputs written. Entries may be -Inf where
 * fewer than k logits are larger. */
typedef struct pcp_top_logits_args {
  int64_t n_rows;           /* 0 .. 2^31 - 1                                             */
  int64_t vocab;            /* V, 1 .. PCP_DISTILL_MAX_VOCAB                             */
  int64_t row_stride;       /* elements between rows; 0 => vocab                         */
  int32_t k;                /* entries per row, 1 .. min(V, PCP_TOP_LOGITS_MAX)          */
  int32_t logits_dtype;     /* PCP_BF16 | PCP_F16 | PCP_F32                              */
  int32_t ids_dtype;        /* PCP_I32 | PCP_I64                                         */
  float temperature;        /* > 0, finite: scales lse only                              */
  const void* logits;       /* rows at any element                                       */
  float* values;            /* [n_rows, k] the logits themselves                         */
  void* ids;                /* [n_rows, k]                                               */
  float* lse;               /* [n_rows], or NULL                                         */
  uint32_t flags;           /* PCP_FLAG_ASYNC                                            */
  void* stream;             /* hipStream_t; NULL => the default stream                   */
} pcp_top_logits_args;

/* Defaults: stride 0, bf16 logits, i32 ids, temperature 1. */
void pcp_top_logits_args_init(pcp_top_logits_args* a);
int pcp_top_logits(pcp_ctx* ctx, const pcp_top_logits_args* a);

/* Which way the divergence of teacher p and student q runs. */
typedef enum pcp_divergence {
  PCP_DIVERGENCE_FORWARD = 0,   /* sum p log(p / q): the student covers the teacher      */
  PCP_DIVERGENCE_REVERSE = 1    /* sum q log(q / p): it keeps to what the teacher does;
                                   needs teacher_lse                                      */
} pcp_divergence;

/* The least probability that a teacher's tokens outside its entries are given: half an
 * f32 step of 1, below which an f32 log-sum-exp says nothing about them. */
#define PCP_DISTILL_TAIL_FLOOR 5.9604644775390625e-08 /* 2^-24 */

/*
 * Distillation from a teacher's top logits. A row (s, t) has up to k teacher entries
 * (id, logit); an entry whose id is PCP_IGNORE_INDEX or whose logit is -Inf is unused.
 * With K the used ids, tau the temperature, z the row's student logits and
 * q = softmax(z / tau) over the whole vocabulary:
 *   with teacher_lse:  p_i = exp(t_i / tau - lse), and the other tokens form one class of
 *     probabilities  p_T = max(1 - sum p_i, PCP_DISTILL_TAIL_FLOOR),  q_T = sum_{v not in K} q_v
 *     (no such class where q_T is below 2^-126: every logit outside K masked, by -Inf or by
 *     a finite value far below the others, or K holding every token);
 *   without:           p = softmax(t / tau) over K, no such class.
 *   forward:  l = sum_i p_i log(p_i / q_i) + p_T log(p_T / q_T)
 *   reverse:  l = sum_i q_i log(q_i / p_i) + q_T log(q_T / p_T)
 *   loss = weight * (1 / loss_norm) * sum_s [ sum_t m_{s,t} l_{s,t} ] / max(sum_t m_{s,t}, 1)
 * and dlogits = d loss / d z. Rows, token arrays and the mask are those of
 * pcp_grpo_args; the teacher's arrays are indexed by logits row (as pcp_top_logits
 * writes them for a teacher's logits of the same layout). Rows without weight, without a
 * used entry, or past `rows` have zero dlogits and loss.
 *
 * Reported after the call (or by pcp_sync): a used id outside [0, V)
 * (PCP_ERR_TOKEN_RANGE) and an id used twice in one row (PCP_ERR_INVALID_ARG), in a row
 * with weight: that row has zero dlogits and loss; a non-finite log-sum-exp, NaN in the
 * teacher's entries, a NaN loss or a weight that is not finite (PCP_ERR_NONFINITE). dlogits may be the logits
 * themselves (their element type, the same address). Rows are summed in a fixed order:
 * the same call gives the same bits, but calls with other row counts may deal a row to
 * other numbers of workgroups, so a row's last bits depend on the call's size.
 */
typedef struct pcp_distill_args {
  int64_t n_seq;            /* S                                                          */
  int64_t rows;             /* token-carrying rows per sequence                           */
  int64_t vocab;            /* V, 1 .. PCP_DISTILL_MAX_VOCAB                              */
  int64_t logit_seq_stride; /* rows between sequences; 0 => rows                          */
  int64_t tok_seq_stride;   /* elements between sequences in mask / token_loss; 0 => rows */
  int64_t tok_offset;       /* token index of row t is tok_offset + t                     */

  int32_t k;                /* teacher entries per row, 1 .. PCP_TOP_LOGITS_MAX           */
  int32_t logits_dtype;     /* PCP_BF16 | PCP_F16 | PCP_F32                               */
  int32_t dlogits_dtype;    /* logits_dtype or PCP_F32                                    */
  int32_t ids_dtype;        /* teacher_ids: PCP_I32 | PCP_I64                             */
  int32_t mask_dtype;       /* PCP_F32 | PCP_BOOL (u8); ignored when mask == NULL         */
  int32_t divergence;       /* pcp_divergence                                             */

  const void* logits;             /* [n_seq*logit_seq_stride, V] student logits           */
  const void* teacher_ids;        /* [n_seq*logit_seq_stride, k]                          */
  const float* teacher_logits;    /* [n_seq*logit_seq_stride, k]                          */
  const float* teacher_lse;       /* [n_seq*logit_seq_stride] at the same temperature, or
                                     NULL: the entries renormalised                       */
  const void* mask;               /* token weights; NULL => all ones                      */

  void* dlogits;            /* [n_seq*logit_seq_stride, V]; NULL => forward only          */
  float* token_loss;        /* optional: m_t * l_t at the tokens that rows address        */
  float* loss;              /* optional device scalar                                     */

  float temperature;        /* tau > 0, finite                                            */
  float weight;             /* > 0, finite                                                */
  float loss_norm;          /* divisor of the sequence sum; 0 => n_seq                    */
  uint32_t flags;           /* PCP_FLAG_ASYNC                                             */
  void* stream;             /* hipStream_t; NULL => the default stream                    */
} pcp_distill_args;

/* Defaults: strides and offset 0, bf16 / bf16 / i32 / f32, forward, temperature 1,
 * weight 1, loss_norm 0. */
void pcp_distill_args_init(pcp_distill_args* a);
int pcp_distill_fwd_bwd(pcp_ctx* ctx, const pcp_distill_args* a);

#ifdef __cplusplus
}
#endif

#endif /* PCP_DISTILL_H */
