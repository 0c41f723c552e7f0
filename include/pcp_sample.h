/*
 * pcp_sample.h — the rollout sampler on the GPU.
 *
 * Reference: Sampler.sample (src/core/math.zig:21-58), called once per generated
 * token by GenerationEngine.generateRolloutStreaming
 * (src/nodes/workers/generation_engine.zig:255-268) after a device-to-host copy of
 * the full logits row. Here the logits stay in HBM and only the token id comes back.
 *
 * The random stream stays the caller's: uniforms[r] is the value the reference draws
 * with self.prng.random().float(f32) for row r, so a Zig caller keeps its Sampler's
 * PRNG and passes the draws. Status codes and the context are those of pcp_grpo.h.
 */
#ifndef PCP_SAMPLE_H
#define PCP_SAMPLE_H

#include <stdint.h>

#include "pcp_grpo.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Largest vocabulary and batch per call. */
#define PCP_SAMPLE_MAX_VOCAB (1 << 20)
#define PCP_SAMPLE_MAX_ROWS 65535

/* For each row r < n_rows of logits (dtype PCP_F32 or PCP_BF16, row r at element
 * offset r * row_stride, device memory):
 *  - temperature < 1e-6: the index of the first maximum (math.zig:22-25, argmax
 *    :61-73; NaN never wins; a row with no value above -inf gives 0);
 *  - otherwise the first index i with sum_{j<=i} e_j >= uniforms[r] * sum_j e_j,
 *    e_j = exp((logit_j - max) / temperature) (:27-53); a NaN or +Inf logit, or a row
 *    of -Inf, makes the sum NaN and gives vocab - 1, the reference's fallback (:56).
 *    A NaN temperature is not below 1e-6, so it samples too, and every row gives
 *    vocab - 1 for the same reason; +Inf makes every finite term 1 (uniform draw).
 * 1 <= n_rows <= PCP_SAMPLE_MAX_ROWS. ids[r] receives the token (int64, device). uniforms (device, n_rows floats in
 * [0, 1)) may be NULL when temperature < 1e-6. The kernel sums in a fixed parallel
 * order, not the reference's sequential f32 loop, so a draw whose threshold lies
 * within f32 rounding of a cumulative boundary can pick the neighbouring token. */
int pcp_sample_tokens(pcp_ctx* ctx, const void* logits, int dtype, int64_t n_rows, int64_t vocab,
                      int64_t row_stride, float temperature, const float* uniforms, int64_t* ids,
                      void* stream);
/* The same, enqueued only: one kernel launch on `stream` behind the work that produced
 * the logits (a decode step's forward), the token ids left in device memory, no host
 * synchronisation (as PCP_FLAG_ASYNC; pcp_sync waits for it). For the reference's one
 * sampled row per generated token (generation_engine.zig:255-268) without its
 * device-to-host copy of the row. Calls on one context use its per-row tickets: calls
 * that may overlap on different streams need separate contexts. */
int pcp_sample_tokens_async(pcp_ctx* ctx, const void* logits, int dtype, int64_t n_rows, int64_t vocab,
                            int64_t row_stride, float temperature, const float* uniforms, int64_t* ids,
                            void* stream);

/* Most drafted tokens per sequence of pcp_verify_drafts. */
#define PCP_VERIFY_MAX_DRAFT 64

/*
 * Verification of drafted tokens. The reference generates one token per forward of the
 * policy (generation_engine.zig:255-268) and has no counterpart. A draft (a smaller
 * model, or a lookup) proposes n tokens per sequence; one forward of the target scores
 * them all, and this call keeps the longest prefix that leaves the text distributed as
 * if the target had sampled it token by token, then adds one token.
 *
 * Sequence s has len = draft_lens[s] drafted tokens d_0 .. d_{len-1} (n without
 * draft_lens). Target row i of s scores the token that follows d_0 .. d_{i-1}; with
 * p_i = softmax(target row i / temperature) and q_i the same of draft row i (all of q_i
 * on d_i where draft_logits is NULL), d_i is accepted while
 *     uniforms[s, i] * q_i(d_i) < p_i(d_i).
 * With j the first i that is not accepted (len if all are), the token after them is the
 * first v with  sum_{w<=v} r_w > uniforms[s, n] * sum_w r_w,  r = max(p_j - q_j, 0), or
 * r = p_j for j = len (and where max(p_j - q_j, 0) is zero throughout). A temperature
 * below 1e-6 is greedy, as in pcp_sample_tokens: d_i is accepted while it is the first
 * maximum of target row i, whose first maximum is the token after; draft_logits and
 * uniforms are not read.
 * Every probability, sum and comparison is formed in 64 bits from the logits, so the
 * choice is the formulas' own up to about 1e-14 of a probability.
 *
 * tokens[s, :] receives d_0 .. d_{j-1}, the token after them, then PCP_IGNORE_INDEX;
 * accepted[s] = j; logp[s, i] = log p_i(tokens[s, i]) for i <= j (0 when greedy) and 0
 * after them: at temperature 1 the behaviour policy's log-probs, pcp_grpo_args.old_logp.
 *
 * Reported after the call (or by pcp_sync), for rows that a result depends on: a
 * drafted id outside [0, V) (PCP_ERR_TOKEN_RANGE; it is refused, and the token after
 * comes from p_j), draft_lens outside [0, n] (PCP_ERR_INVALID_ARG; taken as the nearer end),
 * and, when sampling, a row whose log-sum-exp is not finite (PCP_ERR_NONFINITE: its
 * token is refused and the token after is V - 1 with log-prob 0; a draft row alone being so
 * refuses its token for one from p_j).
 * Calls on one context share its work buffer: calls that may overlap on different
 * streams need separate contexts. Under stream capture the work buffer must have grown
 * by an uncaptured call of the same sizes (PCP_ERR_INVALID_ARG before any work if not);
 * it then stays where it is until pcp_release_workspace or pcp_destroy, after which the
 * graph must not be replayed.
 */
typedef struct pcp_verify_args {
  int64_t n_seq;             /* S, 0 .. PCP_SAMPLE_MAX_ROWS                               */
  int64_t n_draft;           /* n, 0 .. PCP_VERIFY_MAX_DRAFT                              */
  int64_t vocab;             /* V, 1 .. PCP_SAMPLE_MAX_VOCAB                              */
  int64_t target_row_stride; /* elements between rows; 0 => vocab                         */
  int64_t draft_row_stride;  /* elements between rows; 0 => vocab                         */
  int32_t logits_dtype;      /* PCP_BF16 | PCP_F16 | PCP_F32, both models                 */
  float temperature;         /* NaN is refused                                            */
  const void* target_logits; /* [S, n + 1] rows, at any element                           */
  const void* draft_logits;  /* [S, n] rows, or NULL                                      */
  const int64_t* draft_ids;  /* [S, n]; may be NULL for n = 0                             */
  const int32_t* draft_lens; /* [S], or NULL                                              */
  const float* uniforms;     /* [S, n + 1] in [0, 1); may be NULL when greedy             */
  int64_t* tokens;           /* [S, n + 1]                                                */
  int32_t* accepted;         /* [S]                                                       */
  float* logp;               /* [S, n + 1], or NULL                                       */
  uint32_t flags;            /* PCP_FLAG_ASYNC                                            */
  void* stream;              /* hipStream_t; NULL => the default stream                   */
  int64_t target_seq_stride; /* elements between sequences; 0 => n + 1 rows               */
  int64_t draft_seq_stride;  /* elements between sequences; 0 => n rows                   */
} pcp_verify_args;

/* Defaults: strides 0, bf16, temperature 1. Strides may be in either order: rows of one
 * drafting step after another, [n, S, V], have a row stride of S * V and a sequence stride
 * of V. */
void pcp_verify_args_init(pcp_verify_args* a);
int pcp_verify_drafts(pcp_ctx* ctx, const pcp_verify_args* a);

#ifdef __cplusplus
}
#endif

#endif /* PCP_SAMPLE_H */
