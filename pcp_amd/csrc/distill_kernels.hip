// Entry point of the distillation from a teacher's top logits (pcp_distill.h): checks, work
// buffers and the choice of kernel. The kernels are in distill_device.hpp, compiled for one
// logits type per file.

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <cstring>

#include "context.hpp"
#include "distill_device.hpp"

namespace pcp {

hipError_t launch_distill_bf16(const DistillArgs& a, bool f32_out, hipStream_t st);
hipError_t launch_distill_f16(const DistillArgs& a, bool f32_out, hipStream_t st);
hipError_t launch_distill_f32(const DistillArgs& a, bool f32_out, hipStream_t st);

namespace {

hipError_t launch_distill(const DistillArgs& a, int in_dtype, int out_dtype, hipStream_t st) {
  const bool f32_out = out_dtype == PCP_F32;
  return in_dtype == PCP_BF16  ? launch_distill_bf16(a, f32_out, st)
         : in_dtype == PCP_F16 ? launch_distill_f16(a, f32_out, st)
                               : launch_distill_f32(a, f32_out, st);
}

inline size_t round256(size_t b) { return (b + 255) & ~static_cast<size_t>(255); }

inline bool misaligned(const void* p, int size) {
  return (reinterpret_cast<uintptr_t>(p) & static_cast<uintptr_t>(size - 1)) != 0;
}

// Rows in parts where they are wide and few: parts | a row to a workgroup, us, forward divergence
// with k = 64, by rows:
//   bf16 151,936   16  18 | 32   64 19 | 34   128 29 | 35   256 51 | 42   512 94 | 74   1024 170 | 142
//   bf16 100,000   16  18 | 29   64 19 | 31   128 23 | 31   256 39 | 35   512 68 | 57   1024 118 | 105
//   bf16  50,257   16  18 | 27   64 19 | 29   128 21 | 30   256 27 | 31   512 45 | 37   1024  72 |  66
//   bf16  33,000   16  19 | 24   64 20 | 25   128 21 | 27   256 24 | 27   512 34 | 33   1024  56 |  53
//   bf16  16,000   16  24 | 24   64 24 | 26   128 25 | 27   256 25 | 27   512 28 | 30   1024  41 |  37
//   f32   50,257   16  17 | 25   64 18 | 27   128 22 | 28   256 38 | 35   512 63 | 59   1024 113 | 105
constexpr int64_t kPartMinVecs = 4096, kPartMaxRows = 320;
constexpr int64_t kPartWideVecs = 12000, kPartMaxRowsWide = 192;
// The loss by the last workgroup to finish, where few take tickets; else by a kernel of its own.
// us per call, along | by its own kernel, by rows:
//   bf16 151,936   4  13 | 16   64 17 | 20   128 26 | 28   256 41 | 42   320 62 | 62   512 73 | 71   1024 144 | 142
//   bf16  50,257   4  14 | 17   64 15 | 18   128 18 | 20   256 23 | 26   320 27 | 29   512 35 | 35   1024  64 |  63
//   f32    1,024   4  17 | 18   64 18 | 20   128 19 | 20   256 19 | 21   320 20 | 21   512 23 | 23   1024  32 |  27
constexpr int64_t kAlongMaxRows = 320;

int distill(pcp_ctx* ctx, const pcp_distill_args* a) {
  if (!a) return fail(ctx, PCP_ERR_INVALID_ARG, "args is NULL");
  if (a->n_seq < 1) return fail(ctx, PCP_ERR_INVALID_ARG, "n_seq must be >= 1 (got %lld)", (long long)a->n_seq);
  if (a->rows < 0) return fail(ctx, PCP_ERR_INVALID_ARG, "rows must be >= 0");
  if (a->vocab < 1 || a->vocab > PCP_DISTILL_MAX_VOCAB)
    return fail(ctx, PCP_ERR_INVALID_ARG, "vocab must be in [1, %d] (got %lld)", PCP_DISTILL_MAX_VOCAB,
                (long long)a->vocab);
  if (a->k < 1 || a->k > PCP_TOP_LOGITS_MAX)
    return fail(ctx, PCP_ERR_INVALID_ARG, "k must be in [1, %d] (got %d)", PCP_TOP_LOGITS_MAX, a->k);
  const int64_t lstride = a->logit_seq_stride ? a->logit_seq_stride : a->rows;
  const int64_t tstride = a->tok_seq_stride ? a->tok_seq_stride : a->rows;
  if (lstride < a->rows || lstride < 1)
    return fail(ctx, PCP_ERR_INVALID_ARG, "logit_seq_stride (%lld) must be >= max(rows, 1)", (long long)lstride);
  if (a->tok_offset < 0 || a->tok_offset > tstride - a->rows)
    return fail(ctx, PCP_ERR_INVALID_ARG, "tok_offset + rows must fit in tok_seq_stride");
  int64_t nrows, tmp;
  if (mul_overflows(a->n_seq, lstride, &nrows) || nrows > INT32_MAX)
    return fail(ctx, PCP_ERR_OVERFLOW, "n_seq * logit_seq_stride exceeds 2^31-1 rows");
  if (mul_overflows(a->n_seq, tstride, &tmp) || mul_overflows(tmp, 4, &tmp))
    return fail(ctx, PCP_ERR_OVERFLOW, "token array size overflows int64");
  if (a->logits_dtype != PCP_BF16 && a->logits_dtype != PCP_F16 && a->logits_dtype != PCP_F32)
    return fail(ctx, PCP_ERR_DTYPE, "logits dtype must be bf16, f16 or f32 (got %d)", a->logits_dtype);
  if (a->dlogits && a->dlogits_dtype != a->logits_dtype && a->dlogits_dtype != PCP_F32)
    return fail(ctx, PCP_ERR_DTYPE, "dlogits dtype must equal the logits dtype or be f32");
  if (a->ids_dtype != PCP_I64 && a->ids_dtype != PCP_I32)
    return fail(ctx, PCP_ERR_DTYPE, "teacher_ids dtype must be i64 or i32 (got %d)", a->ids_dtype);
  if (a->mask && a->mask_dtype != PCP_F32 && a->mask_dtype != PCP_BOOL)
    return fail(ctx, PCP_ERR_DTYPE, "mask dtype must be f32 or bool (got %d)", a->mask_dtype);
  if (!a->logits || !a->teacher_ids || !a->teacher_logits)
    return fail(ctx, PCP_ERR_INVALID_ARG, "logits / teacher_ids / teacher_logits is NULL");
  if (misaligned(a->logits, dtype_bytes(a->logits_dtype)) || misaligned(a->teacher_ids, dtype_bytes(a->ids_dtype)) ||
      misaligned(a->teacher_logits, 4) || misaligned(a->teacher_lse, 4) || misaligned(a->token_loss, 4) ||
      misaligned(a->loss, 4) || (a->mask && misaligned(a->mask, a->mask_dtype == PCP_F32 ? 4 : 1)) ||
      (a->dlogits && misaligned(a->dlogits, dtype_bytes(a->dlogits_dtype))))
    return fail(ctx, PCP_ERR_INVALID_ARG, "pointers must be aligned to their element size");
  if (a->dlogits) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a->logits), d = reinterpret_cast<uintptr_t>(a->dlogits);
    const uintptr_t n = static_cast<uintptr_t>(nrows) * static_cast<uintptr_t>(a->vocab);
    const bool apart = d + n * dtype_bytes(a->dlogits_dtype) <= x || x + n * dtype_bytes(a->logits_dtype) <= d;
    if (!apart && !(x == d && a->dlogits_dtype == a->logits_dtype))
      return fail(ctx, PCP_ERR_INVALID_ARG, "dlogits overlaps the logits without being them");
  }
  if (a->divergence != PCP_DIVERGENCE_FORWARD && a->divergence != PCP_DIVERGENCE_REVERSE)
    return fail(ctx, PCP_ERR_INVALID_ARG, "unknown divergence %d", a->divergence);
  if (a->divergence == PCP_DIVERGENCE_REVERSE && !a->teacher_lse)
    return fail(ctx, PCP_ERR_INVALID_ARG, "the reverse divergence needs teacher_lse");
  const float k2 = static_cast<float>(1.4426950408889634074 / static_cast<double>(a->temperature));
  if (!(a->temperature > 0.f) || !std::isfinite(a->temperature) || !std::isnormal(k2))
    return fail(ctx, PCP_ERR_INVALID_ARG, "temperature must be positive and finite (and its inverse a normal f32)");
  if (!(a->weight > 0.f) || !std::isfinite(a->weight))
    return fail(ctx, PCP_ERR_INVALID_ARG, "weight must be positive and finite");
  if (!(a->loss_norm >= 0.f) || !std::isfinite(a->loss_norm))
    return fail(ctx, PCP_ERR_INVALID_ARG, "loss_norm must be >= 0 and finite");
  if (a->flags & ~PCP_FLAG_ASYNC) return fail(ctx, PCP_ERR_INVALID_ARG, "only PCP_FLAG_ASYNC applies here");
  if (!ctx) return fail(nullptr, PCP_ERR_INVALID_ARG, "context is NULL");
  const DeviceScope scope(ctx->device);
  if (scope.error() != hipSuccess) return hip_fail(ctx, scope.error(), "making the context's device current");
  hipStream_t st = static_cast<hipStream_t>(a->stream);

  const int64_t nv = a->vocab * dtype_bytes(a->logits_dtype) / 16;
  // A row to a workgroup where rows fit and are many or narrow, else in parts.
  const bool together = a->dlogits && (a->dlogits_dtype != a->logits_dtype ||
                                       ((reinterpret_cast<uintptr_t>(a->logits) ^
                                         reinterpret_cast<uintptr_t>(a->dlogits)) & 15u) == 0) &&
                        nv <= kDistillRowVecs &&
                        (nv < kPartMinVecs || nrows > (nv < kPartWideVecs ? kPartMaxRows : kPartMaxRowsWide));
  const int64_t parts = together ? 0 : nv > 0 ? (nv + kPartBlock * kPartU - 1) / (kPartBlock * kPartU) : 1;
  // Scratch: seq_len | seq_scale | seq_val | loss, counters | token_loss | rows' records |
  // entries' ids, logits, weights | parts.
  const size_t sv = round256(sizeof(float) * static_cast<size_t>(a->n_seq));
  const size_t tl = a->token_loss ? 0 : round256(sizeof(float) * static_cast<size_t>(a->n_seq * tstride));
  const size_t pb = round256(sizeof(PartSum) * static_cast<size_t>(nrows) * static_cast<size_t>(parts));
  const size_t tb = round256(sizeof(TeacherRow) * static_cast<size_t>(nrows));
  const size_t eb = round256(sizeof(float) * static_cast<size_t>(nrows) * static_cast<size_t>(a->k));
  const int rc = ensure_scratch_on(ctx, 3 * sv + 512 + tl + tb + 4 * eb + pb, st);
  if (rc != PCP_OK) return rc;
  char* sp = static_cast<char*>(ctx->scratch);
  float* s_len = reinterpret_cast<float*>(sp);
  float* s_scale = reinterpret_cast<float*>(sp + sv);
  float* s_val = reinterpret_cast<float*>(sp + 2 * sv);
  float* s_loss = reinterpret_cast<float*>(sp + 3 * sv);
  int* s_done = reinterpret_cast<int*>(sp + 3 * sv + 256);
  int* s_next = reinterpret_cast<int*>(sp + 3 * sv + 256 + 64);
  float* s_tl = a->token_loss ? a->token_loss : reinterpret_cast<float*>(sp + 3 * sv + 512);

  // weight / loss_norm as one divisor: the loss and every scale below carry both.
  const float norm = (a->loss_norm > 0.f ? a->loss_norm : static_cast<float>(a->n_seq)) / a->weight;
  DistillArgs d;
  std::memset(&d, 0, sizeof(d));
  d.logits = a->logits;
  d.tids = a->teacher_ids;
  d.tlogits = a->teacher_logits;
  d.tlse = a->teacher_lse;
  d.mask = a->mask;
  d.seq_len = s_len;
  d.seq_scale = s_scale;
  d.n_seq = a->n_seq;
  d.done = s_done;
  d.loss_norm = norm;
  d.dlogits = a->dlogits;
  d.token_loss = s_tl;
  char* work = sp + 3 * sv + 512 + tl;
  d.teacher = reinterpret_cast<TeacherRow*>(work);
  d.entry_ids = reinterpret_cast<int*>(work + tb);
  d.entry_z = reinterpret_cast<float*>(work + tb + eb);
  d.entry_w = reinterpret_cast<double*>(work + tb + 2 * eb);
  d.part = reinterpret_cast<PartSum*>(work + tb + 4 * eb);
  d.err = ctx->d_page->err;
  d.next_row = s_next;
  d.nrows = nrows;
  d.vocab = a->vocab;
  d.rows = a->rows;
  d.logit_stride = lstride;
  d.tok_stride = tstride;
  d.tok_offset = a->tok_offset;
  d.inv_tau = 1. / static_cast<double>(a->temperature);
  d.k2 = k2;
  d.k = a->k;
  d.ids_i64 = a->ids_dtype == PCP_I64;
  d.mask_u8 = a->mask_dtype == PCP_BOOL;
  d.forward = a->divergence == PCP_DIVERGENCE_FORWARD;
  d.parts = static_cast<int32_t>(parts);
  d.per = parts ? static_cast<int32_t>((nv + parts - 1) / parts) : 0;
  const bool along = nrows <= kAlongMaxRows;
  if (along) d.loss = a->loss ? a->loss : s_loss;

  const bool timed = prof_begin(ctx, st);
  hipError_t e = launch_distill(d, a->logits_dtype, a->dlogits ? a->dlogits_dtype : a->logits_dtype, st);
  prof_end(ctx, st, timed);
  if (e != hipSuccess) return hip_fail(ctx, e, "distillation launch");
  if (along) return finish_call(ctx, a->flags, st);
  const LossReduceArgs la{s_tl, a->rows, tstride, a->tok_offset, s_len, nullptr, 0, s_val, a->n_seq, norm, s_done,
                          a->loss ? a->loss : s_loss};
  if ((e = launch_loss_reduce_fused(la, st)) != hipSuccess) return hip_fail(ctx, e, "loss reduction launch");
  return finish_call(ctx, a->flags, st);
}

}  // namespace
}  // namespace pcp

using namespace pcp;

extern "C" void pcp_distill_args_init(pcp_distill_args* a) {
  if (!a) return;
  std::memset(a, 0, sizeof(*a));
  a->logits_dtype = PCP_BF16;
  a->dlogits_dtype = PCP_BF16;
  a->ids_dtype = PCP_I32;
  a->mask_dtype = PCP_F32;
  a->divergence = PCP_DIVERGENCE_FORWARD;
  a->temperature = 1.f;
  a->weight = 1.f;
}

extern "C" int pcp_distill_fwd_bwd(pcp_ctx* ctx, const pcp_distill_args* a) { return distill(ctx, a); }
