// The k largest logits of rows with their ids and the rows' log-sum-exp
// (pcp_top_logits, pcp_distill.h).
//
// An element is ordered by a 64-bit key: its logit's bits made monotone, then the id
// complemented, so that no two are equal and equal logits fall by rising id. A workgroup
// streams its part of a row once. It keeps candidates in LDS and a threshold that at least
// k of the elements seen reach: first from a histogram of the maxima of the 16-byte vectors
// of its first batch, later, as the list grows, from a histogram of the candidates. Few
// elements pass it, so the row costs one read, the log-sum-exp's arithmetic and a comparison
// per vector. Rows in any order are right: a batch of which too much passes is taken again
// in small rounds, and a list that a histogram cannot thin (equal values) is sorted. A row
// with one part is ranked and written by its workgroup; else each part leaves its
// candidates and a second kernel merges them.
//
// Bound by the exponentials and HBM with many rows (4096 rows of 151,936 bf16, k = 64: 202 us,
// 6.2 TB/s; 231 while every lane looked at each vector that passed in any, 474 with thresholds from sorted
// lists and a pass of its own for the vectors' maxima), by latency with few: one such row takes
// 7.9 us in 10 parts and 6.3 to merge them. The merge of many long lists costs most: 192 rows,
// k = 256, 25 + 17 us. Rows with fewer than k logits above the masks, or of equal values, have no
// threshold, and every element goes through the candidates' loop: 4096 rows of 151,936 with 40 tokens
// left 961 us (plain 241 in the same run), 512 rows 213 (42), 64 rows 136 (18), one row 111 (14); so does a
// part that holds nothing but masks: half of the vocabulary in a run, 64 rows 102, one row 92.

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <cstring>

#include "context.hpp"
#include "grpo_device.hpp"
#include "pcp_distill.h"
#include "top_device.hpp"

namespace pcp {
namespace {

struct TopArgs {
  const void* logits;
  int64_t n_rows, vocab, row_stride;
  int64_t row0;
  float* values;
  void* ids;
  float* lse;
  uint64_t* part_key;     // [n_rows, parts, part_cap]
  PartSum* part_sum;      // [n_rows, parts]: n the candidates left
  int* err;
  double inv_tau;
  float k2;               // log2(e) / temperature
  int32_t k, ids_i64, parts, per, part_cap;
};

// A lane's largest logit and its sum against it: a batch's in f32, the batches' in f64 (a lane has
// up to 65,536 elements of a row).
struct TopSums {
  float k2, mx, adj;
  double s;
  TermScale ts;

  // Terms against the lane's maximum so far, and the vectors compared by their largest term:
  // no pass for a new maximum unless one has risen far above.
  template <typename TI, int U, typename Held>
  __device__ __forceinline__ bool add(const u32x4 (&x)[U], Held held, float least_x, bool (&near)[U]) {
    constexpr int EPV = 16 / TI::kBytes;
    const float cut = hw_exp2(fmaf(least_x, ts.k, -ts.ref)) * (1.f - 0x1p-16f);
    const float floor = cut > 0x1p-100f ? cut : 0.f;   // rounding above, underflow below
    float acc = 0.f, most = 0.f;
#pragma unroll
    for (int q = 0; q < U; ++q) {
      float e[EPV], ve = 0.f;
      if (held(q)) {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(&x[q]);
#pragma unroll
        for (int j = 0; j < EPV; ++j) {
          e[j] = hw_exp2(fmaf(TI::unpack(w, j), ts.k, -ts.ref));
          acc += e[j];
        }
#pragma unroll
        for (int j = 0; j < EPV; j += 2) ve = max3(ve, e[j], e[j + 1]);
      }
      near[q] = held(q) && ve >= floor;
      most = fmaxf(most, ve);
    }
    if (__any(most > 0x1p40f)) return false;
    s += static_cast<double>(acc * adj);
    return true;
  }
  template <typename TI, int U, typename Held>
  __device__ __forceinline__ void fresh(const u32x4 (&x)[U], Held held, float bx) {
    const float nm = fmaxf(mx, bx);
    ts = term_scale(nm, k2);
    adj = term_adj(nm, ts);
    float acc = 0.f;
#pragma unroll
    for (int q = 0; q < U; ++q)
      if (held(q)) {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(&x[q]);
#pragma unroll
        for (int j = 0; j < 16 / TI::kBytes; ++j) acc += hw_exp2(fmaf(TI::unpack(w, j), ts.k, -ts.ref));
      }
    s = rescale_at(s, mx, nm, k2) + static_cast<double>(acc * adj);
    mx = nm;
  }
};

// The 16-byte vectors [v0, end) of a row interior (sp) through xbuf: every element goes into the lane's
// sums, and those that may be among the k largest into the candidates, which hold `edges` elements
// at the start and at most `left` (>= k) at the end, few more than k where the row lets them. Called by the whole
// workgroup after a barrier; ends with one.
template <typename TI>
__device__ __forceinline__ void scan_part(const RowSpan& sp, __amdgpu_buffer_rsrc_t xbuf, int v0, int end, int edges, int k,
                                          int left, TopSums& sums, Candidates& c, Shared& sh) {
  constexpr int EPV = 16 / TI::kBytes, U = kU, BLOCK = kBlock;
  const int tid = threadIdx.x;
  // The candidates are thinned where they pass `limit`; after the last batch to about k.
  const int room = min(kCut, 2 * k + 128);
  constexpr int kRounds = U * EPV / 4;                   // of 4 elements per lane
  int n = edges;                                         // candidates before the batch
  int round = -1;                                        // >= 0: a batch taken in rounds
  for (int base = v0; base < end;) {
    u32x4 x[U];
    const uint32_t off = static_cast<uint32_t>(base + tid) * 16u;
#pragma unroll
    for (int q = 0; q < U; ++q) x[q] = buf_ld16<true>(xbuf, off + q * (BLOCK * 16u));
    auto held = [&](int q) { return base + q * BLOCK + tid < end; };
    bool near[U];   // this lane's vector may hold an element that passes
    bool fresh = round >= 0 || base == v0 || __any(sums.mx == kNegInf);
    if (!fresh) fresh = !sums.template add<TI>(x, held, c.least_x, near);
    if (fresh) {
      float vm[U], bx = kNegInf;
#pragma unroll
      for (int q = 0; q < U; ++q) {
        vm[q] = held(q) ? vec_max<TI>(kNegInf, x[q]) : kNegInf;
        bx = fmaxf(bx, vm[q]);
      }
      if (round < 0) {
        sums.template fresh<TI>(x, held, bx);
        // k vectors of the first batch reach this, each with one element at least.
        if (base == v0) c.least_x = reached_by(sh, vm, k);
      }
#pragma unroll
      for (int q = 0; q < U; ++q) near[q] = held(q) && (vm[q] >= c.least_x || c.least_x == kNegInf);
    }
    uint32_t left_q = 0;
#pragma unroll
    for (int q = 0; q < U; ++q) left_q |= near[q] ? 1u << q : 0u;
    if (round >= 0) left_q &= 1u << (round / (EPV / 4));
    uint32_t keep = (1u << EPV) - 1u;
    if (round >= 0) keep = 0xf0u >> (EPV == 4 ? 4 : 4 * (round % 2));
    take_vectors<TI>(c, x, left_q, static_cast<uint32_t>(sp.head + (base + tid) * EPV), keep);
    __syncthreads();
    const int was = n;
    n = sh.count;
    __syncthreads();
    if (round < 0 && n > kCap) {   // too many at once: this batch again, in rounds that are sure to fit
      if (tid == 0) sh.count = was;
      n = was;
      round = 0;
    } else if (round < 0 || ++round == kRounds) {
      round = -1;
      base += BLOCK * U;
    }
    if (n > (base >= end ? left : round >= 0 ? kCut : room)) n = c.thin(n, k, base >= end ? left : kCut);
    else __syncthreads();
  }
}

__device__ __forceinline__ void write_entries(const TopArgs& a, int64_t row, Shared& sh, int n) {
  rank_entries(sh, n, a.k, [&](int rank, float x, int64_t id) {
    a.values[row * a.k + rank] = x;
    if (a.ids_i64) static_cast<int64_t*>(a.ids)[row * a.k + rank] = id;
    else static_cast<int32_t*>(a.ids)[row * a.k + rank] = static_cast<int32_t>(id);
  });
}

// From the row's sum against its largest logit, which may leave f32's range divided by the temperature.
__device__ __forceinline__ void write_lse(const TopArgs& a, int64_t row, float mx, float s) {
  const float lse = static_cast<float>(static_cast<double>(mx) * a.inv_tau + ms_lse(0.f, s));
  if (a.lse) a.lse[row] = lse;
  if (!__builtin_isfinite(lse)) raise_error(a.err, kErrNonFinite);
}

// 5 waves a SIMD: at 6 a register is spilled, and 2048 f32 rows of 50,257 take 74 us instead of 69.
template <typename TI>
__global__ void __launch_bounds__(kBlock, 5) top_part_kernel(TopArgs a) {
  constexpr int BLOCK = kBlock;
  __shared__ __align__(16) Shared sh;
  __shared__ float2 wave_sum[kWaves];
  const int tid = threadIdx.x, part = blockIdx.x;
  const int64_t row = a.row0 + blockIdx.y;
  const char* xrow = static_cast<const char*>(a.logits) + row * a.row_stride * TI::kBytes;
  const RowSpan sp = row_span<TI>(xrow, a.vocab);
  const int v0 = part * a.per, end = min(v0 + a.per, sp.nv);
  const __amdgpu_buffer_rsrc_t xbuf = row_rsrc(sp.vec, static_cast<uint32_t>(max(end, 0)) * 16u);
  Candidates c{sh, 0, kNegInf};
  if (tid == 0) sh.count = 0;
  TopSums sums{a.k2, kNegInf, 1.f, 0., TermScale{a.k2, 0.f}};
  __syncthreads();
  if (part == 0 && tid < 64) {   // the elements outside the interior
    const int ek = edge_index<TI>(sp, tid);
    float xe = kNegInf;
    if (ek >= 0) {
      xe = TI::load1(xrow, ek);
      sums.mx = fmaxf(sums.mx, xe);
      sums.s = hw_exp2((xe - ms_ref(sums.mx)) * a.k2);
    }
    c.add(ek >= 0, element_key(xe, static_cast<uint32_t>(ek)));
  }
  scan_part<TI>(sp, xbuf, v0, end, part == 0 ? sp.head + sp.tail : 0, a.k, a.parts == 1 ? a.k + 64 : a.part_cap, sums, c,
                sh);
  __syncthreads();
  const int n = sh.count;
  float mx = sums.mx, sum = static_cast<float>(sums.s);
  block_merge_at<BLOCK>(mx, sum, a.k2, wave_sum);
  if (a.parts == 1) {
    write_entries(a, row, sh, n);
    if (tid == 0) write_lse(a, row, mx, sum);
  } else {
    uint64_t* out = a.part_key + (row * a.parts + part) * a.part_cap;
    for (int i = tid; i < n; i += BLOCK) out[i] = sh.key[i];
    if (tid == 0) a.part_sum[row * a.parts + part] = PartSum{mx, sum, n, 0};
  }
}

__global__ void __launch_bounds__(kBlock) top_merge_kernel(TopArgs a) {
  __shared__ __align__(16) Shared sh;
  const int tid = threadIdx.x;
  const int64_t row = a.row0 + blockIdx.x;
  const PartSum* sums = a.part_sum + row * a.parts;
  const uint64_t* in = a.part_key + row * a.parts * a.part_cap;
  const int n = merge_parts([&](int i) { return in[i]; }, a.parts, a.part_cap, a.k, [&](int p) { return sums[p].n; }, sh);
  write_entries(a, row, sh, n);
  if (tid < 64) {
    float mx = kNegInf, s = 0.f;
    if (tid < a.parts) {
      mx = sums[tid].mx;
      s = sums[tid].s;
    }
    lanes_merge_at<64>(mx, s, a.k2);
    if (tid == 0) write_lse(a, row, mx, s);
  }
}

template <typename TI>
hipError_t launch_top(TopArgs a, hipStream_t st) {
  constexpr int64_t kRows = 65535;   // grid.y
  for (int64_t r0 = 0; r0 < a.n_rows; r0 += kRows) {
    a.row0 = r0;
    const unsigned n = static_cast<unsigned>(a.n_rows - r0 < kRows ? a.n_rows - r0 : kRows);
    top_part_kernel<TI><<<dim3(static_cast<unsigned>(a.parts), n), dim3(kBlock), 0, st>>>(a);
    if (a.parts > 1) top_merge_kernel<<<dim3(n), dim3(kBlock), 0, st>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

inline bool misaligned(const void* p, int size) {
  return (reinterpret_cast<uintptr_t>(p) & static_cast<uintptr_t>(size - 1)) != 0;
}

int top_logits(pcp_ctx* ctx, const pcp_top_logits_args* a) {
  if (!a) return fail(ctx, PCP_ERR_INVALID_ARG, "args is NULL");
  if (a->n_rows < 0 || a->n_rows > INT32_MAX)
    return fail(ctx, PCP_ERR_INVALID_ARG, "n_rows must be in [0, 2^31-1] (got %lld)", (long long)a->n_rows);
  if (a->vocab < 1 || a->vocab > PCP_DISTILL_MAX_VOCAB)
    return fail(ctx, PCP_ERR_INVALID_ARG, "vocab must be in [1, %d] (got %lld)", PCP_DISTILL_MAX_VOCAB,
                (long long)a->vocab);
  if (a->k < 1 || a->k > PCP_TOP_LOGITS_MAX || a->k > a->vocab)
    return fail(ctx, PCP_ERR_INVALID_ARG, "k must be in [1, min(vocab, %d)] (got %d)", PCP_TOP_LOGITS_MAX, a->k);
  const int64_t stride = a->row_stride ? a->row_stride : a->vocab;
  if (stride < a->vocab)
    return fail(ctx, PCP_ERR_INVALID_ARG, "row_stride (%lld) must be >= vocab", (long long)stride);
  int64_t tmp;
  if (mul_overflows(a->n_rows, stride, &tmp) || mul_overflows(tmp, 4, &tmp))
    return fail(ctx, PCP_ERR_OVERFLOW, "logits byte size overflows int64");
  if (a->logits_dtype != PCP_BF16 && a->logits_dtype != PCP_F16 && a->logits_dtype != PCP_F32)
    return fail(ctx, PCP_ERR_DTYPE, "logits dtype must be bf16, f16 or f32 (got %d)", a->logits_dtype);
  if (a->ids_dtype != PCP_I64 && a->ids_dtype != PCP_I32)
    return fail(ctx, PCP_ERR_DTYPE, "ids dtype must be i64 or i32 (got %d)", a->ids_dtype);
  const float k2 = static_cast<float>(1.4426950408889634074 / static_cast<double>(a->temperature));
  if (!(a->temperature > 0.f) || !std::isfinite(a->temperature) || !std::isnormal(k2))
    return fail(ctx, PCP_ERR_INVALID_ARG, "temperature must be positive and finite (and its inverse a normal f32)");
  if (a->flags & ~PCP_FLAG_ASYNC) return fail(ctx, PCP_ERR_INVALID_ARG, "only PCP_FLAG_ASYNC applies here");
  if (a->n_rows > 0 && (!a->logits || !a->values || !a->ids))
    return fail(ctx, PCP_ERR_INVALID_ARG, "logits / values / ids is NULL");
  if (misaligned(a->logits, dtype_bytes(a->logits_dtype)) || misaligned(a->ids, dtype_bytes(a->ids_dtype)) ||
      misaligned(a->values, 4) || misaligned(a->lse, 4))
    return fail(ctx, PCP_ERR_INVALID_ARG, "pointers must be aligned to their element size");
  if (!ctx) return fail(nullptr, PCP_ERR_INVALID_ARG, "context is NULL");
  if (a->n_rows == 0) return PCP_OK;
  const DeviceScope scope(ctx->device);
  if (scope.error() != hipSuccess) return hip_fail(ctx, scope.error(), "making the context's device current");
  hipStream_t st = static_cast<hipStream_t>(a->stream);

  // Workgroups per row: one from 512 rows on, which need no merge then; below, no more than it takes
  // to fill the chip (2048), at least a batch each. us for 2048 | 1024 workgroups in all | one per row:
  //   bf16 151,936, k 64    128 rows 21 | 23 | 34   256 29 | 32 | 36   400 39 | 40 | 42   512 49 | 42 | 42   1024 69 | 60 | 59
  //   f16  151,936, k 256   128      37 | 34 | 56   256 41 | 44 | 49   400 54 | 55 | 56   512 66 | 57 | 56   1024 89 | 76 | 76
  //   f32   50,257, k 20    128      16 | 16 | 21   256 21 | 20 | 22   400 26 | 24 | 24   512 29 | 29 | 25   1024 50 | 41 | 40
  //   bf16  50,257, k 64    128      16 | 15 | 17   256 20 | 19 | 18   400 24 | 25 | 21   512 26 | 26 | 21   1024 40 | 28 | 29
  const int64_t nv = a->vocab * dtype_bytes(a->logits_dtype) / 16;
  const int64_t batches = nv > 0 ? (nv + kBlock * kU - 1) / (kBlock * kU) : 1;
  int64_t parts = a->n_rows < 512 ? (2048 + a->n_rows - 1) / a->n_rows : 1;
  if (parts > batches) parts = batches;
  if (parts > 64) parts = 64;   // one wave merges their sums
  const int64_t per_batches = (batches + parts - 1) / parts;
  parts = (batches + per_batches - 1) / per_batches;
  const int64_t part_cap = a->k + 64;
  const size_t keys = parts > 1 ? sizeof(uint64_t) * static_cast<size_t>(a->n_rows) * parts * part_cap : 0;
  const size_t sums = parts > 1 ? sizeof(PartSum) * static_cast<size_t>(a->n_rows) * parts + 16 : 0;
  const int rc = ensure_scratch_on(ctx, keys + sums, st);
  if (rc != PCP_OK) return rc;

  TopArgs t;
  std::memset(&t, 0, sizeof(t));
  t.logits = a->logits;
  t.n_rows = a->n_rows;
  t.vocab = a->vocab;
  t.row_stride = stride;
  t.values = a->values;
  t.ids = a->ids;
  t.lse = a->lse;
  t.part_key = static_cast<uint64_t*>(ctx->scratch);
  t.part_sum = reinterpret_cast<PartSum*>(static_cast<char*>(ctx->scratch) + ((keys + 15) & ~static_cast<size_t>(15)));
  t.err = ctx->d_page->err;
  t.inv_tau = 1. / static_cast<double>(a->temperature);
  t.k2 = k2;
  t.k = a->k;
  t.ids_i64 = a->ids_dtype == PCP_I64;
  t.parts = static_cast<int32_t>(parts);
  t.per = static_cast<int32_t>(per_batches * kBlock * kU);
  t.part_cap = static_cast<int32_t>(part_cap);
  const bool timed = prof_begin(ctx, st);
  const hipError_t e = a->logits_dtype == PCP_F32    ? launch_top<F32T>(t, st)
                       : a->logits_dtype == PCP_BF16 ? launch_top<BF16T>(t, st)
                                                     : launch_top<F16T>(t, st);
  prof_end(ctx, st, timed);
  if (e != hipSuccess) return hip_fail(ctx, e, "top logits launch");
  return finish_call(ctx, a->flags, st);
}

}  // namespace
}  // namespace pcp

using namespace pcp;

extern "C" void pcp_top_logits_args_init(pcp_top_logits_args* a) {
  if (!a) return;
  std::memset(a, 0, sizeof(*a));
  a->k = 1;
  a->logits_dtype = PCP_BF16;
  a->ids_dtype = PCP_I32;
  a->temperature = 1.f;
}

extern "C" int pcp_top_logits(pcp_ctx* ctx, const pcp_top_logits_args* a) { return top_logits(ctx, a); }
