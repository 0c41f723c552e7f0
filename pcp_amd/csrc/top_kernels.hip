// The k largest logits of rows with their ids and the rows' log-sum-exp
// (pcp_top_logits, pcp_distill.h).
//
// An element is ordered by a 64-bit key: its logit's bits made monotone, then the id
// complemented, so that no two are equal and equal logits fall by rising id. A workgroup
// streams its part of a row once. It keeps candidates in LDS and a threshold that at least
// k of the elements seen reach: at first the k-th largest of its lanes' maxima over the
// first batch, later the k-th candidate whenever the list is cut back. Few elements pass
// it, so the row costs one read, the log-sum-exp's arithmetic and a comparison each; rows
// in any order are right, falling back to cuts every 1,024 elements where they pass in
// numbers. A row with one part is sorted and written by its workgroup; else each part
// leaves its k best and a second kernel merges them.

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <cstring>

#include "context.hpp"
#include "grpo_device.hpp"
#include "pcp_distill.h"

namespace pcp {
namespace {

constexpr int kBlock = 256;
constexpr int kU = 8;              // 16-byte vectors per lane and batch
constexpr int kCap = 2048;         // candidates held
constexpr int kCut = 1024;         // cut back past this many: a cautious round adds at most kCap - kCut

struct TopArgs {
  const void* logits;
  int64_t n_rows, vocab, row_stride;
  int64_t row0;
  float* values;
  void* ids;
  float* lse;
  uint64_t* part_key;     // [n_rows, parts, k]
  float2* part_ms;        // [n_rows, parts]
  int* err;
  float k2;               // log2(e) / temperature
  double to_nat;          // ln 2: base-2 state to natural units
  int32_t k, ids_i64, parts, per;
};

// Monotone in x; -0 as 0, NaN below everything.
__device__ __forceinline__ uint32_t order_bits(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return x == x ? (b & 0x80000000u ? ~b : b | 0x80000000u) : 0u;
}
__device__ __forceinline__ float from_order(uint32_t k) {
  return k == 0u ? __builtin_nanf("") : __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ uint64_t element_key(float x, uint32_t id) {
  return static_cast<uint64_t>(order_bits(x)) << 32 | (0xffffffffu - id);
}

// c[0, n) into falling order (n <= kCap; the rest up to a power of two becomes 0).
__device__ __forceinline__ void sort_falling(uint64_t* c, int n) {
  int size = 2;
  while (size < n) size <<= 1;
  for (int i = n + threadIdx.x; i < size; i += kBlock) c[i] = 0;
  __syncthreads();
  for (int span = 2; span <= size; span <<= 1)
    for (int step = span >> 1; step > 0; step >>= 1) {
      for (int t = threadIdx.x; t < size / 2; t += kBlock) {
        const int i = 2 * t - (t & (step - 1)), j = i + step;
        const uint64_t a = c[i], b = c[j];
        if ((a < b) == ((i & span) == 0)) {
          c[i] = b;
          c[j] = a;
        }
      }
      __syncthreads();
    }
}

struct Candidates {
  uint64_t* key;       // LDS [kCap]
  int* count;          // LDS
  uint64_t least;      // keys above this pass (0: all)
  float least_x;       // no element below this passes

  // Called by every lane of a wave.
  __device__ __forceinline__ void add(bool pass, uint64_t k) {
    const uint64_t who = __ballot(pass);
    if (who == 0) return;
    const int before = __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(who >> 32),
                                                 __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(who), 0));
    int at = 0;
    if (before == 0 && pass) at = atomicAdd(count, __popcll(who));
    at = __builtin_amdgcn_readlane(at, __builtin_ctzll(who)) + before;
    if (pass && at < kCap) key[at] = k;
  }
  // Keeps the k largest of the n held, in falling order; called by the whole workgroup.
  __device__ __forceinline__ int cut(int n, int k) {
    sort_falling(key, n);
    const int left = min(n, k);
    if (n >= k) {
      least = key[k - 1] - 1;   // the k-th itself is held already, and no other key equals it
      least_x = from_order(static_cast<uint32_t>(key[k - 1] >> 32));
    }
    __syncthreads();
    if (threadIdx.x == 0) *count = left;
    __syncthreads();
    return left;
  }
};

// A row's entries from the sorted candidates.
__device__ __forceinline__ void write_entries(const TopArgs& a, int64_t row, const uint64_t* key) {
  for (int i = threadIdx.x; i < a.k; i += kBlock) {
    const uint64_t v = key[i];
    const int64_t id = 0xffffffffu - static_cast<uint32_t>(v);
    a.values[row * a.k + i] = from_order(static_cast<uint32_t>(v >> 32));
    if (a.ids_i64) static_cast<int64_t*>(a.ids)[row * a.k + i] = id;
    else static_cast<int32_t*>(a.ids)[row * a.k + i] = static_cast<int32_t>(id);
  }
}

__device__ __forceinline__ void write_lse(const TopArgs& a, int64_t row, float m, float s) {
  const double lse = ms_lse(m, s);
  if (a.lse) a.lse[row] = static_cast<float>(lse);
  if (!__builtin_isfinite(lse)) raise_error(a.err, kErrNonFinite);
}

template <typename TI>
__global__ void __launch_bounds__(kBlock) top_part_kernel(TopArgs a) {
  constexpr int EPV = 16 / TI::kBytes, U = kU, BLOCK = kBlock;
  __shared__ uint64_t key[kCap];
  __shared__ __align__(16) float lds[4 * (BLOCK / 64)];
  __shared__ float lane_max[BLOCK];
  __shared__ int count;
  __shared__ float first_least;
  const int tid = threadIdx.x, part = blockIdx.x;
  const int64_t row = a.row0 + blockIdx.y;
  const char* xrow = static_cast<const char*>(a.logits) + row * a.row_stride * TI::kBytes;
  const RowSpan sp = row_span<TI>(xrow, a.vocab);
  const int v0 = part * a.per, end = min(v0 + a.per, sp.nv);
  const __amdgpu_buffer_rsrc_t xbuf = row_rsrc(sp.vec, static_cast<uint32_t>(max(end, 0)) * 16u);
  Candidates c{key, &count, 0, kNegInf};
  if (tid == 0) {
    count = 0;
    first_least = kNegInf;
  }
  float m = kNegInf, s = 0.f;
  __syncthreads();
  if (part == 0 && tid < 64) {   // the elements outside the interior
    const int ek = edge_index<TI>(sp, tid);
    float xe = kNegInf;
    if (ek >= 0) {
      xe = TI::load1(xrow, ek);
      m = fmaxf(m, xe * a.k2);
      s = hw_exp2(fmaf(xe, a.k2, -ms_ref(m)));
    }
    c.add(ek >= 0, element_key(xe, static_cast<uint32_t>(ek)));
  }
  for (int base = v0; base < end; base += BLOCK * U) {
    u32x4 x[U];
    const uint32_t off = static_cast<uint32_t>(base + tid) * 16u;
#pragma unroll
    for (int q = 0; q < U; ++q) x[q] = buf_ld16<true>(xbuf, off + q * (BLOCK * 16u));
    auto held = [&](int q) { return base + q * BLOCK + tid < end; };
    float bx = kNegInf;
#pragma unroll
    for (int q = 0; q < U; ++q)
      if (held(q)) bx = vec_max<TI>(bx, x[q]);
    {
      const float nm = fmaxf(m, bx * a.k2), ref = ms_ref(nm);
      float acc = ms_rescale(s, m, nm);
#pragma unroll
      for (int q = 0; q < U; ++q)
        if (held(q)) {
          const uint32_t* w = reinterpret_cast<const uint32_t*>(&x[q]);
#pragma unroll
          for (int j = 0; j < EPV; ++j) acc += hw_exp2(fmaf(TI::unpack(w, j), a.k2, -ref));
        }
      m = nm;
      s = acc;
    }
    if (base == v0) {
      // The k-th largest of the lanes' maxima: k elements of this batch reach it.
      lane_max[tid] = bx;
      __syncthreads();
      int above = 0;
      for (int i = 0; i < BLOCK; ++i) above += lane_max[i] > bx || (lane_max[i] == bx && i < tid);
      if (above == a.k - 1) first_least = bx;
      __syncthreads();
      c.least_x = first_least;
    }
    auto offer = [&](int q, int j0, int j1) {
#pragma unroll
      for (int j = j0; j < j1; ++j) {
        const float v = TI::unpack(reinterpret_cast<const uint32_t*>(&x[q]), j);
        const bool near = held(q) && !(v < c.least_x);
        if (__any(near)) {
          const uint32_t id = static_cast<uint32_t>(sp.head + (base + q * BLOCK + tid) * EPV + j);
          const uint64_t k = element_key(v, id);
          c.add(near && k > c.least, k);
        }
      }
    };
    __syncthreads();
    const int before = count;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < U; ++q) offer(q, 0, EPV);
    __syncthreads();
    int n = count;
    if (n > kCap) {   // too many at once: this batch again, in rounds that are sure to fit
      __syncthreads();
      if (tid == 0) count = before;
      __syncthreads();
      n = before;
#pragma unroll
      for (int q = 0; q < U; ++q)
#pragma unroll
        for (int h = 0; h < EPV; h += 4) {
          if (n > kCut) n = c.cut(n, a.k);
          offer(q, h, h + 4);
          __syncthreads();
          n = count;
          __syncthreads();
        }
    }
    if (n > kCut) n = c.cut(n, a.k);
  }
  __syncthreads();
  const int n = count;
  float m2 = kNegInf, s2 = 0.f;
  block_merge2<BLOCK>(m, s, m2, s2, lds);
  sort_falling(key, n);
  if (a.parts == 1) {
    write_entries(a, row, key);
    if (tid == 0) write_lse(a, row, m, s);
  } else {
    uint64_t* out = a.part_key + (row * a.parts + part) * a.k;
    for (int i = tid; i < a.k; i += BLOCK) out[i] = i < n ? key[i] : 0;
    if (tid == 0) a.part_ms[row * a.parts + part] = make_float2(m, s);
  }
}

__global__ void __launch_bounds__(kBlock) top_merge_kernel(TopArgs a) {
  __shared__ uint64_t key[kCap];
  __shared__ int count;
  const int tid = threadIdx.x;
  const int64_t row = a.row0 + blockIdx.x;
  const uint64_t* in = a.part_key + row * a.parts * a.k;
  const int total = a.parts * a.k;
  Candidates c{key, &count, 0, kNegInf};
  if (tid == 0) count = 0;
  __syncthreads();
  int n = 0;
  for (int base = 0; base < total; base += kBlock) {
    if (n > kCap - kBlock) n = c.cut(n, a.k);
    const uint64_t k = base + tid < total ? in[base + tid] : 0;
    c.add(k > c.least, k);
    __syncthreads();
    n = count;
    __syncthreads();
  }
  sort_falling(key, n);
  write_entries(a, row, key);
  if (tid < 64) {
    float m = kNegInf, s = 0.f;
    for (int p = tid; p < a.parts; p += 64) {
      const float2 v = a.part_ms[row * a.parts + p];
      const float M = fmaxf(m, v.x);
      s = ms_rescale(s, m, M) + ms_rescale(v.y, v.x, M);
      m = M;
    }
    lanes_merge<64>(m, s);
    if (tid == 0) write_lse(a, row, m, s);
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

  // Workgroups per row: at least a batch each, and no more than it takes to fill the chip.
  const int64_t nv = a->vocab * dtype_bytes(a->logits_dtype) / 16;
  const int64_t batches = nv > 0 ? (nv + kBlock * kU - 1) / (kBlock * kU) : 1;
  int64_t parts = (2048 + a->n_rows - 1) / a->n_rows;
  if (parts > batches) parts = batches;
  const int64_t per_batches = (batches + parts - 1) / parts;
  parts = (batches + per_batches - 1) / per_batches;
  const size_t keys = parts > 1 ? sizeof(uint64_t) * static_cast<size_t>(a->n_rows) * parts * a->k : 0;
  const size_t ms = parts > 1 ? sizeof(float2) * static_cast<size_t>(a->n_rows) * parts : 0;
  const int rc = ensure_scratch_on(ctx, keys + ms, st);
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
  t.part_ms = reinterpret_cast<float2*>(static_cast<char*>(ctx->scratch) + keys);
  t.err = ctx->d_page->err;
  t.k2 = k2;
  t.k = a->k;
  t.ids_i64 = a->ids_dtype == PCP_I64;
  t.parts = static_cast<int32_t>(parts);
  t.per = static_cast<int32_t>(per_batches * kBlock * kU);
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
