// Verification of drafted tokens (pcp_verify_drafts, pcp_sample.h).
//
// Whether a token is accepted and which one follows are comparisons of sums over the
// vocabulary with given numbers, so everything is formed in 64 bits: a row's terms are
// e = 2^((x - max) k), k = log2(e) / temperature.
//   rows:     token i's target and draft row in parts, (max, sum e) of each
//   decide:   merges a sequence's parts and decides its tokens
//   residual: sums of max(p - q, 0) over the parts of the row where the sequence ends
//   pick:     the part, then the element, where the running sum passes the draw
// A large call takes the first tokens' rows, decides them, and leaves out the rows of sequences
// that have ended there. Greedy calls: the rows' first maxima in parts, then one workgroup per
// sequence.
//
// Bound by f64 arithmetic in the rows (16 operations an element) and, with few rows, by the
// chain of dependent loads from a decision to a token. 64 sequences of 8 drafted tokens over
// 151,936 bf16 logits: rows 82, decide 2 x 4.8, residual 18, pick 11 us (rows in one launch 109;
// with the 11-point polynomial alone 150). One sequence of 4: rows 4.5, decide 3.9, residual
// with pick 12.5.
// Deciding in each token's last workgroup, by a ticket, instead of in launches between: the
// tickets cost 28 us for 4,368 workgroups, 50 for 12,000.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstdint>
#include <cstring>

#include "context.hpp"
#include "grpo_device.hpp"
#include "pcp_sample.h"

namespace pcp {
namespace {

constexpr int kBlock = 256;
constexpr int kU = 4;                       // 16-byte vectors per lane of a part
constexpr int kPartVecs = kBlock * kU;      // 16 KB
// The same of the residual's parts: U vectors per lane, 1 where the last workgroup picks along.
constexpr int end_vecs(int U) { return kBlock * U; }
constexpr int kNW = kBlock / 64;

// A part of a row.
struct RowState {
  double sum;   // with the terms' ref (see scale64); greedy: unused
  float max;
  int32_t at;   // greedy: the first maximum's index; sampling: its log-sum-exp is not finite
};

// Token i of a sequence, and its rows.
struct Decision {
  double sum_p, sum_q;   // sum e of the target row, of the draft row, with the terms' ref (see scale64)
  float max_p, max_q;
  float logp;            // of the drafted token
  int32_t flags;
};
constexpr int kAccepted = 1, kInRange = 2, kBadP = 4, kBadQ = 8;

// Where a sequence ends: the row its last token comes from.
struct SeqEnd {
  double scale_p, scale_q;   // 1 / sum e of the target row, of the draft row (0: q is 0)
  float max_p, max_q;
  double log_p;              // log of the target row's sum
  int32_t j;                 // accepted tokens
  int32_t without;           // a lookup's refused token (r is 0 there), or -1
};

// With a kernel's own argument within three cache lines: a fourth, which holds that argument, took the
// decision's kernel from 4.8 to 5.1 us.
struct VerifyArgs {
  const void* target;
  const void* draft;          // nullptr: all of q on the drafted token
  const int64_t* ids;
  const int32_t* lens;
  const float* uniforms;
  int64_t* tokens;
  int32_t* accepted;
  float* logp;
  RowState* part;             // [S, n + 1, 2, parts]; greedy [S, n + 1, parts]
  Decision* decision;         // [S, n + 1]
  double* seg;                // [S, end_parts + 2]: residual sums of head, parts, tail
  int* ended;                 // [S]: one of the first tokens was refused
  unsigned* done;             // [S]: workgroups done with a sequence's residual; zero between calls
  int* err;
  int64_t vocab, tstride, dstride, tseq, dseq;   // elements: between rows, between sequences
  double k;                   // log2(e) / temperature
  float plain;                // see scale64
  int32_t n;
  int32_t parts, end_parts;   // of kPartVecs, end_vecs vectors
  int32_t from;               // the first token of this launch
};
static_assert(sizeof(VerifyArgs) + sizeof(int) <= 192, "");

// 2^y for y <= 0 (0 below 2^-1075, NaN kept): 2^n times a polynomial in y - n that meets 2^f in the
// 11 Chebyshev points of [-1/2, 1/2]. Relative error 4.0e-16 at most of 40,000 arguments, against 60
// digits (with 9 points 1e-12, which over 151,936 tokens would decide some draws).
__device__ __forceinline__ double exp2_64(double y) {
  y = y < -1100. ? -1100. : y;
  const double n = __builtin_rint(y), f = y - n;
  double p = 7.072578846877522e-09;
  p = fma(p, f, 1.0208690285818614e-07);
  p = fma(p, f, 1.3215442633591105e-06);
  p = fma(p, f, 1.5252657260154878e-05);
  p = fma(p, f, 0.00015403530441632557);
  p = fma(p, f, 0.001333355823016538);
  p = fma(p, f, 0.009618129107606982);
  p = fma(p, f, 0.055504108664447716);
  p = fma(p, f, 0.24022650695910097);
  p = fma(p, f, 0.69314718055995);
  p = fma(p, f, 1.0);
  return __builtin_amdgcn_ldexp(p, static_cast<int>(n));
}

// The same for many terms: 2^y with y = Y / 128 as 2^(j/128), from a table in LDS, times a
// polynomial in Y - rint(Y) through 5 Chebyshev points, times 2^e: 16 operations an element instead
// of 27. The polynomial is within 7.6e-17 of 2^f, the table's entries within 3.4e-16, the whole
// within 5.4e-16 at most of 40,000 arguments. (With 16 to 64
// entries and a longer polynomial the rows take 3 to 7 us more of 82: the lookups hide under the
// arithmetic.)
constexpr int kTable = 128;
__device__ __forceinline__ void fill_table(double* table) {
  if (threadIdx.x < kTable) table[threadIdx.x] = exp2_64(threadIdx.x * (1. / kTable));
}
struct Exp2 {
  double head, poly;   // 2^(j/128), 2^(f/128)
  int n;
  __device__ __forceinline__ Exp2(double Y, const double* table) {
    constexpr double kMagic = 6755399441055744.;   // 1.5 2^52: the sum's low word is rint(Y)
    const double t = Y + kMagic, f = Y - (t - kMagic);
    n = static_cast<int>(static_cast<uint32_t>(__builtin_bit_cast(uint64_t, t)));
    head = table[n & (kTable - 1)];
    double p = 3.583033772988275e-11;
    p = fma(p, f, 2.6466433571126926e-08);
    p = fma(p, f, 1.4662262387638751e-05);
    p = fma(p, f, 0.0054152123481238145);
    poly = fma(p, f, 1.);
  }
  // sum + 2^y, y >= -1000: the exponent goes into the table's value. (What lies below adds nothing
  // to a sum that holds a 1.)
  __device__ __forceinline__ double add_to(double sum) const {
    const uint64_t h = __builtin_bit_cast(uint64_t, head);
    const uint32_t hi = static_cast<uint32_t>(h >> 32) + (static_cast<uint32_t>(n & ~(kTable - 1)) << 13);
    return fma(__builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | static_cast<uint32_t>(h)), poly, sum);
  }
  // 2^y, subnormal or 0 from -1022 down.
  __device__ __forceinline__ double value() const { return __builtin_amdgcn_ldexp(head * poly, n >> 7); }
};
static_assert(kTable == 1 << 7, "");

// Terms 2^((x - max) k) of Exp2 as 2^(fma(x, k', -ref) / 128), one instruction. Below |max| =
// a.plain ref is the rounded product with k' = 128 k, below 2^42 and so off by at most 2^-12 (a row
// all at a mask such as -1e30 would otherwise have a product off by 2^50, and anything for a term);
// where sums of different ref meet, adj() takes that out. From there on two f32 logits that differ
// at all lie 2^2048 apart, whatever k' is from 128 k up: it is the next power of two, and the product
// exact.
struct Scale64 {
  double k, ref;
};
__device__ __forceinline__ Scale64 scale64(const VerifyArgs& a, float max) {
  const float m = ms_ref(max);
  double k = a.k * kTable;
  if (!(fabsf(m) < a.plain)) k = __builtin_amdgcn_ldexp(1., __builtin_amdgcn_frexp_exp(k));   // also +inf
  return Scale64{k, m * k};
}
__device__ __forceinline__ double adj(const VerifyArgs& a, float max) {
  const double m = max, k = a.k * kTable;
  return fabsf(max) < a.plain ? fma(fma(m, k, -(m * k)), -0.69314718055994530942 / kTable, 1.) : 1.;
}

template <typename TI>
__device__ __forceinline__ const char* target_row(const VerifyArgs& a, int64_t s, int i) {
  return static_cast<const char*>(a.target) + (s * a.tseq + i * a.tstride) * TI::kBytes;
}
template <typename TI>
__device__ __forceinline__ const char* draft_row(const VerifyArgs& a, int64_t s, int i) {
  return static_cast<const char*>(a.draft) + (s * a.dseq + i * a.dstride) * TI::kBytes;
}

__device__ __forceinline__ int draft_len(const VerifyArgs& a, int64_t s) {
  return a.lens ? min(max(a.lens[s], 0), a.n) : a.n;
}

// Workgroup sum of v in a fixed order, on every thread. lds: one double per wave.
template <int BLOCK>
__device__ __forceinline__ double block_sum64(double v, double* lds) {
  v = wave_sum64(v);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = lds[0];
#pragma unroll
  for (int w = 1; w < BLOCK / 64; ++w) v += lds[w];
  __syncthreads();
  return v;
}

// The larger value, of equals the smaller index; NaN and -inf never win over index INT32_MAX.
__device__ __forceinline__ void better32(float& v, int& i, float v2, int i2) {
  if (v2 > v || (v2 == v && i2 < i)) {
    v = v2;
    i = i2;
  }
}

// ---- greedy ----------------------------------------------------------------------------
template <typename TI>
__global__ void __launch_bounds__(kBlock) verify_first_max_kernel(VerifyArgs a) {
  constexpr int EPV = 16 / TI::kBytes, U = kU, BLOCK = kBlock;
  __shared__ float wmax[kNW];
  __shared__ int wat[kNW];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, part = blockIdx.x, i = blockIdx.z;
  const int64_t s = blockIdx.y;
  if (i > draft_len(a, s)) return;   // rows of tokens that were not drafted
  const char* row = target_row<TI>(a, s, i);
  const RowSpan sp = row_span<TI>(row, a.vocab);
  const int v0 = part * kPartVecs;
  const __amdgpu_buffer_rsrc_t buf = row_rsrc(sp.vec, static_cast<uint32_t>(sp.nv) * 16u);
  u32x4 x[U];
#pragma unroll
  for (int q = 0; q < U; ++q) x[q] = buf_ld16<false>(buf, static_cast<uint32_t>(v0 + q * BLOCK + tid) * 16u);
  const int ek = part == 0 ? edge_index<TI>(sp, tid) : -1;
  const float xe = ek >= 0 ? TI::load1(row, ek) : kNegInf;
  float best = kNegInf;
  int slot = -1;   // a lane's elements come by rising index: the first of equals stays
#pragma unroll
  for (int q = 0; q < U; ++q)
    if (v0 + q * BLOCK + tid < sp.nv)
#pragma unroll
      for (int j = 0; j < EPV; ++j) {
        const float v = TI::unpack(reinterpret_cast<const uint32_t*>(&x[q]), j);
        if (v > best) {
          best = v;
          slot = q * EPV + j;
        }
      }
  int at = slot < 0 ? INT32_MAX : sp.head + (v0 + slot / EPV * BLOCK + tid) * EPV + slot % EPV;
  if (xe > kNegInf) better32(best, at, xe, ek);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) better32(best, at, __shfl_xor(best, o), __shfl_xor(at, o));
  if (lane == 0) {
    wmax[wave] = best;
    wat[wave] = at;
  }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kNW; ++w) better32(best, at, wmax[w], wat[w]);
    a.part[(s * (a.n + 1) + i) * a.parts + part] = RowState{0., best, at};
  }
}

constexpr int kGreedyBlock = 512;

__global__ void __launch_bounds__(kGreedyBlock) verify_greedy_kernel(VerifyArgs a) {
  __shared__ int row_at[PCP_VERIFY_MAX_DRAFT + 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t s = blockIdx.x;
  const int len = draft_len(a, s);
  for (int i = wave; i <= len; i += kGreedyBlock / 64) {
    const RowState* p = a.part + (s * (a.n + 1) + i) * a.parts;
    float m = kNegInf;
    int at = INT32_MAX;
    for (int q = lane; q < a.parts; q += 64) better32(m, at, p[q].max, p[q].at);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) better32(m, at, __shfl_xor(m, o), __shfl_xor(at, o));
    if (lane == 0) row_at[i] = at == INT32_MAX ? 0 : at;
  }
  __syncthreads();
  if (wave != 0) return;
  if (lane == 0 && a.lens && (a.lens[s] < 0 || a.lens[s] > a.n)) raise_error(a.err, kErrDraftLen);
  // Lane i decides token i (n <= 64).
  const int64_t d = lane < len ? a.ids[s * a.n + lane] : 0;
  const uint64_t no = ~__ballot(lane < len && d == row_at[lane]);
  const int j = min(no ? __builtin_ctzll(no) : 64, len);
  if (lane == j && lane < len && !(d >= 0 && d < a.vocab)) raise_error(a.err, kErrTokenRange);
  if (lane == 0) a.accepted[s] = j;
  // Entries 0 .. n (65 at most): the accepted tokens, the one after, then the pad.
  for (int i = lane; i <= a.n; i += 64) {
    a.tokens[s * (a.n + 1) + i] = i < j ? d : i == j ? row_at[j] : PCP_IGNORE_INDEX;
    if (a.logp) a.logp[s * (a.n + 1) + i] = 0.f;
  }
}

// ---- rows ------------------------------------------------------------------------------
template <typename TI>
__global__ void __launch_bounds__(kBlock) verify_rows_kernel(VerifyArgs a, int rows) {
  constexpr int EPV = 16 / TI::kBytes, U = kU, BLOCK = kBlock;
  __shared__ double table[kTable];
  __shared__ double lds[kNW];
  __shared__ float wmax[kNW];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, part = blockIdx.x;
  const bool is_draft = static_cast<int>(blockIdx.z) >= rows;   // rows target rows, then their draft rows
  const int i = a.from + blockIdx.z - (is_draft ? rows : 0);
  const int64_t s = blockIdx.y, token = s * (a.n + 1) + i;
  if (i + is_draft > draft_len(a, s)) return;   // rows of tokens that were not drafted
  if (a.from > 0 && a.ended[s]) return;
  const int v0 = part * kPartVecs;
  const char* row = is_draft ? draft_row<TI>(a, s, i) : target_row<TI>(a, s, i);
  const RowSpan sp = row_span<TI>(row, a.vocab);
  const __amdgpu_buffer_rsrc_t buf = row_rsrc(sp.vec, static_cast<uint32_t>(sp.nv) * 16u);
  u32x4 x[U];
#pragma unroll
  for (int q = 0; q < U; ++q) x[q] = buf_ld16<false>(buf, static_cast<uint32_t>(v0 + q * BLOCK + tid) * 16u);
  const int ek = part == 0 ? edge_index<TI>(sp, tid) : -1;
  const float xe = ek >= 0 ? TI::load1(row, ek) : kNegInf;
  auto held = [&](int q) { return v0 + q * BLOCK + tid < sp.nv; };
  fill_table(table);
  float m = xe;   // maximum: NaN where either is
#pragma unroll
  for (int q = 0; q < U; ++q)
    if (held(q))
#pragma unroll
      for (int j = 0; j < EPV; ++j)
        m = __builtin_elementwise_maximum(m, TI::unpack(reinterpret_cast<const uint32_t*>(&x[q]), j));
  bool nan = __any(m != m);
  m = lanes_max<64>(m);
  if (lane == 0) wmax[wave] = nan ? __builtin_nanf("") : m;
  __syncthreads();
  nan = false;
#pragma unroll
  for (int w = 0; w < kNW; ++w) {
    m = fmaxf(m, wmax[w]);
    nan |= wmax[w] != wmax[w];
  }
  const Scale64 at = scale64(a, m);
  auto term = [&](float v, double sum) {
    return Exp2(fmax(fma(static_cast<double>(v), at.k, -at.ref), -1000. * kTable), table).add_to(sum);
  };
  double sum = ek >= 0 ? term(xe, 0.) : 0.;
#pragma unroll
  for (int q = 0; q < U; ++q)
    if (held(q))
#pragma unroll
      for (int j = 0; j < EPV; ++j) sum = term(TI::unpack(reinterpret_cast<const uint32_t*>(&x[q]), j), sum);
  sum = block_sum64<BLOCK>(sum, lds);
  if (tid == 0) a.part[(token * 2 + is_draft) * a.parts + part] = RowState{sum, m, nan};
}

// ---- decide ----------------------------------------------------------------------------
constexpr int kDecideBlock = 512;

// The tokens from a.from to before `to`.
template <typename TI>
__global__ void __launch_bounds__(kDecideBlock) verify_decide_kernel(VerifyArgs a, int to) {
  __shared__ RowState whole[2 * (PCP_VERIFY_MAX_DRAFT + 1)];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t s = blockIdx.x;
  const int len = draft_len(a, s), n = min(to, len + 1) - a.from;
  if (a.from > 0 && a.ended[s]) return;
  for (int i = wave; i < 2 * n; i += kDecideBlock / 64) {
    if ((i & 1) && !(a.draft && a.from + (i >> 1) < len)) continue;
    const RowState* p = a.part + ((s * (a.n + 1) + a.from) * 2 + i) * a.parts;
    float mm = kNegInf;
    int bad = 0;
    for (int q = lane; q < a.parts; q += 64) {
      mm = fmaxf(mm, p[q].max);
      bad |= p[q].at;
    }
    mm = lanes_max<64>(mm);
    double sum = 0.;
    for (int q = lane; q < a.parts; q += 64)
      if (p[q].max > kNegInf)
        sum += p[q].sum * adj(a, p[q].max) *
               exp2_64((static_cast<double>(p[q].max) - static_cast<double>(mm)) * a.k);
    sum = wave_sum64(sum);
    bad = __any(bad != 0) || !(__builtin_isfinite(mm) && __builtin_isfinite(sum));
    if (lane == 0) whole[i] = RowState{sum, mm, bad};
  }
  __syncthreads();
  bool refused = false;
  if (tid < n) {   // at most 65
    const int i = a.from + tid;
    const int64_t token = s * (a.n + 1) + i;
    const bool drafted = i < len, model = drafted && a.draft;
    const RowState p = whole[2 * tid], q = model ? whole[2 * tid + 1] : RowState{1., 0.f, 0};
    const int64_t d = drafted ? a.ids[s * a.n + i] : 0;
    const bool in = d >= 0 && d < a.vocab;
    Decision o{p.sum * (2. - adj(a, p.max)), q.sum * (2. - adj(a, q.max)), p.max, q.max, 0.f,   // 1 / adj
               (in ? kInRange : 0) | (p.at ? kBadP : 0) | (q.at ? kBadQ : 0)};
    if (drafted && in && !p.at && !q.at) {
      const double y = (static_cast<double>(TI::load1(target_row<TI>(a, s, i), d)) - p.max) * a.k;
      double qd = 1.;
      if (model) qd = exp2_64((static_cast<double>(TI::load1(draft_row<TI>(a, s, i), d)) - q.max) * a.k) / q.sum;
      if (static_cast<double>(a.uniforms[token]) * qd < exp2_64(y) / p.sum) o.flags |= kAccepted;
      o.logp = static_cast<float>(y * 0.69314718055994530942 - log(p.sum));
    }
    a.decision[token] = o;
    refused = drafted && !(o.flags & kAccepted);
  }
  if (to <= a.n) {
    const int any = __syncthreads_or(refused);
    if (tid == 0) a.ended[s] = any;
  }
}

// ---- the sequence's end ----------------------------------------------------------------
// r of one element: max(p - q, 0), p alone where scale_q is 0.
struct Residual {
  Scale64 p, q;
  double scale_p, scale_q;  // 1 / sum e
  int without;
  bool plain;   // p alone: nothing of p lies above q
  const double* table;
  __device__ __forceinline__ double prob(float x, const Scale64& at, double scale) const {
    // Exactly 0 from 2^-1100 down; an element that has any mass can be drawn.
    const double v = Exp2(fmax(fma(static_cast<double>(x), at.k, -at.ref), -1100. * kTable), table).value();
    return v * scale;
  }
  __device__ __forceinline__ double operator()(float x, float y, int id) const {
    const double v = prob(x, p, scale_p);
    if (plain) return v;
    if (scale_q != 0.) return fmax(v - prob(y, q, scale_q), 0.);
    return id == without ? 0. : v;
  }
};

__device__ __forceinline__ Residual residual(const VerifyArgs& a, const SeqEnd& e, bool plain, const double* table) {
  return Residual{scale64(a, e.max_p), scale64(a, e.max_q), e.scale_p, e.scale_q, e.without, plain, table};
}

// The elements of a part: both rows' values, in element order per (chunk, lane, element). The
// draft row may start at another offset of its 16 bytes, so it is read element by element there.
template <typename TI, int U, typename F>
__device__ __forceinline__ void part_elements(const VerifyArgs& a, const SeqEnd& e, int64_t s, const RowSpan& sp, int v0,
                                              F f) {
  constexpr int EPV = 16 / TI::kBytes, BLOCK = kBlock;
  const int tid = threadIdx.x;
  const bool model = e.scale_q != 0.;
  const __amdgpu_buffer_rsrc_t buf = row_rsrc(sp.vec, static_cast<uint32_t>(sp.nv) * 16u);
  const char* drow = model ? draft_row<TI>(a, s, e.j) + sp.head * TI::kBytes : nullptr;
  const bool same = model && (reinterpret_cast<uintptr_t>(drow) & 15u) == 0;
  const __amdgpu_buffer_rsrc_t qbuf = row_rsrc(same ? drow : static_cast<const char*>(sp.vec),
                                               same ? static_cast<uint32_t>(sp.nv) * 16u : 0u);
  u32x4 x[U], y[U];
#pragma unroll
  for (int q = 0; q < U; ++q) {
    const uint32_t off = static_cast<uint32_t>(v0 + q * BLOCK + tid) * 16u;
    x[q] = buf_ld16<false>(buf, off);
    y[q] = buf_ld16<false>(qbuf, off);
  }
#pragma unroll
  for (int q = 0; q < U; ++q) {
    const int v = v0 + q * BLOCK + tid;
    const bool held = v < sp.nv;
#pragma unroll
    for (int j = 0; j < EPV; ++j) {
      float yv = TI::unpack(reinterpret_cast<const uint32_t*>(&y[q]), j);
      if (model && !same && held) yv = TI::load1(drow, static_cast<int64_t>(v) * EPV + j);
      f(q, j, held, TI::unpack(reinterpret_cast<const uint32_t*>(&x[q]), j), yv, sp.head + v * EPV + j);
    }
  }
}

// The token after the accepted ones, by the whole workgroup.
template <typename TI, int U>
__device__ __forceinline__ void pick_token(const VerifyArgs& a, const SeqEnd& e, int64_t s, const char* row,
                                           const RowSpan& sp, const double* table) {
  constexpr int EPV = 16 / TI::kBytes;
  __shared__ double chunk_sum[U][kNW];
  __shared__ int first;       // the smallest element whose running sum passes
  __shared__ int last;        // the largest element with r > 0, where rounding leaves none
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const char* drow = e.scale_q != 0. ? draft_row<TI>(a, s, e.j) : nullptr;
  const double u = static_cast<double>(a.uniforms[s * (a.n + 1) + a.n]);
  const int segs = a.end_parts + 2;
  const double* seg = a.seg + s * segs;
  // Each wave: the total, then the first segment whose running sum passes u * total.
  double total = 0.;
  for (int b = 0; b < segs; b += 64) total += wave_sum64(b + lane < segs ? seg[b + lane] : 0.);
  // Nothing of p above q (equal rows): the token comes from p, whose sums are not in seg; the
  // whole row is then one segment, scanned part by part.
  const bool plain = !(total > 0.);
  const Residual r = residual(a, e, plain, table);
  const double t = u * (plain ? 1. : total);
  int hit = -1, last_seg = -1;
  double before = 0.;
  if (!plain) {
    double run = 0.;
    for (int b = 0; b < segs && hit < 0; b += 64) {
      const double v = b + lane < segs ? seg[b + lane] : 0.;
      const double incl = run + wave_scan(v);
      const uint64_t over = __ballot(b + lane < segs && v > 0. && incl > t);
      const uint64_t some = __ballot(v > 0.);
      if (some) last_seg = b + 63 - __builtin_clzll(some);
      if (over) {
        const int l = __builtin_ctzll(over);
        hit = b + l;
        before = read_lane64(incl - v, l);
      }
      run = read_lane64(incl, 63);
    }
  }
  // Scans segment g from running sum `run`; true once an element passes. Every thread of the
  // workgroup takes part; run becomes the sum after the segment.
  auto scan = [&](int g, double& run) {
    if (tid == 0) {
      first = INT32_MAX;
      last = -1;
    }
    __syncthreads();
    if (g == 0 || g == a.end_parts + 1) {   // the head or the tail: at most 7 elements, each thread alone
      const int n0 = g == 0 ? 0 : sp.head + sp.nv * EPV, n1 = g == 0 ? sp.head : static_cast<int>(a.vocab);
      for (int i = n0; i < n1; ++i) {
        const double v = r(TI::load1(row, i), drow ? TI::load1(drow, i) : 0.f, i);
        run += v;
        if (tid == 0 && v > 0.) {
          last = i;
          if (run > t && first == INT32_MAX) first = i;
        }
      }
    } else {
      double part_sum[U];
      double mine[U][EPV];
#pragma unroll
      for (int q = 0; q < U; ++q) part_sum[q] = 0.;
      part_elements<TI, U>(a, e, s, sp, (g - 1) * end_vecs(U), [&](int q, int j, bool held, float x, float y, int id) {
        mine[q][j] = held ? r(x, y, id) : 0.;
        part_sum[q] += mine[q][j];
      });
      double incl[U];
#pragma unroll
      for (int q = 0; q < U; ++q) {
        incl[q] = wave_scan(part_sum[q]);
        if (lane == 63) chunk_sum[q][wave] = incl[q];
      }
      __syncthreads();
      double base = run;
      int seen = INT32_MAX, most = -1;
#pragma unroll
      for (int q = 0; q < U; ++q) {
        double b = base;
        for (int w = 0; w < kNW; ++w) {
          if (w < wave) b += chunk_sum[q][w];
          base += chunk_sum[q][w];
        }
        double c = b + (incl[q] - part_sum[q]);
#pragma unroll
        for (int j = 0; j < EPV; ++j) {
          c += mine[q][j];
          const int id = sp.head + ((g - 1) * end_vecs(U) + q * kBlock + tid) * EPV + j;
          if (mine[q][j] > 0.) {
            most = max(most, id);
            if (c > t) seen = min(seen, id);
          }
        }
      }
      run = base;
      if (seen != INT32_MAX) atomicMin(&first, seen);
      if (most >= 0) atomicMax(&last, most);
    }
    __syncthreads();
    return first != INT32_MAX;
  };
  // The segment where the sum passes (rounding past the last one: its last element); plain, one
  // after the other.
  int pick = -1;
  double run = before;
  const int end = plain ? segs : hit >= 0 ? hit + 1 : last_seg + 1;
  for (int g = plain ? 0 : end - 1; g < end; ++g) {
    const bool found = scan(g, run);
    if (last >= 0) pick = found ? first : last;
    __syncthreads();   // first / last read before the next segment resets them
    if (found) break;
  }
  if (tid == 0) {
    if (pick < 0) pick = static_cast<int>(a.vocab) - 1;
    const int64_t at = s * (a.n + 1) + e.j;
    a.tokens[at] = pick;
    const double below = static_cast<double>(TI::load1(row, pick)) - e.max_p;
    if (a.logp) a.logp[at] = static_cast<float>(below * a.k * 0.69314718055994530942 - e.log_p);
  }
}

// The end of sequence s, by each wave: false where the row of its last token is bad.
__device__ __forceinline__ bool seq_end(const VerifyArgs& a, int64_t s, SeqEnd& e) {
  const int lane = threadIdx.x & 63;
  const Decision* dec = a.decision + s * (a.n + 1);
  // Lane i has token i, in one load beside the length's (n <= 64). What lies after a refusal may be of
  // another call.
  const Decision mine = dec[min(lane, a.n)];
  const int len = draft_len(a, s);
  const uint64_t no = ~__ballot(lane < len && (mine.flags & kAccepted));
  const int j = min(no ? __builtin_ctzll(no) : 64, len);
  Decision at;
  if (j < 64) {
    at = Decision{read_lane64(mine.sum_p, j), read_lane64(mine.sum_q, j), read_lane(mine.max_p, j),
                  read_lane(mine.max_q, j), 0.f, __builtin_amdgcn_readlane(mine.flags, j)};
  } else {
    at = dec[j];
  }
  const bool refused = j < len, in = at.flags & kInRange;
  const bool model = refused && a.draft && in && !(at.flags & kBadQ);
  e.j = j;
  e.max_p = at.max_p;
  e.scale_p = 1. / at.sum_p;
  e.log_p = log(at.sum_p * adj(a, at.max_p));
  e.max_q = model ? at.max_q : 0.f;
  e.scale_q = model ? 1. / at.sum_q : 0.;
  e.without = refused && !a.draft && in ? static_cast<int32_t>(a.ids[s * a.n + j]) : -1;
  return !(at.flags & kBadP);
}

// The workgroup's count is full: this call comes from its last, and the count is 0 again.
__device__ __forceinline__ bool last_of(unsigned* count, int n) {
  return atomicInc(count, static_cast<unsigned>(n - 1)) == static_cast<unsigned>(n - 1);
}

// PICK: the sequence's last workgroup picks the token.
template <typename TI, int U, bool PICK>
__device__ __forceinline__ void residual_part(const VerifyArgs& a) {
  __shared__ double table[kTable];
  __shared__ double lds[kNW];
  __shared__ int last;
  const int tid = threadIdx.x, lane = tid & 63, part = blockIdx.x;
  const int64_t s = blockIdx.y;
  fill_table(table);
  SeqEnd e;
  const bool good = seq_end(a, s, e);
  if (part == 0 && tid < 64) {
    const Decision* dec = a.decision + s * (a.n + 1);
    int64_t* tok = a.tokens + s * (a.n + 1);
    float* logp = a.logp ? a.logp + s * (a.n + 1) : nullptr;
    // Entries 0 .. n (65 at most): the accepted tokens, the one after (V - 1 where its row is
    // bad; else pick_token's), then the pad.
    for (int i = lane; i <= a.n; i += 64)
      if (i != e.j || !good) {
        tok[i] = i < e.j ? a.ids[s * a.n + i] : i == e.j ? a.vocab - 1 : PCP_IGNORE_INDEX;
        if (logp) logp[i] = i < e.j ? dec[i].logp : 0.f;
      }
    if (lane == 0) {
      const bool refused = e.j < draft_len(a, s);
      a.accepted[s] = e.j;
      if (a.lens && (a.lens[s] < 0 || a.lens[s] > a.n)) raise_error(a.err, kErrDraftLen);
      if (refused && !(dec[e.j].flags & kInRange)) raise_error(a.err, kErrTokenRange);
      if (!good || (refused && (dec[e.j].flags & kBadQ))) raise_error(a.err, kErrNonFinite);
    }
  }
  if (!good) return;
  const char* row = target_row<TI>(a, s, e.j);
  const RowSpan sp = row_span<TI>(row, a.vocab);
  const Residual r = residual(a, e, false, table);
  double* seg = a.seg + s * (a.end_parts + 2);
  __syncthreads();   // the table
  if (part == 0 && tid < 64) {
    const int ek = edge_index<TI>(sp, tid);
    double v = 0.;
    if (ek >= 0) v = r(TI::load1(row, ek), e.scale_q != 0. ? TI::load1(draft_row<TI>(a, s, e.j), ek) : 0.f, ek);
    const double head = wave_sum64(tid < sp.head ? v : 0.), tail = wave_sum64(tid >= sp.head ? v : 0.);
    if (tid == 0) {
      store_coherent(seg, head);
      store_coherent(seg + a.end_parts + 1, tail);
    }
  }
  double sum = 0.;
  part_elements<TI, U>(a, e, s, sp, part * end_vecs(U), [&](int, int, bool held, float x, float y, int id) {
    if (held) sum += r(x, y, id);
  });
  sum = block_sum64<kBlock>(sum, lds);
  if (tid == 0) store_coherent(seg + 1 + part, sum);
  if constexpr (PICK) {
    if (tid == 0) {
      wait_stores();
      last = last_of(a.done + s, a.end_parts);
    }
    __syncthreads();
    if (!last) return;
    acquire_coherent();
    pick_token<TI, U>(a, e, s, row, sp, table);
  }
}

// Scalar registers come in sixteens, of 800 a SIMD, and sixteen more of a wave's are the trap handler's: past
// 80 a CU holds 7 workgroups, not 8, and 1,976 of them take 12.7 us instead of 11.5.
template <typename TI>
__global__ void __launch_bounds__(kBlock) __attribute__((amdgpu_num_sgpr(80))) verify_residual_kernel(VerifyArgs a) {
  residual_part<TI, 2, false>(a);
}
// Few workgroups: with the same limit one sequence takes 21.5 us instead of 20.5.
template <typename TI>
__global__ void __launch_bounds__(kBlock) verify_residual_pick_kernel(VerifyArgs a) {
  residual_part<TI, 1, true>(a);
}

template <typename TI, int U>
__global__ void __launch_bounds__(kBlock) verify_pick_kernel(VerifyArgs a) {
  __shared__ double table[kTable];
  fill_table(table);
  SeqEnd e;
  if (!seq_end(a, blockIdx.x, e)) return;
  const char* row = target_row<TI>(a, blockIdx.x, e.j);
  __syncthreads();   // the table
  pick_token<TI, U>(a, e, blockIdx.x, row, row_span<TI>(row, a.vocab), table);
}

// The residual's last workgroup picks the token along, by a ticket of each of its workgroups (4 KB of a
// row), where all sequences have at most so many, fewer where rows are narrow; else a launch of its
// own does. us for a whole call with 4 drafted tokens, along | by its own launch, by sequences:
//   bf16 151,936, looked up  1  20 | 23   2  22 | 24   4  25 | 26    6  28 | 27   12  37 | 31   64  94 | 61
//   bf16 151,936, a model    1  21 | 24   2  24 | 27   4  27 | 28    6  31 | 31   12  42 | 37   64 123 | 93
//   bf16  50,257, looked up  1  20 | 23   4  21 | 25   8  24 | 26   12  25 | 26   16  28 | 28   32  34 | 32
//   f32   50,257, a model    1  19 | 21   4  22 | 24   6  24 | 25    8  27 | 27   12  31 | 28   32  45 | 36
//   bf16  32,000, a model    1  20 | 24   4  21 | 26   8  24 | 27   16  28 | 29   24  32 | 31   32  34 | 32
//   f32    8,192, looked up  1  17 | 19   4  18 | 20   8  20 | 21   12  21 | 21   16  22 | 22   24  24 | 22
//   bf16   4,096, a model    1  19 | 22   8  20 | 25  32  22 | 26   64  25 | 27   80  26 | 27  128  31 | 28
//   bf16   1,000, a model    1  18 | 20   8  20 | 22  32  21 | 22   80  23 | 23  128  25 | 24  160  26 | 25
constexpr int64_t kPickAlongWorkgroups = 320, kPickAlongNarrow = 96, kNarrowParts = 16;
static_assert(kPickAlongWorkgroups / kNarrowParts <= kPickAlongNarrow, "a count per sequence");
// Rows in two launches from this many workgroups (16 KB of a row each) on: what it leaves out depends on
// how many sequences end in their first half. us for a whole call, two | one, by accepted tokens:
//   of 8, a model     10,336: 3.7  79 |  81   5.8  86 |  80   7.0  89 |  79   8  89 |  78
//                     17,408: 3.8 112 | 123   5.5 118 | 121   6.8 123 | 119   8 124 | 115
//                     20,672: 3.6 121 | 140   5.8 133 | 137   7.3 141 | 135   8 140 | 134
//   of 4, looked up    6,080: 0    47 |  61   0.9  59 |  61   2.4  66 |  61   4  72 |  61
//                     12,160: 0    68 | 100   1.0  83 |  99   2.3  97 | 100   4 109 |  99
// Drafts that are mostly accepted lose a tenth by it, those that are refused early gain more: 14,079
// workgroups of a model's draft with about half of the tokens accepted take 100 | 110, and looked-up
// tokens are refused more often than a model's.
constexpr int64_t kSplitWorkgroups = 8192;

bool picks_along(int64_t n_seq, int64_t nv) {
  const int64_t parts = std::max<int64_t>((nv + end_vecs(1) - 1) / end_vecs(1), 1);
  return n_seq * parts <= (parts < kNarrowParts ? kPickAlongNarrow : kPickAlongWorkgroups);
}

template <typename TI>
hipError_t launch_verify(VerifyArgs a, int64_t n_seq, bool greedy, bool along, hipStream_t st) {
  const unsigned ns = static_cast<unsigned>(n_seq), parts = static_cast<unsigned>(a.parts);
  const dim3 b(kBlock), seqs(ns);
  if (greedy) {
    verify_first_max_kernel<TI><<<dim3(parts, ns, static_cast<unsigned>(a.n + 1)), b, 0, st>>>(a);
    verify_greedy_kernel<<<seqs, dim3(kGreedyBlock), 0, st>>>(a);
    return hipGetLastError();
  }
  const int first = n_seq * (a.draft ? 2 * a.n + 1 : a.n + 1) * a.parts > kSplitWorkgroups ? (a.n + 1) / 2 : 0;
  for (int from = 0, to = first ? first : a.n + 1; from <= a.n; from = to, to = a.n + 1) {
    a.from = from;
    const unsigned rows = static_cast<unsigned>(to - from);
    verify_rows_kernel<TI><<<dim3(parts, ns, a.draft ? 2 * rows : rows), b, 0, st>>>(a, static_cast<int>(rows));
    verify_decide_kernel<TI><<<seqs, dim3(kDecideBlock), 0, st>>>(a, to);
  }
  const dim3 ends(static_cast<unsigned>(a.end_parts), ns);
  if (along) {
    verify_residual_pick_kernel<TI><<<ends, b, 0, st>>>(a);
  } else {
    verify_residual_kernel<TI><<<ends, b, 0, st>>>(a);
    verify_pick_kernel<TI, 2><<<seqs, b, 0, st>>>(a);
  }
  return hipGetLastError();
}

inline bool misaligned(const void* p, int size) {
  return (reinterpret_cast<uintptr_t>(p) & static_cast<uintptr_t>(size - 1)) != 0;
}
inline size_t round256(size_t b) { return (b + 255) & ~static_cast<size_t>(255); }

// The counts that verify_residual_pick_kernel leaves at zero, one per sequence: at most kPickAlongNarrow.
int ensure_verify_done(pcp_ctx* ctx, hipStream_t st) {
  if (ctx->verify_done) return PCP_OK;
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(st, &status) != hipSuccess) (void)hipGetLastError();
  else if (status != hipStreamCaptureStatusNone)
    return fail(ctx, PCP_ERR_INVALID_ARG, "the stream is being captured and the context's counters would have to be "
                                          "made: make one uncaptured call of the same sizes first");
  hipError_t e = hipMalloc(&ctx->verify_done, sizeof(unsigned) * kPickAlongNarrow);
  if (e != hipSuccess) {
    ctx->verify_done = nullptr;
    (void)hipGetLastError();
    return fail(ctx, PCP_ERR_OOM, "hipMalloc of the verification's counters failed");
  }
  if ((e = hipMemset(ctx->verify_done, 0, sizeof(unsigned) * kPickAlongNarrow)) != hipSuccess ||
      (e = hipDeviceSynchronize()) != hipSuccess) {
    (void)hipFree(ctx->verify_done);
    ctx->verify_done = nullptr;
    return hip_fail(ctx, e, "zeroing the verification's counters");
  }
  return PCP_OK;
}

int verify_drafts(pcp_ctx* ctx, const pcp_verify_args* a) {
  if (!a) return fail(ctx, PCP_ERR_INVALID_ARG, "args is NULL");
  if (a->n_seq < 0 || a->n_seq > PCP_SAMPLE_MAX_ROWS)
    return fail(ctx, PCP_ERR_INVALID_ARG, "n_seq must be in [0, %d] (got %lld)", PCP_SAMPLE_MAX_ROWS,
                (long long)a->n_seq);
  if (a->n_draft < 0 || a->n_draft > PCP_VERIFY_MAX_DRAFT)
    return fail(ctx, PCP_ERR_INVALID_ARG, "n_draft must be in [0, %d] (got %lld)", PCP_VERIFY_MAX_DRAFT,
                (long long)a->n_draft);
  if (a->vocab < 1 || a->vocab > PCP_SAMPLE_MAX_VOCAB)
    return fail(ctx, PCP_ERR_INVALID_ARG, "vocab must be in [1, %d] (got %lld)", PCP_SAMPLE_MAX_VOCAB,
                (long long)a->vocab);
  const int64_t ts = a->target_row_stride ? a->target_row_stride : a->vocab;
  const int64_t ds = a->draft_row_stride ? a->draft_row_stride : a->vocab;
  if (ts < a->vocab || ds < a->vocab) return fail(ctx, PCP_ERR_INVALID_ARG, "row strides must be >= vocab");
  int64_t tseq, dseq;
  if (mul_overflows(a->n_draft + 1, ts, &tseq) || mul_overflows(a->n_draft, ds, &dseq))
    return fail(ctx, PCP_ERR_OVERFLOW, "logits byte size overflows int64");
  if (a->target_seq_stride) tseq = a->target_seq_stride;
  if (a->draft_seq_stride) dseq = a->draft_seq_stride;
  if (tseq < a->vocab || (dseq < a->vocab && a->n_draft > 0))
    return fail(ctx, PCP_ERR_INVALID_ARG, "sequence strides must be >= vocab");
  // The bytes up to the last row's end, from above.
  auto too_far = [&](int64_t rows, int64_t row, int64_t seq) {
    int64_t in_seq, all, sum;
    return mul_overflows(rows, row, &in_seq) || mul_overflows(a->n_seq, seq, &all) ||
           __builtin_add_overflow(in_seq, all, &sum) || mul_overflows(sum, 4, &sum);
  };
  if (too_far(a->n_draft + 1, ts, tseq) || too_far(a->n_draft, ds, dseq))
    return fail(ctx, PCP_ERR_OVERFLOW, "logits byte size overflows int64");
  if (a->logits_dtype != PCP_BF16 && a->logits_dtype != PCP_F16 && a->logits_dtype != PCP_F32)
    return fail(ctx, PCP_ERR_DTYPE, "logits dtype must be bf16, f16 or f32 (got %d)", a->logits_dtype);
  if (!(a->temperature == a->temperature)) return fail(ctx, PCP_ERR_INVALID_ARG, "temperature is NaN");
  const bool greedy = a->temperature < 1e-6f;
  if (!greedy && !std::isfinite(a->temperature))
    return fail(ctx, PCP_ERR_INVALID_ARG, "temperature must be finite");
  if (a->flags & ~PCP_FLAG_ASYNC) return fail(ctx, PCP_ERR_INVALID_ARG, "only PCP_FLAG_ASYNC applies here");
  if (a->n_seq > 0) {
    if (!a->target_logits || !a->tokens || !a->accepted)
      return fail(ctx, PCP_ERR_INVALID_ARG, "target_logits / tokens / accepted is NULL");
    if (a->n_draft > 0 && !a->draft_ids) return fail(ctx, PCP_ERR_INVALID_ARG, "draft_ids is NULL");
    if (!greedy && !a->uniforms)
      return fail(ctx, PCP_ERR_INVALID_ARG, "uniforms is NULL and temperature is not below 1e-6");
  }
  const int size = dtype_bytes(a->logits_dtype);
  if (misaligned(a->target_logits, size) || misaligned(a->draft_logits, size) || misaligned(a->draft_ids, 8) ||
      misaligned(a->draft_lens, 4) || misaligned(a->uniforms, 4) || misaligned(a->tokens, 8) ||
      misaligned(a->accepted, 4) || misaligned(a->logp, 4))
    return fail(ctx, PCP_ERR_INVALID_ARG, "pointers must be aligned to their element size");
  if (!ctx) return fail(nullptr, PCP_ERR_INVALID_ARG, "context is NULL");
  if (a->n_seq == 0) return PCP_OK;
  const DeviceScope scope(ctx->device);
  if (scope.error() != hipSuccess) return hip_fail(ctx, scope.error(), "making the context's device current");
  hipStream_t st = static_cast<hipStream_t>(a->stream);

  const bool model = !greedy && a->draft_logits && a->n_draft > 0;
  const int64_t nv = a->vocab * size / 16;
  const int64_t parts = nv > 0 ? (nv + kPartVecs - 1) / kPartVecs : 1;
  const bool along = !greedy && picks_along(a->n_seq, nv);
  const int64_t ev = end_vecs(along ? 1 : 2), end_parts = nv > 0 ? (nv + ev - 1) / ev : 1;
  const size_t S = static_cast<size_t>(a->n_seq), tokens = S * static_cast<size_t>(a->n_draft + 1);
  const size_t o_dec = round256(sizeof(RowState) * tokens * (greedy ? 1 : 2) * parts);
  const size_t o_seg = o_dec + (greedy ? 0 : round256(sizeof(Decision) * tokens));
  const size_t o_ended = o_seg + (greedy ? 0 : round256(sizeof(double) * S * (end_parts + 2)));
  int rc = ensure_scratch_on(ctx, o_ended + (greedy ? 0 : sizeof(int) * S), st);
  if (rc == PCP_OK && along) rc = ensure_verify_done(ctx, st);
  if (rc != PCP_OK) return rc;
  char* sp = static_cast<char*>(ctx->scratch);

  VerifyArgs v;
  std::memset(&v, 0, sizeof(v));
  v.target = a->target_logits;
  v.draft = model ? a->draft_logits : nullptr;
  v.ids = a->draft_ids;
  v.lens = a->draft_lens;
  v.uniforms = a->uniforms;
  v.tokens = a->tokens;
  v.accepted = a->accepted;
  v.logp = a->logp;
  v.part = reinterpret_cast<RowState*>(sp);
  v.decision = reinterpret_cast<Decision*>(sp + o_dec);
  v.seg = reinterpret_cast<double*>(sp + o_seg);
  v.ended = reinterpret_cast<int*>(sp + o_ended);
  v.done = ctx->verify_done;
  v.err = ctx->d_page->err;
  v.vocab = a->vocab;
  v.tstride = ts;
  v.dstride = ds;
  v.tseq = tseq;
  v.dseq = dseq;
  v.k = 1.4426950408889634074 * (greedy ? 1. : 1. / static_cast<double>(a->temperature));
  const double plain = 0x1p42 / (v.k * kTable);
  v.plain = plain < static_cast<double>(FLT_MAX) ? static_cast<float>(plain) : HUGE_VALF;
  v.n = static_cast<int32_t>(a->n_draft);
  v.parts = static_cast<int32_t>(parts);
  v.end_parts = static_cast<int32_t>(end_parts);
  const bool timed = prof_begin(ctx, st);
  const hipError_t e = a->logits_dtype == PCP_F32    ? launch_verify<F32T>(v, a->n_seq, greedy, along, st)
                       : a->logits_dtype == PCP_BF16 ? launch_verify<BF16T>(v, a->n_seq, greedy, along, st)
                                                     : launch_verify<F16T>(v, a->n_seq, greedy, along, st);
  prof_end(ctx, st, timed);
  if (e != hipSuccess) return hip_fail(ctx, e, "draft verification launch");
  return finish_call(ctx, a->flags, st);
}

}  // namespace
}  // namespace pcp

using namespace pcp;

extern "C" void pcp_verify_args_init(pcp_verify_args* a) {
  if (!a) return;
  std::memset(a, 0, sizeof(*a));
  a->logits_dtype = PCP_BF16;
  a->temperature = 1.f;
}

extern "C" int pcp_verify_drafts(pcp_ctx* ctx, const pcp_verify_args* a) { return verify_drafts(ctx, a); }
