// Verification of drafted tokens (pcp_verify_drafts, pcp_sample.h).
//
// Whether a token is accepted and which one follows are comparisons of sums over the
// vocabulary with given numbers, so everything is formed in 64 bits: a row's terms are
// e = 2^((x - max) k), k = log2(e) / temperature, by a polynomial (exp2_64), and f64 multiply-adds run at the rate of f32 ones on this chip.
//   rows:     every target and draft row in parts, (max, sum e) of each
//   decide:   one workgroup per sequence merges its rows' parts and finds the first refusal
//   residual: sums of max(p - q, 0) over the parts of the row where the sequence ends
//   pick:     the part, then the element, where the running sum passes the draw
// Greedy calls take the first two only, with (first maximum) in place of (max, sum).

#include <hip/hip_runtime.h>

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
constexpr int kMaxRows = 2 * PCP_VERIFY_MAX_DRAFT + 1;

struct RowState {
  double sum;   // greedy: unused
  float max;
  int32_t at;   // greedy: the first maximum's index; sampling: NaN seen
};

// Where a sequence ends: the row its last token comes from.
struct SeqEnd {
  double scale_p, scale_q;   // 1 / sum e of the target row, of the draft row (0: q is 0)
  double max_p, max_q;
  double lse_p;              // natural units, of logits / temperature
  int32_t j;                 // accepted tokens
  int32_t without;           // a lookup's refused token (r is 0 there), or -1
  int32_t bad;               // the target row's sum is not finite
  int32_t pad;
};

struct VerifyArgs {
  const void* target;
  const void* draft;          // nullptr: all of q on the drafted token
  const int64_t* ids;
  const int32_t* lens;
  const float* uniforms;
  int64_t* tokens;
  int32_t* accepted;
  float* logp;
  RowState* part;             // [S, 2n + 1, parts]
  double* seg;                // [S, parts + 2]: residual sums of head, parts, tail
  SeqEnd* end;                // [S]
  int* err;
  int64_t vocab, tstride, dstride;   // elements
  double k;                   // log2(e) / temperature
  double inv_t;
  int32_t n, n_rows;          // drafted tokens, rows per sequence (n + 1, or 2n + 1 with a draft model)
  int32_t parts, greedy;
};

// 2^y for y <= 0, to the rounding of 64 bits (0 below 2^-1075, NaN kept): 2^n times a polynomial
// in y - n that meets 2^f in the 11 Chebyshev points of [-1/2, 1/2] (relative error 3e-16; with
// 9 points 1e-12, which over 151,936 tokens would decide some draws).
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

template <typename TI>
__device__ __forceinline__ const char* target_row(const VerifyArgs& a, int64_t s, int i) {
  return static_cast<const char*>(a.target) + (s * (a.n + 1) + i) * a.tstride * TI::kBytes;
}
template <typename TI>
__device__ __forceinline__ const char* draft_row(const VerifyArgs& a, int64_t s, int i) {
  return static_cast<const char*>(a.draft) + (s * a.n + i) * a.dstride * TI::kBytes;
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

// ---- rows ------------------------------------------------------------------------------
template <typename TI, bool GREEDY>
__global__ void __launch_bounds__(kBlock) verify_rows_kernel(VerifyArgs a) {
  constexpr int EPV = 16 / TI::kBytes, U = kU, BLOCK = kBlock;
  __shared__ double lds64[BLOCK / 64];
  __shared__ float wmax[BLOCK / 64];
  __shared__ int wat[BLOCK / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, part = blockIdx.x, i = blockIdx.y;
  const int64_t s = blockIdx.z;
  const int len = draft_len(a, s);
  const bool is_target = i <= a.n;
  if (is_target ? i > len : i - a.n - 1 >= len) return;   // rows of tokens that were not drafted
  const char* row = is_target ? target_row<TI>(a, s, i) : draft_row<TI>(a, s, i - a.n - 1);
  const RowSpan sp = row_span<TI>(row, a.vocab);
  const int v0 = part * kPartVecs;
  const __amdgpu_buffer_rsrc_t buf = row_rsrc(sp.vec, static_cast<uint32_t>(sp.nv) * 16u);
  u32x4 x[U];
#pragma unroll
  for (int q = 0; q < U; ++q) x[q] = buf_ld16<false>(buf, static_cast<uint32_t>(v0 + q * BLOCK + tid) * 16u);
  const int ek = part == 0 ? edge_index<TI>(sp, tid) : -1;
  const float xe = ek >= 0 ? TI::load1(row, ek) : kNegInf;
  auto held = [&](int q) { return v0 + q * BLOCK + tid < sp.nv; };
  RowState* out = a.part + ((s * a.n_rows + i) * a.parts + part);
  if constexpr (GREEDY) {
    float best = kNegInf;
    int at = INT32_MAX;
    if (xe > kNegInf) {
      best = xe;
      at = ek;
    }
#pragma unroll
    for (int q = 0; q < U; ++q)
      if (held(q))
#pragma unroll
        for (int j = 0; j < EPV; ++j) {
          const float v = TI::unpack(reinterpret_cast<const uint32_t*>(&x[q]), j);
          const int e = sp.head + (v0 + q * BLOCK + tid) * EPV + j;
          if (v > kNegInf) better32(best, at, v, e);
        }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) better32(best, at, __shfl_xor(best, o), __shfl_xor(at, o));
    if (lane == 0) {
      wmax[wave] = best;
      wat[wave] = at;
    }
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < BLOCK / 64; ++w) better32(best, at, wmax[w], wat[w]);
      *out = RowState{0., best, at};
    }
  } else {
    float m = xe;
    bool nan = !(xe == xe);
#pragma unroll
    for (int q = 0; q < U; ++q)
      if (held(q)) {
        m = vec_max<TI>(m, x[q]);
#pragma unroll
        for (int j = 0; j < EPV; ++j) {
          const float v = TI::unpack(reinterpret_cast<const uint32_t*>(&x[q]), j);
          nan |= !(v == v);
        }
      }
    m = lanes_max<64>(m);
    if (lane == 0) wmax[wave] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < BLOCK / 64; ++w) m = fmaxf(m, wmax[w]);
    const double ref = -static_cast<double>(ms_ref(m)) * a.k;
    double sum = exp2_64(fma(static_cast<double>(xe), a.k, ref));   // 0 for threads without one
#pragma unroll
    for (int q = 0; q < U; ++q)
      if (held(q))
#pragma unroll
        for (int j = 0; j < EPV; ++j)
          sum += exp2_64(fma(static_cast<double>(TI::unpack(reinterpret_cast<const uint32_t*>(&x[q]), j)), a.k, ref));
    sum = block_sum64<BLOCK>(sum, lds64);
    const int any_nan = __syncthreads_or(nan);
    if (tid == 0) *out = RowState{sum, m, any_nan};
  }
}

// ---- decide ----------------------------------------------------------------------------
constexpr int kDecideBlock = 512;

template <typename TI, bool GREEDY>
__global__ void __launch_bounds__(kDecideBlock) verify_decide_kernel(VerifyArgs a) {
  __shared__ double row_sum[kMaxRows];
  __shared__ float row_max[kMaxRows];
  __shared__ int row_at[kMaxRows];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t s = blockIdx.x;
  const int len = draft_len(a, s);
  for (int i = wave; i < a.n_rows; i += kDecideBlock / 64) {
    if (i <= a.n ? i > len : i - a.n - 1 >= len) continue;
    const RowState* p = a.part + (s * a.n_rows + i) * a.parts;
    float m = kNegInf;
    if constexpr (GREEDY) {
      int at = INT32_MAX;
      for (int q = lane; q < a.parts; q += 64) better32(m, at, p[q].max, p[q].at);
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) better32(m, at, __shfl_xor(m, o), __shfl_xor(at, o));
      if (lane == 0) row_at[i] = at == INT32_MAX ? 0 : at;
    } else {
      int nan = 0;
      for (int q = lane; q < a.parts; q += 64) {
        m = fmaxf(m, p[q].max);
        nan |= p[q].at;
      }
      m = lanes_max<64>(m);
      double sum = 0.;
      for (int q = lane; q < a.parts; q += 64)
        if (p[q].max > kNegInf) sum += p[q].sum * exp2_64((static_cast<double>(p[q].max) - static_cast<double>(m)) * a.k);
      sum = wave_sum64(sum);
      if (lane == 0) {
        row_sum[i] = sum;
        row_max[i] = m;
        row_at[i] = __builtin_isfinite(m) && __builtin_isfinite(sum);
      }
      const bool any = __any(nan != 0);
      if (lane == 0 && any) row_at[i] = 0;
    }
  }
  __syncthreads();
  if (wave != 0) return;
  if (lane == 0 && a.lens && (a.lens[s] < 0 || a.lens[s] > a.n)) raise_error(a.err, kErrDraftLen);
  // Lane i decides token i (n <= 64).
  const int64_t d = lane < len ? a.ids[s * a.n + lane] : 0;
  const bool in = d >= 0 && d < a.vocab;
  bool ok = false, bad_p = false, bad_q = false;
  float lp = 0.f;
  if (lane < len) {
    if constexpr (GREEDY) {
      ok = d == row_at[lane];
    } else {
      bad_p = !row_at[lane];
      bad_q = a.draft && !row_at[a.n + 1 + lane];
      if (in && !bad_p && !bad_q) {
        const double y = fma(static_cast<double>(TI::load1(target_row<TI>(a, s, lane), d)), a.k,
                             -static_cast<double>(row_max[lane]) * a.k);
        const double p = exp2_64(y) / row_sum[lane];
        double q = 1.;
        if (a.draft) {
          const int r = a.n + 1 + lane;
          q = exp2_64(fma(static_cast<double>(TI::load1(draft_row<TI>(a, s, lane), d)), a.k,
                          -static_cast<double>(row_max[r]) * a.k)) / row_sum[r];
        }
        ok = static_cast<double>(a.uniforms[s * (a.n + 1) + lane]) * q < p;
        lp = static_cast<float>(y * 0.69314718055994530942 - log(row_sum[lane]));
      }
    }
  }
  const uint64_t no = ~__ballot(ok);
  const int j = min(no ? __builtin_ctzll(no) : 64, len);
  if (lane == j && lane < len && !in) raise_error(a.err, kErrTokenRange);
  if (lane == 0) a.accepted[s] = j;
  int64_t* tok = a.tokens + s * (a.n + 1);
  float* logp = a.logp ? a.logp + s * (a.n + 1) : nullptr;
  // Entries 0 .. n (65 at most): the accepted tokens, the one after, then the pad.
  for (int i = lane; i <= a.n; i += 64) {
    if (i < j) {
      tok[i] = d;
      if (logp) logp[i] = lp;
    } else if (i > j) {
      tok[i] = PCP_IGNORE_INDEX;
      if (logp) logp[i] = 0.f;
    } else if (GREEDY) {
      tok[i] = row_at[j];
      if (logp) logp[i] = 0.f;
    }
  }
  if constexpr (!GREEDY) {
    const bool refused = j < len;
    const bool q_bad = refused && __builtin_amdgcn_readlane(bad_q, j);
    const bool out = refused && !__builtin_amdgcn_readlane(in, j);
    if (lane == 0) {
      SeqEnd e;
      e.j = j;
      e.bad = !row_at[j];
      e.max_p = ms_ref(row_max[j]);
      e.scale_p = 1. / row_sum[j];
      e.lse_p = e.max_p * a.inv_t + log(row_sum[j]);
      const bool model = refused && a.draft && !q_bad && !out;
      const int r = a.n + 1 + j;
      e.max_q = model ? row_max[r] : 0.;
      e.scale_q = model ? 1. / row_sum[r] : 0.;
      e.without = refused && !a.draft && !out ? static_cast<int32_t>(a.ids[s * a.n + j]) : -1;
      e.pad = 0;
      a.end[s] = e;
      if (e.bad || q_bad) raise_error(a.err, kErrNonFinite);
    }
  }
}

// ---- residual --------------------------------------------------------------------------
// r of one element: max(p - q, 0), p alone where scale_q is 0.
struct Residual {
  double k, ref_p, ref_q, scale_p, scale_q;
  int without;
  bool plain;   // p alone: nothing of p lies above q
  __device__ __forceinline__ double operator()(float x, float y, int id) const {
    const double p = exp2_64(fma(static_cast<double>(x), k, ref_p)) * scale_p;
    if (plain) return p;
    if (scale_q != 0.) return fmax(p - exp2_64(fma(static_cast<double>(y), k, ref_q)) * scale_q, 0.);
    return id == without ? 0. : p;
  }
};

__device__ __forceinline__ Residual residual(const VerifyArgs& a, const SeqEnd& e, bool plain) {
  return Residual{a.k, -e.max_p * a.k, -e.max_q * a.k, e.scale_p, e.scale_q, e.without, plain};
}

// The elements of a part: both rows' values, in element order per (chunk, lane, element). The
// draft row may start at another offset of its 16 bytes, so it is read element by element there.
template <typename TI, typename F>
__device__ __forceinline__ void part_elements(const VerifyArgs& a, const SeqEnd& e, int64_t s, const RowSpan& sp, int v0,
                                              F f) {
  constexpr int EPV = 16 / TI::kBytes, U = kU, BLOCK = kBlock;
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

template <typename TI>
__global__ void __launch_bounds__(kBlock) verify_residual_kernel(VerifyArgs a) {
  __shared__ double lds[kBlock / 64];
  const int tid = threadIdx.x, part = blockIdx.x;
  const int64_t s = blockIdx.y;
  const SeqEnd e = a.end[s];
  if (e.bad) return;
  const char* row = target_row<TI>(a, s, e.j);
  const RowSpan sp = row_span<TI>(row, a.vocab);
  const Residual r = residual(a, e, false);
  double* seg = a.seg + s * (a.parts + 2);
  if (part == 0 && tid < 64) {
    const int ek = edge_index<TI>(sp, tid);
    double v = 0.;
    if (ek >= 0) v = r(TI::load1(row, ek), e.scale_q != 0. ? TI::load1(draft_row<TI>(a, s, e.j), ek) : 0.f, ek);
    const double head = wave_sum64(tid < sp.head ? v : 0.), tail = wave_sum64(tid >= sp.head ? v : 0.);
    if (tid == 0) {
      seg[0] = head;
      seg[a.parts + 1] = tail;
    }
  }
  double sum = 0.;
  part_elements<TI>(a, e, s, sp, part * kPartVecs, [&](int, int, bool held, float x, float y, int id) {
    if (held) sum += r(x, y, id);
  });
  sum = block_sum64<kBlock>(sum, lds);
  if (tid == 0) seg[1 + part] = sum;
}

// ---- pick ------------------------------------------------------------------------------
template <typename TI>
__global__ void __launch_bounds__(kBlock) verify_pick_kernel(VerifyArgs a) {
  constexpr int EPV = 16 / TI::kBytes, U = kU, NW = kBlock / 64;
  __shared__ double chunk_sum[U][NW];
  __shared__ int first;       // the smallest element whose running sum passes
  __shared__ int last;        // the largest element with r > 0, where rounding leaves none
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t s = blockIdx.x;
  const SeqEnd e = a.end[s];
  int64_t* tok = a.tokens + s * (a.n + 1) + e.j;
  float* logp = a.logp ? a.logp + s * (a.n + 1) + e.j : nullptr;
  if (e.bad) {
    if (tid == 0) {
      *tok = a.vocab - 1;
      if (logp) *logp = 0.f;
    }
    return;
  }
  const char* row = target_row<TI>(a, s, e.j);
  const char* drow = e.scale_q != 0. ? draft_row<TI>(a, s, e.j) : nullptr;
  const RowSpan sp = row_span<TI>(row, a.vocab);
  const double u = static_cast<double>(a.uniforms[s * (a.n + 1) + a.n]);
  const double* seg = a.seg + s * (a.parts + 2);
  const int segs = a.parts + 2;
  // Each wave: the total, then the first segment whose running sum passes u * total.
  double total = 0.;
  for (int b = 0; b < segs; b += 64) total += wave_sum64(b + lane < segs ? seg[b + lane] : 0.);
  // Nothing of p above q (equal rows): the token comes from p, whose sums are not in seg; the
  // whole row is then one segment, scanned part by part.
  const bool plain = !(total > 0.);
  const Residual r = residual(a, e, plain);
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
    if (g == 0 || g == a.parts + 1) {   // the head or the tail: at most 7 elements, each thread alone
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
      part_elements<TI>(a, e, s, sp, (g - 1) * kPartVecs, [&](int q, int j, bool held, float x, float y, int id) {
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
        for (int w = 0; w < NW; ++w) {
          if (w < wave) b += chunk_sum[q][w];
          base += chunk_sum[q][w];
        }
        double c = b + (incl[q] - part_sum[q]);
#pragma unroll
        for (int j = 0; j < EPV; ++j) {
          c += mine[q][j];
          const int id = sp.head + ((g - 1) * kPartVecs + q * kBlock + tid) * EPV + j;
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
  int pick = -1;
  if (!plain) {
    double run = before;
    const int g = hit >= 0 ? hit : last_seg;   // rounding past the last segment: its last element
    pick = scan(g, run) ? first : last;
  } else {
    double run = 0.;
    for (int g = 0; g < segs; ++g) {
      const bool found = scan(g, run);
      if (last >= 0) pick = found ? first : last;
      const bool stop = found;
      __syncthreads();   // first / last read before the next segment resets them
      if (stop) break;
    }
  }
  if (tid == 0) {
    if (pick < 0) pick = static_cast<int>(a.vocab) - 1;
    *tok = pick;
    if (logp) *logp = static_cast<float>(static_cast<double>(TI::load1(row, pick)) * a.inv_t - e.lse_p);
  }
}

template <typename TI>
hipError_t launch_verify(const VerifyArgs& a, int64_t n_seq, hipStream_t st) {
  const unsigned parts = static_cast<unsigned>(a.parts), ns = static_cast<unsigned>(n_seq);
  const dim3 rows(parts, static_cast<unsigned>(a.n_rows), ns), b(kBlock);
  if (a.greedy) {
    verify_rows_kernel<TI, true><<<rows, b, 0, st>>>(a);
    verify_decide_kernel<TI, true><<<dim3(ns), dim3(kDecideBlock), 0, st>>>(a);
  } else {
    verify_rows_kernel<TI, false><<<rows, b, 0, st>>>(a);
    verify_decide_kernel<TI, false><<<dim3(ns), dim3(kDecideBlock), 0, st>>>(a);
    verify_residual_kernel<TI><<<dim3(parts, ns), b, 0, st>>>(a);
    verify_pick_kernel<TI><<<dim3(ns), b, 0, st>>>(a);
  }
  return hipGetLastError();
}

inline bool misaligned(const void* p, int size) {
  return (reinterpret_cast<uintptr_t>(p) & static_cast<uintptr_t>(size - 1)) != 0;
}
inline size_t round256(size_t b) { return (b + 255) & ~static_cast<size_t>(255); }

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
  int64_t tmp;
  if (mul_overflows(a->n_seq * (a->n_draft + 1), ts, &tmp) || mul_overflows(tmp, 4, &tmp) ||
      mul_overflows(a->n_seq * a->n_draft, ds, &tmp) || mul_overflows(tmp, 4, &tmp))
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
  const int64_t n_rows = a->n_draft + 1 + (model ? a->n_draft : 0);
  const size_t S = static_cast<size_t>(a->n_seq);
  const size_t o_seg = round256(sizeof(RowState) * S * n_rows * parts);
  const size_t o_end = o_seg + round256(sizeof(double) * S * (parts + 2));
  const int rc = ensure_scratch_on(ctx, o_end + sizeof(SeqEnd) * S, st);
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
  v.seg = reinterpret_cast<double*>(sp + o_seg);
  v.end = reinterpret_cast<SeqEnd*>(sp + o_end);
  v.err = ctx->d_page->err;
  v.vocab = a->vocab;
  v.tstride = ts;
  v.dstride = ds;
  v.inv_t = greedy ? 1. : 1. / static_cast<double>(a->temperature);
  v.k = 1.4426950408889634074 * v.inv_t;
  v.n = static_cast<int32_t>(a->n_draft);
  v.n_rows = static_cast<int32_t>(n_rows);
  v.parts = static_cast<int32_t>(parts);
  v.greedy = greedy;
  const bool timed = prof_begin(ctx, st);
  const hipError_t e = a->logits_dtype == PCP_F32    ? launch_verify<F32T>(v, a->n_seq, st)
                       : a->logits_dtype == PCP_BF16 ? launch_verify<BF16T>(v, a->n_seq, st)
                                                     : launch_verify<F16T>(v, a->n_seq, st);
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
