// Scores of given tokens (pcp_score.h): log-probs, entropy and the top alternatives of rows of
// logits, and the gradient of a function of the log-probs and entropies.
//
// Forward: one read of a row. With m the largest logit, d = (x - m) log2(e) / temperature, s = sum 2^d and
// t = sum 2^d d, the log-sum-exp is m / temperature + ln s and the entropy ln s - ln 2 t / s, two parts that are not
// negative: a row with one likely token keeps its entropy to 2^-24, the rounding of its largest term. A batch of eight
// 16-byte vectors a lane gives a lane's maximum (two 16-bit elements an instruction), then s and t against it; the next
// batch's loads are out meanwhile. The alternatives come after the pass: the lanes have kept their groups' maxima, what k
// of those reach rules out all but about k groups, and these are read again. Few rows are cut into parts, whose sums and
// candidates the last part to finish merges; there a part is one batch, and its candidates come from its registers.
//
// Bound by HBM with many rows, and by their last ones: 4096 rows of 151,936 bf16 192 us (6.5 TB/s, 65% of the VALU's
// time), with 5/8 of them live 126 (6.2 TB/s), with k = 20 207 and 139. By latency with few: one row 7.9 us, with
// k = 20 11.1 (meta data 0.4, the pass 1.6, sums 0.6, candidates 2.3, stores and ticket 1.0, merge 3, ranking 1); 64
// f32 rows 12 and with k = 5 17. Rows of masks with fewer than k tokens left take one more pass (4096 such rows
// 393 us; by select_exact, as first written, 2097), rows of a few equal values six (select_exact, 2490).
//
// Backward: one read of the logits, one write (or update) of dlogits, elementwise from the forward's
// statistics; 4096 rows of 151,936 bf16, 5/8 of them live, 349 us (5.8 TB/s), added to what was there 384 (6.1).

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstddef>
#include <cstdint>
#include <cstring>

#include "context.hpp"
#include "grpo_device.hpp"
#include "pcp_score.h"
#include "score_split.hpp"
#include "top_device.hpp"

namespace pcp {
namespace {

constexpr double kLn2d = 0.69314718055994530942;

// The token arrays of a call and the rows that they weigh.
struct TokenArrays {
  const void* ids;      // nullptr: no row has a token
  const void* mask;     // nullptr: all ones
  int64_t rows, tok_stride, tok_offset, vocab;
  int* err;
  int32_t ids_i64, mask_u8;
};

struct ScoreRow {
  int64_t at;      // index in the token arrays
  int64_t id;      // -1: no token
  bool live;
};

__device__ __forceinline__ ScoreRow score_row(const TokenArrays& a, int64_t s, int64_t t) {
  ScoreRow r{s * a.tok_stride + a.tok_offset + t, -1, true};
  if (a.ids != nullptr)   // (read along with the mask: one latency for both)
    r.id = a.ids_i64 ? static_cast<const int64_t*>(a.ids)[r.at] : static_cast<const int32_t*>(a.ids)[r.at];
  if (a.mask != nullptr)
    r.live = a.mask_u8 ? static_cast<const uint8_t*>(a.mask)[r.at] != 0 : static_cast<const float*>(a.mask)[r.at] != 0.f;
  if (a.ids != nullptr && r.live && (r.id < 0 || r.id >= a.vocab)) {
    if (r.id != PCP_IGNORE_INDEX && threadIdx.x == 0) raise_error(a.err, kErrTokenRange);
    r.live = false;
  }
  return r;
}

// ---- forward ----------------------------------------------------------------------------

// A part of a row as its workgroup leaves it.
struct alignas(16) ScorePart {
  double s, t;
  float mx;
  int32_t n;               // its candidates
  int64_t pad;
};

struct ScoreArgs {
  TokenArrays tok;
  const void* logits;
  int64_t row_stride, seq_stride;
  int64_t row0;            // of this launch
  float* logp;
  float* entropy;
  float* row_max;
  float* log_sum;
  float* top_logp;
  void* top_ids;
  uint64_t* part_key;      // [row, parts, part_cap]
  ScorePart* part;         // [row, parts]
  unsigned* done;          // [row] parts that are, 0 between launches
  double inv_tau;
  float k2;                // log2(e) / temperature
  int32_t k, top_i64, parts, per, part_cap;
  int32_t group;           // batches per group (gather_top)
};

// Loads at agent scope (sc1), for what other workgroups have stored with store_coherent.
constexpr int kBufAgent = 16;
__device__ __forceinline__ u32x4 buf_ld16_coherent(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, kBufAgent));
}
__device__ __forceinline__ uint64_t buf_ld8_coherent(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  return __builtin_bit_cast(uint64_t, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, kBufAgent));
}

// An exponent this low is a term of 0, whose product with it then is 0 too (and not NaN at -inf).
constexpr float kLeastExp = -1024.f;

// A sum of terms and one of terms times their exponents (both against m), against M >= m.
__device__ __forceinline__ void score_rebase(double& s, double& t, float m, float M, float k) {
  const float d = fmaxf((m - ms_ref(M)) * k, kLeastExp);
  const double w = hw_exp2(d);
  t = s == 0. ? 0. : w * (t + d * s);
  s = s == 0. ? 0. : w * s;
}

// Of a lane: its largest logit mx, and against it the sum s of the terms 2^d, d = (x - mx) k, and the sum t of
// 2^d d. The sums of a batch are f32 against the rounded product ref of mx and k, whose residue r is
// taken out once per batch: of terms 2^d it leaves 2^-r s and 2^-r (t - r s). A batch has 64 terms at most, so that f32 loses
// less than 4e-6 of them at worst (measured against 64 bits: 2e-7), and f64 would take a conversion and two adds of half the rate
// per term of a kernel whose VALU is 65% busy; everything above a batch is f64.
struct ScoreSums {
  float k2, mx;
  double s, t;
  bool masked;

  // CLAMP: exponents of -inf, or near it, may be among them, whose products would be NaN.
  template <typename TI, bool CLAMP, int U, typename Held>
  __device__ __forceinline__ void terms(const u32x4 (&x)[U], Held held, const TermScale& ts, float& s1, float& t1) {
    s1 = t1 = 0.f;
#pragma unroll
    for (int q = 0; q < U; ++q)
      if (held(q)) {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(&x[q]);
#pragma unroll
        for (int j = 0; j < 16 / TI::kBytes; ++j) {
          const float d = fmaf(TI::unpack(w, j), ts.k, -ts.ref);
          const float e = hw_exp2(d);
          s1 += e;
          t1 = fmaf(e, CLAMP ? fmaxf(d, kLeastExp) : d, t1);
        }
      }
  }
  // A batch whose largest logit is bx. A masked element's product 0 * -inf makes t1 NaN: then once more, and
  // from there on, with exponents clamped.
  template <typename TI, int U, typename Held>
  __device__ __forceinline__ void add(const u32x4 (&x)[U], Held held, float bx) {
    const float nm = fmaxf(mx, bx);
    const TermScale ts = term_scale(nm, k2);
    float s1, t1;
    if (!masked) {
      terms<TI, false>(x, held, ts, s1, t1);
      masked = __any(t1 != t1);
    }
    if (masked) {
      // Opaque copies: the compiler would else keep every exponent and term of the first pass for this one.
      u32x4 y[U];
#pragma unroll
      for (int q = 0; q < U; ++q) {
        y[q] = x[q];
        asm volatile("" : "+v"(y[q]));
      }
      terms<TI, true>(y, held, ts, s1, t1);
    }
    score_rebase(s, t, mx, nm, k2);
    const float r = term_residue(nm, ts), adj = hw_exp2(-r);
    s += static_cast<double>(s1 * adj);
    t += static_cast<double>(fmaf(-r, s1, t1) * adj);
    mx = nm;
  }
};

// The largest element of a batch, two 16-bit ones an instruction. bf16 values compare as 16-bit integers where one is
// positive; a lane that holds negative ones alone (or none), or a NaN, which is above all as an integer, makes its wave
// look again.
template <typename TI, int U, typename Held>
__device__ __forceinline__ float batch_max(const u32x4 (&x)[U], Held held) {
  typedef short i16x2 __attribute__((ext_vector_type(2)));
  float m = kNegInf;
  if constexpr (__is_same(TI, BF16T)) {
    i16x2 top = {-32768, -32768};
#pragma unroll
    for (int q = 0; q < U; ++q)
      if (held(q)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t w = x[q][i];   // (a variable: __builtin_bit_cast of a vector's element takes the first one)
          top = __builtin_elementwise_max(top, __builtin_bit_cast(i16x2, w));
        }
      }
    const uint32_t t = __builtin_bit_cast(uint32_t, top);
    const float even = __uint_as_float(t << 16), odd = __uint_as_float(t & 0xffff0000u);
    if (!__any((top[0] < 0 && top[1] < 0) || __builtin_isunordered(even, odd))) return fmaxf(even, odd);
    m = kNegInf;
#pragma unroll
    for (int q = 0; q < U; ++q) m = held(q) ? vec_max<TI>(m, x[q]) : m;
  } else if constexpr (__is_same(TI, F16T)) {
    f16x2 top = {-__builtin_inff16(), -__builtin_inff16()};
#pragma unroll
    for (int q = 0; q < U; ++q)
      if (held(q)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t w = x[q][i];
          top = __builtin_elementwise_max(top, __builtin_bit_cast(f16x2, w));
        }
      }
    m = fmaxf(static_cast<float>(top[0]), static_cast<float>(top[1]));
  } else {
#pragma unroll
    for (int q = 0; q < U; ++q) m = held(q) ? vec_max<TI>(m, x[q]) : m;
  }
  return m;
}

// ---- the k largest of a part ----
// The pass over the part leaves each lane's largest logit of every group of batches (at most kGroups groups). What k of
// those reach, k elements reach, each in a group of its own; so only groups that reach it are read again, about
// k of a row's thousands, and what reaches it there are the candidates, few more than k.

constexpr int kGroups = kScoreGroups;
static_assert(kBlock == kScoreBlock && kU == kScoreU, "score_split.hpp");

struct PartShared {
  union {
    Shared sh;
    float group[kGroups][kBlock];   // until the candidates are gathered
  };
};
static_assert(offsetof(Shared, key) == 0 && sizeof(float) * kGroups * kBlock <= sizeof(uint64_t) * kCap,
              "groups lie over the keys alone");

// The part's candidates where values may be equal in any number: the exact k-th largest by its bits, eight a pass,
// then those above it and as many of its equals as are missing, by rising id. Called by the whole workgroup with sh free;
// returns their number, min(k, elements). Six passes: for parts of masks or of few values.
template <typename TI>
__device__ __forceinline__ int select_exact(const char* xrow, const RowSpan& sp, __amdgpu_buffer_rsrc_t xbuf, int v0, int end,
                                            bool edges, int k, Shared& sh) {
  constexpr int EPV = 16 / TI::kBytes;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int total = max(end - v0, 0) * EPV + (edges ? sp.head + sp.tail : 0);
  const int ek = edges ? edge_index<TI>(sp, tid) : -1;
  const uint32_t edge = ek >= 0 ? order_bits(TI::load1(xrow, ek)) : 0u;
  int need = min(k, total);
  uint32_t prefix = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    for (int i = tid; i < kBins; i += kBlock) sh.bin[i] = 0;
    __syncthreads();
    auto count = [&](bool is, uint32_t b) {
      const uint32_t rest = shift == 24 ? 0u : (b ^ prefix) >> (shift + 8);
      const int bin = is && rest == 0 ? static_cast<int>(b >> shift & 255u) : -1;
      // One lane for all where a wave's elements are alike, as masks are.
      const int other = __builtin_amdgcn_readfirstlane(bin);
      if (__all(bin == other)) {
        if (lane == 0 && bin >= 0) atomicAdd(&sh.bin[bin], 64);
      } else if (bin >= 0) {
        atomicAdd(&sh.bin[bin], 1);
      }
    };
    for (int base = v0; base < end; base += kBlock) {
      const bool is = base + tid < end;
      const u32x4 x = buf_ld16<false>(xbuf, static_cast<uint32_t>(base + tid) * 16u);
#pragma unroll
      for (int j = 0; j < EPV; ++j) count(is, order_bits(TI::unpack(reinterpret_cast<const uint32_t*>(&x), j)));
    }
    if (ek >= 0) {
      const uint32_t rest = shift == 24 ? 0u : (edge ^ prefix) >> (shift + 8);
      if (rest == 0) atomicAdd(&sh.bin[edge >> shift & 255u], 1);
    }
    __syncthreads();
    // Every wave finds the bin of the need-th largest: lane l has bins 4 (63 - l) .. + 3.
    const int first = 4 * (63 - lane);
    const int4 c = *reinterpret_cast<const int4*>(&sh.bin[first]);
    const int all = c.x + c.y + c.z + c.w;
    int above = lanes_scan(all) - all, at = first + 3;
    const int counts[4] = {c.w, c.z, c.y, c.x};
    const uint64_t who = __ballot(above + all >= need);
    bool found = false;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (!found) {
        if (above + counts[i] >= need) {
          found = true;
          at = first + 3 - i;
        } else {
          above += counts[i];
        }
      }
    const int owner = __builtin_ctzll(who);
    need -= __builtin_amdgcn_readlane(above, owner);
    prefix |= static_cast<uint32_t>(__builtin_amdgcn_readlane(at, owner)) << shift;
  }
  // prefix: the k-th largest, need: its equals to take, by rising id: head, interior, tail.
  __syncthreads();
  if (tid == 0) sh.count = 0;
  int taken = 0;
  __syncthreads();
  Candidates c{sh, 0, kNegInf};
  auto step = [&](const u32x4& x, bool is, uint32_t id0, int n_el) {   // up to EPV elements of rising id per lane
    uint32_t b[EPV];
    int mine = 0;
#pragma unroll
    for (int j = 0; j < EPV; ++j) {
      b[j] = order_bits(TI::unpack(reinterpret_cast<const uint32_t*>(&x), j));
      mine += is && j < n_el && b[j] == prefix;
    }
    const int incl = lanes_scan(mine);
    if (lane == 63) sh.bin[wave] = incl;
    __syncthreads();
    int before = taken + incl - mine, sum = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      before += w < wave ? sh.bin[w] : 0;
      sum += sh.bin[w];
    }
    __syncthreads();
    taken += sum;
#pragma unroll
    for (int j = 0; j < EPV; ++j) {
      const bool there = is && j < n_el, same = there && b[j] == prefix;
      c.add((there && b[j] > prefix) || (same && before < need),
            static_cast<uint64_t>(b[j]) << 32 | (0xffffffffu - (id0 + static_cast<uint32_t>(j))));
      before += same;
    }
  };
  auto one = [&](int at) {
    u32x4 x = {};
    const float v = TI::load1(xrow, at);
    x[0] = TI::kBytes == 4 ? __float_as_uint(v) : __is_same(TI, BF16T) ? __float_as_uint(v) >> 16 : pack2<F16T>(v, 0.f);
    return x;
  };
  if (edges) step(one(min(tid, max(sp.head - 1, 0))), tid < sp.head, static_cast<uint32_t>(tid), 1);
  for (int base = v0; base < end; base += kBlock)
    step(buf_ld16<false>(xbuf, static_cast<uint32_t>(base + tid) * 16u), base + tid < end,
         static_cast<uint32_t>(sp.head + (base + tid) * EPV), EPV);
  const int tail0 = sp.head + sp.nv * EPV;
  if (edges)
    step(one(tail0 + min(tid, max(sp.tail - 1, 0)) - (sp.tail == 0)), tid < sp.tail, static_cast<uint32_t>(tail0 + tid), 1);
  __syncthreads();
  return min(k, total);
}

// The candidates of a part where fewer than k values lie above masks: those, and of the masked ones, if all are
// equal, the first k elements of the part (at least as many as are missing are among them, unless some are NaN). Called by
// the whole workgroup; ends with a barrier.
template <typename TI>
__device__ __forceinline__ int gather_masked(const char* xrow, const RowSpan& sp, __amdgpu_buffer_rsrc_t xbuf, int v0, int end,
                                             bool edges, int k, Shared& sh) {
  constexpr int EPV = 16 / TI::kBytes, U = 4;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int total = max(end - v0, 0) * EPV + (edges ? sp.head + sp.tail : 0);
  __syncthreads();
  if (tid == 0) sh.count = 0;
  __syncthreads();
  Candidates c{sh, 0, kMasked + 0x1p-9f};   // the least f32 above kMasked
  float lo = __builtin_inff(), hi = kNegInf;   // of the masked elements
  auto masked = [&](bool is, float e) {
    is = is && e <= kMasked;
    lo = is ? fminf(lo, e) : lo;
    hi = is ? fmaxf(hi, e) : hi;
  };
  if (edges && tid < 64) {
    const int ek = edge_index<TI>(sp, tid);
    const float e = ek >= 0 ? TI::load1(xrow, ek) : kNegInf;
    masked(ek >= 0, e);
    c.add(ek >= 0 && e >= c.least_x, element_key(e, static_cast<uint32_t>(ek)));
  }
  for (int base = v0; base < end; base += kBlock * U) {
    u32x4 x[U];
#pragma unroll
    for (int q = 0; q < U; ++q) x[q] = buf_ld16<false>(xbuf, static_cast<uint32_t>(base + q * kBlock + tid) * 16u);
    uint32_t left_q = 0;
#pragma unroll
    for (int q = 0; q < U; ++q) {
      const bool is = base + q * kBlock + tid < end;
#pragma unroll
      for (int j = 0; j < EPV; ++j) masked(is, TI::unpack(reinterpret_cast<const uint32_t*>(&x[q]), j));
      left_q |= is && vec_max<TI>(kNegInf, x[q]) >= c.least_x ? 1u << q : 0u;
    }
    take_vectors<TI>(c, x, left_q, static_cast<uint32_t>(sp.head + (base + tid) * EPV), (1u << EPV) - 1u);
  }
  lo = -lanes_max<64>(-lo);
  hi = lanes_max<64>(hi);
  if (lane == 0) {
    sh.low[wave] = lo;
    sh.high[wave] = hi;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    lo = fminf(lo, sh.low[w]);
    hi = fmaxf(hi, sh.high[w]);
  }
  const int first = edges ? 0 : sp.head + v0 * EPV;
  const float e = tid < min(k, total) ? TI::load1(xrow, first + tid) : 0.f;
  c.add(tid < min(k, total) && e <= kMasked, element_key(e, static_cast<uint32_t>(first + tid)));
  __syncthreads();
  const int n = sh.count;
  __syncthreads();
  return n >= min(k, total) && n <= kCap && !(lo < hi) ? n : select_exact<TI>(xrow, sp, xbuf, v0, end, edges, k, sh);
}

// The candidates of a part whose lanes have left their groups' largest logits (batches: batches per group, groups:
// how many), k or more of them where the part has as many elements. Called by the whole workgroup; ends with a barrier.
template <typename TI>
__device__ __forceinline__ int gather_top(const char* xrow, const RowSpan& sp, __amdgpu_buffer_rsrc_t xbuf, int v0, int end,
                                          bool edges, int k, int batches, int groups, PartShared& ps) {
  constexpr int EPV = 16 / TI::kBytes, U = kU;
  Shared& sh = ps.sh;
  const int tid = threadIdx.x;
  float v[kGroups], lane_max[1] = {kNegInf};
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    v[g] = g < groups ? ps.group[g][tid] : kNegInf;
    lane_max[0] = fmaxf(lane_max[0], v[g]);
  }
  // Up to 64 of the lanes' own maxima are nearly as high as the groups', and 256 values sooner counted than 4096.
  const float least = k <= 64 ? reached_by(sh, lane_max, k) : reached_by(sh, v, k);
  uint32_t left = 0;
#pragma unroll
  for (int g = 0; g < kGroups; ++g) left |= g < groups && v[g] >= least ? 1u << g : 0u;
  __syncthreads();
  if (tid == 0) sh.count = 0;
  __syncthreads();
  const int total = max(end - v0, 0) * EPV + (edges ? sp.head + sp.tail : 0);
  const bool all = least == kNegInf;   // fewer than k values above masks: a short part's elements all
  if (all && total > kCap) return gather_masked<TI>(xrow, sp, xbuf, v0, end, edges, k, sh);
  if (all) left = (1u << groups) - 1u;
  Candidates c{sh, 0, least};
  if (edges && tid < 64) {
    const int ek = edge_index<TI>(sp, tid);
    const float x = ek >= 0 ? TI::load1(xrow, ek) : kNegInf;
    c.add(ek >= 0 && (x >= least || all), element_key(x, static_cast<uint32_t>(ek)));
  }
  while (__any(left != 0)) {
    const bool mine = left != 0;
    const int g = __builtin_ctz(left | 1u << kGroups);
    left &= left - 1;
    for (int b = 0; b < batches; ++b) {
      const int at = v0 + (g * batches + b) * (kBlock * U) + tid;
      u32x4 x[U];
#pragma unroll
      for (int q = 0; q < U; ++q) x[q] = buf_ld16<false>(xbuf, mine ? static_cast<uint32_t>(at + q * kBlock) * 16u : 0u);
      uint32_t left_q = 0;
#pragma unroll
      for (int q = 0; q < U; ++q)
        left_q |= mine && at + q * kBlock < end && (vec_max<TI>(kNegInf, x[q]) >= least || all) ? 1u << q : 0u;
      take_vectors<TI>(c, x, left_q, static_cast<uint32_t>(sp.head + at * EPV), (1u << EPV) - 1u);
    }
  }
  __syncthreads();
  const int n = sh.count;
  __syncthreads();
  return n <= kCap ? n : select_exact<TI>(xrow, sp, xbuf, v0, end, edges, k, sh);
}

// The same for a part of one batch, which is still in x; lane_max: the lane's largest logit.
template <typename TI, int U>
__device__ __forceinline__ int gather_one(const char* xrow, const RowSpan& sp, __amdgpu_buffer_rsrc_t xbuf, int v0, int end,
                                          bool edges, int k, const u32x4 (&x)[U], float lane_max, Shared& sh) {
  constexpr int EPV = 16 / TI::kBytes;
  const int tid = threadIdx.x;
  float v[U];
#pragma unroll
  for (int q = 0; q < U; ++q) v[q] = v0 + q * kBlock + tid < end ? vec_max<TI>(kNegInf, x[q]) : kNegInf;
  const float own[1] = {lane_max};
  const float least = k <= 64 ? reached_by(sh, own, k) : reached_by(sh, v, k);
  if (tid == 0) sh.count = 0;
  __syncthreads();
  const int total = max(end - v0, 0) * EPV + (edges ? sp.head + sp.tail : 0);
  const bool all = least == kNegInf;
  if (all && total > kCap) return gather_masked<TI>(xrow, sp, xbuf, v0, end, edges, k, sh);
  Candidates c{sh, 0, least};
  if (edges && tid < 64) {
    const int ek = edge_index<TI>(sp, tid);
    const float e = ek >= 0 ? TI::load1(xrow, ek) : kNegInf;
    c.add(ek >= 0 && (e >= least || all), element_key(e, static_cast<uint32_t>(ek)));
  }
  uint32_t left_q = 0;
#pragma unroll
  for (int q = 0; q < U; ++q) left_q |= v0 + q * kBlock + tid < end && (v[q] >= least || all) ? 1u << q : 0u;
  take_vectors<TI>(c, x, left_q, static_cast<uint32_t>(sp.head + (v0 + tid) * EPV), (1u << EPV) - 1u);
  __syncthreads();
  const int n = sh.count;
  __syncthreads();
  return n <= kCap ? n : select_exact<TI>(xrow, sp, xbuf, v0, end, edges, k, sh);
}

// The merge of the first N lanes' sums, on every lane, in a fixed order.
template <int N>
__device__ __forceinline__ void score_merge(float& mx, double& s, double& t, float k) {
  const float M = lanes_max<N>(mx);
  score_rebase(s, t, mx, M, k);
  const int lane = threadIdx.x & 63;
  s = wave_sum64(lane < N ? s : 0.);
  t = wave_sum64(lane < N ? t : 0.);
  mx = M;
}

// ln s, s >= 1, to 2^-24 and near 1 to a few 2^-24 of itself: s = 2^k m with m in [1/sqrt 2, sqrt 2), of which f32 has the
// logarithm of the nearest f32 f, and (m - f) / f is added. f64's logarithm took 0.9 us more of the 30 of 1520 f16 rows of
// 50,257 with k = 8.
__device__ __forceinline__ double score_log(double s) {
  int k = __builtin_amdgcn_frexp_exp(s);
  double m = __builtin_amdgcn_frexp_mant(s);
  if (m < 0.70710678118654752440) {
    m += m;
    k -= 1;
  }
  const float f = static_cast<float>(m), rest = static_cast<float>(m - static_cast<double>(f));
  return static_cast<double>(k) * kLn2d + static_cast<double>(logf(f) + rest * __builtin_amdgcn_rcpf(f));
}

// A row's outputs: the alternatives by the threads that rank them, the rest by thread 0.
template <bool TOP>
__device__ __forceinline__ void score_write(const ScoreArgs& a, const ScoreRow& r, float token, Shared& sh, int n, float mx,
                                            double s, double t) {
  // The largest logit's own term is 1 and no exponent is above 0. Rounding misses either by 2^-24, and a row of one
  // likely token would have a positive log-prob and a negative entropy. (NaN, and a sum of 0, stay and are reported.)
  if (s > 0. && s < 1.) s = 1.;
  if (t > 0.) t = 0.;
  const double log_sum = score_log(s);
  auto log_p = [&](float x) {
    return static_cast<float>((static_cast<double>(x) - static_cast<double>(mx)) * a.inv_tau - log_sum);
  };
  if constexpr (TOP) {
    // (Sorted instead, 600 candidates of one row took 16 us more.)
    if (n > 2 * kBlock) n = Candidates{sh, 0, kNegInf}.thin(n, a.k, 2 * kBlock);
    rank_entries(sh, n, a.k, [&](int rank, float x, int64_t id) {
      const int64_t at = r.at * a.k + rank;
      a.top_logp[at] = log_p(x);
      if (a.top_i64) static_cast<int64_t*>(a.top_ids)[at] = id;
      else static_cast<int32_t*>(a.top_ids)[at] = static_cast<int32_t>(id);
    });
  }
  if (threadIdx.x != 0) return;
  if (!__builtin_isfinite(mx) || !__builtin_isfinite(log_sum)) raise_error(a.tok.err, kErrNonFinite);
  if (a.logp) a.logp[r.at] = r.id < 0 ? 0.f : log_p(token);
  if (a.entropy) a.entropy[r.at] = static_cast<float>(log_sum - t / s * kLn2d);
  if (a.row_max) a.row_max[r.at] = mx;
  if (a.log_sum) a.log_sum[r.at] = static_cast<float>(log_sum);
}

__device__ __forceinline__ void score_dead(const ScoreArgs& a, const ScoreRow& r) {
  for (int i = threadIdx.x; i < a.k; i += kBlock) {
    const int64_t at = r.at * a.k + i;
    a.top_logp[at] = 0.f;
    if (a.top_i64) static_cast<int64_t*>(a.top_ids)[at] = PCP_IGNORE_INDEX;
    else static_cast<int32_t*>(a.top_ids)[at] = PCP_IGNORE_INDEX;
  }
  if (threadIdx.x != 0) return;
  if (a.logp) a.logp[r.at] = 0.f;
  if (a.entropy) a.entropy[r.at] = 0.f;
  if (a.row_max) a.row_max[r.at] = 0.f;
  if (a.log_sum) a.log_sum[r.at] = 0.f;
}

// ONE: rows in parts of at most a batch each.
template <typename TI, bool TOP, bool ONE>
__global__ void __launch_bounds__(kBlock, 5) score_kernel(ScoreArgs a) {
  constexpr int BLOCK = kBlock, U = kU;
  __shared__ __align__(16) PartShared ps;
  Shared& sh = ps.sh;
  __shared__ double wave_s[kWaves], wave_t[kWaves];
  __shared__ float wave_mx[kWaves];
  __shared__ unsigned turn;
  __shared__ int counts[kScoreParts];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t of = blockIdx.x / static_cast<uint32_t>(a.parts);
  const int part = static_cast<int>(blockIdx.x - of * static_cast<uint32_t>(a.parts));
  const int64_t row = a.row0 + of;
  const int64_t seq = static_cast<uint32_t>(row) / static_cast<uint32_t>(a.tok.rows);
  const int64_t t = row - seq * a.tok.rows;
  const ScoreRow r = score_row(a.tok, seq, t);
  if (!r.live) {
    if (part == 0) score_dead(a, r);
    return;
  }
  const char* xrow = static_cast<const char*>(a.logits) + (seq * a.seq_stride + t * a.row_stride) * TI::kBytes;
  const RowSpan sp = row_span<TI>(xrow, a.tok.vocab);
  const int v0 = part * a.per, end = min(v0 + a.per, sp.nv);
  const __amdgpu_buffer_rsrc_t xbuf = row_rsrc(sp.vec, static_cast<uint32_t>(max(end, 0)) * 16u);
  ScoreSums sums{a.k2, kNegInf, 0., 0., false};
  const float token = r.id >= 0 ? TI::load1(xrow, r.id) : 0.f;   // (ahead of the row: nothing waits for it at the end)
  if (part == 0 && tid < 64) {   // the elements outside the interior
    const int ek = edge_index<TI>(sp, tid);
    if (ek >= 0) {
      sums.mx = fmaxf(sums.mx, TI::load1(xrow, ek));
      sums.s = hw_exp2((TI::load1(xrow, ek) - ms_ref(sums.mx)) * a.k2);
    }
  }
  u32x4 x[U];
  float bx = kNegInf, group = kNegInf;
  int b = 0;
  auto load = [&](u32x4 (&to)[U], int base) {
    const uint32_t off = static_cast<uint32_t>(base + tid) * 16u;
#pragma unroll
    for (int q = 0; q < U; ++q) to[q] = buf_ld16<true>(xbuf, off + q * (BLOCK * 16u));
  };
  auto batch = [&](auto held) {
    bx = batch_max<TI>(x, held);
    sums.template add<TI>(x, held, bx);
    if constexpr (TOP && !ONE) {
      group = b % a.group == 0 ? bx : fmaxf(group, bx);
      ps.group[b / a.group][tid] = group;
      ++b;
    }
  };
  // Whole batches without a test for each vector, then what is left; the next batch's loads go out ahead.
  int base = v0;
  if (base < end || ONE) load(x, base);
  if constexpr (!ONE)
    for (; base + BLOCK * U <= end; base += BLOCK * U) {
      u32x4 next[U];
      load(next, base + BLOCK * U);
      batch([](int) { return true; });
#pragma unroll
      for (int q = 0; q < U; ++q) x[q] = next[q];
    }
  if (base < end || ONE) batch([&](int q) { return base + q * BLOCK + tid < end; });
  float mx = sums.mx;
  double s = sums.s, tt = sums.t;
  score_merge<64>(mx, s, tt, a.k2);
  if (lane == 0) {
    wave_mx[wave] = mx;
    wave_s[wave] = s;
    wave_t[wave] = tt;
  }
  __syncthreads();
  mx = wave_mx[lane & (kWaves - 1)];
  s = wave_s[lane & (kWaves - 1)];
  tt = wave_t[lane & (kWaves - 1)];
  score_merge<kWaves>(mx, s, tt, a.k2);
  int n = 0;
  if constexpr (TOP && ONE) n = gather_one<TI>(xrow, sp, xbuf, v0, end, part == 0, a.k, x, bx, sh);
  else if constexpr (TOP)
    n = gather_top<TI>(xrow, sp, xbuf, v0, end, part == 0, a.k, a.group, (b + a.group - 1) / a.group, ps);
  if (a.parts == 1) {
    score_write<TOP>(a, r, token, sh, n, mx, s, tt);
    return;
  }
  if constexpr (TOP)
    if (n > a.part_cap) n = Candidates{sh, 0, kNegInf}.thin(n, a.k, a.part_cap);
  // The part's candidates and sums for the last of the row's workgroups to finish, which merges them.
  ScorePart* parts = a.part + static_cast<int64_t>(of) * a.parts;
  uint64_t* keys = a.part_key + static_cast<int64_t>(of) * a.parts * a.part_cap;
  if constexpr (TOP)
    for (int i = tid; i < n; i += BLOCK) store_coherent(keys + static_cast<int64_t>(part) * a.part_cap + i, sh.key[i]);
  if (tid == 0) {
    store_coherent(&parts[part].s, s);
    store_coherent(&parts[part].t, tt);
    store_coherent(&parts[part].mx, mx);
    store_coherent(&parts[part].n, n);
  }
  wait_stores();
  __syncthreads();
  if (tid == 0) turn = __hip_atomic_fetch_add(a.done + of, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (turn + 1 != static_cast<unsigned>(a.parts)) return;
  if (tid == 0) store_coherent(a.done + of, 0u);
  // Read at the level that the stores went to, past the caches, which then need no invalidation (an XCD's whole L2,
  // for every row: 400 rows of 50,257 in four parts each took 50 us instead of 16).
  const __amdgpu_buffer_rsrc_t pbuf = row_rsrc(parts, static_cast<uint32_t>(a.parts) * sizeof(ScorePart));
  const __amdgpu_buffer_rsrc_t kbuf = row_rsrc(keys, static_cast<uint32_t>(a.parts * a.part_cap) * 8u);
  auto key_at = [&](int i) { return buf_ld8_coherent(kbuf, static_cast<uint32_t>(i) * 8u); };
  // Few slots are read along with the parts' counts, whatever they hold.
  constexpr int R = 4;
  const int slots = TOP ? a.parts * a.part_cap : 0;
  uint64_t key[R] = {};
  if (TOP && slots <= R * BLOCK) {
#pragma unroll
    for (int q = 0; q < R; ++q) key[q] = key_at(q * BLOCK + tid);   // (past the last: 0)
  }
  const u32x4 p0 = buf_ld16_coherent(pbuf, lane * sizeof(ScorePart));
  const u32x4 p1 = buf_ld16_coherent(pbuf, lane * sizeof(ScorePart) + 16);
  const bool is = lane < a.parts;
  s = is ? __builtin_bit_cast(double, static_cast<uint64_t>(p0[1]) << 32 | p0[0]) : 0.;
  tt = is ? __builtin_bit_cast(double, static_cast<uint64_t>(p0[3]) << 32 | p0[2]) : 0.;
  mx = is ? __uint_as_float(p1[0]) : kNegInf;
  if constexpr (TOP) {
    const int left = is ? static_cast<int>(p1[1]) : 0;
    if (tid < 64) counts[tid] = left;
    if (slots <= R * BLOCK) {
      __syncthreads();
      float v[R];
#pragma unroll
      for (int q = 0; q < R; ++q) {
        const int at = q * BLOCK + tid, p = at / a.part_cap;
        key[q] = at < slots && at - p * a.part_cap < counts[p] ? key[q] : 0;   // no key is 0
        v[q] = key[q] ? from_order(static_cast<uint32_t>(key[q] >> 32)) : kNegInf;
      }
      Candidates c{sh, 0, reached_by(sh, v, a.k, (slots + BLOCK - 1) / BLOCK)};
      if (tid == 0) sh.count = 0;
      __syncthreads();
#pragma unroll
      for (int q = 0; q < R; ++q)
        if (q * BLOCK < slots) c.add(key[q] != 0 && (v[q] >= c.least_x || c.least_x == kNegInf), key[q]);
      __syncthreads();
      n = sh.count;
      __syncthreads();
    } else {
      n = merge_parts(key_at, a.parts, a.part_cap, a.k, [&](int p) { return counts[p]; }, sh);
    }
  }
  score_merge<64>(mx, s, tt, a.k2);
  score_write<TOP>(a, r, token, sh, n, mx, s, tt);
}

template <typename TI>
hipError_t launch_score(ScoreArgs a, int64_t n_rows, hipStream_t st) {
  constexpr int64_t kRows = 1 << 22;   // of a launch: 2^30 lanes, and rows in parts are fewer
  for (int64_t r0 = 0; r0 < n_rows; r0 += kRows) {
    a.row0 = r0;
    const unsigned grid = static_cast<unsigned>((n_rows - r0 < kRows ? n_rows - r0 : kRows) * a.parts);
    const bool one = a.parts > 1 && a.per <= kBlock * kU;
    if (a.k > 0 && one) score_kernel<TI, true, true><<<grid, kBlock, 0, st>>>(a);
    else if (a.k > 0) score_kernel<TI, true, false><<<grid, kBlock, 0, st>>>(a);
    else if (one) score_kernel<TI, false, true><<<grid, kBlock, 0, st>>>(a);
    else score_kernel<TI, false, false><<<grid, kBlock, 0, st>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

// ---- backward ---------------------------------------------------------------------------

struct ScoreBwdArgs {
  TokenArrays tok;
  const void* logits;
  void* dlogits;
  int64_t row_stride, seq_stride, drow_stride, dseq_stride, logit_rows;
  int64_t row0;
  const float* row_max;
  const float* log_sum;
  const float* entropy;
  const float* dlogp;
  const float* dentropy;
  float k2, inv_tau;
  int32_t blocks;          // workgroups per row
};

// 16 bytes of dlogits each: the logits of the same elements (16 or 8 bytes) at any element's address.
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef u32x2 u32x2_any __attribute__((aligned(2)));

// Groups per lane: 16 bytes of dlogits each, so that 16-bit logits of f32 dlogits come 8 bytes a group. us with 1 | 2 | 4, 5/8
// of the rows live:
//   bf16 -> f32, 2048 rows of 50,257   142 | 112 | 104        f32 -> f32, 1024 rows of 151,936   209 | 169 | 176
//   bf16 -> bf16, 4096 rows of 151,936 466 | 349 | 347, added 427 | 384 | 410
template <typename TI, typename TO>
constexpr int grad_unroll() { return TI::kBytes == 2 && TO::kBytes == 4 ? 4 : 2; }

// Stores at system scope (sc0 sc1), which suit the whole-model updates, took as long here and, on rows off 16 bytes, 87 us
// for 68. A row's gradient is one pass: dz = p (A + B d) with d = (x - m) k2 - log2 sum, p = 2^d, and the token's
// own term.
template <typename TI, typename TO, bool ACC>
__global__ void __launch_bounds__(kBlock) score_grad_kernel(ScoreBwdArgs a) {
  constexpr int N = 16 / TO::kBytes, U = grad_unroll<TI, TO>();   // elements per group
  const int tid = threadIdx.x;
  const uint32_t of = blockIdx.x / static_cast<uint32_t>(a.blocks);
  const int block = static_cast<int>(blockIdx.x - of * static_cast<uint32_t>(a.blocks));
  const int64_t row = a.row0 + of;
  const int64_t seq = static_cast<uint32_t>(row) / static_cast<uint32_t>(a.logit_rows);
  const int64_t t = row - seq * a.logit_rows;
  ScoreRow r{0, -1, false};
  if (t < a.tok.rows) r = score_row(a.tok, seq, t);
  float gl = 0.f, gh = 0.f;
  if (r.live) {
    if (a.dlogp) gl = a.dlogp[r.at];
    if (a.dentropy) gh = a.dentropy[r.at];
    r.live = gl != 0.f || gh != 0.f;
  }
  if (ACC && !r.live) return;
  char* drow = static_cast<char*>(a.dlogits) + (seq * a.dseq_stride + t * a.drow_stride) * TO::kBytes;
  const int V = static_cast<int>(a.tok.vocab);
  // Group g: elements first + N g on, 16-byte aligned in dlogits; the first and the last may be cut.
  const int first = -static_cast<int>((reinterpret_cast<uintptr_t>(drow) & 15u) / TO::kBytes);
  const int e0 = first + (block * (U * kBlock) + tid) * N;
  if (!r.live) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int e = e0 + u * (kBlock * N);
      if (e >= 0 && e + N <= V) {
        __builtin_nontemporal_store(u32x4{0, 0, 0, 0}, reinterpret_cast<u32x4*>(drow + static_cast<int64_t>(e) * TO::kBytes));
      } else {
        for (int j = max(-e, 0); j < min(N, V - e); ++j) store1<TO>(drow, e + j, 0.f);
      }
    }
    return;
  }
  const char* xrow = static_cast<const char*>(a.logits) + (seq * a.seq_stride + t * a.row_stride) * TI::kBytes;
  const float m = a.row_max[r.at], ls = a.log_sum[r.at], h = a.dentropy ? a.entropy[r.at] : 0.f;
  const float l2 = ls * kLog2e;
  float A = -fmaf(gh, h, gl) * a.inv_tau;
  const float B = -gh * kLn2 * a.inv_tau, at_token = gl * a.inv_tau;
  if (!__builtin_isfinite(m) || !__builtin_isfinite(ls) || !__builtin_isfinite(A) || !__builtin_isfinite(B)) {
    A = __builtin_nanf("");
    if (tid == 0 && block == 0) raise_error(a.tok.err, kErrNonFinite);
  }
  const int y = static_cast<int>(r.id);
  auto grad = [&](float x, int e) {
    const float d = fmaxf(fmaf(x - m, a.k2, -l2), kLeastExp);
    const float g = hw_exp2(d) * fmaf(B, d, A);
    return e == y ? g + at_token : g;
  };
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int e = e0 + u * (kBlock * N);
    const char* xp = xrow + static_cast<int64_t>(e) * TI::kBytes;
    u32x4* dp = reinterpret_cast<u32x4*>(drow + static_cast<int64_t>(e) * TO::kBytes);
    if (e >= 0 && e + N <= V) {
      uint32_t w[4] = {}, b[4] = {};
      if constexpr (N * TI::kBytes == 16) {
        const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(xp));
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = v[i];
      } else {
        const u32x2 v = __builtin_nontemporal_load(reinterpret_cast<const u32x2_any*>(xp));
        w[0] = v[0];
        w[1] = v[1];
      }
      if constexpr (ACC) {
        const u32x4 v = __builtin_nontemporal_load(dp);
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = v[i];
      }
      float o[N];
#pragma unroll
      for (int j = 0; j < N; ++j) {
        o[j] = grad(TI::unpack(w, j), e + j);
        if constexpr (ACC) o[j] += TO::unpack(b, j);
      }
      store_vals<TO, N, true>(dp, 0, o);
    } else {
      for (int j = max(-e, 0); j < min(N, V - e); ++j) {
        float o = grad(TI::load1(xrow, e + j), e + j);
        if constexpr (ACC) o += TO::load1(drow, e + j);
        store1<TO>(drow, e + j, o);
      }
    }
  }
}

template <typename TI, typename TO>
hipError_t launch_grad(ScoreBwdArgs a, int64_t n_rows, bool accumulate, hipStream_t st) {
  constexpr int N = 16 / TO::kBytes, U = grad_unroll<TI, TO>();
  // The groups of a row that begins up to N - 1 elements past an aligned address.
  const int64_t groups = (a.tok.vocab + N - 1 + N - 1) / N;
  a.blocks = static_cast<int32_t>((groups + kBlock * U - 1) / (kBlock * U));
  const int64_t rows = (int64_t(1) << 23) / a.blocks > 0 ? (int64_t(1) << 23) / a.blocks : 1;   // of a launch
  for (int64_t r0 = 0; r0 < n_rows; r0 += rows) {
    a.row0 = r0;
    const unsigned grid = static_cast<unsigned>((n_rows - r0 < rows ? n_rows - r0 : rows) * a.blocks);
    if (accumulate) score_grad_kernel<TI, TO, true><<<grid, kBlock, 0, st>>>(a);
    else score_grad_kernel<TI, TO, false><<<grid, kBlock, 0, st>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

// ---- entry points -----------------------------------------------------------------------

inline bool misaligned(const void* p, int size) {
  return (reinterpret_cast<uintptr_t>(p) & static_cast<uintptr_t>(size - 1)) != 0;
}

// Elements from the first to past the last of n_seq x rows rows (0 where there are none);
// false where that overflows.
bool extent_of(int64_t n_seq, int64_t rows, int64_t row_stride, int64_t seq_stride, int64_t vocab, int64_t* out) {
  *out = 0;
  if (n_seq == 0 || rows == 0) return true;
  int64_t a, b, bytes;
  if (mul_overflows(n_seq - 1, seq_stride, &a) || mul_overflows(rows - 1, row_stride, &b) ||
      __builtin_add_overflow(a, b, &a) || __builtin_add_overflow(a, vocab, &a) || mul_overflows(a, 8, &bytes))
    return false;
  *out = a;
  return true;
}

// What both calls check alike, and the token arrays that follow from it.
template <typename Args>
int score_common(pcp_ctx* ctx, const Args* a, TokenArrays* tok, float* k2) {
  if (a->n_seq < 0) return fail(ctx, PCP_ERR_INVALID_ARG, "n_seq must be >= 0 (got %lld)", (long long)a->n_seq);
  if (a->rows < 0) return fail(ctx, PCP_ERR_INVALID_ARG, "rows must be >= 0 (got %lld)", (long long)a->rows);
  if (a->vocab < 1 || a->vocab > PCP_SCORE_MAX_VOCAB)
    return fail(ctx, PCP_ERR_INVALID_ARG, "vocab must be in [1, %d] (got %lld)", PCP_SCORE_MAX_VOCAB, (long long)a->vocab);
  if (a->logits_dtype != PCP_BF16 && a->logits_dtype != PCP_F16 && a->logits_dtype != PCP_F32)
    return fail(ctx, PCP_ERR_DTYPE, "logits dtype must be bf16, f16 or f32 (got %d)", a->logits_dtype);
  if (a->ids && a->ids_dtype != PCP_I64 && a->ids_dtype != PCP_I32)
    return fail(ctx, PCP_ERR_DTYPE, "ids dtype must be i64 or i32 (got %d)", a->ids_dtype);
  if (a->mask && a->mask_dtype != PCP_F32 && a->mask_dtype != PCP_BOOL)
    return fail(ctx, PCP_ERR_DTYPE, "mask dtype must be f32 or bool (got %d)", a->mask_dtype);
  *k2 = static_cast<float>(1.4426950408889634074 / static_cast<double>(a->temperature));
  if (!(a->temperature > 0.f) || !std::isfinite(a->temperature) || !std::isnormal(*k2))
    return fail(ctx, PCP_ERR_INVALID_ARG, "temperature must be positive and finite (and its inverse a normal f32)");
  if (a->flags & ~PCP_FLAG_ASYNC) return fail(ctx, PCP_ERR_INVALID_ARG, "only PCP_FLAG_ASYNC applies here");
  const int64_t ts = a->tok_seq_stride ? a->tok_seq_stride : a->rows;
  if (a->tok_offset < 0 || a->rows > ts || a->tok_offset > ts - a->rows)
    return fail(ctx, PCP_ERR_INVALID_ARG, "tok_offset + rows must fit in tok_seq_stride");
  int64_t tmp;
  if (mul_overflows(a->n_seq, ts, &tmp) || mul_overflows(tmp, 8 * PCP_SCORE_TOP_MAX, &tmp))
    return fail(ctx, PCP_ERR_OVERFLOW, "token array size overflows int64");
  if (misaligned(a->logits, dtype_bytes(a->logits_dtype)) || (a->ids && misaligned(a->ids, dtype_bytes(a->ids_dtype))) ||
      (a->mask && a->mask_dtype == PCP_F32 && misaligned(a->mask, 4)))
    return fail(ctx, PCP_ERR_INVALID_ARG, "pointers must be aligned to their element size");
  *tok = TokenArrays{a->ids, a->mask, a->rows, ts, a->tok_offset, a->vocab, nullptr, a->ids_dtype == PCP_I64,
                     a->mask_dtype == PCP_BOOL};
  return PCP_OK;
}

int score_fwd(pcp_ctx* ctx, const pcp_score_args* a) {
  if (!a) return fail(ctx, PCP_ERR_INVALID_ARG, "args is NULL");
  ScoreArgs t;
  std::memset(&t, 0, sizeof(t));
  const int rc0 = score_common(ctx, a, &t.tok, &t.k2);
  if (rc0 != PCP_OK) return rc0;
  if (a->k < 0 || a->k > PCP_SCORE_TOP_MAX || a->k > a->vocab)
    return fail(ctx, PCP_ERR_INVALID_ARG, "k must be in [0, min(vocab, %d)] (got %d)", PCP_SCORE_TOP_MAX, a->k);
  t.row_stride = a->row_stride ? a->row_stride : a->vocab;
  if (t.row_stride < a->vocab)
    return fail(ctx, PCP_ERR_INVALID_ARG, "row_stride (%lld) must be >= vocab", (long long)t.row_stride);
  int64_t n_rows, extent;
  if (mul_overflows(a->n_seq, a->rows, &n_rows) || n_rows > INT32_MAX)
    return fail(ctx, PCP_ERR_OVERFLOW, "n_seq * rows exceeds 2^31-1 rows");
  if (a->seq_stride) t.seq_stride = a->seq_stride;
  else if (mul_overflows(a->rows, t.row_stride, &t.seq_stride))
    return fail(ctx, PCP_ERR_OVERFLOW, "logits byte size overflows int64");
  if (a->n_seq > 1 && a->rows > 0 && t.seq_stride < a->vocab)
    return fail(ctx, PCP_ERR_INVALID_ARG, "seq_stride (%lld) must be >= vocab", (long long)t.seq_stride);
  if (!extent_of(a->n_seq, a->rows, t.row_stride, t.seq_stride, a->vocab, &extent))
    return fail(ctx, PCP_ERR_OVERFLOW, "logits byte size overflows int64");
  if (a->k > 0 && a->top_ids_dtype != PCP_I64 && a->top_ids_dtype != PCP_I32)
    return fail(ctx, PCP_ERR_DTYPE, "top_ids dtype must be i64 or i32 (got %d)", a->top_ids_dtype);
  if (n_rows > 0 && (!a->logits || (a->k > 0 && (!a->top_logp || !a->top_ids))))
    return fail(ctx, PCP_ERR_INVALID_ARG, "logits, or top_logp / top_ids with k > 0, is NULL");
  if (!a->ids && a->logp) return fail(ctx, PCP_ERR_INVALID_ARG, "logp needs ids");
  if (misaligned(a->logp, 4) || misaligned(a->entropy, 4) || misaligned(a->row_max, 4) || misaligned(a->log_sum, 4) ||
      (a->k > 0 && (misaligned(a->top_logp, 4) || misaligned(a->top_ids, dtype_bytes(a->top_ids_dtype)))))
    return fail(ctx, PCP_ERR_INVALID_ARG, "pointers must be aligned to their element size");
  if (!ctx) return fail(nullptr, PCP_ERR_INVALID_ARG, "context is NULL");
  if (n_rows == 0) return PCP_OK;
  const DeviceScope scope(ctx->device);
  if (scope.error() != hipSuccess) return hip_fail(ctx, scope.error(), "making the context's device current");
  hipStream_t st = static_cast<hipStream_t>(a->stream);

  const ScoreSplit split = score_split(n_rows, a->vocab, dtype_bytes(a->logits_dtype));
  const int64_t parts = split.parts;
  const int64_t part_cap = a->k > 0 ? a->k + 16 + a->k / 4 : 0;   // a part seldom has more, and is thinned then
  const size_t keys = parts > 1 ? sizeof(uint64_t) * static_cast<size_t>(n_rows) * parts * part_cap : 0;
  const size_t sums = parts > 1 ? sizeof(ScorePart) * static_cast<size_t>(n_rows) * parts + 16 : 0;
  if (parts > 1) {
    const int rc = ensure_scratch_on(ctx, keys + sums, st);
    if (rc != PCP_OK) return rc;
  }
  t.tok.err = ctx->d_page->err;
  t.logits = a->logits;
  t.logp = a->logp;
  t.entropy = a->entropy;
  t.row_max = a->row_max;
  t.log_sum = a->log_sum;
  t.top_logp = a->top_logp;
  t.top_ids = a->top_ids;
  t.part_key = static_cast<uint64_t*>(ctx->scratch);
  t.part = reinterpret_cast<ScorePart*>(static_cast<char*>(ctx->scratch) + ((keys + 15) & ~static_cast<size_t>(15)));
  t.done = ctx->d_score_done;
  t.inv_tau = 1. / static_cast<double>(a->temperature);
  t.k = a->k;
  t.top_i64 = a->top_ids_dtype == PCP_I64;
  t.parts = static_cast<int32_t>(parts);
  t.per = static_cast<int32_t>(split.per);
  t.part_cap = static_cast<int32_t>(part_cap);
  t.group = split.group;
  const bool timed = prof_begin(ctx, st);
  const hipError_t e = a->logits_dtype == PCP_F32    ? launch_score<F32T>(t, n_rows, st)
                       : a->logits_dtype == PCP_BF16 ? launch_score<BF16T>(t, n_rows, st)
                                                     : launch_score<F16T>(t, n_rows, st);
  prof_end(ctx, st, timed);
  if (e != hipSuccess) return hip_fail(ctx, e, "token scores launch");
  return finish_call(ctx, a->flags, st);
}

int score_bwd(pcp_ctx* ctx, const pcp_score_bwd_args* a) {
  if (!a) return fail(ctx, PCP_ERR_INVALID_ARG, "args is NULL");
  ScoreBwdArgs t;
  std::memset(&t, 0, sizeof(t));
  const int rc0 = score_common(ctx, a, &t.tok, &t.k2);
  if (rc0 != PCP_OK) return rc0;
  if (a->dlogits_dtype != a->logits_dtype && a->dlogits_dtype != PCP_F32)
    return fail(ctx, PCP_ERR_DTYPE, "dlogits dtype must equal the logits dtype or be f32");
  t.logit_rows = a->logit_rows ? a->logit_rows : a->rows;
  if (t.logit_rows < a->rows)
    return fail(ctx, PCP_ERR_INVALID_ARG, "logit_rows (%lld) must be >= rows", (long long)a->logit_rows);
  t.row_stride = a->row_stride ? a->row_stride : a->vocab;
  t.drow_stride = a->drow_stride ? a->drow_stride : a->vocab;
  if (t.row_stride < a->vocab || t.drow_stride < a->vocab)
    return fail(ctx, PCP_ERR_INVALID_ARG, "row_stride and drow_stride must be >= vocab");
  int64_t n_rows, extent, dextent;
  if (mul_overflows(a->n_seq, t.logit_rows, &n_rows) || n_rows > INT32_MAX)
    return fail(ctx, PCP_ERR_OVERFLOW, "n_seq * logit_rows exceeds 2^31-1 rows");
  t.seq_stride = a->seq_stride;
  t.dseq_stride = a->dseq_stride;
  if ((!a->seq_stride && mul_overflows(t.logit_rows, t.row_stride, &t.seq_stride)) ||
      (!a->dseq_stride && mul_overflows(t.logit_rows, t.drow_stride, &t.dseq_stride)))
    return fail(ctx, PCP_ERR_OVERFLOW, "logits byte size overflows int64");
  if (a->n_seq > 1 && n_rows > 0 && (t.seq_stride < a->vocab || t.dseq_stride < a->vocab))
    return fail(ctx, PCP_ERR_INVALID_ARG, "seq_stride and dseq_stride must be >= vocab");
  if (!extent_of(a->n_seq, a->rows, t.row_stride, t.seq_stride, a->vocab, &extent) ||
      !extent_of(a->n_seq, t.logit_rows, t.drow_stride, t.dseq_stride, a->vocab, &dextent))
    return fail(ctx, PCP_ERR_OVERFLOW, "logits byte size overflows int64");
  {
    // Rows of dlogits apart: sequences after one another, or row by row beside one another.
    int64_t one = 0, all = 0;
    (void)extent_of(1, t.logit_rows, t.drow_stride, t.dseq_stride, a->vocab, &one);
    (void)extent_of(a->n_seq, 1, t.drow_stride, t.dseq_stride, a->vocab, &all);
    if (a->n_seq > 1 && t.logit_rows > 1 && t.dseq_stride < one && t.drow_stride < all)
      return fail(ctx, PCP_ERR_INVALID_ARG, "rows of dlogits overlap");
  }
  if (n_rows > 0 && !a->dlogits) return fail(ctx, PCP_ERR_INVALID_ARG, "dlogits is NULL");
  if (extent > 0 && (!a->logits || !a->row_max || !a->log_sum))
    return fail(ctx, PCP_ERR_INVALID_ARG, "logits / row_max / log_sum is NULL");
  if (a->dlogp && !a->ids) return fail(ctx, PCP_ERR_INVALID_ARG, "dlogp needs ids");
  if (a->dentropy && !a->entropy) return fail(ctx, PCP_ERR_INVALID_ARG, "dentropy needs the forward's entropy");
  if (misaligned(a->dlogits, dtype_bytes(a->dlogits_dtype)) || misaligned(a->row_max, 4) || misaligned(a->log_sum, 4) ||
      misaligned(a->entropy, 4) || misaligned(a->dlogp, 4) || misaligned(a->dentropy, 4))
    return fail(ctx, PCP_ERR_INVALID_ARG, "pointers must be aligned to their element size");
  {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a->logits), d = reinterpret_cast<uintptr_t>(a->dlogits);
    const uintptr_t xn = static_cast<uintptr_t>(extent) * dtype_bytes(a->logits_dtype);
    const uintptr_t dn = static_cast<uintptr_t>(dextent) * dtype_bytes(a->dlogits_dtype);
    const bool same = x == d && a->logits_dtype == a->dlogits_dtype && t.row_stride == t.drow_stride &&
                      t.seq_stride == t.dseq_stride;
    if (extent > 0 && !same && x < d + dn && d < x + xn)
      return fail(ctx, PCP_ERR_INVALID_ARG, "dlogits overlap the logits without being the same rows");
  }
  if (!ctx) return fail(nullptr, PCP_ERR_INVALID_ARG, "context is NULL");
  if (n_rows == 0) return PCP_OK;
  const DeviceScope scope(ctx->device);
  if (scope.error() != hipSuccess) return hip_fail(ctx, scope.error(), "making the context's device current");
  hipStream_t st = static_cast<hipStream_t>(a->stream);
  t.tok.err = ctx->d_page->err;
  t.logits = a->logits;
  t.dlogits = a->dlogits;
  t.row_max = a->row_max;
  t.log_sum = a->log_sum;
  t.entropy = a->entropy;
  t.dlogp = a->dlogp;
  t.dentropy = a->dentropy;
  t.inv_tau = static_cast<float>(1. / static_cast<double>(a->temperature));
  const bool acc = a->accumulate != 0, wide = a->dlogits_dtype == PCP_F32;
  const bool timed = prof_begin(ctx, st);
  const hipError_t e = a->logits_dtype == PCP_F32 ? launch_grad<F32T, F32T>(t, n_rows, acc, st)
                       : a->logits_dtype == PCP_BF16
                           ? (wide ? launch_grad<BF16T, F32T>(t, n_rows, acc, st) : launch_grad<BF16T, BF16T>(t, n_rows, acc, st))
                           : (wide ? launch_grad<F16T, F32T>(t, n_rows, acc, st) : launch_grad<F16T, F16T>(t, n_rows, acc, st));
  prof_end(ctx, st, timed);
  if (e != hipSuccess) return hip_fail(ctx, e, "token scores' gradient launch");
  return finish_call(ctx, a->flags, st);
}

}  // namespace
}  // namespace pcp

using namespace pcp;

extern "C" {

void pcp_score_args_init(pcp_score_args* a) {
  if (!a) return;
  std::memset(a, 0, sizeof(*a));
  a->logits_dtype = PCP_BF16;
  a->ids_dtype = PCP_I64;
  a->mask_dtype = PCP_F32;
  a->top_ids_dtype = PCP_I32;
  a->temperature = 1.f;
}

int pcp_score_fwd(pcp_ctx* ctx, const pcp_score_args* a) { return score_fwd(ctx, a); }

void pcp_score_bwd_args_init(pcp_score_bwd_args* a) {
  if (!a) return;
  std::memset(a, 0, sizeof(*a));
  a->logits_dtype = a->dlogits_dtype = PCP_BF16;
  a->ids_dtype = PCP_I64;
  a->mask_dtype = PCP_F32;
  a->temperature = 1.f;
}

int pcp_score_bwd(pcp_ctx* ctx, const pcp_score_bwd_args* a) { return score_bwd(ctx, a); }

}  // extern "C"
