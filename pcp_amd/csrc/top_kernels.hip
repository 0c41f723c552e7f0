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

namespace pcp {
namespace {

constexpr int kBlock = 256;
constexpr int kWaves = kBlock / 64;
constexpr int kU = 8;              // 16-byte vectors per lane and batch
constexpr int kCap = 2048;         // candidates held
constexpr int kCut = 1024;         // thinned past this many: a cautious round adds at most kCap - kCut
constexpr int kBins = 256;
// A logit this low is a mask (-inf, or a type's lowest value): it stays out of the histograms,
// whose range it would take up.
constexpr float kMasked = -32768.f;

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

struct Shared {
  uint64_t key[kCap];
  int bin[kBins];
  float low[kWaves], high[kWaves];
  int count;
};

__device__ __forceinline__ float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }

// Inclusive sum over the lanes up to this one.
__device__ __forceinline__ int lanes_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return v;
}

// A value that at least k of the workgroup's values v[] reach, and not many more unless they
// lie close together: the lower edge of a bin of a histogram over their range; -inf where
// fewer than k lie above kMasked. Called by the whole workgroup; sh.bin is free again after
// the caller's next barrier.
// used: the values past this many of v are no one's.
template <int M>
__device__ __forceinline__ float reached_by(Shared& sh, const float (&v)[M], int k, int used = M) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float lo = __builtin_inff(), hi = kNegInf;
#pragma unroll
  for (int i = 0; i < M; ++i) {
    if (i >= used) break;
    const bool plain = v[i] > kMasked && v[i] < __builtin_inff();
    lo = plain ? fminf(lo, v[i]) : lo;
    hi = plain ? fmaxf(hi, v[i]) : hi;
  }
  lo = -lanes_max<64>(-lo);
  hi = lanes_max<64>(hi);
  if (lane == 0) {
    sh.low[wave] = lo;
    sh.high[wave] = hi;
  }
  for (int i = threadIdx.x; i < kBins; i += kBlock) sh.bin[i] = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    lo = fminf(lo, sh.low[w]);
    hi = fmaxf(hi, sh.high[w]);
  }
  const float range = hi - lo;
  const float scale = range > 0.f && range < __builtin_inff() ? (kBins - 1) / range : 0.f;
#pragma unroll
  for (int i = 0; i < M; ++i)
    if (i < used && v[i] >= lo)   // +inf counts in the last bin
      atomicAdd(&sh.bin[v[i] > hi ? kBins - 1 : min(static_cast<int>((v[i] - lo) * scale), kBins - 1)], 1);
  __syncthreads();
  // Lane l: the bins 4 (63 - l) .. + 3, from the last bin down.
  const int first = 4 * (63 - lane);
  const int4 c = *reinterpret_cast<const int4*>(&sh.bin[first]);
  const int incl = lanes_scan(c.x + c.y + c.z + c.w);
  const uint64_t enough = __ballot(incl >= k);
  if (enough == 0) return kNegInf;
  const int above = incl - (c.x + c.y + c.z + c.w);
  int at = first;
  if (above + c.w >= k) at = first + 3;
  else if (above + c.w + c.z >= k) at = first + 2;
  else if (above + c.w + c.z + c.y >= k) at = first + 1;
  at = __builtin_amdgcn_readlane(at, __builtin_ctzll(enough));
  // Below the edge by more than the rounding of the bins' arithmetic.
  return at == 0 || scale == 0.f ? lo : lo + (at / scale - 0x1p-20f * (fabsf(lo) + fabsf(hi)));
}

struct Candidates {
  Shared& sh;
  uint64_t least;      // keys above this pass (0: all)
  float least_x;       // no element below this passes

  // Called by every lane of a wave.
  __device__ __forceinline__ void add(bool pass, uint64_t k) {
    const uint64_t who = __ballot(pass);
    if (who == 0) return;
    const int before = __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(who >> 32),
                                                 __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(who), 0));
    // One lane adds for all; the offset that the compiler cannot see through keeps it from
    // wrapping the single atomic in a reduction of its own.
    int at = 0, zero = 0;
    asm volatile("" : "+v"(zero));
    if (before == 0 && pass) at = atomicAdd(&sh.count + zero, __popcll(who));
    at = __builtin_amdgcn_readlane(at, __builtin_ctzll(who)) + before;
    if (pass && at < kCap) sh.key[at] = k;
  }
  // The n candidates held become those of the k largest, and few more: at most `most` (>= k).
  // Called by the whole workgroup after a barrier; ends with one.
  __device__ __forceinline__ int thin(int n, int k, int most) {
    constexpr int M = kCap / kBlock;
    uint64_t key[M];
    float v[M];
#pragma unroll
    for (int i = 0; i < M; ++i) {
      key[i] = 0;
      v[i] = kNegInf;
      if (i * kBlock < n) {
        const int at = i * kBlock + static_cast<int>(threadIdx.x);
        if (at < n) {
          key[i] = sh.key[at];
          v[i] = from_order(static_cast<uint32_t>(key[i] >> 32));
        }
      }
    }
    const float x = reached_by(sh, v, k, (n + kBlock - 1) / kBlock);
    least_x = fmaxf(least_x, x);
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < M; ++i)
      if (i * kBlock < n) add(i * kBlock + static_cast<int>(threadIdx.x) < n && !(v[i] < x), key[i]);
    __syncthreads();
    n = sh.count;
    if (n > most) {   // too many near the k-th: exactly
      sort_falling(sh.key, n);
      least = sh.key[k - 1] - 1;   // the k-th itself is held already, and no other key equals it
      n = k;
      __syncthreads();
      if (threadIdx.x == 0) sh.count = k;
    }
    __syncthreads();
    return n;
  }
};

// A row's entries from its n candidates (>= k of them), each put where its rank says: the
// number of larger ones, counted over LDS reads that every lane shares.
__device__ __forceinline__ void write_entries(const TopArgs& a, int64_t row, Shared& sh, int n) {
  if (n > 2 * kBlock) {
    sort_falling(sh.key, n);
    n = a.k;
  } else {
    if (threadIdx.x == 0) sh.key[n] = 0;   // pairs below
    __syncthreads();
  }
  for (int i = threadIdx.x; i < n; i += kBlock) {
    const uint64_t v = sh.key[i];
    int rank = 0;
    for (int o = 0; o < n; o += 2) {
      const ulonglong2 w = *reinterpret_cast<const ulonglong2*>(&sh.key[o]);
      rank += (w.x > v) + (w.y > v);
    }
    if (rank >= a.k) continue;
    const int64_t id = 0xffffffffu - static_cast<uint32_t>(v);
    a.values[row * a.k + rank] = from_order(static_cast<uint32_t>(v >> 32));
    if (a.ids_i64) static_cast<int64_t*>(a.ids)[row * a.k + rank] = id;
    else static_cast<int32_t*>(a.ids)[row * a.k + rank] = static_cast<int32_t>(id);
  }
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
  constexpr int EPV = 16 / TI::kBytes, U = kU, BLOCK = kBlock;
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
  // The lane's largest logit and its sum against it: a batch's in f32, the batches' in f64 (a lane has
  // up to 65,536 elements of a row).
  float mx = kNegInf, adj = 1.f;
  double s = 0.;
  TermScale ts{a.k2, 0.f};
  __syncthreads();
  if (part == 0 && tid < 64) {   // the elements outside the interior
    const int ek = edge_index<TI>(sp, tid);
    float xe = kNegInf;
    if (ek >= 0) {
      xe = TI::load1(xrow, ek);
      mx = fmaxf(mx, xe);
      s = hw_exp2((xe - ms_ref(mx)) * a.k2);
    }
    c.add(ek >= 0, element_key(xe, static_cast<uint32_t>(ek)));
  }
  // The candidates are thinned where they pass `limit`; after the last batch to about k.
  const int room = min(kCut, 2 * a.k + 128), left = a.parts == 1 ? a.k + 64 : a.part_cap;
  constexpr int kRounds = U * EPV / 4;                   // of 4 elements per lane
  int n = part == 0 ? sp.head + sp.tail : 0;             // candidates before the batch
  int round = -1;                                        // >= 0: a batch taken in rounds
  for (int base = v0; base < end;) {
    u32x4 x[U];
    const uint32_t off = static_cast<uint32_t>(base + tid) * 16u;
#pragma unroll
    for (int q = 0; q < U; ++q) x[q] = buf_ld16<true>(xbuf, off + q * (BLOCK * 16u));
    auto held = [&](int q) { return base + q * BLOCK + tid < end; };
    bool near[U];   // this lane's vector may hold an element that passes
    bool fresh = round >= 0 || base == v0 || __any(mx == kNegInf);
    if (!fresh) {
      // Terms against the lane's maximum so far, and the vectors compared by their largest term:
      // no pass for a new maximum unless one has risen far above.
      const float cut = hw_exp2(fmaf(c.least_x, ts.k, -ts.ref)) * (1.f - 0x1p-16f);
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
      fresh = __any(most > 0x1p40f);
      if (!fresh) s += static_cast<double>(acc * adj);
    }
    if (fresh) {
      float vm[U], bx = kNegInf;
#pragma unroll
      for (int q = 0; q < U; ++q) {
        vm[q] = held(q) ? vec_max<TI>(kNegInf, x[q]) : kNegInf;
        bx = fmaxf(bx, vm[q]);
      }
      if (round < 0) {
        const float nm = fmaxf(mx, bx);
        ts = term_scale(nm, a.k2);
        adj = term_adj(nm, ts);
        float acc = 0.f;
#pragma unroll
        for (int q = 0; q < U; ++q)
          if (held(q)) {
            const uint32_t* w = reinterpret_cast<const uint32_t*>(&x[q]);
#pragma unroll
            for (int j = 0; j < EPV; ++j) acc += hw_exp2(fmaf(TI::unpack(w, j), ts.k, -ts.ref));
          }
        s = rescale_at(s, mx, nm, a.k2) + static_cast<double>(acc * adj);
        mx = nm;
        // k vectors of the first batch reach this, each with one element at least.
        if (base == v0) c.least_x = reached_by(sh, vm, a.k);
      }
#pragma unroll
      for (int q = 0; q < U; ++q) near[q] = held(q) && (vm[q] >= c.least_x || c.least_x == kNegInf);
    }
    // While nothing is ruled out NaN is taken too, which ranks below all.
    const bool all = c.least_x == kNegInf;
    // Each lane takes its own vectors one after the other: about a dozen of a wave's 512 pass, so
    // that two turns serve all.
    uint32_t left_q = 0;
#pragma unroll
    for (int q = 0; q < U; ++q) left_q |= near[q] ? 1u << q : 0u;
    if (round >= 0) left_q &= 1u << (round / (EPV / 4));
    while (__any(left_q != 0)) {
      const int mine = __builtin_ctz(left_q | 1u << U);
      u32x4 w = x[0];
#pragma unroll
      for (int q = 1; q < U; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = mine == q ? x[q][i] : w[i];
      // Bit EPV - 1 - j: element j passes. Few lanes have any, fewer have two.
      uint32_t bits = 0;
#pragma unroll
      for (int j = 0; j < EPV; ++j) {
        const float v = TI::unpack(reinterpret_cast<const uint32_t*>(&w), j);
        bits = 2 * bits + ((v >= c.least_x || all) ? 1u : 0u);
      }
      if (left_q == 0) bits = 0;
      left_q &= left_q - 1;
      if (round >= 0) bits &= 0xf0u >> (EPV == 4 ? 4 : 4 * (round % 2));
      const uint32_t first = static_cast<uint32_t>(sp.head + (base + mine * BLOCK + tid) * EPV);
      while (__any(bits != 0)) {
        const int j = EPV - 32 + __builtin_clz(bits | 1u);   // the first that is left
        uint32_t u = w[0];
        const int word = TI::kBytes == 4 ? j : j >> 1;
#pragma unroll
        for (int i = 1; i < 4; ++i) u = word == i ? w[i] : u;
        if constexpr (TI::kBytes == 2) u >>= 16 * (j & 1);
        const uint64_t k = element_key(TI::unpack(&u, 0), first + j);
        c.add(bits != 0 && k > c.least, k);
        bits &= ~((1u << (EPV - 1)) >> j);
      }
    }
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
    if (n > (base >= end ? left : round >= 0 ? kCut : room)) n = c.thin(n, a.k, base >= end ? left : kCut);
    else __syncthreads();
  }
  __syncthreads();
  n = sh.count;
  float sum = static_cast<float>(s);
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

// The parts' candidates, kMergeKeys per lane at a time: a histogram of the first ones finds what
// k of them reach, as in the first kernel.
constexpr int kMergeKeys = 12;

__global__ void __launch_bounds__(kBlock) top_merge_kernel(TopArgs a) {
  constexpr int R = kMergeKeys, kPer = 4;   // keys per lane: of a round, of a cautious one
  static_assert(R % kPer == 0 && kBlock * kPer <= kCap - kCut, "cautious rounds fit");
  __shared__ __align__(16) Shared sh;
  const int tid = threadIdx.x;
  const int64_t row = a.row0 + blockIdx.x;
  const uint64_t* in = a.part_key + row * a.parts * a.part_cap;
  const PartSum* sums = a.part_sum + row * a.parts;
  const int total = a.parts * a.part_cap;
  Candidates c{sh, 0, kNegInf};
  if (tid == 0) sh.count = 0;
  __syncthreads();
  int n = 0, round = -1;
  for (int base = 0; base < total;) {
    uint64_t k[R];
    float v[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int at = base + i * kBlock + tid, p = at / a.part_cap;
      const bool is = at < total && at - p * a.part_cap < sums[p].n;
      k[i] = is ? in[at] : 0;   // no key is 0
    }
#pragma unroll
    for (int i = 0; i < R; ++i) v[i] = k[i] ? from_order(static_cast<uint32_t>(k[i] >> 32)) : kNegInf;
    if (base == 0 && round < 0) c.least_x = reached_by(sh, v, a.k);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (round >= 0 && i / kPer != round) continue;
      c.add(k[i] > c.least && (v[i] >= c.least_x || c.least_x == kNegInf), k[i]);
    }
    __syncthreads();
    const int was = n;
    n = sh.count;
    __syncthreads();
    if (round < 0 && n > kCap) {
      if (tid == 0) sh.count = was;
      n = was;
      round = 0;
    } else if (round < 0 || ++round == R / kPer) {
      round = -1;
      base += kBlock * R;
    }
    if (n > (base >= total ? a.k + 64 : kCut)) n = c.thin(n, a.k, kCut);
    else __syncthreads();
  }
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
