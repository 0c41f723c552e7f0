// The k largest logits of a row: elements as 64-bit keys, candidates of them in LDS, a threshold that at least k
// reach, and the ranking of what is left (top_kernels.hip and score_kernels.hip say how they come by them).
#pragma once

#include "grpo_device.hpp"

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

// A row's k entries from its n candidates (>= k of them), each put where its rank says: the
// number of larger ones, counted over LDS reads that every lane shares. put(rank, logit, id).
template <typename Put>
__device__ __forceinline__ void rank_entries(Shared& sh, int n, int k, Put put) {
  constexpr int kRead = 8;   // keys read at once
  if (n > 2 * kBlock) {
    sort_falling(sh.key, n);
    n = k;
  }
  if (threadIdx.x < kRead && n + static_cast<int>(threadIdx.x) < kCap) sh.key[n + threadIdx.x] = 0;   // read below
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kBlock) {
    const uint64_t v = sh.key[i];
    int rank = 0;
    for (int o = 0; o < n; o += kRead) {
      ulonglong2 w[kRead / 2];
#pragma unroll
      for (int j = 0; j < kRead / 2; ++j) w[j] = *reinterpret_cast<const ulonglong2*>(&sh.key[o + 2 * j]);
#pragma unroll
      for (int j = 0; j < kRead / 2; ++j) rank += (w[j].x > v) + (w[j].y > v);
    }
    if (rank < k)
      put(rank, from_order(static_cast<uint32_t>(v >> 32)), static_cast<int64_t>(0xffffffffu - static_cast<uint32_t>(v)));
  }
}

// The elements of this lane's vectors left_q (bit q: x[q], whose first element is first + q kBlock EPV) that pass go into
// the candidates, of those that keep has (bit EPV - 1 - j: element j). Each lane takes its own vectors one
// after the other: about a dozen of a wave's 512 pass, so that two turns serve all. Called by every lane of a wave.
template <typename TI, int U>
__device__ __forceinline__ void take_vectors(Candidates& c, const u32x4 (&x)[U], uint32_t left_q, uint32_t first, uint32_t keep) {
  constexpr int EPV = 16 / TI::kBytes;
  // While nothing is ruled out NaN is taken too, which ranks below all.
  const bool all = c.least_x == kNegInf;
  while (__any(left_q != 0)) {
    const int mine = __builtin_ctz(left_q | 1u << U);
    u32x4 w = x[0];
#pragma unroll
    for (int q = 1; q < U; ++q)
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = mine == q ? x[q][i] : w[i];
    // Few lanes have any element that passes, fewer have two.
    uint32_t bits = 0;
#pragma unroll
    for (int j = 0; j < EPV; ++j) {
      const float v = TI::unpack(reinterpret_cast<const uint32_t*>(&w), j);
      bits = 2 * bits + ((v >= c.least_x || all) ? 1u : 0u);
    }
    if (left_q == 0) bits = 0;
    left_q &= left_q - 1;
    bits &= keep;
    while (__any(bits != 0)) {
      const int j = EPV - 32 + __builtin_clz(bits | 1u);   // the first that is left
      uint32_t u = w[0];
      const int word = TI::kBytes == 4 ? j : j >> 1;
#pragma unroll
      for (int i = 1; i < 4; ++i) u = word == i ? w[i] : u;
      if constexpr (TI::kBytes == 2) u >>= 16 * (j & 1);
      const uint64_t key = element_key(TI::unpack(&u, 0), first + static_cast<uint32_t>(mine * kBlock * EPV + j));
      c.add(bits != 0 && key > c.least, key);
      bits &= ~((1u << (EPV - 1)) >> j);
    }
  }
}

// The candidates of a row's parts, kMergeKeys per lane at a time: a histogram of the first ones finds what
// k of them reach, as in the scan. n_of(part): what a part has left, part_cap keys apart, key_at(i) the i-th
// of all. Leaves them in sh, and returns their number; called by the whole workgroup with sh free.
constexpr int kMergeKeys = 12;

template <typename KeyAt, typename NOf>
__device__ __forceinline__ int merge_parts(KeyAt key_at, int parts, int part_cap, int k, NOf n_of, Shared& sh) {
  constexpr int R = kMergeKeys, kPer = 4;   // keys per lane: of a round, of a cautious one
  static_assert(R % kPer == 0 && kBlock * kPer <= kCap - kCut, "cautious rounds fit");
  const int tid = threadIdx.x;
  const int total = parts * part_cap;
  Candidates c{sh, 0, kNegInf};
  if (tid == 0) sh.count = 0;
  __syncthreads();
  int n = 0, round = -1;
  for (int base = 0; base < total;) {
    uint64_t key[R];
    float v[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int at = base + i * kBlock + tid, p = at / part_cap;
      const bool is = at < total && at - p * part_cap < n_of(p);
      key[i] = is ? key_at(at) : 0;   // no key is 0
    }
#pragma unroll
    for (int i = 0; i < R; ++i) v[i] = key[i] ? from_order(static_cast<uint32_t>(key[i] >> 32)) : kNegInf;
    if (base == 0 && round < 0) c.least_x = reached_by(sh, v, k);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (round >= 0 && i / kPer != round) continue;
      c.add(key[i] > c.least && (v[i] >= c.least_x || c.least_x == kNegInf), key[i]);
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
    if (n > (base >= total ? k + 64 : kCut)) n = c.thin(n, k, kCut);
    else __syncthreads();
  }
  return n;
}

}  // namespace
}  // namespace pcp
