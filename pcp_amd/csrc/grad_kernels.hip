// A model's gradients where the backward pass left them (pcp_step.h): their norm and the coefficient
// that clips it, the clipped gradients, and the Nesterov update of many tensors with that coefficient.
//
// A 0.5B model's 290 bf16 gradients: norm 162 us (0.99 GB, 6.1 TB/s in two launches), clipped into a flat f32 buffer
// 485 (2.96 GB, 6.1 TB/s), update with f32 weights and velocities and a bf16 copy 1655 (9.88 GB, 6.0 TB/s). f32 gradients:
// norm 314 (6.3 TB/s), update 1873 (10.9 GB, 5.8). The gradients are read twice, for the norm and with the
// coefficient: they are four times what the caches hold, and visiting them in falling order the second time gained 0.5%.
//
// All three are HBM-bound streams over a list of tensors. The list travels in the kernels' arguments
// (under 4 KB), so a call uploads nothing and keeps nothing; long lists take several launches. A tensor
// is cut into pieces below 2^28 elements, a piece into chunks, so that every index within one is 32-bit.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <new>
#include <vector>

#include "context.hpp"
#include "grpo_device.hpp"
#include "pcp_step.h"

// Products and sums round one by one, as in the update of one flat buffer.
#pragma clang fp contract(off)

namespace pcp {
namespace {

constexpr int kBlock = 256;
constexpr int64_t kPiece = int64_t(1) << 28;
constexpr uint32_t kCount = (1u << 29) - 1;    // of a piece's word: its elements, and above them its types
constexpr int kTypeShift = 30;
constexpr int kLaunchChunks = 1 << 23;         // 2^31 lanes: the next launch takes what follows

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef u32x2 u32x2_any __attribute__((aligned(2)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));

// Type codes of a piece's word: PCP_F16, PCP_BF16, PCP_F32 as they are (0, 1, 2).
template <typename F>
__device__ __forceinline__ void with_type(uint32_t code, F f) {
  if (code == PCP_F32) f(F32T{});
  else if (code == PCP_BF16) f(BF16T{});
  else f(F16T{});
}

// The piece of chunk c: first[t] <= c < first[t + 1].
__device__ __forceinline__ int piece_of(const int* first, int pieces, int c) {
  int t = 0, hi = pieces;
  while (hi - t > 1) {
    const int mid = (t + hi) / 2;
    if (first[mid] <= c) t = mid;
    else hi = mid;
  }
  return t;
}

// ---- norm -------------------------------------------------------------------------------

constexpr int kNormPieces = 240;
constexpr int kNormChunk = 16384, kNormSmall = 4096;
constexpr int kNormGrid = 2048;    // workgroups of a launch: eight on each CU

struct NormArgs {
  const void* g[kNormPieces];
  uint32_t n[kNormPieces];
  int first[kNormPieces + 1];
  int pieces;
  int chunk;              // elements
  int block0;             // workgroups of earlier launches
  int blocks;             // of all launches
  float max_norm;
  double* parts;
  unsigned* done;
  float* norm;
  float* coef;
  int* err;
};
static_assert(sizeof(NormArgs) <= 4096, "kernel arguments");

// Bound by HBM: f64 sums, f32 sums of 16 squares and the maximum alone read at the same 6.8 to 6.9 TB/s in a flat loop over one
// tensor. What cost were lookups between chunks (0.99 GB of 290 tensors 260 us; stretches 189), registers (eight loads a lane
// in flight 107 of them; four, 64) and one ticket for 2048 workgroups (an atomic after the other): 189 -> 162 us with
// those two, 117 MB of 110 tensors 39 -> 27.
//
// Squares of N elements in f64, or their largest magnitude as f32 bits, which order NaN above infinity.
template <int TYPE, int N>
__device__ __forceinline__ void norm_add(double& s, uint32_t& top, const float (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if constexpr (TYPE == PCP_NORM_L2) {
      const double d = static_cast<double>(x[i]);
      s = __builtin_fma(d, d, s);   // d * d is exact
    } else {
      top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
    }
  }
}

template <int TYPE, typename TI>
__device__ __forceinline__ void norm_chunk(const char* g, int n, double& s, uint32_t& top) {
  constexpr int EPV = 16 / TI::kBytes, U = 4;
  const int nv = n / EPV;
  const u32x4_any* v = reinterpret_cast<const u32x4_any*>(g);
  int i = threadIdx.x;
  for (; i + (U - 1) * kBlock < nv; i += U * kBlock) {
    u32x4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = __builtin_nontemporal_load(v + i + u * kBlock);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[EPV];
#pragma unroll
      for (int j = 0; j < EPV; ++j) x[j] = TI::unpack(reinterpret_cast<const uint32_t*>(&w[u]), j);
      norm_add<TYPE>(s, top, x);
    }
  }
  for (; i < nv; i += kBlock) {
    const u32x4 w = v[i];
    float x[EPV];
#pragma unroll
    for (int j = 0; j < EPV; ++j) x[j] = TI::unpack(reinterpret_cast<const uint32_t*>(&w), j);
    norm_add<TYPE>(s, top, x);
  }
  const int r = nv * EPV + static_cast<int>(threadIdx.x);
  if (r < n) {
    const float x[1] = {TI::load1(g, r)};
    norm_add<TYPE>(s, top, x);
  }
}

// A workgroup's sum of s, or its largest top, as a number on thread 0 (bits are exact in f64).
template <int TYPE>
__device__ __forceinline__ double norm_block(double s, uint32_t top, double* lds) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if constexpr (TYPE == PCP_NORM_L2) {
    s = wave_sum64(s);
  } else {
    for (int i = 32; i > 0; i >>= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), i)));
    s = static_cast<double>(top);
  }
  if (lane == 0) lds[wave] = s;
  __syncthreads();
  double o = lds[0];
#pragma unroll
  for (int w = 1; w < kBlock / 64; ++w) o = TYPE == PCP_NORM_L2 ? o + lds[w] : fmax(o, lds[w]);
  return o;
}

template <int TYPE>
__global__ void __launch_bounds__(kBlock) norm_kernel(NormArgs a) {
  __shared__ double lds[kBlock / 64];
  __shared__ unsigned turn;
  const int chunks = a.first[a.pieces];
  const int c0 = static_cast<int>(static_cast<int64_t>(chunks) * blockIdx.x / gridDim.x);
  const int c1 = static_cast<int>(static_cast<int64_t>(chunks) * (blockIdx.x + 1) / gridDim.x);
  double s = 0.;
  uint32_t top = 0;
  // A workgroup's chunks lie one after another: what they have of a piece is read as one stretch, with no lookup (three
  // dependent scalar loads) between chunks.
  if (c0 < c1) {
    int t = piece_of(a.first, a.pieces, c0);
    for (int c = c0; c < c1; ++t) {
      const uint32_t word = a.n[t];
      const int from = c - a.first[t], to = min(c1, a.first[t + 1]) - a.first[t];
      const int64_t e0 = static_cast<int64_t>(from) * a.chunk;
      const int n = static_cast<int>(min(static_cast<int64_t>(to) * a.chunk, static_cast<int64_t>(word & kCount)) - e0);
      with_type(word >> kTypeShift, [&](auto type) {
        using TI = decltype(type);
        norm_chunk<TYPE, TI>(static_cast<const char*>(a.g[t]) + e0 * TI::kBytes, n, s, top);
      });
      c += to - from;
    }
  }
  const double mine = norm_block<TYPE>(s, top, lds);
  if (threadIdx.x == 0) {
    store_coherent(a.parts + a.block0 + blockIdx.x, mine);
    wait_stores();
    // The last of a group of workgroups counts for it: one counter for all of them would take an atomic after the other.
    const int block = a.block0 + static_cast<int>(blockIdx.x), g = block % kNormGroups;
    const unsigned of_group = static_cast<unsigned>((a.blocks - g + kNormGroups - 1) / kNormGroups);
    const unsigned groups = static_cast<unsigned>(min(a.blocks, kNormGroups));
    unsigned* const mine = a.done + (1 + g) * kNormApart;
    turn = 0;
    if (__hip_atomic_fetch_add(mine, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == of_group) {
      store_coherent(mine, 0u);
      turn = __hip_atomic_fetch_add(a.done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == groups;
      if (turn) store_coherent(a.done, 0u);
    }
  }
  __syncthreads();
  if (!turn) return;
  acquire_coherent();
  s = 0.;
  top = 0;
  for (int i = threadIdx.x; i < a.blocks; i += kBlock) {
    if constexpr (TYPE == PCP_NORM_L2) s += a.parts[i];
    else top = max(top, static_cast<uint32_t>(a.parts[i]));
  }
  const double all = norm_block<TYPE>(s, top, lds);
  if (threadIdx.x != 0) return;
  const double norm = TYPE == PCP_NORM_L2 ? sqrt(all) : static_cast<double>(__uint_as_float(static_cast<uint32_t>(all)));
  const float rounded = static_cast<float>(norm);
  const bool fine = __builtin_isfinite(rounded);
  if (!fine) raise_error(a.err, kErrNonFinite);
  *a.norm = rounded;
  const double most = static_cast<double>(a.max_norm);
  *a.coef = !fine ? __builtin_nanf("") : norm > most ? static_cast<float>(most / norm) : 1.f;
}

// ---- clipping ---------------------------------------------------------------------------

constexpr int kClipPieces = 160;

struct ClipArgs {
  const void* g[kClipPieces];
  void* out[kClipPieces];
  uint32_t n[kClipPieces];       // elements, and out's type above them
  uint8_t from[kClipPieces];     // g's type
  int first[kClipPieces + 1];
  int pieces;
  const float* coef;
};
static_assert(sizeof(ClipArgs) <= 4096, "kernel arguments");

// Elements per lane and group: 16 bytes of the wider type; and groups per lane. us for 494 M elements with 1 | 2 | 4:
// bf16 to f32 610 | 501 | 485, f32 to f32 636 | 651 | 672; for 576 M, bf16 to bf16 382 | 362 | 376 (in place the same), f32
// to bf16 657 | 530 | 558.
constexpr __host__ __device__ inline int clip_group(int from, int to) { return from == 4 || to == 4 ? 4 : 8; }
constexpr __host__ __device__ inline int clip_unroll(int from, int to) { return from == 4 ? 1 : to == 4 ? 4 : 2; }

// Chunks begin where out is aligned to its group: the first group of a tensor may begin before it.
constexpr __host__ __device__ inline int clip_lead(uintptr_t out, int bytes, int group) {
  return static_cast<int>((out / bytes) & static_cast<uintptr_t>(group - 1));
}

template <int N, typename TI>
__device__ __forceinline__ void load_group(const char* p, float (&x)[N]) {
  if constexpr (N * TI::kBytes == 16) {
    const u32x4 w = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(p));
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = TI::unpack(reinterpret_cast<const uint32_t*>(&w), j);
  } else {
    const u32x2 w = __builtin_nontemporal_load(reinterpret_cast<const u32x2_any*>(p));
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = TI::unpack(reinterpret_cast<const uint32_t*>(&w), j);
  }
}

// The f32 product, rounded: for f16 the compiler would else form v_fma_mixlo_f16, which rounds the
// exact product to f16 at once and so differs where f32's rounding makes a tie.
template <typename TO>
__device__ __forceinline__ float f32_product(float a, float b) {
  float y = a * b;
  if constexpr (__is_same(TO, F16T)) asm("" : "+v"(y));
  return y;
}

template <typename TI, typename TO>
__device__ __forceinline__ void clip_chunk(const char* g, char* out, int n, int c, float coef) {
  constexpr int N = clip_group(TI::kBytes, TO::kBytes), U = clip_unroll(TI::kBytes, TO::kBytes);
  const int first = -clip_lead(reinterpret_cast<uintptr_t>(out), TO::kBytes, N);
  const int e0 = first + (c * (U * kBlock) + static_cast<int>(threadIdx.x)) * N;
  float x[U][N];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int e = e0 + u * kBlock * N;
    if (e >= 0 && e + N <= n) load_group<N, TI>(g + static_cast<int64_t>(e) * TI::kBytes, x[u]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int e = e0 + u * kBlock * N;
    if (e >= 0 && e + N <= n) {
#pragma unroll
      for (int j = 0; j < N; ++j) x[u][j] = f32_product<TO>(coef, x[u][j]);
      store_vals<TO, N, true>(out, e, x[u]);
    } else {
      for (int j = max(-e, 0); j < min(N, n - e); ++j) store1<TO>(out, e + j, f32_product<TO>(coef, TI::load1(g, e + j)));
    }
  }
}

__global__ void __launch_bounds__(kBlock) clip_kernel(ClipArgs a) {
  const int t = piece_of(a.first, a.pieces, static_cast<int>(blockIdx.x));
  const uint32_t word = a.n[t];
  const char* g = static_cast<const char*>(a.g[t]);
  char* out = static_cast<char*>(a.out[t]);
  float coef = *a.coef;
  if (coef != coef) coef = 1.f;
  if (coef == 1.f && g == out) return;
  const int n = static_cast<int>(word & kCount), c = static_cast<int>(blockIdx.x) - a.first[t];
  with_type(a.from[t], [&](auto from) {
    with_type(word >> kTypeShift, [&](auto to) { clip_chunk<decltype(from), decltype(to)>(g, out, n, c, coef); });
  });
}

// ---- update -----------------------------------------------------------------------------

constexpr int kUpdatePieces = 100;
constexpr int kUpdateChunk = 4 * kBlock;   // a group of four per lane: waves with few stores each write fastest

struct UpdateArgs {
  float* p[kUpdatePieces];
  float* v[kUpdatePieces];
  const void* g[kUpdatePieces];
  uint16_t* copy[kUpdatePieces];
  uint32_t n[kUpdatePieces];       // elements, and the gradient's type above them
  int first[kUpdatePieces + 1];
  int pieces;
  const float* coef;
  float lr, mu;
};
static_assert(sizeof(UpdateArgs) <= 4096, "kernel arguments");

template <int MODE>
__device__ __forceinline__ void update_one(float& p, float& v, float g, float lr, float mu) {
  if constexpr (MODE == PCP_NESTEROV_SUTSKEVER) {
    v = mu * v + g;
    p = p - lr * (g + mu * v);
  } else {
    v = mu * v + lr * g;
    p = p - v;
  }
}

template <int MODE, typename TI>
__device__ __forceinline__ void update_chunk(float* p, float* v, const char* g, uint16_t* copy, int n, int c, float coef,
                                             float lr, float mu) {
  const int e = (c * kBlock + static_cast<int>(threadIdx.x)) * 4 - clip_lead(reinterpret_cast<uintptr_t>(p), 4, 4);
  if (e >= 0 && e + 4 <= n) {
    f32x4 pp = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p + e));
    f32x4 vv = __builtin_nontemporal_load(reinterpret_cast<const f32x4_any*>(v + e));
    float gg[4];
    load_group<4, TI>(g + static_cast<int64_t>(e) * TI::kBytes, gg);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float pj = pp[j], vj = vv[j];
      update_one<MODE>(pj, vj, coef * gg[j], lr, mu);
      pp[j] = pj;
      vv[j] = vj;
    }
    store_nt_sys(__builtin_bit_cast(u32x4, pp), p + e);
    store_nt_sys(__builtin_bit_cast(u32x4, vv), v + e);
    if (copy != nullptr) {
      const u32x2 b = {pack2<BF16T>(pp[0], pp[1]), pack2<BF16T>(pp[2], pp[3])};
      if ((reinterpret_cast<uintptr_t>(copy + e) & 3u) == 0) {
        store_nt_sys(b, copy + e);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) store1<BF16T>(copy, e + j, pp[j]);
      }
    }
    return;
  }
  for (int i = max(e, 0); i < min(e + 4, n); ++i) {
    float pi = p[i], vi = v[i];
    update_one<MODE>(pi, vi, coef * TI::load1(g, i), lr, mu);
    p[i] = pi;
    v[i] = vi;
    if (copy != nullptr) store1<BF16T>(copy, i, pi);
  }
}

template <int MODE>
__global__ void __launch_bounds__(kBlock) update_kernel(UpdateArgs a) {
  const int t = piece_of(a.first, a.pieces, static_cast<int>(blockIdx.x));
  const uint32_t word = a.n[t];
  const float coef = a.coef ? *a.coef : 1.f;
  if (!__builtin_isfinite(coef)) return;
  const int n = static_cast<int>(word & kCount), c = static_cast<int>(blockIdx.x) - a.first[t];
  with_type(word >> kTypeShift, [&](auto type) {
    update_chunk<MODE, decltype(type)>(a.p[t], a.v[t], static_cast<const char*>(a.g[t]), a.copy[t], n, c, coef, a.lr, a.mu);
  });
}

// ---- host -------------------------------------------------------------------------------

inline bool misaligned(const void* p, int size) {
  return (reinterpret_cast<uintptr_t>(p) & static_cast<uintptr_t>(size - 1)) != 0;
}

inline bool float_type(int dt) { return dt == PCP_F32 || dt == PCP_BF16 || dt == PCP_F16; }

// Memory that a call writes, or reads.
struct Range {
  uintptr_t at, end;
  bool written;
};

// One of a call's lists: where it lies, and whether its tensors follow one another.
struct Extent {
  uintptr_t lo = UINTPTR_MAX, hi = 0;
  bool written = false, rising = true;
};

// Whether a written range meets any other; each(f) calls f(list, address, bytes, written) for all, lists numbered below
// kLists. Lists that each lie in a stretch of their own, the written ones rising, as pieces of flat buffers do, need no
// sorting (3 us of a 26-tensor update).
template <typename Each>
bool ranges_meet(Each each) {
  constexpr int kLists = 5;
  Extent e[kLists];
  size_t n = 0;
  each([&](int list, uintptr_t at, uintptr_t bytes, bool written) {
    Extent& x = e[list];
    x.rising = x.rising && at >= x.hi;
    x.written = x.written || written;
    x.lo = std::min(x.lo, at);
    x.hi = std::max(x.hi, at + bytes);
    ++n;
  });
  bool apart = true;
  for (int i = 0; i < kLists; ++i) {
    apart = apart && (!e[i].written || e[i].rising);
    for (int j = 0; j < i; ++j) apart = apart && (!(e[i].written || e[j].written) || e[i].hi <= e[j].lo || e[j].hi <= e[i].lo);
  }
  if (apart) return false;
  std::vector<Range> r;
  r.reserve(n);
  each([&](int, uintptr_t at, uintptr_t bytes, bool written) { r.push_back({at, at + bytes, written}); });
  std::sort(r.begin(), r.end(), [](const Range& x, const Range& y) { return x.at < y.at; });
  uintptr_t written = 0, any = 0;   // the furthest end of what began before
  for (const Range& x : r) {
    if (x.at < written || (x.written && x.at < any)) return true;
    any = std::max(any, x.end);
    if (x.written) written = std::max(written, x.end);
  }
  return false;
}

int check_list(pcp_ctx* ctx, int64_t n_tensors, const int64_t* counts, int64_t* elements) {
  *elements = 0;
  if (n_tensors < 0 || n_tensors > PCP_GRAD_MAX_TENSORS)
    return fail(ctx, PCP_ERR_INVALID_ARG, "n_tensors must be in [0, %d] (got %lld)", PCP_GRAD_MAX_TENSORS, (long long)n_tensors);
  if (n_tensors > 0 && !counts) return fail(ctx, PCP_ERR_INVALID_ARG, "counts is NULL");
  for (int64_t i = 0; i < n_tensors; ++i) {
    if (counts[i] < 0) return fail(ctx, PCP_ERR_INVALID_ARG, "counts[%lld] < 0", (long long)i);
    if (counts[i] > (int64_t(1) << 44) - *elements) return fail(ctx, PCP_ERR_OVERFLOW, "more than 2^44 elements");
    *elements += counts[i];
  }
  return PCP_OK;
}

// Walks the pieces of a list: next() is the piece's tensor, first element and elements, false at the end.
struct Pieces {
  const int64_t* counts;
  int64_t n_tensors, tensor = 0, at = 0, from = 0, size = 0;
  bool next() {
    while (tensor < n_tensors && at >= counts[tensor]) {
      ++tensor;
      at = 0;
    }
    if (tensor >= n_tensors) return false;
    from = at;
    size = std::min(kPiece, counts[tensor] - at);
    at += size;
    return true;
  }
};

hipError_t launch_norm(pcp_ctx* ctx, const pcp_grad_clip_args* a, int64_t elements, hipStream_t st) {
  // The launches, and how many workgroups each may have: kNormBlocks in all.
  int64_t pieces = elements == 0 ? 0 : a->n_tensors;
  if (elements > kPiece || pieces > kNormPieces) {
    pieces = 0;
    for (Pieces p{a->counts, a->n_tensors}; p.next();) ++pieces;
  }
  const int64_t launches = std::max<int64_t>(1, (pieces + kNormPieces - 1) / kNormPieces);
  const int most = static_cast<int>(std::min<int64_t>(kNormGrid, kNormBlocks / launches));
  // Chunks small enough that a small model's gradients occupy the chip, and large enough that a vector's loads are wide.
  const int chunk = elements < int64_t(kNormGrid) * kNormChunk ? kNormSmall : kNormChunk;
  static_assert((PCP_GRAD_MAX_TENSORS + 65536) / kNormPieces + 1 <= kNormBlocks, "a workgroup for every launch");
  NormArgs b;
  b.chunk = chunk;
  b.max_norm = a->max_norm;
  b.parts = ctx->d_norm_parts;
  b.done = ctx->d_norm_done;
  b.norm = a->norm;
  b.coef = a->coef;
  b.err = ctx->d_page->err;
  // With several launches two walks: the workgroups are counted before the first, since each needs their number.
  for (int launch = launches > 1 ? 0 : 1; launch < 2; ++launch) {
    Pieces p{a->counts, a->n_tensors};
    bool more = p.next();
    int blocks = 0;
    do {
      b.pieces = 0;
      b.first[0] = 0;
      for (; more && b.pieces < kNormPieces; more = p.next()) {
        const int dt = a->dtypes ? a->dtypes[p.tensor] : PCP_F32;
        b.g[b.pieces] = static_cast<const char*>(a->grads[p.tensor]) + p.from * dtype_bytes(dt);
        b.n[b.pieces] = static_cast<uint32_t>(p.size) | static_cast<uint32_t>(dt) << kTypeShift;
        b.first[b.pieces + 1] = b.first[b.pieces] + static_cast<int>((p.size + chunk - 1) / chunk);
        ++b.pieces;
      }
      const int grid = std::max(1, std::min(most, b.first[b.pieces]));
      if (launch == 1) {
        b.block0 = blocks;
        if (launches == 1) b.blocks = grid;
        if (a->norm_type == PCP_NORM_L2) norm_kernel<PCP_NORM_L2><<<grid, kBlock, 0, st>>>(b);
        else norm_kernel<PCP_NORM_MAX><<<grid, kBlock, 0, st>>>(b);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
      }
      blocks += grid;
    } while (more);
    b.blocks = blocks;
  }
  return hipSuccess;
}

hipError_t launch_clip(const pcp_grad_clip_args* a, hipStream_t st) {
  ClipArgs b;
  b.coef = a->coef;
  Pieces p{a->counts, a->n_tensors};
  for (bool more = p.next(); more;) {
    b.pieces = 0;
    b.first[0] = 0;
    for (; more && b.pieces < kClipPieces; more = p.next()) {
      const int from = a->dtypes ? a->dtypes[p.tensor] : PCP_F32, to = a->out_dtypes ? a->out_dtypes[p.tensor] : from;
      const int group = clip_group(dtype_bytes(from), dtype_bytes(to));
      char* out = static_cast<char*>(a->out[p.tensor]) + p.from * dtype_bytes(to);
      b.g[b.pieces] = static_cast<const char*>(a->grads[p.tensor]) + p.from * dtype_bytes(from);
      b.out[b.pieces] = out;
      b.n[b.pieces] = static_cast<uint32_t>(p.size) | static_cast<uint32_t>(to) << kTypeShift;
      b.from[b.pieces] = static_cast<uint8_t>(from);
      const int64_t chunk = clip_unroll(dtype_bytes(from), dtype_bytes(to)) * kBlock * group;
      const int64_t span = p.size + clip_lead(reinterpret_cast<uintptr_t>(out), dtype_bytes(to), group);
      b.first[b.pieces + 1] = b.first[b.pieces] + static_cast<int>((span + chunk - 1) / chunk);
      ++b.pieces;
      if (b.first[b.pieces] > kLaunchChunks) {
        more = p.next();
        break;
      }
    }
    clip_kernel<<<b.first[b.pieces], kBlock, 0, st>>>(b);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

int grad_clip(pcp_ctx* ctx, const pcp_grad_clip_args* a) {
  if (!a) return fail(ctx, PCP_ERR_INVALID_ARG, "args is NULL");
  int64_t elements;
  const int rc = check_list(ctx, a->n_tensors, a->counts, &elements);
  if (rc != PCP_OK) return rc;
  if (a->norm_type != PCP_NORM_L2 && a->norm_type != PCP_NORM_MAX)
    return fail(ctx, PCP_ERR_INVALID_ARG, "unknown norm_type %d", a->norm_type);
  if (!(a->max_norm > 0.f)) return fail(ctx, PCP_ERR_INVALID_ARG, "max_norm must be > 0");
  if (a->flags & ~PCP_FLAG_ASYNC) return fail(ctx, PCP_ERR_INVALID_ARG, "only PCP_FLAG_ASYNC applies here");
  if (!a->norm || !a->coef || (a->n_tensors > 0 && !a->grads))
    return fail(ctx, PCP_ERR_INVALID_ARG, "norm, coef or grads is NULL");
  if (misaligned(a->norm, 4) || misaligned(a->coef, 4))
    return fail(ctx, PCP_ERR_INVALID_ARG, "pointers must be aligned to their element size");
  for (int64_t i = 0; i < a->n_tensors; ++i) {
    const int from = a->dtypes ? a->dtypes[i] : PCP_F32, to = a->out_dtypes ? a->out_dtypes[i] : from;
    if (!float_type(from) || (a->out && !float_type(to)))
      return fail(ctx, PCP_ERR_DTYPE, "tensor %lld: types must be f32, bf16 or f16", (long long)i);
    if (a->counts[i] == 0) continue;
    if (!a->grads[i] || (a->out && !a->out[i])) return fail(ctx, PCP_ERR_INVALID_ARG, "tensor %lld is NULL", (long long)i);
    if (misaligned(a->grads[i], dtype_bytes(from)) || (a->out && misaligned(a->out[i], dtype_bytes(to))))
      return fail(ctx, PCP_ERR_INVALID_ARG, "pointers must be aligned to their element size");
  }
  const uintptr_t norm = reinterpret_cast<uintptr_t>(a->norm), coef = reinterpret_cast<uintptr_t>(a->coef);
  bool scalars = norm < coef + 4 && coef < norm + 4;
  if (!a->out)   // (with outputs their ranges are among the lists': below. Gradients may overlap one another here.)
    for (int64_t i = 0; i < a->n_tensors; ++i) {
      const uintptr_t g = reinterpret_cast<uintptr_t>(a->grads[i]);
      const uintptr_t end = g + static_cast<uintptr_t>(a->counts[i]) * dtype_bytes(a->dtypes ? a->dtypes[i] : PCP_F32);
      scalars = scalars || (norm < end && g < norm + 4 && g < end) || (coef < end && g < coef + 4 && g < end);
    }
  if (scalars) return fail(ctx, PCP_ERR_INVALID_ARG, "norm or coef overlaps a gradient, or one the other");
  try {
    const bool meet = a->out && ranges_meet([&](auto add) {
      for (int64_t i = 0; i < a->n_tensors; ++i) {
        if (a->counts[i] == 0) continue;
        const int from = a->dtypes ? a->dtypes[i] : PCP_F32, to = a->out_dtypes ? a->out_dtypes[i] : from;
        const uintptr_t g = reinterpret_cast<uintptr_t>(a->grads[i]), o = reinterpret_cast<uintptr_t>(a->out[i]);
        const uintptr_t n = static_cast<uintptr_t>(a->counts[i]);
        if (g != o || from != to) add(0, g, n * dtype_bytes(from), false);   // (else in place: one range)
        add(1, o, n * dtype_bytes(to), true);
      }
      add(2, reinterpret_cast<uintptr_t>(a->norm), 4, true);
      add(3, reinterpret_cast<uintptr_t>(a->coef), 4, true);
    });
    if (meet) return fail(ctx, PCP_ERR_INVALID_ARG, "an output overlaps a gradient other than its own, or another output");
  } catch (const std::bad_alloc&) {
    return fail(ctx, PCP_ERR_OOM, "no host memory to check the tensors");
  }
  if (!ctx) return fail(nullptr, PCP_ERR_INVALID_ARG, "context is NULL");
  const DeviceScope scope(ctx->device);
  if (scope.error() != hipSuccess) return hip_fail(ctx, scope.error(), "making the context's device current");
  hipStream_t st = static_cast<hipStream_t>(a->stream);
  hipError_t e = launch_norm(ctx, a, elements, st);
  if (e != hipSuccess) return hip_fail(ctx, e, "gradient norm launch");
  if (a->out && elements > 0 && (e = launch_clip(a, st)) != hipSuccess) return hip_fail(ctx, e, "gradient clipping launch");
  return finish_call(ctx, a->flags, st);
}

int nesterov_many(pcp_ctx* ctx, const pcp_nesterov_many_args* a) {
  if (!a) return fail(ctx, PCP_ERR_INVALID_ARG, "args is NULL");
  int64_t elements;
  const int rc = check_list(ctx, a->n_tensors, a->counts, &elements);
  if (rc != PCP_OK) return rc;
  if (a->mode != PCP_NESTEROV_SUTSKEVER && a->mode != PCP_NESTEROV_MLIR)
    return fail(ctx, PCP_ERR_INVALID_ARG, "unknown Nesterov mode %d", a->mode);
  if (!std::isfinite(a->learning_rate) || !std::isfinite(a->momentum))
    return fail(ctx, PCP_ERR_INVALID_ARG, "learning_rate and momentum must be finite");
  if (a->flags & ~PCP_FLAG_ASYNC) return fail(ctx, PCP_ERR_INVALID_ARG, "only PCP_FLAG_ASYNC applies here");
  if (a->n_tensors > 0 && (!a->params || !a->velocities || !a->grads))
    return fail(ctx, PCP_ERR_INVALID_ARG, "params, velocities or grads is NULL");
  if (misaligned(a->coef, 4)) return fail(ctx, PCP_ERR_INVALID_ARG, "pointers must be aligned to their element size");
  for (int64_t i = 0; i < a->n_tensors; ++i) {
    const int dt = a->dtypes ? a->dtypes[i] : PCP_F32;
    if (!float_type(dt)) return fail(ctx, PCP_ERR_DTYPE, "tensor %lld: gradients must be f32, bf16 or f16", (long long)i);
    if (a->counts[i] == 0) continue;
    if (!a->params[i] || !a->velocities[i] || !a->grads[i])
      return fail(ctx, PCP_ERR_INVALID_ARG, "tensor %lld is NULL", (long long)i);
    if (misaligned(a->params[i], 4) || misaligned(a->velocities[i], 4) || misaligned(a->grads[i], dtype_bytes(dt)) ||
        (a->param_copies && misaligned(a->param_copies[i], 2)))
      return fail(ctx, PCP_ERR_INVALID_ARG, "pointers must be aligned to their element size");
  }
  try {
    const bool meet = ranges_meet([&](auto add) {
      for (int64_t i = 0; i < a->n_tensors; ++i) {
        const uintptr_t n = static_cast<uintptr_t>(a->counts[i]);
        if (n == 0) continue;
        add(0, reinterpret_cast<uintptr_t>(a->params[i]), n * 4, true);
        add(1, reinterpret_cast<uintptr_t>(a->velocities[i]), n * 4, true);
        add(2, reinterpret_cast<uintptr_t>(a->grads[i]), n * dtype_bytes(a->dtypes ? a->dtypes[i] : PCP_F32), false);
        if (a->param_copies && a->param_copies[i]) add(3, reinterpret_cast<uintptr_t>(a->param_copies[i]), n * 2, true);
      }
      if (a->coef) add(4, reinterpret_cast<uintptr_t>(a->coef), 4, false);
    });
    if (meet) return fail(ctx, PCP_ERR_INVALID_ARG, "a parameter, velocity or copy overlaps another tensor of the call");
  } catch (const std::bad_alloc&) {
    return fail(ctx, PCP_ERR_OOM, "no host memory to check the tensors");
  }
  if (!ctx) return fail(nullptr, PCP_ERR_INVALID_ARG, "context is NULL");
  if (elements == 0) return PCP_OK;
  const DeviceScope scope(ctx->device);
  if (scope.error() != hipSuccess) return hip_fail(ctx, scope.error(), "making the context's device current");
  hipStream_t st = static_cast<hipStream_t>(a->stream);
  UpdateArgs b;
  b.coef = a->coef;
  b.lr = a->learning_rate;
  b.mu = a->momentum;
  Pieces p{a->counts, a->n_tensors};
  for (bool more = p.next(); more;) {
    b.pieces = 0;
    b.first[0] = 0;
    for (; more && b.pieces < kUpdatePieces; more = p.next()) {
      const int dt = a->dtypes ? a->dtypes[p.tensor] : PCP_F32;
      b.p[b.pieces] = a->params[p.tensor] + p.from;
      b.v[b.pieces] = a->velocities[p.tensor] + p.from;
      b.g[b.pieces] = static_cast<const char*>(a->grads[p.tensor]) + p.from * dtype_bytes(dt);
      void* const copy = a->param_copies ? a->param_copies[p.tensor] : nullptr;
      b.copy[b.pieces] = copy ? static_cast<uint16_t*>(copy) + p.from : nullptr;
      b.n[b.pieces] = static_cast<uint32_t>(p.size) | static_cast<uint32_t>(dt) << kTypeShift;
      const int64_t span = p.size + clip_lead(reinterpret_cast<uintptr_t>(b.p[b.pieces]), 4, 4);
      b.first[b.pieces + 1] = b.first[b.pieces] + static_cast<int>((span + kUpdateChunk - 1) / kUpdateChunk);
      ++b.pieces;
      if (b.first[b.pieces] > kLaunchChunks) {
        more = p.next();
        break;
      }
    }
    if (a->mode == PCP_NESTEROV_SUTSKEVER) update_kernel<PCP_NESTEROV_SUTSKEVER><<<b.first[b.pieces], kBlock, 0, st>>>(b);
    else update_kernel<PCP_NESTEROV_MLIR><<<b.first[b.pieces], kBlock, 0, st>>>(b);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return hip_fail(ctx, e, "Nesterov launch");
  }
  return finish_call(ctx, a->flags, st);
}

}  // namespace
}  // namespace pcp

using namespace pcp;

extern "C" {

void pcp_grad_clip_args_init(pcp_grad_clip_args* a) {
  if (!a) return;
  std::memset(a, 0, sizeof(*a));
  a->norm_type = PCP_NORM_L2;
  a->max_norm = __builtin_inff();
}

int pcp_grad_clip(pcp_ctx* ctx, const pcp_grad_clip_args* a) { return grad_clip(ctx, a); }

void pcp_nesterov_many_args_init(pcp_nesterov_many_args* a) {
  if (!a) return;
  std::memset(a, 0, sizeof(*a));
  a->learning_rate = 0.01f;
  a->momentum = 0.9f;
  a->mode = PCP_NESTEROV_SUTSKEVER;
}

int pcp_nesterov_update_many(pcp_ctx* ctx, const pcp_nesterov_many_args* a) { return nesterov_many(ctx, a); }

}  // extern "C"
