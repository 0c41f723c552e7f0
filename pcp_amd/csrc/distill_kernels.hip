// Distillation from a teacher's top logits (pcp_distill.h): the loss of a row against up
// to 256 teacher entries, and its gradient over the whole vocabulary.
//
// With x a row's logits, k2 = log2(e) / tau, K the used teacher ids and T the rest of the
// vocabulary, the rows' sums are kept apart: (m_T, s_T) over T while the row streams past
// (the entries' own elements are replaced by -inf where they sit in registers), and
// (m_K, s_K) from the k gathered logits. The tail's mass Q_T = s_T 2^(m_T - lse) is then a
// sum of its own and keeps its relative precision where the teacher's entries hold nearly
// everything (1 - sum q_i would lose it all). Outside K the gradient is one factor of
// 2^(x k2 - m_T):
//   forward:  c (P 2^(m_T - lse) - p_T / s_T),   reverse:  c 2^(m_T - lse) (log(Q_T/p_T) - l),
// with c = weight m / (loss_norm L tau) and P = sum p_i + p_T; on K each entry has its own
// value, which takes the element's place before its vector is stored.

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <cstring>

#include "context.hpp"
#include "grpo_device.hpp"
#include "grpo_launch.hpp"
#include "pcp_distill.h"

namespace pcp {
namespace {

constexpr int kMaxEntries = PCP_TOP_LOGITS_MAX;
constexpr int kWave = 64;
constexpr int kSlots = kMaxEntries / kWave;   // entries per lane: entry i is slot i / 64 of lane i % 64

struct DistillArgs {
  const void* logits;
  const void* tids;
  const float* tlogits;
  const float* tlse;        // nullptr: the entries renormalised
  const void* mask;         // nullptr: all ones
  const float* seq_scale;   // [n_seq]: weight / (loss_norm * max(sum mask, 1))
  void* dlogits;
  float* token_loss;
  float4* part;             // [nrows, parts]: (m_T, s_T, an id is used twice, -)
  float* part_z;            // [nrows, k] the entries' logits (dlogits may replace them)
  int* err;
  int64_t nrows, vocab, rows, logit_stride, tok_stride, tok_offset;
  int64_t row0;             // first row of this launch
  double inv_tau;
  float k2;                 // log2(e) / tau
  int32_t k, ids_i64, mask_u8, forward;
  int32_t parts, per;       // workgroups per row, 16-byte vectors per workgroup
};

struct DistillRow {
  int64_t row, tix;
  float w;
  int32_t seq;
  bool tok;
};

__device__ __forceinline__ DistillRow distill_row(const DistillArgs& a, int64_t row) {
  DistillRow r;
  r.row = row;
  const int64_t s = static_cast<uint32_t>(row) / static_cast<uint32_t>(a.logit_stride);
  const int64_t t = row - s * a.logit_stride;
  r.seq = static_cast<int32_t>(s);
  r.tok = t < a.rows;
  r.tix = s * a.tok_stride + a.tok_offset + t;
  r.w = 0.f;
  if (r.tok) {
    if (a.mask == nullptr) r.w = 1.f;
    else if (a.mask_u8) r.w = static_cast<const uint8_t*>(a.mask)[r.tix] ? 1.f : 0.f;
    else r.w = static_cast<const float*>(a.mask)[r.tix];
  }
  return r;
}

// Entry i of a row: its id, or -1 when it is unused, -2 when its id is out of range.
__device__ __forceinline__ int entry_id(const DistillArgs& a, int64_t row, int i, float& t) {
  t = kNegInf;
  if (i >= a.k) return -1;
  const int64_t e = row * a.k + i;
  const int64_t id = a.ids_i64 ? static_cast<const int64_t*>(a.tids)[e]
                               : static_cast<int64_t>(static_cast<const int32_t*>(a.tids)[e]);
  t = a.tlogits[e];
  if (id == PCP_IGNORE_INDEX || t == kNegInf) return -1;
  return id >= 0 && id < a.vocab ? static_cast<int>(id) : -2;
}

// Where a workgroup of BLOCK lanes that holds vectors [v0, v0 + U * BLOCK) of a row's interior
// has element `it` of it, as chunk << 16 | thread << 4 | element of the lane's chunk; -1 if it
// has not. SPLIT: the two-halves layout of load_chunk.
template <typename TI, bool SPLIT, int BLOCK, int U>
__device__ __forceinline__ int entry_place(int it, int v0) {
  constexpr int EPV = 16 / TI::kBytes;
  const int rel = it - v0 * EPV;
  if (it < 0 || rel < 0 || rel >= U * BLOCK * EPV) return -1;
  if constexpr (SPLIT) {
    const int g = rel >> 2, r = g % (2 * BLOCK);
    return (g / (2 * BLOCK)) << 16 | (64 * (r >> 7) + (r & 63)) << 4 | 4 * ((r >> 6) & 1) | (rel & 3);
  } else {
    const int v = rel / EPV;
    return (v / BLOCK) << 16 | (v % BLOCK) << 4 | rel % EPV;
  }
}

// Lane `lane`'s element `slot` of a vector becomes -inf.
template <typename TI>
__device__ __forceinline__ void mask_element(u32x4& v, bool here, int slot) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if constexpr (TI::kBytes == 4) {
      if (here && slot == w) v[w] = 0xff800000u;
    } else {
      constexpr uint32_t kInf = __is_same(TI, BF16T) ? 0xff80u : 0xfc00u;
      const uint32_t keep = (slot & 1) ? 0xffffu : 0xffff0000u, put = (slot & 1) ? kInf << 16 : kInf;
      if (here && (slot >> 1) == w) v[w] = (v[w] & keep) | put;
    }
  }
}

// The entries' elements that this wave holds become -inf; true if one of their ids is used
// twice. id / place: the lane's entries (slots of the wave).
template <typename TI, int U>
__device__ __forceinline__ bool mask_entries(u32x4 (&x)[U], const int (&id)[kSlots], const int (&place)[kSlots]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  bool twice = false;
#pragma unroll
  for (int s = 0; s < kSlots; ++s) {
    uint64_t mine = __ballot(place[s] >= 0 && ((place[s] >> 10) & 15) == wave);
    while (mine) {
      const int src = __builtin_ctzll(mine);
      mine &= mine - 1;
      const int p = __builtin_amdgcn_readlane(place[s], src), want = __builtin_amdgcn_readlane(id[s], src);
      int n = 0;
#pragma unroll
      for (int o = 0; o < kSlots; ++o) n += __popcll(__ballot(id[o] == want));
      twice |= n > 1;
      const int q = p >> 16;
      const bool here = ((p >> 4) & 63) == lane;
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (k == q) mask_element<TI>(x[k], here, p & 15);
    }
  }
  return twice;
}

// The thread (one of the first 14) that handles a row's element outside its interior.
template <typename TI>
__device__ __forceinline__ int edge_thread(const RowSpan& sp, int id) {
  constexpr int EPV = 16 / TI::kBytes;
  if (id < 0) return -1;
  if (id < sp.head) return id;
  const int past = id - sp.head - sp.nv * EPV;
  return past >= 0 ? sp.head + past : -1;
}

// The same for the head and tail elements: xe is this lane's (wave 0 only).
template <typename TI>
__device__ __forceinline__ bool mask_edges(const RowSpan& sp, float& xe, const int (&id)[kSlots]) {
  bool twice = false;
#pragma unroll
  for (int s = 0; s < kSlots; ++s) {
    const int owner = edge_thread<TI>(sp, id[s]);
    uint64_t at = __ballot(owner >= 0);
    while (at) {
      const int src = __builtin_ctzll(at);
      at &= at - 1;
      const int want = __builtin_amdgcn_readlane(id[s], src), thread = __builtin_amdgcn_readlane(owner, src);
      int n = 0;
#pragma unroll
      for (int o = 0; o < kSlots; ++o) n += __popcll(__ballot(id[o] == want));
      twice |= n > 1;
      if (static_cast<int>(threadIdx.x) == thread) xe = kNegInf;
    }
  }
  return twice;
}

// A row's teacher, staged in LDS by the first wave for the whole workgroup.
struct Teacher {
  double log_p[kMaxEntries];
  int id[kMaxEntries];
  float z[kMaxEntries];     // the student's logits there
  float p[kMaxEntries];
  double sum_p;
  float mk, sk;             // the entries' log-sum-exp state, base 2
  int used, bad;
};

// z_at(i, id): the student's logit at entry i. Called by all lanes of one wave.
template <typename F>
__device__ __forceinline__ void stage_teacher(const DistillArgs& a, const DistillRow& r, Teacher& te, F z_at) {
  const int lane = threadIdx.x & 63;
  int id[kSlots];
  float t[kSlots], z[kSlots];
  bool out = false, any = false;
  float tmax = kNegInf, zmax = kNegInf;
#pragma unroll
  for (int s = 0; s < kSlots; ++s) {
    id[s] = entry_id(a, r.row, lane + kWave * s, t[s]);
    out |= id[s] == -2;
    any |= id[s] >= 0;
    if (id[s] < 0) t[s] = kNegInf;
    z[s] = id[s] >= 0 ? z_at(lane + kWave * s, id[s]) : kNegInf;
    tmax = fmaxf(tmax, t[s]);
    zmax = fmaxf(zmax, z[s]);
  }
  const float mk = lanes_max<64>(zmax) * a.k2;
  double ref;
  if (a.tlse) ref = static_cast<double>(a.tlse[r.row]);
  else {
    const double m = static_cast<double>(ms_ref(lanes_max<64>(tmax))) * a.inv_tau;
    double e = 0.;
#pragma unroll
    for (int s = 0; s < kSlots; ++s)
      if (id[s] >= 0) e += exp(static_cast<double>(t[s]) * a.inv_tau - m);
    ref = m + log(wave_sum64(e));
  }
  double sum_p = 0.;
  float sk = 0.f;
#pragma unroll
  for (int s = 0; s < kSlots; ++s) {
    const int i = lane + kWave * s;
    const double lp = static_cast<double>(t[s]) * a.inv_tau - ref;
    const double p = id[s] >= 0 ? exp(lp) : 0.;
    sum_p += p;
    if (id[s] >= 0) sk += hw_exp2(fmaf(z[s], a.k2, -ms_ref(mk)));
    te.id[i] = id[s];
    te.z[i] = z[s];
    te.p[i] = static_cast<float>(p);
    te.log_p[i] = lp;
  }
  sum_p = wave_sum64(sum_p);
  sk = lanes_sum<64>(sk);
  const bool bad = __any(out), used = __any(any);
  if (lane == 0) {
    te.sum_p = sum_p;
    te.mk = mk;
    te.sk = sk;
    te.used = used;
    te.bad = bad;
    if (bad) raise_error(a.err, kErrTokenRange);
    else if (used && !__builtin_isfinite(ref)) raise_error(a.err, kErrNonFinite);
  }
}

// What a row's gradient needs: out = tail * 2^(x k2 - ref) outside K, g[] at this lane's
// entries; token: m * l.
struct RowTerms {
  float tail, ref, token;
  float g[kSlots];
};

// mt, st: the state outside K. Every wave of the workgroup computes the same.
__device__ __forceinline__ RowTerms row_terms(const DistillArgs& a, const DistillRow& r, const Teacher& te, float mt,
                                              float st) {
  const int lane = threadIdx.x & 63;
  RowTerms o;
  const float m = fmaxf(mt, te.mk), rm = ms_ref(m);
  const float ft = st == 0.f ? 0.f : hw_exp2(mt - rm);
  const float s = (st == 0.f ? 0.f : st * ft) + (te.sk == 0.f ? 0.f : te.sk * hw_exp2(te.mk - rm));
  const double lse = ms_lse(m, s);
  const float inv_s = 1.f / s;
  const float qt = st * ft * inv_s;
  const bool tail = a.tlse != nullptr && qt >= 0x1p-126f;
  const double pt = tail ? fmax(1. - te.sum_p, PCP_DISTILL_TAIL_FLOOR) : 0.;
  const double tail_gap = tail ? log(pt) - (ms_lse(mt, st) - lse) : 0.;   // log(p_T / q_T)
  const float c = static_cast<float>(static_cast<double>(a.seq_scale[r.seq] * r.w) * a.inv_tau);
  double gap[kSlots], l = 0.;
  float q[kSlots];
#pragma unroll
  for (int e = 0; e < kSlots; ++e) {
    const int i = lane + kWave * e;
    q[e] = 0.f;
    gap[e] = 0.;
    if (kWave * e >= a.k || te.id[i] < 0) continue;
    q[e] = hw_exp2(fmaf(te.z[i], a.k2, -rm)) * inv_s;
    const double log_q = static_cast<double>(te.z[i]) * static_cast<double>(a.k2) * 0.69314718055994530942 - lse;
    gap[e] = te.log_p[i] - log_q;                                         // log(p_i / q_i)
    if (a.forward ? te.p[i] > 0.f : q[e] > 0.f) l += a.forward ? te.p[i] * gap[e] : -q[e] * gap[e];
  }
  l = wave_sum64(l);
  if (a.forward) {
    l += pt > 0. ? pt * tail_gap : 0.;
    const float big_p = static_cast<float>(te.sum_p + pt);
    o.tail = st == 0.f ? 0.f : c * (big_p * ft * inv_s - static_cast<float>(pt) / st);
#pragma unroll
    for (int e = 0; e < kSlots; ++e) o.g[e] = kWave * e < a.k ? c * (q[e] * big_p - te.p[lane + kWave * e]) : 0.f;
  } else {
    l -= tail ? qt * tail_gap : 0.;
    const float lf = static_cast<float>(l);
    o.tail = st == 0.f ? 0.f : -c * (ft * inv_s) * (static_cast<float>(tail_gap) + lf);
#pragma unroll
    for (int e = 0; e < kSlots; ++e) o.g[e] = q[e] > 0.f ? -c * q[e] * (static_cast<float>(gap[e]) + lf) : 0.f;
  }
  o.ref = ms_ref(mt);
  o.token = r.w * static_cast<float>(l);
  if (threadIdx.x == 0 && !(__builtin_isfinite(lse) && __builtin_isfinite(te.sum_p) && l == l))
    raise_error(a.err, kErrNonFinite);
  return o;
}

// ---------------------------------------------------------------------------
// Rows in parts: workgroups of 256 lanes take `per` vectors of a row each. The first kernel
// leaves each part's (m_T, s_T); in the second every workgroup of a row merges them for
// itself and forms its part of dlogits from a second read of the row.
// ---------------------------------------------------------------------------
constexpr int kPartBlock = 256;
constexpr int kPartU = 8;

template <typename TI>
__global__ void __launch_bounds__(kPartBlock) distill_part_kernel(DistillArgs a) {
  constexpr int EPV = 16 / TI::kBytes, U = kPartU, BLOCK = kPartBlock;
  __shared__ __align__(16) float lds[4 * (BLOCK / 64)];
  __shared__ int any_twice;
  const int tid = threadIdx.x, part = blockIdx.x;
  const int64_t row = a.row0 + blockIdx.y;
  const DistillRow r = distill_row(a, row);
  if (r.w == 0.f) return;
  const char* xrow = static_cast<const char*>(a.logits) + row * a.vocab * TI::kBytes;
  const RowSpan sp = row_span<TI>(xrow, a.vocab);
  const int v0 = part * a.per, end = min(v0 + a.per, sp.nv);
  const __amdgpu_buffer_rsrc_t xbuf = row_rsrc(sp.vec, static_cast<uint32_t>(max(end, 0)) * 16u);
  const uint32_t off = static_cast<uint32_t>(v0 + tid) * 16u;
  u32x4 x[U];
#pragma unroll
  for (int q = 0; q < U; ++q) x[q] = buf_ld16<false>(xbuf, off + q * (BLOCK * 16u));   // read again for dlogits
  if (tid == 0) any_twice = 0;
  int id[kSlots], place[kSlots];
#pragma unroll
  for (int s = 0; s < kSlots; ++s) {
    float t;
    const int i = (tid & 63) + kWave * s;
    id[s] = entry_id(a, row, i, t);
    place[s] = id[s] >= 0 && id[s] - sp.head < end * EPV ? entry_place<TI, false, BLOCK, U>(id[s] - sp.head, v0) : -1;
    if (part == 0 && tid < 64 && i < a.k) a.part_z[row * a.k + i] = id[s] >= 0 ? TI::load1(xrow, id[s]) : 0.f;
  }
  bool twice = mask_entries<TI, U>(x, id, place);
  float xe = kNegInf;
  if (part == 0 && tid < 64) {
    const int ek = edge_index<TI>(sp, tid);
    if (ek >= 0) xe = TI::load1(xrow, ek);
    twice |= mask_edges<TI>(sp, xe, id);
  }
  float bx = xe;
#pragma unroll
  for (int q = 0; q < U; ++q)
    if (v0 + q * BLOCK + tid < end) bx = vec_max<TI>(bx, x[q]);
  float m = bx * a.k2, s = 0.f, m0 = kNegInf, s0 = 0.f;
  const float ref = ms_ref(m);
  s = hw_exp2(fmaf(xe, a.k2, -ref));
#pragma unroll
  for (int q = 0; q < U; ++q)
    if (v0 + q * BLOCK + tid < end) {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(&x[q]);
#pragma unroll
      for (int j = 0; j < EPV; ++j) s += hw_exp2(fmaf(TI::unpack(w, j), a.k2, -ref));
    }
  __syncthreads();
  if (twice && (tid & 63) == 0) any_twice = 1;
  block_merge2<BLOCK>(m, s, m0, s0, lds);
  if (tid == 0) a.part[row * a.parts + part] = make_float4(m, s, any_twice ? 1.f : 0.f, 0.f);
}

// The row's state outside K from its parts, and whether an id is used twice.
__device__ __forceinline__ void merge_tail(const DistillArgs& a, int64_t row, float& m, float& s, bool& twice) {
  const int lane = threadIdx.x & 63;
  m = kNegInf;
  s = 0.f;
  bool t = false;
  for (int p = lane; p < a.parts; p += 64) {
    const float4 v = a.part[row * a.parts + p];
    const float M = fmaxf(m, v.x);
    s = ms_rescale(s, m, M) + ms_rescale(v.y, v.x, M);
    m = M;
    t |= v.z != 0.f;
  }
  lanes_merge<64>(m, s);
  twice = __any(t);
}

// GRAD false: one wave per row, the loss alone. SCALAR: dlogits rows that do not split as the
// logits rows do (another address mod 16), stored element by element.
template <typename TI, typename TO, bool GRAD, bool SCALAR>
__global__ void __launch_bounds__(kPartBlock) distill_part_grad_kernel(DistillArgs a) {
  constexpr int EPV = 16 / TI::kBytes, U = kPartU, BLOCK = kPartBlock;
  constexpr bool kSplit = TI::kBytes == 2 && TO::kBytes == 4;
  constexpr uint32_t kOutVec = EPV * TO::kBytes;
  static_assert(!(SCALAR && kSplit), "f32 dlogits of 16-bit rows are stored at any element");
  __shared__ Teacher te;
  const int tid = threadIdx.x, part = blockIdx.x;
  const int64_t row = a.row0 + blockIdx.y, row_elem = row * a.vocab;
  const DistillRow r = distill_row(a, row);
  const char* xrow = static_cast<const char*>(a.logits) + row_elem * TI::kBytes;
  const RowSpan sp = row_span<TI>(xrow, a.vocab);
  const int ek = part == 0 ? edge_index<TI>(sp, tid) : -1;
  const int v0 = part * a.per, end = max(min(v0 + a.per, sp.nv), 0);
  char* drow0 = static_cast<char*>(a.dlogits) + (row_elem + sp.head) * TO::kBytes;
  const __amdgpu_buffer_rsrc_t drow = row_rsrc(drow0, GRAD ? static_cast<uint32_t>(end) * kOutVec : 0u);
  const uint32_t sgrp = split_group<TI, TO, BLOCK>(tid);
  auto group = [&](int q, int h) { return static_cast<uint32_t>(2 * (v0 + q * BLOCK) + 64 * h) + sgrp; };
  u32x4 x[U];
  float xe = 0.f;
  bool live = r.w != 0.f;
  float mt = kNegInf, st = 0.f;
  if (live) {
    if constexpr (GRAD) {
      const __amdgpu_buffer_rsrc_t xbuf = row_rsrc(sp.vec, static_cast<uint32_t>(end) * 16u);
#pragma unroll
      for (int q = 0; q < U; ++q) {
        if constexpr (kSplit) {
          const u32x2 lo = buf_ld8<true>(xbuf, group(q, 0) * 8u), hi = buf_ld8<true>(xbuf, group(q, 1) * 8u);
          x[q] = u32x4{lo[0], lo[1], hi[0], hi[1]};
        } else {
          x[q] = buf_ld16<true>(xbuf, static_cast<uint32_t>(v0 + q * BLOCK + tid) * 16u);
        }
      }
      if (ek >= 0) xe = TI::load1(xrow, ek);
    }
    if (tid < 64) stage_teacher(a, r, te, [&](int i, int) { return a.part_z[row * a.k + i]; });
    bool twice;
    merge_tail(a, row, mt, st, twice);
    __syncthreads();
    if (twice && part == 0 && tid == 0) raise_error(a.err, kErrTeacherTwice);
    live = te.used && !te.bad && !twice;
  }
  RowTerms t;
  t.tail = t.ref = t.token = 0.f;
#pragma unroll
  for (int s = 0; s < kSlots; ++s) t.g[s] = 0.f;
  int place[kSlots], edge[kSlots];
#pragma unroll
  for (int s = 0; s < kSlots; ++s) place[s] = edge[s] = -1;
  if (live) {
    t = row_terms(a, r, te, mt, st);
    if constexpr (GRAD) {
#pragma unroll
      for (int s = 0; s < kSlots; ++s) {
        const int id = te.id[(tid & 63) + kWave * s];
        place[s] = id >= 0 && id - sp.head < end * EPV ? entry_place<TI, kSplit, BLOCK, U>(id - sp.head, v0) : -1;
        if (place[s] >= 0 && ((place[s] >> 10) & 15) != (tid >> 6)) place[s] = -1;
        if (part == 0 && tid < 64) edge[s] = edge_thread<TI>(sp, id);
      }
    }
  }
  if (part == 0 && tid == 0 && r.tok && a.token_loss) a.token_loss[r.tix] = t.token;
  if constexpr (GRAD) {
#pragma unroll
    for (int q = 0; q < U; ++q) {
      float o[EPV];
      if (live) {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(&x[q]);
#pragma unroll
        for (int j = 0; j < EPV; ++j) o[j] = t.tail * hw_exp2(fmaf(TI::unpack(w, j), a.k2, -t.ref));
#pragma unroll
        for (int s = 0; s < kSlots; ++s) {
          uint64_t at = __ballot(place[s] >= 0 && (place[s] >> 16) == q);
          while (at) {
            const int src = __builtin_ctzll(at);
            at &= at - 1;
            const int p = __builtin_amdgcn_readlane(place[s], src);
            const float g = read_lane(t.g[s], src);
            const bool here = ((p >> 4) & 63) == (tid & 63);
#pragma unroll
            for (int j = 0; j < EPV; ++j)
              if (here && j == (p & 15)) o[j] = g;
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < EPV; ++j) o[j] = 0.f;
      }
      if constexpr (kSplit) {
        const float (&o0)[4] = reinterpret_cast<const float (&)[4]>(o[0]);
        const float (&o1)[4] = reinterpret_cast<const float (&)[4]>(o[4]);
        buf_store_vals<TO, 4, true>(drow, group(q, 0) * 16u, o0);
        buf_store_vals<TO, 4, true>(drow, group(q, 1) * 16u, o1);
      } else if constexpr (SCALAR) {
        const int vi = v0 + q * BLOCK + tid;
        if (vi < end) {
#pragma unroll
          for (int j = 0; j < EPV; ++j) store1<TO>(drow0, static_cast<int64_t>(vi) * EPV + j, o[j]);
        }
      } else {
        buf_store_vals<TO, EPV, true>(drow, static_cast<uint32_t>(v0 + q * BLOCK + tid) * kOutVec, o);
      }
    }
    if (part == 0 && tid < 64) {
      float o = live && ek >= 0 ? t.tail * hw_exp2(fmaf(xe, a.k2, -t.ref)) : 0.f;
      if (live) {
#pragma unroll
        for (int s = 0; s < kSlots; ++s) {
          uint64_t at = __ballot(edge[s] >= 0);
          while (at) {
            const int src = __builtin_ctzll(at);
            at &= at - 1;
            const int thread = __builtin_amdgcn_readlane(edge[s], src);
            const float g = read_lane(t.g[s], src);
            if (tid == thread) o = g;
          }
        }
      }
      if (ek >= 0) store1<TO>(a.dlogits, row_elem + ek, o);
    }
  }
}

// ---------------------------------------------------------------------------
// Launches.
// ---------------------------------------------------------------------------
template <typename TI, typename TO>
hipError_t launch_parts(DistillArgs a, hipStream_t st) {
  const bool scalar = a.dlogits && TI::kBytes == TO::kBytes &&
                      ((reinterpret_cast<uintptr_t>(a.logits) ^ reinterpret_cast<uintptr_t>(a.dlogits)) & 15u) != 0;
  constexpr int64_t kRows = 65535;   // grid.y
  for (int64_t r0 = 0; r0 < a.nrows; r0 += kRows) {
    a.row0 = r0;
    const unsigned n = static_cast<unsigned>(a.nrows - r0 < kRows ? a.nrows - r0 : kRows);
    const dim3 g(static_cast<unsigned>(a.parts), n), b(kPartBlock);
    distill_part_kernel<TI><<<g, b, 0, st>>>(a);
    if (!a.dlogits) {
      distill_part_grad_kernel<TI, TO, false, false><<<dim3(1, n), dim3(64), 0, st>>>(a);
    } else if constexpr (TI::kBytes == TO::kBytes) {
      if (scalar) distill_part_grad_kernel<TI, TO, true, true><<<g, b, 0, st>>>(a);
      else distill_part_grad_kernel<TI, TO, true, false><<<g, b, 0, st>>>(a);
    } else {
      distill_part_grad_kernel<TI, TO, true, false><<<g, b, 0, st>>>(a);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

hipError_t launch_distill(const DistillArgs& a, int in_dtype, int out_dtype, hipStream_t st) {
  if (in_dtype == PCP_BF16)
    return out_dtype == PCP_F32 ? launch_parts<BF16T, F32T>(a, st) : launch_parts<BF16T, BF16T>(a, st);
  if (in_dtype == PCP_F16)
    return out_dtype == PCP_F32 ? launch_parts<F16T, F32T>(a, st) : launch_parts<F16T, F16T>(a, st);
  return launch_parts<F32T, F32T>(a, st);
}

inline size_t round256(size_t b) { return (b + 255) & ~static_cast<size_t>(255); }

inline bool misaligned(const void* p, int size) {
  return (reinterpret_cast<uintptr_t>(p) & static_cast<uintptr_t>(size - 1)) != 0;
}

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
  const int64_t parts = nv > 0 ? (nv + kPartBlock * kPartU - 1) / (kPartBlock * kPartU) : 1;
  // Scratch: seq_len | seq_scale | seq_val | loss, ticket | token_loss | parts | entries' logits.
  const size_t sv = round256(sizeof(float) * static_cast<size_t>(a->n_seq));
  const size_t tl = a->token_loss ? 0 : round256(sizeof(float) * static_cast<size_t>(a->n_seq * tstride));
  const size_t pb = round256(sizeof(float4) * static_cast<size_t>(nrows) * static_cast<size_t>(parts));
  const size_t zb = sizeof(float) * static_cast<size_t>(nrows) * static_cast<size_t>(a->k);
  const int rc = ensure_scratch_on(ctx, 3 * sv + 512 + tl + pb + zb, st);
  if (rc != PCP_OK) return rc;
  char* sp = static_cast<char*>(ctx->scratch);
  float* s_len = reinterpret_cast<float*>(sp);
  float* s_scale = reinterpret_cast<float*>(sp + sv);
  float* s_val = reinterpret_cast<float*>(sp + 2 * sv);
  float* s_loss = reinterpret_cast<float*>(sp + 3 * sv);
  int* s_done = reinterpret_cast<int*>(sp + 3 * sv + 256);
  float* s_tl = a->token_loss ? a->token_loss : reinterpret_cast<float*>(sp + 3 * sv + 512);

  // weight / loss_norm as one divisor: the loss and every scale below carry both.
  const float norm = (a->loss_norm > 0.f ? a->loss_norm : static_cast<float>(a->n_seq)) / a->weight;
  StepPrepArgs pa;
  std::memset(&pa, 0, sizeof(pa));
  pa.mask = a->mask;
  pa.mask_u8 = a->mask_dtype == PCP_BOOL;
  pa.n_seq = a->n_seq;
  pa.rows = a->rows;
  pa.tok_stride = tstride;
  pa.tok_offset = a->tok_offset;
  pa.loss_norm = norm;
  pa.seq_len = s_len;
  pa.seq_scale = s_scale;
  pa.zero[0] = s_done;

  DistillArgs d;
  std::memset(&d, 0, sizeof(d));
  d.logits = a->logits;
  d.tids = a->teacher_ids;
  d.tlogits = a->teacher_logits;
  d.tlse = a->teacher_lse;
  d.mask = a->mask;
  d.seq_scale = s_scale;
  d.dlogits = a->dlogits;
  d.token_loss = s_tl;
  d.part = reinterpret_cast<float4*>(sp + 3 * sv + 512 + tl);
  d.part_z = reinterpret_cast<float*>(sp + 3 * sv + 512 + tl + pb);
  d.err = ctx->d_page->err;
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
  d.mask_u8 = pa.mask_u8;
  d.forward = a->divergence == PCP_DIVERGENCE_FORWARD;
  d.parts = static_cast<int32_t>(parts);
  d.per = static_cast<int32_t>((nv + parts - 1) / parts);

  hipError_t e = launch_step_prep(pa, st);
  if (e != hipSuccess) return hip_fail(ctx, e, "step prep launch");
  const bool timed = prof_begin(ctx, st);
  e = launch_distill(d, a->logits_dtype, a->dlogits ? a->dlogits_dtype : a->logits_dtype, st);
  prof_end(ctx, st, timed);
  if (e != hipSuccess) return hip_fail(ctx, e, "distillation launch");
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
