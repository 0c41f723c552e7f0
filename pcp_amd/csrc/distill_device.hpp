// Kernels of the distillation from a teacher's top logits (pcp_distill.h): the loss of a row against up
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
#pragma once

#include <hip/hip_runtime.h>

#include <atomic>
#include <cstdint>

#include "grpo_device.hpp"
#include "grpo_launch.hpp"
#include "pcp_distill.h"

namespace pcp {

// The widest rows that a workgroup keeps in registers, in 16-byte vectors.
constexpr int64_t kDistillRowVecs = 1024 * 19;

constexpr int kMaxEntries = PCP_TOP_LOGITS_MAX;
constexpr int kWave = 64;
// Entry i is slot i / 64 of lane i % 64; kernels are compiled for 1 slot (k <= 64) and for 4.
constexpr int kMaxSlots = kMaxEntries / kWave;

// What a row's teacher comes to, whatever the student.
struct TeacherRow {
  double sum_p;     // of the entries
  double log_pt;    // of the tail's class, if there is one
  double lse;       // the entries' probabilities are exp(t / tau - lse)
  float pt;
  int32_t state;    // kUnused, kUsed; kBad: an id out of range
};
constexpr int kUnused = 0, kUsed = 1, kBad = 2;

struct DistillArgs {
  const void* logits;
  const void* tids;
  const float* tlogits;
  const float* tlse;        // nullptr: the entries renormalised
  const void* mask;         // nullptr: all ones
  float* seq_len;           // [n_seq]: max(sum mask, 1), and
  float* seq_scale;         // [n_seq]: weight / (loss_norm * seq_len), by the preparation
  void* dlogits;
  float* token_loss;
  float4* part;             // [nrows, parts]: (m_T, s_T, an id is used twice, -)
  float* part_z;            // [nrows, k] the entries' logits (dlogits may replace them)
  TeacherRow* teacher;      // [nrows], by the preparation, and
  float* teacher_p;         // [nrows, k]
  int* err;
  int* next_row;            // rows handed out past the first grid (zeroed earlier on the stream)
  int64_t nrows, vocab, rows, logit_stride, tok_stride, tok_offset;
  int64_t row0;             // first row of this launch
  double inv_tau;
  int64_t n_seq;
  int* done;                // the loss reduction's ticket
  float loss_norm;          // loss_norm / weight
  float k2;                 // log2(e) / tau
  int32_t k, ids_i64, mask_u8, forward;
  int32_t parts, per;       // workgroups per row (0: a row to a workgroup), 16-byte vectors per workgroup
  int32_t turn;             // rows dealt in grid strides: how far on each stride starts
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
template <typename TI, int U, int NS>
__device__ __forceinline__ bool mask_entries(u32x4 (&x)[U], const int (&id)[NS], const int (&place)[NS]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  bool twice = false;
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    uint64_t mine = __ballot(place[s] >= 0 && ((place[s] >> 10) & 15) == wave);
    while (mine) {
      const int src = __builtin_ctzll(mine);
      mine &= mine - 1;
      const int p = __builtin_amdgcn_readlane(place[s], src), want = __builtin_amdgcn_readlane(id[s], src);
      int n = 0;
#pragma unroll
      for (int o = 0; o < NS; ++o) n += __popcll(__ballot(id[o] == want));
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
template <typename TI, int NS>
__device__ __forceinline__ bool mask_edges(const RowSpan& sp, float& xe, const int (&id)[NS]) {
  bool twice = false;
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    const int owner = edge_thread<TI>(sp, id[s]);
    uint64_t at = __ballot(owner >= 0);
    while (at) {
      const int src = __builtin_ctzll(at);
      at &= at - 1;
      const int want = __builtin_amdgcn_readlane(id[s], src), thread = __builtin_amdgcn_readlane(owner, src);
      int n = 0;
#pragma unroll
      for (int o = 0; o < NS; ++o) n += __popcll(__ballot(id[o] == want));
      twice |= n > 1;
      if (static_cast<int>(threadIdx.x) == thread) xe = kNegInf;
    }
  }
  return twice;
}

// ---- the preparation -------------------------------------------------------------------
// Everything that needs 64-bit exponentials and logarithms is done ahead, one wave per row:
// in the row kernel their constants alone took 60 registers of its 128.

// Sequence s: its length and scale, summed in a fixed order by the workgroup.
constexpr int kPrepBlock = 256;
__device__ __forceinline__ void prepare_sequence(const DistillArgs& a, int64_t s, float* lds) {
  float acc = 0.f;
  const int64_t base = s * a.tok_stride + a.tok_offset;
  for (int64_t t = threadIdx.x; t < a.rows; t += kPrepBlock)
    acc += a.mask == nullptr ? 1.f
           : a.mask_u8       ? (static_cast<const uint8_t*>(a.mask)[base + t] ? 1.f : 0.f)
                             : static_cast<const float*>(a.mask)[base + t];
  acc = lanes_sum<64>(acc);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = acc;
  __syncthreads();
  if (threadIdx.x != 0) return;
  float total = 0.f;
  for (int w = 0; w < kPrepBlock / 64; ++w) total += lds[w];
  const float len = fmaxf(total, 1.f);
  a.seq_len[s] = len;
  a.seq_scale[s] = 1.f / (a.loss_norm * len);
  if (s == 0) {
    *a.done = 0;
    *a.next_row = 0;
  }
}

// Row `row`'s teacher, by one wave.
__device__ __forceinline__ void prepare_teacher(const DistillArgs& a, int64_t row) {
  if (distill_row(a, row).w == 0.f) return;
  const int lane = threadIdx.x & 63;
  int id[kMaxSlots];
  float t[kMaxSlots], tmax = kNegInf;
  bool out = false, any = false;
#pragma unroll
  for (int s = 0; s < kMaxSlots; ++s) {
    id[s] = -1;
    if (kWave * s < a.k) id[s] = entry_id(a, row, lane + kWave * s, t[s]);
    out |= id[s] == -2;
    any |= id[s] >= 0;
    if (id[s] >= 0) tmax = fmaxf(tmax, t[s]);
  }
  TeacherRow o;
  if (a.tlse) {
    o.lse = static_cast<double>(a.tlse[row]);
  } else {
    const double m = static_cast<double>(ms_ref(lanes_max<64>(tmax))) * a.inv_tau;
    double sum = 0.;
#pragma unroll
    for (int s = 0; s < kMaxSlots; ++s)
      if (id[s] >= 0) sum += exp(static_cast<double>(t[s]) * a.inv_tau - m);
    o.lse = m + log(wave_sum64(sum));
  }
  double sum_p = 0.;
#pragma unroll
  for (int s = 0; s < kMaxSlots; ++s) {
    const int i = lane + kWave * s;
    if (i >= a.k) continue;
    const double p = id[s] >= 0 ? exp(static_cast<double>(t[s]) * a.inv_tau - o.lse) : 0.;
    sum_p += p;
    a.teacher_p[row * a.k + i] = static_cast<float>(p);
  }
  o.sum_p = wave_sum64(sum_p);
  const double pt = fmax(1. - o.sum_p, PCP_DISTILL_TAIL_FLOOR);
  o.log_pt = log(pt);
  o.pt = static_cast<float>(pt);
  o.state = __any(out) ? kBad : __any(any) ? kUsed : kUnused;
  if (lane != 0) return;
  a.teacher[row] = o;
  if (o.state == kBad) raise_error(a.err, kErrTokenRange);
  else if (o.state == kUsed && !(__builtin_isfinite(o.lse) && __builtin_isfinite(o.sum_p)))
    raise_error(a.err, kErrNonFinite);
}

// Workgroup `block` of the preparation: a sequence, or a row per wave.
__device__ __forceinline__ void prepare(const DistillArgs& a, int64_t block, float* lds) {
  if (block < a.n_seq) {
    prepare_sequence(a, block, lds);
    return;
  }
  const int64_t row = (block - a.n_seq) * (kPrepBlock / 64) + (threadIdx.x >> 6);
  if (row < a.nrows) prepare_teacher(a, row);
}
inline int64_t prepare_blocks(const DistillArgs& a) {
  return a.n_seq + (a.nrows + kPrepBlock / 64 - 1) / (kPrepBlock / 64);
}

// A kernel template like the others, so that every type's file may hold it.
template <int BLOCK>
__global__ void __launch_bounds__(BLOCK) distill_prepare_kernel(DistillArgs a) {
  __shared__ float lds[BLOCK / 64];
  prepare(a, blockIdx.x, lds);
}

// ---- a row's terms -----------------------------------------------------------------------
// A row's teacher and the student's logits there, in LDS for the whole workgroup.
struct Teacher {
  TeacherRow row;
  int id[kMaxEntries];
  float t[kMaxEntries];
  float p[kMaxEntries];
  float z[kMaxEntries];     // the student's logits
  float mk, sk;             // their log-sum-exp state, base 2
};

// What a row's gradient needs: tail * 2^(x k2 - ref) outside K, g[] at the entries.
struct RowTerms {
  float tail, ref;
  float g[kMaxEntries];
};

// A row's entries to LDS, by one wave, in steps: the loads, the stores, the student's part.
template <int NS>
struct Entries {
  int id[NS];
  float t[NS], p[NS];
};
template <int NS>
__device__ __forceinline__ void load_entries(const DistillArgs& a, int64_t row, Entries<NS>& e) {
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    const int i = static_cast<int>(threadIdx.x & 63) + kWave * s;
    e.id[s] = entry_id(a, row, i, e.t[s]);
    e.p[s] = i < a.k ? a.teacher_p[row * a.k + i] : 0.f;
  }
}
template <int NS>
__device__ __forceinline__ void put_entries(const DistillArgs& a, int64_t row, Teacher& te, const Entries<NS>& e) {
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    const int i = static_cast<int>(threadIdx.x & 63) + kWave * s;
    te.id[i] = e.id[s];
    te.t[i] = e.t[s];
    te.p[i] = e.p[s];
  }
  if ((threadIdx.x & 63) == 0) te.row = a.teacher[row];
}
template <int NS>
__device__ __forceinline__ void put_student(const DistillArgs& a, Teacher& te, const float (&z)[NS]) {
  const int lane = threadIdx.x & 63;
  float zmax = kNegInf, sk = 0.f;
  bool used[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    used[s] = te.id[lane + kWave * s] >= 0;
    te.z[lane + kWave * s] = z[s];
    if (used[s]) zmax = fmaxf(zmax, z[s]);
  }
  const float mk = lanes_max<64>(zmax) * a.k2;
#pragma unroll
  for (int s = 0; s < NS; ++s)
    if (used[s]) sk += hw_exp2(fmaf(z[s], a.k2, -ms_ref(mk)));
  sk = lanes_sum<64>(sk);
  if (lane == 0) {
    te.mk = mk;
    te.sk = sk;
  }
}

// By all lanes of one wave, into LDS; returns m * l. mt, st: the state outside K.
template <int NS>
__device__ __forceinline__ float row_terms(const DistillArgs& a, const DistillRow& r, const Teacher& te, float mt,
                                           float st, RowTerms& o) {
  const int lane = threadIdx.x & 63;
  const float m = fmaxf(mt, te.mk), rm = ms_ref(m);
  const float ft = st == 0.f ? 0.f : hw_exp2(mt - rm);
  const float s = (st == 0.f ? 0.f : st * ft) + (te.sk == 0.f ? 0.f : te.sk * hw_exp2(te.mk - rm));
  const double lse = ms_lse(m, s);
  const float inv_s = 1.f / s;
  const float qt = st * ft * inv_s;
  const bool tail = a.tlse != nullptr && qt >= 0x1p-126f;
  const float pt = tail ? te.row.pt : 0.f;
  const double tail_gap = tail ? te.row.log_pt - (ms_lse(mt, st) - lse) : 0.;   // log(p_T / q_T)
  const float c = static_cast<float>(static_cast<double>(a.seq_scale[r.seq] * r.w) * a.inv_tau);
  double gap[NS], l = 0.;
  float q[NS];
#pragma unroll
  for (int e = 0; e < NS; ++e) {
    const int i = lane + kWave * e;
    q[e] = 0.f;
    gap[e] = 0.;
    if (kWave * e >= a.k || te.id[i] < 0) continue;
    q[e] = hw_exp2(fmaf(te.z[i], a.k2, -rm)) * inv_s;
    const double log_q = static_cast<double>(te.z[i]) * static_cast<double>(a.k2) * 0.69314718055994530942 - lse;
    gap[e] = static_cast<double>(te.t[i]) * a.inv_tau - te.row.lse - log_q;   // log(p_i / q_i)
    if (a.forward ? te.p[i] > 0.f : q[e] > 0.f) l += a.forward ? te.p[i] * gap[e] : -q[e] * gap[e];
  }
  l = wave_sum64(l);
  float tail_factor;
  if (a.forward) {
    l += pt > 0.f ? pt * tail_gap : 0.;
    const float big_p = static_cast<float>(te.row.sum_p + pt);
    tail_factor = st == 0.f ? 0.f : c * (big_p * ft * inv_s - pt / st);
#pragma unroll
    for (int e = 0; e < NS; ++e)
      if (kWave * e < a.k) o.g[lane + kWave * e] = c * (q[e] * big_p - te.p[lane + kWave * e]);
  } else {
    l -= tail ? qt * tail_gap : 0.;
    const float lf = static_cast<float>(l);
    tail_factor = st == 0.f ? 0.f : -c * (ft * inv_s) * (static_cast<float>(tail_gap) + lf);
#pragma unroll
    for (int e = 0; e < NS; ++e)
      if (kWave * e < a.k) o.g[lane + kWave * e] = q[e] > 0.f ? -c * q[e] * (static_cast<float>(gap[e]) + lf) : 0.f;
  }
  if (lane == 0) {
    o.tail = tail_factor;
    o.ref = ms_ref(mt);
  }
  if (lane == 0 && !(__builtin_isfinite(lse) && l == l))
    raise_error(a.err, kErrNonFinite);
  return r.w * static_cast<float>(l);
}

// ---------------------------------------------------------------------------
// Rows in parts: workgroups of 256 lanes take `per` vectors of a row each. The first kernel
// leaves each part's (m_T, s_T); in the second every workgroup of a row merges them for
// itself and forms its part of dlogits from a second read of the row.
// ---------------------------------------------------------------------------
constexpr int kPartBlock = 256;
constexpr int kPartU = 8;

template <typename TI, int NS>
__global__ void __launch_bounds__(kPartBlock) distill_part_kernel(DistillArgs a, int n) {
  constexpr int EPV = 16 / TI::kBytes, U = kPartU, BLOCK = kPartBlock;
  __shared__ __align__(16) float lds[4 * (BLOCK / 64)];
  __shared__ int any_twice;
  const int tid = threadIdx.x, part = blockIdx.x;
  static_assert(kPartBlock == kPrepBlock, "the preparation's workgroup");
  if (blockIdx.y >= static_cast<unsigned>(n)) {   // past the rows: the preparation
    if (part == 0) prepare(a, blockIdx.y - n, lds);
    return;
  }
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
  int id[NS], place[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    float t;
    const int i = (tid & 63) + kWave * s;
    id[s] = entry_id(a, row, i, t);
    place[s] = id[s] >= 0 && id[s] - sp.head < end * EPV ? entry_place<TI, false, BLOCK, U>(id[s] - sp.head, v0) : -1;
    if (part == 0 && tid < 64 && i < a.k) a.part_z[row * a.k + i] = id[s] >= 0 ? TI::load1(xrow, id[s]) : 0.f;
  }
  bool twice = mask_entries<TI>(x, id, place);
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
template <typename TI, typename TO, int NS, bool GRAD, bool SCALAR>
__global__ void __launch_bounds__(kPartBlock) distill_part_grad_kernel(DistillArgs a) {
  constexpr int EPV = 16 / TI::kBytes, U = kPartU, BLOCK = kPartBlock;
  constexpr bool kSplit = TI::kBytes == 2 && TO::kBytes == 4;
  constexpr uint32_t kOutVec = EPV * TO::kBytes;
  static_assert(!(SCALAR && kSplit), "f32 dlogits of 16-bit rows are stored at any element");
  __shared__ Teacher te;
  __shared__ RowTerms terms;
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
    if (tid < 64) {
      Entries<NS> e;
      float z[NS];
      load_entries(a, row, e);
#pragma unroll
      for (int s = 0; s < NS; ++s) z[s] = e.id[s] >= 0 ? a.part_z[row * a.k + tid + kWave * s] : kNegInf;
      float mt, st;
      bool twice;
      merge_tail(a, row, mt, st, twice);
      put_entries(a, row, te, e);
      put_student(a, te, z);
      if (tid == 0 && twice) {
        te.row.state = kBad;
        if (part == 0) raise_error(a.err, kErrTeacherTwice);
      }
      float token = 0.f;
      if (te.row.state == kUsed) token = row_terms<NS>(a, r, te, mt, st, terms);
      if (part == 0 && tid == 0 && a.token_loss) a.token_loss[r.tix] = token;
    }
    __syncthreads();
    live = te.row.state == kUsed;
  } else if (part == 0 && tid == 0 && r.tok && a.token_loss) {
    a.token_loss[r.tix] = 0.f;
  }
  float g[NS], tail = 0.f, ref = 0.f;
  int place[NS], edge[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    place[s] = edge[s] = -1;
    g[s] = 0.f;
  }
  if (live) {
    if constexpr (GRAD) {
      tail = terms.tail;
      ref = terms.ref;
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const int id = te.id[(tid & 63) + kWave * s];
        if (id >= 0) g[s] = terms.g[(tid & 63) + kWave * s];
        place[s] = id >= 0 && id - sp.head < end * EPV ? entry_place<TI, kSplit, BLOCK, U>(id - sp.head, v0) : -1;
        if (place[s] >= 0 && ((place[s] >> 10) & 15) != (tid >> 6)) place[s] = -1;
        if (part == 0 && tid < 64) edge[s] = edge_thread<TI>(sp, id);
      }
    }
  }
  if constexpr (GRAD) {
#pragma unroll
    for (int q = 0; q < U; ++q) {
      float o[EPV];
      if (live) {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(&x[q]);
#pragma unroll
        for (int j = 0; j < EPV; ++j) o[j] = tail * hw_exp2(fmaf(TI::unpack(w, j), a.k2, -ref));
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          uint64_t at = __ballot(place[s] >= 0 && (place[s] >> 16) == q);
          while (at) {
            const int src = __builtin_ctzll(at);
            at &= at - 1;
            const int p = __builtin_amdgcn_readlane(place[s], src);
            const float ge = read_lane(g[s], src);
            const bool here = ((p >> 4) & 63) == (tid & 63);
#pragma unroll
            for (int j = 0; j < EPV; ++j)
              if (here && j == (p & 15)) o[j] = ge;
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
      float o = live && ek >= 0 ? tail * hw_exp2(fmaf(xe, a.k2, -ref)) : 0.f;
      if (live) {
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          uint64_t at = __ballot(edge[s] >= 0);
          while (at) {
            const int src = __builtin_ctzll(at);
            at &= at - 1;
            const int thread = __builtin_amdgcn_readlane(edge[s], src);
            const float ge = read_lane(g[s], src);
            if (tid == thread) o = ge;
          }
        }
      }
      if (ek >= 0) store1<TO>(a.dlogits, row_elem + ek, o);
    }
  }
}


// ---------------------------------------------------------------------------
// A row to a workgroup, kept in registers from its one read to its gradient's write.
// Persistent: while a row's gradient is stored, each chunk's registers take the next row's
// load, so the CU reads and writes at once; the next row's entries come the same way (ids and
// probabilities at the top of this row, the student's logits there after its merge, their
// sum after its stores, all by the first wave, through the other half of te).
// Requirements (checked on the host): the row's interior fits BLOCK * NCH vectors; dlogits
// rows split like the logits rows, or hold f32 for 16-bit logits (dword-aligned stores).
// ---------------------------------------------------------------------------
// Narrow rows are dealt in grid strides, each starting `turn` further on, wide ones from a
// counter, for the reasons given at grpo_resident_kernel.
template <int BLOCK, int NCH>
constexpr bool kDealt = BLOCK * NCH <= 2048;

template <typename TI, typename TO, int BLOCK, int NCH, int NS>
__global__ void __launch_bounds__(BLOCK) distill_row_kernel(DistillArgs a) {
  constexpr int EPV = 16 / TI::kBytes, NW = BLOCK / 64;
  constexpr bool kSplit = TI::kBytes == 2 && TO::kBytes == 4, kStatic = kDealt<BLOCK, NCH>;
  constexpr uint32_t kOutVec = EPV * TO::kBytes;
  __shared__ Teacher te[2];
  __shared__ RowTerms terms;
  __shared__ float4 merge[NW];
  __shared__ int s_next[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t voff = tid * 16u, sgrp = split_group<TI, TO, BLOCK>(tid);
  const char* logits = static_cast<const char*>(a.logits);
  auto span_of = [&](int64_t row) { return row_span<TI>(logits + row * a.vocab * TI::kBytes, a.vocab); };
  auto buffer_of = [&](const RowSpan& sp, bool on) {   // off: loads return 0 without an access
    return row_rsrc(sp.vec, on ? static_cast<uint32_t>(sp.nv) * 16u : 0u);
  };
  int64_t stride0 = 0;                                 // static: the current stride's first row
  uint32_t at = blockIdx.x;
  auto deal = [&]() -> int64_t {                       // static: the row after this one
    stride0 += gridDim.x;
    at += static_cast<uint32_t>(a.turn);
    if (at >= gridDim.x) at -= gridDim.x;
    return stride0 + at;
  };
  int64_t row = blockIdx.x, next = kStatic ? deal() : static_cast<int64_t>(blockIdx.x) + gridDim.x;
  DistillRow r = distill_row(a, row);
  RowSpan sp = span_of(row);
  u32x4 xv[NCH];
  float xe = 0.f;
  {
    const __amdgpu_buffer_rsrc_t buf = buffer_of(sp, r.w != 0.f);
#pragma unroll
    for (int k = 0; k < NCH; ++k) xv[k] = load_chunk<TI, TO, BLOCK>(buf, k, voff, sgrp);
    if (r.w != 0.f) {
      const int ek = edge_index<TI>(sp, tid);
      if (ek >= 0) xe = TI::load1(logits + row * a.vocab * TI::kBytes, ek);
      if (wave == 0) {
        Entries<NS> e;
        float z[NS];
        load_entries(a, row, e);
#pragma unroll
        for (int s = 0; s < NS; ++s)
          z[s] = e.id[s] >= 0 ? TI::load1(logits + row * a.vocab * TI::kBytes, e.id[s]) : kNegInf;
        put_entries(a, row, te[0], e);
        put_student(a, te[0], z);
      }
    }
  }
  __syncthreads();
  for (int i = 0;; ++i) {
    const Teacher& t = te[i & 1];
    const int64_t row_elem = row * a.vocab;
    // What the next row needs first.
    const bool more = next < a.nrows;
    DistillRow rn = distill_row(a, more ? next : row);
    const bool want = more && rn.w != 0.f;
    Teacher& tn = te[(i + 1) & 1];
    Entries<NS> en;
    if (wave == 0 && want) load_entries(a, next, en);
    int claimed = INT32_MAX;
    if (!kStatic && tid == 0 && a.nrows > 2 * static_cast<int64_t>(gridDim.x))
      claimed = atomicAdd(a.next_row, 1) + 2 * static_cast<int>(gridDim.x);

    const int nv = sp.nv;
    // kSplit: half h of chunk k of this lane holds row values (past the row end it read 0).
    auto held = [&](int k, int h) {
      return kSplit ? static_cast<int64_t>(k) * 2 * BLOCK + 64 * h + sgrp < 2 * static_cast<int64_t>(nv)
                    : k * BLOCK + tid < nv;
    };
    bool live = r.w != 0.f && t.row.state == kUsed;
    float token = 0.f;
    if (live) {
      bool twice;
      const int ek = edge_index<TI>(sp, tid);
      float x1 = ek >= 0 ? xe : kNegInf;
      {
        int id[NS], place[NS];
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          id[s] = t.id[lane + kWave * s];
          place[s] = id[s] >= 0 && id[s] - sp.head < nv * EPV ? entry_place<TI, kSplit, BLOCK, NCH>(id[s] - sp.head, 0) : -1;
        }
        twice = mask_entries<TI>(xv, id, place);
        if (wave == 0) twice |= mask_edges<TI>(sp, x1, id);
      }
      float mx = x1;
#pragma unroll
      for (int k = 0; k < NCH; ++k) {
        if constexpr (kSplit) {
          const uint32_t* w = reinterpret_cast<const uint32_t*>(&xv[k]);
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (held(k, h)) {
#pragma unroll
              for (int j = 4 * h; j < 4 * h + 4; ++j) mx = fmaxf(mx, TI::unpack(w, j));
            }
        } else if (held(k, 0)) {
          mx = vec_max<TI>(mx, xv[k]);
        }
      }
      float m = mx * a.k2;
      const float ref = ms_ref(m);
      float s = hw_exp2(fmaf(x1, a.k2, -ref));
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int k = 0; k < NCH; ++k) {
        uint32_t u[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          u[q] = xv[k][q];
          asm volatile("" : "+v"(u[q]));   // else the unpacked maxima stay live
        }
        if constexpr (kSplit) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (held(k, h)) {
#pragma unroll
              for (int j = 4 * h; j < 4 * h + 4; ++j) s += hw_exp2(fmaf(TI::unpack(u, j), a.k2, -ref));
            }
        } else if (held(k, 0)) {
#pragma unroll
          for (int j = 0; j < EPV; ++j) s += hw_exp2(fmaf(TI::unpack(u, j), a.k2, -ref));
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      lanes_merge<64>(m, s);
      if (lane == 0) merge[wave] = make_float4(m, s, twice ? 1.f : 0.f, 0.f);
      __syncthreads();
      const float4 w = merge[lane & (NW - 1)];
      live = !__any(w.z != 0.f);
      if (wave == 0) {
        m = w.x;
        s = w.y;
        lanes_merge<NW>(m, s);
        if (live) token = row_terms<NS>(a, r, t, m, s, terms);
        else if (lane == 0) raise_error(a.err, kErrTeacherTwice);
      }
      __syncthreads();
    }
    if (wave == 0 && want) put_entries(a, next, tn, en);
    if (!live) {
#pragma unroll
      for (int k = 0; k < NCH; ++k) xv[k] = u32x4{0u, 0u, 0u, 0u};
    }
    // This wave's entries and their gradients.
    const float tail = live ? terms.tail : 0.f, ref = live ? terms.ref : 0.f;
    int place[NS];
    float g[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      place[s] = -1;
      g[s] = 0.f;
      if (live) {
        const int id = t.id[lane + kWave * s];
        if (id >= 0 && id - sp.head < nv * EPV) place[s] = entry_place<TI, kSplit, BLOCK, NCH>(id - sp.head, 0);
        if (place[s] >= 0 && ((place[s] >> 10) & 15) != wave) place[s] = -1;
        if (place[s] >= 0) g[s] = terms.g[lane + kWave * s];
      }
    }
    if (tid == 0 && r.tok) a.token_loss[r.tix] = token;
    const char* nrow = logits + (more ? next : row) * a.vocab * TI::kBytes;
    const RowSpan spn = span_of(more ? next : row);
    float en_z[NS];
    if (wave == 0 && want) {
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const int id = tn.id[lane + kWave * s];
        en_z[s] = id >= 0 ? TI::load1(nrow, id) : kNegInf;
      }
    }
    const __amdgpu_buffer_rsrc_t nbuf = buffer_of(spn, want);
    const __amdgpu_buffer_rsrc_t drow = row_rsrc(static_cast<char*>(a.dlogits) + (row_elem + sp.head) * TO::kBytes,
                                                 static_cast<uint32_t>(nv) * kOutVec);
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      uint32_t u[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        u[q] = xv[k][q];
        asm volatile("" : "+v"(u[q]));   // else the sum pass's unpacked values stay live
      }
      float out[EPV];
#pragma unroll
      for (int j = 0; j < EPV; ++j) out[j] = tail * hw_exp2(fmaf(TI::unpack(u, j), a.k2, -ref));
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        uint64_t mine = __ballot(place[s] >= 0 && (place[s] >> 16) == k);
        while (mine) {
          const int src = __builtin_ctzll(mine);
          mine &= mine - 1;
          const int p = __builtin_amdgcn_readlane(place[s], src);
          const float ge = read_lane(g[s], src);
          const bool here = ((p >> 4) & 63) == lane;
#pragma unroll
          for (int j = 0; j < EPV; ++j)
            if (here && j == (p & 15)) out[j] = ge;
        }
      }
      // Vectors past the row end sit past the descriptor: their stores are dropped.
      if constexpr (kSplit) {
        const float (&o0)[4] = reinterpret_cast<const float (&)[4]>(out[0]);
        const float (&o1)[4] = reinterpret_cast<const float (&)[4]>(out[4]);
        buf_store_vals<TO, 4, true, kBufNTSystem>(drow, fresh_off(sgrp * 16u, k * 2 * BLOCK * 16u), o0);
        buf_store_vals<TO, 4, true, kBufNTSystem>(drow, fresh_off(sgrp * 16u, k * 2 * BLOCK * 16u + 1024u), o1);
      } else {
        buf_store_vals<TO, EPV, true, kBufNTSystem>(drow, fresh_off(tid * kOutVec, k * BLOCK * kOutVec), out);
      }
      xv[k] = load_chunk<TI, TO, BLOCK>(nbuf, k, voff, sgrp);
    }
    if (wave == 0) {
      const int ek = edge_index<TI>(sp, tid);
      float oe = live && ek >= 0 ? tail * hw_exp2(fmaf(xe, a.k2, -ref)) : 0.f;
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const int edge = live ? edge_thread<TI>(sp, t.id[lane + kWave * s]) : -1;
        const float ge = edge >= 0 ? terms.g[lane + kWave * s] : 0.f;
        uint64_t mine = __ballot(edge >= 0);
        while (mine) {
          const int src = __builtin_ctzll(mine);
          mine &= mine - 1;
          if (tid == __builtin_amdgcn_readlane(edge, src)) oe = read_lane(ge, src);
        }
      }
      if (ek >= 0) store1<TO>(a.dlogits, row_elem + ek, oe);
      if (want) {
        const int en_k = edge_index<TI>(spn, tid);
        if (en_k >= 0) xe = TI::load1(nrow, en_k);
        put_student(a, tn, en_z);
      }
    }
    if (!kStatic && tid == 0) s_next[i & 1] = claimed;
    __syncthreads();
    if (!more) break;
    row = next;
    r = rn;
    sp = spn;
    next = kStatic ? deal() : static_cast<int64_t>(__builtin_amdgcn_readfirstlane(s_next[i & 1]));
  }
}

// ---------------------------------------------------------------------------
// Launches of one pair of element types.
// ---------------------------------------------------------------------------
template <typename TI, typename TO, int NS>
hipError_t launch_parts(DistillArgs a, hipStream_t st) {
  const bool scalar = a.dlogits && TI::kBytes == TO::kBytes &&
                      ((reinterpret_cast<uintptr_t>(a.logits) ^ reinterpret_cast<uintptr_t>(a.dlogits)) & 15u) != 0;
  constexpr int64_t kRows = 65535;   // grid.y
  // The preparation goes with the first kernel where its workgroups fit that grid.
  const int64_t prep = prepare_blocks(a);
  const bool with = a.nrows + prep <= kRows;
  if (!with) distill_prepare_kernel<kPrepBlock><<<dim3(static_cast<unsigned>(prep)), dim3(kPrepBlock), 0, st>>>(a);
  for (int64_t r0 = 0; r0 < a.nrows; r0 += kRows) {
    a.row0 = r0;
    const unsigned n = static_cast<unsigned>(a.nrows - r0 < kRows ? a.nrows - r0 : kRows);
    const dim3 g(static_cast<unsigned>(a.parts), n), b(kPartBlock);
    const dim3 g1(static_cast<unsigned>(a.parts), with ? n + static_cast<unsigned>(prep) : n);
    distill_part_kernel<TI, NS><<<g1, b, 0, st>>>(a, static_cast<int>(n));
    if (!a.dlogits) {
      distill_part_grad_kernel<TI, TO, NS, false, false><<<dim3(1, n), dim3(64), 0, st>>>(a);
    } else if constexpr (TI::kBytes == TO::kBytes) {
      if (scalar) distill_part_grad_kernel<TI, TO, NS, true, true><<<g, b, 0, st>>>(a);
      else distill_part_grad_kernel<TI, TO, NS, true, false><<<g, b, 0, st>>>(a);
    } else {
      distill_part_grad_kernel<TI, TO, NS, true, false><<<g, b, 0, st>>>(a);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <typename TI, typename TO, int BLOCK, int NCH, int NS>
hipError_t launch_row(DistillArgs a, hipStream_t st) {
  static std::atomic<int> cached{0};   // workgroups that the device holds at once
  int slots = cached.load(std::memory_order_relaxed);
  if (slots <= 0) {
    int dev = 0, cus = 0, occ = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e == hipSuccess) e = hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev);
    if (e == hipSuccess)
      e = hipOccupancyMaxActiveBlocksPerMultiprocessor(
          &occ, reinterpret_cast<const void*>(&distill_row_kernel<TI, TO, BLOCK, NCH, NS>), BLOCK, 0);
    if (e != hipSuccess) return e;
    slots = cus * (occ > 0 ? occ : 1);
    cached.store(slots, std::memory_order_relaxed);
  }
  const int64_t grid = a.nrows < slots ? a.nrows : slots;
  distill_prepare_kernel<kPrepBlock><<<dim3(static_cast<unsigned>(prepare_blocks(a))), dim3(kPrepBlock), 0, st>>>(a);
  if (kDealt<BLOCK, NCH>) a.turn = resident_turn(grid, a.logit_stride, a.mask != nullptr);
  distill_row_kernel<TI, TO, BLOCK, NCH, NS><<<dim3(static_cast<unsigned>(grid)), dim3(BLOCK), 0, st>>>(a);
  return hipGetLastError();
}

template <typename TI, typename TO, int NS>
hipError_t launch_rows_of(const DistillArgs& a, int64_t nv, hipStream_t st) {
  if (nv <= 256) return launch_row<TI, TO, 256, 1, NS>(a, st);
  if (nv <= 512) return launch_row<TI, TO, 256, 2, NS>(a, st);
  if (nv <= 1024) return launch_row<TI, TO, 256, 4, NS>(a, st);
  if (nv <= 2048) return launch_row<TI, TO, 256, 8, NS>(a, st);
  if (nv <= 4096) return launch_row<TI, TO, 1024, 4, NS>(a, st);
  if (nv <= 8192) return launch_row<TI, TO, 1024, 8, NS>(a, st);
  if (nv <= 12288) return launch_row<TI, TO, 1024, 12, NS>(a, st);
  if (nv <= 16384) return launch_row<TI, TO, 1024, 16, NS>(a, st);
  if (nv <= kDistillRowVecs) return launch_row<TI, TO, 1024, 19, NS>(a, st);
  return hipErrorInvalidValue;
}

template <typename TI, typename TO>
hipError_t launch_pair(const DistillArgs& a, hipStream_t st) {
  const bool few = a.k <= kWave;
  if (a.parts > 0) return few ? launch_parts<TI, TO, 1>(a, st) : launch_parts<TI, TO, kMaxSlots>(a, st);
  const int64_t nv = a.vocab * TI::kBytes / 16;
  return few ? launch_rows_of<TI, TO, 1>(a, nv, st) : launch_rows_of<TI, TO, kMaxSlots>(a, nv, st);
}

}  // namespace pcp
