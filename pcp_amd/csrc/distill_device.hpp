// Kernels of the distillation from a teacher's top logits (pcp_distill.h): the loss of a row against up
// to 256 teacher entries, and its gradient over the whole vocabulary.
//
// With x a row's logits, k2 = log2(e) / tau, K the used teacher ids and T the rest of the
// vocabulary, the rows' sums are kept apart: (m_T, s_T) over T while the row streams past
// (the entries' own elements are replaced by -inf where they sit in registers), and s_K from
// the k gathered logits. Maxima are logits and sums relative to them (see term_scale). The tail's
// mass Q_T = s_T 2^((m_T - R) k2) / s is then a sum of its own and keeps its relative precision
// where the teacher's entries hold nearly everything (1 - sum q_i would lose it all). Per element
// the arithmetic is f32; what a row has once (s_K, the merge of its waves' sums, the logarithms,
// the divergence) f64, since the divergence may be far below its terms. Outside K the gradient is
// one factor of 2^((x - m_T) k2):
//   forward:  c (P Q_T - p_T) / s_T,   reverse:  c (Q_T / s_T) (log(Q_T/p_T) - l),
// with c = weight m / (loss_norm L tau) and P = sum p_i + p_T; on K each entry has its own
// value, which takes the element's place before its vector is stored.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
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
// Entry i is slot i / 64 of lane i % 64; the kernels of rows in parts are compiled for 1 slot
// (k <= 64) and for 4.
constexpr int kMaxSlots = kMaxEntries / kWave;

// What the preparation makes of a row. zref is the student's largest logit at an entry (0 and sk 0
// where all are -inf); the row kernel takes its first sums against it.
struct TeacherRow {
  double sum_p;     // of the entries
  double log_pt;    // of the tail's class, if there is one
  double lse;       // the entries' probabilities are exp((t - tref) / tau - lse) (see log_base)
  double sk;        // sum exp((z - zref) / tau) over the entries
  double adj;       // term_adj of zref and at, in 64 bits
  float pt;
  float zref;
  TermScale at;     // term_scale of zref
  float tref;
  float w;          // the row's weight
  int32_t state;    // kUnused, kUsed; kBad: an id out of range
  int32_t pad;
};
// What log-probabilities of a row with largest logit m are taken relative to: 0, where (x - 0) / tau and
// a log-sum-exp in 64 bits lose nothing; else m, since a row of huge logits (each -1e30, say) has
// its log-probabilities in the last bits of neither.
__device__ __forceinline__ float log_base(float m) { return fabsf(m) < 0x1p16f ? 0.f : m; }
constexpr int kUnused = 0, kUsed = 1, kBad = 2;
constexpr int kRowWords = sizeof(TeacherRow) / 4;
constexpr double kLn2F64 = 0.69314718055994530942;

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
  PartSum* part;            // [nrows, parts]: m_T, s_T, n: an id is used twice
  TeacherRow* teacher;      // [nrows], by the preparation, and per entry, [nrows, k]:
  int* entry_ids;           // used_id,
  double* entry_w;          // forward: its probability; reverse: exp((z - zref) / tau),
  float* entry_z;           // the student's logit (dlogits may replace it)
  int* err;
  int* next_row;            // rows handed out past the first grid (zeroed earlier on the stream)
  int64_t nrows, vocab, rows, logit_stride, tok_stride, tok_offset;
  int64_t row0;             // first row of this launch
  double inv_tau;
  int64_t n_seq;
  int* done;                // the loss reduction's ticket
  float* loss;              // formed by the last workgroup to finish, or nullptr: by loss_reduce_kernel
  float loss_norm;          // loss_norm / weight
  float k2;                 // log2(e) / tau
  int32_t k, ids_i64, mask_u8, forward;
  int32_t parts, per;       // workgroups per row (0: a row to a workgroup), 16-byte vectors per workgroup
  int32_t turn;             // rows dealt in grid strides: how far on each stride starts
};

struct DistillRow {
  int64_t tix;
  float w;
  int32_t seq;
  bool tok;
};

__device__ __forceinline__ DistillRow distill_row(const DistillArgs& a, int64_t row) {
  DistillRow r;
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

// An entry's id, or -1 when it is unused, -2 when its id is out of range.
__device__ __forceinline__ int used_id(const DistillArgs& a, int64_t id, float t) {
  if (id == PCP_IGNORE_INDEX || t == kNegInf) return -1;
  return id >= 0 && id < a.vocab ? static_cast<int>(id) : -2;
}
// Entry i of a row.
__device__ __forceinline__ int entry_id(const DistillArgs& a, int64_t row, int i, float& t) {
  t = kNegInf;
  if (i >= a.k) return -1;
  const int64_t e = row * a.k + i;
  const int64_t id = a.ids_i64 ? static_cast<const int64_t*>(a.tids)[e]
                               : static_cast<int64_t>(static_cast<const int32_t*>(a.tids)[e]);
  t = a.tlogits[e];
  return used_id(a, id, t);
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

// Row `row`, by one wave.
template <typename TI>
__device__ __forceinline__ void prepare_row(const DistillArgs& a, int64_t row) {
  const int lane = threadIdx.x & 63;
  TeacherRow o;
  o.sum_p = o.log_pt = o.lse = o.sk = 0.;
  o.adj = 1.;
  o.pt = o.zref = o.tref = 0.f;
  o.at = TermScale{a.k2, 0.f};
  o.w = distill_row(a, row).w;
  o.state = kUnused;
  o.pad = 0;
  if (o.w != 0.f) {
    const char* xrow = static_cast<const char*>(a.logits) + row * a.vocab * TI::kBytes;
    int id[kMaxSlots];
    float t[kMaxSlots], z[kMaxSlots], tmax = kNegInf, zmax = kNegInf;
    bool out = false, any = false;
#pragma unroll
    for (int s = 0; s < kMaxSlots; ++s) {
      id[s] = -1;
      z[s] = kNegInf;
      if (kWave * s < a.k) id[s] = entry_id(a, row, lane + kWave * s, t[s]);
      if (id[s] >= 0) z[s] = TI::load1(xrow, id[s]);
      out |= id[s] == -2;
      any |= id[s] >= 0;
      if (id[s] >= 0) tmax = fmaxf(tmax, t[s]);
      zmax = fmaxf(zmax, z[s]);
    }
    if (a.tlse) {
      o.lse = static_cast<double>(a.tlse[row]);
    } else {
      const float m = ms_ref(lanes_max<64>(tmax));
      double sum = 0.;
#pragma unroll
      for (int s = 0; s < kMaxSlots; ++s)
        if (id[s] >= 0) sum += exp((static_cast<double>(t[s]) - m) * a.inv_tau);
      o.tref = log_base(m);
      o.lse = static_cast<double>(m - o.tref) * a.inv_tau + log(wave_sum64(sum));
    }
    o.zref = ms_ref(lanes_max<64>(zmax));
    o.at = term_scale(o.zref, a.k2);
    o.adj = exp(-term_residue(o.zref, o.at) * kLn2F64);
    double sum_p = 0., sk = 0.;
#pragma unroll
    for (int s = 0; s < kMaxSlots; ++s) {
      const int i = lane + kWave * s;
      if (i >= a.k) continue;
      double p = 0., e = 0.;
      if (id[s] >= 0) {
        p = exp((static_cast<double>(t[s]) - o.tref) * a.inv_tau - o.lse);
        e = exp((static_cast<double>(z[s]) - o.zref) * a.inv_tau);
      }
      sum_p += p;
      sk += e;
      a.entry_ids[row * a.k + i] = id[s];
      a.entry_w[row * a.k + i] = a.forward ? p : e;
      a.entry_z[row * a.k + i] = z[s];
    }
    o.sk = wave_sum64(sk);
    o.sum_p = wave_sum64(sum_p);
    const double pt = fmax(1. - o.sum_p, PCP_DISTILL_TAIL_FLOOR);
    o.log_pt = log(pt);
    o.pt = static_cast<float>(pt);
    o.state = __any(out) ? kBad : __any(any) ? kUsed : kUnused;
  }
  if (lane != 0) return;
  a.teacher[row] = o;
  if (o.state == kBad) raise_error(a.err, kErrTokenRange);
  else if (o.state == kUsed && !(__builtin_isfinite(o.lse) && __builtin_isfinite(o.sum_p) && __builtin_isfinite(o.w)))
    raise_error(a.err, kErrNonFinite);
}

// Workgroup `block` of the preparation: a sequence, or a row per wave.
template <typename TI>
__device__ __forceinline__ void prepare(const DistillArgs& a, int64_t block, float* lds) {
  if (block < a.n_seq) {
    prepare_sequence(a, block, lds);
    return;
  }
  const int64_t row = (block - a.n_seq) * (kPrepBlock / 64) + (threadIdx.x >> 6);
  if (row < a.nrows) prepare_row<TI>(a, row);
}
inline int64_t prepare_blocks(const DistillArgs& a) {
  return a.n_seq + (a.nrows + kPrepBlock / 64 - 1) / (kPrepBlock / 64);
}

template <typename TI>
__global__ void __launch_bounds__(kPrepBlock) distill_prepare_kernel(DistillArgs a, int64_t block0) {
  __shared__ float lds[kPrepBlock / 64];
  prepare<TI>(a, block0 + blockIdx.x, lds);
}
// A grid has fewer than 2^32 threads: calls of some ten million rows and more take several.
template <typename TI>
void launch_prepare(const DistillArgs& a, hipStream_t st) {
  constexpr int64_t kMost = (int64_t{1} << 31) / kPrepBlock;
  const int64_t blocks = prepare_blocks(a);
  for (int64_t b = 0; b < blocks; b += kMost)
    distill_prepare_kernel<TI>
        <<<dim3(static_cast<unsigned>(std::min(blocks - b, kMost))), dim3(kPrepBlock), 0, st>>>(a, b);
}

// ---- a row's terms -----------------------------------------------------------------------
// A row's record and entries in LDS, for the whole workgroup.
struct Teacher {
  TeacherRow row;
  int id[kMaxEntries];
  float t[kMaxEntries];
  float z[kMaxEntries];
  uint32_t w_lo[kMaxEntries], w_hi[kMaxEntries];   // all five arrays at one offset per lane
  __device__ __forceinline__ double w(int i) const {
    return __builtin_bit_cast(double, static_cast<uint64_t>(w_hi[i]) << 32 | w_lo[i]);
  }
};

// What a row's gradient needs: tail * 2^(x at.k - at.ref) outside K, g[] at the entries.
struct RowTerms {
  float tail;
  TermScale at;
  float g[kMaxEntries];
};

// A row on its way to LDS: lane l's entry of group w by wave w, and word l of the record. The loads
// are the same for every lane and their values are only looked at when they go to LDS.
struct LateRow {
  int id;
  float t, z;
  double w;
  uint32_t word;
};
// Through buffer descriptors, which need no address in registers from row to row and give 0 past
// the row's k entries. group: the same in the whole wave.
__device__ __forceinline__ LateRow load_late(const DistillArgs& a, int64_t row, int group) {
  const int lane = threadIdx.x & 63;
  const int64_t base = row * a.k + kWave * group;
  const uint32_t n = static_cast<uint32_t>(a.k - kWave * group), off = lane * 4u;
  auto word = [&](const void* p, uint32_t bytes) {
    return static_cast<uint32_t>(__builtin_amdgcn_raw_buffer_load_b32(row_rsrc(p, bytes), off, 0, 0));
  };
  LateRow l;
  l.id = static_cast<int>(word(a.entry_ids + base, n * 4u));
  l.t = __uint_as_float(word(a.tlogits + base, n * 4u));
  l.z = __uint_as_float(word(a.entry_z + base, n * 4u));
  l.w = __builtin_bit_cast(double, __builtin_amdgcn_raw_buffer_load_b64(row_rsrc(a.entry_w + base, n * 8u),
                                                                         lane * 8u, 0, 0));
  l.word = word(a.teacher + row, sizeof(TeacherRow));
  return l;
}
__device__ __forceinline__ void put_late(const DistillArgs& a, Teacher& te, int group, const LateRow& l) {
  const int lane = threadIdx.x & 63, i = lane + kWave * group;
  te.id[i] = i < a.k ? l.id : -1;
  te.t[i] = l.t;
  te.w_lo[i] = static_cast<uint32_t>(__builtin_bit_cast(uint64_t, l.w));
  te.w_hi[i] = static_cast<uint32_t>(__builtin_bit_cast(uint64_t, l.w) >> 32);
  te.z[i] = l.z;
  if (group == 0 && lane < kRowWords) reinterpret_cast<uint32_t*>(&te.row)[lane] = l.word;
}
__device__ __forceinline__ int groups_of(const DistillArgs& a) { return (a.k + kWave - 1) / kWave; }

// A row's factors, the same in every lane of any wave that forms them.
struct RowFactors {
  float tail;           // the gradient outside K: tail * 2^(x at.k - at.ref)
  TermScale at;
  float c, r, inv_s;    // the coefficient; q_i = 2^((z - r) k2) inv_s
  float big_p, lf;      // forward: P; reverse: l
  float ek;             // 2^((zref - r) k2)
  double s;             // the whole row's sum over exp(r / tau)
  double qt, log_qt;    // the tail's mass; 0: no tail
  double lse;           // log q_i = (z - zbase) / tau - lse; these and log_qt only after set_logs
  float zbase;
};

// log(s) to 1e-12, by atanh's series. Its constants are set where they are used: over the row
// kernel's loop the compiler would keep them all in registers.
__device__ __forceinline__ double log64(double s) {
  if (s == 0.) return -__builtin_inf();
  int k = __builtin_amdgcn_frexp_exp(s);
  double m = __builtin_amdgcn_frexp_mant(s);
  if (m < 0.70710678118654752) {
    m *= 2.;
    --k;
  }
  const double t = (m - 1.) / (m + 1.), u = t * t;
  double p = 0.;
#pragma unroll
  for (int i = 17; i >= 1; i -= 2) {
    double c = 1. / i;
    asm volatile("" : "+s"(c));
    p = fma(p, u, c);
  }
  double ln2 = kLn2F64;
  asm volatile("" : "+s"(ln2));
  return fma(2. * t, p, k * ln2);
}

// A value that is the same in every lane, in a scalar register (two vector registers fewer where the
// widest rows leave none).
__device__ __forceinline__ float first_lane(float v) {
  return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v)));
}
__device__ __forceinline__ float entry_prob(const DistillArgs& a, const Teacher& te, const RowFactors& f, int i) {
  return hw_exp2((te.z[i] - f.r) * a.k2) * f.inv_s;
}
// log(p_i / q_i)
__device__ __forceinline__ double entry_gap(const DistillArgs& a, const Teacher& te, const RowFactors& f, int i) {
  return (static_cast<double>(te.t[i] - first_lane(te.row.tref)) - (te.z[i] - first_lane(f.zbase))) * a.inv_tau -
         (te.row.lse - f.lse);
}
// The gradient at entry i.
__device__ __forceinline__ float entry_grad(const DistillArgs& a, const Teacher& te, const RowFactors& f, int i) {
  const float q = entry_prob(a, te, f, i);
  if (a.forward) return f.c * (q * f.big_p - static_cast<float>(te.w(i)));
  return q > 0.f ? -f.c * q * (static_cast<float>(entry_gap(a, te, f, i)) + f.lf) : 0.f;
}

__device__ __forceinline__ void set_logs(const DistillArgs& a, RowFactors& f) {
  f.zbase = log_base(f.r);
  f.lse = static_cast<double>(f.r - f.zbase) * a.inv_tau + log64(f.s);
  f.log_qt = f.qt > 0. ? log64(f.qt) : 0.;
}

// The row's divergence l, by a whole wave, after set_logs. Formed in 64 bits: l may be far below
// its terms.
__device__ __forceinline__ double row_loss(const DistillArgs& a, const Teacher& te, const RowFactors& f) {
  const int lane = threadIdx.x & 63, groups = groups_of(a);
  double l = 0.;
  for (int w = 0; w < groups; ++w) {
    const int i = lane + kWave * w;
    if (te.id[i] < 0) continue;
    const double weight = a.forward ? te.w(i) : -te.w(i) * f.ek / f.s;
    if (weight != 0.) l += weight * entry_gap(a, te, f, i);
  }
  l = wave_sum64(l);
  if (f.qt > 0.) {
    const double gap = te.row.log_pt - f.log_qt;   // log(p_T / q_T)
    l += a.forward ? te.row.pt * gap : -f.qt * gap;
  }
  if (lane == 0 && !(__builtin_isfinite(f.lse) && l == l)) raise_error(a.err, kErrNonFinite);
  return l;
}

// st: the sum outside K, relative to mt, its largest logit or the row's zref. The forward gradient does
// without the loss, the reverse one holds it (loss: l, formed here if reverse).
// weight: the row's scale times its weight.
__device__ __forceinline__ RowFactors row_factors(const DistillArgs& a, float weight, const Teacher& te, float mt,
                                                  double st, double& loss) {
  RowFactors f;
  f.r = ms_ref(te.row.sk == 0. ? mt : fmaxf(mt, te.row.zref));
  f.ek = te.row.sk == 0. ? 0.f : hw_exp2((te.row.zref - f.r) * a.k2);
  const double ft = st == 0. ? 0. : hw_exp2((mt - f.r) * a.k2);
  f.s = te.row.sk * f.ek + st * ft;
  const double inv = 1. / f.s;
  f.inv_s = static_cast<float>(inv);
  f.qt = st * ft * inv;
  f.qt = a.tlse != nullptr && f.qt >= 0x1p-126 ? f.qt : 0.;
  f.c = static_cast<float>(static_cast<double>(weight) * a.inv_tau);
  f.big_p = f.lf = 0.f;
  f.lse = f.log_qt = 0.;
  f.zbase = 0.f;
  if (a.forward) {
    const double pt = f.qt > 0. ? te.row.pt : 0.;
    f.big_p = static_cast<float>(te.row.sum_p + pt);
    f.tail = st == 0. ? 0.f : f.c * static_cast<float>((te.row.sum_p + pt) * (ft * inv) - pt / st);
  } else {
    set_logs(a, f);
    loss = row_loss(a, te, f);
    f.lf = static_cast<float>(loss);
    const double gap = f.qt > 0. ? te.row.log_pt - f.log_qt : 0.;
    f.tail = st == 0. ? 0.f : -f.c * static_cast<float>(ft * inv * (gap + loss));
  }
  f.at = term_scale(mt, a.k2);
  f.tail *= term_adj(mt, f.at);
  return f;
}

// The loss from the token losses, which are stored through to the coherent level: by the last of
// `n` workgroups to come here, each after its last one; in a fixed order.
template <int BLOCK>
__device__ __forceinline__ void finish_loss(const DistillArgs& a, int n) {
  __shared__ double sums[BLOCK / 64];
  __shared__ int last;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  wait_stores();     // this wave's token losses ...
  __syncthreads();   // ... and every wave's, before the ticket
  if (tid == 0) last = atomicAdd(a.done, 1) == n - 1;
  __syncthreads();
  if (!last) return;
  acquire_coherent();
  double sum = 0.;
  for (int64_t s = wave; s < a.n_seq; s += BLOCK / 64) {
    const float* t = a.token_loss + s * a.tok_stride + a.tok_offset;
    double l = 0.;
    for (int64_t i = lane; i < a.rows; i += 64) l += t[i];
    sum += wave_sum64(l) / a.seq_len[s];
  }
  if (lane == 0) sums[wave] = sum;
  __syncthreads();
  if (tid != 0) return;
  for (int w = 1; w < BLOCK / 64; ++w) sum += sums[w];
  *a.loss = static_cast<float>(sum / a.loss_norm);
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
  __shared__ float2 lds[BLOCK / 64];
  __shared__ int any_twice;
  const int tid = threadIdx.x, part = blockIdx.x;
  static_assert(kPartBlock == kPrepBlock, "the preparation's workgroup");
  if (blockIdx.y >= static_cast<unsigned>(n)) {   // past the rows: the preparation
    if (part == 0) prepare<TI>(a, blockIdx.y - n, &lds[0].x);
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
  const TermScale ts = term_scale(bx, a.k2);
  float s = hw_exp2(fmaf(xe, ts.k, -ts.ref));
#pragma unroll
  for (int q = 0; q < U; ++q)
    if (v0 + q * BLOCK + tid < end) {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(&x[q]);
#pragma unroll
      for (int j = 0; j < EPV; ++j) s += hw_exp2(fmaf(TI::unpack(w, j), ts.k, -ts.ref));
    }
  s *= term_adj(bx, ts);
  __syncthreads();
  if (twice && (tid & 63) == 0) any_twice = 1;
  block_merge_at<BLOCK>(bx, s, a.k2, lds);
  if (tid == 0) a.part[row * a.parts + part] = PartSum{bx, s, any_twice, 0};
}

// The row's state outside K from its parts, and whether an id is used twice.
__device__ __forceinline__ void merge_tail(const DistillArgs& a, int64_t row, float& m, float& s, bool& twice) {
  const int lane = threadIdx.x & 63;
  m = kNegInf;
  s = 0.f;
  bool t = false;
  for (int p = lane; p < a.parts; p += 64) {
    const PartSum v = a.part[row * a.parts + p];
    const float M = fmaxf(m, v.mx);
    s = rescale_at(s, m, M, a.k2) + rescale_at(v.s, v.mx, M, a.k2);
    m = M;
    t |= v.n != 0;
  }
  lanes_merge_at<64>(m, s, a.k2);
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
    const int groups = groups_of(a);
    for (int w = __builtin_amdgcn_readfirstlane(tid >> 6); w < groups; w += static_cast<int>(blockDim.x) >> 6)
      put_late(a, te, w, load_late(a, row, w));
    __syncthreads();
    if (tid < 64) {
      float mt, st;
      bool twice;
      merge_tail(a, row, mt, st, twice);
      if (tid == 0 && twice) {
        te.row.state = kBad;
        if (part == 0) raise_error(a.err, kErrTeacherTwice);
      }
      float token = 0.f;
      if (te.row.state == kUsed) {
        double l = 0.;
        RowFactors f = row_factors(a, a.seq_scale[r.seq] * r.w, te, mt, st, l);
        for (int w = 0; w < groups; ++w) {
          const int i = tid + kWave * w;
          terms.g[i] = te.id[i] >= 0 ? entry_grad(a, te, f, i) : 0.f;
        }
        terms.tail = f.tail;
        terms.at = f.at;
        if (part == 0) {
          if (a.forward) {
            set_logs(a, f);
            l = row_loss(a, te, f);
          }
          token = r.w * static_cast<float>(l);
        }
      }
      if (part == 0 && tid == 0) store_coherent(a.token_loss + r.tix, token);
    }
    __syncthreads();
    live = te.row.state == kUsed;
  } else if (part == 0 && tid == 0 && r.tok) {
    store_coherent(a.token_loss + r.tix, 0.f);
  }
  float g[NS], tail = 0.f;
  TermScale ts{0.f, 0.f};
  int place[NS], edge[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    place[s] = edge[s] = -1;
    g[s] = 0.f;
  }
  if (live) {
    if constexpr (GRAD) {
      tail = terms.tail;
      ts = terms.at;
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const int id = kWave * s < a.k ? te.id[(tid & 63) + kWave * s] : -1;
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
        for (int j = 0; j < EPV; ++j) o[j] = tail * hw_exp2(fmaf(TI::unpack(w, j), ts.k, -ts.ref));
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
      float o = live && ek >= 0 ? tail * hw_exp2(fmaf(xe, ts.k, -ts.ref)) : 0.f;
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
  if (part == 0 && a.loss) finish_loss<GRAD ? BLOCK : 64>(a, static_cast<int>(a.nrows));
}

// ---------------------------------------------------------------------------
// A row to a workgroup, kept in registers from its one read to its gradient's write, by a
// persistent grid. A wave's loads and stores complete in order here, so a value loaded after a
// row's stores can be had only when they have gone out to memory, several microseconds later:
// nothing is loaded then but the row's chunks. Its record and entries, which the preparation
// has made, come with the row before's chunks and go to LDS before its stores. The sums need no
// maximum of their own: they are taken against the largest of the entries' logits, which is the
// row's largest or near it, and formed again against the true maximum where they are 2^60 off (a
// tail that is masked, or far above what the teacher named).
// Bound by memory and, nearly as much, by the two exponentials per element (the second instead
// of a second unpacked copy: 19 chunks of 16-bit logits fill the registers of 4 waves a SIMD).
// 8 sequences of 512 rows of 151,936 in bf16, part of them masked: 381 us; with the entries and
// the 64-bit arithmetic in the row's own workgroup 496, with them loaded after the row before's
// stores 441, with a few registers of the loop spilled to scratch memory 391 (a reload waits for
// the stores too: hence the buffer descriptors, 32-bit compares and wave-uniform indexes here).
// 512-thread workgroups, two to a CU, up to 8192 vectors: 16 sequences of 256 rows
// of 50,257 take 158 us (one of 1024 threads: 170). kBufNT stores against kBufNTSystem: 5 us
// less.
// Requirements (checked on the host): the row's interior fits BLOCK * NCH vectors; dlogits
// rows split like the logits rows, or hold f32 for 16-bit logits (dword-aligned stores).
// ---------------------------------------------------------------------------
// Narrow rows are dealt in grid strides, each starting `turn` further on, wide ones from a
// counter, for the reasons given at grpo_resident_kernel.
template <int BLOCK, int NCH>
constexpr bool kDealt = BLOCK * NCH <= 2048;

__device__ __forceinline__ float uniform(float v) { return read_lane(v, 0); }

// A wave's entries lie in lane-held lists: entry list[l] of the row with its place, lane l of
// group 0 in registers, of further groups (over 64 entries in one wave's part of the row: ids
// that lie close together) in LDS.
struct Owned {
  int place;         // of group 0's entry; -1
  int n;
  uint32_t chunks;   // bit k: chunk k holds one of them
};

template <typename TI, typename TO, int BLOCK, int NCH, int FULL>
__global__ void __launch_bounds__(BLOCK, 4) distill_row_kernel(DistillArgs a) {
  constexpr int EPV = 16 / TI::kBytes, NW = BLOCK / 64;
  constexpr bool kSplit = TI::kBytes == 2 && TO::kBytes == 4, kStatic = kDealt<BLOCK, NCH>;
  constexpr uint32_t kOutVec = EPV * TO::kBytes;
  static_assert(NW >= kMaxSlots, "a wave per group of entries");
  __shared__ Teacher te3[3];                   // of the row before (its loss comes with this row), this one, the next
  __shared__ RowFactors factors[NW];           // each wave its own copy of the same: out of registers under the stores
  __shared__ uint8_t list[NW][kMaxEntries];
  __shared__ float2 merge[NW];
  __shared__ int s_next[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), groups = groups_of(a);
  const uint32_t voff = tid * 16u, sgrp = split_group<TI, TO, BLOCK>(tid);
  const char* logits = static_cast<const char*>(a.logits);
  auto row_of = [&](int64_t row) { return logits + row * a.vocab * TI::kBytes; };
  // kSplit: half h of chunk k of this lane holds values of a row of nv vectors. (The chunk goes to
  // the uniform side: k * BLOCK + tid would be a register kept for each.)
  auto held = [&](int nv, int k, int h) {
    return k < FULL || (kSplit ? static_cast<int>(sgrp) < 2 * nv - k * 2 * BLOCK - 64 * h : tid < nv - k * BLOCK);
  };
  int64_t stride0 = 0;                                 // static: the last stride dealt
  uint32_t at = blockIdx.x;
  auto deal = [&]() -> int64_t {
    stride0 += gridDim.x;
    at += static_cast<uint32_t>(a.turn);
    if (at >= gridDim.x) at -= gridDim.x;
    return stride0 + at;
  };
  const int64_t grid = gridDim.x;
  int64_t row = blockIdx.x, next = kStatic ? deal() : blockIdx.x + grid;
  auto place_of = [&](int id, const RowSpan& sp) {     // -1 outside the interior
    return id >= 0 && id - sp.head < sp.nv * EPV ? entry_place<TI, kSplit, BLOCK, NCH>(id - sp.head, 0) : -1;
  };
  // This wave's entries of a row, into its list.
  auto own = [&](const Teacher& te, const RowSpan& sp) {
    int n = 0;
    for (int w = 0; w < groups; ++w) {
      const int p = place_of(te.id[lane + kWave * w], sp);
      const bool mine = p >= 0 && ((p >> 10) & 15) == wave;
      const uint64_t who = __ballot(mine);
      const int before = __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(who >> 32),
                                                   __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(who), 0));
      if (mine) list[wave][n + before] = static_cast<uint8_t>(lane + kWave * w);
      n += __popcll(who);
    }
    __builtin_amdgcn_wave_barrier();
    Owned o;
    o.n = n;
    o.place = lane < n ? place_of(te.id[list[wave][lane]], sp) : -1;
    o.chunks = n > kWave ? ~0u : 0u;
    for (int e = 0; e < min(n, kWave); ++e) o.chunks |= 1u << (__builtin_amdgcn_readlane(o.place, e) >> 16);
    return o;
  };
  // f(place, lane of the list, list group) for each of the wave's entries in chunk k.
  auto each_in_chunk = [&](const Teacher& te, const RowSpan& sp, const Owned& o, int k, auto f) {
    if ((o.chunks >> k & 1) == 0) return;
    uint64_t in = __ballot(o.place >= 0 && (o.place >> 16) == k);
    int place = o.place;
    for (int w = 0;;) {
      while (in) {
        const int src = __builtin_ctzll(in);
        in &= in - 1;
        f(__builtin_amdgcn_readlane(place, src), src, w);
      }
      if (++w * kWave >= o.n) break;
      place = kWave * w + lane < o.n ? place_of(te.id[list[wave][kWave * w + lane]], sp) : -1;
      in = __ballot(place >= 0 && (place >> 16) == k);
    }
  };
  // Adds chunk k's terms outside the entries to s, at ts; the entries' elements become -inf.
  auto sum_chunk = [&](u32x4& x, const Teacher& te, const RowSpan& sp, const Owned& o, int k, const TermScale& ts,
                       float& s) {
    each_in_chunk(te, sp, o, k, [&](int p, int, int) { mask_element<TI>(x, ((p >> 4) & 63) == lane, p & 15); });
    uint32_t u[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      u[q] = x[q];
      asm volatile("" : "+v"(u[q]));   // unpacked here and again for the gradient, not kept between
    }
    if constexpr (kSplit) {
#pragma unroll
      for (int q = 0; q < 2; ++q)
        if (held(sp.nv, k, q)) {
#pragma unroll
          for (int j = 4 * q; j < 4 * q + 4; ++j) s += hw_exp2(fmaf(TI::unpack(u, j), ts.k, -ts.ref));
        }
    } else if (held(sp.nv, k, 0)) {
#pragma unroll
      for (int j = 0; j < EPV; ++j) s += hw_exp2(fmaf(TI::unpack(u, j), ts.k, -ts.ref));
    }
    asm volatile("" : "+v"(s));   // here, not after the last chunk's entries
  };
  // Whether the wave's list has an id twice (equal ids have one place, so one wave has both).
  auto used_twice = [&](const Teacher& te, int n) {
    bool twice = false;
    const int mine = lane < n ? te.id[list[wave][lane]] : -1;
    for (int o = 0; o < min(n, kWave); ++o)
      twice |= lane < n && o != lane && __builtin_amdgcn_readlane(mine, o) == mine;
    for (int w = 1; kWave * w < n; ++w) {   // further groups against all before
      const int later = kWave * w + lane < n ? te.id[list[wave][kWave * w + lane]] : -1;
      for (int o = 0; o < min(n, kWave * w + kWave); ++o)
        twice |= kWave * w + lane < n && o < kWave * w + lane && te.id[list[wave][o]] == later;
    }
    return __any(twice);
  };
  // The same for the row's head and tail; this lane's element x of them becomes -inf where an entry
  // has it, or where there is none.
  auto mask_row_edges = [&](const Teacher& te, const RowSpan& sp, float& x) {
    const int ek = edge_index<TI>(sp, tid);
    int n = 0;
    if (ek >= 0)
      for (int i = 0; i < a.k; ++i) n += te.id[i] == ek;
    if (ek < 0 || n > 0) x = kNegInf;
    return __any(n > 1);
  };

  // The token of row i, -1 for a pad row.
  auto token_of = [&](int64_t i) -> int64_t {
    const uint32_t s = static_cast<uint32_t>(i) / static_cast<uint32_t>(a.logit_stride);
    const uint32_t t = static_cast<uint32_t>(i) - s * static_cast<uint32_t>(a.logit_stride);   // 64 bits: a vector compare
    return t < static_cast<uint32_t>(a.rows) ? s * a.tok_stride + a.tok_offset + t : -1;
  };
  auto scale_of = [&](int64_t i) { return a.seq_scale[static_cast<uint32_t>(i) / static_cast<uint32_t>(a.logit_stride)]; };
  auto pay = [&](const Teacher& te, int64_t owed) {    // by wave NW - 1: token `owed`'s loss
    RowFactors f = factors[wave];
    set_logs(a, f);
    const float l = static_cast<float>(row_loss(a, te, f));
    if (lane == 0) store_coherent(a.token_loss + owed, te.row.w * l);
  };

  if (wave < groups) put_late(a, te3[0], wave, load_late(a, row, wave));
  float scale = uniform(scale_of(row));
  int64_t owed = -1;
  int c = 0;                                           // te3[c]: this row's
  __syncthreads();
  for (int i = 0;; ++i) {
    const int cn = c == 2 ? 0 : c + 1, cp = c == 0 ? 2 : c - 1;
    const Teacher& te = te3[c];
    const float weight = uniform(te.row.w);
    const int64_t row_elem = row * a.vocab, token = token_of(row);
    const bool more = next < a.nrows;
    const RowSpan sp = row_span<TI>(row_of(row), a.vocab);
    const int ek = wave == 0 ? edge_index<TI>(sp, tid) : -1;
    const __amdgpu_buffer_rsrc_t drow = row_rsrc(static_cast<char*>(a.dlogits) + (row_elem + sp.head) * TO::kBytes,
                                                 static_cast<uint32_t>(sp.nv) * kOutVec);
    // (Under the loads its 64-bit arithmetic would need registers that they fill.)
    if (wave == NW - 1 && owed >= 0) pay(te3[cp], owed);
    owed = -1;
    __builtin_amdgcn_sched_barrier(0);
    u32x4 xv[NCH];
    float xe = 0.f;
    if (weight != 0.f) {
      const __amdgpu_buffer_rsrc_t buf = row_rsrc(sp.vec, static_cast<uint32_t>(sp.nv) * 16u);
#pragma unroll
      for (int k = 0; k < NCH; ++k) xv[k] = load_chunk<TI, TO, BLOCK>(buf, k, voff, sgrp);
    }
    // Ahead: the next row, and a claim for the one after it.
    const LateRow late = load_late(a, more ? next : row, min(wave, groups - 1));
    const float late_scale = scale_of(more ? next : row);
    int claimed = 0;
    if (!kStatic && tid == 0 && a.nrows > 2 * grid) claimed = atomicAdd(a.next_row, 1);
    Owned mine{-1, 0, 0u};                             // this wave's entries
    float g = 0.f, tail = 0.f;                         // the gradient at this lane's entry; elsewhere
    TermScale gs{0.f, 0.f};
    double loss = 0.;
    bool live = false;
    if (weight != 0.f) {
      mine = own(te, sp);
      bool twice = used_twice(te, mine.n);
      const TermScale ts{uniform(te.row.at.k), uniform(te.row.at.ref)};
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < NCH; ++k) {
        __builtin_amdgcn_sched_barrier(0);
        sum_chunk(xv[k], te, sp, mine, k, ts, s);
      }
      __builtin_amdgcn_sched_barrier(0);
      if (wave == 0) {
        if (ek >= 0) xe = TI::load1(row_of(row), ek);
        float x1 = xe;
        twice |= mask_row_edges(te, sp, x1);
        s += hw_exp2(fmaf(x1, ts.k, -ts.ref));
      }
      // The workgroup's sum, in a fixed order.
      s = lanes_sum<64>(s);
      if (lane == 0) merge[wave] = make_float2(s, twice ? 1.f : 0.f);
    }
    // What was loaded ahead goes out of registers before the row's factors need theirs.
    if (wave < groups) put_late(a, te3[cn], wave, late);
    if (!kStatic && tid == 0) s_next[i & 1] = a.nrows > 2 * grid ? claimed + 2 * static_cast<int>(grid) : INT32_MAX;
    const float scale_n = uniform(late_scale);
    __builtin_amdgcn_sched_barrier(0);
    if (weight != 0.f) {
      __syncthreads();
      const float2 w = merge[lane & (NW - 1)];
      float m = uniform(te.row.zref);
      const double first = wave_sum64(lane < NW ? static_cast<double>(w.x) : 0.);
      double st = first * te.row.adj;
      const bool any_twice = __any(w.y != 0.f);
      live = te.row.state == kUsed && !any_twice;
      if (live && !(first > 0x1p-60 && first < 0x1p60)) {
        // Too far from the entries: elements next to the tail's largest could leave f32's range. The
        // true maximum (the entries' elements are -inf by now), then the sum.
        float x1 = kNegInf;
        if (wave == 0) {
          x1 = xe;
          mask_row_edges(te, sp, x1);
        }
        float mx = x1;
#pragma unroll
        for (int k = 0; k < NCH; ++k)
#pragma unroll
          for (int j = 0; j < EPV; ++j)
            if (held(sp.nv, k, kSplit ? j / 4 : 0)) mx = fmaxf(mx, TI::unpack(reinterpret_cast<const uint32_t*>(&xv[k]), j));
        const TermScale own_ts = term_scale(mx, a.k2);
        float ss = hw_exp2(fmaf(x1, own_ts.k, -own_ts.ref));
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
          uint32_t u[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            u[q] = xv[k][q];
            asm volatile("" : "+v"(u[q]));
          }
#pragma unroll
          for (int j = 0; j < EPV; ++j)
            if (held(sp.nv, k, kSplit ? j / 4 : 0)) ss += hw_exp2(fmaf(TI::unpack(u, j), own_ts.k, -own_ts.ref));
          asm volatile("" : "+v"(ss));
        }
        __builtin_amdgcn_sched_barrier(0);
        ss *= term_adj(mx, own_ts);
        lanes_merge_at<64>(mx, ss, a.k2);
        __syncthreads();   // every wave has read the first sums
        if (lane == 0) merge[wave] = make_float2(mx, ss);
        __syncthreads();
        const float2 v = merge[lane & (NW - 1)];
        m = v.x;
        float st1 = v.y;
        lanes_merge_at<NW>(m, st1, a.k2);
        st = st1;
      }
      if (live) {
        const RowFactors f = row_factors(a, scale * weight, te, m, st, loss);
        if (lane == 0) factors[wave] = f;
        tail = uniform(f.tail);
        gs = TermScale{uniform(f.at.k), uniform(f.at.ref)};
        if (mine.place >= 0) g = entry_grad(a, te, f, list[wave][lane]);
      } else if (tid == 0 && any_twice && te.row.state == kUsed) {
        raise_error(a.err, kErrTeacherTwice);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    // Vectors past the row end sit past the descriptor: their stores are dropped.
    if (live) {
#pragma unroll
      for (int k = 0; k < NCH; ++k) {
        uint32_t u[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          u[q] = xv[k][q];
          asm volatile("" : "+v"(u[q]));
        }
        float out[EPV];
#pragma unroll
        for (int j = 0; j < EPV; ++j) out[j] = tail * hw_exp2(fmaf(TI::unpack(u, j), gs.k, -gs.ref));
        each_in_chunk(te, sp, mine, k, [&](int p, int src, int w) {
          const float ge = w == 0 ? read_lane(g, src) : entry_grad(a, te, factors[wave], list[wave][kWave * w + src]);
          const bool here = ((p >> 4) & 63) == lane;
#pragma unroll
          for (int j = 0; j < EPV; ++j)
            if (here && j == (p & 15)) out[j] = ge;
        });
        if constexpr (kSplit) {
          const float (&o0)[4] = reinterpret_cast<const float (&)[4]>(out[0]);
          const float (&o1)[4] = reinterpret_cast<const float (&)[4]>(out[4]);
          buf_store_vals<TO, 4, true>(drow, fresh_off(sgrp * 16u, k * 2 * BLOCK * 16u), o0);
          buf_store_vals<TO, 4, true>(drow, fresh_off(sgrp * 16u, k * 2 * BLOCK * 16u + 1024u), o1);
        } else {
          buf_store_vals<TO, EPV, true>(drow, fresh_off(tid * kOutVec, k * BLOCK * kOutVec), out);
        }
      }
    } else {
      const u32x4 zero = {0u, 0u, 0u, 0u};   // 0 bits are 0 in every output type
#pragma unroll
      for (int k = 0; k < NCH; ++k) {
        if constexpr (kSplit) {
#pragma unroll
          for (int q = 0; q < 2; ++q) buf_st16<true>(drow, zero, (k * 2 * BLOCK + 64 * q + sgrp) * 16u);
        } else {
#pragma unroll
          for (uint32_t q = 0; q < kOutVec; q += 16) buf_st16<true>(drow, zero, (k * BLOCK + tid) * kOutVec + q);
        }
      }
    }
    if (wave == 0) {
      if (ek >= 0) {
        float oe = live ? tail * hw_exp2(fmaf(xe, gs.k, -gs.ref)) : 0.f;
        if (live)
          for (int e = 0; e < a.k; ++e)
            if (te.id[e] == ek) oe = entry_grad(a, te, factors[0], e);
        store1<TO>(a.dlogits, row_elem + ek, oe);
      }
      if (tid == 0 && token >= 0 && !(live && a.forward))
        store_coherent(a.token_loss + token, live ? weight * static_cast<float>(loss) : 0.f);
    }
    if (live && a.forward) owed = token;
    if (!more) {
      if (wave == NW - 1 && owed >= 0) pay(te, owed);
      break;
    }
    __syncthreads();   // what was put ahead is there
    row = next;
    scale = scale_n;
    next = kStatic ? deal() : static_cast<int64_t>(__builtin_amdgcn_readfirstlane(s_next[i & 1]));
    c = cn;
  }
  if (a.loss) finish_loss<BLOCK>(a, static_cast<int>(gridDim.x));
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
  if (!with) launch_prepare<TI>(a, st);
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

template <typename TI, typename TO, int BLOCK, int NCH, int FULL>
hipError_t launch_row(DistillArgs a, hipStream_t st) {
  static std::atomic<int> cached{0};   // workgroups that the device holds at once
  int slots = cached.load(std::memory_order_relaxed);
  if (slots <= 0) {
    int dev = 0, cus = 0, occ = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e == hipSuccess) e = hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev);
    if (e == hipSuccess)
      e = hipOccupancyMaxActiveBlocksPerMultiprocessor(
          &occ, reinterpret_cast<const void*>(&distill_row_kernel<TI, TO, BLOCK, NCH, FULL>), BLOCK, 0);
    if (e != hipSuccess) return e;
    slots = cus * (occ > 0 ? occ : 1);
    cached.store(slots, std::memory_order_relaxed);
  }
  const int64_t grid = a.nrows < slots ? a.nrows : slots;
  launch_prepare<TI>(a, st);
  if (kDealt<BLOCK, NCH>) a.turn = resident_turn(grid, a.logit_stride, a.mask != nullptr);
  distill_row_kernel<TI, TO, BLOCK, NCH, FULL><<<dim3(static_cast<unsigned>(grid)), dim3(BLOCK), 0, st>>>(a);
  return hipGetLastError();
}

template <typename TI, typename TO>
hipError_t launch_rows_of(const DistillArgs& a, int64_t nv, hipStream_t st) {
  // FULL: chunks that every row of the configuration fills (its interior has nv - 1 vectors at least).
  if (nv <= 256) return launch_row<TI, TO, 256, 1, 0>(a, st);
  if (nv <= 512) return launch_row<TI, TO, 256, 2, 1>(a, st);
  if (nv <= 1024) return launch_row<TI, TO, 256, 4, 2>(a, st);
  if (nv <= 2048) return launch_row<TI, TO, 256, 8, 4>(a, st);
  if (nv <= 4096) return launch_row<TI, TO, 512, 8, 4>(a, st);
  if (nv <= 6656) return launch_row<TI, TO, 512, 13, 8>(a, st);
  if (nv <= 8192) return launch_row<TI, TO, 512, 16, 13>(a, st);
  if (nv <= 12288) return launch_row<TI, TO, 1024, 12, 8>(a, st);
  if (nv <= 16384) return launch_row<TI, TO, 1024, 16, 12>(a, st);
  if (nv <= kDistillRowVecs) return launch_row<TI, TO, 1024, 19, 16>(a, st);
  return hipErrorInvalidValue;
}

template <typename TI, typename TO>
hipError_t launch_pair(const DistillArgs& a, hipStream_t st) {
  if (a.parts > 0) return a.k <= kWave ? launch_parts<TI, TO, 1>(a, st) : launch_parts<TI, TO, kMaxSlots>(a, st);
  return launch_rows_of<TI, TO>(a, a.vocab * TI::kBytes / 16, st);
}

}  // namespace pcp
