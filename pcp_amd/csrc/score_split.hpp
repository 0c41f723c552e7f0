// How a call of token scores deals its rows to workgroups (score_kernels.hip). Host arithmetic alone.
#pragma once

#include <algorithm>
#include <cstdint>

namespace pcp {

// Rows of fewer than this may share a row between workgroups (a ticket each), about as many of those in all: the CUs.
constexpr int kScoreTickets = 256;
constexpr int kScoreBlock = 256;   // threads of a workgroup
constexpr int kScoreU = 8;         // 16-byte vectors per lane and batch
constexpr int kScoreGroups = 16;   // groups of batches that a lane keeps maxima of
constexpr int kScoreParts = 64;    // most parts of a row: one wave merges their sums

struct ScoreSplit {
  int64_t parts;   // of a row
  int64_t per;     // vectors of a part
  int32_t group;   // batches of a group, 1 or more
};

// Workgroups per row: about one on each CU in all, so that few wait for the ticket at a time, and a batch (kLeastPart vectors) each
// or more. us with 1024 workgroups in all | 512 | 256, by then of several batches each:
//   64 f32 rows of 151,936, k 0   16.0 | 12.7 | 12.0     k 5   19.8 | 18.3 | 17.0     100 bf16 rows, k 0   12.4 | 12.8 | 14.4
//   200 bf16 rows                 18.8 | 19.1 | 18.3           27.5 | 25.9 | 24.2     500 bf16 rows        36.3 | 34.8 | 31.9
// Half a batch each took one bf16 row of 151,936 with k = 20 from 12 to 19 us. 1520 f16 rows of 50,257 in 8192 took 25 us for 26,
// but 1024 bf16 rows of 151,936 62 for 54 and 4096 of them 133 for 129.
inline ScoreSplit score_split(int64_t n_rows, int64_t vocab, int elem_bytes) {
  constexpr int64_t kBlock = kScoreBlock, kLeastPart = kScoreU * kBlock;
  const int64_t nv = vocab * elem_bytes / 16;
  int64_t parts = 1, per = (nv + kBlock - 1) / kBlock * kBlock;
  if (n_rows < kScoreTickets && nv > kLeastPart) {   // (a ticket per row)
    parts = std::min<int64_t>((kScoreTickets + n_rows - 1) / n_rows, kScoreParts);
    per = ((nv + parts - 1) / parts + kBlock - 1) / kBlock * kBlock;
    // A part of one batch is gathered from registers: as long as that leaves no CU two.
    const int64_t ones = (nv + kLeastPart - 1) / kLeastPart;
    if (per < kLeastPart || (per <= 2 * kLeastPart && ones <= kScoreParts && n_rows * ones <= kScoreTickets)) per = kLeastPart;
    parts = (nv + per - 1) / per;
  }
  const int64_t of_group = kLeastPart * kScoreGroups;
  return {parts, per, static_cast<int32_t>(std::max<int64_t>(1, (per + of_group - 1) / of_group))};   // (per 0: no whole vector)
}

}  // namespace pcp
