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

// Workgroups per row: about one on each CU in all, so that few wait for the ticket at a time, and a batch (kLeastPart vectors)
// each or more. us of rows of 151,936 with 1024 workgroups in all | 512 | 256, by then of several batches each:
//   64 f32 rows     k 0   14.0 | 12.4 | 11.9     k 5   19.4 | 17.8 | 17.1
//   32 bf16 rows           8.9 |  9.0 |  8.8           12.9 | 12.9 | 14.0
//   64 bf16 rows          10.5 | 10.4 | 10.1           15.2 | 16.2 | 15.7
//   100 bf16 rows         11.9 | 12.5 | 14.3           17.5 | 19.3 | 20.5
//   200 bf16 rows         16.9 | 18.7 | 17.8           25.1 | 25.8 | 24.2
//   255 bf16 rows         19.6 | 19.6 | 18.4           27.1 | 26.9 | 24.8     (256, one part each: 16.5, 20.8)
// It suits numbers of rows that divide the CUs; the 300 workgroups of 100 rows and the 510 of 255 leave some CUs one more than
// others. Half a batch each took one bf16 row of 151,936 with k = 20 from 12 to 19 us. 1520 f16 rows of 50,257 in 8192 took
// 25 us for 26, but 1024 bf16 rows of 151,936 62 for 54 and 4096 of them 133 for 129.
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
