// Groups of neighbouring sequences that begin alike: which rows of a call are theirs, and how many blocks of rows they ask for.  Whole-number
// arithmetic shared by the kernels, their launchers and a host program of the test suite.
//
// Boundaries come from device arrays, which nobody has checked.  Where they ascend, and the first rows of the sequences at them do, each row is in one
// group at most: the blocks of all groups fit the grid that the host sizes for them, and whoever looks for a row's sums finds sums of this call.
// Where they do not, nothing is read once (worth_sharing), and every sequence walks over all of its keys.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define KQ_ANYWHERE __host__ __device__ __forceinline__
#else
#define KQ_ANYWHERE inline
#endif

namespace kq {
namespace groups {

// Groups of a launch: a kernel keeps what it found of each in shared memory; more come in turns.
constexpr uint32_t kAtOnce = 128;

struct Range {
  int begin, end;
};
KQ_ANYWHERE int between(int x, int low, int high) { return x < low ? low : x > high ? high : x; }

// First row of sequence b's new tokens, 0 <= b <= sequences; without starts every sequence has one.
KQ_ANYWHERE int row_of(const int* starts, int b, int tokens) { return between(starts ? starts[b] : b, 0, tokens); }
// Sequences of a group between two boundaries, and its rows.
KQ_ANYWHERE Range sequences_of(int first, int next, int sequences) {
  const int begin = between(first, 0, sequences);
  return Range{begin, between(next, begin, sequences)};
}
KQ_ANYWHERE Range rows_of(const Range& group, const int* starts, int tokens) {
  const int begin = row_of(starts, group.begin, tokens), end = row_of(starts, group.end, tokens);
  return Range{begin, end < begin ? begin : end};
}
// Of all groups of a call: their rows are disjoint, and in order.
KQ_ANYWHERE bool in_order(int first, int next, const int* starts, int sequences, int tokens) {
  return first <= next && row_of(starts, between(first, 0, sequences), tokens) <= row_of(starts, between(next, 0, sequences), tokens);
}

// Blocks of `block` query rows, at most, that groups (or sequences) with more than `beyond` of them ask for: full ones, and one begun for each.
inline uint64_t most_blocks(uint64_t rows, uint32_t block, uint64_t groups, uint32_t beyond) {
  const uint64_t large = rows / (static_cast<uint64_t>(beyond) + 1);
  return rows / block + (groups < large ? groups : large);
}

}  // namespace groups
}  // namespace kq
