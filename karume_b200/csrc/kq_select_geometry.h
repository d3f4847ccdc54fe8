// How many new tokens a block of the summaries' kernel goes through: host arithmetic, shared by the launcher and a host program of the test suite.
#pragma once

#include <cstdint>

namespace kq {
namespace select {

constexpr uint64_t kMostBlocks = 0x7FFFFFFFull;  // of a grid

inline uint64_t summary_blocks(uint32_t tokens, uint32_t heads, uint32_t each) { return (static_cast<uint64_t>(tokens) + each - 1) / each * heads; }
// One token a sequence: every one has a page, a block for each; else one of sixteen, or less, so four to a block.  More where a grid has not so many blocks.
inline uint32_t summary_rows(uint32_t tokens, uint32_t heads, bool one_each) {
  uint32_t each = one_each ? 1 : 4;
  while (summary_blocks(tokens, heads, each) > kMostBlocks) each *= 2;
  return each;
}

}  // namespace select
}  // namespace kq
