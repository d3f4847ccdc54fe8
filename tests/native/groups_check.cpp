// Host-side check of karume_b200/csrc/kq_groups.h over random boundaries, in order and not: groups that are in order have disjoint rows, which ask for no
// more blocks than the launcher's grid has, and whoever finds itself in a group has its rows among the group's.  Prints how many calls were in
// order, and how many out of order would have asked for more blocks than there are.
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "kq_groups.h"

namespace {

int failures = 0;
#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); ++failures; } } while (0)

struct Call {
  std::vector<int> first, starts;
  int sequences, tokens;
  uint32_t heads, block, beyond;
  const int* at() const { return starts.empty() ? nullptr : starts.data(); }
};

bool ordered(const Call& c) {
  bool all = true;
  for (size_t g = 0; g + 1 < c.first.size(); ++g) all &= kq::groups::in_order(c.first[g], c.first[g + 1], c.at(), c.sequences, c.tokens);
  return all;
}
// Blocks that the groups ask for beyond those that there are.
long long excess(const Call& c) {
  long long asked = 0;
  for (size_t g = 0; g + 1 < c.first.size(); ++g) {
    const kq::groups::Range rows = kq::groups::rows_of(kq::groups::sequences_of(c.first[g], c.first[g + 1], c.sequences), c.at(), c.tokens);
    const uint64_t n = static_cast<uint64_t>(rows.end - rows.begin) * c.heads;
    CHECK(rows.begin >= 0 && rows.begin <= rows.end && rows.end <= c.tokens);
    if (n > c.beyond) asked += static_cast<long long>((n + c.block - 1) / c.block);
  }
  return asked - static_cast<long long>(kq::groups::most_blocks(static_cast<uint64_t>(c.tokens) * c.heads, c.block, c.first.size() - 1, c.beyond));
}
void in_order_is_enough(const Call& c) {
  CHECK(excess(c) <= 0);
  int end = 0;
  for (size_t g = 0; g + 1 < c.first.size(); ++g) {
    const kq::groups::Range of = kq::groups::sequences_of(c.first[g], c.first[g + 1], c.sequences), rows = kq::groups::rows_of(of, c.at(), c.tokens);
    if (rows.end == rows.begin) continue;
    CHECK(rows.begin >= end);
    end = rows.end;
  }
  // the group that halving finds for each sequence
  for (int b = 0; b < c.sequences; ++b) {
    size_t lo = 0, hi = c.first.size() - 1;
    while (hi - lo > 1) {
      const size_t mid = (lo + hi) / 2;
      (c.first[mid] <= b ? lo : hi) = mid;
    }
    if (c.first[lo] > b || c.first[lo + 1] <= b) continue;
    const kq::groups::Range rows = kq::groups::rows_of(kq::groups::sequences_of(c.first[lo], c.first[lo + 1], c.sequences), c.at(), c.tokens);
    const int begin = kq::groups::row_of(c.at(), b, c.tokens), next = c.starts.empty() ? std::min(b + 1, c.tokens) : std::max(begin, kq::groups::row_of(c.at(), b + 1, c.tokens));
    if (c.starts.empty() || (c.starts[std::max(c.first[lo], 0)] <= begin && c.starts[std::min(c.first[lo + 1], c.sequences)] >= next))
      CHECK(rows.begin <= begin && next <= rows.end);
  }
}

}  // namespace

int main() {
  std::mt19937 rng(7);
  const auto pick = [&](int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); };
  long long good = 0, wild = 0;
  for (int i = 0; i < 200000; ++i) {
    Call c;
    c.sequences = pick(1, 80);
    const int groups = pick(1, c.sequences);
    c.heads = 1u << pick(0, 5);
    c.block = pick(0, 1) ? 128 : 256;
    c.beyond = pick(0, 1) ? 32 : 0;
    if (pick(0, 1)) {
      c.starts.push_back(pick(0, 3) ? 0 : pick(-3, 5));
      for (int b = 0; b < c.sequences; ++b) c.starts.push_back(c.starts.back() + pick(0, 9));
      c.tokens = std::max(c.starts.back() + (pick(0, 2) ? 0 : pick(-5, 5)), 1);
      if (pick(0, 3) == 0) std::swap(c.starts[pick(0, c.sequences)], c.starts[pick(0, c.sequences)]);
    } else {
      c.tokens = c.sequences;
    }
    for (int g = 0; g <= groups; ++g) c.first.push_back(pick(0, 9) ? pick(0, c.sequences) : pick(-(1 << 30), 1 << 30));
    if (pick(0, 2)) std::sort(c.first.begin(), c.first.end());
    if (ordered(c)) {
      ++good;
      in_order_is_enough(c);
    } else {
      wild += excess(c) > 0;
    }
  }
  // groups that take turns at the same 63 sequences
  Call c{{}, {}, 64, 64, 32, 256, 0};
  for (int g = 0; g < 64; ++g) c.first.push_back(g % 2 ? 63 : 0);
  c.first.push_back(64);
  CHECK(!ordered(c) && excess(c) > 0);
  std::printf("%lld %lld\n", good, wild);
  return failures != 0;
}
