// Host-side check of karume_b200/csrc/kq_select_geometry.h: every new token of every call that is not refused belongs to a block, and the blocks fit a grid.
#include <cstdio>
#include <initializer_list>

#include "kq_select_geometry.h"

int main() {
  int failures = 0;
  const uint32_t tokens[] = {1, 2, 3, 4, 5, 63, 64, 1000, 1u << 20, (1u << 23) - 1, 1u << 23, (1u << 24) - 1, 1u << 24, (1u << 30) - 3, 1u << 30};
  const uint32_t heads[] = {1, 2, 3, 8, 127, 128, 129, 255, 256, 300, 511, 512, 1023, 1024};
  for (const uint32_t t : tokens)
    for (const uint32_t h : heads)
      for (const bool one_each : {false, true}) {
        if (static_cast<uint64_t>(t) * h > (1ull << 33) || (one_each && t > (1u << 24))) continue;  // refused
        const uint32_t each = kq::select::summary_rows(t, h, one_each);
        const uint64_t blocks = kq::select::summary_blocks(t, h, each), least = one_each ? 1 : 4;
        // the last block's last token; half as many tokens a block would not fit; small calls as they were
        if (blocks > 0x7FFFFFFFull || blocks / h * each < t || (blocks / h - 1) * each + each > 0xFFFFFFFFull || each < least ||
            (each > least && kq::select::summary_blocks(t, h, each / 2) <= 0x7FFFFFFFull)) {
          std::printf("%u tokens, %u heads: %u a block, %llu blocks\n", t, h, each, (unsigned long long)blocks);
          ++failures;
        }
      }
  return failures != 0;
}
