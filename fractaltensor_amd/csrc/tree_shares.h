// How many workgroups of a head of keys the work of trees is shared out to (paged_attn.h), and of how many keys its grains are.  No HIP in here.
#pragma once

#include <limits.h>

#include <algorithm>
#include <cmath>

namespace ftk {

constexpr int kPartsMost = 256;  // parts of a row: what joins them has registers for the weights of so many

struct TreeShares {
  int shares;                    // 0: the work cannot be shared out
  int grain_shift;               // grains of 2^grain_shift keys
};

// capacity: positions that a sequence has room for; row_blocks: blocks of rows that one may have.
inline TreeShares share_trees(long long sequences, long long row_blocks, int heads, long long capacity, int cus) {
  TreeShares s{0, 7};
  // The least grains whose number over all sequences and blocks of rows has 32 bits, whatever lengths the device finds; there may be none.
  const auto grains = [&](int shift) { return (double)sequences * row_blocks * ((double)(std::min<long long>(capacity, INT_MAX) >> shift) + 1.0); };
  while (s.grain_shift < 30 && grains(s.grain_shift) > 1e9) ++s.grain_shift;
  // (the kernels have a lane for each block of rows of a sequence)
  if (row_blocks > 64 || grains(s.grain_shift) > 1e9) return s;
  // As many as there are compute units, or twice as many and more where the heads divide those badly, but no fewer than blocks of rows, each of which begins with a workgroup of its own.
  long long shares = 0;
  double used = 0.0;
  for (int rounds = 1; rounds <= 4 && used < 0.9; ++rounds) {
    const long long n = std::max<long long>(rounds * (long long)cus / heads, 1);
    const double u = (double)n * heads / (std::ceil((double)n * heads / cus) * cus);
    if (u > used) {
      used = u;
      shares = n;
    }
  }
  // (one sequence may be left in as many parts as there are shares)
  s.shares = (int)std::min<long long>(std::max(shares, row_blocks), kPartsMost);
  return s;
}

}  // namespace ftk
