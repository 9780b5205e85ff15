// share_trees (fractaltensor_amd/csrc/tree_shares.h) over sizes of any order of magnitude: it ends, and what it says fits what the kernels hold.  Prints what does not and ends with 1.
#include <cstdio>

#include "../fractaltensor_amd/csrc/tree_shares.h"

int main() {
  int bad = 0, shared = 0, refused = 0;
  const long long sequences[] = {1, 2, 3, 16, 70, 4096, 1 << 20, 1 << 27, INT_MAX}, blocks[] = {1, 2, 7, 64, 65, 262144, 1 << 27};
  const long long capacities[] = {16, 8192, 131072, 1 << 24, INT_MAX, (long long)INT_MAX << 10};
  const int heads[] = {1, 2, 3, 5, 8, 12, 16, 96, 300, 100000};
  for (long long n : sequences)
    for (long long k : blocks)
      for (long long c : capacities)
        for (int h : heads)
          for (int cus : {1, 64, 256, 304, 1000}) {
            const ftk::TreeShares s = ftk::share_trees(n, k, h, c, cus);
            if (s.shares == 0) {
              ++refused;
              continue;
            }
            ++shared;
            // all lines' grains are added up in 32 bits, a line of a lane each
            const long long keys = std::min<long long>(c, INT_MAX);
            const bool fits = s.grain_shift >= 7 && s.grain_shift <= 30 && (double)n * k * (double)((keys + (1LL << s.grain_shift) - 1) >> s.grain_shift) <= INT_MAX;
            if (!fits || k > 64 || s.shares < k || s.shares > ftk::kPartsMost) {
              std::printf("%lld sequences, %lld blocks, %d heads, %lld positions, %d units: %d shares of 2^%d keys\n", n, k, h, c, cus, s.shares, s.grain_shift);
              ++bad;
            }
          }
  // sizes as they are met are shared out, to one workgroup of each unit
  const ftk::TreeShares usual = ftk::share_trees(16, 1, 8, 8192, 256);
  if (usual.shares != 32 || usual.grain_shift != 7) {
    std::printf("16 sequences, 8 heads: %d shares of 2^%d keys\n", usual.shares, usual.grain_shift);
    ++bad;
  }
  if (!shared || !refused) ++bad;
  return bad != 0;
}
