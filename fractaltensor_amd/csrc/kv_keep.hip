// Caches of limited length: which positions of a sequence stay (by the weights that they have gathered), and moving the rows that stay together.
//
// select.  The budget's heaviest positions, without sorting: a workgroup to a (sequence, head) finds the weight at the border by counting.  Weights are
// taken as whole numbers that have their order; the range that holds the border, at first from the least to the greatest, is cut into 1024 or 2048 equal
// parts, the positions of each are counted in LDS, and the part that holds the border is the next range: mostly two rounds, since a range of some binades
// has hundreds of parts in each, and at most four (32 bits by 10; 32 by 11 take three; the upper and the lower 16 bits by 11 two each).  (Cutting by the bits from the top instead puts nearly all positions into a few parts, whose counting takes turns.)
// Then every wave writes the positions of its own stretch in their order, behind those of the waves before it.
//
// keep.  Row kept[j] of a list that ascends goes to place j <= kept[j].  In place, that is safe without a second buffer as long as no place
// is written before it has been read: rows of later j come from behind all places of earlier ones, so a workgroup takes the list in order, some
// pieces of 16 bytes a thread at a time, with all of a step's reads done before its first write.  Rows are cut into slices of 32 to 256 bytes, each a workgroup's of its own with
// nothing to wait for, where sequences and heads alone leave compute units idle.  The first slice's workgroup moves a row's exponent too, that of K its weight.  Bound by reading
// and writing each moved byte once, beside whole lines for the exponents and weights of rows that lie apart.
#include <algorithm>

#include "kv_common.h"

namespace ftk {

// ---- select -----------------------------------------------------------------------------

struct SelectArgs {
  const float* weights;          // [pages, heads, 2^page_shift]
  int pages, heads, page_shift;
  KvBatch batch;                 // (starts and tokens are not looked at)
  int* kept;                     // [sequences, heads, budget]
  int budget, sinks, recent;
};

// A weight as a whole number with its order, from 2^16 up; both zeros alike, NaN below all.  Zero is left for what is not chosen from.
__device__ __forceinline__ unsigned ordered(float x) {
  const unsigned u = __float_as_uint(x + 0.0f);
  return x != x ? 0x10000u : u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}

// A wave has a stretch of whole 256 positions, a lane four neighbours of each 256.  The keys of the first CHUNKS of these are held: whole, or, PACKED, their upper 16 bits, two
// to a register, which find the border but for its lower 16 bits; those of the few positions whose upper bits are the border's are read again.
template <int WAVES, int CHUNKS, bool PACKED>
__global__ __launch_bounds__(WAVES * 64) void kv_select_kernel(SelectArgs a) {
  constexpr int THREADS = WAVES * 64, BINS = WAVES == 16 ? 2048 : 1024, LOG = WAVES == 16 ? 11 : 10, PER = BINS / THREADS, UNIT = PACKED ? 16 : 0;
  constexpr int GROUP = CHUNKS < 8 ? CHUNKS : 8;                 // chunks whose loads are on their way together
  __shared__ unsigned bins[BINS], sums[WAVES][2], found[3];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int b = blockIdx.x / a.heads, head = blockIdx.x - b * a.heads;
  const int len = min(max(load_uniform(a.batch.lens, b), 0), kv_capacity(a.batch, a.page_shift));
  int* const kept = a.kept + (long long)blockIdx.x * a.budget;
  if (len <= a.budget) {                                         // all stay
    for (int i = tid; i < a.budget; i += THREADS) kept[i] = i < len ? i : -1;
    return;
  }
  // [from, to): the positions that are chosen from; sinks + recent <= budget < len
  const int from = a.sinks, to = len - a.recent;
  const int stretch = (len + 256 * WAVES - 1) / (256 * WAVES) * 256, begin = wave * stretch + 4 * lane, steps = stretch / 256;
  const int* const table = a.batch.table + (long long)b * a.batch.width;
  const auto look = [&](int p) __attribute__((always_inline)) {
    return p < len ? table[p >> a.page_shift] : -1;
  };
  const auto read = [&](int p, int page) __attribute__((always_inline)) {
    const bool there = page >= 0 && page < a.pages;
    return *reinterpret_cast<const v4f*>(a.weights + (there ? (((long long)page * a.heads + head) << a.page_shift) + (p & ((1 << a.page_shift) - 1)) : 0));
  };
  // the keys of four positions, zero for those that are not chosen from; of these, the bits of those in the sequence
  const auto keys_of = [&](int p, int page, v4f w, unsigned (&k)[4]) __attribute__((always_inline)) {
    unsigned sure = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool open = p + e >= from && p + e < to;
      k[e] = !open ? 0u : page >= 0 && page < a.pages ? ordered(w[e]) : 0x10000u;
      if (!open && p + e < len) sure |= 1u << e;
    }
    return sure;
  };
  // from memory.  (What one pass has compared or worked out is not to be kept for the next, here and for the keys that are held: it would be far more than there are registers.)
  const auto loose = [&](int i, unsigned (&k)[4]) __attribute__((always_inline)) {
    int p = begin + 256 * i;
    asm volatile("" : "+v"(p));
    const int page = look(p);
    return keys_of(p, page, read(p, page), k);
  };
  constexpr int WORDS = (CHUNKS + 7) / 8, REGS = PACKED ? 2 : 4;
  unsigned h[CHUNKS][REGS], stay[WORDS], tied[WORDS];            // four bits a chunk: of those that stay, and of those at the border
#pragma unroll
  for (int w = 0; w < WORDS; ++w) stay[w] = tied[w] = 0;
#pragma unroll
  for (int g = 0; g < CHUNKS; g += GROUP) {
    if (g < steps) {
      int page[GROUP];
      v4f w[GROUP];
#pragma unroll
      for (int u = 0; u < GROUP; ++u) page[u] = look(begin + 256 * (g + u));
#pragma unroll
      for (int u = 0; u < GROUP; ++u) w[u] = read(begin + 256 * (g + u), page[u]);
#pragma unroll
      for (int u = 0; u < GROUP; ++u) {
        unsigned k[4];
        unsigned sure = keys_of(begin + 256 * (g + u), page[u], w[u], k);
        if (g + u >= steps) {                                    // the next wave's
          sure = 0;
          k[0] = k[1] = k[2] = k[3] = 0;
        }
        stay[(g + u) / 8] |= sure << (4 * ((g + u) % 8));
        if constexpr (PACKED) {
          h[g + u][0] = k[0] >> 16 | (k[1] & 0xffff0000u);
          h[g + u][1] = k[2] >> 16 | (k[3] & 0xffff0000u);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) h[g + u][e] = k[e];
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
#pragma unroll
      for (int u = 0; u < GROUP; ++u)
#pragma unroll
        for (int j = 0; j < REGS; ++j) h[g + u][j] = 0;
    }
  }
  // f(chunk, its four keys >> UNIT) for what is held.
  const auto for_held = [&](auto&& f) __attribute__((always_inline)) {
#pragma unroll
    for (int g = 0; g < CHUNKS; g += GROUP)
      if (g < steps) {
#pragma unroll
        for (int i = g; i < g + GROUP; ++i) {
          unsigned k[4];
          if constexpr (PACKED) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              asm volatile("" : "+v"(h[i][j]));
              k[2 * j] = h[i][j] & 0xffffu;
              k[2 * j + 1] = h[i][j] >> 16;
            }
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              asm volatile("" : "+v"(h[i][j]));
              k[j] = h[i][j];
            }
          }
          f(i, k);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
  };
  // f(key >> UNIT) for all that a lane has, zeros among it
  const auto for_upper = [&](auto&& f) __attribute__((always_inline)) {
    for_held([&](int, const unsigned (&k)[4]) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < 4; ++e) f(k[e]);
    });
    for (int i = CHUNKS; i < steps; ++i) {
      unsigned k[4];
      loose(i, k);
#pragma unroll
      for (int e = 0; e < 4; ++e) f(k[e] >> UNIT);
    }
  };
  // The border among the keys that each(f) hands to f, all between low and high: keys above *border stay, and the first *ties of those at it.
  const auto find = [&](auto&& each, unsigned low, unsigned high, unsigned need, unsigned* border, unsigned* ties) __attribute__((always_inline)) {
    for (int round = 0; round < 4; ++round) {                    // 32 bits by 10
      const int shift = max(0, 32 - (int)__builtin_clz((high - low) | 1u) - LOG);   // parts of 2^shift keys
#pragma unroll
      for (int i = 0; i < PER; ++i) bins[i * THREADS + tid] = 0;
      __syncthreads();
      each([&](unsigned k) __attribute__((always_inline)) {
        if (k - low <= high - low) atomicAdd(&bins[(k - low) >> shift], 1u);
      });
      __syncthreads();
      // from the top: thread i has the bins below those of thread i - 1
      unsigned own[PER], sum = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        own[i] = bins[BINS - 1 - (tid * PER + i)];
        sum += own[i];
      }
      unsigned end = sum;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const unsigned y = (unsigned)__shfl_up((int)end, o);
        if (lane >= o) end += y;
      }
      if (lane == 63) sums[wave][0] = end;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < WAVES; ++i)
        if (i < wave) end += sums[i][0];
      unsigned above = end - sum;
      if (above < need && end >= need) {                         // one thread
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          if (above < need && above + own[i] >= need) {
            found[0] = BINS - 1 - (tid * PER + i);
            found[1] = above;
            found[2] = own[i];
          }
          above += own[i];
        }
      }
      __syncthreads();
      low += found[0] << shift;
      need -= found[1];
      if (found[2] == need && low > 0) {                         // all of the part stay
        *border = low - 1;
        *ties = 0;
        return;
      }
      if (shift == 0) break;
      high = min(high, low + ((1u << shift) - 1));
    }
    *border = low;
    *ties = need;
  };
  unsigned border = 0xffffffffu >> UNIT, ties = 0;               // of upper keys
  const unsigned need = a.budget - a.sinks - a.recent;
  if (need > 0) {
    unsigned low = 0xffffffffu, high = 0;                        // (low is one less)
    for_upper([&](unsigned k) __attribute__((always_inline)) {
      low = min(low, k - 1);
      high = max(high, k);
    });
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      low = min(low, (unsigned)__shfl_xor((int)low, o));
      high = max(high, (unsigned)__shfl_xor((int)high, o));
    }
    if (lane == 0) {
      sums[wave][0] = low;
      sums[wave][1] = high;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
      low = min(low, sums[i][0]);
      high = max(high, sums[i][1]);
    }
    find(for_upper, low + 1, high, need, &border, &ties);
  }
  // PACKED: the lower bits, of those whose upper ones are the border's
  unsigned whole = 0xffffffffu, whole_ties = ties;               // the border of whole keys
  bool split = false;
  if constexpr (PACKED) {
    split = ties > 0;
    if (split) {
      const auto for_whole = [&](auto&& f) __attribute__((always_inline)) {
        for_held([&](int i, const unsigned (&u)[4]) __attribute__((always_inline)) {
          if (u[0] == border || u[1] == border || u[2] == border || u[3] == border) {
            unsigned k[4];
            loose(i, k);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (k[e] >> 16 == border) f(k[e]);
          }
        });
        for (int i = CHUNKS; i < steps; ++i) {
          unsigned k[4];
          loose(i, k);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (k[e] >> 16 == border) f(k[e]);
        }
      };
      find(for_whole, border << 16, border << 16 | 0xffffu, ties, &whole, &whole_ties);
    }
  }
  const unsigned quota = PACKED ? (split ? whole_ties : 0) : ties;
  // ---- which stay
  const auto bits_of = [&](const unsigned (&k)[4], unsigned* at) __attribute__((always_inline)) {   // of whole keys
    unsigned in = 0;
    *at = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool above = PACKED ? k[e] >> 16 > border || (split && k[e] >> 16 == border && k[e] > whole) : k[e] > border;
      if (above) in |= 1u << e;
      if (quota > 0 && k[e] == (PACKED ? whole : border)) *at |= 1u << e;
    }
    return in;
  };
  for_held([&](int i, const unsigned (&u)[4]) __attribute__((always_inline)) {
    unsigned in = 0, t = 0;
    if constexpr (PACKED) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (u[e] > border) in |= 1u << e;
      if (split && (u[0] == border || u[1] == border || u[2] == border || u[3] == border)) {
        unsigned k[4];
        loose(i, k);
        in = bits_of(k, &t);
      }
    } else {
      in = bits_of(u, &t);
    }
    stay[i / 8] |= in << (4 * (i % 8));
    tied[i / 8] |= t << (4 * (i % 8));
  });
  const auto nibble = [&](const unsigned (&x)[WORDS], int i) __attribute__((always_inline)) { return x[i / 8] >> (4 * (i % 8)) & 15u; };
  // how many of a number of 0 to 4 the lanes in front have
  const auto in_front = [&](unsigned n, unsigned* all) __attribute__((always_inline)) {
    unsigned before = 0, total = 0;
#pragma unroll
    for (int bit = 0; bit < 3; ++bit) {
      const unsigned long long m = __builtin_amdgcn_ballot_w64(n >> bit & 1);
      before += (unsigned)__builtin_amdgcn_mbcnt_hi((unsigned)(m >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)m, 0u)) << bit;
      total += (unsigned)__popcll(m) << bit;
    }
    *all = total;
    return before;
  };
  const auto wave_total = [&](unsigned n) __attribute__((always_inline)) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) n += (unsigned)__shfl_xor((int)n, o);
    return n;
  };
  // waves in front of this one
  const auto waves_in_front = [&](unsigned n, int which) __attribute__((always_inline)) {
    if (lane == 0) sums[wave][which] = n;
    __syncthreads();
    unsigned before = 0;
#pragma unroll
    for (int i = 0; i < WAVES; ++i)
      if (i < wave) before += sums[i][which];
    return before;
  };
  // the first `quota` of those at the border stay too
  unsigned rank = 0;                                             // of the next at the border
  const auto settle = [&](unsigned in, unsigned t) __attribute__((always_inline)) {
    unsigned all;
    unsigned r = rank + in_front(__builtin_popcount(t), &all);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (t >> e & 1) {
        if (r < quota) in |= 1u << e;
        ++r;
      }
    rank += all;
    return in;
  };
  if (quota > 0) {
    unsigned n = 0;
#pragma unroll
    for (int w = 0; w < WORDS; ++w) n += __builtin_popcount(tied[w]);
    for (int i = CHUNKS; i < steps; ++i) {
      unsigned k[4], t;
      loose(i, k);
      bits_of(k, &t);
      n += __builtin_popcount(t);
    }
    __syncthreads();
    rank = waves_in_front(wave_total(n), 0);
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      const unsigned t = nibble(tied, i);
      if (__builtin_amdgcn_ballot_w64(t != 0) != 0) stay[i / 8] |= settle(0, t) << (4 * (i % 8));
    }
  }
  const unsigned loose_rank = rank;
  unsigned n = 0;
#pragma unroll
  for (int w = 0; w < WORDS; ++w) n += __builtin_popcount(stay[w]);
  for (int i = CHUNKS; i < steps; ++i) {
    unsigned k[4], t;
    const unsigned sure = loose(i, k);
    n += __builtin_popcount(settle(sure | bits_of(k, &t), t));
  }
  unsigned at = waves_in_front(wave_total(n), 1);
  const auto write = [&](unsigned in, int i) __attribute__((always_inline)) {
    unsigned all;
    unsigned place = at + in_front(__builtin_popcount(in), &all);
    while (in != 0) {
      if (place < (unsigned)a.budget) kept[place] = begin + 256 * i + __builtin_ctz(in);
      in &= in - 1;
      ++place;
    }
    at += all;
  };
#pragma unroll
  for (int w = 0; w < WORDS; ++w)
#pragma unroll 1
    for (int i = 8 * w; i < min(min(8 * w + 8, CHUNKS), steps); ++i) write(stay[w] >> (4 * (i % 8)) & 15u, i);
  rank = loose_rank;
  for (int i = CHUNKS; i < steps; ++i) {
    unsigned k[4], t;
    const unsigned sure = loose(i, k);
    const unsigned in = sure | bits_of(k, &t);
    write(settle(in, t), i);
  }
}

// ---- keep -------------------------------------------------------------------------------

struct KeepArgs {
  KvPages pages;
  KvBatch batch;                 // starts NULL: rows are counted from a sequence's first position, else from that of its first new token
  const int* kept;               // [sequences, lists, most]
  int most, per_head;            // per_head: a list for each head
  float* weights;                // may be NULL
  int* lens;                     // [sequences], results
  int row_bytes, slices, lanes;  // of a row; slices of 16 * lanes bytes
};

constexpr int kKeepThreads = 512, kKeepItems = 8;
constexpr int kKeepList = 2048;                      // entries of a list whose rows are looked up at once

// Every lane loads, those whose row does not move the cache's first: only loads that are always there can be waited for by their number.  (In the place of exponents and weights
// that another workgroup moves, and may be writing, it is the list's first entry.)
template <int LANES, bool EXPS, bool WEIGHTS>
__global__ __launch_bounds__(kKeepThreads, 4) void kv_keep_kernel(KeepArgs a) {
  constexpr int ROWS = kKeepThreads / LANES, STEP = ROWS * kKeepItems;
  static_assert(kKeepList % STEP == 0);
  __shared__ long long sources[kKeepList], places[kKeepList];  // cache rows; place -1: the row stays where it is, or there is none
  __shared__ int count, ends, some;
  const int tid = threadIdx.x, piece = tid % LANES, in = tid / LANES;
  int id = blockIdx.x;
  const int slice = id % a.slices;
  id /= a.slices;
  const bool values = id & 1;
  id >>= 1;
  const int b = id / a.pages.heads, head = id - b * a.pages.heads;
  const int all = max(load_uniform(a.batch.lens, b), 0), len = min(all, kv_capacity(a.batch, a.pages.page_shift)), shift = a.pages.page_shift;
  const int first = a.batch.starts ? first_position(all, load_uniform(a.batch.starts, b), load_uniform(a.batch.starts, b + 1)) : 0;
  const int* const kept = a.kept + (a.per_head ? (long long)b * a.pages.heads + head : b) * a.most;
  const int* const table = a.batch.table + (long long)b * a.batch.width;
  unsigned char* const data = (values ? a.pages.v : a.pages.k) + slice * 16 * LANES + 16 * piece;
  signed char* const exps = values ? a.pages.v_exps : a.pages.k_exps;
  const bool with_exps = EXPS && slice == 0 && piece == 0, with_weights = WEIGHTS && slice == 0 && piece == 0 && !values;
  const signed char* const exps_from = slice == 0 ? exps : reinterpret_cast<const signed char*>(kept);
  const float* const weights_from = slice == 0 && !values ? a.weights : reinterpret_cast<const float*>(kept);
  const long long exps_mask = slice == 0 ? -1 : 0, weights_mask = slice == 0 && !values ? -1 : 0;
  const bool counts = slice == 0 && !values && head == 0;        // one workgroup of a sequence says how many stay
  // the cache row of a position, -1: it has none
  const auto row_of = [&](long long position) __attribute__((always_inline)) -> long long {
    const bool in_sequence = position >= 0 && position < len;
    const int p = in_sequence ? (int)position : 0, page = in_sequence ? table[p >> shift] : -1;
    return page < 0 || page >= a.pages.pages ? -1 : (((long long)page * a.pages.heads + head) << shift) + (p & ((1 << shift) - 1));
  };
  if (tid == 0) count = 0;
  for (int l0 = 0; l0 < a.most; l0 += kKeepList) {
    const int entries = min(a.most - l0, kKeepList), steps = (entries + STEP - 1) / STEP;
    __syncthreads();
    if (tid == 0) ends = some = 0;
    __syncthreads();
    int n = 0;
#pragma unroll
    for (int t = 0; t < kKeepList / kKeepThreads; ++t) {
      const int i = t * kKeepThreads + tid;
      if (i - tid >= steps * STEP) break;
      const int k = i < entries ? kept[l0 + i] : -1;
      n += k >= 0;
      const bool moves = k >= 0 && k != l0 + i;
      const long long from = moves ? row_of((long long)first + k) : -1, to = moves ? row_of((long long)first + l0 + i) : -1;
      sources[i] = from >= 0 && to >= 0 ? from : 0;
      places[i] = from >= 0 ? to : -1;
      if (from >= 0) some = 1;
      if (i < entries && k < 0) ends = 1;                        // a list ends at its first negative entry
    }
    if (counts && n) atomicAdd(&count, n);
    __syncthreads();
    // What is read in a step is written in the next but one half: the rows of step s + 1 come from behind all places of step s, and are asked for in front of its writes.
    v4u x[2][kKeepItems];
    int e[2][kKeepItems];
    float w[2][kKeepItems];
    const auto ask = [&](int s, v4u (&x)[kKeepItems], int (&e)[kKeepItems], float (&w)[kKeepItems]) __attribute__((always_inline)) {
      long long from[kKeepItems];
#pragma unroll
      for (int u = 0; u < kKeepItems; ++u) from[u] = sources[s * STEP + u * ROWS + in];
#pragma unroll
      for (int u = 0; u < kKeepItems; ++u) {
        x[u] = *reinterpret_cast<const v4u*>(data + from[u] * a.row_bytes);
        if constexpr (EXPS) e[u] = exps_from[from[u] & exps_mask];
        if constexpr (WEIGHTS) w[u] = weights_from[from[u] & weights_mask];
      }
    };
    const auto write = [&](int s, v4u (&x)[kKeepItems], int (&e)[kKeepItems], float (&w)[kKeepItems]) __attribute__((always_inline)) {
      // all that the workgroup reads in this step is in registers before any of its places is written
#pragma unroll
      for (int u = 0; u < kKeepItems; ++u) {
        asm volatile("" : "+v"(x[u]));
        if constexpr (EXPS) asm volatile("" : "+v"(e[u]));
        if constexpr (WEIGHTS) asm volatile("" : "+v"(w[u]));
      }
      asm volatile("s_barrier" ::: "memory");
#pragma unroll
      for (int u = 0; u < kKeepItems; ++u) {
        const long long to = places[s * STEP + u * ROWS + in];
        if (to < 0) continue;
        *reinterpret_cast<v4u*>(data + to * a.row_bytes) = x[u];
        if constexpr (EXPS) {
          if (with_exps) exps[to] = (signed char)e[u];
        }
        if constexpr (WEIGHTS) {
          if (with_weights) a.weights[to] = w[u];
        }
      }
    };
    const bool last = ends;
    if (some) {
      ask(0, x[0], e[0], w[0]);
      for (int s = 0; s < steps; s += 2) {
        if (s + 1 < steps) ask(s + 1, x[1], e[1], w[1]);
        write(s, x[0], e[0], w[0]);
        if (s + 1 >= steps) break;
        if (s + 2 < steps) ask(s + 2, x[0], e[0], w[0]);
        write(s + 1, x[1], e[1], w[1]);
      }
    }
    if (last) break;
  }
  if (counts) {
    __syncthreads();
    if (tid == 0) a.lens[b] = (int)min(max((long long)first + count, 0LL), (long long)INT_MAX);
  }
}

static int check_weights(const char* who, const float* weights, int pages, int heads, int page_size) {
  if (!weights || !aligned16(weights)) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: weights must be non-NULL and 16-byte aligned", who);
  if (pages <= 0 || heads <= 0) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: pages and heads must be positive", who);
  if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1)))
    return fail(FTK_ERR_UNSUPPORTED_SHAPE, "%s: page size must be a power of two from 16 to 1024, got %d", who, page_size);
  return FTK_OK;
}

}  // namespace ftk

extern "C" {

int ftk_kv_cache_select(const float* weights, int pages, int heads, int page_size, const int* table, const int* lens, int sequences, int table_width, int budget,
                        int sinks, int recent, int max_keys, int* kept, ftk_stream_t stream) {
  using namespace ftk;
  const char* who = "ftk_kv_cache_select";
  if (int rc = check_weights(who, weights, pages, heads, page_size)) return rc;
  if (sequences < 0 || table_width < 0 || max_keys < 0) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: sequences, table width and max_keys must not be negative", who);
  if (budget <= 0 || sinks < 0 || recent < 0 || (long long)sinks + recent > budget)
    return fail(FTK_ERR_INVALID_ARGUMENT, "%s: the budget must be positive and have room for %d first and %d last positions, got %d", who, sinks, recent, budget);
  if (sequences == 0) return FTK_OK;
  if (table_width == 0) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: the table has no columns", who);
  if (!table || !lens || !kept || (((uintptr_t)table | (uintptr_t)lens | (uintptr_t)kept) & 3))
    return fail(FTK_ERR_INVALID_ARGUMENT, "%s: table, lens and kept must be non-NULL and 4-byte aligned", who);
  if ((long long)sequences * heads > INT_MAX) return fail(FTK_ERR_UNSUPPORTED_SHAPE, "%s: too many sequences and heads", who);
  const int shift = __builtin_ctz((unsigned)page_size);
  const long long capacity = (long long)table_width << shift, most = max_keys > 0 ? std::min<long long>(max_keys, capacity) : capacity;
  const SelectArgs a{weights, pages, heads, shift, KvBatch{table, lens, nullptr, sequences, table_width, 0}, kept, budget, sinks, recent};
  const dim3 grid((unsigned)(sequences * (long long)heads));
  const hipStream_t s = (hipStream_t)stream;
  // Four waves up to 4096 positions, sixteen beyond; all of up to 16384, or the upper halves of 131072, are held in registers, and more are read again each time.
  if (most <= 4096) hipLaunchKernelGGL((kv_select_kernel<4, 4, false>), grid, dim3(256), 0, s, a);
  else if (most <= 16384) hipLaunchKernelGGL((kv_select_kernel<16, 4, false>), grid, dim3(1024), 0, s, a);
  else hipLaunchKernelGGL((kv_select_kernel<16, 32, true>), grid, dim3(1024), 0, s, a);
  return check_launch("kv_select_kernel");
}

int ftk_kv_cache_keep(const ftk_kv_pages* pages, const int* table, const int* lens, const int* starts, int sequences, int table_width, const int* kept, int most,
                      int per_head, float* weights, int* new_lens, ftk_stream_t stream) {
  using namespace ftk;
  const char* who = "ftk_kv_cache_keep";
  KeepArgs a;
  if (int rc = check_kv_pages(who, pages, &a.pages)) return rc;
  if (sequences < 0 || table_width < 0 || most < 0) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: sequences, table width and the lists' length must not be negative", who);
  if (sequences == 0) return FTK_OK;
  if (new_lens == lens) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: the new lengths must not be where the old ones are", who);
  if (!new_lens || !lens || (most > 0 && (!table || !kept))) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: table, lens, kept and the new lengths must be non-NULL", who);
  if (most > 0 && table_width == 0) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: the table has no columns", who);
  if (((uintptr_t)table | (uintptr_t)lens | (uintptr_t)starts | (uintptr_t)kept | (uintptr_t)weights | (uintptr_t)new_lens) & 3)
    return fail(FTK_ERR_INVALID_ARGUMENT, "%s: table, lens, starts, kept and weights must be 4-byte aligned", who);
  const DeviceProps* d = nullptr;
  if (int rc = device_props(&d)) return rc;
  a.batch = KvBatch{table, lens, starts, sequences, table_width, 0};
  a.kept = kept;
  a.most = most;
  a.per_head = per_head != 0;
  a.weights = weights;
  a.lens = new_lens;
  const bool exps = pages->k_exps != nullptr;
  a.row_bytes = pages->head_size * (exps ? 1 : 2);
  // the largest power of two that divides a row, then half of it while workgroups are few
  int bytes = a.row_bytes & -a.row_bytes;
  const long long units = 2LL * sequences * pages->heads;
  while (bytes > 64 && units * (a.row_bytes / bytes) < 2LL * d->cus) bytes /= 2;
  a.lanes = bytes / 16;
  a.slices = a.row_bytes / bytes;
  const long long blocks = units * a.slices;
  if (blocks > INT_MAX) return fail(FTK_ERR_UNSUPPORTED_SHAPE, "%s: grid too large", who);
  auto launch = [&](auto lanes, auto e, auto w) -> int {
    hipLaunchKernelGGL((kv_keep_kernel<decltype(lanes)::value, decltype(e)::value, decltype(w)::value>), dim3((unsigned)blocks), dim3(kKeepThreads), 0, (hipStream_t)stream, a);
    return check_launch("kv_keep_kernel");
  };
  auto with_extras = [&](auto lanes) -> int {
    using yes = std::true_type;
    using no = std::false_type;
    if (exps) return weights ? launch(lanes, yes{}, yes{}) : launch(lanes, yes{}, no{});
    return weights ? launch(lanes, no{}, yes{}) : launch(lanes, no{}, no{});
  };
  switch (a.lanes) {
    case 2: return with_extras(std::integral_constant<int, 2>{});
    case 4: return with_extras(std::integral_constant<int, 4>{});
    case 8: return with_extras(std::integral_constant<int, 8>{});
    default: return with_extras(std::integral_constant<int, 16>{});
  }
}

}  // extern "C"
