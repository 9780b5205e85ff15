// Caches of limited length: which positions of a sequence stay (by the weights that they have gathered), and moving the rows that stay together.
//
// select.  The budget's heaviest positions, without sorting: a workgroup to a (sequence, head) finds the weight at the border by counting.  Weights are
// taken as whole numbers that have their order; the range that holds the border, at first from the least to the greatest, is cut into 1024 or 2048 equal
// parts, the positions of each are counted in LDS, and the part that holds the border is the next range: three rounds at most, mostly two, since a range of some binades
// has hundreds of parts in each.  (Cutting by the bits from the top instead puts nearly all positions into a few parts, whose counting takes turns.)
// Then every wave writes the positions of its own stretch in their order, behind those of the waves before it.
//
// keep.  Row kept[j] of a list that ascends goes to place j <= kept[j].  In place, that is safe without a second buffer as long as no place
// is written before it has been read: rows of later j come from behind all places of earlier ones, so a workgroup takes the list in order, 256 pieces of 16
// bytes or more at a time, with all of a step's reads done before its first write.  Rows are cut into slices of 16 to 256 bytes, each a workgroup's of its own with
// nothing to wait for, where sequences and heads alone leave compute units idle.  Bound by reading and writing each moved byte once.
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

// A weight as a whole number with its order; NaN below all, both zeros alike.
__device__ __forceinline__ unsigned ordered(float x) {
  const unsigned u = __float_as_uint(x + 0.0f);
  return x != x ? 0u : u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}

template <int WAVES, int ITEMS>
__global__ __launch_bounds__(WAVES * 64) void kv_select_kernel(SelectArgs a) {
  constexpr int THREADS = WAVES * 64, BINS = WAVES == 16 ? 2048 : 1024, PER = BINS / THREADS;
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
  unsigned need = a.budget - a.sinks - a.recent;
  // a wave has a stretch of whole 256 positions, a lane four neighbours of each 256; the keys of the first ITEMS are held
  const int stretch = (len + 256 * WAVES - 1) / (256 * WAVES) * 256, begin = wave * stretch, steps = stretch / 256;
  const auto load = [&](int i, unsigned (&x)[4]) __attribute__((always_inline)) {
    const int p = begin + 256 * i + 4 * lane;
    v4f w = {0.f, 0.f, 0.f, 0.f};
    bool there = false;
    if (p < len) {
      const int page = a.batch.table[(long long)b * a.batch.width + (p >> a.page_shift)];
      there = page >= 0 && page < a.pages;
      if (there) w = *reinterpret_cast<const v4f*>(a.weights + ((((long long)page * a.heads + head) << a.page_shift) + (p & ((1 << a.page_shift) - 1))));
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = there ? ordered(w[e]) : 0u;
  };
  unsigned held[ITEMS][4];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i)
    if (i < steps) load(i, held[i]);
  // f(key, position) for what a lane has between from and to
  const auto for_each = [&](auto&& f) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
      if (i < steps) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int p = begin + 256 * i + 4 * lane + e;
          if (p >= from && p < to) f(held[i][e]);
        }
      }
    for (int i = ITEMS; i < steps; ++i) {
      unsigned x[4];
      load(i, x);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int p = begin + 256 * i + 4 * lane + e;
        if (p >= from && p < to) f(x[e]);
      }
    }
  };
  // ---- the border: positions with a key above `border` stay, and the first `ties` of those at it
  unsigned border = 0xffffffffu, ties = 0;
  if (need > 0) {
    unsigned low = 0xffffffffu, high = 0;
    for_each([&](unsigned k) __attribute__((always_inline)) {
      low = min(low, k);
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
    for (int round = 0; round < 4; ++round) {                    // 32 bits by 10
      // parts of 2^shift keys
      const int shift = max(0, 32 - (int)__builtin_clz((high - low) | 1u) - (BINS == 2048 ? 11 : 10));
#pragma unroll
      for (int i = 0; i < PER; ++i) bins[i * THREADS + tid] = 0;
      __syncthreads();
      for_each([&](unsigned k) __attribute__((always_inline)) {
        if (k >= low && k <= high) atomicAdd(&bins[(k - low) >> shift], 1u);
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
      const unsigned here = found[2];
      if (here == need && low > 0) {                             // all of the part stay
        border = low - 1;
        break;
      }
      if (shift == 0) {
        border = low;
        ties = need;
        break;
      }
      high = min(high, low + ((1u << shift) - 1));
    }
    __syncthreads();
  }
  // ---- how many stay in front of each wave, then their positions
  const auto marks = [&](const unsigned (&x)[4], int i, unsigned long long (&in)[4], unsigned long long (&tie)[4]) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int p = begin + 256 * i + 4 * lane + e;
      const bool free_choice = p >= from && p < to;
      in[e] = __builtin_amdgcn_ballot_w64(p < len && (!free_choice || x[e] > border));
      tie[e] = __builtin_amdgcn_ballot_w64(free_choice && x[e] == border && ties > 0);
    }
  };
  unsigned sure = 0, tied = 0;
  const auto count = [&](const unsigned (&x)[4], int i) __attribute__((always_inline)) {
    unsigned long long in[4], tie[4];
    marks(x, i, in, tie);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      sure += __popcll(in[e]);
      tied += __popcll(tie[e]);
    }
  };
#pragma unroll
  for (int i = 0; i < ITEMS; ++i)
    if (i < steps) count(held[i], i);
  for (int i = ITEMS; i < steps; ++i) {
    unsigned x[4];
    load(i, x);
    count(x, i);
  }
  if (lane == 0) {
    sums[wave][0] = sure;
    sums[wave][1] = tied;
  }
  __syncthreads();
  unsigned at = 0, ties_before = 0;
#pragma unroll
  for (int i = 0; i < WAVES; ++i)
    if (i < wave) {
      at += sums[i][0];
      ties_before += sums[i][1];
    }
  at += min(ties_before, ties);
  const auto write = [&](const unsigned (&x)[4], int i) __attribute__((always_inline)) {
    unsigned long long in[4], tie[4];
    marks(x, i, in, tie);
    const unsigned long long below = (1ULL << lane) - 1;
    unsigned t = ties_before;                                    // ties in front of this lane's, then of each of its four
    unsigned n = 0;                                              // sure ones in front
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      t += __popcll(tie[e] & below);
      n += __popcll(in[e] & below);
    }
    unsigned place = at + n + min(t, ties) - min(ties_before, ties);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool is = in[e] >> lane & 1, is_tie = tie[e] >> lane & 1;
      const bool stays = is || (is_tie && t < ties);
      if (stays && place < (unsigned)a.budget) kept[place] = begin + 256 * i + 4 * lane + e;
      place += stays;
      t += is_tie;
    }
    unsigned all_ties = 0, all = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      all += __popcll(in[e]);
      all_ties += __popcll(tie[e]);
    }
    at += all + min(ties_before + all_ties, ties) - min(ties_before, ties);
    ties_before += all_ties;
  };
#pragma unroll
  for (int i = 0; i < ITEMS; ++i)
    if (i < steps) write(held[i], i);
  for (int i = ITEMS; i < steps; ++i) {
    unsigned x[4];
    load(i, x);
    write(x, i);
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
  int exps;                      // whether rows have exponents
};

constexpr int kKeepThreads = 256, kKeepItems = 8;

template <int LANES>
__global__ __launch_bounds__(kKeepThreads) void kv_keep_kernel(KeepArgs a) {
  constexpr int ROWS = kKeepThreads / LANES;
  const int tid = threadIdx.x, piece = tid % LANES, in = tid / LANES;
  int id = blockIdx.x;
  const int slice = id % a.slices;
  id /= a.slices;
  const bool values = id & 1;
  id >>= 1;
  const int b = id / a.pages.heads, head = id - b * a.pages.heads;
  const int all = max(load_uniform(a.batch.lens, b), 0), len = min(all, kv_capacity(a.batch, a.pages.page_shift));
  const int first = a.batch.starts ? first_position(all, load_uniform(a.batch.starts, b), load_uniform(a.batch.starts, b + 1)) : 0;
  const int* const kept = a.kept + (a.per_head ? (long long)b * a.pages.heads + head : b) * a.most;
  const int* const table = a.batch.table + (long long)b * a.batch.width;
  unsigned char* const data = (values ? a.pages.v : a.pages.k) + slice * 16 * LANES + 16 * piece;
  signed char* const exps = values ? a.pages.v_exps : a.pages.k_exps;
  const bool extra = slice == 0 && piece == 0, with_exps = extra && a.exps, with_weights = extra && !values && a.weights;
  // the cache row of a position, -1: it has none
  const auto row_of = [&](long long position) __attribute__((always_inline)) -> long long {
    if (position < 0 || position >= len) return -1;
    const int page = table[position >> a.pages.page_shift];
    if (page < 0 || page >= a.pages.pages) return -1;
    return (((long long)page * a.pages.heads + head) << a.pages.page_shift) + (position & ((1 << a.pages.page_shift) - 1));
  };
  __shared__ int count;
  const bool counts = blockIdx.x == (unsigned)(b * a.pages.heads * 2 * a.slices);    // one workgroup of a sequence says how many stay
  if (counts && tid == 0) count = 0;
  if (counts) __syncthreads();
  for (int j0 = 0; j0 < a.most; j0 += ROWS * kKeepItems) {
    long long from[kKeepItems], to[kKeepItems];
    bool listed = false;
#pragma unroll
    for (int u = 0; u < kKeepItems; ++u) {
      const int j = j0 + u * ROWS + in, k = j < a.most ? kept[j] : -1;
      const bool moves = k >= 0 && k != j;
      listed |= k >= 0;
      from[u] = moves ? row_of((long long)first + k) : -1;
      to[u] = moves ? row_of((long long)first + j) : -1;
      if (counts && piece == 0 && k >= 0) atomicAdd(&count, 1);
    }
    v4u x[kKeepItems];
    signed char e[kKeepItems];
    float w[kKeepItems];
#pragma unroll
    for (int u = 0; u < kKeepItems; ++u) {
      x[u] = v4u{0, 0, 0, 0};
      e[u] = 0;
      w[u] = 0.0f;
      if (from[u] >= 0 && to[u] >= 0) {
        x[u] = *reinterpret_cast<const v4u*>(data + from[u] * a.row_bytes);
        if (with_exps) e[u] = exps[from[u]];
        if (with_weights) w[u] = a.weights[from[u]];
      }
    }
    // all that the workgroup reads in this step is in registers before any of it is written
    int flag[kKeepItems];
#pragma unroll
    for (int u = 0; u < kKeepItems; ++u) {
      flag[u] = e[u];
      asm volatile("" : "+v"(x[u]), "+v"(flag[u]), "+v"(w[u]));
    }
    const bool more = __syncthreads_or(listed);
#pragma unroll
    for (int u = 0; u < kKeepItems; ++u) {
      if (from[u] >= 0 && to[u] >= 0) {
        *reinterpret_cast<v4u*>(data + to[u] * a.row_bytes) = x[u];
        if (with_exps) exps[to[u]] = (signed char)flag[u];
        if (with_weights) a.weights[to[u]] = w[u];
      }
    }
    if (!more) break;                                            // a list ends at its first negative entry
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
  // Four waves up to 4096 positions, sixteen beyond; up to 16384 positions, or the first 65536, stay in registers.
  if (most <= 4096) hipLaunchKernelGGL((kv_select_kernel<4, 4>), grid, dim3(256), 0, s, a);
  else if (most <= 16384) hipLaunchKernelGGL((kv_select_kernel<16, 4>), grid, dim3(1024), 0, s, a);
  else hipLaunchKernelGGL((kv_select_kernel<16, 16>), grid, dim3(1024), 0, s, a);
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
  a.exps = pages->k_exps != nullptr;
  a.row_bytes = pages->head_size * (a.exps ? 1 : 2);
  // the largest power of two that divides a row, then half of it while workgroups are few
  int bytes = a.row_bytes & -a.row_bytes;
  const long long units = 2LL * sequences * pages->heads;
  while (bytes > 64 && units * (a.row_bytes / bytes) < 2LL * d->cus) bytes /= 2;
  a.lanes = bytes / 16;
  a.slices = a.row_bytes / bytes;
  const long long blocks = units * a.slices;
  if (blocks > INT_MAX) return fail(FTK_ERR_UNSUPPORTED_SHAPE, "%s: grid too large", who);
  auto launch = [&](auto lanes) -> int {
    hipLaunchKernelGGL((kv_keep_kernel<decltype(lanes)::value>), dim3((unsigned)blocks), dim3(kKeepThreads), 0, (hipStream_t)stream, a);
    return check_launch("kv_keep_kernel");
  };
  switch (a.lanes) {
    case 2: return launch(std::integral_constant<int, 2>{});
    case 4: return launch(std::integral_constant<int, 4>{});
    case 8: return launch(std::integral_constant<int, 8>{});
    default: return launch(std::integral_constant<int, 16>{});
  }
}

}  // extern "C"
