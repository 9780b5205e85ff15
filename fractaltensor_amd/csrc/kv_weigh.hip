// The attention weights that new tokens give to the positions of a paged cache, gathered position by position.
//
// weights[k] = decay * weights[k] + sum over new tokens t and heads of the group of exp(scale q_t . k - lse_t), the sum of a column of the
// attention matrix where attention itself needs the sums of its rows.  So a workgroup has KEYS and walks the rows (row r is token r / G, head
// r % G): four waves of 64 keys each over rows of Q in LDS, which they share.  The product is S = Q K^T with a key to a lane, so that a lane adds up its own
// key's weights in one register, and only the two or four lanes of a key meet at the end.  There are no atomics: the sum of a key has one order.
//
//   few rows   (at most 64 to a sequence: decoding, drafts) are bound by reading K, straight into registers.  64 sequences of up to 8192 keys, 8 heads of 128 in e4m3: 83 us,
//              4.4 TB/s with all that is read and written; in bf16 5.2, and 6.0 for one sequence of 131072.  (A lane's 16 bytes lie beside those of three others of its row: copies of
//              whole lines, whose rows the product could not use, were 6 % faster.)
//   many rows  (chunks, prompts): the keys' fragments stay in registers, and the products of 32 rows go beside the exponentials of the 32 in front of them (32x32x16:
//              with 16x16x32 the two pipes got in each other's way).  Four prompts of 4096, 16 heads of 128, fp16: 168 us under a causal mask, 0.82 PFLOP/s, three quarters
//              of what a large library product reaches beside it, and 340 without one.  There it is the card's power that bounds it: without the exponentials 1.0, and neither
//              less LDS traffic nor fewer instructions changed the time.  Prompts of unlike lengths end unevenly: 4096, 1749 and 3648 tokens, 864 workgroups of up to 2048 rows on
//              the 512 that there is room for, take 126 us, 0.54 PFLOP/s; in parts of 1024 rows 140, of 512 161, since each begins with 3 to 4 us.  (At D 128 six registers spill.)
//
// Scores and sums are fp32; codes of 8 bits enter the product as they are, exact in both 16-bit types, and the power of two of a key's row multiplies its scores.
#include <float.h>

#include <algorithm>
#include <cmath>

#include "kv_common.h"

namespace ftk {

constexpr int kWeighRows = 64;   // rows of Q in LDS at once
constexpr int kBlock = 256;      // keys of a workgroup

struct WeighArgs {
  const void* q;
  const float* lse;                // [tokens, heads]
  long long q_token, q_head;       // strides, elements
  KvPages pages;                   // (v is not looked at)
  KvBatch batch;
  float* weights;                  // [pages, kv heads, 2^page_shift]
  int heads, group;                // query heads, query heads of a kv head
  unsigned inverse;                // ceil(2^32 / group): r / group of any row (1: 0)
  float scale_log2e, decay;
  int causal, window;
  int even_blocks;                 // 64 rows are whole tokens, and begin within 2 GB of one another
  int tiles;                       // blocks of keys of a (sequence, head) that the grid has
  int parts, part_rows;            // many rows: how they are cut
  float* sums;                     // [sequences, kv heads, parts, tiles * 256], where they are
};

__device__ __forceinline__ int token_of(const WeighArgs& a, unsigned row) { return a.group == 1 ? (int)row : (int)__umulhi(row, a.inverse); }

// 16 bytes a lane from an address of its own into LDS.
__device__ __forceinline__ void lds_dma16_each(const void* from, void* lds_base) {
  const unsigned lds_addr = (unsigned)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void*)lds_base);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(lds_addr), "v"(from) : "memory", "m0");
}

__device__ __forceinline__ void lds_dma4_each(const void* from, void* lds_base) {
  const unsigned lds_addr = (unsigned)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void*)lds_base);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" : : "s"(lds_addr), "v"(from) : "memory", "m0");
}

__device__ __forceinline__ void lds_dma4(const void* gbase, unsigned byte_off, void* lds_base) {
  const unsigned lds_addr = (unsigned)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void*)lds_base);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" : : "s"(lds_addr), "v"(byte_off), "s"(gbase) : "memory", "m0");
}

// The 16-byte slot that chunk c of a row of Q takes is c ^ turn(row): 16 rows' reads of one chunk then lie in different banks.
template <int BYTES>
__device__ __forceinline__ int turn(int row) {
  if constexpr (BYTES == 256) return row & 15;
  else if constexpr (BYTES == 128) return (row >> 1) & 7;
  else return (row >> 2) & 3;      // 192 and 64
}

template <int D>
struct WeighShape {
  static constexpr int BYTES = 2 * D, Q = kWeighRows * BYTES;
  static constexpr int ROWS = kWeighRows * 4;                  // lse in powers of two
  static constexpr int BLOCK = Q + ROWS, BLOCKS = 4, LDS = BLOCKS * BLOCK;
  static constexpr int LOADS = Q / 4096 + 1;                   // of a wave for a block
};

// A row of the cache as a lane of the product holds its key: of 16 (KG = 4 lanes share a row) or 32 (KG = 2) keys the lane has elements 8 KG s + 8 kg of the row in
// fragment s, or, of codes, 16 neighbours a load in two fragments, where the row has them.  (The product takes the elements in any order, if Q's reads have the same.)
template <typename T, KvFormat F, int D, int KG>
struct KeyRow {
  static constexpr int KS = D / (8 * KG), CACHED = F == kSame ? 2 * D : D, PAIRS = F == kSame ? KS : KS / 2;
  v4u whole[PAIRS > 0 ? PAIRS : 1];
  v2u last;
  __device__ __forceinline__ void load(const WeighArgs& a, long long row, int kg) {
    const unsigned char* const from = a.pages.k + (size_t)row * CACHED;
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) whole[i] = *reinterpret_cast<const v4u*>(from + 16 * KG * i + 16 * kg);
    if constexpr (F != kSame && KS % 2) last = *reinterpret_cast<const v2u*>(from + 16 * KG * PAIRS + 8 * kg);
  }
  __device__ __forceinline__ typename T::v8 fragment(int s) const {
    if constexpr (F == kSame) {
      return __builtin_bit_cast(typename T::v8, whole[s]);
    } else {
      if (KS % 2 && s == KS - 1) return decode8<T, F>(last, 1.0f);
      const v4u w = whole[s / 2];
      return s % 2 ? decode8<T, F>(v2u{w[2], w[3]}, 1.0f) : decode8<T, F>(v2u{w[0], w[1]}, 1.0f);
    }
  }
  // the 16 bytes of a row of Q that go with it
  static __device__ __forceinline__ int chunk(int s, int kg) { return F != kSame && (s | 1) < KS ? 2 * KG * (s / 2) + 2 * kg + (s & 1) : KG * s + kg; }
};

// How many rows of a sequence belong to tokens in front of `token`: those rows r that see a position, under a causal mask from the position's own on, are r >= rows_before(position -
// first), so that a mask compares rows and needs no division.
__device__ __forceinline__ int rows_before(const WeighArgs& a, const KvChunk& c, long long token) { return (int)min(max(token, 0LL), (long long)c.n) * a.group; }
__device__ __forceinline__ int first_row(const WeighArgs& a, const KvChunk& c, int key) { return a.causal ? rows_before(a, c, (long long)key - c.first) : 0; }
__device__ __forceinline__ int end_row(const WeighArgs& a, const KvChunk& c, int key) { return a.window > 0 ? rows_before(a, c, (long long)key - c.first + a.window) : c.n * a.group; }

// Blocks of 64 rows of Q and their lse on their way into LDS; a wave copies rows 16 wave .. + 15 of a block.  Where a group divides 64 a lane's rows lie at the same
// distances from each block's first row, and no block but the last costs vector instructions, of which there are none to spare.
template <typename T, int D>
struct RowStage {
  using S = WeighShape<D>;
  using scalar = typename T::scalar;
  static constexpr int CH = S::BYTES / 16, COPIES = S::Q / 4096;
  const WeighArgs& a;
  const KvChunk& c;
  int kv_head, row_hi, wave, lane;
  unsigned off[COPIES], lse_off;                               // bytes from a block's first row
  __device__ __forceinline__ int piece(int i) const { return 64 * (wave * COPIES + i) + lane; }
  __device__ __forceinline__ void begin() {
#pragma unroll
    for (int i = 0; i < COPIES; ++i) {
      const int in = piece(i) / CH, slot = piece(i) % CH, t = token_of(a, (unsigned)in);
      off[i] = (unsigned)(t * a.q_token + (in - t * a.group) * a.q_head) * 2 + 16 * (slot ^ turn<S::BYTES>(in));
    }
    const int in = 16 * wave + (lane & 15), t = token_of(a, (unsigned)in);
    lse_off = 4 * (unsigned)(t * a.heads + in - t * a.group);
  }
  // asks for rows row0 .. + 63, into LDS at `to`: LOADS loads
  __device__ __forceinline__ void ask(int row0, unsigned char* to) {
    unsigned char* const dst = to + 1024 * wave * COPIES;
    if (a.even_blocks && row0 + kWeighRows <= row_hi) {
      const int t = token_of(a, (unsigned)row0);
      const scalar* const q = (const scalar*)a.q + (long long)(c.start + t) * a.q_token + (long long)kv_head * a.group * a.q_head;
      const float* const lse = a.lse + (long long)(c.start + t) * a.heads + kv_head * a.group;
#pragma unroll
      for (int i = 0; i < COPIES; ++i) lds_dma16(q, off[i], dst + 1024 * i);
      if (lane < 16) lds_dma4(lse, lse_off, to + S::Q + 64 * wave);
      return;
    }
    // rows from row_hi on repeat the last
#pragma unroll
    for (int i = 0; i < COPIES; ++i) {
      const int in = piece(i) / CH, slot = piece(i) % CH, row = min(row0 + in, row_hi - 1), t = token_of(a, (unsigned)row);
      const scalar* const q = (const scalar*)a.q + (long long)(c.start + t) * a.q_token + (long long)(kv_head * a.group + row - t * a.group) * a.q_head;
      lds_dma16_each(q + 8 * (slot ^ turn<S::BYTES>(in)), dst + 1024 * i);
    }
    if (lane < 16) {
      const int row = min(row0 + 16 * wave + lane, row_hi - 1), t = token_of(a, (unsigned)row);
      lds_dma4_each(a.lse + (long long)(c.start + t) * a.heads + kv_head * a.group + row - t * a.group, to + S::Q + 64 * wave);
    }
  }
  // Once a wave's loads of a block are there: its lse as exponents of two.  A row that sees nothing gives nothing.
  __device__ __forceinline__ void finish(unsigned char* to) const {
    if (lane < 16) {
      float* const at = reinterpret_cast<float*>(to + S::Q) + 16 * wave + lane;
      const float x = *at;
      *at = x == -INFINITY ? INFINITY : x * 1.4426950408889634f;
    }
  }
};

// The weight of position `key` of a sequence, and what it has gathered before; NULL: it has none.
__device__ __forceinline__ float* weight_of(const WeighArgs& a, int page, int kv_head, int key, int len) {
  if (key >= len || page < 0 || page >= a.pages.pages) return nullptr;
  return a.weights + (((long long)page * a.pages.heads + kv_head) << a.pages.page_shift) + (key & ((1 << a.pages.page_shift) - 1));
}
__device__ __forceinline__ float gathered(const WeighArgs& a, const KvChunk& c, const float* at, int key) {
  return at && key < c.first && a.decay != 0.0f ? *at * a.decay : 0.0f;
}

// ---- few rows -----------------------------------------------------------------------

// At most 16 TILES rows to a sequence: they stay in LDS, and every wave walks blocks of 64 keys of its own.  A block's keys are asked for as soon as the products of the one in front
// have taken the registers' contents, its pages are looked up a block earlier, and there are few registers and so many waves: what is on its way at once
// is what counts.
template <typename T, KvFormat F, int D, int TILES>
__global__ __launch_bounds__(256, TILES == 1 ? (F == kSame && D > 64 ? 4 : 5) : TILES == 2 ? 3 : 2) void kv_weigh_few_kernel(WeighArgs a) {
  using S = WeighShape<D>;
  using Key = KeyRow<T, F, D, 4>;
  using v8 = typename T::v8;
  constexpr int KS = D / 32;
  __shared__ __attribute__((aligned(1024))) unsigned char q[S::BLOCK];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m = lane & 15, kg = lane >> 4;
  const int kv_head = blockIdx.x % a.pages.heads, rest = blockIdx.x / a.pages.heads;
  const int b = rest / a.tiles, part = rest - b * a.tiles;
  const KvChunk c = kv_chunk(a.batch, b);
  const int len = min(c.len, kv_capacity(a.batch, a.pages.page_shift)), shift = a.pages.page_shift;
  if (c.n == 0 || part * kBlock >= len) return;
  const int rows = min(c.n * a.group, 16 * TILES);
  const int* const table = a.batch.table + (long long)b * a.batch.width;
  const int blocks = (len - 1) / 64 + 1, step = 4 * a.tiles;
  auto look = [&](int block) __attribute__((always_inline)) { return table[min(64 * block + lane, len - 1) >> shift]; };
  Key keys[4];
  signed char exponent = 0;                                      // of the lane's own key
  float* at = nullptr;
  float before = 0.0f;
  auto ask = [&](int block, int page, bool read) __attribute__((always_inline)) {
    const int key = 64 * block + lane;
    if (read) {
#pragma unroll
      for (int nb = 0; nb < 4; ++nb) {
        const int first = min(64 * block + 16 * nb, (len - 1) & ~15);    // blocks of 16 behind the last repeat it, keys behind the last that one
        const int p = min(max(__builtin_amdgcn_readlane(page, 16 * nb), 0), a.pages.pages - 1);
        keys[nb].load(a, (((long long)p * a.pages.heads + kv_head) << shift) + (first & ((1 << shift) - 1)) + min(m, len - 1 - first), kg);
      }
      if constexpr (F != kSame) {
        const int k = min(key, len - 1), p = min(max(page, 0), a.pages.pages - 1);
        exponent = a.pages.k_exps[(((long long)p * a.pages.heads + kv_head) << shift) + (k & ((1 << shift) - 1))];
      }
    }
    at = weight_of(a, page, kv_head, key, len);
    before = gathered(a, c, at, key);
  };
  // under a window, positions in front of all that is seen are left alone, or only decay
  const int seen = a.window > 0 ? (int)(min(max((long long)c.first - a.window + 1, 0LL), (long long)len) / 64) : 0;
  int block = min((a.decay == 1.0f ? seen : 0) + 4 * part + wave, blocks);   // blocks: this wave has none
  int page = look(block);
  RowStage<T, D> stage{a, c, kv_head, rows, wave, lane};
  stage.begin();
  if (16 * wave < rows) stage.ask(0, q);
  if (block < blocks) ask(block, page, block >= seen);
  page = look(min(block + step, blocks));
  __builtin_amdgcn_s_waitcnt(0x0F70);                            // vmcnt(0): the rows
  if (16 * wave < rows) stage.finish(q);
  __syncthreads();
  for (; block < blocks; block += step) {
    const int key0 = 64 * block, next = block + step;
    const bool read = block >= seen;
    v4f sc[TILES][4];
    float factor[4];
    if (read) {
#pragma unroll
      for (int nb = 0; nb < 4; ++nb) factor[nb] = F == kSame ? a.scale_log2e : ldexpf(a.scale_log2e, __shfl((int)exponent, 16 * nb + m));
#pragma unroll
      for (int t = 0; t < TILES; ++t)
#pragma unroll
        for (int nb = 0; nb < 4; ++nb) sc[t][nb] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        v8 kf[4];
#pragma unroll
        for (int nb = 0; nb < 4; ++nb) kf[nb] = keys[nb].fragment(s);
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
          const v8 qf = *reinterpret_cast<const v8*>(q + (16 * t + m) * S::BYTES + 16 * (Key::chunk(s, kg) ^ turn<S::BYTES>(16 * t + m)));
#pragma unroll
          for (int nb = 0; nb < 4; ++nb) sc[t][nb] = T::mma16(qf, kf[nb], sc[t][nb]);
        }
      }
    }
    float* const here = at;
    const float old = before;
    __builtin_amdgcn_sched_barrier(0);
    if (next < blocks) {
      ask(next, page, next >= seen);
      page = look(min(next + step, blocks));
    }
    __builtin_amdgcn_sched_barrier(0);
    float mine = 0.0f;
    if (read) {
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        const v4f lse = *reinterpret_cast<const v4f*>(q + S::Q + 4 * (16 * t + 4 * kg));
#pragma unroll
        for (int nb = 0; nb < 4; ++nb) {
          const int from = first_row(a, c, key0 + 16 * nb + m), to = min(end_row(a, c, key0 + 16 * nb + m), rows);   // the rows that see a lane's key
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int of = 16 * t + 4 * kg + r;
            const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][nb][r], factor[nb], -lse[r]));
            acc[nb] += of >= from && of < to ? w : 0.0f;
          }
        }
      }
      // the four lanes of a key meet; lane 16 nb + m takes key m of block nb
#pragma unroll
      for (int nb = 0; nb < 4; ++nb) {
        float x = acc[nb];
        x += __shfl_xor(x, 16);
        x += __shfl_xor(x, 32);
        if (kg == nb) mine = x;
      }
    }
    if (here) *here = old + finite_or_nan(mine);
  }
}

// ---- many rows ----------------------------------------------------------------------

// A block of a sequence's keys, from key0 on: the rows [lo, hi) that see some of it.
struct BlockRows {
  int lo, hi;
};
__device__ __forceinline__ BlockRows rows_that_see(const WeighArgs& a, const KvChunk& c, int key0, int end) {
  return {first_row(a, c, key0), end_row(a, c, end - 1)};
}

// How many parts the rows of a sequence are cut into: part p has rows p part_rows .. + part_rows - 1, the last all that are left.
__device__ __forceinline__ int parts_of(const WeighArgs& a, const KvChunk& c, int len) {
  return a.parts == 1 || len > a.tiles * kBlock ? 1 : min((c.n * a.group + a.part_rows - 1) / a.part_rows, a.parts);
}
__device__ __forceinline__ BlockRows rows_of_part(const WeighArgs& a, BlockRows r, int part, int parts) {
  return {part == 0 ? r.lo : max(r.lo, part * a.part_rows), part == parts - 1 ? r.hi : min(r.hi, (part + 1) * a.part_rows)};
}

template <typename T, KvFormat F, int D>
__global__ __launch_bounds__(256, 2) void kv_weigh_kernel(WeighArgs a) {
  using S = WeighShape<D>;
  using Key = KeyRow<T, F, D, 2>;
  using v8 = typename T::v8;
  constexpr int KS = D / 16, KEYS = 64;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  constexpr auto vmcnt = [](int n) { return 0x0F70 | (n & 15) | ((n >> 4) << 14); };

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m = lane & 31, kg = lane >> 5;
  // the head goes fastest, the block of keys slowest: under a causal mask the first blocks are seen by most rows, and go out first
  const int kv_head = blockIdx.x % a.pages.heads;
  int rest = blockIdx.x / a.pages.heads;
  const int b = rest % a.batch.sequences;
  rest /= a.batch.sequences;
  const int part = rest % a.parts, tile0 = rest / a.parts;
  const KvChunk c = kv_chunk(a.batch, b);
  const int len = min(c.len, kv_capacity(a.batch, a.pages.page_shift)), parts = parts_of(a, c, len), shift = a.pages.page_shift;
  if (c.n == 0 || part >= parts) return;

  for (int block0 = tile0 * kBlock; block0 < len; block0 = (int)min((long long)block0 + (long long)a.tiles * kBlock, (long long)INT_MAX)) {
    const int key0 = block0 + wave * KEYS;
    const BlockRows rows = rows_of_part(a, rows_that_see(a, c, block0, min(block0 + kBlock, len)), part, parts);
    const int row_lo = rows.lo, row_hi = rows.hi;
    if (row_lo >= row_hi && (parts > 1 || a.decay == 1.0f)) continue;

    // ---- this wave's keys, and the rows that see a lane's
    v8 kf[2][KS];
    float factor[2], acc[2];
    int from[2], to[2];
    if (row_lo < row_hi) {
#pragma unroll
      for (int nb = 0; nb < 2; ++nb) {
        long long base[2];                                     // of two blocks of 16, each in one page; those behind the last repeat it, keys behind the last that one
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int first = min(key0 + 32 * nb + 16 * h, (len - 1) & ~15);
          base[h] = (((long long)kv_page(a.batch, b, first >> shift, a.pages.pages) * a.pages.heads + kv_head) << shift) + (first & ((1 << shift) - 1)) +
                    min(m & 15, len - 1 - first);
        }
        Key key;
        const long long row = m & 16 ? base[1] : base[0];
        key.load(a, row, kg);
#pragma unroll
        for (int s = 0; s < KS; ++s) kf[nb][s] = key.fragment(s);
        factor[nb] = F == kSame ? a.scale_log2e : ldexpf(a.scale_log2e, a.pages.k_exps[row]);
        from[nb] = first_row(a, c, key0 + 32 * nb + m);
        to[nb] = min(end_row(a, c, key0 + 32 * nb + m), row_hi);
      }
    }
    acc[0] = acc[1] = 0.0f;
    // [all_lo, all_hi): the rows that see each of this wave's keys; [some_lo, some_hi): some of them
    const int last = min(key0 + KEYS, len) - 1, all_hi = min(end_row(a, c, key0), row_hi), some_hi = end_row(a, c, last);
    const int all_lo = key0 >= len ? INT_MAX : first_row(a, c, last), some_lo = key0 >= len ? INT_MAX : first_row(a, c, key0);
    // where the sums go, and what has been gathered before: lane i has key key0 + i
    const int key = key0 + lane;
    float* const at = key >= len ? nullptr
                      : parts > 1 ? a.sums + (((long long)b * a.pages.heads + kv_head) * a.parts + part) * (a.tiles * (long long)kBlock) + key
                                  : weight_of(a, a.batch.table[(long long)b * a.batch.width + (key >> shift)], kv_head, key, len);
    float before = parts > 1 ? 0.0f : gathered(a, c, at, key);

    // ---- rows, 64 at a time, 32 to a product: 0 and 1
    v16f sc[2][2];                                             // [rows][keys]
    v4f l[2][4];
    const int at_m = m * S::BYTES, chunk_m = turn<S::BYTES>(m);   // (32 rows on, both are the same but for the row's offset)
    auto products = [&](const unsigned char* q, auto i_c) __attribute__((always_inline)) {
      constexpr int i = decltype(i_c)::value;
#pragma unroll
      for (int g = 0; g < 4; ++g) l[i][g] = *reinterpret_cast<const v4f*>(q + S::Q + 4 * (32 * i + 8 * g + 4 * kg));
#pragma unroll
      for (int nb = 0; nb < 2; ++nb)
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[i][nb][e] = 0.0f;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const v8 qf = *reinterpret_cast<const v8*>(q + 32 * i * S::BYTES + at_m + 16 * (Key::chunk(s, kg) ^ chunk_m));
#pragma unroll
        for (int nb = 0; nb < 2; ++nb) sc[i][nb] = T::mma32(qf, kf[nb][s], sc[i][nb]);
      }
    };
    auto weights = [&](auto i_c) __attribute__((always_inline)) {
      constexpr int i = decltype(i_c)::value;
#pragma unroll
      for (int nb = 0; nb < 2; ++nb)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[nb] += __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i][nb][e], factor[nb], -l[i][e >> 2][e & 3]));
    };
    auto masked_weights = [&](int row0, auto i_c) __attribute__((always_inline)) {
      constexpr int i = decltype(i_c)::value;
#pragma unroll
      for (int nb = 0; nb < 2; ++nb)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int row = row0 + 32 * i + 8 * (e >> 2) + 4 * kg + (e & 3);
          const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i][nb][e], factor[nb], -l[i][e >> 2][e & 3]));
          acc[nb] += row >= from[nb] && row < to[nb] ? w : 0.0f;
        }
    };
    // Products of rows i of a block beside the weights of the others of before: after each product the reads of the one AHEAD steps on and two weights' vector
    // instructions, in this order, which keeps both pipes fed; early holds the first AHEAD fragments, and at the end those of the rows behind.
    constexpr int AHEAD = KS < 4 ? KS : 4;
    v8 early[AHEAD];
    auto fragment = [&](const unsigned char* q, int i, int s) __attribute__((always_inline)) {
      return *reinterpret_cast<const v8*>(q + 32 * i * S::BYTES + at_m + 16 * (Key::chunk(s, kg) ^ chunk_m));
    };
    auto phase = [&](const unsigned char* q, auto i_c, auto weights_c) __attribute__((always_inline)) {
      constexpr int i = decltype(i_c)::value, STEPS = 2 * KS, EACH = (32 + STEPS - 1) / STEPS;
      v8 f[KS];
      float y[32];
      static_for<AHEAD>([&](auto n_c) __attribute__((always_inline)) { f[decltype(n_c)::value] = early[decltype(n_c)::value]; });
      __builtin_amdgcn_sched_barrier(0);
      static_for<STEPS>([&](auto n_c) __attribute__((always_inline)) {
        constexpr int n = decltype(n_c)::value, s = n / 2, nb = n % 2;
        v16f zero;
#pragma unroll
        for (int e = 0; e < 16; ++e) zero[e] = 0.0f;
        sc[i][nb] = T::mma32(f[s], kf[nb][s], s == 0 ? zero : sc[i][nb]);
        if constexpr (nb == 0 && s + AHEAD < KS) f[s + AHEAD] = fragment(q, i, s + AHEAD);
        if constexpr (nb == 0 && s + AHEAD >= KS && i == 0) early[s + AHEAD - KS] = fragment(q, 1, s + AHEAD - KS);
        if constexpr (nb == 1 && s < 4) l[i][s] = *reinterpret_cast<const v4f*>(q + S::Q + 4 * (32 * i + 8 * s + 4 * kg));
        if constexpr (KS < 4 && n == STEPS - 1) {
#pragma unroll
          for (int g = KS; g < 4; ++g) l[i][g] = *reinterpret_cast<const v4f*>(q + S::Q + 4 * (32 * i + 8 * g + 4 * kg));
        }
        if constexpr (decltype(weights_c)::value) {
#pragma unroll
          for (int w = 0; w < EACH; ++w) {
            const int k = EACH * n + w;
            if (k < 32) y[k] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[1 - i][k / 16][k % 16], factor[k / 16], -l[1 - i][k % 16 >> 2][k % 4]));
            const int done = k - EACH;
            if (done >= 0 && done < 32) acc[done / 16] += y[done];
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      });
      if constexpr (decltype(weights_c)::value) {
#pragma unroll
        for (int k = EACH * (STEPS - 1); k < 32; ++k) acc[k / 16] += y[k];
      }
    };
    auto begin = [&](const unsigned char* q) __attribute__((always_inline)) {
#pragma unroll
      for (int s = 0; s < AHEAD; ++s) early[s] = fragment(q, 0, s);
    };
    using yes = std::true_type;
    using no = std::false_type;
    using first = std::integral_constant<int, 0>;
    using second = std::integral_constant<int, 1>;
    if (row_lo < row_hi) {
      // Blocks of rows are asked for three ahead, into the place of the one before this, whose reads the barrier ends; their lse are finished one ahead.
      RowStage<T, D> stage{a, c, kv_head, row_hi, wave, lane};
      stage.begin();
#pragma unroll
      for (int i = 0; i < S::BLOCKS - 1; ++i)
        if (row_lo + i * kWeighRows < row_hi) stage.ask(row_lo + i * kWeighRows, smem + i * S::BLOCK);
      // the keys are there before the loop, which would otherwise wait for all that is on its way wherever they are used
#pragma unroll
      for (int nb = 0; nb < 2; ++nb) {
#pragma unroll
        for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(kf[nb][s]));
        asm volatile("" : "+v"(factor[nb]));
      }
      asm volatile("" : "+v"(before));
      __builtin_amdgcn_s_waitcnt(vmcnt(0));
      stage.finish(smem);
      int r0 = row_lo, at_block = 0;
      // the block of rows r0: there once this has been called
      auto arrive = [&]() __attribute__((always_inline)) {
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (r0 + 3 * kWeighRows < row_hi) {
          stage.ask(r0 + 3 * kWeighRows, smem + ((at_block + 3) & (S::BLOCKS - 1)) * S::BLOCK);
          __builtin_amdgcn_s_waitcnt(vmcnt(2 * S::LOADS));
        } else {
          __builtin_amdgcn_s_waitcnt(vmcnt(0));
        }
        asm volatile("" ::: "memory");
        if (r0 + kWeighRows < row_hi) stage.finish(smem + ((at_block + 1) & (S::BLOCKS - 1)) * S::BLOCK);
        return (const unsigned char*)smem + at_block * S::BLOCK;
      };
      auto on = [&]() __attribute__((always_inline)) {
        r0 += kWeighRows;
        at_block = (at_block + 1) & (S::BLOCKS - 1);
      };
      while (r0 < row_hi) {
        const unsigned char* q = arrive();
        if (r0 >= all_lo && r0 <= all_hi - kWeighRows) {
          // All rows see all keys, for as long as that is so: products go beside the weights of the 32 rows in front of them.
          begin(q);
          phase(q, first{}, no{});
          phase(q, second{}, yes{});
          for (on(); r0 <= all_hi - kWeighRows; on()) {
            q = arrive();
            begin(q);
            phase(q, first{}, yes{});
            phase(q, second{}, yes{});
          }
          weights(second{});
        } else {
          if (r0 > some_lo - kWeighRows && r0 < some_hi) {
            products(q, first{});
            masked_weights(r0, first{});
            products(q, second{});
            masked_weights(r0, second{});
          }
          on();
        }
      }
      __syncthreads();                                         // (the next keys' rows go where these lie)
    }
    // the two lanes of a key meet; lane 32 nb + m takes key m of block nb
    const float x = acc[0] + __shfl_xor(acc[0], 32), y = acc[1] + __shfl_xor(acc[1], 32);
    const float mine = kg ? y : x;
    if (at) *at = before + (parts > 1 ? mine : finite_or_nan(mine));
  }
}

// The parts' sums of a key, one behind the other.
__global__ __launch_bounds__(kBlock) void kv_weigh_join_kernel(WeighArgs a) {
  const int kv_head = blockIdx.x % a.pages.heads, rest = blockIdx.x / a.pages.heads;
  const int b = rest % a.batch.sequences, block0 = rest / a.batch.sequences * kBlock, key = block0 + threadIdx.x;
  const KvChunk c = kv_chunk(a.batch, b);
  const int len = min(c.len, kv_capacity(a.batch, a.pages.page_shift)), parts = parts_of(a, c, len);
  if (c.n == 0 || parts == 1 || key >= len) return;
  float* const at = weight_of(a, a.batch.table[(long long)b * a.batch.width + (key >> a.pages.page_shift)], kv_head, key, len);
  const BlockRows all = rows_that_see(a, c, block0, min(block0 + kBlock, len));
  const float* const from = a.sums + ((long long)b * a.pages.heads + kv_head) * a.parts * (a.tiles * (long long)kBlock) + key;
  float sum = 0.0f;
#pragma unroll 8
  for (int p = 0; p < parts; ++p) {
    const BlockRows r = rows_of_part(a, all, p, parts);
    if (r.lo < r.hi) sum += from[(long long)p * a.tiles * kBlock];
  }
  if (at) *at = gathered(a, c, at, key) + finite_or_nan(sum);
}

// Rows in parts of 2048, or of fewer while there are less than four workgroups to a compute unit; the results are joined by a second launch.  (A workgroup needs 3 to 4 us
// before its first product: a prompt of 4096 tokens, 16 heads of 128: 71 us in parts of 2048, 68 in 1024 or 512; four such prompts 168, 185 and 213; one of 2048 tokens, 8 heads
// on one of keys: 82, 48 and 34.  Workgroups are counted from the sizes that the call could have, among them those of sequences that pause and of blocks behind shorter ones' ends.)
struct RowCut {
  int parts, rows;
};
static RowCut cut_rows(long long pairs, long long most, long long most_rows, int cus, size_t room) {
  const long long tiles = std::max(1LL, (most + kBlock - 1) / kBlock);
  long long rows = 2048;
  while (rows > 512 && pairs * tiles * ((most_rows + rows - 1) / rows) < 4 * cus) rows /= 2;
  const long long parts = (most_rows + rows - 1) / rows;
  if (parts <= 1 || pairs * tiles * parts > INT_MAX / 2 || (size_t)(pairs * tiles * parts * kBlock) > room / sizeof(float)) return {1, INT_MAX};
  return {(int)parts, (int)rows};
}

}  // namespace ftk

extern "C" {

size_t ftk_kv_cache_weigh_workspace_bytes(const ftk_kv_pages* pages, const ftk_kv_batch* batch, int heads, int max_queries, int max_keys) {
  using namespace ftk;
  const DeviceProps* d = nullptr;
  if (!pages || !batch || pages->heads <= 0 || heads <= 0 || heads % pages->heads || batch->tokens <= 0 || batch->sequences <= 0 || batch->table_width <= 0 ||
      pages->page_size <= 0 || device_props(&d))
    return 0;
  const long long capacity = std::min<long long>((long long)batch->table_width * pages->page_size, INT_MAX);
  const long long most = max_keys > 0 ? std::min<long long>(max_keys, capacity) : capacity, pairs = (long long)batch->sequences * pages->heads;
  const long long rows = (long long)(max_queries > 0 ? std::min(max_queries, batch->tokens) : batch->tokens) * (heads / pages->heads);
  if (rows <= kWeighRows) return 0;
  const RowCut cut = cut_rows(pairs, most, rows, d->cus, SIZE_MAX);
  return cut.parts > 1 ? (size_t)(pairs * cut.parts * ((most + kBlock - 1) / kBlock) * kBlock) * sizeof(float) : 0;
}

int ftk_kv_cache_weigh(const void* q, int type, long long q_token_stride, long long q_head_stride, const float* lse, const ftk_kv_pages* pages, float* weights,
                       const ftk_kv_batch* batch, int heads, float scale, float decay, int causal, int window, int max_queries, int max_keys,
                       void* workspace, size_t workspace_bytes, ftk_stream_t stream) {
  using namespace ftk;
  const char* who = "ftk_kv_cache_weigh";
  WeighArgs a;
  ftk_kv_pages keys = pages ? *pages : ftk_kv_pages{};
  keys.v = keys.k;
  keys.v_exps = keys.k_exps;
  int rc = check_kv_pages(who, pages ? &keys : nullptr, &a.pages);
  if (rc || (rc = check_kv_batch(who, batch, &a.batch))) return rc;
  if (heads <= 0 || heads % pages->heads) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: query heads must be a multiple of the kv heads, got %d and %d", who, heads, pages->heads);
  if (type != FTK_F16 && type != FTK_BF16) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: queries must be fp16 or bf16", who);
  if ((pages->type == FTK_F16 || pages->type == FTK_BF16) && pages->type != type) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: pages of 16 bits must have the type of the queries", who);
  if (!(scale > 0.0f) || !(scale * 1.4426950408889634f <= FLT_MAX)) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: scale must be positive, and its product with log2(e) finite", who);
  if (!(decay >= 0.0f) || !(decay <= 1.0f)) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: decay must be from 0 to 1", who);
  if (window < 0 || max_queries < 0 || max_keys < 0) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: window, max_queries and max_keys must not be negative", who);
  if (a.batch.tokens == 0) return FTK_OK;
  if (!q || !lse || !weights || !aligned16(q)) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: q, lse and weights must be non-NULL and q 16-byte aligned", who);
  if (((uintptr_t)lse | (uintptr_t)weights) & 3) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: lse and weights must be 4-byte aligned", who);
  if (q_token_stride < 0 || q_head_stride < 0 || q_token_stride % 8 || q_head_stride % 8) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: strides must be multiples of 8 elements", who);
  if (workspace && !aligned16(workspace)) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: the workspace must be 16-byte aligned", who);
  a.group = heads / pages->heads;
  // rows are numbered in 31 bits, and rows / group is a product with the inverse, exact below 2^32 / group
  if ((long long)a.batch.tokens * a.group > INT_MAX / 2 || (long long)a.batch.tokens * a.group >= (1LL << 32) / a.group) return fail(FTK_ERR_UNSUPPORTED_SHAPE, "%s: too many rows", who);
  const DeviceProps* d = nullptr;
  if ((rc = device_props(&d))) return rc;
  a.q = q;
  a.lse = lse;
  a.q_token = q_token_stride;
  a.q_head = q_head_stride;
  a.weights = weights;
  a.heads = heads;
  a.inverse = a.group == 1 ? 0u : (unsigned)(((1ULL << 32) + a.group - 1) / a.group);
  a.scale_log2e = scale * 1.4426950408889634f;
  a.decay = decay;
  a.causal = causal != 0;
  a.window = window;
  a.even_blocks = 64 % a.group == 0 && (64 / a.group) * (double)q_token_stride + (double)heads * q_head_stride < (1 << 30) && 64LL * heads < (1 << 29);
  a.parts = 1;
  a.part_rows = INT_MAX;
  a.sums = nullptr;
  const long long capacity = std::min<long long>((long long)a.batch.width << a.pages.page_shift, INT_MAX);
  const long long most = max_keys > 0 ? std::min<long long>(max_keys, capacity) : capacity;
  const long long pairs = (long long)a.batch.sequences * pages->heads;
  const long long most_rows = (long long)(max_queries > 0 ? std::min(max_queries, a.batch.tokens) : a.batch.tokens) * a.group;
  return with_kv_types(type, pages->type, pages->head_size, [&](auto t, auto f, auto dc) -> int {
    using T = decltype(t);
    constexpr KvFormat F = decltype(f)::value;
    constexpr int D = decltype(dc)::value;
    if (pairs > INT_MAX / 2) return fail(FTK_ERR_UNSUPPORTED_SHAPE, "%s: too many sequences", who);
    // (a workgroup takes every a.tiles-th block; with more than one part they are all there)
    const auto launch = [&](const char* name, auto kernel, long long tiles, int parts, int lds) -> int {
      a.tiles = (int)std::min(std::max(1LL, tiles), (INT_MAX / 2) / pairs);
      hipLaunchKernelGGL(kernel, dim3((unsigned)(a.tiles * pairs * parts)), dim3(256), lds, (hipStream_t)stream, a);
      return check_launch(name);
    };
    if (most_rows <= kWeighRows) {
      // four blocks of 64 keys to a wave (2 to 16: all within 8 % for 64 sequences of up to 8192 keys), or fewer while there are less than four workgroups to a compute unit
      const long long blocks = (most + kBlock - 1) / kBlock;     // of a workgroup
      const long long tiles = std::max(std::min(blocks, (4LL * d->cus + pairs - 1) / pairs), (blocks + 3) / 4);
      const auto few = [&](auto n) { return launch("kv_weigh_few_kernel", kv_weigh_few_kernel<T, F, D, decltype(n)::value>, tiles, 1, 0); };
      if (most_rows <= 16) return few(std::integral_constant<int, 1>{});
      return most_rows <= 32 ? few(std::integral_constant<int, 2>{}) : few(std::integral_constant<int, 4>{});
    }
    const RowCut cut = cut_rows(pairs, most, most_rows, d->cus, workspace ? workspace_bytes : 0);
    a.parts = cut.parts;
    a.part_rows = cut.rows;
    a.sums = (float*)workspace;
    static DeviceOnce once;
    unsigned bit;
    if (once.pending(&bit)) {
      FTK_HIP(hipFuncSetAttribute((const void*)kv_weigh_kernel<T, F, D>, hipFuncAttributeMaxDynamicSharedMemorySize, WeighShape<D>::LDS));
      once.done(bit);
    }
    const int bad = launch("kv_weigh_kernel", kv_weigh_kernel<T, F, D>, (most + kBlock - 1) / kBlock, a.parts, WeighShape<D>::LDS);
    if (bad || a.parts == 1) return bad;
    hipLaunchKernelGGL(kv_weigh_join_kernel, dim3((unsigned)(a.tiles * pairs)), dim3(kBlock), 0, (hipStream_t)stream, a);
    return check_launch("kv_weigh_join_kernel");
  });
}

}  // extern "C"
