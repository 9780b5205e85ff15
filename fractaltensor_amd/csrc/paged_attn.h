// Attention of the new tokens of a batch of sequences over a paged cache of keys and values, grouped heads included.
//
// The G = query heads / kv heads query heads that share a kv head, times the new tokens of a sequence, are the ROWS of one
// product with that head's keys: row r is token r / G, head r % G.  Two kernels by the number of rows:
//
//   narrow  (at most 64 rows: decoding, drafts): bound by reading the cache once.  A workgroup has 16 NQ rows, 16 or 32; its four waves cut the
//           KEYS, each walking every fourth 32-key tile from copies straight into its own LDS, with no barrier in the loop.  The two
//           to four workgroups of more rows run next to one another, and all but one find what they read in the caches.
//   wide    (chunks and prompts): bound by the matrix pipe.  A wave has 32 rows, and the eight waves of a workgroup share 64-key tiles.
//
// Products are transposed in both, so that a lane has one row: S^T = K Q^T, O^T = V^T P^T with P as it comes out of the
// first product (the contraction takes the keys in the order a lane holds them).  Long sequences are cut into parts of
// `part_keys` keys, a workgroup each, which leave (reference, sum, unnormalised O) for a second launch to join.
//
// Rounding: scores, softmax state and O are fp32 and Q is not scaled beforehand.  Weights enter P V in 16 bits.  In the narrow form, which leaves the matrix unit
// time for a second product, a weight is the rounded one and what that leaves, also in 16 bits (2^-22 of it fp16, 2^-16 bf16), so that a result is off by its own rounding
// alone, whatever else the call holds.  In the wide form, bound by the matrix pipe, of which a second product would take half as much again, it is the rounded one
// alone, half a step (2^-11 of it fp16, 2^-8 bf16), which with the result's own rounding makes sqrt(2) of the error of that alone in the mean.  A cache of 8
// bits enters the products as its exact values, which fp16 rows and bf16 rows have in their own type; with queries in fp16, those of bf16 rows that fp16 does not
// have are rounded to it, tile by tile on a way of its own.
//
// TREE: the new tokens of a sequence are a tree of drafts.  Each sees the cache in front of them, its ancestors and itself, so that only the tiles that hold new tokens'
// own keys differ: there a row has a bit for each of those keys, found by walking up from it through the parents, a lane a row, which are passed from lane to
// lane.  (Position and depth differ in a tree; a window counts the steps on the way.)  The narrow form has up to 16 rows of them, and the wide form
// more: up to 128 rows by both halves of a workgroup, on different keys, and the work of sequences of different lengths shared
// out evenly.  Sequences of up to 64 rows have their weights as two operands on either, by their own rows alone, so that a tree's results are no less exact than those of the same tokens
// one behind the other, nor for a larger tree beside it; the wide form has a second body for them.  (16 sequences of 2064 to 8192 positions in e4m3, 8 heads of keys, 64 rows: 89 us, 74 with
// weights rounded once, 92 by the narrow form; 16 bits 87, 86 and 107.)
#pragma once

#include <float.h>

#include <algorithm>
#include <cmath>

#include "kv_common.h"
#include "tree_shares.h"

namespace ftk {

constexpr int kWaves = 4;
constexpr float kNoRef = -3.402823466e38f;   // the reference before any score: finite, so that -inf minus it is -inf
constexpr int kSmallRows = 16;                // sequences of at most so many rows, beside larger ones, are small
constexpr int kNarrowRows = 64;               // calls of no more rows to a sequence are narrow (trees: have weights as narrow ones do)
constexpr int kTreeMost = 256;                // new tokens of a tree

// Weights are 2^(score - reference), and the reference is moved to the largest score less kLift, so that the largest weight is 2^kLift then.  fp16 has 15
// binades above 1 and no more below it than down to 2^-24: with weights of at most 1, those of many keys beside one that outweighs them (a sink,
// whose value may be zero) were subnormal, or zero, while their sum counted them.  (4096 keys in fp16, one of a score 20 above the others' with a value
// of zero: all of the result was lost.)  With nine binades a weight is off by at most 2^-34 of the largest besides its own rounding, which the result's own
// finest step hides.  bf16 has the range of fp32.
template <typename T>
constexpr float kLift = std::is_same<T, Half>::value ? 9.0f : 0.0f;
template <typename T>
constexpr float kSlack = std::is_same<T, Half>::value ? 6.0f : 8.0f;   // narrow: the reference moves when a weight would be above 2^(kLift + kSlack)

// How the keys of a sequence are cut: at most nparts parts of part_keys keys, the last of which takes what is left.
struct Cut {
  int nparts, part_keys;
};

struct AttnArgs {
  const void* q;
  void* o;
  float* lse;                                 // may be NULL
  long long q_token, q_head;                  // strides, elements
  KvPages pages;
  KvBatch batch;
  int heads, group;                           // query heads, query heads of a kv head
  float scale_log2e;
  int causal, window;
  int slots, slots_per_seq;                   // blocks of rows, and those of a sequence (0: they are numbered over the packed rows)
  Cut cut, small;                             // `small` for sequences of at most small_rows rows
  int small_rows;
  long long small_first;                      // parts of small sequences stand behind these many
  float *part_o, *part_ml;                    // [tokens * heads][cut.nparts] parts, then [sequences][kv heads][kSmallRows][small.nparts]: D floats; two
  const int* parents;                         // trees: of each packed row, by its number among the sequence's new tokens; negative: none
  int shares, grain_shift, block_shift, row_blocks;  // trees, wide: workgroups of a kv head that the work is shared out to (0: a workgroup to a block of rows), of
                                              // grains of 2^grain_shift keys; blocks of 2^block_shift rows, as many as a sequence may have
};

// ---- which rows and which keys a workgroup has ----------------------------------------

struct Job {
  int b, start, n, first;      // the sequence, its first packed row, its new tokens, the position of the first
  int row0, rows;              // first row of this workgroup, rows of the sequence
  int len;                     // keys there are
  int lo, hi;                  // keys [lo, hi) that the rows of this workgroup and its part see
  int sure_lo, sure_hi;        // keys that each of its rows sees
  int part, parts;             // parts of this sequence
  bool small;
  long long left;              // trees, wide, parts > 1: where the first row's is left, in parts
};

// The keys that some row of the sequence sees begin here (a multiple of 64).
__device__ __forceinline__ int seq_first_key(const AttnArgs& a, int first) {
  return a.window > 0 ? (int)max(0LL, (long long)first - a.window + 1) & ~63 : 0;
}
__device__ __forceinline__ int seq_parts(const AttnArgs& a, const Cut& cut, int first, int len) {
  if (cut.nparts == 1) return 1;
  const int keys = max(0, len - seq_first_key(a, first));
  return min(max((int)(((long long)keys + cut.part_keys - 1) / cut.part_keys), 1), cut.nparts);
}
__device__ __forceinline__ int clamp_position(long long x, int len) { return (int)(x < 0 ? 0 : x > len ? len : x); }

// The sequence and the block of R of its rows that a slot stands for; false: none.
template <int R>
__device__ __forceinline__ bool find_rows(const AttnArgs& a, int slot, int* b, int* tile) {
  if (a.slots_per_seq > 0) {
    // Row blocks go out in three passes over the sequences, the last third of every sequence's first: the blocks of a sequence share
    // its keys in the caches, and a launch ends with blocks that see few keys under a causal mask.  (Four prompts of up to 4096 tokens: 177 us, 183 in
    // one pass, 218 with the last block of every sequence first.)
    int left = a.slots_per_seq, r = slot;
    for (int pass = 3;; --pass) {
      const int take = (left + pass - 1) / pass;
      if (pass == 1 || r < take * a.batch.sequences) {
        *b = min(r / max(take, 1), a.batch.sequences - 1);
        *tile = left - 1 - (r - *b * take);
        return *tile >= 0;
      }
      r -= take * a.batch.sequences;
      left -= take;
    }
  }
  // sequence b has the slots from starts[b] * G / R + b on, at least as many as it needs; the last go out first
  const int from_end = a.slots - 1 - slot;
  const auto first_slot = [&](int i) { return (long long)min(max(a.batch.starts[i], 0), a.batch.tokens) * a.group / R + i; };
  *b = __builtin_amdgcn_readfirstlane(max(count_at_most(a.batch.sequences, from_end, first_slot) - 1, 0));
  const long long t = from_end - first_slot(*b);
  *tile = __builtin_amdgcn_readfirstlane((int)t);
  return t >= 0;
}

// False: there is nothing to do.  small: the sequence is one of at most small_rows rows, or is not meant.
template <int R, bool TREE>
__device__ __forceinline__ bool find_job(const AttnArgs& a, int b, int tile, int part, bool small, Job& j) {
  j.b = b;
  const KvChunk c = kv_chunk(a.batch, b);
  j.start = c.start;
  j.n = TREE ? min(c.n, kTreeMost) : c.n;
  j.first = c.first;
  j.rows = j.n * a.group;
  j.row0 = tile * R;
  if (tile >= (j.rows + R - 1) / R || (j.rows <= a.small_rows) != small) return false;
  j.len = min(c.len, kv_capacity(a.batch, a.pages.page_shift));
  const int t_lo = j.row0 / a.group, t_hi = (min(j.row0 + R, j.rows) - 1) / a.group;
  // (in a tree a token may see no other new one, and be no deeper than the root or as deep as its number)
  const long long p_lo = (long long)c.first + (TREE ? 0 : t_lo), p_hi = (long long)c.first + t_hi;
  j.hi = TREE || a.causal ? clamp_position(p_hi + 1, j.len) : j.len;
  j.sure_hi = TREE ? clamp_position(c.first, j.len) : a.causal ? clamp_position(p_lo + 1, j.len) : j.len;
  j.lo = a.window > 0 ? clamp_position(p_lo - a.window + 1, j.len) : 0;
  j.sure_lo = a.window > 0 ? clamp_position(p_hi - a.window + 1, j.len) : 0;
  j.part = part;
  j.small = small;
  const Cut cut = small ? a.small : a.cut;
  j.parts = seq_parts(a, cut, c.first, j.len);
  if (part >= j.parts) return false;
  if (j.parts > 1) {
    const long long from = (long long)seq_first_key(a, c.first) + (long long)part * cut.part_keys;
    j.lo = max(j.lo, clamp_position(from, j.len));
    if (part < j.parts - 1) j.hi = min(j.hi, clamp_position(from + cut.part_keys, j.len));
  }
  return true;
}

// The first part of a row among all parts; at: its place among the packed rows times heads.
__device__ __forceinline__ long long first_part(const AttnArgs& a, bool small, int b, int kv_head, int row, long long at) {
  return small ? a.small_first + (((long long)b * a.pages.heads + kv_head) * kSmallRows + row) * a.small.nparts : at * a.cut.nparts;
}

// The keys [lo, hi) that a row sees, and its place among the packed rows times heads.  In a tree lo is that of the root, until the row's depth is known, and
// loose says that the row's own key has no room in the table, so that it may see nothing all the same.
struct Row {
  int lo, hi;
  long long at;
  bool loose;
};
template <bool TREE>
__device__ __forceinline__ Row row_of(const AttnArgs& a, const Job& j, int kv_head, int row) {
  const int t = row / a.group, g = row - t * a.group;
  const long long p = (long long)j.first + t;
  Row r;
  r.hi = TREE || a.causal ? clamp_position(p + 1, j.len) : j.len;
  r.lo = a.window > 0 ? clamp_position((TREE ? (long long)j.first : p) - a.window + 1, j.len) : 0;
  r.loose = TREE && p >= j.len;
  r.at = (long long)(j.start + t) * a.heads + kv_head * a.group + g;
  return r;
}

// The way from a new token up to its root, as a bit for each token on it that the window holds; `depth` of them lie above it.  WORDS 64-bit words, bit i + shift for token
// i.  All lanes of a wave call it, a token each.
template <int WORDS>
__device__ __forceinline__ void walk_up(const AttnArgs& a, const Job& j, int token, int shift, unsigned long long (&bits)[WORDS], int* depth) {
  constexpr int CHUNKS = WORDS == 1 ? 1 : kTreeMost / 64;
  const int lane = threadIdx.x & 63;
  int up[CHUNKS];                                              // a parent comes before its child, or is none
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int i = 64 * c + lane;
    up[c] = i < j.n ? a.parents[j.start + i] : -1;
    if (up[c] >= i) up[c] = -1;
  }
#pragma unroll
  for (int w = 0; w < WORDS; ++w) bits[w] = 0;
  int at = token, steps = 0;
  while (__builtin_amdgcn_ballot_w64(at >= 0) != 0) {          // (at falls with every step)
    if (at >= 0) {
      const int place = at + shift;
      if (a.window == 0 || steps < a.window) {
#pragma unroll
        for (int w = 0; w < WORDS; ++w)
          if (WORDS == 1 || place >> 6 == w) bits[w] |= 1ULL << (place & 63);
      }
      ++steps;
    }
    int next = __shfl(up[0], at & 63);
#pragma unroll
    for (int c = 1; c < CHUNKS; ++c) {
      if (64 * c >= j.n) break;
      const int x = __shfl(up[c], at & 63);
      if (at >> 6 == c) next = x;
    }
    at = at >= 0 ? next : -1;
  }
  *depth = steps - 1;
}

template <typename T>
__device__ __forceinline__ const typename T::scalar* query_of(const AttnArgs& a, const Job& j, int kv_head, int row) {
  const int t = row / a.group, g = row - t * a.group;
  return (const typename T::scalar*)a.q + (j.start + t) * a.q_token + (long long)(kv_head * a.group + g) * a.q_head;
}

// The same pointer, known to be that of every lane.
__device__ __forceinline__ const unsigned char* uniform(const unsigned char* p) {
  const unsigned long long x = (unsigned long long)p;
  const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)x), hi = __builtin_amdgcn_readfirstlane((unsigned)(x >> 32));
  return (const unsigned char*)(((unsigned long long)hi << 32) | lo);
}

// First cache row (of a kv head) of the block of 16 keys that begins at `key`, a multiple of 16, or 16 times that of the key nearest to it
// in [lo, hi) where the block lies outside: a block that holds no key of the range is never looked at.
__device__ __forceinline__ long long block_row(const AttnArgs& a, int b, int kv_head, int key, int lo, int hi) {
  const int inside = min(max(key, lo & ~15), (hi - 1) & ~15);
  const int page = kv_page(a.batch, b, inside >> a.pages.page_shift, a.pages.pages);
  return (((long long)page * a.pages.heads + kv_head) << a.pages.page_shift) + (inside & ((1 << a.pages.page_shift) - 1));
}

// The 16-byte slot that chunk c of a tile's row takes: c ^ swizzle(row), for the reads of one chunk of 16 rows (K, rows of BYTES bytes).
template <int BYTES>
__device__ __forceinline__ int swizzle(int row) {
  if constexpr (BYTES == 256) return row & 15;
  else if constexpr (BYTES == 128) return (row >> 1) & 7;
  else if constexpr (BYTES == 192 || BYTES == 64) return (row >> 2) & 3;
  else return (row >> 3) & 1;                       // 96 and 32
}

// Which of eight elements are not finite, a bit each.
template <typename T>
__device__ __forceinline__ unsigned not_finite(typename T::v8 x) {
  const v4u w = __builtin_bit_cast(v4u, x);
  unsigned bits = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if ((w[i] & T::kExpMask) == T::kExpMask) bits |= 1u << (2 * i);
    if ((w[i] & (T::kExpMask << 16)) == (T::kExpMask << 16)) bits |= 2u << (2 * i);
  }
  return bits;
}
template <typename T>
__device__ __forceinline__ typename T::v8 ones_at(unsigned bits) {
  v4u w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = T::pack(bits & (1u << (2 * i)) ? 1.0f : 0.0f, bits & (2u << (2 * i)) ? 1.0f : 0.0f);
  return __builtin_bit_cast(typename T::v8, w);
}
template <typename T>
__device__ __forceinline__ typename T::v8 zeros_at(typename T::v8 x, unsigned bits) {
  v4u w = __builtin_bit_cast(v4u, x);
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] &= (bits & (1u << (2 * i)) ? 0u : 0xffffu) | (bits & (2u << (2 * i)) ? 0u : 0xffff0000u);
  return __builtin_bit_cast(typename T::v8, w);
}

// log of the sum of exponentials from the reference (in powers of two) and the sum
__device__ __forceinline__ float log_sum(float ref, float l) { return (ref + __builtin_log2f(l)) * 0.6931471805599453f; }

// ---- narrow ---------------------------------------------------------------------------

template <KvFormat F, int D>
struct NarrowShape {
  static constexpr int BYTES = F == kSame ? 2 * D : D;        // of a row of the cache
  static constexpr int TILE = 32 * BYTES;                     // of a K or V tile of 32 keys
  static constexpr int COPIES = TILE / 1024;
  static constexpr int EXPS = F == kSame ? 0 : 256;           // the exponents of a tile's keys and values, one copy of 4 bytes a lane
  static constexpr int STAGE = 2 * TILE + EXPS;
  static constexpr int K_LOADS = COPIES + (F == kSame ? 0 : 1);   // (the exponents of both come with K)
  static constexpr int STAGES = TILE >= 6144 ? 1 : TILE >= 4096 ? 2 : TILE >= 3072 ? 3 : 4;
  static constexpr int RING = kWaves * STAGES * STAGE;
  static constexpr int JOIN = kWaves * (D / 16) * 64 * 16 + kWaves * 16 * 8;
  static constexpr int LDS = RING > JOIN ? RING : JOIN;
};

// 16 (4) bytes a lane from an address of its own, otherwise as lds_dma16_once (lds_dma16).  A call reads a byte of the cache once, and
// the next call reads another layer's: copies that leave no lines are 10 % faster (64 sequences of up to 8192 keys 140 -> 126 us).  KEPT: another workgroup
// is about to read the same.
template <bool KEPT>
__device__ __forceinline__ void lds_dma16_from(const unsigned char* from, void* lds_base) {
  const unsigned lds_addr = (unsigned)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void*)lds_base);
  if constexpr (KEPT) asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(lds_addr), "v"(from) : "memory", "m0");
  else asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off nt" : : "s"(lds_addr), "v"(from) : "memory", "m0");
}
__device__ __forceinline__ void lds_dma4_from(const signed char* from, void* lds_base) {
  const unsigned lds_addr = (unsigned)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void*)lds_base);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" : : "s"(lds_addr), "v"(from) : "memory", "m0");
}

// tid: of the 256 threads that work together
template <typename T, KvFormat F, int D, int NQ, bool KEPT, bool TREE>
__device__ __forceinline__ void narrow_attention(const AttnArgs& a, const Job& j, int kv_head, unsigned char* smem, int tid) {
  using S = NarrowShape<F, D>;
  using v8 = typename T::v8;
  using scalar = typename T::scalar;
  constexpr int KS = D / 32, DT = D / 16, CH = S::BYTES / 16, STAGES = S::STAGES;
  using lds_v4s = __attribute__((address_space(3))) v4s;
  using lds_v2i = __attribute__((address_space(3))) v2i;
  typedef short v8s __attribute__((ext_vector_type(8)));

  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m = lane & 15, kg = lane >> 4;
  const int base = j.lo & ~31;
  const int ntiles = j.hi > j.lo ? (j.hi - base + 31) / 32 : 0;
  unsigned char* const ring = smem + wave * (STAGES * S::STAGE);
  const int mine = ntiles > wave ? (ntiles - wave + kWaves - 1) / kWaves : 0;

  // a tile's two blocks of 16 keys, each in one page
  struct Blocks {
    long long r0, r1;
  };
  auto blocks_of = [&](int i) __attribute__((always_inline)) {
    const int key0 = base + 32 * (wave + kWaves * i);
    return Blocks{block_row(a, j.b, kv_head, key0, j.lo, j.hi), block_row(a, j.b, kv_head, key0 + 16, j.lo, j.hi)};
  };
  // Where the 16 bytes that a lane copies lie from the first row of their block; a copy's rows repeat every 16, so that both blocks
  // share these, but for rows of 96 and 32 bytes, of which a copy has rows of both blocks.
  constexpr bool WHOLE = 16 * S::BYTES % 1024 == 0;
  constexpr int OFFS = WHOLE ? 16 * S::BYTES / 1024 : S::COPIES;
  unsigned off[OFFS];
#pragma unroll
  for (int c = 0; c < OFFS; ++c) {
    const int p = 64 * c + lane, row = p / CH, slot = p - row * CH;
    off[c] = (row & 15) * S::BYTES + 16 * (slot ^ swizzle<S::BYTES>(row));
  }
  // VALUES: the tile of V, else that of K, and the exponents of both
  auto issue = [&](int i, int stage, const Blocks& at, auto values_c) __attribute__((always_inline)) {
    constexpr bool VALUES = decltype(values_c)::value;
    const int key0 = base + 32 * (wave + kWaves * i);
    unsigned char* const dst = ring + stage * S::STAGE;
    unsigned char* const to = VALUES ? dst + S::TILE : dst;
    const unsigned char* const from = VALUES ? a.pages.v : a.pages.k;
    const int least = j.lo - key0, most = j.hi - 1 - key0;
    if (least <= 0 && most >= 31) {
      const unsigned char *const b0 = from + at.r0 * S::BYTES, *const b1 = from + at.r1 * S::BYTES;
#pragma unroll
      for (int c = 0; c < S::COPIES; ++c) {
        if constexpr (WHOLE && KEPT) lds_dma16(c < OFFS ? b0 : b1, off[c % OFFS], to + 1024 * c);
        else if constexpr (WHOLE) lds_dma16_once(c < OFFS ? b0 : b1, off[c % OFFS], to + 1024 * c);
        else lds_dma16_from<KEPT>(((64 * c + lane) / CH >= 16 ? b1 : b0) + off[c], to + 1024 * c);
      }
    } else {
      // rows outside [lo, hi) repeat the nearest key inside: their weights are zero, and what they hold is finite if the cache is
#pragma unroll
      for (int c = 0; c < S::COPIES; ++c) {
        const int p = 64 * c + lane, row = p / CH, slot = p - row * CH;
        const int key = min(max(row, least), most);
        const long long at_row = key >= 16 ? at.r1 + key - 16 : at.r0 + key;
        lds_dma16_from<KEPT>(from + (size_t)at_row * S::BYTES + 16 * (slot ^ swizzle<S::BYTES>(row)), to + 1024 * c);
      }
    }
    if constexpr (F != kSame && !VALUES) {
      // lanes 0..7: the exponents of K, four keys each, lanes 8..15: of V
      const int four = 4 * (lane & 7), key = min(max(four, least & ~3), most & ~3);
      const long long at_row = key >= 16 ? at.r1 + key - 16 : at.r0 + key;
      lds_dma4_from((lane & 8 ? a.pages.v_exps : a.pages.k_exps) + at_row, dst + 2 * S::TILE);
    }
  };
  using keys_c = std::false_type;
  using values_c = std::true_type;

  v8 qf[NQ][KS];
  int row_lo[NQ], row_hi[NQ];
#pragma unroll
  for (int nq = 0; nq < NQ; ++nq) {
    const int row = min(j.row0 + 16 * nq + m, j.rows - 1);
    const Row r = row_of<TREE>(a, j, kv_head, row);
    row_lo[nq] = r.lo;
    row_hi[nq] = r.hi;
    const scalar* const q = query_of<T>(a, j, kv_head, row) + 8 * kg;
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[nq][s] = *reinterpret_cast<const v8*>(q + 32 * s);
  }
  asm volatile("" ::: "memory");

  v4f o[NQ][DT];
  float ref[NQ], l[NQ];
#pragma unroll
  for (int nq = 0; nq < NQ; ++nq) {
    ref[nq] = kNoRef;
    l[nq] = 0.0f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[nq][dt] = v4f{0.f, 0.f, 0.f, 0.f};
  }

  Blocks next{0, 0};
#pragma unroll
  for (int i = 0; i < STAGES; ++i) {
    if (i < mine) {
      const Blocks at = blocks_of(i);
      issue(i, i, at, keys_c{});
      issue(i, i, at, values_c{});
    }
  }
  if (STAGES < mine) next = blocks_of(STAGES);
  unsigned long long way[NQ][1];                               // TREE: the new tokens that each row sees
  if constexpr (TREE) {
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq) {
      int depth;
      walk_up<1>(a, j, min(j.row0 + 16 * nq + m, j.rows - 1) / a.group, 0, way[nq], &depth);
      if (a.window > 0) row_lo[nq] = clamp_position((long long)j.first + depth - a.window + 1, j.len);
    }
  }
  // the queries are there before the loop, which would otherwise wait for all that is on its way wherever they are used
#pragma unroll
  for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
    for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(qf[nq][s]));
  // One tile.  MASKED: some row does not see all of it.  ODD: some row of the cache has an exponent that fp16 elements do not.
  // keys_read and values_read come where the tile of K, and that of V, has been read.
  auto step = [&](int key0, const unsigned char* kt, auto masked_c, auto odd_c, auto&& keys_read, auto&& values_read) __attribute__((always_inline)) {
    constexpr bool MASKED = decltype(masked_c)::value, ODD = decltype(odd_c)::value;
    const unsigned char* const vt = kt + S::TILE;
    // lane (row m, kg) has keys 16 h + 4 kg + r: the factors of their scores (scale, and the power of two of K's row), and those of V's rows
    float kfac[2][4];
    int vexp[2][4];
    if constexpr (F != kSame) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const unsigned ke = *reinterpret_cast<const unsigned*>(kt + 2 * S::TILE + 16 * h + 4 * kg);
        const unsigned ve = *reinterpret_cast<const unsigned*>(kt + 2 * S::TILE + 32 + 16 * h + 4 * kg);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          kfac[h][r] = ODD ? a.scale_log2e : ldexpf(a.scale_log2e, (signed char)(ke >> (8 * r)));
          vexp[h][r] = (signed char)(ve >> (8 * r));
          if constexpr (MASKED) {                                  // what lies behind a sequence's keys has no exponent
            const int key = key0 + 16 * h + 4 * kg + r;
            if (key < j.lo || key >= j.hi) {
              kfac[h][r] = 0.0f;
              vexp[h][r] = 0;
            }
          }
        }
      }
    }
    v4f sc[NQ][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int nq = 0; nq < NQ; ++nq) sc[nq][h] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int row = 16 * h + m;
        v8 kf;
        if constexpr (F == kSame) {
          kf = *reinterpret_cast<const v8*>(kt + row * S::BYTES + (((4 * s + kg) ^ swizzle<S::BYTES>(row)) * 16));
        } else {
          const v2u w = *reinterpret_cast<const v2u*>(kt + row * S::BYTES + (((2 * s + (kg >> 1)) ^ swizzle<S::BYTES>(row)) * 16) + 8 * (kg & 1));
          if constexpr (ODD) kf = decode8_rounded<T, F>(w, ldexpf(1.0f, (signed char)kt[2 * S::TILE + row]));
          else kf = decode8<T, F>(w, 1.0f);
        }
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq) sc[nq][h] = T::mma16(kf, qf[nq][s], sc[nq][h]);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    keys_read();
    v8 p[NQ], rest[NQ];                                           // weights as two operands: rounded, and what that leaves
    unsigned seen[NQ];                                            // MASKED: which of the lane's eight keys its row sees
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r) sc[nq][h][r] *= F == kSame ? a.scale_log2e : kfac[h][r];
      if constexpr (MASKED) {
        seen[nq] = 255;
        unsigned drawn = ~0u;                                      // TREE: the tile's 32 keys, a bit each, but for bounds
        if constexpr (TREE) {
          const int off = key0 - j.first;
          if (off > -32) drawn = off >= 64 ? 0u : off >= 0 ? (unsigned)(way[nq][0] >> off) : (unsigned)(way[nq][0] << -off) | ((1u << -off) - 1);
          drawn >>= 4 * kg;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int key = key0 + 16 * h + 4 * kg + r;
            if (key < max(row_lo[nq], j.lo) || key >= min(row_hi[nq], j.hi) || (TREE && !(drawn >> (16 * h + r) & 1))) {
              sc[nq][h][r] = -INFINITY;
              seen[nq] &= ~(1u << (4 * h + r));
            }
          }
      }
      float mx = fmaxf(fmaxf(fmaxf(sc[nq][0][0], sc[nq][0][1]), fmaxf(sc[nq][0][2], sc[nq][0][3])),
                       fmaxf(fmaxf(sc[nq][1][0], sc[nq][1][1]), fmaxf(sc[nq][1][2], sc[nq][1][3])));
      if (__builtin_amdgcn_ballot_w64(!(mx <= ref[nq] + (kLift<T> + kSlack<T>))) != 0) {
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const float moved = fmaxf(ref[nq], mx - kLift<T>);
        const float alpha = __builtin_amdgcn_exp2f(ref[nq] - moved);
        ref[nq] = moved;
        l[nq] *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int r = 0; r < 4; ++r) o[nq][dt][r] *= alpha;
      }
      // bf16 weights take the power of two of their value's row with them; those of fp16 could leave its range, and V takes it
      unsigned w[4], u[4];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
          float p0 = __builtin_amdgcn_exp2f(sc[nq][h][r] - ref[nq]), p1 = __builtin_amdgcn_exp2f(sc[nq][h][r + 1] - ref[nq]);
          l[nq] += p0 + p1;
          if constexpr (F != kSame && std::is_same<T, Brain>::value) {
            p0 = ldexpf(p0, vexp[h][r]);
            p1 = ldexpf(p1, vexp[h][r + 1]);
          }
          const unsigned pair = T::pack(p0, p1);
          w[2 * h + r / 2] = pair;
          u[2 * h + r / 2] = T::pack(p0 - T::low(pair), p1 - T::high(pair));
        }
      p[nq] = __builtin_bit_cast(v8, (v4u{w[0], w[1], w[2], w[3]}));
      rest[nq] = __builtin_bit_cast(v8, (v4u{u[0], u[1], u[2], u[3]}));
    }
    v2h vpair[4];
    if constexpr (F != kSame && !ODD && std::is_same<T, Half>::value) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 4; r += 2) vpair[2 * h + r / 2] = v2h{(_Float16)ldexpf(1.0f, vexp[h][r]), (_Float16)ldexpf(1.0f, vexp[h][r + 1])};
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      v8 vf;
      if constexpr (F == kSame) {
        // 16 lanes hand in a block of 4 keys x 16 columns
        const int a4 = (lane & 15) >> 2, b4 = lane & 3;
        v4s half[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = 16 * h + 4 * kg + a4;
          half[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (lds_v4s*)(vt + row * S::BYTES + (((2 * dt + (b4 >> 1)) ^ swizzle<S::BYTES>(row)) * 16) + 8 * (b4 & 1)));
        }
        const v8s both = {half[0][0], half[0][1], half[0][2], half[0][3], half[1][0], half[1][1], half[1][2], half[1][3]};
        vf = __builtin_bit_cast(v8, both);
      } else {
        // 16 lanes hand in 8 keys x 16 columns, a pair of lanes a key
        const int a8 = (lane & 15) >> 1;
        const int row = 16 * (a8 >> 2) + 4 * kg + (a8 & 3);
        const v2i w = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i*)(vt + row * S::BYTES + ((dt ^ swizzle<S::BYTES>(row)) * 16) + 8 * (lane & 1)));
        vf = decode8<T, F>(__builtin_bit_cast(v2u, w), 1.0f);
        if constexpr (std::is_same<T, Half>::value) {
          v4u pairs = __builtin_bit_cast(v4u, vf);
#pragma unroll
          for (int i2 = 0; i2 < 4; ++i2) {
            const unsigned pair = pairs[i2];                      // (a bit cast of a vector's element itself takes the first element)
            if constexpr (ODD) pairs[i2] = T::pack(ldexpf(T::low(pair), vexp[i2 / 2][2 * (i2 % 2)]), ldexpf(T::high(pair), vexp[i2 / 2][2 * (i2 % 2) + 1]));
            else pairs[i2] = __builtin_bit_cast(unsigned, __builtin_bit_cast(v2h, pair) * vpair[i2]);
          }
          vf = __builtin_bit_cast(v8, pairs);
        }
      }
      if constexpr (MASKED) {
        // A value that is not finite must not reach the rows that do not see it (0 x inf): it leaves the product, and makes NaN of
        // the rows that do see it.
        const unsigned bad = not_finite<T>(vf);
        if (__builtin_amdgcn_ballot_w64(bad != 0) != 0) {
          vf = zeros_at<T>(vf, bad);
          const v8 flags = ones_at<T>(bad);
#pragma unroll
          for (int nq = 0; nq < NQ; ++nq) {
            const v4f hits = T::mma16(flags, ones_at<T>(seen[nq]), v4f{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (hits[r] > 0.0f) o[nq][dt][r] = __builtin_nanf("");
          }
        }
      }
#pragma unroll
      for (int nq = 0; nq < NQ; ++nq) {
        o[nq][dt] = T::mma16(vf, p[nq], o[nq][dt]);
        o[nq][dt] = T::mma16(vf, rest[nq], o[nq][dt]);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    values_read();
  };

  // Copies go out as soon as what lies in their place has been read, K's and V's apart, so that 2 STAGES - 1 of 2 STAGES tiles are on
  // their way while one is worked on; they land in the order they went out.
  constexpr int KL = S::K_LOADS, VL = S::COPIES;
  constexpr int BEHIND_K = (STAGES - 1) * (KL + VL) + VL, BEHIND_V = STAGES * KL + (STAGES - 1) * VL;   // loads behind K of tile i, behind its V
  static_assert(BEHIND_K < 64 && BEHIND_V < 64, "vmcnt counts to 63");
  constexpr auto vmcnt = [](int n) { return 0x0F70 | (n & 15) | ((n >> 4) << 14); };
  int stage = 0;
  for (int i = 0; i < mine; ++i) {
    const int key0 = base + 32 * (wave + kWaves * i);
    const bool more = i + STAGES < mine;
    if (i + STAGES <= mine) __builtin_amdgcn_s_waitcnt(vmcnt(BEHIND_K));
    else __builtin_amdgcn_s_waitcnt(vmcnt(0));
    asm volatile("" ::: "memory");
    auto keys_read = [&]() __attribute__((always_inline)) {
      if (more) {
        issue(i + STAGES, stage, next, keys_c{});
        __builtin_amdgcn_s_waitcnt(vmcnt(BEHIND_V));
      } else {
        __builtin_amdgcn_s_waitcnt(vmcnt(0));
      }
      asm volatile("" ::: "memory");
    };
    auto values_read = [&]() __attribute__((always_inline)) {
      if (more) {
        issue(i + STAGES, stage, next, values_c{});
        if (i + STAGES + 1 < mine) next = blocks_of(i + STAGES + 1);
      }
    };
    const unsigned char* const kt = ring + stage * S::STAGE;
    const bool masked = key0 < j.sure_lo || key0 + 32 > j.sure_hi || key0 < j.lo || key0 + 32 > j.hi;
    bool odd = false;
    if constexpr (F != kSame && std::is_same<T, Half>::value) {     // a lane looks at four of the tile's 64 exponents
      const unsigned e = *reinterpret_cast<const unsigned*>(kt + 2 * S::TILE + 4 * (lane & 15));
      odd = __builtin_amdgcn_ballot_w64(!(fits_half<F>((signed char)e) && fits_half<F>((signed char)(e >> 8)) && fits_half<F>((signed char)(e >> 16)) &&
                                          fits_half<F>((signed char)(e >> 24)))) != 0;
      if (__builtin_expect(odd, 0)) step(key0, kt, std::true_type{}, std::true_type{}, keys_read, values_read);
    }
    if (!odd) {
      if (masked) step(key0, kt, std::true_type{}, std::false_type{}, keys_read, values_read);
      else step(key0, kt, std::false_type{}, std::false_type{}, keys_read, values_read);
    }
    stage = stage == STAGES - 1 ? 0 : stage + 1;
  }

  // ---- the four waves meet, 16 rows at a time: O as [wave][tile][lane] in LDS, (ref, l) behind it
  v4f* const so = reinterpret_cast<v4f*>(smem);
  float* const sml = reinterpret_cast<float*>(smem + kWaves * DT * 64 * sizeof(v4f));   // [wave][row][2]
#pragma unroll
  for (int nq = 0; nq < NQ; ++nq) {
    if (j.row0 + 16 * nq >= j.rows) break;
    l[nq] += __shfl_xor(l[nq], 16);
    l[nq] += __shfl_xor(l[nq], 32);
    __syncthreads();
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) so[(wave * DT + dt) * 64 + lane] = o[nq][dt];
    if (kg == 0) {
      sml[(wave * 16 + m) * 2] = ref[nq];
      sml[(wave * 16 + m) * 2 + 1] = l[nq];
    }
    __syncthreads();
    const int q = tid & 15, row = j.row0 + 16 * nq + q;
    if (row < j.rows) {
      float top = kNoRef, sum = 0.0f, w[kWaves];
#pragma unroll
      for (int i = 0; i < kWaves; ++i) top = fmaxf(top, sml[(i * 16 + q) * 2]);
#pragma unroll
      for (int i = 0; i < kWaves; ++i) {
        w[i] = __builtin_amdgcn_exp2f(sml[(i * 16 + q) * 2] - top);
        sum += w[i] * sml[(i * 16 + q) * 2 + 1];
      }
      const Row r = row_of<TREE>(a, j, kv_head, row);
      const bool none = r.hi <= r.lo || (TREE && r.loose && sum == 0.0f);
      const float inv = none ? 0.0f : 1.0f / sum;
      for (int g = tid >> 4; g < D / 4; g += kWaves * 4) {   // columns 4 g .. +3: tile g / 4, lane group g % 4
        v4f acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < kWaves; ++i) {
          const v4f v = so[(i * DT + (g >> 2)) * 64 + 16 * (g & 3) + q];
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[e] += w[i] * v[e];
        }
        if (j.parts == 1) {
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[e] = finite_or_nan(acc[e]);
          *reinterpret_cast<v2u*>((scalar*)a.o + r.at * D + 4 * g) = v2u{T::pack(acc[0] * inv, acc[1] * inv), T::pack(acc[2] * inv, acc[3] * inv)};
        } else {
          *reinterpret_cast<v4f*>(a.part_o + (first_part(a, j.small, j.b, kv_head, row, r.at) + j.part) * D + 4 * g) = acc;
        }
      }
      if (tid < 16) {
        if (j.parts > 1) {
          float* const ml = a.part_ml + 2 * (first_part(a, j.small, j.b, kv_head, row, r.at) + j.part);
          ml[0] = top;
          ml[1] = sum;
        } else if (a.lse) {
          a.lse[r.at] = none ? -INFINITY : log_sum(top, sum);
        }
      }
    }
  }
}

// The slots are `tiles` row blocks of each of `sequences`.  Workgroups that are 8 apart run on one XCD, at about the same time: the row blocks of a (sequence, head, part)
// are, and the head goes fastest.
template <typename T, KvFormat F, int D, int NQ, bool KEPT, bool TREE>
__global__ __launch_bounds__(kWaves * 64, 2) void paged_narrow_kernel(AttnArgs a, int tiles) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  int id = blockIdx.x, tile = 0;
  if (KEPT) {
    const int units = gridDim.x / tiles, group = id / (8 * tiles) * 8, width = min(8, units - group), in = id - group * tiles;   // the last group may be narrower
    tile = in / width;
    id = group + in - tile * width;
  }
  const int kv_head = id % a.pages.heads, rest = id / a.pages.heads;
  const int b = rest / a.cut.nparts, part = rest % a.cut.nparts;
  Job j;
  if (!find_job<16 * NQ, TREE>(a, b, tile, part, false, j)) return;
  narrow_attention<T, F, D, NQ, KEPT, TREE>(a, j, kv_head, smem, threadIdx.x);
}

// ---- wide -----------------------------------------------------------------------------

// Eight waves of 32 rows.  A wave alternates between a phase of matrix instructions, M(t): O^T += V(t)^T P(t)^T and then the scores of
// tile t + 1, and a phase of vector instructions, S(t): the weights of tile t; waves 4 to 7 run one phase behind waves 0 to 3, so that of the two
// waves of a SIMD one feeds the matrix unit while the other works out weights.  A barrier ends every phase.  Waves 0 to 3 bring V(t + 1),
// which is read from their M(t + 1) on, into one of three places, waves 4 to 7 K(t + 2) into that of K(t).  16-bit elements are copied straight into
// LDS; codes of 8 bits go through registers, a tile earlier, and are written as 16-bit elements.
//
// PAIRED, for trees, most of which have 128 rows or fewer: waves 4 to 7 have the rows of waves 0 to 3, and every other tile, each half of them tiles of K and V
// of its own; the two sums are joined at the end.
constexpr int kWideWaves = 8, kWideRows = 32 * kWideWaves, kPairedRows = kWideRows / 2;
constexpr float kMostSum = 32768.0f;          // a lane's sum of 32 weights above this moves the reference, to where it is at most 32 * 2^kLift

template <int D, bool TREE, bool PAIRED>
struct WideShape {
  static constexpr int BYTES = 2 * D, TILE = 64 * BYTES;
  static constexpr int ROWS = PAIRED ? kPairedRows : kWideRows;
  static constexpr int ORS = BYTES + 16;                       // a padded row of the O tiles that the waves turn round at the end
  static constexpr int RING = (PAIRED ? 8 : 5) * TILE;         // two tiles of K, three of V; PAIRED: two of each, twice
  static constexpr int FLAGS = 64 * D / 8;                     // TREE: of a place of V, a bit for each value that was not finite, [key][chunk of 8]
  static constexpr int NOTES = 64 + (TREE ? 4 * FLAGS : 0);  // of each place of V and wave; flags
  static constexpr int ENDS = kWideWaves * 32 * ORS;           // PAIRED: four waves' rows, and what the other four have of them
  static constexpr int TILES_LDS = RING + NOTES > ENDS ? RING + NOTES : ENDS;
  static constexpr int WORDS = kTreeMost / 64 + 1;             // TREE, behind those: of each row, which new tokens it sees
  static constexpr int LDS = TILES_LDS + (TREE ? ROWS * WORDS * 8 : 0);
  static_assert(!PAIRED || ROWS * ORS + ROWS * D * 4 + ROWS * 32 <= RING, "what halves hand to one another lies in the ring, behind the rows");
};

// V: the transposing read of a 32-lane pass covers 4 keys x 64 bytes, which these bring into four different groups of 64 bytes
template <int D>
__device__ __forceinline__ int v_swizzle(int row) {
  if constexpr (D == 128) return 4 * (row & 3);
  else if constexpr (D == 64) return 4 * ((row >> 1) & 1);
  else return 0;                                               // rows of 192 and 64 bytes lie that way
}

// TWO: weights as two operands.
template <typename T, KvFormat F, int D, bool TREE, bool PAIRED, bool TWO>
__device__ __forceinline__ void wide_attention(const AttnArgs& a, const Job& j, int kv_head, unsigned char* smem) {
  using S = WideShape<D, TREE, PAIRED>;
  using v8 = typename T::v8;
  using scalar = typename T::scalar;
  constexpr int DS = D / 16, DT = D / 32, CH = S::BYTES / 16;
  using lds_v4s = __attribute__((address_space(3))) v4s;
  typedef short v8s __attribute__((ext_vector_type(8)));

  using yes = std::true_type;
  using no = std::false_type;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = wave >> 2, cw = wave & 3;                   // which of the two run behind; whose 16 keys of a tile this wave brings
  const int jr = lane & 31, hh = lane >> 5;
  unsigned char* const tiles = smem + (PAIRED ? half * (4 * S::TILE) : 0);
  unsigned char* const Kb = tiles;
  unsigned char* const Vb = tiles + 2 * S::TILE;
  const int base = j.lo & ~63;
  const int ntiles = j.hi > j.lo ? (j.hi - base + 63) / 64 : 0;

  // rows of this wave
  const int in_rows = 32 * (PAIRED ? cw : wave);
  const int wrow0 = j.row0 + in_rows;
  const bool idle = wrow0 >= j.rows;
  const int row = min(wrow0 + jr, j.rows - 1);
  const Row r = row_of<TREE>(a, j, kv_head, row);
  int wave_lo, wave_hi, sure_lo, sure_hi;                      // keys that some, and that each, of the wave's rows see
  {
    const int t_lo = min(wrow0, j.rows - 1) / a.group, t_hi = (min(wrow0 + 32, j.rows) - 1) / a.group;
    const long long p_lo = (long long)j.first + (TREE ? 0 : t_lo), p_hi = (long long)j.first + t_hi;
    wave_hi = idle ? 0 : min(TREE || a.causal ? clamp_position(p_hi + 1, j.len) : j.len, j.hi);
    sure_hi = min(TREE ? clamp_position(j.first, j.len) : a.causal ? clamp_position(p_lo + 1, j.len) : j.len, j.hi);
    wave_lo = max(a.window > 0 ? clamp_position(p_lo - a.window + 1, j.len) : 0, j.lo);
    sure_lo = max(a.window > 0 ? clamp_position(p_hi - a.window + 1, j.len) : 0, j.lo);
  }
  int my_lo = max(r.lo, j.lo);
  const int my_hi = min(r.hi, j.hi);
  // TREE: which of the 64 keys of a tile a row sees; those of new tokens stand in words that begin where tiles do
  unsigned long long* const ways = reinterpret_cast<unsigned long long*>(smem + S::TILES_LDS) + (in_rows + jr) * S::WORDS;
  auto way_of = [&](int t) __attribute__((always_inline)) {
    const int key0 = base + 64 * t, word = (key0 - (j.first & ~63)) / 64;    // (both are multiples of 64)
    const int lo = my_lo - key0, hi = my_hi - key0;
    unsigned long long bits = word < 0 ? ~0ULL : word < S::WORDS ? ways[word] : 0ULL;
    bits &= lo <= 0 ? ~0ULL : lo < 64 ? ~0ULL << lo : 0ULL;
    return bits & (hi >= 64 ? ~0ULL : hi > 0 ? (1ULL << hi) - 1 : 0ULL);
  };
  auto sees = [&](int t) __attribute__((always_inline)) { return base + 64 * t < wave_hi && base + 64 * t + 64 > wave_lo; };
  auto masked = [&](int t) __attribute__((always_inline)) { return base + 64 * t < sure_lo || base + 64 * t + 64 > sure_hi; };

  v8 qf[DS];
  {
    const scalar* const q = query_of<T>(a, j, kv_head, row) + 8 * hh;
#pragma unroll
    for (int s = 0; s < DS; ++s) qf[s] = *reinterpret_cast<const v8*>(q + 16 * s);
  }
  asm volatile("" ::: "memory");

  // ---- tiles into LDS: a wave brings the 16 keys from 16 cw on, which lie in one page; waves 0 to 3 those of V, the others those of K (PAIRED: each those of both)
  constexpr int CP = D / 32;                                   // 1 KB copies of 16 rows of 16-bit elements
  const int shift = a.pages.page_shift;
  const long long page_rows = (long long)a.pages.heads << shift;
  const long long head_row = (long long)kv_head << shift;
  const int* const table = a.batch.table + (long long)j.b * a.batch.width;
  constexpr int LD = (D + 63) / 64;                            // 8 bits, 16 codes a lane: 16-byte pieces of a block of 16 rows, D of them, by 64 lanes
  struct Bring {
    bool keys;
    const unsigned char* from;
    const signed char* exps;
    unsigned src[D == 96 ? CP : 1];
    v4u codes[LD];
    std::conditional_t<TREE, int, float> power[LD];            // of two; TREE: the exponent as it is held, since what is made of it waits for it
  };
  // Cache row (from this head's first) of the 16 keys of this wave in tile t; of the nearest 16 in [lo, hi) where those lie outside (INSIDE: they
  // do not).
  auto block_at = [&](int t, auto inside_c) __attribute__((always_inline)) {
    int key = base + 64 * t + 16 * cw;
    if constexpr (!decltype(inside_c)::value) key = min(max(key, j.lo & ~15), (j.hi - 1) & ~15);
    const int page = min(max(load_uniform(table, key >> shift), 0), a.pages.pages - 1);
    return page * page_rows + (key & ((1 << shift) - 1));
  };
  // Where a lane's 16 bytes of a copy lie: with 64 and 128 elements the swizzle makes copy i's places those of the first with some bits turned over.
  auto begin = [&](Bring& b, bool of_keys) __attribute__((always_inline)) {
    b.keys = of_keys;
    b.from = (of_keys ? a.pages.k : a.pages.v) + head_row * (F == kSame ? S::BYTES : D);
    b.exps = F == kSame ? nullptr : (of_keys ? a.pages.k_exps : a.pages.v_exps) + head_row;
#pragma unroll
    for (int i = 0; i < (D == 96 ? CP : 1); ++i) {
      const int p = 64 * i + lane, rw = p / CH, slot = p - rw * CH, in_tile = 16 * cw + rw;
      b.src[i] = rw * S::BYTES + 16 * (slot ^ (of_keys ? swizzle<S::BYTES>(in_tile) : v_swizzle<D>(in_tile)));
    }
  };
  auto source = [&](const Bring& b, int i) __attribute__((always_inline)) {
    const unsigned turned = b.keys && D != 96 ? 64 : 0;
    return D == 96 ? b.src[D == 96 ? i : 0] : (b.src[0] ^ (i * turned)) + 1024 * i;
  };
  // 16 rows of tile t, `at` what block_at gave, into the tile at `to`
  auto copy = [&](const Bring& b, unsigned char* to, int t, long long at, auto inside_c) __attribute__((always_inline)) {
    const int key0 = base + 64 * t + 16 * cw;
    const unsigned char* const block = uniform(b.from + at * S::BYTES);
    unsigned char* const dst = to + cw * (16 * S::BYTES);
    if (decltype(inside_c)::value || (key0 >= j.lo && key0 + 16 <= j.hi)) {
#pragma unroll
      for (int i = 0; i < CP; ++i) lds_dma16(block, source(b, i), dst + 1024 * i);
    } else {                                                   // rows outside [lo, hi) repeat the nearest key inside
      const int inside = min(max(key0, j.lo & ~15), (j.hi - 1) & ~15);   // where `at` begins
      const int least = max(j.lo - inside, 0), most = min(j.hi - 1 - inside, 15);
#pragma unroll
      for (int i = 0; i < CP; ++i) {
        const int rw = (64 * i + lane) / CH;
        lds_dma16(block, source(b, i) + (min(max(key0 + rw - inside, least), most) - rw) * S::BYTES, dst + 1024 * i);
      }
    }
  };
  // 8 bits.  (TREE: from addresses of the whole wave, which frees registers there; chunks and prompts have none to spare for them: four prompts of 4096 in int8, 16 heads of
  // 128, fp16, 197 us, and 211 that way.)
  auto load = [&](Bring& b, int t, long long at, auto inside_c) __attribute__((always_inline)) {
    const int key0 = base + 64 * t + 16 * cw;
    const int inside = min(max(key0, j.lo & ~15), (j.hi - 1) & ~15);
    const int least = max(j.lo - inside, 0), most = min(j.hi - 1 - inside, 15);
#pragma unroll
    for (int i = 0; i < LD; ++i) {
      const int p = min(64 * i + lane, D - 1), rw = p / (D / 16), piece = p - rw * (D / 16);
      const int row = decltype(inside_c)::value ? rw : min(max(key0 + rw - inside, least), most);
      if constexpr (TREE) {
        const unsigned char *const block = uniform(b.from + at * D), *const block_exps = uniform((const unsigned char*)b.exps + at);
        b.codes[i] = *reinterpret_cast<const v4u*>(block + (decltype(inside_c)::value ? 16u * p : (unsigned)row * D + 16u * piece));
        b.power[i] = (signed char)block_exps[(unsigned)row];
      } else {
        const long long row_at = at + row;
        b.codes[i] = *reinterpret_cast<const v4u*>(b.from + row_at * D + 16 * piece);
        b.power[i] = ldexpf(1.0f, b.exps[row_at]);
      }
    }
  };
  auto store = [&](const Bring& b, unsigned char* to) __attribute__((always_inline)) {
    if constexpr (F != kSame) {
#pragma unroll
      for (int i = 0; i < LD; ++i) {
        const int p = 64 * i + lane, rw = p / (D / 16), piece = p - rw * (D / 16), in_tile = 16 * cw + rw;
        const int swz = b.keys ? swizzle<S::BYTES>(in_tile) : v_swizzle<D>(in_tile);
        const float scale = TREE ? ldexpf(1.0f, (int)b.power[i]) : (float)b.power[i];
        auto put = [&](auto decode) __attribute__((always_inline)) {
          if (D % 64 == 0 || p < D) {
#pragma unroll
            for (int c = 0; c < 2; ++c)
              *reinterpret_cast<v8*>(to + in_tile * S::BYTES + 16 * ((2 * piece + c) ^ swz)) = decode(v2u{b.codes[i][2 * c], b.codes[i][2 * c + 1]}, scale);
          }
        };
        // (the conversion of e4m3 rounds once whatever the scale)
        constexpr bool LOOK = std::is_same<T, Half>::value && F == kInt8;
        if (LOOK && __builtin_expect(__builtin_amdgcn_ballot_w64(!(scale >= 0x1p-24f && scale <= 0x1p9f)) != 0, 0)) put(decode8_rounded<T, F>);
        else put(decode8<T, F>);
      }
    }
  };
  Bring mine, keys;                                            // PAIRED: V and K; else the one that this wave brings
  begin(mine, PAIRED ? false : half != 0);
  if constexpr (PAIRED) begin(keys, true);

  // ---- fragments: K row 32 h + jr, bytes [32 s + 16 hh, +16); V the block of 4 keys x 16 columns that 16 lanes hand in
  // (The swizzles touch bits of the chunk's index that are zero in a row's address, so that a step's offset is the first one's with some bits turned
  // over, and what they leave alone is added.)
  constexpr int KX = D == 128 ? 15 : D == 64 ? 7 : 3, VX = D == 128 ? 12 : D == 64 ? 4 : 0;   // those bits
  const unsigned k_off = jr * S::BYTES + ((hh ^ swizzle<S::BYTES>(jr)) * 16);
  const int v_row = 4 * hh + ((lane & 15) >> 2);
  const unsigned v_off = v_row * S::BYTES + v_swizzle<D>(v_row) * 16 + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
  auto read_k = [&](const unsigned char* kt, int h, int s) __attribute__((always_inline)) {
    return *reinterpret_cast<const v8*>(kt + 32 * h * S::BYTES + (k_off ^ (16 * (2 * s & KX))) + 16 * (2 * s & ~KX));
  };
  auto read_v = [&](const unsigned char* vt, int key, int dt) __attribute__((always_inline)) {   // keys key + 4 hh + .. and 8 more
    const unsigned char* const p = vt + key * S::BYTES + (v_off ^ (16 * (4 * dt & VX))) + 16 * (4 * dt & ~VX);
    const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(p));
    const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(p + 8 * S::BYTES));
    const v8s both = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    return __builtin_bit_cast(v8, both);
  };

  v16f o[DT], sc[2];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[dt][e] = 0.0f;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int e = 0; e < 16; ++e) sc[h][e] = 0.0f;
  float ref = kNoRef, l = 0.0f;
  v8 pf[2][2], rest[2][2];                                     // weights as operands, and (TWO) what their rounding leaves

  // The weights of the tile's scores as operands of P V; returns this lane's share of their sum.  (TWO: still in 32 bits, in p.)
  float p[TWO ? 32 : 1];
  auto weights = [&]() __attribute__((always_inline)) {
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        v4u w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[h][8 * s + 2 * i], a.scale_log2e, -ref));
          const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[h][8 * s + 2 * i + 1], a.scale_log2e, -ref));
          sum[i] += p0;
          sum[i] += p1;
          if constexpr (TWO) {
            p[16 * h + 8 * s + 2 * i] = p0;
            p[16 * h + 8 * s + 2 * i + 1] = p1;
          } else {
            w[i] = T::pack(p0, p1);
          }
        }
        if constexpr (!TWO) pf[h][s] = __builtin_bit_cast(v8, w);
      }
    return (sum[0] + sum[1]) + (sum[2] + sum[3]);
  };
  auto two_operands = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v4u w, left;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p0 = p[8 * k + 2 * i], p1 = p[8 * k + 2 * i + 1];
        unsigned pair = T::pack(p0, p1);
        asm("" : "+v"(pair));                                  // (taken out of the pair: the compiler would round each once more)
        w[i] = pair;
        left[i] = T::pack(__builtin_fmaf(T::low(pair), -1.0f, p0), __builtin_fmaf(T::high(pair), -1.0f, p1));
      }
      pf[k / 2][k % 2] = __builtin_bit_cast(v8, w);
      rest[k / 2][k % 2] = __builtin_bit_cast(v8, left);
    }
  };
  // The reference is not compared with every tile's maximum: weights are worked out against it as it is, and only when a lane's sum says that
  // one of them may not fit 16 bits (or came out infinite, as all do before there is a reference) are the maxima taken, the reference moved, O and the sums
  // rescaled and the tile's weights worked out again.  Any reference gives the same O / l.
  auto phase_s = [&](int t, auto clean_c) __attribute__((always_inline)) {
    if (!decltype(clean_c)::value && masked(t)) {
      const int key0 = base + 64 * t + 4 * hh;
      unsigned long long drawn = 0;
      if constexpr (TREE) drawn = way_of(t) >> (4 * hh);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int in = 32 * h + 8 * (e >> 2) + (e & 3), key = key0 + in;
          if (TREE ? !(drawn >> in & 1) : key < my_lo || key >= my_hi) sc[h][e] = -INFINITY;
        }
    }
    float psum = weights();
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(!(psum <= kMostSum)) != 0, 0)) {
      float mx = sc[0][0];
#pragma unroll
      for (int e = 1; e < 32; ++e) mx = fmaxf(mx, sc[e >> 4][e & 15]);
      const float moved = fmaxf(ref, max_with_other_half(mx) * a.scale_log2e - kLift<T>);
      const float alpha = __builtin_amdgcn_exp2f(ref - moved);
      ref = moved;
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[dt][e] *= alpha;
      psum = weights();
    }
    if constexpr (TWO) two_operands();
    l += psum;
  };

  constexpr int LA = 4;                                        // fragments read ahead of the matrix instruction that uses them
  constexpr int NPV = 4 * DT, NQK = 2 * DS;
  static_assert(LA <= NPV && LA <= NQK);
  // PV: P V of a tile; QK: the scores of the next
  auto phase_m = [&](const unsigned char* vt, const unsigned char* kt, auto pv_c, auto qk_c) __attribute__((always_inline)) {
    constexpr bool PV = decltype(pv_c)::value, QK = decltype(qk_c)::value;
    constexpr int N0 = PV ? NPV : 0, N = N0 + (QK ? NQK : 0);
    auto read = [&](auto n_c) __attribute__((always_inline)) {
      constexpr int n = decltype(n_c)::value;
      if constexpr (n < N0) return read_v(vt, 32 * (n / (2 * DT)) + 16 * ((n % (2 * DT)) / DT), n % DT);
      else return read_k(kt, (n - N0) % 2, (n - N0) / 2);
    };
    v8 fr[N];
    static_for<LA>([&](auto i_c) __attribute__((always_inline)) { fr[decltype(i_c)::value] = read(i_c); });
    __builtin_amdgcn_s_setprio(3);
    __builtin_amdgcn_sched_barrier(0);
    static_for<N>([&](auto i_c) __attribute__((always_inline)) {
      constexpr int i = decltype(i_c)::value;
      if constexpr (i < N0) {
        constexpr int h = i / (2 * DT), s = (i % (2 * DT)) / DT, dt = i % DT;
        o[dt] = T::mma32(fr[i], pf[h][s], o[dt]);
        if constexpr (TWO) o[dt] = T::mma32(fr[i], rest[h][s], o[dt]);
      } else {
        constexpr int s = (i - N0) / 2, h = (i - N0) % 2;
        v16f zero;
#pragma unroll
        for (int e = 0; e < 16; ++e) zero[e] = 0.0f;
        sc[h] = T::mma32(fr[i], qf[s], s == 0 ? zero : sc[h]);
      }
      if constexpr (i + LA < N) fr[i + LA] = read(std::integral_constant<int, i + LA>{});
      __builtin_amdgcn_sched_barrier(0);
    });
    __builtin_amdgcn_s_setprio(0);
  };
  // Waves 0 to 3 (PAIRED: all) look whether their 16 keys of a tile of V hold anything that is not finite, and leave word for all.
  unsigned* const words = reinterpret_cast<unsigned*>(smem + S::RING) + (PAIRED ? 8 * half : 0);   // [three places of V][wave]; PAIRED: [two][wave], twice
  unsigned char* const flags = smem + S::RING + 64 + (PAIRED ? 2 * S::FLAGS * half : 0);
  auto look = [&](unsigned char* vt, int place) __attribute__((always_inline)) {
    unsigned bad = 0;
#pragma unroll
    for (int i = 0; i < CP; ++i) bad |= not_finite<T>(*reinterpret_cast<const v8*>(vt + cw * (16 * S::BYTES) + 1024 * i + 16 * lane));
    const bool any = __builtin_amdgcn_ballot_w64(bad != 0) != 0;
    if (lane == 0) words[4 * place + cw] = any;
    if constexpr (TREE) {
      if (__builtin_expect(any, 0)) {                            // those leave the tile, for 0 x inf, and a bit is left for each
#pragma unroll 1
        for (int i = 0; i < CP; ++i) {
          const int p = 64 * i + lane, key = 16 * cw + p / CH, chunk = (p % CH) ^ v_swizzle<D>(key);
          v8* const at = reinterpret_cast<v8*>(vt + cw * (16 * S::BYTES) + 16 * p);
          const v8 x = *at;
          const unsigned bits = not_finite<T>(x);
          *at = zeros_at<T>(x, bits);
          flags[place * S::FLAGS + key * (D / 8) + chunk] = (unsigned char)bits;
        }
      }
    }
  };
  // TREE: NaN for the rows that see a key whose value was not finite
  auto mark = [&](int t, int place) __attribute__((always_inline)) {
    const unsigned long long drawn = way_of(t);
#pragma unroll 1
    for (int key = 0; key < 64; ++key) {
      if (words[4 * place + (key >> 4)] == 0) continue;
      const bool sees_it = drawn >> key & 1;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const unsigned four = *reinterpret_cast<const unsigned*>(flags + place * S::FLAGS + key * (D / 8) + 4 * dt) >> (4 * hh);   // (chunks 4 dt .. +3)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (sees_it && (four >> (8 * (e >> 2) + (e & 3)) & 1)) o[dt][e] = __builtin_nanf("");
      }
    }
  };
  auto all_finite = [&](int place) __attribute__((always_inline)) {
    const v4u w = *reinterpret_cast<const v4u*>(words + 4 * place);
    return __builtin_amdgcn_readfirstlane((w[0] | w[1]) | (w[2] | w[3])) == 0;
  };
  // P V of a tile whose keys not every row sees and whose values are not all finite: those leave the product (0 x inf), and make NaN
  // of the rows that do see them.
  auto careful_pv = [&](const unsigned char* vt, int t) __attribute__((always_inline)) {
#pragma unroll 1
    for (int step = 0; step < 4; ++step) {
      const v8 p = step == 0 ? pf[0][0] : step == 1 ? pf[0][1] : step == 2 ? pf[1][0] : pf[1][1];
      const int key0 = base + 64 * t + 16 * step + 4 * hh;
      unsigned seen = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int in = 8 * (e >> 2) + (e & 3), key = key0 + in;
        if (key >= my_lo && key < my_hi) seen |= 1u << e;
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const v8 vf = read_v(vt, 16 * step, dt);
        const unsigned bad = not_finite<T>(vf);
        v16f hits;
#pragma unroll
        for (int e = 0; e < 16; ++e) hits[e] = 0.0f;
        hits = T::mma32(ones_at<T>(bad), ones_at<T>(seen), hits);
        o[dt] = T::mma32(zeros_at<T>(vf, bad), p, o[dt]);
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (hits[e] > 0.0f) o[dt][e] = __builtin_nanf("");
      }
    }
  };
  // a barrier that waits for nothing of the wave's own: whoever wrote what the barrier publishes has waited before it
  auto phase_barrier = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  if (ntiles > 0) {
    // V(0) by waves 0 to 3, K(0) by the others, and K(1) behind it
    constexpr int AHEAD = F == kSame ? 0 : 1;                  // codes go through registers a tile earlier
    // TREE: what lies behind the last tile is the nearest 16 keys once more; rows in front of and behind [lo, hi) that share 16 keys with it come as they are, and
    // no row sees them
    if constexpr (PAIRED) {
      const long long at0 = block_at(half, no{}), at1 = block_at(half + 2, no{});
      if constexpr (F == kSame) {
        copy(keys, Kb, half, at0, yes{});
        copy(mine, Vb, half, at0, yes{});
        copy(keys, Kb + S::TILE, half + 2, at1, yes{});
      } else {
        Bring second = keys;
        load(keys, half, at0, yes{});
        load(mine, half, at0, yes{});
        load(second, half + 2, at1, yes{});
        store(keys, Kb);
        store(mine, Vb);
        store(second, Kb + S::TILE);
        load(mine, half + 2, at1, yes{});
        load(keys, half + 4, block_at(half + 4, no{}), yes{});
      }
    } else if constexpr (TREE) {
      const long long at0 = block_at(0, no{}), at1 = block_at(1, no{});
      if constexpr (F == kSame) {
        copy(mine, half ? Kb : Vb, 0, at0, yes{});
        if (half) copy(mine, Kb + S::TILE, 0, at1, yes{});
      } else {
        Bring second = mine;
        load(mine, 0, at0, yes{});
        if (half) load(second, 0, at1, yes{});
        store(mine, half ? Kb : Vb);
        if (half) store(second, Kb + S::TILE);
        load(mine, 0, half ? block_at(2, no{}) : at1, yes{});
      }
    } else if constexpr (F == kSame) {
      copy(mine, half ? Kb : Vb, 0, block_at(0, no{}), no{});
      if (half && ntiles > 1) copy(mine, Kb + S::TILE, 1, block_at(1, no{}), no{});
    } else {
      load(mine, 0, block_at(0, no{}), no{});
      store(mine, half ? Kb : Vb);
      if (ntiles > 1) load(mine, 1, block_at(1, no{}), no{});
      if (half) {
        if (ntiles > 1) store(mine, Kb + S::TILE);
        if (ntiles > 2) load(mine, 2, block_at(2, no{}), no{});
      }
    }
    const int ahead = PAIRED ? 2 * (2 + AHEAD) : (half ? 2 : 1) + AHEAD;          // S(t) asks for tile t + ahead; PAIRED: that one of K, the one before it of V
    const int asked = (PAIRED ? half : 0) + ahead;
    long long next = TREE || asked < ntiles ? block_at(asked, no{}) : 0;
    if (TREE && (j.hi > (j.first & ~63) || a.window > 0)) {    // (no tile of another part has a word)
      unsigned long long bits[S::WORDS];
      int depth;
      const int before = j.first & 63;                         // keys in front of the new tokens in the first word
      walk_up<S::WORDS>(a, j, row / a.group, before, bits, &depth);
      bits[0] |= (1ULL << before) - 1;
      if (hh == 0 && (!PAIRED || half == 0)) {
#pragma unroll
        for (int w = 0; w < S::WORDS; ++w) ways[w] = bits[w];
      }
      if (a.window > 0) my_lo = max(clamp_position((long long)j.first + depth - a.window + 1, j.len), j.lo);
    }
    __builtin_amdgcn_s_waitcnt(0x0F70);                        // vmcnt(0)
    __syncthreads();
    phase_m(Vb, Kb, no{}, yes{});
    if constexpr (TREE) {
      // One turn for all tiles, as code that runs once takes longer to fetch than to run: what a turn asks for and puts away behind the last tile is that tile once more,
      // and its scores go nowhere.
      constexpr int STEP = PAIRED ? 2 : 1;                     // from a wave's tile to its next
      if constexpr (PAIRED) phase_barrier();                   // waves 0 to 3 are about to write where K(0) was read
      int kcur = 0, knext = S::TILE;                           // K(t), that of the next
      int vcur = 2 * S::TILE, vnext = 3 * S::TILE, vfree = (PAIRED ? 2 : 4) * S::TILE;   // V(t), the next, and the place of the one behind: PAIRED, that of V(t)
      long long behind = PAIRED ? block_at(asked - 2, no{}) : 0;
      if (half) phase_barrier();
      const int first_tile = PAIRED ? half : 0;                // PAIRED: both halves take as many turns, the last of which may have no tile for waves 4 to 7
      for (int t = first_tile; t < ntiles + first_tile; t += STEP) {
        if constexpr (PAIRED && F == kSame) {
          copy(keys, tiles + kcur, 0, next, yes{});
          copy(mine, tiles + vnext, 0, behind, yes{});
        } else if constexpr (PAIRED) {
          store(keys, tiles + kcur);
          store(mine, tiles + vnext);
          load(keys, 0, next, yes{});
          load(mine, 0, behind, yes{});
        } else if constexpr (F == kSame) {
          copy(mine, tiles + (half ? kcur : vnext), 0, next, yes{});
        } else {
          store(mine, tiles + (half ? kcur : vnext));
          load(mine, 0, next, yes{});
        }
        behind = next;
        next = block_at(t + ahead + STEP, no{});
        __builtin_amdgcn_sched_barrier(0);                     // the copies go out before the weights are begun
        const bool works = !idle && t < ntiles;
        const bool some = base + 64 * t < max(j.sure_lo, j.lo) || base + 64 * t + 64 > min(j.sure_hi, j.hi);   // some wave's rows do not see all of it
        const int place = vcur / S::TILE - 2;
        if (works) phase_s(t, no{});
        if (some && (PAIRED || !half)) look(tiles + vcur, place);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");     // what was written to LDS
        phase_barrier();
        if (works) phase_m(tiles + vcur, tiles + knext, yes{}, yes{});
        if (some && works && __builtin_expect(!all_finite(place), 0)) mark(t, place);
        if constexpr (F == kSame) __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0): the copies that this wave asked for in S(t)
        phase_barrier();
        const int k = kcur, v = vcur;
        kcur = knext;
        knext = k;
        vcur = vnext;
        vnext = vfree;
        vfree = PAIRED ? vcur : v;
      }
      if (!half) phase_barrier();
    } else {
      int vcur = 2 * S::TILE, vnext = 3 * S::TILE, vfree = 4 * S::TILE;           // V(t), V(t + 1), the place of V(t + 2)
      int kcur = 0, knext = S::TILE;                                              // K(t), K(t + 1)
      // Tiles [clean, dirty): every row sees all of them, and the tiles that they ask for lie inside [lo, hi)
      const int whole = (j.hi - base) / 64;
      const int clean = (max(j.sure_lo, j.lo) - base + 63) / 64, dirty = min((min(j.sure_hi, j.hi) - base) / 64, whole - 2 - AHEAD - 1);
      auto turn = [&](int t, auto clean_c) __attribute__((always_inline)) {
        constexpr bool CLEAN = decltype(clean_c)::value;
        // K(t) was last read in the phase before this one, V(t - 2) two before
        const int bring = t + ahead;
        if constexpr (F == kSame) {
          if (CLEAN || bring < ntiles) copy(mine, smem + (half ? kcur : vnext), bring, next, clean_c);
        } else {
          if (CLEAN || bring - 1 < ntiles) store(mine, smem + (half ? kcur : vnext));
          if (CLEAN || bring < ntiles) load(mine, bring, next, clean_c);
        }
        if (CLEAN || bring + 1 < ntiles) next = block_at(bring + 1, clean_c);
        __builtin_amdgcn_sched_barrier(0);                     // the copies go out before the weights are begun
        if (CLEAN || sees(t)) phase_s(t, clean_c);
        if (!CLEAN && !half) look(smem + vcur, vcur / S::TILE - 2);
        if constexpr (!CLEAN || F != kSame) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // what was written to LDS
        phase_barrier();
        const unsigned char *const vt = smem + vcur, *const kt = smem + knext;
        if constexpr (CLEAN) {
          phase_m(vt, kt, yes{}, yes{});
        } else {
          if (sees(t)) {
            if (masked(t) && __builtin_expect(!all_finite(vcur / S::TILE - 2), 0)) careful_pv(vt, t);
            else phase_m(vt, kt, yes{}, no{});
          }
          if (t + 1 < ntiles) phase_m(vt, kt, no{}, yes{});
        }
        if constexpr (F == kSame) __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0): the copies that this wave asked for in S(t)
        phase_barrier();
        const int v = vcur, k = kcur;
        vcur = vnext;
        vnext = vfree;
        vfree = v;
        kcur = knext;
        knext = k;
      };
      if (half) phase_barrier();
      for (int t = 0; t < ntiles; ++t) {
        if (t == clean)
          for (; t < dirty; ++t) turn(t, yes{});
        turn(t, no{});
      }
      if (!half) phase_barrier();
    }
  }
  // PAIRED: each half has the first or the last of the columns in the end, and hands the others over
  const auto columns = [&](auto&& f) __attribute__((always_inline)) {
    static_for<DT>([&](auto dt) __attribute__((always_inline)) {
      if (!PAIRED || (decltype(dt)::value < (DT + 1) / 2) == (half == 0)) f(dt);
    });
  };
  if constexpr (PAIRED) {
    v4f* const so = reinterpret_cast<v4f*>(smem + S::ROWS * S::ORS) + cw * (DT * 4 * 64) + lane;
    float* const sml = reinterpret_cast<float*>(smem + S::ROWS * (S::ORS + D * 4)) + (cw * 64 + lane) * 2;
    __syncthreads();
    static_for<DT>([&](auto dt_c) __attribute__((always_inline)) {
      constexpr int dt = decltype(dt_c)::value;
      if ((dt < (DT + 1) / 2) == (half != 0)) {
#pragma unroll
        for (int g = 0; g < 4; ++g) so[64 * (4 * dt + g)] = v4f{o[dt][4 * g], o[dt][4 * g + 1], o[dt][4 * g + 2], o[dt][4 * g + 3]};
      }
    });
    sml[8 * 64 * half] = ref;
    sml[8 * 64 * half + 1] = l;
    __syncthreads();
    const float its = sml[8 * 64 * (1 - half)], top = fmaxf(ref, its), wa = __builtin_amdgcn_exp2f(ref - top), wb = __builtin_amdgcn_exp2f(its - top);
    ref = top;
    l = l * wa + sml[8 * 64 * (1 - half) + 1] * wb;
    columns([&](auto dt_c) __attribute__((always_inline)) {
      constexpr int dt = decltype(dt_c)::value;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const v4f x = so[64 * (4 * dt + g)];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[dt][4 * g + e] = o[dt][4 * g + e] * wa + x[e] * wb;
      }
    });
  }
  l += __shfl_xor(l, 32);
  if (j.parts > 1) {
    if (wrow0 + jr < j.rows) {
      const long long left = TREE ? j.left + in_rows + jr : r.at * a.cut.nparts + j.part;
      float* const po = a.part_o + left * D;
      columns([&](auto dt_c) __attribute__((always_inline)) {
        constexpr int dt = decltype(dt_c)::value;
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<v4f*>(po + 32 * dt + 8 * g + 4 * hh) = v4f{o[dt][4 * g], o[dt][4 * g + 1], o[dt][4 * g + 2], o[dt][4 * g + 3]};
      });
      if (hh == 0 && (!PAIRED || half == 0)) {
        float* const ml = a.part_ml + 2 * left;
        ml[0] = ref;
        ml[1] = l;
      }
    }
    return;
  }
  if (!PAIRED && idle) return;
  // the wave (PAIRED: two of them) turns its 32 x D tile round through LDS (nobody reads tiles any more) and stores whole rows
  const bool none = r.hi <= r.lo || (TREE && r.loose && l == 0.0f);
  const float inv = none ? 0.0f : 1.0f / l;
  unsigned char* const ot = smem + in_rows * S::ORS;
  columns([&](auto dt_c) __attribute__((always_inline)) {
    constexpr int dt = decltype(dt_c)::value;
#pragma unroll
    for (int e = 0; e < 16; ++e) o[dt][e] = finite_or_nan(o[dt][e]);
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<v2u*>(ot + jr * S::ORS + 2 * (32 * dt + 8 * g + 4 * hh)) =
          v2u{T::pack(o[dt][4 * g] * inv, o[dt][4 * g + 1] * inv), T::pack(o[dt][4 * g + 2] * inv, o[dt][4 * g + 3] * inv)};
  });
  if (a.lse && hh == 0 && wrow0 + jr < j.rows && (!PAIRED || half == 0)) a.lse[r.at] = none ? -INFINITY : log_sum(ref, l);
  if constexpr (PAIRED) __syncthreads();
  else asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  for (int idx = lane + (PAIRED ? 64 * half : 0); idx < 32 * CH; idx += PAIRED ? 128 : 64) {
    const int rw = idx / CH, c = idx - rw * CH;
    if (wrow0 + rw >= j.rows) break;
    const Row to = row_of<TREE>(a, j, kv_head, wrow0 + rw);
    *reinterpret_cast<v4u*>((unsigned char*)a.o + to.at * S::BYTES + 16 * c) = *reinterpret_cast<const v4u*>(ot + rw * S::ORS + 16 * c);
  }
}

// Trees: how the work of a kv head is shared out to `shares` workgroups, which the arrays on the device say alone.  The keys of the sequences that are not small, in
// grains and one sequence behind the other, are a line for each block of rows (the k-th line of those sequences that have more than k of them), and each
// workgroup has as many grains of one line, of one sequence or of several, whose block of rows it works on one after the other; a block of rows that more than one
// workgroup has is left in parts.  (16 sequences of 2064 to 8192 positions, 60 tokens each, 8 heads, e4m3: 133 us, 227 by a
// workgroup to a block of rows; 25 tokens 92 and 159.)
constexpr int kLeastGrains = 4;

// The sum of the lanes up to a lane's own, from register to register: a shuffle through LDS takes twenty times as long.
template <int DPP, int ROWS>
__device__ __forceinline__ int plus_moved(int x) {
  return x + __builtin_amdgcn_update_dpp(0, x, DPP, ROWS, 0xf, false);
}
__device__ __forceinline__ int wave_scan(int x) {
  x = plus_moved<0x111, 0xf>(x);                               // lanes 1, 2, 4 and 8 to the left in its row of 16
  x = plus_moved<0x112, 0xf>(x);
  x = plus_moved<0x114, 0xf>(x);
  x = plus_moved<0x118, 0xf>(x);
  x = plus_moved<0x142, 0xa>(x);                               // the last of the row before, into rows 1 and 3
  return plus_moved<0x143, 0xc>(x);                            // the last of the first half, into the second
}
__device__ __forceinline__ int wave_sum(int x) { return __builtin_amdgcn_readlane(wave_scan(x), 63); }

struct Shares {
  int each;                    // grains
  int grains, groups, before;  // lane k: of line k, the workgroups that have them, and those of the lines before
};

// Sequence i, a lane's own: its grains, and its blocks of rows.
__device__ __forceinline__ int share_work(const AttnArgs& a, int i, int* blocks) {
  *blocks = 0;
  if (i >= a.batch.sequences) return 0;
  const int start = min(max(a.batch.starts[i], 0), a.batch.tokens), end = a.batch.starts[i + 1], all = max(a.batch.lens[i], 0);
  const int rows = min(min(max(end, start), a.batch.tokens) - start, kTreeMost) * a.group;
  if (rows <= a.small_rows) return 0;
  *blocks = min((rows + (1 << a.block_shift) - 1) >> a.block_shift, a.row_blocks);
  const int keys = max(min(all, kv_capacity(a.batch, a.pages.page_shift)) - seq_first_key(a, first_position(all, start, end)), 1);
  return (int)(((long long)keys + (1LL << a.grain_shift) - 1) >> a.grain_shift);
}

// All lanes of a wave call these.
__device__ __forceinline__ Shares share_out(const AttnArgs& a) {
  const int lane = threadIdx.x & 63;
  Shares s{0, 0, 0, 0};
  for (int from = 0; from < a.batch.sequences; from += 64) {
    int blocks;
    const int grains = share_work(a, from + lane, &blocks);
    for (int k = 0; k < a.row_blocks; ++k) {
      const int sum = wave_sum(blocks > k ? grains : 0);
      if (lane == k) s.grains += sum;
    }
  }
  s.each = max((int)(((unsigned)wave_sum(s.grains) + a.shares - 1) / (unsigned)a.shares), kLeastGrains);
  for (;;) {                                                   // (it ends: there are as many shares as lines at least)
    s.groups = (int)(((unsigned)s.grains + s.each - 1) / (unsigned)s.each);
    const int before = wave_scan(s.groups);
    s.before = before - s.groups;
    if (__builtin_amdgcn_readlane(before, 63) <= a.shares) break;
    s.each += s.each / 32 + 1;
  }
  return s;
}
// Which workgroup of which line the w-th is: lines have no more of them than those before, and the same one of all lines, which read the same keys, go together.
__device__ __forceinline__ bool share_of(const AttnArgs& a, const Shares& s, int w, int* line, int* at) {
  int done = 0;
  for (int k = a.row_blocks; k > 0; --k) {
    const int groups = __builtin_amdgcn_readlane(s.groups, k - 1), here = (groups - done) * k;
    if (w < here) {
      *at = done + (int)((unsigned)w / (unsigned)k);
      *line = (int)((unsigned)w % (unsigned)k);
      return true;
    }
    w -= here;
    done = groups;
  }
  return false;
}
// The sequence that has grain x of a line, or (seek >= 0) sequence `seek` itself; where it begins there, and how many it has.
__device__ __forceinline__ int share_find(const AttnArgs& a, int line, int x, int seek, int* begin, int* grains) {
  const int lane = threadIdx.x & 63;
  int base = 0;
  for (int from = 0; from < a.batch.sequences; from += 64) {
    int blocks;
    int mine = share_work(a, from + lane, &blocks);
    if (blocks <= line) mine = 0;
    const int upto = base + wave_scan(mine);
    const unsigned long long here = __builtin_amdgcn_ballot_w64(seek >= 0 ? from + lane == seek : mine > 0 && x < upto);
    if (here) {
      const int l = (int)__builtin_ctzll(here);
      *grains = __builtin_amdgcn_readlane(mine, l);
      *begin = __builtin_amdgcn_readlane(upto, l) - *grains;
      return from + l;
    }
    base = __builtin_amdgcn_readlane(upto, 63);
  }
  return -1;
}

// Grains [from, to) of `grains` of sequence b for a line's block of rows.
__device__ __forceinline__ void share_job(const AttnArgs& a, int b, int line, int from, int to, int grains, Job& j) {
  j.b = b;
  const KvChunk c = kv_chunk(a.batch, b);
  j.start = c.start;
  j.n = min(c.n, kTreeMost);
  j.first = c.first;
  j.rows = j.n * a.group;
  j.row0 = line << a.block_shift;
  j.len = min(c.len, kv_capacity(a.batch, a.pages.page_shift));
  const long long p_hi = (long long)c.first + (min(j.row0 + (1 << a.block_shift), j.rows) - 1) / a.group, key0 = seq_first_key(a, c.first);
  j.hi = clamp_position(p_hi + 1, j.len);
  j.sure_hi = clamp_position(c.first, j.len);
  j.lo = a.window > 0 ? clamp_position((long long)c.first - a.window + 1, j.len) : 0;
  j.sure_lo = a.window > 0 ? clamp_position(p_hi - a.window + 1, j.len) : 0;
  if (from > 0) j.lo = max(j.lo, clamp_position(key0 + ((long long)from << a.grain_shift), j.len));
  if (to < grains) j.hi = min(j.hi, clamp_position(key0 + ((long long)to << a.grain_shift), j.len));
  j.part = 0;
  j.parts = from > 0 || to < grains ? 2 : 1;
  j.small = false;
}

// The workgroups behind the first `wide` take sequences of at most small_rows = 16 rows, which would leave seven of the eight waves without
// any: two (sequence, head, part) each, by four waves that cut the keys as in the narrow kernel.  They read on the compute units that the others
// leave free, or have left, while those multiply.  (A chunk of 512 tokens beside five sequences that decode, 16 heads, 4 of keys, up to
// 16384 of them, in int8: 165 us with all on the wide form, 108 so, and 12 for joining.)
template <typename T, KvFormat F, int D, bool TREE, bool PAIRED>
__global__ __launch_bounds__(kWideWaves * 64, 1) void paged_wide_kernel(AttnArgs a, int wide) {
  constexpr int R = WideShape<D, TREE, PAIRED>::ROWS;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  Job j;
  if constexpr (!TREE) {
    if ((int)blockIdx.x >= wide) {
      const int half = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
      const int item = 2 * (blockIdx.x - wide) + half, kv_head = item % a.pages.heads, rest = item / a.pages.heads;
      const int b = rest / a.small.nparts, part = rest - b * a.small.nparts;
      if (b < a.batch.sequences && find_job<16, false>(a, b, 0, part, true, j)) {
        narrow_attention<T, F, D, 1, false, false>(a, j, kv_head, smem + half * NarrowShape<F, D>::LDS, threadIdx.x & 255);
      } else {                                                     // the other half's two barriers
        __syncthreads();
        __syncthreads();
      }
      return;
    }
  }
  // the head goes fastest, so that the row blocks of a head meet on the XCDs that have its keys
  const int id = blockIdx.x, kv_head = id % a.pages.heads, rest = id / a.pages.heads;
  if constexpr (TREE) {
    const bool shared = a.shares > 0;
    Shares s{1, 0, 0, 0};
    int line = 0, at = 0, x0 = 0, x = 0, end = 1;
    if (shared) {
      s = share_out(a);
      if (!share_of(a, s, rest, &line, &at)) return;
      x = x0 = at * s.each;
      end = min(x0 + s.each, __builtin_amdgcn_readlane(s.grains, line));
    }
    const long long slot = ((long long)(__builtin_amdgcn_readlane(s.before, line) + at) * a.pages.heads + kv_head) * 2;
    while (x < end) {
      int b, tile, begin, grains;
      if (shared) {
        b = share_find(a, line, x, -1, &begin, &grains);
        if (b < 0) return;
        const int to = min(end - begin, grains);
        share_job(a, __builtin_amdgcn_readfirstlane(b), line, x - begin, to, grains, j);
        j.left = (slot + (x > x0)) * R;
        x = begin + to;
      } else {
        if (!find_rows<R>(a, rest, &b, &tile) || !find_job<R, TREE>(a, b, tile, 0, false, j)) return;
        x = end;
      }
      if (j.rows <= kNarrowRows) wide_attention<T, F, D, TREE, PAIRED, true>(a, j, kv_head, smem);
      else wide_attention<T, F, D, TREE, PAIRED, false>(a, j, kv_head, smem);
      if (x < end) __syncthreads();
    }
  } else {
    const int slot = rest / a.cut.nparts, part = rest - slot * a.cut.nparts;
    int b, tile;
    if (!find_rows<R>(a, slot, &b, &tile) || !find_job<R, TREE>(a, b, tile, part, false, j)) return;
    wide_attention<T, F, D, TREE, PAIRED, false>(a, j, kv_head, smem);
  }
}

// ---- parts ------------------------------------------------------------------------------

// The parts of the sequence that row `at` of the packed rows times heads belongs to (1: nothing to join), the first of them, and the keys [*lo, *hi) that the row
// sees.  first_token: that of the wave's first lane.
__device__ __forceinline__ int row_parts(const AttnArgs& a, long long at, int first_token, int* lo, int* hi, long long* first_of) {
  const int token = (int)(at / a.heads), head = (int)(at - (long long)token * a.heads);
  int b = count_at_most(a.batch.sequences, first_token, [&](int k) { return a.batch.starts[k + 1]; });
  while (b < a.batch.sequences && a.batch.starts[b + 1] <= token) ++b;
  if (b >= a.batch.sequences) return 1;
  const int start = min(max(a.batch.starts[b], 0), a.batch.tokens), end = min(max(a.batch.starts[b + 1], start), a.batch.tokens);
  if (token < start || token >= end) return 1;
  const int all = max(a.batch.lens[b], 0), first = first_position(all, start, a.batch.starts[b + 1]), len = min(all, kv_capacity(a.batch, a.pages.page_shift));
  const long long position = (long long)first + (token - start);
  *hi = a.causal ? clamp_position(position + 1, len) : len;
  *lo = a.window > 0 ? clamp_position(position - a.window + 1, len) : 0;
  const int kv_head = head / a.group;
  const bool small = (end - start) * a.group <= a.small_rows;
  *first_of = first_part(a, small, b, kv_head, (token - start) * a.group + head - kv_head * a.group, at);
  return seq_parts(a, small ? a.small : a.cut, first, len);
}

// m = max m_p, l = sum l_p 2^(m_p - m), O = sum O_p 2^(m_p - m) / l over the parts of a row.  A wave (WAVES = 4: the four of a block) to a row: the
// weights 2^(m_p - m) first, a lane a part, then the sums of O, D / 4 lanes a part, by loads that do not wait for one another.  A wave is given `rows` rows: one, or
// many where only small sequences are cut and most waves find nothing to do.
template <typename T, int D, int WAVES>
__global__ __launch_bounds__(256) void paged_merge_kernel(AttnArgs a, int rows) {
  constexpr int L = D / 4, SL = 64 / L, K = kPartsMost / 64;    // lanes of a part, parts of a wave at once
  constexpr int TURN = SL * WAVES, PRE = WAVES == 4 ? kPartsMost / TURN : std::min(8, 64 / TURN);    // parts at once; turns whose loads go out first
  __shared__ v4f so[WAVES == 4 ? 4 * L : 1];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, slice = lane / L, c = lane - slice * L;
  const int mine = (WAVES == 4 ? wave * SL : 0) + slice;
  const long long all_rows = (long long)a.batch.tokens * a.heads;
  const long long row0 = ((long long)blockIdx.x * (WAVES == 4 ? 1 : 4) + (WAVES == 4 ? 0 : wave)) * rows;
  if (row0 >= all_rows) return;
  int lo = 0, hi = 0;
  long long first = 0;
  const int parts = row_parts(a, min(row0 + min(lane, rows - 1), all_rows - 1), __builtin_amdgcn_readfirstlane((int)(row0 / a.heads)), &lo, &hi, &first);
  unsigned long long todo = __builtin_amdgcn_ballot_w64(lane < rows && row0 + lane < all_rows && parts > 1);
  while (todo) {
    const int r = (int)__builtin_ctzll(todo);
    todo &= todo - 1;
    const long long at = row0 + r;
    const int n = __builtin_amdgcn_readlane(parts, r);
    const bool none = __builtin_amdgcn_readlane(hi, r) <= __builtin_amdgcn_readlane(lo, r);
    const long long part0 = (long long)(((unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)(first >> 32), r) << 32) |
                                        (unsigned)__builtin_amdgcn_readlane((int)first, r));
    const float* const ml = a.part_ml + 2 * part0;
    // the first PRE turns' sums are asked for beside (m, l): all of them where four waves share a row
    const float* const po = a.part_o + part0 * D + 4 * c;
    v4f early[PRE];
#pragma unroll
    for (int i = 0; i < PRE; ++i) {
      const int p = i * TURN + mine;
      early[i] = p < n && slice < SL ? *reinterpret_cast<const v4f*>(po + (size_t)p * D) : v4f{0.f, 0.f, 0.f, 0.f};
    }
    float m[K], w[K], top = kNoRef, sum = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int p = 64 * k + lane;
      m[k] = p < n ? ml[2 * p] : kNoRef;
      w[k] = p < n ? ml[2 * p + 1] : 0.0f;
      top = fmaxf(top, m[k]);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const float e = __builtin_amdgcn_exp2f(m[k] - top);
      sum += e * w[k];
      w[k] = e;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    v4f acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < PRE; ++i) {
      const float weight = __shfl(w[i * TURN / 64], (i * TURN + mine) & 63);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += weight * early[i][e];
    }
    if constexpr (WAVES == 1) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int last = min(n - 64 * k, 64);
#pragma unroll 4
        for (int p0 = k == 0 ? PRE * TURN : 0; p0 < last; p0 += TURN) {
          const int p = p0 + slice;
          const float weight = __shfl(w[k], p & 63);
          if (p < last && slice < SL) {
            const v4f v = *reinterpret_cast<const v4f*>(po + (size_t)(64 * k + p) * D);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] += weight * v[e];
          }
        }
      }
    }
#pragma unroll
    for (int o = SL / 2; o > 0; o >>= 1)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += __shfl(acc[e], lane + o * L);
    if constexpr (WAVES == 4) {
      if (lane < L) so[wave * L + lane] = acc;
      __syncthreads();
      if (wave == 0 && lane < L) {
#pragma unroll
        for (int i = 1; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[e] += so[i * L + lane][e];
      }
    }
    if ((WAVES == 1 || wave == 0) && lane < L) {
      const float inv = none ? 0.0f : 1.0f / sum;
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = finite_or_nan(acc[e]);
      *reinterpret_cast<v2u*>((typename T::scalar*)a.o + at * D + 4 * c) = v2u{T::pack(acc[0] * inv, acc[1] * inv), T::pack(acc[2] * inv, acc[3] * inv)};
      if (a.lse && lane == 0) a.lse[at] = none ? -INFINITY : log_sum(top, sum);
    }
  }
}

// The same for trees: a wave has ROWS heads of a token.  Lanes have columns, so that a part's weight is the same for all of them.  Rows in at most four parts, which most
// are where there are many, are joined at once, everything of theirs being asked for before any of it is needed; others one after the other, their
// weights a lane each.  (25 tokens, 32 heads, 32 parts: 7 us, 19 by the kernel above.)
template <typename T, int D, int ROWS>
__global__ __launch_bounds__(256) void tree_join_kernel(AttnArgs a) {
  constexpr int VEC = D > 64 ? 2 : 1, TURN = 16, K = kPartsMost / 64, FEW = 4;
  typedef float vec __attribute__((ext_vector_type(VEC)));
  typedef float v2f __attribute__((ext_vector_type(2)));
  const int lane = threadIdx.x & 63;
  const int chunks = (a.heads + ROWS - 1) / ROWS, unit = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  const int token = unit / chunks, head0 = (unit - token * chunks) * ROWS;
  if (token >= a.batch.tokens) return;
  // the sequence, and what it says of the token
  int start = 0, place = 0, all = 0, b = -1;
  for (int from = 0; from < a.batch.sequences && b < 0; from += 64) {
    const int i = min(from + lane, a.batch.sequences - 1), s0 = a.batch.starts[i], s1 = a.batch.starts[i + 1], n = a.batch.lens[i];
    const unsigned long long here = __builtin_amdgcn_ballot_w64(from + lane < a.batch.sequences && max(s0, 0) <= token && token < s1);
    if (here) {
      const int l = (int)__builtin_ctzll(here);
      b = from + l;
      start = max(__builtin_amdgcn_readlane(s0, l), 0);
      place = __builtin_amdgcn_readlane(s1, l);
      all = max(__builtin_amdgcn_readlane(n, l), 0);
    }
  }
  if (b < 0 || token - start >= kTreeMost) return;
  const int first = first_position(all, start, place), len = min(all, kv_capacity(a.batch, a.pages.page_shift));
  const long long position = (long long)first + (token - start);
  const int hi = clamp_position(position + 1, len), lo = a.window > 0 ? clamp_position((long long)first - a.window + 1, len) : 0;
  const bool some = hi > lo, loose = position >= len;
  Shares s{0, 0, 0, 0};
  if (a.shares > 0) s = share_out(a);
  // where the first part of each row is, the second, and how far those behind are from one another
  int n[ROWS], line = -1, parts = 1, after = 0, kv_head = (int)((unsigned)head0 / (unsigned)a.group), in_group = head0 - kv_head * a.group;
  long long part0[ROWS], part1[ROWS], slot = 0;
  const long long step = a.shares > 0 ? 2LL * a.pages.heads << a.block_shift : 1;
  const int own_parts = a.shares > 0 ? 1 : seq_parts(a, a.cut, first, len);
  bool few = true;
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    if (a.shares == 0) {
      n[r] = own_parts;
      part0[r] = ((long long)token * a.heads + min(head0 + r, a.heads - 1)) * a.cut.nparts;
      part1[r] = part0[r] + 1;
    } else {
      const int row = (token - start) * a.group + in_group, in_block = row & ((1 << a.block_shift) - 1);
      if (line != row >> a.block_shift) {
        line = row >> a.block_shift;
        if (line >= a.row_blocks) return;
        int begin, grains;
        share_find(a, line, 0, b, &begin, &grains);
        const int group0 = (int)((unsigned)begin / (unsigned)s.each);
        parts = (int)((unsigned)(begin + max(grains, 1) - 1) / (unsigned)s.each) - group0 + 1;
        after = begin > group0 * s.each;
        slot = (long long)(__builtin_amdgcn_readlane(s.before, line) + group0) * a.pages.heads * 2;
      }
      n[r] = parts;
      part1[r] = ((slot + 2 * kv_head) << a.block_shift) + in_block + step;
      part0[r] = part1[r] - step + ((long long)after << a.block_shift);
    }
    few = few && n[r] <= FEW;
    if (head0 + r + 1 < a.heads && ++in_group == a.group) {
      in_group = 0;
      ++kv_head;
    }
  }
  const int col = min(lane * VEC, D - VEC);
  const float* const po = a.part_o + col;
  const auto finish = [&](int head, vec acc, float top, float sum) __attribute__((always_inline)) {
    const long long at = (long long)token * a.heads + head;
    const bool none = !some || (loose && sum == 0.0f);
    const float inv = none ? 0.0f : 1.0f / sum;
    if (lane * VEC < D) {
      typename T::scalar* const o = (typename T::scalar*)a.o + at * D + col;
      const unsigned pair = T::pack(finite_or_nan(acc[0]) * inv, finite_or_nan(acc[VEC - 1]) * inv);
      if constexpr (VEC == 2) *reinterpret_cast<unsigned*>(o) = pair;
      else *reinterpret_cast<unsigned short*>(o) = (unsigned short)pair;
    }
    if (a.lse && lane == 0) a.lse[at] = none ? -INFINITY : log_sum(top, sum);
  };
  if (few) {
    vec x[ROWS][FEW];
    v2f ml[ROWS][FEW];
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int p = 0; p < FEW; ++p) {
        if (n[r] <= 1 || p >= n[r]) continue;
        const long long at = p == 0 ? part0[r] : part1[r] + (p - 1) * step;
        ml[r][p] = *reinterpret_cast<const v2f*>(a.part_ml + 2 * at);
        x[r][p] = *reinterpret_cast<const vec*>(po + at * D);
      }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      if (n[r] <= 1 || head0 + r >= a.heads) continue;
      float top = kNoRef, sum = 0.0f;
      vec acc = 0.0f;
#pragma unroll
      for (int p = 0; p < FEW; ++p)
        if (p < n[r]) top = fmaxf(top, ml[r][p][0]);
#pragma unroll
      for (int p = 0; p < FEW; ++p) {
        if (p >= n[r]) continue;
        const float w = __builtin_amdgcn_exp2f(ml[r][p][0] - top);
        sum += w * ml[r][p][1];
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] += w * x[r][p][e];
      }
      finish(head0 + r, acc, top, sum);
    }
    return;
  }
#pragma unroll 1
  for (int r = 0; r < ROWS; ++r) {
    int count = n[0];
    long long at0 = part0[0], at1 = part1[0];
#pragma unroll
    for (int i = 1; i < ROWS; ++i)
      if (r == i) {
        count = n[i];
        at0 = part0[i];
        at1 = part1[i];
      }
    if (count <= 1 || head0 + r >= a.heads) continue;
    const auto part_at = [&](int p) { return p == 0 ? at0 : at1 + (p - 1) * step; };
    vec x[TURN];
#pragma unroll
    for (int i = 0; i < TURN; ++i) x[i] = *reinterpret_cast<const vec*>(po + part_at(min(i, count - 1)) * D);
    float m[K], w[K], top = kNoRef, sum = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int p = 64 * k + lane;
      const v2f ml = *reinterpret_cast<const v2f*>(a.part_ml + 2 * part_at(min(p, count - 1)));
      m[k] = p < count ? ml[0] : kNoRef;
      w[k] = p < count ? ml[1] : 0.0f;
      top = fmaxf(top, m[k]);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const float e = __builtin_amdgcn_exp2f(m[k] - top);
      sum += e * w[k];
      w[k] = e;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    vec acc = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll 1
      for (int p0 = 0; p0 < min(count - 64 * k, 64); p0 += TURN) {
        if (k + p0 > 0) {
#pragma unroll
          for (int i = 0; i < TURN; ++i) x[i] = *reinterpret_cast<const vec*>(po + part_at(min(64 * k + p0 + i, count - 1)) * D);
        }
#pragma unroll
        for (int i = 0; i < TURN; ++i) {
          const float weight = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w[k]), p0 + i));
          if (64 * k + p0 + i < count) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[e] += weight * x[i][e];
          }
        }
      }
    }
    finish(head0 + r, acc, top, sum);
  }
}

// ---- host side ----------------------------------------------------------------------------

// How a call is run.
struct Plan {
  bool narrow;
  int nq;                  // narrow: blocks of 16 rows of a workgroup, 1 or 2
  int slots, slots_per_seq;
  Cut cut, small;
  int small_rows;
  size_t large, all;       // parts that there is room for: of sequences that are not small, and with those that are
  int shares, grain_shift, block_rows; // trees, wide
};

static size_t parts_of(long long rows, int nparts) { return nparts > 1 ? (size_t)rows * nparts : 0; }
static size_t workspace_of(size_t parts, int D) { return parts * (D + 2) * 4; }

// us of a launch of the narrow kernel: rounds of two workgroups to a compute unit, 3 us each until the first tile is there, and their share of 5.8 TB/s, or
// the 17 KB a us that one workgroup gets through.  The lengths of several sequences are not known here, only the greatest: the mean of that with all of them alike
// and that with two thirds of the work, where workgroups follow one another as they end and no round is waited for.  (Five tokens each of 16 sequences
// of up to 4096 keys: 31 us with three parts, as all alike would have it, 26 with four.)
static double narrow_cost(double workgroups, int part_keys, int held, int cus, bool alike) {
  const double at_once = std::min(workgroups, 2.0 * cus), rounds = std::ceil(workgroups / (2.0 * cus)), kb = part_keys * (held / 1000.0);
  const double same = rounds * (3.0 + kb / std::min(17.0, 5800.0 / at_once));
  return alike ? same : 0.5 * (same + 3.0 + std::max(workgroups * kb * (2.0 / 3) / 5800.0, kb / 17.0));
}

// The same of the wide kernel: rounds of one workgroup to a compute unit, which takes 2 us for a tile of 64 keys of 128; then what is left of `small` us of
// other workgroups when these have filled the last round.
static double wide_cost(double workgroups, double part_keys, int D, int cus, double small) {
  const double each = 6.0 + part_keys / 64 * (2.0 * D / 128), rounds = std::ceil(workgroups / cus);
  return rounds * each + std::max(0.0, small - (rounds * cus - workgroups) * each) / cus;
}

// Leaving parts and joining them: a launch, and fp32 sums written and read at 4 TB/s.
static double join_cost(double rows, int D, int nparts) { return nparts > 1 ? 5.0 + rows * nparts * D * 8 / 4e6 : 0.0; }

static Cut cut_into(int keys, long long n) {
  Cut c;
  c.part_keys = (int)(((keys + n - 1) / n + 127) / 128 * 128);
  c.nparts = std::max(1, (keys + c.part_keys - 1) / c.part_keys);
  return c;
}

// The number of parts that cost() finds cheapest by 3 %, among those whose results have room.
template <typename C>
static Cut best_cut(int keys, int least_keys, long long rows, int D, size_t room, C&& cost) {
  Cut best = cut_into(keys, 1);
  double least = cost(best);
  for (int n = 2; n <= kPartsMost; n += n < 4 ? 1 : n / 4) {
    const Cut c = cut_into(keys, n);
    if (c.part_keys < least_keys || workspace_of(parts_of(rows, c.nparts), D) > room) break;
    const double t = cost(c);
    if (t < 0.97 * least) {
      least = t;
      best = c;
    }
  }
  return best;
}

static Plan plan(const ftk_kv_pages& pages, const KvBatch& b, int page_shift, int heads, int window, int max_queries, int max_keys, int cus, size_t room, bool tree) {
  const int D = pages.head_size, group = heads / pages.heads;
  Plan p;
  const long long most = max_queries > 0 ? std::min(max_queries, b.tokens) : b.tokens;   // new tokens of a sequence
  const long long most_rows = most * group, rows = (long long)b.tokens * heads;
  p.narrow = most_rows <= (tree ? kSmallRows : kNarrowRows);
  const long long capacity = (long long)b.width << page_shift;
  long long seen = max_keys > 0 ? std::min<long long>(max_keys, capacity) : capacity;
  if (window > 0) seen = std::min(seen, most + window + 64);   // from the first key that the first new token sees, down to a multiple of 64
  const int keys = (int)std::min<long long>(seen, INT_MAX - 1024);
  // 32 rows to a narrow workgroup read the keys half as often as 16; those are the faster ones where even parts of 256 keys are fewer than the compute
  // units.  (16 sequences of up to 4096 keys, 8 heads of them, 20 rows: 48 us by 32 rows and 54 by 16 at D 128, int8 46 and 48, 25 and 28 at D 64; 48 rows: 65 and 67, int8 69 and 71, but
  // 38 and 34 at D 64; two sequences of up to 1000 keys, 48 rows: 15 and 12.)
  p.nq = most_rows <= 16 || (p.narrow && ((most_rows + 31) / 32) * b.sequences * pages.heads * ((keys + 255) / 256) < cus) ? 1 : 2;
  p.block_rows = most_rows <= kPairedRows ? kPairedRows : kWideRows;
  const int R = p.narrow ? 16 * p.nq : tree ? p.block_rows : kWideRows;
  const long long per_seq = (most_rows + R - 1) / R, packed = (long long)b.tokens * group / R + b.sequences;
  // numbered by row blocks, unless most of such slots would be empty (as those of narrow workgroups, four to a sequence at most, cannot be)
  p.slots_per_seq = p.narrow || b.sequences * per_seq <= 2 * packed ? (int)per_seq : 0;
  p.slots = (int)std::min<long long>(p.slots_per_seq ? b.sequences * per_seq : packed, INT_MAX);
  p.small_rows = p.narrow || tree || b.sequences == 1 ? 0 : kSmallRows;
  const int held = pages.type == FTK_F16 || pages.type == FTK_BF16 ? 4 * D : 2 * D + 2;   // bytes of a position and head
  const long long small_rows = (long long)b.sequences * pages.heads * kSmallRows;
  p.small = Cut{1, keys};
  p.shares = 0;
  p.grain_shift = 7;
  if (p.narrow) {
    const double units = (double)p.slots * pages.heads;
    p.cut = best_cut(keys, 256, rows, D, room, [&](const Cut& c) { return narrow_cost(units * c.nparts, c.part_keys, held, cus, b.sequences == 1) + join_cost(rows, D, c.nparts); });
  } else if (tree) {
    // Work shared out, unless a workgroup for each block of rows is expected to be done sooner: us as in wide_cost(), several sequences being two thirds as long as
    // the longest in the mean.
    const double turn = (p.block_rows == kPairedRows ? 2.4 : 4.0) * D / 128, turns = std::ceil(keys / 128.0), units = (double)b.sequences * per_seq * pages.heads;
    const double whole = std::ceil(units / cus) * (8.0 + turns * turn);
    p.cut = cut_into(keys, 1);
    const TreeShares s = share_trees(b.sequences, per_seq, pages.heads, capacity, cus);
    p.grain_shift = s.grain_shift;
    const double rounds = std::ceil((double)s.shares * pages.heads / cus);
    const double shared = 18.0 + rounds * 6.0 + std::max(units * turns * (b.sequences > 1 ? 2.0 / 3 : 1.0) / ((double)s.shares * pages.heads), (double)kLeastGrains) * turn * rounds;
    const size_t parts = (size_t)s.shares * pages.heads * 2 * p.block_rows;
    if (s.shares > 0 && shared < whole && workspace_of(parts, D) <= room) {
      p.shares = s.shares;
      p.slots = p.shares;
      p.large = parts;
      p.all = parts;
      return p;
    }
    p.large = p.all = 0;
    return p;
  } else {
    // the small sequences: as many as there can be beside ones of `most` tokens, in parts of some 20 us
    double small = 0.0;
    if (p.small_rows > 0) {
      p.small = cut_into(keys, std::min({std::max(1, (int)((long long)keys * held / (20 * 17000))), keys / 256 + 1, kPartsMost}));
      while (p.small.nparts > 1 && workspace_of(parts_of(small_rows, p.small.nparts), D) > room) p.small = cut_into(keys, p.small.nparts - 1);
      room -= workspace_of(parts_of(small_rows, p.small.nparts), D);
      const double sequences = std::max(0.0, b.sequences - std::ceil((double)(b.tokens - b.sequences) / std::max(1LL, most - 1)));
      small = sequences * pages.heads * p.small.nparts / 2 * (3.0 + p.small.part_keys * (held / 17000.0));
    }
    // whole row blocks; a chunk that sees itself under a causal mask works on half of its own keys
    const double units = (double)std::max<long long>(1, b.tokens * (long long)group / R) * pages.heads, own = std::min<double>(most, keys) / 2;
    p.cut = best_cut(keys, 512, rows, D, room,
                     [&](const Cut& c) { return wide_cost(units * c.nparts, c.part_keys * (1 - own / keys), D, cus, small) + join_cost(rows, D, c.nparts); });
  }
  p.large = parts_of(rows, p.cut.nparts);
  p.all = p.large + parts_of(small_rows, p.small.nparts);
  return p;
}

static int check_attention(const char* who, int heads, const ftk_kv_pages* pages) {
  if (heads <= 0 || heads % pages->heads) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: query heads must be a multiple of the kv heads, got %d and %d", who, heads, pages->heads);
  return FTK_OK;
}

template <typename K, typename... Args>
static int launch_with_lds(const char* who, const char* name, K kernel, DeviceOnce& once, long long blocks, int waves, int lds, hipStream_t s, Args... args) {
  if (blocks > INT_MAX) return fail(FTK_ERR_UNSUPPORTED_SHAPE, "%s: grid too large", who);
  unsigned bit;
  if (once.pending(&bit)) {
    FTK_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    once.done(bit);
  }
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(waves * 64), lds, s, args...);
  return check_launch(name);
}

// A sequence's new tokens at most.
static int most_tokens(int max_queries, int tokens) { return max_queries > 0 ? std::min(max_queries, tokens) : tokens; }

static size_t attend_workspace_bytes(const ftk_kv_pages* pages, const ftk_kv_batch* batch, int heads, int window, int max_queries, int max_keys, bool tree) {
  const DeviceProps* d = nullptr;
  if (!pages || !batch || pages->heads <= 0 || heads <= 0 || heads % pages->heads || batch->tokens <= 0 || batch->sequences <= 0 || batch->table_width <= 0 ||
      pages->page_size <= 0 || window < 0 || (tree && most_tokens(max_queries, batch->tokens) > kTreeMost) || device_props(&d))
    return 0;
  KvBatch b{};
  b.tokens = batch->tokens;
  b.sequences = batch->sequences;
  b.width = batch->table_width;
  const Plan p = plan(*pages, b, __builtin_ctz((unsigned)pages->page_size), heads, window, max_queries, max_keys, d->cus, SIZE_MAX, tree);
  return workspace_of(p.all, pages->head_size);
}

template <bool TREE>
static int attend(const char* who, const void* q, int type, long long q_token_stride, long long q_head_stride, const ftk_kv_pages* pages, const ftk_kv_batch* batch,
                  const int* parents, void* o, float* lse, int heads, float scale, int causal, int window, int max_queries, int max_keys, void* workspace,
                   size_t workspace_bytes, ftk_stream_t stream) {
  AttnArgs a;
  int rc = check_kv_pages(who, pages, &a.pages);
  if (rc || (rc = check_kv_batch(who, batch, &a.batch)) || (rc = check_attention(who, heads, pages))) return rc;
  if (type != FTK_F16 && type != FTK_BF16) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: queries must be fp16 or bf16", who);
  if ((pages->type == FTK_F16 || pages->type == FTK_BF16) && pages->type != type) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: pages of 16 bits must have the type of the queries", who);
  if (!(scale > 0.0f) || !(scale * 1.4426950408889634f <= FLT_MAX)) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: scale must be positive, and its product with log2(e) finite", who);
  if (window < 0 || max_queries < 0 || max_keys < 0) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: window, max_queries and max_keys must not be negative", who);
  if (a.batch.tokens == 0) return FTK_OK;
  if constexpr (TREE) {
    if (!parents || ((uintptr_t)parents & 3)) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: parents must be non-NULL and 4-byte aligned", who);
    const int most = most_tokens(max_queries, a.batch.tokens);
    if (most > kTreeMost) return fail(FTK_ERR_UNSUPPORTED_SHAPE, "%s: trees of at most %d tokens, max_queries says how many there may be, got %d", who, kTreeMost, most);
  }
  if (!q || !o || !aligned16(q) || !aligned16(o)) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: q and o must be non-NULL and 16-byte aligned", who);
  if ((uintptr_t)lse & 3) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: lse must be 4-byte aligned", who);
  if (q_token_stride < 0 || q_head_stride < 0 || q_token_stride % 8 || q_head_stride % 8) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: strides must be multiples of 8 elements", who);
  if ((long long)a.batch.tokens * (heads / pages->heads) > INT_MAX / 2) return fail(FTK_ERR_UNSUPPORTED_SHAPE, "%s: too many rows", who);
  const DeviceProps* d = nullptr;
  if ((rc = device_props(&d))) return rc;
  if (workspace && !aligned16(workspace)) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: the workspace must be 16-byte aligned", who);
  const Plan p = plan(*pages, a.batch, a.pages.page_shift, heads, window, max_queries, max_keys, d->cus, workspace ? workspace_bytes : 0, TREE);
  a.q = q;
  a.o = o;
  a.lse = lse;
  a.q_token = q_token_stride;
  a.q_head = q_head_stride;
  a.heads = heads;
  a.group = heads / pages->heads;
  a.scale_log2e = scale * 1.4426950408889634f;
  a.causal = causal != 0;
  a.window = window;
  a.slots = p.slots;
  a.slots_per_seq = p.slots_per_seq;
  a.cut = p.cut;
  a.small = p.small;
  a.small_rows = p.small_rows;
  a.small_first = (long long)p.large;
  a.shares = p.shares;
  a.grain_shift = p.grain_shift;
  a.block_shift = __builtin_ctz((unsigned)p.block_rows);
  a.row_blocks = p.narrow ? 0 : (int)((most_tokens(max_queries, a.batch.tokens) * (long long)a.group + p.block_rows - 1) / p.block_rows);
  const long long rows = (long long)a.batch.tokens * heads;
  a.part_o = (float*)workspace;
  a.part_ml = a.part_o + p.all * pages->head_size;
  a.parents = parents;
  const long long blocks = (long long)p.slots * pages->heads * p.cut.nparts;
  const long long pairs = p.small_rows ? ((long long)a.batch.sequences * pages->heads * p.small.nparts + 1) / 2 : 0;
  const hipStream_t s = (hipStream_t)stream;
  return with_kv_types(type, pages->type, pages->head_size, [&](auto t, auto f, auto dc) -> int {
    using T = decltype(t);
    constexpr KvFormat F = decltype(f)::value;
    constexpr int D = decltype(dc)::value;
    int bad;
    if (p.narrow) {
      using yes = std::true_type;
      using no = std::false_type;
      auto launch = [&](auto nq, auto kept) -> int {
        static DeviceOnce once;
        return launch_with_lds(who, "paged_narrow_kernel", paged_narrow_kernel<T, F, D, decltype(nq)::value, decltype(kept)::value, TREE>, once, blocks, kWaves, NarrowShape<F, D>::LDS, s,
                               a, p.slots_per_seq);
      };
      if constexpr (TREE) {                                      // (one block of 16 rows to a sequence and head)
        bad = launch(std::integral_constant<int, 1>{}, no{});
      } else {
        auto with_kept = [&](auto nq) { return p.slots_per_seq == 1 ? launch(nq, no{}) : launch(nq, yes{}); };
        bad = p.nq == 2 ? with_kept(std::integral_constant<int, 2>{}) : with_kept(std::integral_constant<int, 1>{});
      }
    } else {
      auto launch = [&](auto paired) -> int {
        static DeviceOnce once;
        constexpr bool PAIRED = decltype(paired)::value;
        constexpr int lds = std::max(WideShape<D, TREE, PAIRED>::LDS, TREE ? 0 : 2 * NarrowShape<F, D>::LDS);
        return launch_with_lds(who, "paged_wide_kernel", paged_wide_kernel<T, F, D, TREE, PAIRED>, once, blocks + pairs, kWideWaves, lds, s, a, (int)blocks);
      };
      if constexpr (TREE) bad = p.block_rows == kPairedRows ? launch(std::true_type{}) : launch(std::false_type{});
      else bad = launch(std::false_type{});
    }
    if (bad || p.all == 0) return bad;
    if constexpr (TREE) {
      // a wave to a row while the compute units have room for all of them
      auto join = [&](auto each) -> int {
        constexpr int ROWS = decltype(each)::value;
        const long long jblocks = ((long long)a.batch.tokens * ((heads + ROWS - 1) / ROWS) + 3) / 4;
        if (jblocks > INT_MAX / 4) return fail(FTK_ERR_UNSUPPORTED_SHAPE, "%s: grid too large", who);
        hipLaunchKernelGGL((tree_join_kernel<T, D, ROWS>), dim3((unsigned)jblocks), dim3(256), 0, s, a);
        return FTK_OK;
      };
      if ((bad = rows <= 16 * d->cus ? join(std::integral_constant<int, 1>{}) : join(std::integral_constant<int, 4>{}))) return bad;
      return check_launch("tree_join_kernel");
    } else {
      // few rows of many parts: a block to each; only small sequences cut: 16 rows to a wave, most of which have nothing to join
      if (rows <= 4096 && std::max(p.cut.nparts, p.small.nparts) >= 16) {
        hipLaunchKernelGGL((paged_merge_kernel<T, D, 4>), dim3((unsigned)rows), dim3(256), 0, s, a, 1);
      } else {
        const int per_wave = p.cut.nparts > 1 ? 1 : 16;
        const long long mblocks = (rows + 4 * per_wave - 1) / (4 * per_wave);
        if (mblocks > INT_MAX) return fail(FTK_ERR_UNSUPPORTED_SHAPE, "%s: grid too large", who);
        hipLaunchKernelGGL((paged_merge_kernel<T, D, 1>), dim3((unsigned)mblocks), dim3(256), 0, s, a, per_wave);
      }
      return check_launch("paged_merge_kernel");
    }
  });
}

}  // namespace ftk
