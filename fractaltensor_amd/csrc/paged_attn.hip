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
#include <float.h>

#include <algorithm>
#include <cmath>

#include "kv_common.h"

namespace ftk {

constexpr int kWaves = 4;
constexpr float kNoRef = -3.402823466e38f;   // the reference before any score: finite, so that -inf minus it is -inf
constexpr int kSmallRows = 16;                // sequences of at most so many rows, beside larger ones, are small

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
template <int R>
__device__ __forceinline__ bool find_job(const AttnArgs& a, int b, int tile, int part, bool small, Job& j) {
  j.b = b;
  const KvChunk c = kv_chunk(a.batch, b);
  j.start = c.start;
  j.n = c.n;
  j.first = c.first;
  j.rows = c.n * a.group;
  j.row0 = tile * R;
  if (tile >= (j.rows + R - 1) / R || (j.rows <= a.small_rows) != small) return false;
  j.len = min(c.len, kv_capacity(a.batch, a.pages.page_shift));
  const int t_lo = j.row0 / a.group, t_hi = (min(j.row0 + R, j.rows) - 1) / a.group;
  const long long p_lo = (long long)c.first + t_lo, p_hi = (long long)c.first + t_hi;
  j.hi = a.causal ? clamp_position(p_hi + 1, j.len) : j.len;
  j.sure_hi = a.causal ? clamp_position(p_lo + 1, j.len) : j.len;
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

// The keys [lo, hi) that a row sees, and its place among the packed rows times heads.
struct Row {
  int lo, hi;
  long long at;
};
__device__ __forceinline__ Row row_of(const AttnArgs& a, const Job& j, int kv_head, int row) {
  const int t = row / a.group, g = row - t * a.group;
  const long long p = (long long)j.first + t;
  Row r;
  r.hi = a.causal ? clamp_position(p + 1, j.len) : j.len;
  r.lo = a.window > 0 ? clamp_position(p - a.window + 1, j.len) : 0;
  r.at = (long long)(j.start + t) * a.heads + kv_head * a.group + g;
  return r;
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

// A sum over values as it leaves: one that is infinite, because a value is, as NaN, which it is already where a weight of zero met that value, or a mask cut its tile.
__device__ __forceinline__ float finite_or_nan(float x) { return __builtin_fmaf(x, 0.0f, x); }

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
template <typename T, KvFormat F, int D, int NQ, bool KEPT>
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
    const Row r = row_of(a, j, kv_head, row);
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
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int key = key0 + 16 * h + 4 * kg + r;
            if (key < max(row_lo[nq], j.lo) || key >= min(row_hi[nq], j.hi)) {
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
      const Row r = row_of(a, j, kv_head, row);
      const bool none = r.hi <= r.lo;
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
template <typename T, KvFormat F, int D, int NQ, bool KEPT>
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
  if (!find_job<16 * NQ>(a, b, tile, part, false, j)) return;
  narrow_attention<T, F, D, NQ, KEPT>(a, j, kv_head, smem, threadIdx.x);
}

// ---- wide -----------------------------------------------------------------------------

// Eight waves of 32 rows.  A wave alternates between a phase of matrix instructions, M(t): O^T += V(t)^T P(t)^T and then the scores of
// tile t + 1, and a phase of vector instructions, S(t): the weights of tile t; waves 4 to 7 run one phase behind waves 0 to 3, so that of the two
// waves of a SIMD one feeds the matrix unit while the other works out weights.  A barrier ends every phase.  Waves 0 to 3 bring V(t + 1),
// which is read from their M(t + 1) on, into one of three places, waves 4 to 7 K(t + 2) into that of K(t).  16-bit elements are copied straight into
// LDS; codes of 8 bits go through registers, a tile earlier, and are written as 16-bit elements.
constexpr int kWideWaves = 8, kWideRows = 32 * kWideWaves;
constexpr float kMostSum = 32768.0f;          // a lane's sum of 32 weights above this moves the reference, to where it is at most 32 * 2^kLift

template <int D>
struct WideShape {
  static constexpr int BYTES = 2 * D, TILE = 64 * BYTES;
  static constexpr int ORS = BYTES + 16;                       // a padded row of the O tiles that the waves turn round at the end
  static constexpr int RING = 5 * TILE;                        // two tiles of K, three of V
  static constexpr int LDS = RING + 64 > kWideWaves * 32 * ORS ? RING + 64 : kWideWaves * 32 * ORS;
};

// V: the transposing read of a 32-lane pass covers 4 keys x 64 bytes, which these bring into four different groups of 64 bytes
template <int D>
__device__ __forceinline__ int v_swizzle(int row) {
  if constexpr (D == 128) return 4 * (row & 3);
  else if constexpr (D == 64) return 4 * ((row >> 1) & 1);
  else return 0;                                               // rows of 192 and 64 bytes lie that way
}

template <typename T, KvFormat F, int D>
__device__ __forceinline__ void wide_attention(const AttnArgs& a, const Job& j, int kv_head, unsigned char* smem) {
  using S = WideShape<D>;
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
  unsigned char* const Kb = smem;
  unsigned char* const Vb = smem + 2 * S::TILE;
  const int base = j.lo & ~63;
  const int ntiles = j.hi > j.lo ? (j.hi - base + 63) / 64 : 0;

  // rows of this wave
  const int wrow0 = j.row0 + 32 * wave;
  const bool idle = wrow0 >= j.rows;
  const int row = min(wrow0 + jr, j.rows - 1);
  const Row r = row_of(a, j, kv_head, row);
  int wave_lo, wave_hi, sure_lo, sure_hi;                      // keys that some, and that each, of the wave's rows see
  {
    const int t_lo = min(wrow0, j.rows - 1) / a.group, t_hi = (min(wrow0 + 32, j.rows) - 1) / a.group;
    const long long p_lo = (long long)j.first + t_lo, p_hi = (long long)j.first + t_hi;
    wave_hi = idle ? 0 : min(a.causal ? clamp_position(p_hi + 1, j.len) : j.len, j.hi);
    sure_hi = min(a.causal ? clamp_position(p_lo + 1, j.len) : j.len, j.hi);
    wave_lo = max(a.window > 0 ? clamp_position(p_lo - a.window + 1, j.len) : 0, j.lo);
    sure_lo = max(a.window > 0 ? clamp_position(p_hi - a.window + 1, j.len) : 0, j.lo);
  }
  const int my_lo = max(r.lo, j.lo), my_hi = min(r.hi, j.hi);
  auto sees = [&](int t) __attribute__((always_inline)) { return base + 64 * t < wave_hi && base + 64 * t + 64 > wave_lo; };
  auto masked = [&](int t) __attribute__((always_inline)) { return base + 64 * t < sure_lo || base + 64 * t + 64 > sure_hi; };

  v8 qf[DS];
  {
    const scalar* const q = query_of<T>(a, j, kv_head, row) + 8 * hh;
#pragma unroll
    for (int s = 0; s < DS; ++s) qf[s] = *reinterpret_cast<const v8*>(q + 16 * s);
  }
  asm volatile("" ::: "memory");

  // ---- tiles into LDS: a wave brings the 16 keys from 16 cw on, which lie in one page; waves 0 to 3 those of V, the others those of K
  constexpr int CP = D / 32;                                   // 1 KB copies of 16 rows of 16-bit elements
  const int shift = a.pages.page_shift;
  const long long page_rows = (long long)a.pages.heads << shift;
  const long long head_row = (long long)kv_head << shift;
  const int* const table = a.batch.table + (long long)j.b * a.batch.width;
  const unsigned char* const from = (half ? a.pages.k : a.pages.v) + head_row * (F == kSame ? S::BYTES : D);
  const signed char* const from_exps = F == kSame ? nullptr : (half ? a.pages.k_exps : a.pages.v_exps) + head_row;
  // Cache row (from this head's first) of the 16 keys of this wave in tile t; of the nearest 16 in [lo, hi) where those lie outside (INSIDE: they
  // do not).
  auto block_at = [&](int t, auto inside_c) __attribute__((always_inline)) {
    int key = base + 64 * t + 16 * cw;
    if constexpr (!decltype(inside_c)::value) key = min(max(key, j.lo & ~15), (j.hi - 1) & ~15);
    const int page = min(max(load_uniform(table, key >> shift), 0), a.pages.pages - 1);
    return page * page_rows + (key & ((1 << shift) - 1));
  };
  // Where a lane's 16 bytes of a copy lie: with 64 and 128 elements the swizzle makes copy i's places those of the first with some bits turned over.
  unsigned src[D == 96 ? CP : 1];
#pragma unroll
  for (int i = 0; i < (D == 96 ? CP : 1); ++i) {
    const int p = 64 * i + lane, rw = p / CH, slot = p - rw * CH, in_tile = 16 * cw + rw;
    src[i] = rw * S::BYTES + 16 * (slot ^ (half ? swizzle<S::BYTES>(in_tile) : v_swizzle<D>(in_tile)));
  }
  const unsigned turned = half && D != 96 ? 64 : 0;
  auto source = [&](int i) __attribute__((always_inline)) { return D == 96 ? src[D == 96 ? i : 0] : (src[0] ^ (i * turned)) + 1024 * i; };
  // 16 rows of tile t, `at` what block_at gave, into the tile at `to`
  auto copy = [&](unsigned char* to, int t, long long at, auto inside_c) __attribute__((always_inline)) {
    const int key0 = base + 64 * t + 16 * cw;
    const unsigned char* const block = uniform(from + at * S::BYTES);
    unsigned char* const dst = to + cw * (16 * S::BYTES);
    if (decltype(inside_c)::value || (key0 >= j.lo && key0 + 16 <= j.hi)) {
#pragma unroll
      for (int i = 0; i < CP; ++i) lds_dma16(block, source(i), dst + 1024 * i);
    } else {                                                   // rows outside [lo, hi) repeat the nearest key inside
      const int inside = min(max(key0, j.lo & ~15), (j.hi - 1) & ~15);   // where `at` begins
      const int least = max(j.lo - inside, 0), most = min(j.hi - 1 - inside, 15);
#pragma unroll
      for (int i = 0; i < CP; ++i) {
        const int rw = (64 * i + lane) / CH;
        lds_dma16(block, source(i) + (min(max(key0 + rw - inside, least), most) - rw) * S::BYTES, dst + 1024 * i);
      }
    }
  };
  // 8 bits: 16 codes a lane
  constexpr int LD = (D + 63) / 64;                            // 16-byte pieces of a block of 16 rows, D of them, by 64 lanes
  v4u codes[LD];
  float scale[LD];
  auto load = [&](int t, long long at, auto inside_c) __attribute__((always_inline)) {
    const int key0 = base + 64 * t + 16 * cw;
    const int inside = min(max(key0, j.lo & ~15), (j.hi - 1) & ~15);
    const int least = max(j.lo - inside, 0), most = min(j.hi - 1 - inside, 15);
#pragma unroll
    for (int i = 0; i < LD; ++i) {
      const int p = min(64 * i + lane, D - 1), rw = p / (D / 16), piece = p - rw * (D / 16);
      const long long row_at = at + (decltype(inside_c)::value ? rw : min(max(key0 + rw - inside, least), most));
      codes[i] = *reinterpret_cast<const v4u*>(from + row_at * D + 16 * piece);
      scale[i] = ldexpf(1.0f, from_exps[row_at]);
    }
  };
  auto store = [&](unsigned char* to) __attribute__((always_inline)) {
    if constexpr (F != kSame) {
#pragma unroll
      for (int i = 0; i < LD; ++i) {
        const int p = 64 * i + lane, rw = p / (D / 16), piece = p - rw * (D / 16), in_tile = 16 * cw + rw;
        const int swz = half ? swizzle<S::BYTES>(in_tile) : v_swizzle<D>(in_tile);
        auto put = [&](auto decode) __attribute__((always_inline)) {
          if (D % 64 == 0 || p < D) {
#pragma unroll
            for (int c = 0; c < 2; ++c)
              *reinterpret_cast<v8*>(to + in_tile * S::BYTES + 16 * ((2 * piece + c) ^ swz)) = decode(v2u{codes[i][2 * c], codes[i][2 * c + 1]}, scale[i]);
          }
        };
        // (the conversion of e4m3 rounds once whatever the scale)
        constexpr bool LOOK = std::is_same<T, Half>::value && F == kInt8;
        if (LOOK && __builtin_expect(__builtin_amdgcn_ballot_w64(!(scale[i] >= 0x1p-24f && scale[i] <= 0x1p9f)) != 0, 0)) put(decode8_rounded<T, F>);
        else put(decode8<T, F>);
      }
    }
  };

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
  v8 pf[2][2];

  // the weights of the tile's scores as operands of P V; returns this lane's share of their sum
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
          w[i] = T::pack(p0, p1);
        }
        pf[h][s] = __builtin_bit_cast(v8, w);
      }
    return (sum[0] + sum[1]) + (sum[2] + sum[3]);
  };
  // The reference is not compared with every tile's maximum: weights are worked out against it as it is, and only when a lane's sum says that
  // one of them may not fit 16 bits (or came out infinite, as all do before there is a reference) are the maxima taken, the reference moved, O and the sums
  // rescaled and the tile's weights worked out again.  Any reference gives the same O / l.
  auto phase_s = [&](int t, auto clean_c) __attribute__((always_inline)) {
    if (!decltype(clean_c)::value && masked(t)) {
      const int key0 = base + 64 * t + 4 * hh;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int key = key0 + 32 * h + 8 * (e >> 2) + (e & 3);
          if (key < my_lo || key >= my_hi) sc[h][e] = -INFINITY;
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
  // Waves 0 to 3 look whether their 16 keys of a tile of V hold anything that is not finite, and leave word for all.
  unsigned* const words = reinterpret_cast<unsigned*>(smem + S::RING);   // [three places of V][wave]
  auto look = [&](const unsigned char* vt, int place) __attribute__((always_inline)) {
    unsigned bad = 0;
#pragma unroll
    for (int i = 0; i < CP; ++i) bad |= not_finite<T>(*reinterpret_cast<const v8*>(vt + cw * (16 * S::BYTES) + 1024 * i + 16 * lane));
    const bool any = __builtin_amdgcn_ballot_w64(bad != 0) != 0;
    if (lane == 0) words[4 * place + cw] = any;
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
        const int key = key0 + 8 * (e >> 2) + (e & 3);
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
    if constexpr (F == kSame) {
      copy(half ? Kb : Vb, 0, block_at(0, no{}), no{});
      if (half && ntiles > 1) copy(Kb + S::TILE, 1, block_at(1, no{}), no{});
    } else {
      load(0, block_at(0, no{}), no{});
      store(half ? Kb : Vb);
      if (ntiles > 1) load(1, block_at(1, no{}), no{});
      if (half) {
        if (ntiles > 1) store(Kb + S::TILE);
        if (ntiles > 2) load(2, block_at(2, no{}), no{});
      }
    }
    const int ahead = (half ? 2 : 1) + AHEAD;                  // S(t) asks for tile t + ahead
    long long next = ahead < ntiles ? block_at(ahead, no{}) : 0;
    __builtin_amdgcn_s_waitcnt(0x0F70);                        // vmcnt(0)
    __syncthreads();
    phase_m(Vb, Kb, no{}, yes{});
    int vcur = 2 * S::TILE, vnext = 3 * S::TILE, vfree = 4 * S::TILE;             // V(t), V(t + 1), the place of V(t + 2)
    int kcur = 0, knext = S::TILE;                                                // K(t), K(t + 1)
    // Tiles [clean, dirty): every row sees all of them, and the tiles that they ask for lie inside [lo, hi)
    const int whole = (j.hi - base) / 64;
    const int clean = (max(j.sure_lo, j.lo) - base + 63) / 64, dirty = min((min(j.sure_hi, j.hi) - base) / 64, whole - 2 - AHEAD - 1);
    auto turn = [&](int t, auto clean_c) __attribute__((always_inline)) {
      constexpr bool CLEAN = decltype(clean_c)::value;
      // K(t) was last read in the phase before this one, V(t - 2) two before
      const int bring = t + ahead;
      if constexpr (F == kSame) {
        if (CLEAN || bring < ntiles) copy(smem + (half ? kcur : vnext), bring, next, clean_c);
      } else {
        if (CLEAN || bring - 1 < ntiles) store(smem + (half ? kcur : vnext));
        if (CLEAN || bring < ntiles) load(bring, next, clean_c);
      }
      if (CLEAN || bring + 1 < ntiles) next = block_at(bring + 1, clean_c);
      __builtin_amdgcn_sched_barrier(0);                       // the copies go out before the weights are begun
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
  l += __shfl_xor(l, 32);
  if (j.parts > 1) {
    if (wrow0 + jr < j.rows) {
      float* const po = a.part_o + (r.at * a.cut.nparts + j.part) * D;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<v4f*>(po + 32 * dt + 8 * g + 4 * hh) = v4f{o[dt][4 * g], o[dt][4 * g + 1], o[dt][4 * g + 2], o[dt][4 * g + 3]};
      if (hh == 0) {
        float* const ml = a.part_ml + 2 * (r.at * a.cut.nparts + j.part);
        ml[0] = ref;
        ml[1] = l;
      }
    }
    return;
  }
  if (idle) return;
  // the wave turns its 32 x D tile round through LDS (nobody reads tiles any more) and stores whole rows
  const bool none = r.hi <= r.lo;
  const float inv = none ? 0.0f : 1.0f / l;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[dt][e] = finite_or_nan(o[dt][e]);
  unsigned char* const ot = smem + wave * (32 * S::ORS);
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<v2u*>(ot + jr * S::ORS + 2 * (32 * dt + 8 * g + 4 * hh)) =
          v2u{T::pack(o[dt][4 * g] * inv, o[dt][4 * g + 1] * inv), T::pack(o[dt][4 * g + 2] * inv, o[dt][4 * g + 3] * inv)};
  if (a.lse && hh == 0 && wrow0 + jr < j.rows) a.lse[r.at] = none ? -INFINITY : log_sum(ref, l);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  for (int idx = lane; idx < 32 * CH; idx += 64) {
    const int rw = idx / CH, c = idx - rw * CH;
    if (wrow0 + rw >= j.rows) break;
    const Row to = row_of(a, j, kv_head, wrow0 + rw);
    *reinterpret_cast<v4u*>((unsigned char*)a.o + to.at * S::BYTES + 16 * c) = *reinterpret_cast<const v4u*>(ot + rw * S::ORS + 16 * c);
  }
}

// The workgroups behind the first `wide` take sequences of at most small_rows = 16 rows, which would leave seven of the eight waves without
// any: two (sequence, head, part) each, by four waves that cut the keys as in the narrow kernel.  They read on the compute units that the others
// leave free, or have left, while those multiply.  (A chunk of 512 tokens beside five sequences that decode, 16 heads, 4 of keys, up to
// 16384 of them, in int8: 165 us with all on the wide form, 108 so, and 12 for joining.)
template <typename T, KvFormat F, int D>
__global__ __launch_bounds__(kWideWaves * 64, 1) void paged_wide_kernel(AttnArgs a, int wide) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  Job j;
  if ((int)blockIdx.x >= wide) {
    const int half = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
    const int item = 2 * (blockIdx.x - wide) + half, kv_head = item % a.pages.heads, rest = item / a.pages.heads;
    const int b = rest / a.small.nparts, part = rest - b * a.small.nparts;
    if (b < a.batch.sequences && find_job<16>(a, b, 0, part, true, j)) {
      narrow_attention<T, F, D, 1, false>(a, j, kv_head, smem + half * NarrowShape<F, D>::LDS, threadIdx.x & 255);
    } else {                                                     // the other half's two barriers
      __syncthreads();
      __syncthreads();
    }
    return;
  }
  // the head goes fastest, so that the row blocks of a head meet on the XCDs that have its keys
  const int id = blockIdx.x, kv_head = id % a.pages.heads, rest = id / a.pages.heads;
  const int slot = rest / a.cut.nparts, part = rest - slot * a.cut.nparts;
  int b, tile;
  if (!find_rows<kWideRows>(a, slot, &b, &tile) || !find_job<kWideRows>(a, b, tile, part, false, j)) return;
  wide_attention<T, F, D>(a, j, kv_head, smem);
}

// ---- parts ------------------------------------------------------------------------------

constexpr int kPartsMost = 256;

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

// ---- host side ----------------------------------------------------------------------------

// How a call is run.
struct Plan {
  bool narrow;
  int nq;                  // narrow: blocks of 16 rows of a workgroup, 1 or 2
  int slots, slots_per_seq;
  Cut cut, small;
  int small_rows;
  size_t large, all;       // parts that there is room for: of sequences that are not small, and with those that are
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

static Plan plan(const ftk_kv_pages& pages, const KvBatch& b, int page_shift, int heads, int window, int max_queries, int max_keys, int cus, size_t room) {
  const int D = pages.head_size, group = heads / pages.heads;
  Plan p;
  const long long most = max_queries > 0 ? std::min(max_queries, b.tokens) : b.tokens;   // new tokens of a sequence
  const long long most_rows = most * group, rows = (long long)b.tokens * heads;
  p.narrow = most_rows <= 64;
  const long long capacity = (long long)b.width << page_shift;
  long long seen = max_keys > 0 ? std::min<long long>(max_keys, capacity) : capacity;
  if (window > 0) seen = std::min(seen, most + window + 64);   // from the first key that the first new token sees, down to a multiple of 64
  const int keys = (int)std::min<long long>(seen, INT_MAX - 1024);
  // 32 rows to a narrow workgroup read the keys half as often as 16; those are the faster ones where even parts of 256 keys are fewer than the compute
  // units.  (16 sequences of up to 4096 keys, 8 heads of them, 20 rows: 48 us by 32 rows and 54 by 16 at D 128, int8 46 and 48, 25 and 28 at D 64; 48 rows: 65 and 67, int8 69 and 71, but
  // 38 and 34 at D 64; two sequences of up to 1000 keys, 48 rows: 15 and 12.)
  p.nq = most_rows <= 16 || (p.narrow && ((most_rows + 31) / 32) * b.sequences * pages.heads * ((keys + 255) / 256) < cus) ? 1 : 2;
  const int R = p.narrow ? 16 * p.nq : kWideRows;
  const long long per_seq = (most_rows + R - 1) / R, packed = (long long)b.tokens * group / R + b.sequences;
  // numbered by row blocks, unless most of such slots would be empty (as those of narrow workgroups, four to a sequence at most, cannot be)
  p.slots_per_seq = p.narrow || b.sequences * per_seq <= 2 * packed ? (int)per_seq : 0;
  p.slots = (int)std::min<long long>(p.slots_per_seq ? b.sequences * per_seq : packed, INT_MAX);
  p.small_rows = p.narrow || b.sequences == 1 ? 0 : kSmallRows;
  const int held = pages.type == FTK_F16 || pages.type == FTK_BF16 ? 4 * D : 2 * D + 2;   // bytes of a position and head
  const long long small_rows = (long long)b.sequences * pages.heads * kSmallRows;
  p.small = Cut{1, keys};
  if (p.narrow) {
    const double units = (double)p.slots * pages.heads;
    p.cut = best_cut(keys, 256, rows, D, room, [&](const Cut& c) { return narrow_cost(units * c.nparts, c.part_keys, held, cus, b.sequences == 1) + join_cost(rows, D, c.nparts); });
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
static int launch_with_lds(const char* name, K kernel, DeviceOnce& once, long long blocks, int waves, int lds, hipStream_t s, Args... args) {
  if (blocks > INT_MAX) return fail(FTK_ERR_UNSUPPORTED_SHAPE, "ftk_paged_attn: grid too large");
  unsigned bit;
  if (once.pending(&bit)) {
    FTK_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    once.done(bit);
  }
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(waves * 64), lds, s, args...);
  return check_launch(name);
}

}  // namespace ftk

extern "C" {

size_t ftk_paged_attn_workspace_bytes(const ftk_kv_pages* pages, const ftk_kv_batch* batch, int heads, int window, int max_queries, int max_keys) {
  using namespace ftk;
  const DeviceProps* d = nullptr;
  if (!pages || !batch || pages->heads <= 0 || heads <= 0 || heads % pages->heads || batch->tokens <= 0 || batch->sequences <= 0 || batch->table_width <= 0 ||
      pages->page_size <= 0 || window < 0 || device_props(&d))
    return 0;
  KvBatch b{};
  b.tokens = batch->tokens;
  b.sequences = batch->sequences;
  b.width = batch->table_width;
  const Plan p = plan(*pages, b, __builtin_ctz((unsigned)pages->page_size), heads, window, max_queries, max_keys, d->cus, SIZE_MAX);
  return workspace_of(p.all, pages->head_size);
}

int ftk_paged_attn(const void* q, int type, long long q_token_stride, long long q_head_stride, const ftk_kv_pages* pages, const ftk_kv_batch* batch,
                   void* o, float* lse, int heads, float scale, int causal, int window, int max_queries, int max_keys, void* workspace,
                   size_t workspace_bytes, ftk_stream_t stream) {
  using namespace ftk;
  const char* who = "ftk_paged_attn";
  AttnArgs a;
  int rc = check_kv_pages(who, pages, &a.pages);
  if (rc || (rc = check_kv_batch(who, batch, &a.batch)) || (rc = check_attention(who, heads, pages))) return rc;
  if (type != FTK_F16 && type != FTK_BF16) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: queries must be fp16 or bf16", who);
  if ((pages->type == FTK_F16 || pages->type == FTK_BF16) && pages->type != type) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: pages of 16 bits must have the type of the queries", who);
  if (!(scale > 0.0f) || !(scale * 1.4426950408889634f <= FLT_MAX)) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: scale must be positive, and its product with log2(e) finite", who);
  if (window < 0 || max_queries < 0 || max_keys < 0) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: window, max_queries and max_keys must not be negative", who);
  if (a.batch.tokens == 0) return FTK_OK;
  if (!q || !o || !aligned16(q) || !aligned16(o)) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: q and o must be non-NULL and 16-byte aligned", who);
  if ((uintptr_t)lse & 3) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: lse must be 4-byte aligned", who);
  if (q_token_stride < 0 || q_head_stride < 0 || q_token_stride % 8 || q_head_stride % 8) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: strides must be multiples of 8 elements", who);
  if ((long long)a.batch.tokens * (heads / pages->heads) > INT_MAX / 2) return fail(FTK_ERR_UNSUPPORTED_SHAPE, "%s: too many rows", who);
  const DeviceProps* d = nullptr;
  if ((rc = device_props(&d))) return rc;
  if (workspace && !aligned16(workspace)) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: the workspace must be 16-byte aligned", who);
  const Plan p = plan(*pages, a.batch, a.pages.page_shift, heads, window, max_queries, max_keys, d->cus, workspace ? workspace_bytes : 0);
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
  const long long rows = (long long)a.batch.tokens * heads;
  a.part_o = (float*)workspace;
  a.part_ml = a.part_o + p.all * pages->head_size;
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
        return launch_with_lds("paged_narrow_kernel", paged_narrow_kernel<T, F, D, decltype(nq)::value, decltype(kept)::value>, once, blocks, kWaves, NarrowShape<F, D>::LDS, s,
                               a, p.slots_per_seq);
      };
      auto with_kept = [&](auto nq) { return p.slots_per_seq == 1 ? launch(nq, no{}) : launch(nq, yes{}); };
      bad = p.nq == 2 ? with_kept(std::integral_constant<int, 2>{}) : with_kept(std::integral_constant<int, 1>{});
    } else {
      static DeviceOnce once;
      constexpr int lds = std::max(WideShape<D>::LDS, 2 * NarrowShape<F, D>::LDS);
      bad = launch_with_lds("paged_wide_kernel", paged_wide_kernel<T, F, D>, once, blocks + pairs, kWideWaves, lds, s, a, (int)blocks);
    }
    if (bad || p.all == 0) return bad;
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
  });
}

}  // extern "C"
