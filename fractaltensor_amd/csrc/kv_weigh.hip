// The attention weights that new tokens give to the positions of a paged cache, gathered position by position.
//
// weights[k] = decay * weights[k] + sum over new tokens t and heads of the group of exp(scale q_t . k - lse_t), the sum of a column of the
// attention matrix where attention itself needs the sums of its rows.  So a workgroup has KEYS and walks the rows (row r is token r / G, head
// r % G): four waves of 16 NB keys each, whose fragments stay in registers, over blocks of 64 rows of Q in LDS, copied there while the last are worked on.
// The product is S = Q K^T with a key to a lane (16x16x32: lane (m, kg) has the scores of key m with rows 4 kg .. + 3), so that a lane adds up its own
// key's weights in one register, and only the four lanes of a key meet at the end.  Nothing is joined between workgroups and there are no
// atomics: the sum of a key has one order, which depends on the call's sizes alone.
//
// Decoding reads K once and is bound by that; prompts are bound by the exponentials (16 cycles for a wave's 64, beside 8 of other vector work
// and 16 of matrix work at D 128).  Scores and sums are fp32, codes of 8 bits enter the product as they are, exact in both 16-bit types, and the
// power of two of a key's row multiplies its scores.
#include <float.h>

#include <algorithm>
#include <cmath>

#include "kv_common.h"

namespace ftk {

constexpr int kWeighRows = 64;   // rows of Q in LDS at once

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
  int tiles;                       // blocks of keys of a (sequence, head) that the grid has
};

__device__ __forceinline__ int token_of(const WeighArgs& a, unsigned row) { return a.group == 1 ? (int)row : (int)__umulhi(row, a.inverse); }

// 16 bytes a lane from an address of its own into LDS.
__device__ __forceinline__ void lds_dma16_each(const void* from, void* lds_base) {
  const unsigned lds_addr = (unsigned)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void*)lds_base);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(lds_addr), "v"(from) : "memory", "m0");
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
  static constexpr int ROWS = kWeighRows * 12;                 // lse, and the positions that a row sees: from, to
  static constexpr int LDS = 2 * (Q + ROWS);
};

template <typename T, KvFormat F, int D, int NB>
__global__ __launch_bounds__(256, NB == 4 && D >= 96 ? 3 : 4) void kv_weigh_kernel(WeighArgs a) {
  using S = WeighShape<D>;
  using v8 = typename T::v8;
  using scalar = typename T::scalar;
  constexpr int KS = D / 32, CH = S::BYTES / 16, KEYS = 16 * NB, CACHED = F == kSame ? 2 * D : D;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[S::LDS];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m = lane & 15, kg = lane >> 4;
  // the head goes fastest, the block of keys slowest: under a causal mask the first blocks are seen by most rows, and go out first
  const int kv_head = blockIdx.x % a.pages.heads, rest = blockIdx.x / a.pages.heads;
  const int b = rest % a.batch.sequences, tile0 = rest / a.batch.sequences;
  const KvChunk c = kv_chunk(a.batch, b);
  const int len = min(c.len, kv_capacity(a.batch, a.pages.page_shift));
  if (c.n == 0) return;

  for (int block0 = tile0 * 4 * KEYS; block0 < len; block0 = (int)min((long long)block0 + (long long)a.tiles * 4 * KEYS, (long long)INT_MAX)) {
    const int key0 = block0 + wave * KEYS;
    // rows that see some key of the workgroup's: those of tokens [t_lo, t_hi)
    const long long last = min((long long)block0 + 4 * KEYS, (long long)len) - 1;
    const int t_lo = a.causal ? (int)min(max((long long)block0 - c.first, 0LL), (long long)c.n) : 0;
    const int t_hi = a.window > 0 ? (int)min(max(last + a.window - c.first, 0LL), (long long)c.n) : c.n;
    const int row_lo = t_lo * a.group, row_hi = t_hi * a.group, rows = max(row_hi - row_lo, 0);

    // ---- this wave's keys
    v8 kf[NB][KS];
    float kfac[NB];
    if (rows > 0) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const int first = min(key0 + 16 * nb, (len - 1) & ~15);    // blocks behind the last repeat it, keys behind the last that one
        const int page = kv_page(a.batch, b, first >> a.pages.page_shift, a.pages.pages);
        const long long row = (((long long)page * a.pages.heads + kv_head) << a.pages.page_shift) + (first & ((1 << a.pages.page_shift) - 1)) + min(m, len - 1 - first);
        const unsigned char* const from = a.pages.k + (size_t)row * CACHED;
        if constexpr (F == kSame) {
#pragma unroll
          for (int s = 0; s < KS; ++s) kf[nb][s] = *reinterpret_cast<const v8*>(from + 64 * s + 16 * kg);
          kfac[nb] = a.scale_log2e;
        } else {
          // 16 codes a load where there are 64 to a row: the product takes the elements in another order, that of Q's reads below
#pragma unroll
          for (int s = 0; s + 1 < KS; s += 2) {
            const v4u w = *reinterpret_cast<const v4u*>(from + 32 * s + 16 * kg);
            kf[nb][s] = decode8<T, F>(v2u{w[0], w[1]}, 1.0f);
            kf[nb][s + 1] = decode8<T, F>(v2u{w[2], w[3]}, 1.0f);
          }
          if constexpr (KS % 2) kf[nb][KS - 1] = decode8<T, F>(*reinterpret_cast<const v2u*>(from + 32 * (KS - 1) + 8 * kg), 1.0f);
          kfac[nb] = ldexpf(a.scale_log2e, a.pages.k_exps[row]);
        }
      }
    }
    // what has been gathered before: lane i has key key0 + i
    const int key = key0 + lane;
    float* at = nullptr;
    float before = 0.0f;
    if (lane < KEYS && key < len) {
      const int page = a.batch.table[(long long)b * a.batch.width + (key >> a.pages.page_shift)];
      if (page >= 0 && page < a.pages.pages) {
        at = a.weights + (((long long)page * a.pages.heads + kv_head) << a.pages.page_shift) + (key & ((1 << a.pages.page_shift) - 1));
        if (key < c.first && a.decay != 0.0f) before = *at * a.decay;
      }
    }

    // ---- rows, 64 at a time
    auto stage = [&](int r0, unsigned char* to) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < S::Q / 4096; ++i) {
        const int p = 64 * (wave * (S::Q / 4096) + i) + lane, in = p / CH, slot = p - in * CH;
        const unsigned row = (unsigned)min(r0 + in, row_hi - 1);
        const int t = token_of(a, row), g = (int)row - t * a.group;
        const scalar* const q = (const scalar*)a.q + (long long)(c.start + t) * a.q_token + (long long)(kv_head * a.group + g) * a.q_head;
        lds_dma16_each(q + 8 * (slot ^ turn<S::BYTES>(in)), to + 1024 * (wave * (S::Q / 4096) + i));
      }
      if (tid < kWeighRows) {
        const unsigned row = (unsigned)min(r0 + tid, row_hi - 1);
        const int t = token_of(a, row), g = (int)row - t * a.group;
        const float x = a.lse[(long long)(c.start + t) * a.heads + kv_head * a.group + g];
        const long long position = (long long)c.first + t;
        const bool none = r0 + tid >= row_hi;
        float* const r = reinterpret_cast<float*>(to + S::Q);
        r[tid] = x == -INFINITY ? INFINITY : x * 1.4426950408889634f;   // a row that sees nothing gives nothing
        int* const sees = reinterpret_cast<int*>(to + S::Q + 4 * kWeighRows);
        sees[tid] = none ? INT_MAX : a.window > 0 ? (int)max(position - a.window + 1, (long long)INT_MIN) : INT_MIN;
        sees[kWeighRows + tid] = a.causal ? (int)min(position, (long long)INT_MAX) : INT_MAX;
      }
    };
    float acc[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) acc[nb] = 0.0f;
    if (rows > 0) {
      stage(row_lo, smem);
      for (int r0 = row_lo, side = 0; r0 < row_hi; r0 += kWeighRows, side ^= 1) {
        __builtin_amdgcn_s_waitcnt(0x0F70);                    // vmcnt(0): this wave's copies
        __syncthreads();
        const unsigned char* const q = smem + side * (S::Q + S::ROWS);
        if (r0 + kWeighRows < row_hi) stage(r0 + kWeighRows, smem + (side ^ 1) * (S::Q + S::ROWS));
        for (int rt = 0; rt < kWeighRows / 16 && r0 + 16 * rt < row_hi; ++rt) {
          // whether each of the 16 rows sees each of the wave's keys, and whether any sees any
          const int tr_lo = token_of(a, (unsigned)(r0 + 16 * rt)), tr_hi = token_of(a, (unsigned)min(r0 + 16 * rt + 15, row_hi - 1));
          const long long p_lo = (long long)c.first + tr_lo, p_hi = (long long)c.first + tr_hi;
          if (key0 >= len || (a.causal && p_hi < key0) || (a.window > 0 && p_lo - a.window >= key0 + KEYS - 1)) continue;
          const bool masked = r0 + 16 * rt + 16 > row_hi || (a.causal && p_lo < key0 + KEYS - 1) || (a.window > 0 && p_hi - a.window >= key0);
          v8 qf[KS];
          const int row = 16 * rt + m;
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            const int chunk = F != kSame && (s | 1) < KS ? 8 * (s / 2) + 2 * kg + (s & 1) : 4 * s + kg;
            qf[s] = *reinterpret_cast<const v8*>(q + row * S::BYTES + 16 * (chunk ^ turn<S::BYTES>(row)));
          }
          const v4f lse = *reinterpret_cast<const v4f*>(q + S::Q + 4 * (16 * rt + 4 * kg));
          v4f sc[NB];
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            sc[nb] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < KS; ++s) sc[nb] = T::mma16(qf[s], kf[nb][s], sc[nb]);
          }
          if (masked) {
            typedef int v4i __attribute__((ext_vector_type(4)));
            const v4i from = *reinterpret_cast<const v4i*>(q + S::Q + 4 * (kWeighRows + 16 * rt + 4 * kg));
            const v4i to = *reinterpret_cast<const v4i*>(q + S::Q + 4 * (2 * kWeighRows + 16 * rt + 4 * kg));
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const int k = key0 + 16 * nb + m;
                const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[nb][r], kfac[nb], -lse[r]));
                acc[nb] += k >= from[r] && k <= to[r] ? w : 0.0f;
              }
          } else {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
              for (int r = 0; r < 4; ++r) acc[nb] += __builtin_amdgcn_exp2f(__builtin_fmaf(sc[nb][r], kfac[nb], -lse[r]));
          }
        }
      }
      __syncthreads();                                         // (the next keys' rows go where these lie)
    }
    // ---- the four lanes of a key meet; lane 16 nb + m takes key m of block nb
    float mine = 0.0f;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float x = acc[nb];
      x += __shfl_xor(x, 16);
      x += __shfl_xor(x, 32);
      if (kg == nb) mine = x;
    }
    if (at) *at = before + mine;
  }
}

}  // namespace ftk

extern "C" {

int ftk_kv_cache_weigh(const void* q, int type, long long q_token_stride, long long q_head_stride, const float* lse, const ftk_kv_pages* pages, float* weights,
                       const ftk_kv_batch* batch, int heads, float scale, float decay, int causal, int window, int max_keys, ftk_stream_t stream) {
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
  if (window < 0 || max_keys < 0) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: window and max_keys must not be negative", who);
  if (a.batch.tokens == 0) return FTK_OK;
  if (!q || !lse || !weights || !aligned16(q)) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: q, lse and weights must be non-NULL and q 16-byte aligned", who);
  if (((uintptr_t)lse | (uintptr_t)weights) & 3) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: lse and weights must be 4-byte aligned", who);
  if (q_token_stride < 0 || q_head_stride < 0 || q_token_stride % 8 || q_head_stride % 8) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: strides must be multiples of 8 elements", who);
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
  const long long capacity = std::min<long long>((long long)a.batch.width << a.pages.page_shift, INT_MAX);
  const long long most = max_keys > 0 ? std::min<long long>(max_keys, capacity) : capacity;
  const long long pairs = (long long)a.batch.sequences * pages->heads;
  return with_kv_types(type, pages->type, pages->head_size, [&](auto t, auto f, auto dc) -> int {
    using T = decltype(t);
    constexpr KvFormat F = decltype(f)::value;
    constexpr int D = decltype(dc)::value;
    auto launch = [&](auto nb) -> int {
      constexpr int NB = decltype(nb)::value;
      const long long tiles = std::max(1LL, (most + 64 * NB - 1) / (64 * NB));
      if (pairs > INT_MAX / 2) return fail(FTK_ERR_UNSUPPORTED_SHAPE, "%s: too many sequences", who);
      a.tiles = (int)std::min(tiles, (long long)(INT_MAX / 2) / pairs);      // (a workgroup takes every a.tiles-th block)
      hipLaunchKernelGGL((kv_weigh_kernel<T, F, D, NB>), dim3((unsigned)(a.tiles * pairs)), dim3(256), 0, (hipStream_t)stream, a);
      return check_launch("kv_weigh_kernel");
    };
    // 256 keys to a workgroup where that leaves two to a compute unit, 64 otherwise
    return pairs * ((most + 255) / 256) >= 2 * d->cus ? launch(std::integral_constant<int, 4>{}) : launch(std::integral_constant<int, 1>{});
  });
}

}  // extern "C"
