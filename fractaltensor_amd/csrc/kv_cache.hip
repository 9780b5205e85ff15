// Keys and values on their way into a paged cache and out of it again.
//
// Both directions move each byte once, 16 bytes of 16-bit elements a lane: the D / 8 lanes of a row are neighbours, a row's
// maximum is taken over them by exchanges, and a lane has ITEMS pieces of keys and as many of values in flight together.  Where the tokens
// of a wave live is looked up once, a lane to a token, and handed to the lanes that need it.
#include "kv_common.h"

namespace ftk {

constexpr int kKvThreads = 256;

// Lanes that share a row: a power of two (D 96 leaves four of sixteen idle).
template <int D>
constexpr int kRowLanes = D == 96 ? 16 : D / 8;

struct KvStrides {
  long long k_token, k_head, v_token, v_head;   // elements
};

// The rows of a wave: `tokens` tokens from token0 on with heads head0 .. of each; row r of them is token r / heads, head r % heads.
struct WaveRows {
  int token0, tokens, head0, heads, rows;
  unsigned inverse;                              // ceil(2^16 / heads): r / heads for the rows of a wave, 64 at most
};
struct KvSplit {
  int tokens, heads;                             // of a wave
};
template <int D, int ITEMS>
constexpr int kWaveRows = ITEMS * (64 / kRowLanes<D>);

__device__ __forceinline__ WaveRows wave_rows(const KvSplit& split, const KvBatch& batch, int heads) {
  WaveRows w;
  const int wave = __builtin_amdgcn_readfirstlane(blockIdx.x * (kKvThreads / 64) + (threadIdx.x >> 6));
  w.token0 = wave * split.tokens;
  w.tokens = min(split.tokens, batch.tokens - w.token0);
  w.head0 = blockIdx.y * split.heads;
  w.heads = min(split.heads, heads - w.head0);
  w.rows = w.tokens * w.heads;
  w.inverse = (65536u + w.heads - 1) / (unsigned)w.heads;
  return w;
}

constexpr int kNoPlace = -1, kNoSequence = -2;

// Where the tokens of a wave live: lane i has the page of the i-th (kNoPlace: the cache has no room for its position or no such page;
// kNoSequence: it is no sequence's) and its row in that page.
struct WavePlaces {
  int page, row;
};
__device__ __forceinline__ WavePlaces wave_places(const KvBatch& batch, const KvPages& pages, const WaveRows& w, int lane) {
  const int first = count_at_most(batch.sequences, w.token0, [&](int i) { return batch.starts[i + 1]; });
  const int token = w.token0 + lane;
  // the ends of the 64 sequences from `first` on; how many of them are at or before a lane's token
  const int end = first + lane < batch.sequences ? batch.starts[first + 1 + lane] : INT_MAX;
  int n = 0;
#pragma unroll
  for (int step = 32; step > 0; step >>= 1)
    if (__shfl(end, n + step - 1) <= token) n += step;
  int b = first + n;
  WavePlaces p{kNoSequence, 0};
  if (lane >= w.tokens) return p;
  if (n == 63)
    while (b < batch.sequences && batch.starts[b + 1] <= token) ++b;
  if (b >= batch.sequences) return p;
  const int start = batch.starts[b], stop = batch.starts[b + 1];
  if (token < start) return p;
  p.page = kNoPlace;
  const long long position = (long long)batch.lens[b] - stop + token;
  if (position < 0 || position >= kv_capacity(batch, pages.page_shift)) return p;
  const int page = batch.table[(long long)b * batch.width + (position >> pages.page_shift)];
  if (page < 0 || page >= pages.pages) return p;
  p.page = page;
  p.row = (int)(position & ((1 << pages.page_shift) - 1));
  return p;
}
__device__ __forceinline__ long long cache_row(const KvPages& pages, int page, int head, int row) {
  return (((long long)page * pages.heads + head) << pages.page_shift) + row;
}

template <typename T, KvFormat F, int D>
__device__ __forceinline__ void write_row(const v4u piece, unsigned char* codes, signed char* exps, long long row, int lane, bool valid) {
  if constexpr (F == kSame) {
    if (valid) *reinterpret_cast<v4u*>(codes + (size_t)row * (2 * D) + 16 * lane) = piece;
  } else {
    using C = Codes<F, T>;
    float x[8], most = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = T::low(piece[i]);
      x[2 * i + 1] = T::high(piece[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(x[i]));   // (a NaN does not count)
#pragma unroll
    for (int o = kRowLanes<D> / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o));
    if (most > C::kReach) {
      most = C::kReach;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (fabsf(x[i]) > C::kReach) x[i] = copysignf(C::kReach, x[i]);
    }
    const int e = row_exponent<F, T>(most);
    const float down = power_of_two(-e);
    const v2u w = {encode4<F>(x[0] * down, x[1] * down, x[2] * down, x[3] * down), encode4<F>(x[4] * down, x[5] * down, x[6] * down, x[7] * down)};
    if (valid) {
      *reinterpret_cast<v2u*>(codes + (size_t)row * D + 8 * lane) = w;
      if (lane == 0) exps[row] = (signed char)e;
    }
  }
}

template <typename T, KvFormat F, int D, int ITEMS>
__global__ __launch_bounds__(kKvThreads) void kv_write_kernel(const typename T::scalar* __restrict__ keys, const typename T::scalar* __restrict__ values,
                                                              KvStrides st, KvPages pages, KvBatch batch, KvSplit split) {
  const WaveRows w = wave_rows(split, batch, pages.heads);
  if (w.tokens <= 0) return;
  const int lane = threadIdx.x & 63, piece = lane % kRowLanes<D>;
  v4u k[ITEMS], v[ITEMS];
  int token[ITEMS], head[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int r = min(i * (64 / kRowLanes<D>) + lane / kRowLanes<D>, w.rows - 1);
    token[i] = r * w.inverse >> 16;
    head[i] = w.head0 + r - token[i] * w.heads;
    const int at = min(piece, D / 8 - 1) * 8;
    k[i] = *reinterpret_cast<const v4u*>(keys + (long long)(w.token0 + token[i]) * st.k_token + head[i] * st.k_head + at);
    v[i] = *reinterpret_cast<const v4u*>(values + (long long)(w.token0 + token[i]) * st.v_token + head[i] * st.v_head + at);
  }
  const WavePlaces places = wave_places(batch, pages, w, lane);
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int page = __shfl(places.page, token[i]), row = __shfl(places.row, token[i]);
    const bool in = i * (64 / kRowLanes<D>) + lane / kRowLanes<D> < w.rows && piece < D / 8 && page >= 0;
    const long long at = cache_row(pages, page, head[i], row);
    write_row<T, F, D>(k[i], pages.k, pages.k_exps, at, piece, in);
    write_row<T, F, D>(v[i], pages.v, pages.v_exps, at, piece, in);
  }
}

// What a lane has of a row in a cache that came from T (kSame: that holds T).
template <typename T, KvFormat F, int D>
struct RowPiece {
  v4u same;
  v2u codes;
  int e;
  __device__ __forceinline__ void load(const unsigned char* from, const signed char* exps, long long row, int lane, bool valid) {
    same = v4u{0, 0, 0, 0};
    codes = v2u{0, 0};
    e = 0;
    if (!valid) return;
    if constexpr (F == kSame) {
      same = *reinterpret_cast<const v4u*>(from + (size_t)row * (2 * D) + 16 * lane);
    } else {
      codes = *reinterpret_cast<const v2u*>(from + (size_t)row * D + 8 * lane);
      e = exps[row];
    }
  }
  template <typename Out>
  __device__ __forceinline__ void store(Out* out) const {
    float x[8];
    if constexpr (F == kSame) {
      if constexpr (std::is_same<Out, typename T::scalar>::value) {
        *reinterpret_cast<v4u*>(out) = same;
        return;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] = T::low(same[i]);
        x[2 * i + 1] = T::high(same[i]);
      }
    } else {
      const float up = ldexpf(1.0f, e);                          // (of any signed byte: 2^-128 too)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if constexpr (F == kInt8) {
#pragma unroll
          for (int j = 0; j < 4; ++j) x[4 * i + j] = int8_code(codes[i], j) * up;
        } else {
          x[4 * i] = __builtin_amdgcn_cvt_f32_fp8((int)codes[i], 0) * up;
          x[4 * i + 1] = __builtin_amdgcn_cvt_f32_fp8((int)codes[i], 1) * up;
          x[4 * i + 2] = __builtin_amdgcn_cvt_f32_fp8((int)codes[i], 2) * up;
          x[4 * i + 3] = __builtin_amdgcn_cvt_f32_fp8((int)codes[i], 3) * up;
        }
      }
    }
    if constexpr (std::is_same<Out, float>::value) {
      *reinterpret_cast<v4f*>(out) = v4f{x[0], x[1], x[2], x[3]};
      *reinterpret_cast<v4f*>(out + 4) = v4f{x[4], x[5], x[6], x[7]};
    } else {
      using O = typename std::conditional<std::is_same<Out, _Float16>::value, Half, Brain>::type;
      *reinterpret_cast<v4u*>(out) = v4u{O::pack(x[0], x[1]), O::pack(x[2], x[3]), O::pack(x[4], x[5]), O::pack(x[6], x[7])};
    }
  }
};

template <typename T, KvFormat F, typename Out, int D, int ITEMS>
__global__ __launch_bounds__(kKvThreads) void kv_read_kernel(KvPages pages, KvBatch batch, Out* __restrict__ keys, Out* __restrict__ values, KvSplit split) {
  const WaveRows w = wave_rows(split, batch, pages.heads);
  if (w.tokens <= 0) return;
  const int lane = threadIdx.x & 63, piece = lane % kRowLanes<D>;
  RowPiece<T, F, D> k[ITEMS], v[ITEMS];
  int out[ITEMS];                                              // row of the result behind token0's first; -1: none
  const WavePlaces places = wave_places(batch, pages, w, lane);
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int r = i * (64 / kRowLanes<D>) + lane / kRowLanes<D>, token = min(r, w.rows - 1) * w.inverse >> 16, head = w.head0 + r - token * w.heads;
    const int page = __shfl(places.page, token), row = __shfl(places.row, token);
    const bool in = r < w.rows && piece < D / 8;
    out[i] = in && page != kNoSequence ? token * pages.heads + head : -1;
    const long long at = cache_row(pages, page, head, row);
    k[i].load(pages.k, pages.k_exps, at, piece, in && page >= 0);
    v[i].load(pages.v, pages.v_exps, at, piece, in && page >= 0);
  }
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    if (out[i] < 0) continue;
    const long long at = ((long long)w.token0 * pages.heads + out[i]) * D + 8 * piece;
    k[i].store(keys + at);
    v[i].store(values + at);
  }
}

// ---- host side ---------------------------------------------------------------------

int check_kv_pages(const char* who, const ftk_kv_pages* p, KvPages* out) {
  if (!p || !p->k || !p->v) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: pages must be non-NULL", who);
  if (p->type < FTK_F16 || p->type > FTK_INT8) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: unknown type of pages %d", who, p->type);
  if (p->pages <= 0 || p->heads <= 0) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: pages and heads must be positive", who);
  if (p->page_size < 16 || p->page_size > 1024 || (p->page_size & (p->page_size - 1)))
    return fail(FTK_ERR_UNSUPPORTED_SHAPE, "%s: page size must be a power of two from 16 to 1024, got %d", who, p->page_size);
  if (p->head_size != 32 && p->head_size != 64 && p->head_size != 96 && p->head_size != 128)
    return fail(FTK_ERR_UNSUPPORTED_SHAPE, "%s: head size must be 32, 64, 96 or 128, got %d", who, p->head_size);
  const bool codes = p->type == FTK_E4M3 || p->type == FTK_INT8;
  if (codes != (p->k_exps != nullptr) || codes != (p->v_exps != nullptr))
    return fail(FTK_ERR_INVALID_ARGUMENT, "%s: exponents belong to pages of 8 bits, and to those only", who);
  if (!aligned16(p->k) || !aligned16(p->v) || !aligned16(p->k_exps) || !aligned16(p->v_exps))
    return fail(FTK_ERR_INVALID_ARGUMENT, "%s: pages and exponents must be 16-byte aligned", who);
  *out = KvPages{(unsigned char*)p->k, (unsigned char*)p->v, (signed char*)p->k_exps, (signed char*)p->v_exps, p->pages, p->heads,
                 __builtin_ctz((unsigned)p->page_size)};
  return FTK_OK;
}

int check_kv_batch(const char* who, const ftk_kv_batch* b, KvBatch* out) {
  if (!b || b->sequences < 0 || b->tokens < 0 || b->table_width < 0) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: sequences, tokens and table width must not be negative", who);
  const bool none = b->sequences == 0 || b->tokens == 0;        // nothing to do
  if (!none && b->table_width == 0) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: the table has no columns", who);
  if (!none && (!b->table || !b->lens || !b->starts)) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: table, lens and starts must be non-NULL", who);
  if (b->tokens > (1 << 28)) return fail(FTK_ERR_UNSUPPORTED_SHAPE, "%s: at most 2^28 tokens", who);
  if (((uintptr_t)b->table | (uintptr_t)b->lens | (uintptr_t)b->starts) & 3) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: table, lens and starts must be 4-byte aligned", who);
  *out = KvBatch{b->table, b->lens, b->starts, b->sequences, b->table_width, none ? 0 : b->tokens};
  return FTK_OK;
}

static int check_same_type(const char* who, int type, int cache) {
  if (type != FTK_F16 && type != FTK_BF16) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: keys and values must be fp16 or bf16", who);
  if ((cache == FTK_F16 || cache == FTK_BF16) && cache != type) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: pages of 16 bits must have the type of the keys and values", who);
  return FTK_OK;
}

// Calls f(rows that a lane has a piece of, grid, tokens and heads of a wave): two rows where that leaves two blocks or more to a compute unit,
// one for less, whose time is the chain of look-ups.  (Prompts of 4750 tokens, 8 heads of 128 in bf16, into int8: 9.1 us with two, 10.5 with one, 9.6 with
// four; 42800 such tokens out of int8: 50 us with two or four, 55 with eight, 62 with a look-up for each row.)
template <int D, typename F>
static int with_items(const char* who, int tokens, int heads, F&& f) {
  const DeviceProps* d = nullptr;
  if (const int rc = device_props(&d)) return rc;
  auto with = [&](auto items) -> int {
    constexpr int R = kWaveRows<D, decltype(items)::value>;
    const KvSplit split{std::max(1, R / heads), std::min(R, heads)};
    const long long blocks = ((long long)tokens + 4LL * split.tokens - 1) / (4LL * split.tokens);
    const int parts = (heads + split.heads - 1) / split.heads;
    if (parts > 65535 || blocks > UINT_MAX / kKvThreads) return fail(FTK_ERR_UNSUPPORTED_SHAPE, "%s: too many heads or tokens for one launch", who);
    return f(items, dim3((unsigned)blocks, (unsigned)parts), split);
  };
  static_assert(kKvThreads == 4 * 64, "four waves");
  const bool many = (long long)tokens * heads >= 4LL * kWaveRows<D, 2> * 2 * d->cus;
  return many ? with(std::integral_constant<int, 2>{}) : with(std::integral_constant<int, 1>{});
}

}  // namespace ftk

extern "C" {

int ftk_kv_cache_write(const void* keys, const void* values, int type, long long key_token_stride, long long key_head_stride,
                       long long value_token_stride, long long value_head_stride, const ftk_kv_pages* pages, const ftk_kv_batch* batch,
                       ftk_stream_t stream) {
  using namespace ftk;
  const char* who = "ftk_kv_cache_write";
  KvPages p;
  KvBatch b;
  int rc = check_kv_pages(who, pages, &p);
  if (rc || (rc = check_kv_batch(who, batch, &b)) || (rc = check_same_type(who, type, pages->type))) return rc;
  if (b.tokens == 0) return FTK_OK;
  if (!keys || !values) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: keys and values must be non-NULL", who);
  const KvStrides st{key_token_stride, key_head_stride, value_token_stride, value_head_stride};
  for (long long s : {st.k_token, st.k_head, st.v_token, st.v_head})
    if (s < 0 || s % 8) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: strides must be multiples of 8 elements", who);
  if (!aligned16(keys) || !aligned16(values)) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: keys and values must be 16-byte aligned", who);
  return with_kv_types(type, pages->type, pages->head_size, [&](auto t, auto f, auto d) -> int {
    using T = decltype(t);
    constexpr KvFormat F = decltype(f)::value;
    constexpr int D = decltype(d)::value;
    return with_items<D>(who, b.tokens, p.heads, [&](auto n, dim3 grid, KvSplit split) -> int {
      constexpr int ITEMS = decltype(n)::value;
      hipLaunchKernelGGL((kv_write_kernel<T, F, D, ITEMS>), grid, dim3(kKvThreads), 0, (hipStream_t)stream, (const typename T::scalar*)keys,
                         (const typename T::scalar*)values, st, p, b, split);
      return check_launch("kv_write_kernel");
    });
  });
}

int ftk_kv_cache_read(const ftk_kv_pages* pages, const ftk_kv_batch* batch, int type, void* keys, void* values, ftk_stream_t stream) {
  using namespace ftk;
  const char* who = "ftk_kv_cache_read";
  KvPages p;
  KvBatch b;
  int rc = check_kv_pages(who, pages, &p);
  if (rc || (rc = check_kv_batch(who, batch, &b))) return rc;
  if (type != FTK_F16 && type != FTK_BF16 && type != FTK_F32) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: keys and values are read as fp16, bf16 or fp32", who);
  const bool codes = pages->type == FTK_E4M3 || pages->type == FTK_INT8;
  if (!codes && type != FTK_F32 && type != pages->type) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: pages of 16 bits are read in their type or in fp32", who);
  if (b.tokens == 0) return FTK_OK;
  if (!keys || !values || !aligned16(keys) || !aligned16(values)) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: keys and values must be non-NULL and 16-byte aligned", who);
  // what codes stand for does not depend on the type they came from
  return with_kv_types(pages->type == FTK_BF16 ? FTK_BF16 : FTK_F16, pages->type, pages->head_size, [&](auto t, auto f, auto d) -> int {
    using T = decltype(t);
    constexpr KvFormat F = decltype(f)::value;
    constexpr int D = decltype(d)::value;
    auto launch = [&](auto out) -> int {
      using Out = decltype(out);
      return with_items<D>(who, b.tokens, p.heads, [&](auto n, dim3 grid, KvSplit split) -> int {
        constexpr int ITEMS = decltype(n)::value;
        hipLaunchKernelGGL((kv_read_kernel<T, F, Out, D, ITEMS>), grid, dim3(kKvThreads), 0, (hipStream_t)stream, p, b, (Out*)keys, (Out*)values, split);
        return check_launch("kv_read_kernel");
      });
    };
    if (type == FTK_F32) return launch(0.0f);
    if constexpr (F == kSame) return launch(typename T::scalar{});
    else return type == FTK_F16 ? launch(_Float16{}) : launch(__bf16{});
  });
}

}  // extern "C"
