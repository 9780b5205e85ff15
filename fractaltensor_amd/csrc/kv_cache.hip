// Keys and values on their way into a paged cache and out of it again.
//
// Both directions move each byte once, 16 bytes of 16-bit elements a lane: the D / 8 lanes of a row are neighbours, a row's
// maximum is taken over them by exchanges, and a thread has ITEMS pieces of keys and as many of values in flight together.  Which
// sequence a row belongs to is looked up once per wave, 64 sequences at a time.
#include "kv_common.h"

namespace ftk {

constexpr int kKvThreads = 256;

// Lanes that share a row: a power of two (D 96 leaves four of sixteen idle).
template <int D>
constexpr int kRowLanes = D == 96 ? 16 : D / 8;

struct KvStrides {
  long long k_token, k_head, v_token, v_head;   // elements
};

struct KvPlace {
  bool valid;          // the row is a sequence's, at a position that the cache has room for, in a page that there is
  bool owned;          // the row is a sequence's
  long long row;       // of the cache: (page * heads + head) * page size + row of the page
};

// Where packed row `token` of head h lives; *b: a sequence at or before the row's, which becomes that.
__device__ __forceinline__ KvPlace kv_place(const KvBatch& batch, int pages, int heads, int page_shift, int token, int h, int* seq) {
  int b = *seq;
  while (b < batch.sequences && batch.starts[b + 1] <= token) ++b;
  *seq = b;
  KvPlace p{false, false, 0};
  if (b >= batch.sequences) return p;
  const int start = batch.starts[b], end = batch.starts[b + 1];
  if (token < start) return p;
  p.owned = true;
  const long long position = (long long)batch.lens[b] - end + token;
  if (position < 0 || position >= kv_capacity(batch, page_shift)) return p;
  const int page = batch.table[(long long)b * batch.width + (position >> page_shift)];
  if (page < 0 || page >= pages) return p;
  p.valid = true;
  p.row = (((long long)page * heads + h) << page_shift) + (position & ((1 << page_shift) - 1));
  return p;
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

// The items (token, head) of a thread: ITEMS of them, a block's apart.
template <int D, int ITEMS>
struct Items {
  long long first;        // of this thread
  int lane;               // in the row
  static constexpr int kStep = kKvThreads / kRowLanes<D>;
  __device__ __forceinline__ Items() : first((long long)blockIdx.x * (ITEMS * kStep) + threadIdx.x / kRowLanes<D>), lane(threadIdx.x % kRowLanes<D>) {}
  __device__ __forceinline__ long long operator[](int i) const { return first + i * kStep; }
};

template <typename T, KvFormat F, int D, int ITEMS>
__global__ __launch_bounds__(kKvThreads) void kv_write_kernel(const typename T::scalar* __restrict__ keys, const typename T::scalar* __restrict__ values,
                                                              KvStrides st, KvPages pages, KvBatch batch, long long items) {
  const Items<D, ITEMS> mine;
  v4u k[ITEMS], v[ITEMS];
  int token[ITEMS], head[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const long long it = min(mine[i], items - 1);
    token[i] = (int)(it / pages.heads);
    head[i] = (int)(it - (long long)token[i] * pages.heads);
    const int piece = min(mine.lane, D / 8 - 1);
    k[i] = *reinterpret_cast<const v4u*>(keys + token[i] * st.k_token + head[i] * st.k_head + 8 * piece);
    v[i] = *reinterpret_cast<const v4u*>(values + token[i] * st.v_token + head[i] * st.v_head + 8 * piece);
  }
  int b = count_at_most(batch.sequences, __builtin_amdgcn_readfirstlane(token[0]), [&](int i) { return batch.starts[i + 1]; });
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const KvPlace p = kv_place(batch, pages.pages, pages.heads, pages.page_shift, token[i], head[i], &b);
    const bool in = mine[i] < items && mine.lane < D / 8 && p.valid;
    write_row<T, F, D>(k[i], pages.k, pages.k_exps, p.row, mine.lane, in);
    write_row<T, F, D>(v[i], pages.v, pages.v_exps, p.row, mine.lane, in);
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
      const float up = power_of_two(e);
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
__global__ __launch_bounds__(kKvThreads) void kv_read_kernel(KvPages pages, KvBatch batch, Out* __restrict__ keys, Out* __restrict__ values,
                                                             long long items) {
  const Items<D, ITEMS> mine;
  RowPiece<T, F, D> k[ITEMS], v[ITEMS];
  bool in[ITEMS];
  const int first = __builtin_amdgcn_readfirstlane((int)(min(mine[0], items - 1) / pages.heads));
  int b = count_at_most(batch.sequences, first, [&](int i) { return batch.starts[i + 1]; });
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const long long it = min(mine[i], items - 1);
    const int token = (int)(it / pages.heads), h = (int)(it - (long long)token * pages.heads);
    const KvPlace p = kv_place(batch, pages.pages, pages.heads, pages.page_shift, token, h, &b);
    in[i] = mine[i] < items && mine.lane < D / 8 && p.owned;
    k[i].load(pages.k, pages.k_exps, p.row, mine.lane, in[i] && p.valid);
    v[i].load(pages.v, pages.v_exps, p.row, mine.lane, in[i] && p.valid);
  }
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    if (!in[i]) continue;
    k[i].store(keys + mine[i] * D + 8 * mine.lane);
    v[i].store(values + mine[i] * D + 8 * mine.lane);
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

// Calls f(items of a thread, blocks): four items where that leaves two blocks of 256 threads or more to a compute unit (the look-ups of a wave then serve four rows), one
// for less, whose time is the chain of look-ups.
template <int D, typename F>
static int with_items(const char* who, long long items, F&& f) {
  const DeviceProps* d = nullptr;
  if (const int rc = device_props(&d)) return rc;
  constexpr long long step = kKvThreads / kRowLanes<D>;
  const bool many = items >= 4 * step * 2 * d->cus;
  const long long per = many ? 4 * step : step, n = (items + per - 1) / per;
  if (n > INT_MAX) return fail(FTK_ERR_UNSUPPORTED_SHAPE, "%s: too many rows for one launch", who);
  return many ? f(std::integral_constant<int, 4>{}, (unsigned)n) : f(std::integral_constant<int, 1>{}, (unsigned)n);
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
  const long long items = (long long)b.tokens * p.heads;
  return with_kv_types(type, pages->type, pages->head_size, [&](auto t, auto f, auto d) -> int {
    using T = decltype(t);
    constexpr KvFormat F = decltype(f)::value;
    constexpr int D = decltype(d)::value;
    return with_items<D>(who, items, [&](auto n, unsigned blocks) -> int {
      constexpr int ITEMS = decltype(n)::value;
      hipLaunchKernelGGL((kv_write_kernel<T, F, D, ITEMS>), dim3(blocks), dim3(kKvThreads), 0, (hipStream_t)stream, (const typename T::scalar*)keys,
                         (const typename T::scalar*)values, st, p, b, items);
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
  const long long items = (long long)b.tokens * p.heads;
  // what codes stand for does not depend on the type they came from
  return with_kv_types(pages->type == FTK_BF16 ? FTK_BF16 : FTK_F16, pages->type, pages->head_size, [&](auto t, auto f, auto d) -> int {
    using T = decltype(t);
    constexpr KvFormat F = decltype(f)::value;
    constexpr int D = decltype(d)::value;
    auto launch = [&](auto out) -> int {
      using Out = decltype(out);
      return with_items<D>(who, items, [&](auto n, unsigned blocks) -> int {
        constexpr int ITEMS = decltype(n)::value;
        hipLaunchKernelGGL((kv_read_kernel<T, F, Out, D, ITEMS>), dim3(blocks), dim3(kKvThreads), 0, (hipStream_t)stream, p, b, (Out*)keys, (Out*)values, items);
        return check_launch("kv_read_kernel");
      });
    };
    if (type == FTK_F32) return launch(0.0f);
    if constexpr (F == kSame) return launch(typename T::scalar{});
    else return type == FTK_F16 ? launch(_Float16{}) : launch(__bf16{});
  });
}

}  // extern "C"
