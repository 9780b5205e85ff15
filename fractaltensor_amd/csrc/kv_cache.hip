// Keys and values on their way into a paged cache and out of it again.
//
// Both directions move each byte once, 16 bytes of 16-bit elements a lane: the D / 8 lanes of a row are neighbours, a row's
// maximum is taken over them by exchanges, and a thread has the key's and the value's piece in flight together.  Which
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

// Where packed row `token` of head h lives.  first: the token of the wave's first lane.
__device__ __forceinline__ KvPlace kv_place(const KvBatch& batch, int pages, int heads, int page_shift, int token, int h) {
  const int first = __builtin_amdgcn_readfirstlane(token);
  int b = count_at_most(batch.sequences, first, [&](int i) { return batch.starts[i + 1]; });
  while (b < batch.sequences && batch.starts[b + 1] <= token) ++b;
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

// x within the reach of the codes; a NaN stays one and does not count in the maximum.
template <typename C>
__device__ __forceinline__ float within(float x, float& most) {
  const float a = fabsf(x);
  const bool over = a > C::kReach;
  if (a <= C::kReach) most = fmaxf(most, a);
  if (over) most = C::kReach;
  return over ? copysignf(C::kReach, x) : x;
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
      x[2 * i] = within<C>(T::low(piece[i]), most);
      x[2 * i + 1] = within<C>(T::high(piece[i]), most);
    }
#pragma unroll
    for (int o = kRowLanes<D> / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o));
    const int e = row_exponent<F, T>(most);
    const float down = power_of_two(-e);
    const v2u w = {encode4<F>(x[0] * down, x[1] * down, x[2] * down, x[3] * down), encode4<F>(x[4] * down, x[5] * down, x[6] * down, x[7] * down)};
    if (valid) {
      *reinterpret_cast<v2u*>(codes + (size_t)row * D + 8 * lane) = w;
      if (lane == 0) exps[row] = (signed char)e;
    }
  }
}

template <typename T, KvFormat F, int D>
__global__ __launch_bounds__(kKvThreads) void kv_write_kernel(const typename T::scalar* __restrict__ keys, const typename T::scalar* __restrict__ values,
                                                              KvStrides st, KvPages pages, KvBatch batch, long long items) {
  constexpr int L = kRowLanes<D>;
  const long long item = ((long long)blockIdx.x * kKvThreads + threadIdx.x) / L;
  const int lane = threadIdx.x % L;
  const bool in = item < items && lane < D / 8;
  const long long it = min(item, items - 1);
  const int token = (int)(it / pages.heads), h = (int)(it - (long long)token * pages.heads);
  v4u k = {0, 0, 0, 0}, v = {0, 0, 0, 0};
  if (in) {
    k = *reinterpret_cast<const v4u*>(keys + token * st.k_token + h * st.k_head + 8 * lane);
    v = *reinterpret_cast<const v4u*>(values + token * st.v_token + h * st.v_head + 8 * lane);
  }
  const KvPlace p = kv_place(batch, pages.pages, pages.heads, pages.page_shift, token, h);
  write_row<T, F, D>(k, pages.k, pages.k_exps, p.row, lane, in && p.valid);
  write_row<T, F, D>(v, pages.v, pages.v_exps, p.row, lane, in && p.valid);
}

// T: the type that the cache came from (F == kSame: that it holds), Out: what is written.
template <typename T, KvFormat F, typename Out, int D>
__device__ __forceinline__ void read_row(const unsigned char* codes, const signed char* exps, long long row, int lane, bool valid, Out* out) {
  float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if constexpr (F == kSame) {
    v4u piece = {0, 0, 0, 0};
    if (valid) piece = *reinterpret_cast<const v4u*>(codes + (size_t)row * (2 * D) + 16 * lane);
    if constexpr (std::is_same<Out, typename T::scalar>::value) {
      *reinterpret_cast<v4u*>(out) = piece;
      return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = T::low(piece[i]);
      x[2 * i + 1] = T::high(piece[i]);
    }
  } else {
    v2u w = {0, 0};
    float up = 0.0f;
    if (valid) {
      w = *reinterpret_cast<const v2u*>(codes + (size_t)row * D + 8 * lane);
      up = power_of_two(exps[row]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (F == kInt8) {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[4 * i + j] = int8_code(w[i], j) * up;
      } else {
        x[4 * i] = __builtin_amdgcn_cvt_f32_fp8((int)w[i], 0) * up;
        x[4 * i + 1] = __builtin_amdgcn_cvt_f32_fp8((int)w[i], 1) * up;
        x[4 * i + 2] = __builtin_amdgcn_cvt_f32_fp8((int)w[i], 2) * up;
        x[4 * i + 3] = __builtin_amdgcn_cvt_f32_fp8((int)w[i], 3) * up;
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

template <typename T, KvFormat F, typename Out, int D>
__global__ __launch_bounds__(kKvThreads) void kv_read_kernel(KvPages pages, KvBatch batch, Out* __restrict__ keys, Out* __restrict__ values,
                                                             long long items) {
  constexpr int L = kRowLanes<D>;
  const long long item = ((long long)blockIdx.x * kKvThreads + threadIdx.x) / L;
  const int lane = threadIdx.x % L;
  const long long it = min(item, items - 1);
  const int token = (int)(it / pages.heads), h = (int)(it - (long long)token * pages.heads);
  const KvPlace p = kv_place(batch, pages.pages, pages.heads, pages.page_shift, token, h);
  if (item >= items || lane >= D / 8 || !p.owned) return;
  read_row<T, F, Out, D>(pages.k, pages.k_exps, p.row, lane, p.valid, keys + it * D + 8 * lane);
  read_row<T, F, Out, D>(pages.v, pages.v_exps, p.row, lane, p.valid, values + it * D + 8 * lane);
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

template <int D>
static int kv_grid(const char* who, long long items, unsigned* blocks) {
  const long long n = (items * kRowLanes<D> + kKvThreads - 1) / kKvThreads;
  if (n > INT_MAX) return fail(FTK_ERR_UNSUPPORTED_SHAPE, "%s: too many rows for one launch", who);
  *blocks = (unsigned)n;
  return FTK_OK;
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
    unsigned blocks;
    if (int bad = kv_grid<D>(who, items, &blocks)) return bad;
    hipLaunchKernelGGL((kv_write_kernel<T, F, D>), dim3(blocks), dim3(kKvThreads), 0, (hipStream_t)stream, (const typename T::scalar*)keys,
                       (const typename T::scalar*)values, st, p, b, items);
    return check_launch("kv_write_kernel");
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
    unsigned blocks;
    if (int bad = kv_grid<D>(who, items, &blocks)) return bad;
    auto launch = [&](auto out) -> int {
      using Out = decltype(out);
      hipLaunchKernelGGL((kv_read_kernel<T, F, Out, D>), dim3(blocks), dim3(kKvThreads), 0, (hipStream_t)stream, p, b, (Out*)keys, (Out*)values, items);
      return check_launch("kv_read_kernel");
    };
    if (type == FTK_F32) return launch(0.0f);
    if constexpr (F == kSame) return launch(typename T::scalar{});
    else return type == FTK_F16 ? launch(_Float16{}) : launch(__bf16{});
  });
}

}  // extern "C"
