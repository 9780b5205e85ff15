// What the kernels on a paged cache of keys and values share: the batch (which packed rows are whose, where a position
// lies), the element types, and the codes of a cache in 8 bits.
#pragma once

#include <limits.h>

#include "fa_common.h"
#include "ftk_common.h"

namespace ftk {

typedef __bf16 v2b __attribute__((ext_vector_type(2)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef int v2i __attribute__((ext_vector_type(2)));

// ---- the batch --------------------------------------------------------------

// Arrays on the device whose contents nobody has checked: every use below clamps what it takes from them.
struct KvBatch {
  const int* table;    // [sequences, width]
  const int* lens;     // [sequences]
  const int* starts;   // [sequences + 1]
  int sequences, width, tokens;
};

struct KvPages {
  unsigned char *k, *v;          // [pages, heads, 2^page_shift, D]
  signed char *k_exps, *v_exps;  // [pages, heads, 2^page_shift], 8-bit types only
  int pages, heads, page_shift;
};

// 32-bit loads through the scalar cache; the address is the same in every lane.
__device__ __forceinline__ int load_uniform(const int* p, long long i) {
  typedef const __attribute__((address_space(4))) int* constant_int;
  return ((constant_int)(uintptr_t)p)[i];
}

// Positions that the table has room for.
__device__ __forceinline__ int kv_capacity(const KvBatch& b, int page_shift) {
  const long long c = (long long)b.width << page_shift;
  return c > INT_MAX ? INT_MAX : (int)c;
}

// How many of the first `n` values of a non-decreasing function of the index are at most x: 64 at a time, a lane each.
template <typename F>
__device__ __forceinline__ int count_at_most(int n, long long x, F&& value) {
  const int lane = threadIdx.x & 63;
  int count = 0;
  for (int i = 0; i < n; i += 64) {
    const bool in = i + lane < n;
    count += __popcll(__builtin_amdgcn_ballot_w64(in && value(i + lane) <= x));
  }
  return count;
}

// The position of packed row `start`, of those from 0 on, in a sequence whose new tokens end at row `end`, which may lie behind the packed rows.
__device__ __forceinline__ int first_position(int len, int start, int end) { return len - max(end - start, 0); }

// The new tokens of sequence b: packed rows [start, start + n), row start + t at position first + t (which may be negative or
// past what the table has room for).
struct KvChunk {
  int start, n, first, len;
};
__device__ __forceinline__ KvChunk kv_chunk(const KvBatch& batch, int b) {
  KvChunk c;
  c.start = min(max(load_uniform(batch.starts, b), 0), batch.tokens);
  const int end = load_uniform(batch.starts, b + 1);
  c.n = min(max(end, c.start), batch.tokens) - c.start;
  c.len = max(load_uniform(batch.lens, b), 0);
  c.first = first_position(c.len, c.start, end);
  return c;
}

__device__ __forceinline__ int kv_page(const KvBatch& batch, int b, int index, int pages) {
  return min(max(load_uniform(batch.table, (long long)b * batch.width + index), 0), pages - 1);
}

// ---- element types ------------------------------------------------------------

struct Half {
  using scalar = _Float16;
  using v8 = v8h;
  static constexpr unsigned kExpMask = 0x7c00;
  static __device__ __forceinline__ v4f mma16(v8 a, v8 b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ v16f mma32(v8 a, v8 b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ unsigned pack(float a, float b) {
    const v2h p = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(unsigned, p);
  }
  static __device__ __forceinline__ float low(unsigned p) { return (float)__builtin_bit_cast(v2h, p)[0]; }
  static __device__ __forceinline__ float high(unsigned p) { return (float)__builtin_bit_cast(v2h, p)[1]; }
};

struct Brain {
  using scalar = __bf16;
  using v8 = v8b;
  static constexpr unsigned kExpMask = 0x7f80;
  static __device__ __forceinline__ v4f mma16(v8 a, v8 b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ v16f mma32(v8 a, v8 b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ unsigned pack(float a, float b) {
    const v2b p = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(unsigned, p);
  }
  static __device__ __forceinline__ float low(unsigned p) { return __uint_as_float(p << 16); }
  static __device__ __forceinline__ float high(unsigned p) { return __uint_as_float(p & 0xffff0000u); }
};

// ---- codes of 8 bits ------------------------------------------------------------
//
// A row of D elements is held as D codes and one exponent e: element = code * 2^e, e the least integer with
// max |row| <= kTop * 2^e, but not below a floor.  With a power of two for a scale, code * 2^e and the quotient
// x * 2^-e are exact, so the code is the nearest one (the even one of two) however it is computed, and what is read back is a value
// that the 16-bit type it came from can hold: rows are first clamped to the largest such value (kReach), and for fp16 the floor
// puts the finest codes 2^-24 apart, as fp16's own finest values are.  (A scale max|row| / 127 in fp32 would keep up to
// one bit more of int8 rows; every product with it would be a rounding.)

enum KvFormat { kSame, kE4m3, kInt8 };

template <KvFormat F, typename T>
struct Codes;
template <typename T>
struct Codes<kE4m3, T> {
  static constexpr bool half = std::is_same<T, Half>::value;
  static constexpr int kTopExp = 8;                  // 448 = 1.75 * 2^8
  static constexpr unsigned kTopMantissa = 0x600000;
  static constexpr int kLeast = half ? -15 : -100;
  static constexpr float kReach = half ? 61440.0f : 3.1901471898837979e38f;   // 1.875 * 2^15, * 2^127
};
template <typename T>
struct Codes<kInt8, T> {
  static constexpr bool half = std::is_same<T, Half>::value;
  static constexpr int kTopExp = 6;                  // 127 = 1.984375 * 2^6
  static constexpr unsigned kTopMantissa = 0x7e0000;
  static constexpr int kLeast = half ? -24 : -100;
  static constexpr float kReach = half ? 65024.0f : 3.3762391092936862e38f;   // 127 * 2^9, * 2^121
};

// The exponent of a row whose largest magnitude (within the reach) is `most`.
template <KvFormat F, typename T>
__device__ __forceinline__ int row_exponent(float most) {
  using C = Codes<F, T>;
  const int e = (int)((__float_as_uint(most) + (0x7fffffu - C::kTopMantissa)) >> 23) - 127 - C::kTopExp;
  return max(e, C::kLeast);   // (zero and subnormal rows are far below the floor)
}

__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }   // -126 .. 127

// Four codes of scaled values, in memory order.
template <KvFormat F>
__device__ __forceinline__ unsigned encode4(float a, float b, float c, float d) {
  if constexpr (F == kE4m3) {
    int p = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, p, true);
  } else {
    // x + 1.5 * 2^23 rounds x to the nearest whole number, the even one of two, which the low bits then hold (a NaN's are zeros)
    const auto bits = [](float x) { return __float_as_uint(x + 12582912.0f); };
    const unsigned low = __builtin_amdgcn_perm(bits(b), bits(a), 0x0c0c0400u), high = __builtin_amdgcn_perm(bits(d), bits(c), 0x04000c0cu);
    return low | high;
  }
}

// Two of four codes (the lower or the upper pair) as fp32 pairs of codes.
__device__ __forceinline__ float int8_code(unsigned w, int i) { return (float)(signed char)(w >> (8 * i)); }

// Eight codes as eight elements of T times `scale`, a power of two; of int8 in fp16 one that fits_half.
template <typename T, KvFormat F>
__device__ __forceinline__ typename T::v8 decode8(v2u w, float scale) {
  unsigned r[4];
  if constexpr (F == kE4m3) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (std::is_same<T, Half>::value) {
        r[2 * i] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w[i], scale, false));
        r[2 * i + 1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w[i], scale, true));
      } else {
        r[2 * i] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w[i], scale, false));
        r[2 * i + 1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w[i], scale, true));
      }
    }
  } else if constexpr (std::is_same<T, Half>::value) {
    // 0x6400 | u is 1024 + u for a byte u = code + 128: two codes in a byte permutation, a subtraction and, unless it is 1, the scale,
    // where a conversion each takes nine instructions for four
    const v2h middle = {(_Float16)1152.0f, (_Float16)1152.0f}, times = {(_Float16)scale, (_Float16)scale};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const unsigned u = w[i] ^ 0x80808080u;
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const unsigned pair = __builtin_amdgcn_perm(0x64646464u, u, p ? 0x04030402u : 0x04010400u);
        v2h h = __builtin_bit_cast(v2h, pair) - middle;
        if (!(__builtin_constant_p(scale) && scale == 1.0f)) h = h * times;
        r[2 * i + p] = __builtin_bit_cast(unsigned, h);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int p = 0; p < 2; ++p) r[2 * i + p] = T::pack(int8_code(w[i], 2 * p) * scale, int8_code(w[i], 2 * p + 1) * scale);
  }
  const v4u all = {r[0], r[1], r[2], r[3]};
  return __builtin_bit_cast(typename T::v8, all);
}

// Whether code * 2^e is an element of fp16, or rounds to one, by a product in fp16: 2^e is a number of fp16, and no code times it is beyond fp16's largest.
template <KvFormat F>
__device__ __forceinline__ bool fits_half(int e) { return e >= -24 && e <= (F == kInt8 ? 9 : 7); }

// decode8 for any power of two: each element rounded to T once, infinite beyond T's largest.  (Codes that were written from bf16, attended to in fp16.)
template <typename T, KvFormat F>
__device__ __forceinline__ typename T::v8 decode8_rounded(v2u w, float scale) {
  unsigned r[4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float x[4];
    if constexpr (F == kE4m3) {
      x[0] = __builtin_amdgcn_cvt_f32_fp8((int)w[i], 0);
      x[1] = __builtin_amdgcn_cvt_f32_fp8((int)w[i], 1);
      x[2] = __builtin_amdgcn_cvt_f32_fp8((int)w[i], 2);
      x[3] = __builtin_amdgcn_cvt_f32_fp8((int)w[i], 3);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = int8_code(w[i], j);
    }
    r[2 * i] = T::pack(x[0] * scale, x[1] * scale);
    r[2 * i + 1] = T::pack(x[2] * scale, x[3] * scale);
  }
  const v4u all = {r[0], r[1], r[2], r[3]};
  return __builtin_bit_cast(typename T::v8, all);
}

// ---- host side -------------------------------------------------------------------

int check_kv_pages(const char* who, const ftk_kv_pages* p, KvPages* out);
int check_kv_batch(const char* who, const ftk_kv_batch* b, KvBatch* out);
inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Calls f(type tag, format constant, head size constant) for a 16-bit type and a cache that fits it.
template <typename F>
int with_kv_types(int type, int cache, int D, F&& f) {
  auto with_d = [&](auto t, auto c) -> int {
    switch (D) {
      case 32: return f(t, c, std::integral_constant<int, 32>{});
      case 64: return f(t, c, std::integral_constant<int, 64>{});
      case 96: return f(t, c, std::integral_constant<int, 96>{});
      default: return f(t, c, std::integral_constant<int, 128>{});
    }
  };
  auto with_c = [&](auto t) -> int {
    switch (cache) {
      case FTK_E4M3: return with_d(t, std::integral_constant<KvFormat, kE4m3>{});
      case FTK_INT8: return with_d(t, std::integral_constant<KvFormat, kInt8>{});
      default: return with_d(t, std::integral_constant<KvFormat, kSame>{});
    }
  };
  return type == FTK_BF16 ? with_c(Brain{}) : with_c(Half{});
}

}  // namespace ftk
