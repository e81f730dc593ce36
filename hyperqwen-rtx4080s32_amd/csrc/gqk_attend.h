// gqk_attend.h - what the attention kernels share: operands' types, the 8-bit types' conversion, the softmax's running sums.
#pragma once
#include "gqk_decode.h"

namespace gqk {
namespace {

typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

// A weight is 2^(score - maximum + kLift): fp16 uses its whole range, so that weights keep their relative precision down to 2^-29 of
// the heaviest and none is lost above 2^-40 (not lifted they do to 2^-14, and a long flat tail of them, each lighter than that, lost
// up to all of its weight).  bf16 has fp32's exponents.
template <typename T> constexpr float kLift = __is_same(T, f16_t) ? 15.f : 0.f;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

// two e4m3 values (bytes 0, 1 or 2, 3 of x) as two values of T, exactly
template <bool HI> __device__ __forceinline__ uint32_t widen(uint32_t x, bf16_t) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.f, HI));
}
template <bool HI> __device__ __forceinline__ uint32_t widen(uint32_t x, f16_t) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.f, HI));
}
template <typename T> __device__ __forceinline__ v4u widen8(uint32_t lo, uint32_t hi) {
  return v4u{widen<false>(lo, T{}), widen<true>(lo, T{}), widen<false>(hi, T{}), widen<true>(hi, T{})};
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  typedef T v2 __attribute__((ext_vector_type(2)));
  v2 p;
  p[0] = (T)lo;
  p[1] = (T)hi;
  return __builtin_bit_cast(uint32_t, p);
}

// Splits of `chunk` keys of the keys [start, len), one at least.  (len - start + chunk can pass 31 bits where the sequence is long.)
__device__ __forceinline__ int splits_of(int start, int len, int chunk) { return len > start ? (len - start - 1) / chunk + 1 : 1; }

// The exponent's base of a running maximum: nothing was seen yet (-inf) must not become -inf - -inf.
__device__ __forceinline__ float base_of(float m) { return m == -__builtin_huge_valf() ? 0.f : m; }

// Partial sums over a split's keys, relative to its maximum (both lifted alike), added up in order.
struct Joined {
  float m = -__builtin_huge_valf(), l = 0.f;
  v4f o{0.f, 0.f, 0.f, 0.f};
  __device__ __forceinline__ void add(v2u stat, v4u sums) {
    float s[2];
    __builtin_memcpy(s, &stat, 8);
    const float mn = fmaxf(m, s[0]), mb = base_of(mn);
    const float f = __builtin_amdgcn_exp2f(m - mb), g = __builtin_amdgcn_exp2f(s[0] - mb);
    m = mn;
    l = l * f + s[1] * g;
    o = o * f + __builtin_bit_cast(v4f, sums) * g;
  }
};

// key / page_size = 2 key magic >> 32 >> shift for keys below 2^31: 2^(31 + bits) / page_size rounded up fits 32 bits, its excess times a
// key stays below 2^(31 + bits)
struct PageDivisor {
  uint32_t magic;
  int shift;
};
inline PageDivisor page_divisor(int page_size) {
  int bits = 0;
  while (((int64_t)1 << bits) < page_size) ++bits;
  return {(uint32_t)((((uint64_t)1 << (31 + bits)) + page_size - 1) / page_size), bits};
}

}  // namespace
}  // namespace gqk
