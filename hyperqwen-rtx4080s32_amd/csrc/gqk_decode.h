// gqk_decode.h - what the kernels around the linear path share (adapters, norm and rotation, paged
// attention, page copies): the 16-bit types' conversions, indexes of either width, error reporting.
#pragma once
#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>
#include "gguf_hip.h"
#include "gqk_common.h"

namespace gqk {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;
struct fp8_t { uint8_t v; };   // OCP e4m3: no infinities, largest 448

template <typename T> __device__ __forceinline__ float to_f(T v) { return (float)v; }
template <> __device__ __forceinline__ float to_f(fp8_t v) { return __builtin_amdgcn_cvt_f32_fp8(v.v, 0); }

// the largest finite value of e4m3: larger ones are stored as it, as the type has no infinity
constexpr float kFp8Max = 448.f;

template <typename T> __device__ __forceinline__ T from_f(float v) { return (T)v; }
template <> __device__ __forceinline__ fp8_t from_f(float v) {
  v = v != v ? v : fminf(fmaxf(v, -kFp8Max), kFp8Max);
  return fp8_t{(uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(v, v, 0, false)};
}

template <int CTRL> __device__ __forceinline__ float dpp_add(float x) {
  return x + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, false));
}
// the sum over 8, 16 or 32 neighbouring lanes: across pairs, quads, halves of a row and a row by DPP, then over two rows
template <int LPH> __device__ __forceinline__ float lane_sum(float x) {
  x = dpp_add<0xB1>(x);    // quad_perm 1, 0, 3, 2
  x = dpp_add<0x4E>(x);    // quad_perm 2, 3, 0, 1
  x = dpp_add<0x141>(x);   // row_half_mirror
  if constexpr (LPH >= 16) x = dpp_add<0x140>(x);   // row_mirror
  if constexpr (LPH >= 32) x += __shfl_xor(x, 16);
  return x;
}

// element i of an index array of 32-bit or 64-bit integers
__device__ __forceinline__ int64_t index_at(const void* p, int wide, int64_t i) {
  return wide ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
}

inline int decode_fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  gqk_set_last_error(buf);
  return code;
}

inline int decode_launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? GQK_OK : decode_fail(GQK_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

// compute units of the current device (256 where none is visible)
int device_cus();

// the argument checks of a cache's pages; 0 or the error that was reported
int check_pages(const char* what, const gqk_pages* p, int q_dtype);

}  // namespace gqk
