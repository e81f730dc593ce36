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
