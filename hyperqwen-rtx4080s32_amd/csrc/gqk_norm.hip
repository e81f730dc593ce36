// gqk_norm.hip - the residual's addition and the RMS norm of whole rows, in 16 bits or in 8 with scales.
//
//   s = x + r,   r' = s rounded to the type,   y_i = s_i rsqrt(mean(s^2) + eps) w_i       (w_i, or 1 + w_i; no weight: 1)
//   in e4m3:  scale = max |y| / 448 over the row or each group of columns,  out = y / scale
//
// The norm is taken of s in 32 bits, not of what r' keeps of it.
#include <algorithm>
#include "gqk_decode.h"

namespace gqk {
namespace {

struct NormArgs {
  const void *x, *r, *w;
  int64_t x_row, r_row, out_row, or_row;
  void *out, *out_r;
  float* scale;
  int64_t rows, row0;   // row0: the launch's first
  int dim, group;       // group 0: the row
  int weight_f32, unit_offset;
  float eps;
};

// Up to eight values of a row: 16 bytes at any address of the type (unaligned 16-byte accesses are the hardware's own), the row's last
// ones one by one.  STREAM: lines that leave the caches first.
typedef uint32_t any4 __attribute__((ext_vector_type(4), aligned(2)));
template <bool STREAM, typename T> __device__ __forceinline__ void load_some(const T* p, int n, T* v) {
  if (n >= 8) {
    if constexpr (STREAM && sizeof(T) == 2) {
      const any4 x = __builtin_nontemporal_load((const any4*)p);
      __builtin_memcpy(v, &x, 16);
    } else {
      __builtin_memcpy(v, p, 8 * sizeof(T));
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < n ? p[e] : (T)0.f;
  }
}
template <bool STREAM, typename T> __device__ __forceinline__ void store_some(T* p, int n, const float* x) {
  T v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = from_f<T>(x[e]);
  if (n >= 8) {
    any4 y;
    __builtin_memcpy(&y, v, 16);
    if constexpr (STREAM) __builtin_nontemporal_store(y, (any4*)p);
    else *(any4*)p = y;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) p[e] = v[e];
  }
}
template <bool STREAM> __device__ __forceinline__ void store_some(fp8_t* p, int n, const float* x) {
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = x[e] != x[e] ? x[e] : fminf(fmaxf(x[e], -kFp8Max), kFp8Max);
  int w[2] = {0, 0};
  w[0] = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], w[0], false);
  w[0] = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], w[0], true);
  w[1] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4], v[5], w[1], false);
  w[1] = __builtin_amdgcn_cvt_pk_fp8_f32(v[6], v[7], w[1], true);
  if (n >= 8) {
    __builtin_memcpy(p, w, 8);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) p[e].v = (uint8_t)(w[e >> 2] >> (8 * (e & 3)));
  }
}

// The largest |y| as bits: NaN's are above infinity's, so a NaN wins.
__device__ __forceinline__ uint32_t wave_max(uint32_t x, int lanes) {
  for (int o = 1; o < lanes; o <<= 1) x = max(x, (uint32_t)__shfl_xor((int)x, o));
  return x;
}

// What the type's largest value stands for: a maximum below 2^-100 counts as that (a row of zeros is zeros times it).
__device__ __forceinline__ float top_of(uint32_t bits) { return __builtin_bit_cast(float, max(bits, 27u << 23)); }

// TR threads take a row, eight columns of it at a time; a row stays in registers from its one load to its store.  One pass over the bytes,
// which bound it: 8191 rows of 5120, 336 MB in 58 us (5.8 TB/s; with lines that stay in the caches 85, with a wave for a row 78 and 109),
// to 8 bits 294 MB in 52 (5.7); 96 rows of 17408 8 us, of one row 3: a launch and three trips to memory.
template <typename T, typename O, int TR, int NC, bool STREAM>
__global__ __launch_bounds__(TR) void add_norm_kernel(NormArgs a) {
  constexpr bool F8 = sizeof(O) == 1;
  constexpr int W = TR / 64;   // waves of a row
  __shared__ float part[2][16];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = a.row0 + blockIdx.x;
  const int tid = threadIdx.x, dim = a.dim;
  const T* x = (const T*)a.x + row * a.x_row;
  const T* r = (const T*)a.r + row * a.r_row;
  float s[NC][8];
  {
    T vx[NC][8], vr[NC][8];
#pragma unroll
    for (int i = 0; i < NC; ++i) load_some<STREAM>(x + (int64_t)(i * TR + tid) * 8, dim - (i * TR + tid) * 8, vx[i]);
    if (a.r)
#pragma unroll
      for (int i = 0; i < NC; ++i) load_some<STREAM>(r + (int64_t)(i * TR + tid) * 8, dim - (i * TR + tid) * 8, vr[i]);
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) s[i][e] = to_f(vx[i][e]) + (a.r ? to_f(vr[i][e]) : 0.f);
  }
  float w[NC][8];   // on their way while the row is summed up
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int d = (i * TR + tid) * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) w[i][e] = 1.f;
    if (!a.w) continue;
    if (a.weight_f32) {
      load_some<false>((const float*)a.w + d, dim - d, w[i]);
    } else {
      T t[8];
      load_some<false>((const T*)a.w + d, dim - d, t);
#pragma unroll
      for (int e = 0; e < 8; ++e) w[i][e] = to_f(t[e]);
    }
  }
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < NC; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      ss += s[i][e] * s[i][e];
      w[i][e] += a.unit_offset ? 1.f : 0.f;
    }
  if (a.out_r)   // after the row's loads, before any of its threads' other stores: it may be x or r
#pragma unroll
    for (int i = 0; i < NC; ++i)
      store_some<STREAM>((T*)a.out_r + row * a.or_row + (int64_t)(i * TR + tid) * 8, dim - (i * TR + tid) * 8, s[i]);
  ss = lane_sum<32>(ss);
  ss += __shfl_xor(ss, 32);
  if constexpr (W > 1) {
    if ((tid & 63) == 0) part[0][wave] = ss;
    __syncthreads();
    ss = 0.f;
#pragma unroll
    for (int k = 0; k < W; ++k) ss += part[0][k];
  }
  const float f = rsqrtf(ss / dim + a.eps);
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int d = (i * TR + tid) * 8, n = dim - d;
    if (n <= 0) continue;
#pragma unroll
    for (int e = 0; e < 8; ++e) s[i][e] = e < n ? s[i][e] * f * w[i][e] : 0.f;
    if constexpr (!F8) store_some<STREAM>((O*)a.out + row * a.out_row + d, n, s[i]);
  }
  if constexpr (F8) {
    uint32_t top[NC], all = 0;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      top[i] = 0;
      if ((i * TR + tid) * 8 < dim)
#pragma unroll
        for (int e = 0; e < 8; ++e) top[i] = max(top[i], __builtin_bit_cast(uint32_t, s[i][e]) & 0x7fffffffu);
      all = max(all, top[i]);
    }
    if (a.group) {   // a group's columns are neighbouring lanes'
      const int lanes = a.group >> 3, groups = dim / a.group;
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        top[i] = wave_max(top[i], lanes);
        const int d = (i * TR + tid) * 8;
        if (d < dim && (tid & (lanes - 1)) == 0) a.scale[row * groups + d / a.group] = top_of(top[i]) / kFp8Max;
      }
    } else {
      all = wave_max(all, 64);
      if constexpr (W > 1) {
        if ((tid & 63) == 0) part[1][wave] = __builtin_bit_cast(float, all);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < W; ++k) all = max(all, __builtin_bit_cast(uint32_t, part[1][k]));
      }
#pragma unroll
      for (int i = 0; i < NC; ++i) top[i] = all;
      if (tid == 0) a.scale[row] = top_of(all) / kFp8Max;
    }
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int d = (i * TR + tid) * 8, n = dim - d;
      if (n <= 0) continue;
      const float inv = kFp8Max / top_of(top[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[i][e] *= inv;
      store_some<STREAM>((O*)a.out + row * a.out_row + d, n, s[i]);
    }
  }
}

// A launch has fewer than 2^32 threads: more rows than that go in turns.
template <typename T, typename O, int TR, bool STREAM>
void launch(const NormArgs& all, hipStream_t st) {
  constexpr int64_t most = 0xffffffffll / TR;
  const int nc = (all.dim + 8 * TR - 1) / (8 * TR);
  NormArgs a = all;
  for (; a.row0 < a.rows; a.row0 += most) {
    const dim3 grid((unsigned)std::min(most, a.rows - a.row0));
    if (nc <= 1) add_norm_kernel<T, O, TR, 1, STREAM><<<grid, TR, 0, st>>>(a);
    else if (nc == 2) add_norm_kernel<T, O, TR, 2, STREAM><<<grid, TR, 0, st>>>(a);
    else if (nc == 3) add_norm_kernel<T, O, TR, 3, STREAM><<<grid, TR, 0, st>>>(a);
    else add_norm_kernel<T, O, TR, 4, STREAM><<<grid, TR, 0, st>>>(a);
  }
}

// 1024 threads to a row where a thread of 256 would have more than four chunks of it, or in short batches more than one (512 rows of 5120: 8.0
// -> 7.2 us).  What passes the caches by far leaves them first (2048 rows of 5120, 84 MB: 22.0 -> 19.6; 1024 rows the same either way).
template <typename T, typename O>
void launch(const NormArgs& a, hipStream_t st) {
  const bool wide = a.dim > 8192 || (a.rows < 1024 && a.dim > 2048);
  if (a.rows * a.dim >= 8 << 20) {
    if (wide) launch<T, O, 1024, true>(a, st);
    else launch<T, O, 256, true>(a, st);
  } else {
    if (wide) launch<T, O, 1024, false>(a, st);
    else launch<T, O, 256, false>(a, st);
  }
}

}  // namespace
}  // namespace gqk

using namespace gqk;

extern "C" int gqk_add_rms_norm(const void* x, int64_t x_row, const void* residual, int64_t residual_row, int dtype, int64_t rows,
                                int dim, const void* weight, int weight_dtype, float eps, int flags, void* out, int64_t out_row,
                                int out_dtype, float* scale, int group, void* out_residual, int64_t out_residual_row, void* stream) {
  const char* what = "add_rms_norm";
  if (dtype != GQK_DTYPE_BF16 && dtype != GQK_DTYPE_F16) return decode_fail(GQK_ERR_ARG, "%s: dtype %d", what, dtype);
  const bool f8 = out_dtype == GQK_DTYPE_FP8;
  if (!f8 && out_dtype != dtype) return decode_fail(GQK_ERR_ARG, "%s: rows of type %d to outputs of type %d", what, dtype, out_dtype);
  if (weight && weight_dtype != dtype && weight_dtype != GQK_DTYPE_F32)
    return decode_fail(GQK_ERR_ARG, "%s: weights of type %d", what, weight_dtype);
  if (!weight && flags) return decode_fail(GQK_ERR_ARG, "%s: an offset without weights", what);
  if (rows < 0 || rows > 0x7fffffff || dim < 1 || dim > GQK_NORM_MAX_DIM)
    return decode_fail(GQK_ERR_SHAPE, "%s: %lld rows of %d (1 to %d)", what, (long long)rows, dim, GQK_NORM_MAX_DIM);
  if (f8 ? (group && (group < 32 || group > 512 || (group & (group - 1)) || dim % group)) : group != 0)
    return decode_fail(GQK_ERR_SHAPE, "%s: groups of %d columns of %d (0, or a power of two from 32 to 512 that divides them; for 8 bits)",
                       what, group, dim);
  if (rows == 0) return GQK_OK;
  if (!x || !out || (f8 && !scale) || (out_residual && !residual)) return decode_fail(GQK_ERR_ARG, "%s: null pointer", what);
  if (rows > 1 && (x_row < dim || out_row < dim || (residual && residual_row < dim) || (out_residual && out_residual_row < dim)))
    return decode_fail(GQK_ERR_SHAPE, "%s: rows of %d overlap", what, dim);
  if ((((uintptr_t)x | (uintptr_t)residual | (uintptr_t)out_residual | (f8 ? 0 : (uintptr_t)out)) & 1) ||
      (uintptr_t)weight % (weight_dtype == GQK_DTYPE_F32 ? 4 : 2) || (uintptr_t)scale & 3)
    return decode_fail(GQK_ERR_SHAPE, "%s: unaligned values", what);
  NormArgs a{};
  a.x = x; a.r = residual; a.w = weight; a.x_row = x_row; a.r_row = residual_row; a.out_row = out_row; a.or_row = out_residual_row;
  a.out = out; a.out_r = out_residual; a.scale = scale; a.rows = rows; a.dim = dim; a.group = group;
  a.weight_f32 = weight_dtype == GQK_DTYPE_F32; a.unit_offset = flags & GQK_ROPE_UNIT_OFFSET; a.eps = eps;
  const hipStream_t st = (hipStream_t)stream;
  const bool bf = dtype == GQK_DTYPE_BF16;
  if (bf && f8) launch<bf16_t, fp8_t>(a, st);
  else if (bf) launch<bf16_t, bf16_t>(a, st);
  else if (f8) launch<f16_t, fp8_t>(a, st);
  else launch<f16_t, f16_t>(a, st);
  return decode_launched(what);
}
