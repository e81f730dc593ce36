// gqk_rope.hip - the heads of queries and keys, normalized, rotated and stored in one pass.
//
//   n_i = x_i rsqrt(mean(x^2) + eps) w_i             (w_i, or 1 + w_i; no weight: n = x)
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t) (pairs (i, i + rot / 2) or (2 i, 2 i + 1) of the first rot dims)
//
// with cos t | sin t of pair i at [position][i] | [position][rot / 2 + i] of a table in 32 bits.  Keys
// and values of a token with a slot go into its page of the cache.
#include <algorithm>
#include "gqk_decode.h"

namespace gqk {
namespace {

struct RopeArgs {
  const void *q, *k, *v;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;
  const void *q_weight, *k_weight;
  const void* positions;
  const float* table;
  int64_t table_rows;
  void *out_q, *out_k;
  int64_t oq_row, oq_head, ok_row, ok_head;
  gqk_pages kv;
  const void* slots;
  int q_heads, k_heads, dim, rot, tokens;
  float eps;
  int wide_positions, wide_slots, unit_offset, interleaved, weight_f32, store;
};

// Any even rot, and tables or weights off 16 bytes: one wave per (token, head), q heads, k heads, then v heads (stored only); the
// normalized head in LDS.  The general form, not the fast one: it looks up a token's angles again for each head, and a wave has no
// second head on its way while it waits.  8191 tokens of 40 + 8 + 8 heads of 96 dims, 24 of them rotated, stored: 276 us (26 waves a CU, 56% of
// their time waiting), where the vector form takes 49 (32 rotated) and the bytes 37 at a copy's rate; one token 4.2 us, as there.
template <typename T, typename C>
__global__ __launch_bounds__(64) void rope_any_kernel(RopeArgs a) {
  const int h = blockIdx.x, lane = threadIdx.x, D = a.dim;
  const int64_t t = blockIdx.y;
  const bool is_q = h < a.q_heads, is_v = h >= a.q_heads + a.k_heads;
  const int hh = is_q ? h : is_v ? h - a.q_heads - a.k_heads : h - a.q_heads;
  const T* x = is_q ? (const T*)a.q + t * a.q_row + hh * a.q_head
                    : is_v ? (const T*)a.v + t * a.v_row + hh * a.v_head : (const T*)a.k + t * a.k_row + hh * a.k_head;
  const void* w = is_q ? a.q_weight : is_v ? nullptr : a.k_weight;
  const float nan = __builtin_nanf("");
  __shared__ float n[256];
  float ss = 0.f;
  for (int d = lane; d < D; d += 64) ss += to_f(x[d]) * to_f(x[d]);
  for (int o = 32; o > 0; o >>= 1) ss += __shfl_xor(ss, o);
  const float r = w ? rsqrtf(ss / D + a.eps) : 1.f;
  for (int d = lane; d < D; d += 64) {
    const float wd = !w ? 1.f : (a.weight_f32 ? ((const float*)w)[d] : to_f(((const T*)w)[d])) + (a.unit_offset ? 1.f : 0.f);
    n[d] = to_f(x[d]) * r * wd;
  }
  __syncthreads();
  const int64_t pos = is_v ? 0 : index_at(a.positions, a.wide_positions, t);
  const bool in = pos >= 0 && pos < a.table_rows;
  const int64_t slot = a.store && !is_q ? index_at(a.slots, a.wide_slots, t) : -1;
  const bool keep = slot >= 0 && slot < (int64_t)a.kv.pages * a.kv.page_size;
  const int half = a.rot / 2;
  for (int d = lane; d < D; d += 64) {
    float y = n[d];
    if (!is_v && d < a.rot) {
      const int i = a.interleaved ? d >> 1 : d < half ? d : d - half;
      const bool second = a.interleaved ? d & 1 : d >= half;
      const float c = in ? a.table[pos * a.rot + i] : nan, s = in ? a.table[pos * a.rot + half + i] : nan;
      const float other = n[a.interleaved ? d ^ 1 : second ? d - half : d + half];
      y = second ? y * c + other * s : y * c - other * s;
    } else if (!is_v && !in) {
      y = nan;
    }
    if (is_q) ((T*)a.out_q)[t * a.oq_row + hh * a.oq_head + d] = from_f<T>(y);
    if (!is_q && !is_v && a.out_k) ((T*)a.out_k)[t * a.ok_row + hh * a.ok_head + d] = from_f<T>(y);
    if (keep) {
      const int64_t page = slot / a.kv.page_size, at = slot % a.kv.page_size;
      const float* sc = is_v ? a.kv.v_scale : a.kv.k_scale;
      C* to = is_v ? (C*)a.kv.v + page * a.kv.v_page + at * a.kv.v_token + hh * a.kv.v_head
                   : (C*)a.kv.k + page * a.kv.k_page + at * a.kv.k_token + hh * a.kv.k_head;
      to[d] = from_f<C>(sc ? y / sc[hh] : y);
    }
  }
}

typedef uint32_t v4u __attribute__((ext_vector_type(4)));
constexpr int kWaves = 4;
constexpr int64_t kTokens = 32768;   // of one launch

// x of eight dims
template <typename T> __device__ __forceinline__ void load8(const T* p, float* x) {
  T v[8];
  __builtin_memcpy(v, __builtin_assume_aligned(p, 8 * sizeof(T)), 8 * sizeof(T));
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = to_f(v[e]);
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float* x) {
  T v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = from_f<T>(x[e]);
  __builtin_memcpy(__builtin_assume_aligned(p, 8 * sizeof(T)), v, 8 * sizeof(T));
}
template <> __device__ __forceinline__ void store8(fp8_t* p, const float* x) {
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = x[e] != x[e] ? x[e] : fminf(fmaxf(x[e], -kFp8Max), kFp8Max);
  int lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4], v[5], hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6], v[7], hi, true);
  *(int2*)p = make_int2(lo, hi);
}

// Eight dims to a lane, DP / 8 lanes to a head, so that a wave reads 64 x 16 bytes of neighbouring heads at once.  A round
// is 64 LPH heads of one kind (queries, keys, values), the same for the whole wave; a token's waves deal its rounds.
// The rotation of a normalized head is  y = r (x A + x' B)  with x' the other dim of the pair, A = w cos and B = -+ w' sin:
// A and B are made once for a token and kept in registers, and r is the head's own.  Pairs that are rot / 2 apart meet
// by a shuffle of the packed values (rot a multiple of 16: a lane's dims have their partners in one other lane);
// interleaved pairs are a lane's own (rot a multiple of 8).  Arithmetic is in 32 bits, rounded once.  One pass over the bytes, which
// bound it: 8191 tokens of 40 + 8 + 8 heads of 128 dims, keys kept and stored, 256 MB in 56 us (4.6 TB/s, a copy's rate); one
// token 4.4 us, a launch and three dependent loads.
template <typename T, typename C, int DP, bool INTER>
__global__ __launch_bounds__(64 * kWaves) void rope_kernel(RopeArgs a, int waves) {
  constexpr int LPH = DP / 8, HPW = 64 / LPH;   // lanes of a head, heads of a round
  struct alignas(16) Raw { uint32_t w[4]; };
  const int64_t item = (int64_t)blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t t = item / waves;
  const int part = (int)(item - t * waves);
  if (t >= a.tokens) return;
  const int lane = threadIdx.x & 63, sub = lane & (LPH - 1), own = lane / LPH, d = sub * 8, D = a.dim, half = a.rot >> 1;
  const bool live = d < D;
  const int at = live ? d : 0;
  const float nan = __builtin_nanf("");
  const int rq = (a.q_heads + HPW - 1) / HPW, rk = (a.k_heads + HPW - 1) / HPW;
  const int rounds = rq + rk + (a.store ? (a.kv.heads + HPW - 1) / HPW : 0);
  // round i: the kind, the lane's head of it, whether there is one
  auto kind_of = [&](int i) { return i < rq ? 0 : i < rq + rk ? 1 : 2; };
  auto head_of = [&](int i, int kind) { return (kind == 0 ? i : kind == 1 ? i - rq : i - rq - rk) * HPW + own; };
  auto count_of = [&](int kind) { return kind == 0 ? a.q_heads : kind == 1 ? a.k_heads : a.kv.heads; };
  auto load = [&](int i) {
    Raw x{};
    const int kind = kind_of(i), h = head_of(i, kind);
    const T* base = kind == 0 ? (const T*)a.q + t * a.q_row : kind == 1 ? (const T*)a.k + t * a.k_row : (const T*)a.v + t * a.v_row;
    const int64_t stride = kind == 0 ? a.q_head : kind == 1 ? a.k_head : a.v_head;
    if (live && h < count_of(kind)) {
      const v4u z = __builtin_nontemporal_load((const v4u*)(base + h * stride + d));   // read once: 56.6 -> 55.2 us (8191 tokens)
      __builtin_memcpy(&x, &z, 16);
    }
    return x;
  };
  Raw next{};
  if (part < rounds) next = load(part);   // on its way while the angles are looked up
  const int64_t pos = index_at(a.positions, a.wide_positions, t);
  const bool in = pos >= 0 && pos < a.table_rows;
  const bool turned = live && d < a.rot, second = !INTER && d >= half;
  const int mate = INTER || !turned ? lane : second ? lane - half / 8 : lane + half / 8;
  float cs[8], sn[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) { cs[e] = in ? 1.f : nan; sn[e] = 0.f; }   // a position that is not in the table: NaN
  if (turned && in) {
    if constexpr (INTER) {
      const float4 c = *(const float4*)(a.table + pos * a.rot + (d >> 1)), s = *(const float4*)(a.table + pos * a.rot + half + (d >> 1));
      cs[0] = cs[1] = c.x; cs[2] = cs[3] = c.y; cs[4] = cs[5] = c.z; cs[6] = cs[7] = c.w;
      sn[0] = -s.x; sn[1] = s.x; sn[2] = -s.y; sn[3] = s.y; sn[4] = -s.z; sn[5] = s.z; sn[6] = -s.w; sn[7] = s.w;
    } else {
      const float* row = a.table + pos * a.rot + (second ? d - half : d);
      load8(row, cs);
      load8(row + half, sn);
#pragma unroll
      for (int e = 0; e < 8; ++e) sn[e] = second ? sn[e] : -sn[e];
    }
  }
  float A[2][8], B[2][8];   // of queries and of keys
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    // the wave's first round that is not before the kind's
    const int begin = k ? rq : 0, end = k ? rq + rk : rq, i = begin <= part ? part : part + (begin - part + waves - 1) / waves * waves;
    if (i >= end) continue;   // none of the kind
    const void* w = k ? a.k_weight : a.q_weight;
    float own_w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) own_w[e] = 1.f;
    if (w) {
      if (a.weight_f32) load8((const float*)w + at, own_w);
      else load8((const T*)w + at, own_w);
      if (a.unit_offset)
#pragma unroll
        for (int e = 0; e < 8; ++e) own_w[e] += 1.f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      A[k][e] = own_w[e] * cs[e];
      B[k][e] = (INTER ? own_w[e ^ 1] : __shfl(own_w[e], mate)) * sn[e];
    }
  }
  int64_t page = 0, place = 0;
  bool keep = false;
  if (a.store) {
    const int64_t slot = index_at(a.slots, a.wide_slots, t);
    const int64_t room = (int64_t)a.kv.pages * a.kv.page_size;
    keep = slot >= 0 && slot < room;
    if (keep) {
      page = room >> 32 ? slot / a.kv.page_size : (uint32_t)slot / (uint32_t)a.kv.page_size;   // a division in 64 bits costs
      place = slot - page * a.kv.page_size;
    }
  }
  for (int i = part; i < rounds; i += waves) {
    const Raw raw = next;
    if (i + waves < rounds) next = load(i + waves);   // no head is written by another's round, in place either
    const int kind = kind_of(i), h = head_of(i, kind);
    float y[8];
    T v[8];
    __builtin_memcpy(v, &raw, 16);
    if (kind == 2) {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = to_f(v[e]);
    } else {
      Raw other = raw;
      if constexpr (!INTER)
#pragma unroll
        for (int w = 0; w < 4; ++w) other.w[w] = turned ? __shfl(raw.w[w], mate) : 0;
      T o[8];
      __builtin_memcpy(o, &other, 16);
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss += to_f(v[e]) * to_f(v[e]);
      ss = lane_sum<LPH>(ss);
      const float r = (kind ? a.k_weight : a.q_weight) ? rsqrtf(ss / D + a.eps) : 1.f;
      auto turn = [&](const float (&fa)[8], const float (&fb)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          // what is not turned has no other: not 0 times one that is not finite
          const float z = INTER ? (turned ? to_f(v[e ^ 1]) : 0.f) : to_f(o[e]);
          y[e] = r * (to_f(v[e]) * fa[e] + z * fb[e]);
        }
      };
      if (kind == 0) turn(A[0], B[0]);
      else turn(A[1], B[1]);
    }
    if (!live || h >= count_of(kind)) continue;
    if (kind == 0) store8((T*)a.out_q + t * a.oq_row + h * a.oq_head + d, y);
    else if (kind == 1 && a.out_k) store8((T*)a.out_k + t * a.ok_row + h * a.ok_head + d, y);
    if (kind > 0 && keep) {
      const float* sc = kind == 2 ? a.kv.v_scale : a.kv.k_scale;
      C* to = kind == 2 ? (C*)a.kv.v + page * a.kv.v_page + place * a.kv.v_token + h * a.kv.v_head
                        : (C*)a.kv.k + page * a.kv.k_page + place * a.kv.k_token + h * a.kv.k_head;
      if (sc) {
        const float s = sc[h];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] /= s;
      }
      store8(to + d, y);
    }
  }
}

template <typename T, typename C, int DP>
void launch(const RopeArgs& a, bool inter, hipStream_t st) {
  constexpr int HPW = 512 / DP;   // heads of a round
  auto of = [](int heads) { return (heads + HPW - 1) / HPW; };
  const int rounds = of(a.q_heads) + of(a.k_heads) + (a.store ? of(a.kv.heads) : 0);
  // Waves of a token: one for each round until the launch has 4096 (16 a CU), then as many as make that, as a wave spends as
  // long on looking up a token's angles as on some rounds (8191 tokens of 14 rounds: 1 wave 55 us, 2 63, 4 75, 14 123)
  const int waves = std::max(1, std::min(rounds, 4096 / a.tokens));
  const dim3 grid((unsigned)(((int64_t)a.tokens * waves + kWaves - 1) / kWaves));
  if (inter) rope_kernel<T, C, DP, true><<<grid, 64 * kWaves, 0, st>>>(a, waves);
  else rope_kernel<T, C, DP, false><<<grid, 64 * kWaves, 0, st>>>(a, waves);
}

template <typename T, typename C>
void launch(const RopeArgs& a, hipStream_t st) {
  // whole lanes of pairs, tables and weights that take 16-byte loads: the vector form; else a wave per head
  const bool inter = a.interleaved;
  const uint64_t bits = (uintptr_t)a.table | (uintptr_t)a.q_weight | (uintptr_t)a.k_weight;
  if (a.rot % (inter ? 8 : 16) == 0 && !(bits & 15)) {
    if (a.dim <= 64) launch<T, C, 64>(a, inter, st);
    else if (a.dim <= 128) launch<T, C, 128>(a, inter, st);
    else launch<T, C, 256>(a, inter, st);
    return;
  }
  const int heads = a.q_heads + a.k_heads + (a.store ? a.kv.heads : 0);
  rope_any_kernel<T, C><<<dim3(heads, (unsigned)a.tokens), 64, 0, st>>>(a);
}

}  // namespace
}  // namespace gqk

using namespace gqk;

extern "C" int gqk_qk_norm_rope(const gqk_heads* q, const gqk_heads* k, const gqk_heads* v, int dtype, int64_t tokens,
                                int dim, const void* positions, int positions_64, const float* table, int64_t table_rows,
                                int rot, const void* q_weight, const void* k_weight, int weight_dtype, float eps,
                                int flags, const gqk_heads* out_q, const gqk_heads* out_k, const gqk_pages* pages,
                                const void* slots, int slots_64, void* stream) {
  const char* what = "qk_norm_rope";
  if (dtype != GQK_DTYPE_BF16 && dtype != GQK_DTYPE_F16) return decode_fail(GQK_ERR_ARG, "%s: dtype %d", what, dtype);
  if (!q || !out_q || q->heads < 1 || (k && (k->heads < 1))) return decode_fail(GQK_ERR_ARG, "%s: no heads", what);
  if (dim < 8 || dim > 256 || dim % 8 || rot < 0 || rot > dim || rot % 2)
    return decode_fail(GQK_ERR_SHAPE, "%s: %d rotated dims of %d (even; the dim a multiple of 8 in 8..256)", what, rot, dim);
  if (tokens < 0 || tokens > 0x7fffffff || table_rows < 0) return decode_fail(GQK_ERR_SHAPE, "%s: %lld tokens", what, (long long)tokens);
  if ((q_weight || k_weight) && weight_dtype != dtype && weight_dtype != GQK_DTYPE_F32)
    return decode_fail(GQK_ERR_ARG, "%s: weights of type %d", what, weight_dtype);
  if (out_q->heads != q->heads || (out_k && (!k || out_k->heads != k->heads)))
    return decode_fail(GQK_ERR_SHAPE, "%s: outputs with other heads than the inputs", what);
  if (k && !out_k && !pages) return decode_fail(GQK_ERR_ARG, "%s: the keys go nowhere", what);
  if (pages) {
    if (const int rc = check_pages(what, pages, dtype)) return rc;
    if (!k || !v || !slots || k->heads != pages->heads || v->heads != pages->heads || pages->dim != dim)
      return decode_fail(GQK_ERR_SHAPE, "%s: keys and values of %d heads of %d are stored with a slot each", what, pages->heads,
                         pages->dim);
  } else if (v || slots) {
    return decode_fail(GQK_ERR_ARG, "%s: values and slots without pages", what);
  }
  if (tokens == 0) return GQK_OK;
  if (!positions || (!table && rot > 0)) return decode_fail(GQK_ERR_ARG, "%s: null pointer", what);
  const gqk_heads* all[5] = {q, k, v, out_q, out_k};
  for (const gqk_heads* x : all) {
    if (!x) continue;
    if (!x->data) return decode_fail(GQK_ERR_ARG, "%s: null pointer", what);
    if ((uintptr_t)x->data & 15 || (x->row | x->head) & 7)
      return decode_fail(GQK_ERR_SHAPE, "%s: heads are 16-byte aligned with strides that are multiples of 8", what);
  }
  if ((uintptr_t)table & 3) return decode_fail(GQK_ERR_SHAPE, "%s: table must be 4-byte aligned", what);
  RopeArgs a{};
  a.q = q->data; a.q_row = q->row; a.q_head = q->head; a.q_heads = q->heads;
  if (k) { a.k = k->data; a.k_row = k->row; a.k_head = k->head; a.k_heads = k->heads; }
  if (v) { a.v = v->data; a.v_row = v->row; a.v_head = v->head; }
  a.out_q = out_q->data; a.oq_row = out_q->row; a.oq_head = out_q->head;
  if (out_k) { a.out_k = out_k->data; a.ok_row = out_k->row; a.ok_head = out_k->head; }
  a.q_weight = q_weight; a.k_weight = k_weight; a.positions = positions; a.table = table; a.table_rows = table_rows;
  a.slots = slots; a.dim = dim; a.rot = rot; a.tokens = (int)tokens; a.eps = eps;
  a.wide_positions = positions_64; a.wide_slots = slots_64; a.unit_offset = flags & GQK_ROPE_UNIT_OFFSET;
  a.interleaved = flags & GQK_ROPE_INTERLEAVED; a.weight_f32 = weight_dtype == GQK_DTYPE_F32;
  if (pages) { a.kv = *pages; a.store = 1; }
  const hipStream_t st = (hipStream_t)stream;
  const bool bf = dtype == GQK_DTYPE_BF16, f8 = pages && pages->dtype == GQK_DTYPE_FP8;
  for (int64_t t0 = 0; t0 < tokens; t0 += kTokens) {   // a grid's dimensions are limited
    a.tokens = (int)std::min<int64_t>(tokens - t0, kTokens);
    if (bf && f8) launch<bf16_t, fp8_t>(a, st);
    else if (bf) launch<bf16_t, bf16_t>(a, st);
    else if (f8) launch<f16_t, fp8_t>(a, st);
    else launch<f16_t, f16_t>(a, st);
    a.q = (const char*)a.q + 2 * kTokens * a.q_row;
    if (a.k) a.k = (const char*)a.k + 2 * kTokens * a.k_row;
    if (a.v) a.v = (const char*)a.v + 2 * kTokens * a.v_row;
    a.out_q = (char*)a.out_q + 2 * kTokens * a.oq_row;
    if (a.out_k) a.out_k = (char*)a.out_k + 2 * kTokens * a.ok_row;
    a.positions = (const char*)a.positions + kTokens * (positions_64 ? 8 : 4);
    if (a.slots) a.slots = (const char*)a.slots + kTokens * (slots_64 ? 8 : 4);
  }
  return decode_launched(what);
}
