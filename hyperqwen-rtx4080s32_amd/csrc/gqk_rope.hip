// gqk_rope.hip - the heads of queries and keys, normalized, rotated and stored in one pass.
//
//   n_i = x_i rsqrt(mean(x^2) + eps) w_i             (w_i, or 1 + w_i; no weight: n = x)
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t) (pairs (i, i + rot / 2) or (2 i, 2 i + 1) of the first rot dims)
//
// with cos t | sin t of pair i at [position][i] | [position][rot / 2 + i] of a table in 32 bits.  Keys
// and values of a token with a slot go into its page of the cache.
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

// One wave per (token, head): q heads, k heads, then v heads (stored only).
template <typename T, typename C>
__global__ __launch_bounds__(64) void rope_kernel(RopeArgs a) {
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
  const int heads = a.q_heads + a.k_heads + (pages ? pages->heads : 0);
  for (int64_t t0 = 0; t0 < tokens; t0 += 32768) {   // the grid's second dimension is limited
    const dim3 grid(heads, (unsigned)(tokens - t0 < 32768 ? tokens - t0 : 32768));
    if (bf && f8) rope_kernel<bf16_t, fp8_t><<<grid, 64, 0, st>>>(a);
    else if (bf) rope_kernel<bf16_t, bf16_t><<<grid, 64, 0, st>>>(a);
    else if (f8) rope_kernel<f16_t, fp8_t><<<grid, 64, 0, st>>>(a);
    else rope_kernel<f16_t, f16_t><<<grid, 64, 0, st>>>(a);
    const int64_t step = 32768;
    a.q = (const char*)a.q + 2 * step * a.q_row;
    if (a.k) a.k = (const char*)a.k + 2 * step * a.k_row;
    if (a.v) a.v = (const char*)a.v + 2 * step * a.v_row;
    a.out_q = (char*)a.out_q + 2 * step * a.oq_row;
    if (a.out_k) a.out_k = (char*)a.out_k + 2 * step * a.ok_row;
    a.positions = (const char*)a.positions + step * (positions_64 ? 8 : 4);
    if (a.slots) a.slots = (const char*)a.slots + step * (slots_64 ? 8 : 4);
  }
  return decode_launched(what);
}
