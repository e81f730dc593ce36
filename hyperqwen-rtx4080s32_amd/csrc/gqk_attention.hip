// gqk_attention.hip - attention of one new token per sequence over a paged key-value cache.
//
//   o = sum_j exp(scale q.k_j - m) v_j / sum_j exp(scale q.k_j - m),   m = max_j scale q.k_j
//
// over the keys j in [max(0, length - window), length) of the sequence; no key: zeros.
#include "gqk_decode.h"

namespace gqk {

int device_cus() {
  int dev = 0, cus = 0;
  if (hipGetDevice(&dev) != hipSuccess ||
      hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0) {
    (void)hipGetLastError();   // leave no error behind for the next launch check
    cus = 256;
  }
  return cus;
}

int check_pages(const char* what, const gqk_pages* p, int q_dtype) {
  if (!p || !p->k || !p->v) return decode_fail(GQK_ERR_ARG, "%s: null pages", what);
  if (p->dtype != q_dtype && p->dtype != GQK_DTYPE_FP8)
    return decode_fail(GQK_ERR_ARG, "%s: pages of type %d with heads of type %d", what, p->dtype, q_dtype);
  if (p->pages < 1 || p->page_size < 1 || p->heads < 1)
    return decode_fail(GQK_ERR_SHAPE, "%s: %d pages of %d tokens, %d heads", what, p->pages, p->page_size, p->heads);
  if (p->dim < 8 || p->dim > 256 || p->dim % 8)
    return decode_fail(GQK_ERR_SHAPE, "%s: head dim %d is not a multiple of 8 in 8..256", what, p->dim);
  const int64_t size = p->dtype == GQK_DTYPE_FP8 ? 1 : 2, align = 8 * size;
  const int64_t strides[6] = {p->k_page, p->k_token, p->k_head, p->v_page, p->v_token, p->v_head};
  for (int64_t s : strides)
    if (s < 0 || s % 8) return decode_fail(GQK_ERR_SHAPE, "%s: page strides are multiples of 8 elements, not %lld", what, (long long)s);
  if ((uintptr_t)p->k % align || (uintptr_t)p->v % align)
    return decode_fail(GQK_ERR_SHAPE, "%s: pages must be %lld-byte aligned", what, (long long)align);
  if ((uintptr_t)p->k_scale % 4 || (uintptr_t)p->v_scale % 4)
    return decode_fail(GQK_ERR_SHAPE, "%s: scales must be 4-byte aligned", what);
  return GQK_OK;
}

namespace {

struct AttnArgs {
  const void* q;
  int64_t q_row, q_head;
  gqk_pages kv;
  const int32_t* table;
  int64_t table_row;
  const int32_t* lengths;
  void* out;
  int64_t out_row, out_head;
  float* lse;
  int q_heads, max_length, window;
  float scale;
};

// One wave per (sequence, query head): 64 keys at a time, a lane per key for the scores, a lane per
// dim for the values.
template <typename T, typename C>
__global__ __launch_bounds__(64) void attention_kernel(AttnArgs a) {
  const int h = blockIdx.x, b = blockIdx.y, lane = threadIdx.x;
  const int kvh = h / (a.q_heads / a.kv.heads), D = a.kv.dim, ps = a.kv.page_size;
  const int len = max(0, a.lengths[b]);
  const float ks = a.kv.k_scale ? a.kv.k_scale[kvh] : 1.f, vs = a.kv.v_scale ? a.kv.v_scale[kvh] : 1.f;
  const T* q = (const T*)a.q + b * a.q_row + h * a.q_head;
  __shared__ float sq[256], sp[64];
  __shared__ int64_t vo[64];
  for (int d = lane; d < D; d += 64) sq[d] = to_f(q[d]) * (a.scale * ks);
  __syncthreads();
  const float kInf = __builtin_huge_valf();
  float m = -kInf, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  bool bad = len > a.max_length;
  const int first = a.window > 0 ? max(0, len - a.window) : 0;
  for (int j0 = first; j0 < len && !bad; j0 += 64) {
    const int j = min(j0 + lane, len - 1);
    const int page = a.table[b * a.table_row + j / ps];
    const bool out = (uint32_t)page >= (uint32_t)a.kv.pages;
    bad = __any(out);
    if (bad) break;
    const C* kp = (const C*)a.kv.k + page * a.kv.k_page + (j % ps) * a.kv.k_token + kvh * a.kv.k_head;
    float s = 0.f;
    for (int d = 0; d < D; ++d) s += sq[d] * to_f(kp[d]);
    if (j0 + lane >= len) s = -kInf;
    float top = s;
    for (int x = 32; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
    const float mn = fmaxf(m, top), base = mn == -kInf ? 0.f : mn;
    const float p = __expf(s - base), c = __expf(m - base);
    float sum = p;
    for (int x = 32; x > 0; x >>= 1) sum += __shfl_xor(sum, x);
    l = l * c + sum;
    m = mn;
    __syncthreads();
    sp[lane] = p;
    vo[lane] = page * a.kv.v_page + (j % ps) * a.kv.v_token + kvh * a.kv.v_head;
    __syncthreads();
    for (int i = 0; i < 4; ++i) o[i] *= c;
    for (int t = 0; t < min(64, len - j0); ++t)
      for (int i = 0; i < 4; ++i)
        if (lane + 64 * i < D) o[i] += sp[t] * to_f(((const C*)a.kv.v)[vo[t] + lane + 64 * i]);
  }
  const float nan = __builtin_nanf(""), r = bad ? nan : l > 0.f ? vs / l : l == 0.f ? 0.f : nan;
  for (int i = 0; i < 4; ++i)
    if (lane + 64 * i < D) ((T*)a.out)[b * a.out_row + h * a.out_head + lane + 64 * i] = from_f<T>(o[i] * r);
  if (a.lse && lane == 0) a.lse[(int64_t)b * a.q_heads + h] = bad ? nan : l == 0.f ? -kInf : m + __logf(l);
}

}  // namespace
}  // namespace gqk

using namespace gqk;

extern "C" {

int64_t gqk_paged_attention_workspace_bytes(int batch, int q_heads, int kv_heads, int dim, int max_length, int window) {
  if (batch < 0 || kv_heads < 1 || q_heads < kv_heads || q_heads % kv_heads || dim < 8 || dim > 256 || dim % 8 ||
      max_length < 0 || window < 0)
    return decode_fail(GQK_ERR_SHAPE, "paged_attention: %d sequences, %d / %d heads of %d, max_length %d, window %d", batch,
                       q_heads, kv_heads, dim, max_length, window);
  return 0;
}

int gqk_paged_attention(const void* q, int64_t q_row, int64_t q_head, int dtype, int batch, int q_heads,
                        const gqk_pages* pages, const int32_t* table, int64_t table_row, int table_width,
                        const int32_t* lengths, int max_length, int window, float scale, void* out, int64_t out_row,
                        int64_t out_head, float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
  if (dtype != GQK_DTYPE_BF16 && dtype != GQK_DTYPE_F16) return decode_fail(GQK_ERR_ARG, "paged_attention: dtype %d", dtype);
  if (const int rc = check_pages("paged_attention", pages, dtype)) return rc;
  if (batch < 0 || batch > 65535 || q_heads < 1 || q_heads % pages->heads)
    return decode_fail(GQK_ERR_SHAPE, "paged_attention: %d sequences of %d query heads over %d", batch, q_heads, pages->heads);
  if (window < 0 || max_length < 0 || table_width < 0 ||
      (int64_t)max_length > (int64_t)table_width * pages->page_size)
    return decode_fail(GQK_ERR_SHAPE, "paged_attention: window %d, lengths up to %d in %d pages of %d tokens", window, max_length,
                       table_width, pages->page_size);
  if (batch == 0) return GQK_OK;
  if (!q || !out || !lengths || (!table && max_length > 0)) return decode_fail(GQK_ERR_ARG, "paged_attention: null pointer");
  if (((uintptr_t)q | (uintptr_t)out) & 15 || (q_row | q_head | out_row | out_head) & 7)
    return decode_fail(GQK_ERR_SHAPE, "paged_attention: q and out are 16-byte aligned with strides that are multiples of 8");
  const int64_t need = gqk_paged_attention_workspace_bytes(batch, q_heads, pages->heads, pages->dim, max_length, window);
  if (need < 0) return (int)need;
  if (need > 0 && (!workspace || workspace_bytes < need || (uintptr_t)workspace & 255))
    return decode_fail(GQK_ERR_SHAPE, "paged_attention: workspace %lld bytes < %lld (or not 256-byte aligned)",
                       (long long)workspace_bytes, (long long)need);
  AttnArgs a{q, q_row, q_head, *pages, table, table_row, lengths, out, out_row, out_head, lse, q_heads, max_length, window, scale};
  const dim3 grid(q_heads, batch);
  const hipStream_t st = (hipStream_t)stream;
  const bool bf = dtype == GQK_DTYPE_BF16;
  if (pages->dtype == GQK_DTYPE_FP8) {
    if (bf) attention_kernel<bf16_t, fp8_t><<<grid, 64, 0, st>>>(a);
    else attention_kernel<f16_t, fp8_t><<<grid, 64, 0, st>>>(a);
  } else if (bf) {
    attention_kernel<bf16_t, bf16_t><<<grid, 64, 0, st>>>(a);
  } else {
    attention_kernel<f16_t, f16_t><<<grid, 64, 0, st>>>(a);
  }
  return decode_launched("paged_attention");
}

}  // extern "C"
