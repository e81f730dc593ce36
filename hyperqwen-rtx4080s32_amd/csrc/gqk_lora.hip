// gqk_lora.hip - low-rank adapters of many requests beside a shared projection.
//
//   out[m, n] = y[m, n] + s_i sum_r B_i[n, r] h[m, p(n), r],   h[m, p, r] = sum_k A_i[p, r, k] x[m, k]
//
// with i = ids[m] the row's adapter (negative: out = y) and p(n) the part (q, k, v; gate, up) that
// column n belongs to.  h is kept in 32 bits in the workspace, after its counter region.
#include "gqk_decode.h"

namespace gqk {
namespace {

constexpr int kParts = 8;
struct LoraArgs {
  const void *y, *x, *a, *b;
  void* out;
  int64_t y_row, x_row, out_row, K, N;
  const void* ids;
  const float* scales;
  float* h;
  int M, slots, parts, rank, wide_ids;
  int64_t ends[kParts];   // one past each part's last column
};

// a wave per (row, part and rank)
template <typename T>
__global__ __launch_bounds__(64) void lora_down_kernel(LoraArgs a) {
  const int64_t m = blockIdx.y;
  const int pr = blockIdx.x, lane = threadIdx.x;
  const int64_t i = index_at(a.ids, a.wide_ids, m);
  if (i < 0 || i >= a.slots) return;
  const T* A = (const T*)a.a + (i * a.parts * a.rank + pr) * a.K;
  const T* x = (const T*)a.x + m * a.x_row;
  float s = 0.f;
  for (int64_t k = lane; k < a.K; k += 64) s += to_f(A[k]) * to_f(x[k]);
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if (lane == 0) a.h[(m * a.parts * a.rank) + pr] = s;
}

// a thread per (row, column)
template <typename T>
__global__ __launch_bounds__(256) void lora_up_kernel(LoraArgs a) {
  const int64_t m = blockIdx.y, n = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (n >= a.N) return;
  const int64_t i = index_at(a.ids, a.wide_ids, m);
  float d = 0.f;
  if (i >= a.slots) {
    d = __builtin_nanf("");
  } else if (i >= 0) {
    int p = 0;
    while (n >= a.ends[p]) ++p;
    const T* B = (const T*)a.b + (i * a.N + n) * a.rank;
    const float* h = a.h + (m * a.parts + p) * a.rank;
    for (int r = 0; r < a.rank; ++r) d += to_f(B[r]) * h[r];
    d *= a.scales ? a.scales[i] : 1.f;
  }
  ((T*)a.out)[m * a.out_row + n] = from_f<T>(to_f(((const T*)a.y)[m * a.y_row + n]) + d);
}

}  // namespace
}  // namespace gqk

using namespace gqk;

extern "C" {

int64_t gqk_lora_workspace_bytes(int M, int64_t K, int parts, int rank) {
  if (M < 0 || K < 0 || parts < 1 || parts > kParts || rank < 8 || rank > 256 || rank % 8)
    return decode_fail(GQK_ERR_SHAPE, "lora: %d rows of %lld, %d parts (at most %d), rank %d (a multiple of 8 in 8..256)", M,
                       (long long)K, parts, kParts, rank);
  return GQK_CTR_BYTES + (int64_t)M * parts * rank * 4;
}

int gqk_lora_add(const void* y, int64_t y_row, const void* x, int64_t x_row, int M, int64_t K, const void* a, const void* b,
                 int slots, int parts, const int64_t* n_outs, int rank, const void* ids, int ids_64, const float* scales,
                 int dtype, void* out, int64_t out_row, void* workspace, int64_t workspace_bytes, void* stream) {
  if (dtype != GQK_DTYPE_BF16 && dtype != GQK_DTYPE_F16) return decode_fail(GQK_ERR_ARG, "lora_add: dtype %d", dtype);
  const int64_t need = gqk_lora_workspace_bytes(M, K, parts, rank);
  if (need < 0) return (int)need;
  if (K % 8 || slots < 0 || !n_outs) return decode_fail(GQK_ERR_SHAPE, "lora_add: K %lld (a multiple of 8), %d slots", (long long)K, slots);
  LoraArgs g{};
  for (int p = 0; p < parts; ++p) {
    if (n_outs[p] < 1) return decode_fail(GQK_ERR_SHAPE, "lora_add: part %d has %lld columns", p, (long long)n_outs[p]);
    g.N += n_outs[p];
    g.ends[p] = g.N;
  }
  if (g.N >= (int64_t)1 << 31) return decode_fail(GQK_ERR_SHAPE, "lora_add: %lld columns", (long long)g.N);
  if (y_row < g.N || out_row < g.N || x_row < K)
    return decode_fail(GQK_ERR_SHAPE, "lora_add: row strides %lld, %lld, %lld of %lld and %lld columns", (long long)y_row,
                       (long long)out_row, (long long)x_row, (long long)g.N, (long long)K);
  if (M == 0) return GQK_OK;
  if (!y || !x || !ids || !out || (slots > 0 && (!a || !b))) return decode_fail(GQK_ERR_ARG, "lora_add: null pointer");
  if (((uintptr_t)x | (uintptr_t)a | (uintptr_t)b) & 15 || x_row & 7)
    return decode_fail(GQK_ERR_SHAPE, "lora_add: x, a and b are 16-byte aligned, x's row stride a multiple of 8");
  if (!workspace || workspace_bytes < need || (uintptr_t)workspace & 255)
    return decode_fail(GQK_ERR_SHAPE, "lora_add: workspace %lld bytes < %lld (or not 256-byte aligned)", (long long)workspace_bytes,
                       (long long)need);
  g.y = y; g.x = x; g.a = a; g.b = b; g.out = out; g.y_row = y_row; g.x_row = x_row; g.out_row = out_row; g.K = K;
  g.ids = ids; g.wide_ids = ids_64; g.scales = scales; g.h = (float*)((char*)workspace + GQK_CTR_BYTES);
  g.M = M; g.slots = slots; g.parts = parts; g.rank = rank;
  const hipStream_t st = (hipStream_t)stream;
  if (M > 65535) return decode_fail(GQK_ERR_SHAPE, "lora_add: %d rows (at most 65535)", M);
  const dim3 down(parts * rank, M), up((unsigned)((g.N + 255) / 256), M);
  if (dtype == GQK_DTYPE_BF16) {
    lora_down_kernel<bf16_t><<<down, 64, 0, st>>>(g);
    lora_up_kernel<bf16_t><<<up, 256, 0, st>>>(g);
  } else {
    lora_down_kernel<f16_t><<<down, 64, 0, st>>>(g);
    lora_up_kernel<f16_t><<<up, 256, 0, st>>>(g);
  }
  return decode_launched("lora_add");
}

}  // extern "C"
