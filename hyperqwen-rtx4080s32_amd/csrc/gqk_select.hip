// gqk_select.hip - the pages that a decoded token attends to in a long cache: bounds of each page's keys, and the choice by them.
//
//   lo, hi[page, h, d] = min, max over the page's keys of k[., h, d]
//   score(b, h, j) = max over the query heads g of key head h of  sum_d max(q_gd lo_jhd, q_gd hi_jhd)
//
// No key of page j has a larger product with any of the queries.  The first and the last pages of a sequence are always taken, the others
// by their scores, the lowest page first among equals.
#include <algorithm>
#include "gqk_decode.h"

namespace gqk {
namespace {

// x of eight values of a page
__device__ __forceinline__ void load8(const bf16_t* p, float* x) {
  bf16_t v[8];
  __builtin_memcpy(v, __builtin_assume_aligned(p, 16), 16);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = to_f(v[e]);
}
__device__ __forceinline__ void load8(const f16_t* p, float* x) {
  f16_t v[8];
  __builtin_memcpy(v, __builtin_assume_aligned(p, 16), 16);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = to_f(v[e]);
}
__device__ __forceinline__ void load8(const fp8_t* p, float* x) {
  uint32_t w[2];
  __builtin_memcpy(w, __builtin_assume_aligned(p, 8), 8);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    x[4 * i] = __builtin_amdgcn_cvt_f32_fp8(w[i], 0);
    x[4 * i + 1] = __builtin_amdgcn_cvt_f32_fp8(w[i], 1);
    x[4 * i + 2] = __builtin_amdgcn_cvt_f32_fp8(w[i], 2);
    x[4 * i + 3] = __builtin_amdgcn_cvt_f32_fp8(w[i], 3);
  }
}
template <typename C> __device__ __forceinline__ void store8(C* p, const float* x) {
  C v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = from_f<C>(x[e]);
  __builtin_memcpy(__builtin_assume_aligned(p, 8 * sizeof(C)), v, 8 * sizeof(C));
}

// ---- bounds ----------------------------------------------------------------------------------

struct BoundsArgs {
  const void* k;
  int64_t k_page, k_token, k_head;
  const int32_t* table;
  int64_t table_row;
  const int32_t* lengths;
  void* bounds;
  int pages, page_size, heads, dim, width, count, page0;   // page0: of a sequence's, the launch's first
};

// A workgroup takes one page of one key head: its threads the page's keys, eight dims of one at a time.  Everything is in the trips to memory
// that follow one another: the length, the table, the keys, the store.  (One page of 64 keys of 8 heads: 14 us where one thread of a dim
// went through the 16 keys that the others had left, 6 with the waves' own sums first.)
template <typename C, int DP>
__global__ __launch_bounds__(256) void bounds_kernel(BoundsArgs a) {
  constexpr int LPK = DP / 8, KPW = 256 / LPK;   // lanes of a key, keys at once
  __shared__ float ends[2][4][DP];
  const int b = blockIdx.y, h = blockIdx.z, len = a.lengths[b];
  if (len <= 0 || len > (int64_t)a.width * a.page_size) return;
  const int64_t first = max(0, len - a.count) / a.page_size, at_page = first + a.page0 + blockIdx.x;
  if (at_page > (len - 1) / a.page_size) return;
  const int j = (int)at_page;
  const int page = a.table[(int64_t)b * a.table_row + j];
  if ((uint32_t)page >= (uint32_t)a.pages) return;
  const int keys = min(a.page_size, len - j * a.page_size);
  const int at = threadIdx.x / LPK, d = (threadIdx.x % LPK) * 8, wave = threadIdx.x >> 6;
  const bool live = d < a.dim;
  const C* base = (const C*)a.k + page * a.k_page + h * a.k_head + (live ? d : 0);
  const float inf = __builtin_huge_valf(), nan = __builtin_nanf("");
  float lo[8], hi[8];   // a dim with a NaN has NaN for both
#pragma unroll
  for (int e = 0; e < 8; ++e) { lo[e] = inf; hi[e] = -inf; }
  auto lower = [&](float x, float y) { return x != x || y != y ? nan : fminf(x, y); };
  auto upper = [&](float x, float y) { return x != x || y != y ? nan : fmaxf(x, y); };
  for (int i = at; i < keys; i += 4 * KPW) {
    float x[4][8];
#pragma unroll
    for (int k = 0; k < 4; ++k) load8(base + (int64_t)min(i + k * KPW, keys - 1) * a.k_token, x[k]);
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        lo[e] = lower(lo[e], x[k][e]);
        hi[e] = upper(hi[e], x[k][e]);
      }
  }
#pragma unroll
  for (int o = LPK; o < 64; o <<= 1)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      lo[e] = lower(lo[e], __shfl_xor(lo[e], o));
      hi[e] = upper(hi[e], __shfl_xor(hi[e], o));
    }
  if ((threadIdx.x & 63) < LPK)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      ends[0][wave][d + e] = lo[e];
      ends[1][wave][d + e] = hi[e];
    }
  __syncthreads();
  // one thread for each eight dims of a bound
  if (threadIdx.x >= 2 * LPK || !live) return;
  const int which = threadIdx.x / LPK;
  float y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    y[e] = ends[which][0][d + e];
#pragma unroll
    for (int w = 1; w < 4; ++w) y[e] = which ? upper(y[e], ends[1][w][d + e]) : lower(y[e], ends[0][w][d + e]);
  }
  store8((C*)a.bounds + (((int64_t)page * 2 + which) * a.heads + h) * a.dim + d, y);
}

// ---- scores ----------------------------------------------------------------------------------

struct SelectArgs {
  const void* q;
  int64_t q_row, q_head;
  const void* bounds;
  const int32_t* table;
  int64_t table_row;
  const int32_t* lengths;
  int32_t *out, *out_lengths;
  uint64_t* keys;       // [batch of the launch][heads][most]
  int batch0, pages, page_size, heads, dim, group, keep, sink, recent, max_length, most;
};

constexpr uint64_t kTaken = ~0ull;

// a number of 64 bits whose order is the scores': larger for larger; NaN counts as infinity
__device__ __forceinline__ uint64_t order_of(double x) {
  if (x != x) x = __builtin_huge_val();
  const uint64_t bits = __builtin_bit_cast(uint64_t, x + 0.0);   // -0 is 0
  return bits >> 63 ? ~bits : bits | 1ull << 63;
}

// pages of a sequence, -1 where its length is out of range
__device__ __forceinline__ int pages_of(const SelectArgs& a, int len) {
  return len > a.max_length ? -1 : len <= 0 ? 0 : (len - 1) / a.page_size + 1;
}

template <int CTRL> __device__ __forceinline__ double dpp_add(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, 0xf, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, 0xf, 0xf, false);
  return x + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// the sum over 8, 16 or 32 neighbouring lanes
template <int LANES> __device__ __forceinline__ double lane_sum(double x) {
  x = dpp_add<0xB1>(x);    // quad_perm 1, 0, 3, 2
  x = dpp_add<0x4E>(x);    // quad_perm 2, 3, 0, 1
  x = dpp_add<0x141>(x);   // row_half_mirror
  if constexpr (LANES >= 16) x = dpp_add<0x140>(x);   // row_mirror
  if constexpr (LANES >= 32) x += __shfl_xor(x, 16);
  return x;
}

// Eight dims of a page's bounds to a lane; products (exact) and sums in 64 bits, as the comparison of near equals decides which pages are read.  (Products in
// 32 bits are as exact within their range, which bf16's squares pass: a batch took 107 us with them where it takes 109.)  The 64-bit sums bound it in a batch: up to 500 pages of 48 sequences, 8 heads, 40 of queries (31 MB in 8
// bits) 31 us; 2048 pages of one (8 MB) 7.  (Sums in 32 bits first, and those in 64 of the heads within their error of the largest alone: 29 and 10 where this
// took 29 and 7 with products in 32 bits, as the queries' norms, the registers that hold them and the second reading of a query cost what it saves.)
template <typename T, typename C, int DP>
__global__ __launch_bounds__(256) void score_kernel(SelectArgs a) {
  constexpr int LPP = DP / 8, PPW = 256 / LPP;   // lanes of a page, pages at once
  const int b = a.batch0 + blockIdx.z, h = blockIdx.y, len = a.lengths[b], n = pages_of(a, len);
  if (n <= a.keep) return;   // all are taken
  const int at = threadIdx.x / LPP, d = (threadIdx.x % LPP) * 8;
  const bool live = d < a.dim;
  const T* q = (const T*)a.q + b * a.q_row + (int64_t)h * a.group * a.q_head + (live ? d : 0);
  uint64_t* to = a.keys + ((int64_t)blockIdx.z * a.heads + h) * a.most;
  for (int j = blockIdx.x * PPW + at; j < n; j += gridDim.x * PPW) {
    uint64_t key = kTaken;
    // no page outside of the cache is read: it is taken, and the attention answers with NaN
    const int page = j < a.sink || j >= n - a.recent ? -1 : a.table[(int64_t)b * a.table_row + j];
    const bool sound = (uint32_t)page < (uint32_t)a.pages;
    if (sound) {
      const C* from = (const C*)a.bounds + ((int64_t)page * 2 * a.heads + h) * a.dim + (live ? d : 0);
      float lo32[8], hi32[8];
      load8(from, lo32);
      load8(from + (int64_t)a.heads * a.dim, hi32);
      double lo[8], hi[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) { lo[e] = lo32[e]; hi[e] = hi32[e]; }
      double best = -__builtin_huge_val();
      bool bad = false;
      for (int g = 0; g < a.group; ++g) {
        float x[8];
        load8(q + g * a.q_head, x);
        double sum = 0.0;
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = __builtin_fma((double)x[e], x[e] >= 0.f ? hi[e] : lo[e], sum);
        if (!live) sum = 0.0;
        sum = lane_sum<LPP>(sum);
        bad |= sum != sum;
        best = fmax(best, sum);
      }
      key = order_of(bad ? __builtin_huge_val() : best);
    }
    if (threadIdx.x % LPP == 0) to[j] = key;
  }
}

// ---- the choice ------------------------------------------------------------------------------

constexpr int kHeld = 8;

// A workgroup chooses for one key head of one sequence: the keep-th largest key by its digits of eight bits, from the highest in which the keys
// differ, until the digit's bin holds just what is left to take, or few enough keys to be compared with each other by one wave; then the pages
// above it in their order.  A wave's keys are neighbours; up to eight to a lane stay in registers.  500 pages of 8 heads of 48 sequences 8.6 us, of
// 256 threads each (22 of 1024, digit by digit to the end), 2048 pages of 8 heads of one 9 (13): a launch, four trips to memory and some ten barriers.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void select_kernel(SelectArgs a) {
  constexpr int WAVES = THREADS / 64;
  __shared__ int bins[256];
  __shared__ uint32_t ends[2][WAVES];
  __shared__ int counts[2][WAVES];
  __shared__ uint64_t near[64];
  __shared__ int some, found[2];
  __shared__ uint64_t edge;
  const int b = a.batch0 + blockIdx.y, h = blockIdx.x, len = a.lengths[b], n = pages_of(a, len);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int32_t* table = a.table + (int64_t)b * a.table_row;
  int32_t* out = a.out + ((int64_t)b * a.heads + h) * a.keep;
  if (h == 0 && tid == 0) {
    const int over = n - a.keep;
    a.out_lengths[b] = n < 0 ? 0x7fffffff : over <= 0 ? max(0, len) : len - over * a.page_size;
  }
  if (n <= a.keep) {
    for (int j = tid; j < a.keep; j += THREADS) out[j] = j < n ? table[j] : -1;
    return;
  }
  const uint64_t* keys = a.keys + ((int64_t)blockIdx.y * a.heads + h) * a.most;
  const int each = ((n + THREADS - 1) / THREADS) * 64, begin = wave * each;   // of a wave
  const int rounds = each / 64;
  uint64_t held[kHeld];
  auto load = [&](int r0) {
#pragma unroll
    for (int r = 0; r < kHeld; ++r) {
      const int j = begin + (r0 + r) * 64 + lane;
      held[r] = r0 + r < rounds && j < n ? keys[j] : 0;   // no score has the number 0
    }
  };
  load(0);
  const bool all = rounds <= kHeld;
  // where the keys begin to differ: by their upper halves
  uint32_t low = ~0u, high = 0;
  for (int r0 = 0; r0 < rounds; r0 += kHeld) {
    if (!all) load(r0);
#pragma unroll
    for (int r = 0; r < kHeld; ++r)
      if (held[r]) {
        const uint32_t up = held[r] >> 32;
        low = min(low, up);
        high = max(high, held[r] == kTaken ? 0u : up);
      }
  }
  for (int o = 32; o > 0; o >>= 1) {
    low = min(low, (uint32_t)__shfl_xor((int)low, o));
    high = max(high, (uint32_t)__shfl_xor((int)high, o));
  }
  if (lane == 0) { ends[0][wave] = low; ends[1][wave] = high; }
  if (tid < 256) bins[tid] = 0;
  if (tid == 0) some = 0;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < WAVES; ++k) { low = min(low, ends[0][k]); high = max(high, ends[1][k]); }
  high = max(low, high);
  // keys less what they have in common; those always taken are above all others, by as little as there is
  const uint64_t base = (uint64_t)low << 32, top = ((uint64_t)(high - low) + 1) << 32;
  auto rank_of = [&](uint64_t key) { return key == kTaken ? top : key - base; };
  int left = a.keep, bits = 64 - __builtin_clzll(top);
  uint64_t prefix = 0;   // of the keep-th largest rank, its bits above `bits`
  bool exact = false;    // everything at or above prefix is taken
  while (bits > 0) {
    const int digit = min(8, bits);
    bits -= digit;
    for (int r0 = 0; r0 < rounds; r0 += kHeld) {
      if (!all) load(r0);
#pragma unroll
      for (int r = 0; r < kHeld; ++r) {
        const uint64_t x = rank_of(held[r]);
        if (held[r] && x >> bits >> digit == prefix >> bits >> digit) atomicAdd(&bins[(x >> bits) & 255], 1);
      }
    }
    __syncthreads();
    if (wave == 0) {   // the bin in which the sum from the top reaches what is left
      int c[4], own = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) own += c[k] = bins[255 - (lane * 4 + k)];
      int sum = own;
      for (int o = 1; o < 64; o <<= 1) {
        const int up = __shfl_up(sum, o);
        if (lane >= o) sum += up;
      }
      int above = sum - own;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (above < left && above + c[k] >= left) { found[0] = 255 - (lane * 4 + k); found[1] = above; }
        above += c[k];
      }
    }
    __syncthreads();
    const int bin = found[0], held_by = bins[bin];
    left -= found[1];
    prefix |= (uint64_t)bin << bits;
    exact = held_by == left;
    if (exact || bits == 0) break;
    if (held_by <= 64) {
      for (int r0 = 0; r0 < rounds; r0 += kHeld) {
        if (!all) load(r0);
#pragma unroll
        for (int r = 0; r < kHeld; ++r) {
          const uint64_t x = rank_of(held[r]);
          if (held[r] && x >> bits == prefix >> bits) near[atomicAdd(&some, 1)] = x;
        }
      }
      __syncthreads();
      if (wave == 0) {   // the left-th largest of them, and how many of its equals are to be taken
        const uint64_t mine = lane < held_by ? near[lane] : 0;
        int more = 0, same = 0;
        for (int k = 0; k < held_by; ++k) {
          const uint64_t x = near[k];
          more += x > mine;
          same += x == mine;
        }
        if (lane < held_by && more < left && more + same >= left) { edge = mine; found[1] = left - more; }   // (equals write the same)
      }
      __syncthreads();
      prefix = edge;
      left = found[1];
      break;
    }
    __syncthreads();
    if (tid < 256) bins[tid] = 0;
    __syncthreads();
  }
  // What is above is taken, and of the equal ones the first `left` (all, where exact).
  auto above_of = [&](uint64_t key) { return key && (exact ? rank_of(key) >= prefix : rank_of(key) > prefix); };
  auto equal_to = [&](uint64_t key) { return key && !exact && rank_of(key) == prefix; };
  int more = 0, same = 0;
  for (int r0 = 0; r0 < rounds; r0 += kHeld) {
    if (!all) load(r0);
#pragma unroll
    for (int r = 0; r < kHeld; ++r) {
      more += __popcll(__ballot(above_of(held[r])));
      same += __popcll(__ballot(equal_to(held[r])));
    }
  }
  if (lane == 0) { counts[0][wave] = more; counts[1][wave] = same; }
  __syncthreads();
  more = same = 0;
  for (int k = 0; k < wave; ++k) { more += counts[0][k]; same += counts[1][k]; }
  const uint64_t under = (1ull << lane) - 1;
  for (int r0 = 0; r0 < rounds; r0 += kHeld) {
    if (!all) load(r0);
#pragma unroll
    for (int r = 0; r < kHeld; ++r) {
      const uint64_t up = __ballot(above_of(held[r])), eq = __ballot(equal_to(held[r]));
      const int rank = same + __popcll(eq & under);
      const bool mine = (up >> lane & 1) || ((eq >> lane & 1) && rank < left);
      const int place = more + __popcll(up & under) + (exact ? 0 : min(rank, left));
      if (mine && place < a.keep) out[place] = table[begin + (r0 + r) * 64 + lane];
      more += __popcll(up);
      same += __popcll(eq);
    }
  }
}

template <typename T, typename C>
void score(const SelectArgs& a, dim3 grid, hipStream_t st) {
  if (a.dim <= 64) score_kernel<T, C, 64><<<grid, 256, 0, st>>>(a);
  else if (a.dim <= 128) score_kernel<T, C, 128><<<grid, 256, 0, st>>>(a);
  else score_kernel<T, C, 256><<<grid, 256, 0, st>>>(a);
}

template <typename C>
void bounds(const BoundsArgs& a, dim3 grid, hipStream_t st) {
  if (a.dim <= 64) bounds_kernel<C, 64><<<grid, 256, 0, st>>>(a);
  else if (a.dim <= 128) bounds_kernel<C, 128><<<grid, 256, 0, st>>>(a);
  else bounds_kernel<C, 256><<<grid, 256, 0, st>>>(a);
}

int check_shape(const char* what, int dtype, int pages, int page_size, int heads, int dim, int batch, int width) {
  if (dtype != GQK_DTYPE_BF16 && dtype != GQK_DTYPE_F16 && dtype != GQK_DTYPE_FP8) return decode_fail(GQK_ERR_ARG, "%s: pages of type %d", what, dtype);
  if (pages < 1 || page_size < 1 || heads < 1 || heads > 65535 || dim < 8 || dim > 256 || dim % 8)
    return decode_fail(GQK_ERR_SHAPE, "%s: %d pages of %d tokens, %d heads of %d (a multiple of 8 in 8..256)", what, pages, page_size, heads, dim);
  if (batch < 0 || batch > 65535 || width < 0) return decode_fail(GQK_ERR_SHAPE, "%s: %d sequences of %d pages", what, batch, width);
  return GQK_OK;
}

}  // namespace
}  // namespace gqk

using namespace gqk;

extern "C" {

int gqk_page_bounds(const gqk_pages* pages, const int32_t* table, int64_t table_row, int table_width, const int32_t* lengths, int batch,
                    int count, void* bounds_out, void* stream) {
  const char* what = "page_bounds";
  if (!pages || !pages->k) return decode_fail(GQK_ERR_ARG, "%s: null pages", what);
  if (const int rc = check_shape(what, pages->dtype, pages->pages, pages->page_size, pages->heads, pages->dim, batch, table_width)) return rc;
  const int64_t size = pages->dtype == GQK_DTYPE_FP8 ? 1 : 2;
  if (((pages->k_page | pages->k_token | pages->k_head) & 7) || pages->k_page < 0 || pages->k_token < 0 || pages->k_head < 0 ||
      ((uintptr_t)pages->k | (uintptr_t)bounds_out) % (8 * size))
    return decode_fail(GQK_ERR_SHAPE, "%s: pages and bounds are aligned to 8 elements, strides multiples of 8", what);
  if (count < 0) return decode_fail(GQK_ERR_SHAPE, "%s: the last %d keys", what, count);
  if (batch == 0 || count == 0 || table_width == 0) return GQK_OK;
  if (!table || !lengths || !bounds_out) return decode_fail(GQK_ERR_ARG, "%s: null pointer", what);
  BoundsArgs a{};
  a.k = pages->k; a.k_page = pages->k_page; a.k_token = pages->k_token; a.k_head = pages->k_head; a.table = table; a.table_row = table_row;
  a.lengths = lengths; a.bounds = bounds_out; a.pages = pages->pages; a.page_size = pages->page_size; a.heads = pages->heads;
  a.dim = pages->dim; a.width = table_width; a.count = count;
  const int most = (int)std::min<int64_t>(table_width, ((int64_t)count + pages->page_size - 2) / pages->page_size + 1);
  const hipStream_t st = (hipStream_t)stream;
  constexpr int turn = 0xffffff;   // pages of a launch, which has fewer than 2^32 threads
  for (int64_t p0 = 0; p0 < most; p0 += turn) {
    a.page0 = (int)p0;
    const dim3 grid((unsigned)std::min<int64_t>(turn, most - p0), batch, a.heads);
    if (pages->dtype == GQK_DTYPE_FP8) bounds<fp8_t>(a, grid, st);
    else if (pages->dtype == GQK_DTYPE_BF16) bounds<bf16_t>(a, grid, st);
    else bounds<f16_t>(a, grid, st);
  }
  return decode_launched(what);
}

int64_t gqk_select_pages_workspace_bytes(int batch, int heads, int page_size, int max_length) {
  if (batch < 0 || heads < 1 || page_size < 1 || max_length < 0 || max_length > GQK_MAX_KEYS)
    return decode_fail(GQK_ERR_SHAPE, "select_pages: %d sequences of up to %d keys in pages of %d, %d heads", batch, max_length, page_size, heads);
  return GQK_CTR_BYTES + (int64_t)batch * heads * (((int64_t)max_length + page_size - 1) / page_size) * 8;
}

int gqk_select_pages(const void* q, int64_t q_row, int64_t q_head, int dtype, int batch, int q_heads, const void* bounds_in, int bounds_dtype,
                     int pages, int heads, int dim, const int32_t* table, int64_t table_row, int table_width, const int32_t* lengths,
                     int max_length, int page_size, int keep, int sink, int recent, int32_t* out, int32_t* out_lengths, void* workspace,
                     int64_t workspace_bytes, void* stream) {
  const char* what = "select_pages";
  if (dtype != GQK_DTYPE_BF16 && dtype != GQK_DTYPE_F16) return decode_fail(GQK_ERR_ARG, "%s: dtype %d", what, dtype);
  if (const int rc = check_shape(what, bounds_dtype, pages, page_size, heads, dim, batch, table_width)) return rc;
  if (bounds_dtype != dtype && bounds_dtype != GQK_DTYPE_FP8)
    return decode_fail(GQK_ERR_ARG, "%s: bounds of type %d with heads of type %d", what, bounds_dtype, dtype);
  if (q_heads < 1 || q_heads % heads) return decode_fail(GQK_ERR_SHAPE, "%s: %d query heads over %d", what, q_heads, heads);
  if (max_length < 0 || max_length > GQK_MAX_KEYS || (int64_t)max_length > (int64_t)table_width * page_size)
    return decode_fail(GQK_ERR_SHAPE, "%s: lengths up to %d in %d pages of %d tokens", what, max_length, table_width, page_size);
  if (keep < 1 || sink < 0 || recent < 1 || (int64_t)sink + recent > keep)
    return decode_fail(GQK_ERR_SHAPE, "%s: %d pages of which the first %d and the last %d (one at least) are taken always", what, keep, sink, recent);
  if (batch == 0) return GQK_OK;
  if (!q || !bounds_in || !lengths || !out || !out_lengths || (!table && max_length > 0)) return decode_fail(GQK_ERR_ARG, "%s: null pointer", what);
  if ((uintptr_t)q & 15 || (q_row | q_head) & 7 || (uintptr_t)bounds_in % (bounds_dtype == GQK_DTYPE_FP8 ? 8 : 16))
    return decode_fail(GQK_ERR_SHAPE, "%s: q is 16-byte aligned with strides that are multiples of 8, bounds are aligned to 8 elements", what);
  SelectArgs a{};
  a.q = q; a.q_row = q_row; a.q_head = q_head; a.bounds = bounds_in; a.table = table; a.table_row = table_row; a.lengths = lengths;
  a.out = out; a.out_lengths = out_lengths; a.pages = pages; a.page_size = page_size; a.heads = heads; a.dim = dim;
  a.group = q_heads / heads; a.keep = keep; a.sink = sink; a.recent = recent; a.max_length = max_length;
  a.most = (int)(((int64_t)max_length + page_size - 1) / page_size);
  const hipStream_t st = (hipStream_t)stream;
  const bool scored = a.most > keep;   // else all of every sequence's pages are taken
  int turn = batch;                    // sequences whose scores the workspace holds
  if (scored) {
    const int64_t each = (int64_t)heads * a.most * 8, room = workspace ? (workspace_bytes - GQK_CTR_BYTES) / each : 0;
    if (room < 1) return decode_fail(GQK_ERR_SHAPE, "%s: a workspace of %lld bytes does not hold the scores of a sequence (%lld bytes)", what,
                                     (long long)workspace_bytes, (long long)(GQK_CTR_BYTES + each));
    if ((uintptr_t)workspace & 255) return decode_fail(GQK_ERR_SHAPE, "%s: workspace is not 256-byte aligned", what);
    turn = (int)std::min<int64_t>(batch, room);
    a.keys = (uint64_t*)((char*)workspace + GQK_CTR_BYTES);
  }
  for (int b0 = 0; b0 < batch; b0 += turn) {
    const int n = std::min(turn, batch - b0);
    a.batch0 = b0;
    if (scored) {
      const int at_once = 256 / (dim <= 64 ? 8 : dim <= 128 ? 16 : 32);
      const int blocks = std::max(1, std::min((a.most + at_once - 1) / at_once, (8 * device_cus() + n * heads - 1) / (n * heads)));
      const dim3 grid(blocks, heads, n);
      const bool bf = dtype == GQK_DTYPE_BF16;
      if (bounds_dtype == GQK_DTYPE_FP8) {
        if (bf) score<bf16_t, fp8_t>(a, grid, st);
        else score<f16_t, fp8_t>(a, grid, st);
      } else if (bf) {
        score<bf16_t, bf16_t>(a, grid, st);
      } else {
        score<f16_t, f16_t>(a, grid, st);
      }
    }
    // what 256 threads hold in registers, they choose of fastest: fewer waves meet at the barriers
    if (a.most <= 256 * kHeld) select_kernel<256><<<dim3(heads, n), 256, 0, st>>>(a);
    else select_kernel<1024><<<dim3(heads, n), 1024, 0, st>>>(a);
  }
  return decode_launched(what);
}

}  // extern "C"
