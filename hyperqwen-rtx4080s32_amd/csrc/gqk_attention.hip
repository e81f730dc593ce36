// gqk_attention.hip - attention of one new token per sequence over a paged key-value cache.
//
//   o = sum_j exp(scale q.k_j - m) v_j / sum_j exp(scale q.k_j - m),   m = max_j scale q.k_j
//
// over the keys j in [max(0, length - window), length) of the sequence; no key: zeros.
#include <algorithm>
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
  if (p->k_token > GQK_MAX_TOKEN_STRIDE || p->v_token > GQK_MAX_TOKEN_STRIDE || p->k_page > GQK_MAX_PAGE_STRIDE ||
      p->v_page > GQK_MAX_PAGE_STRIDE)
    return decode_fail(GQK_ERR_SHAPE, "%s: pages further apart than %d elements, or their tokens than %d", what, GQK_MAX_PAGE_STRIDE,
                       GQK_MAX_TOKEN_STRIDE);
  if ((uintptr_t)p->k % align || (uintptr_t)p->v % align)
    return decode_fail(GQK_ERR_SHAPE, "%s: pages must be %lld-byte aligned", what, (long long)align);
  if ((uintptr_t)p->k_scale % 4 || (uintptr_t)p->v_scale % 4)
    return decode_fail(GQK_ERR_SHAPE, "%s: scales must be 4-byte aligned", what);
  return GQK_OK;
}

namespace {

typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

constexpr int kWaves = 4;             // waves of a workgroup
constexpr int kTile = 32;             // keys of a wave's step
constexpr int kJoinSplits = 16;       // splits that the last workgroup of a sequence joins, at most
constexpr int kMostSplits = 256;
// A weight is 2^(score - maximum + kLift): fp16 uses its whole range, so that weights keep their relative precision down to 2^-29 of
// the heaviest and none is lost above 2^-40 (not lifted they do to 2^-14, and a long flat tail of them, each lighter than that, lost
// up to all of its weight).  bf16 has fp32's exponents.
template <typename T> constexpr float kLift = __is_same(T, f16_t) ? 15.f : 0.f;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

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
  int* counters;
  float* partials;
  int q_heads, max_length, window;
  float scale;          // of a score, in units of log 2
  int row_waves;        // 16-row tiles of query heads that a workgroup's waves deal among themselves
  int row_blocks;       // workgroups over the query heads of one key head
  int chunk, splits;    // keys of a split, and the most splits of a sequence
  uint32_t magic;       // key / page_size = 2 key magic >> 32 >> shift, exact below 2^31
  int shift;
  int join_apart;       // the splits are joined by a launch of their own
};

__device__ __forceinline__ v4f mfma(v4u a, v4u b, v4f c, bf16_t) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}
__device__ __forceinline__ v4f mfma(v4u a, v4u b, v4f c, f16_t) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

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

// max and sum over the four lanes of a query head (lane, lane ^ 16, lane ^ 32, lane ^ 48)
__device__ __forceinline__ float max4(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float sum4(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
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

// A workgroup takes one split (a.chunk keys) of one sequence's keys of one key head, for up to 16 row_waves query heads
// that share it; its waves deal the 32-key steps of the split (and the 16-row tiles of the heads) among themselves.
//
// Both products run on 16 x 16 x 32 matrix instructions with the keys (then the dims) as the rows and the query
// heads as the columns, so that a lane holds scores, statistics and sums of one head, and nothing but the maximum
// crosses lanes:  S^T = K Q^T: lane l = (head n = l % 16, g = l / 16) gets the scores of keys 8 g .. 8 g + 7 of the step (the
// rows of the two 16-key tiles are dealt so), which is what O^T += V^T P^T wants of it as an operand.  K comes from global
// memory straight as operands (8 dims of a key per lane).  V's operands hold 8 keys of one dim: a lane loads 8 dims of
// each of its 8 keys and transposes the 8 x 8 block in registers, one v_perm per pair.  No barrier in the loop, and no LDS but for
// the queries of 256 dims.
//
// Scores, statistics and sums are in 32 bits; the probabilities become T for the second product (up to 2^-8 of each for bf16, as
// random as the output's own rounding: 1.9e-3 of error against 64 bits where the output's rounding alone has 1.7e-3), two terms
// of T would need twice the instructions.  8-bit keys and values widen to T exactly, their scales go
// into the score's and the output's factor.
//
// Memory bounds it: 2.6 GB of bf16 keys and values (128 sequences of up to 8000) 406 us, 6.5 TB/s; 330 MB (32 of up to 4000)
// 61.8 us, 5.3 TB/s; fp16 heads of 256 dims under a window, 1.5 GB, 245 us, 6.0 TB/s; 268 MB of 8-bit pages of one sequence
// 47 us and 6 for the join.  A sequence of 61 keys takes 5.3 us: a launch, and lengths, table and keys read one after the other.
template <typename T, typename C, int DP, bool FULL, bool P8, bool TIGHT>
__global__ __launch_bounds__(64 * kWaves, DP == 256 ? 2 : 3) void attention_kernel(AttnArgs a) {
  constexpr bool F8 = sizeof(C) == 1;
  constexpr int NM = DP / 32;                 // k-steps of a score
  constexpr int VD = DP == 64 ? 4 : 8;        // dims of a lane's V load
  constexpr int NH = DP / (16 * VD);          // V loads of a key per lane
  constexpr int NT = NH * VD;                 // 16-dim tiles of the output
  constexpr int KW = F8 ? 2 : 4;              // words of 8 dims
  constexpr int RB = DP * (int)sizeof(C);     // bytes of a key (FULL)
  constexpr int RS = DP + 4;                  // row stride of the reduction buffer
  constexpr bool QLDS = DP == 256;
  __shared__ __align__(16) float red[kWaves * 16 * RS];
  __shared__ float stat[kWaves * 16][2];
  __shared__ int flag;

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
  const int b = blockIdx.y, split = blockIdx.z;
  const int kvh = blockIdx.x / a.row_blocks, rb = blockIdx.x % a.row_blocks;
  const int group = a.q_heads / a.kv.heads, D = a.kv.dim;
  const int rows_wg = 16 * a.row_waves, row0 = rb * rows_wg, R = min(rows_wg, group - row0);
  const int len0 = max(0, a.lengths[b]);
  const bool too_long = len0 > a.max_length;
  const int len = too_long ? 0 : len0;
  const int first = a.window > 0 ? max(0, len - a.window) : 0, start = first & ~(kTile - 1);
  const int ns = splits_of(start, len, a.chunk);   // of this sequence
  if (split >= ns) return;
  const int k_begin = start + split * a.chunk, k_end = k_begin + min(a.chunk, len - k_begin);
  const float inf = __builtin_huge_valf();

  const int rt = wave % a.row_waves, kw = wave / a.row_waves, nkw = kWaves / a.row_waves;
  const int row = rt * 16 + n;                                     // of the workgroup's rows
  const int steps_all = (k_end - k_begin + kTile - 1) / kTile;
  const int steps = rt * 16 < R && steps_all > kw ? (steps_all - kw + nkw - 1) / nkw : 0;
  const float scale = a.scale * (a.kv.k_scale ? a.kv.k_scale[kvh] : 1.f);

  v4f acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = v4f{0.f, 0.f, 0.f, 0.f};
  float m = -inf, l = 0.f;
  bool bad = false;

  if (steps > 0) {
    const int32_t* table = a.table + (int64_t)b * a.table_row;
    const char* kb = (const char*)a.kv.k + kvh * a.kv.k_head * (int64_t)sizeof(C);
    const char* vb = (const char*)a.kv.v + kvh * a.kv.v_head * (int64_t)sizeof(C);
    const uint32_t k_page = (uint32_t)a.kv.k_page * sizeof(C), k_tok = TIGHT ? RB : (uint32_t)a.kv.k_token * sizeof(C);
    const uint32_t v_page = (uint32_t)a.kv.v_page * sizeof(C), v_tok = TIGHT ? RB : (uint32_t)a.kv.v_token * sizeof(C);
    const int ps = a.kv.page_size, last = len - 1;
    // first dim of k-step i's operand: 16 bytes of a key per load
    auto dim_at = [&](int i) { return F8 && FULL ? (i >> 1) * 64 + g * 16 + (i & 1) * 8 : i * 32 + g * 8; };
    auto page_of = [&](int key) { return (int)(__umulhi(2u * (uint32_t)key, a.magic) >> a.shift); };

    // Queries stay in registers as operands; at 256 dims, where they would not fit beside K, V and the sums, in the
    // wave's own part of the reduction buffer, which is free until its loop ends.
    v4u q[NM];
    char* const mine = (char*)(red + wave * 16 * RS) + lane * 16;
    {
      const bool live = row < R;
      const T* qp = (const T*)a.q + b * a.q_row + (int64_t)(kvh * group + row0 + (live ? row : 0)) * a.q_head;
#pragma unroll
      for (int i = 0; i < NM; ++i) {
        const int d = dim_at(i);
        q[i] = *(const v4u*)(qp + (FULL || d < D ? d : 0));
        if (!live || !(FULL || d < D)) q[i] = v4u{0, 0, 0, 0};
        if constexpr (QLDS) *(v4u*)(mine + i * 1024) = q[i];
      }
    }

    // The keys of a lane: as rows of K's two tiles, group n / 4 of 8 keys, places n % 4 and 4 + n % 4; for V all 8 of
    // group g.  Keys outside of [first, last] are read as the nearest inside (their weight is 0).
    struct Pages { int page, place; };
    auto find = [&](int key) {
      const int at = page_of(key);
      return Pages{table[at], key - at * ps};
    };
    auto check = [&](Pages& p) {   // a page outside of the cache is not read
      const bool out = (uint32_t)p.page >= (uint32_t)a.kv.pages;
      bad |= out;
      p.page = out ? 0 : p.page;
    };
    auto inside = [&](int base) { return base >= first && base + kTile <= len; };
    // The page of group g's first key and the place of that key in it: 8 keys from a multiple of 8 lie in one page, and
    // so do those of them that are inside.  Where pages do not hold whole groups (P8 false), every load finds its own.
    auto lookup = [&](int base) {
      if constexpr (!P8) return Pages{0, 0};
      return find(min(max(base + g * 8, first), last));
    };
    uint32_t kr[2][NM][KW];   // two 16-key tiles of K
    uint32_t vr[8][NH][VD * (int)sizeof(C) / 4];
    auto take_k = [&](int c, const char* row) {
      if constexpr (F8 && FULL) {
#pragma unroll
        for (int i = 0; i < NM; i += 2) {
          const v4u x = *(const v4u*)(row + dim_at(i));
          kr[c][i][0] = x.x; kr[c][i][1] = x.y; kr[c][i + 1][0] = x.z; kr[c][i + 1][1] = x.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < NM; ++i) {
          const int d = dim_at(i);
          const char* src = row + (FULL || d < D ? d : 0) * (int)sizeof(C);
          if constexpr (F8) {
            const v2u x = *(const v2u*)src;
            kr[c][i][0] = x.x; kr[c][i][1] = x.y;
          } else {
            const v4u x = *(const v4u*)src;
            kr[c][i][0] = x.x; kr[c][i][1] = x.y; kr[c][i][2] = x.z; kr[c][i][3] = x.w;
          }
        }
      }
    };
    // A load of V takes whole lines that nobody reads again: they leave the caches first (2.6 GB of bf16 keys and values 450 ->
    // 406 us, 5.8 -> 6.5 TB/s; caches of 40 MB lose up to 5%).  K's lines are read by two or four loads of a step: the same there
    // costs 3-14%.
    auto take_v = [&](int j, const char* row) {
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        const int d = h * 16 * VD + n * VD;
        const char* src = row + (FULL || d < D ? d : 0) * (int)sizeof(C);
        if constexpr (VD * sizeof(C) == 16) {
          const v4u x = __builtin_nontemporal_load((const v4u*)src);
          vr[j][h][0] = x.x; vr[j][h][1] = x.y; vr[j][h][2] = x.z; vr[j][h][3] = x.w;
        } else if constexpr (VD * sizeof(C) == 8) {
          const v2u x = __builtin_nontemporal_load((const v2u*)src);
          vr[j][h][0] = x.x; vr[j][h][1] = x.y;
        } else {
          vr[j][h][0] = __builtin_nontemporal_load((const uint32_t*)src);
        }
      }
    };
    // A row is at base + page * page stride + place * token stride; inside of the sequence a group's rows follow one
    // another, a constant apart where a page is one run (TIGHT), so that a step's loads share one address.
    auto load_k = [&](int base, const Pages& p) {
      if constexpr (P8) {
        const int src = (n >> 2) * 16;
        const uint32_t page = __shfl(p.page, src);
        const int place = __shfl(p.place, src);
        const char* at = kb + (uint64_t)page * k_page;
        if (inside(base)) {
          const char* row = at + (uint64_t)(uint32_t)(place + (n & 3)) * k_tok;
          take_k(0, row);
          take_k(1, row + 4 * (TIGHT ? (uint32_t)RB : k_tok));
        } else {
          const int own = min(max(base + (n >> 2) * 8, first), last);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int key = min(max(base + (n >> 2) * 8 + c * 4 + (n & 3), first), last);
            take_k(c, at + (uint64_t)(uint32_t)(place + key - own) * k_tok);
          }
        }
      } else {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          Pages one = find(min(max(base + (n >> 2) * 8 + c * 4 + (n & 3), first), last));
          check(one);
          take_k(c, kb + (uint64_t)(uint32_t)one.page * k_page + (uint64_t)(uint32_t)one.place * k_tok);
        }
      }
    };
    auto load_v = [&](int base, const Pages& p) {
      if constexpr (P8) {
        const char* at = vb + (uint64_t)(uint32_t)p.page * v_page + (uint64_t)(uint32_t)p.place * v_tok;
        if (inside(base)) {
#pragma unroll
          for (int j = 0; j < 8; ++j) take_v(j, at + j * (TIGHT ? (uint32_t)RB : v_tok));
        } else {
          const int own = min(max(base + g * 8, first), last);
#pragma unroll
          for (int j = 0; j < 8; ++j) take_v(j, at + (uint32_t)(min(max(base + g * 8 + j, first), last) - own) * v_tok);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          Pages one = find(min(max(base + g * 8 + j, first), last));
          check(one);
          take_v(j, vb + (uint64_t)(uint32_t)one.page * v_page + (uint64_t)(uint32_t)one.place * v_tok);
        }
      }
    };

    const int hop = kTile * nkw;
    int base = k_begin + kTile * kw;
    Pages now = lookup(base);
    check(now);
    load_k(base, now);
    load_v(base, now);
    Pages next = lookup(base + hop);   // past the split: clamped, still a key of the sequence
    for (int s = 0; s < steps; ++s, base += hop) {
      v4f sc[2] = {v4f{0.f, 0.f, 0.f, 0.f}, v4f{0.f, 0.f, 0.f, 0.f}};
      int again = 0;
      if constexpr (QLDS) asm volatile("" : "+v"(again));   // read anew in every step
#pragma unroll
      for (int i = 0; i < NM; ++i) {
        v4u qi;
        if constexpr (QLDS) qi = *(const v4u*)(mine + again + i * 1024);
        else qi = q[i];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          v4u x;
          if constexpr (F8) x = widen8<T>(kr[c][i][0], kr[c][i][1]);
          else x = v4u{kr[c][i][0], kr[c][i][1], kr[c][i][2], kr[c][i][3]};
          if constexpr (!FULL) x = dim_at(i) < D ? x : v4u{0, 0, 0, 0};
          sc[c] = mfma(x, qi, sc[c], T{});
        }
      }
      const bool more = s + 1 < steps;
      if (more) {
        check(next);
        load_k(base + hop, next);
      }
      const bool edge = base < first || base + kTile > k_end;
      float top = -inf;
#pragma unroll
      for (int j = 0; j < 8; ++j) sc[j >> 2][j & 3] *= scale;
      if (edge) {
        asm volatile("");   // a branch: most steps have no edge
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int key = base + g * 8 + j;
          if (key < first || key >= k_end) sc[j >> 2][j & 3] = -inf;
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) top = fmaxf(top, sc[j >> 2][j & 3]);
      const float mn = fmaxf(m, max4(top)), mb = base_of(mn);
      if (__any(mn != m)) {   // rarely, once the first keys were seen
        const float c = __builtin_amdgcn_exp2f(m - mb);
        l *= c;
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t] *= c;
      }
      m = mn;
      float sum = 0.f, p[8];
      const float pb = mb - kLift<T>;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        p[j] = __builtin_amdgcn_exp2f(sc[j >> 2][j & 3] - pb);
        sum += p[j];
      }
      l += sum;
      const v4u pt{pack2<T>(p[0], p[1]), pack2<T>(p[2], p[3]), pack2<T>(p[4], p[5]), pack2<T>(p[6], p[7])};
      if (edge) {   // a weight of 0 does not silence a value that is not finite
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int key = base + g * 8 + j;
          if (key < first || key >= k_end)
#pragma unroll
            for (int h = 0; h < NH; ++h)
#pragma unroll
              for (int w = 0; w < VD * (int)sizeof(C) / 4; ++w) vr[j][h][w] = 0;
        }
      }
#pragma unroll
      for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int w = 0; w < VD * (int)sizeof(C) / 4; ++w) {
          if constexpr (F8) {   // four dims of the lane's keys
#pragma unroll
            for (int hi = 0; hi < 2; ++hi) {
              uint32_t y[4];
#pragma unroll
              for (int j = 0; j < 4; ++j)
                y[j] = __builtin_amdgcn_perm(vr[2 * j + 1][h][w], vr[2 * j][h][w], hi ? 0x07030602 : 0x05010400);
              const int t = h * VD + w * 4 + hi * 2;
              const v4u lo{widen<false>(y[0], T{}), widen<false>(y[1], T{}), widen<false>(y[2], T{}), widen<false>(y[3], T{})};
              const v4u up{widen<true>(y[0], T{}), widen<true>(y[1], T{}), widen<true>(y[2], T{}), widen<true>(y[3], T{})};
              acc[t] = mfma(lo, pt, acc[t], T{});
              acc[t + 1] = mfma(up, pt, acc[t + 1], T{});
            }
          } else {
#pragma unroll
            for (int hi = 0; hi < 2; ++hi) {
              v4u x;
#pragma unroll
              for (int j = 0; j < 4; ++j)
                x[j] = __builtin_amdgcn_perm(vr[2 * j + 1][h][w], vr[2 * j][h][w], hi ? 0x07060302 : 0x05040100);
              acc[h * VD + w * 2 + hi] = mfma(x, pt, acc[h * VD + w * 2 + hi], T{});
            }
          }
        }
      if (more) {
        load_v(base + hop, next);
        next = lookup(base + 2 * hop);
      }
    }
    l = sum4(l);
    if (__any(bad)) l = __builtin_nanf("");
  }

  // the waves' sums, joined: lane (n, g) holds dims h * 16 VD + (4 g + i) VD + t of head n in acc[h VD + t][i]
  {
    float* to = red + (wave * 16 + n) * RS;
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int t = 0; t < VD; t += 4)
          *(v4f*)(to + h * 16 * VD + (4 * g + i) * VD + t) =
              v4f{acc[h * VD + t][i], acc[h * VD + t + 1][i], acc[h * VD + t + 2][i], acc[h * VD + t + 3][i]};
    if (g == 0) {
      stat[wave * 16 + n][0] = m;
      stat[wave * 16 + n][1] = l;
    }
  }
  __syncthreads();
  const float nan = __builtin_nanf("");
  const float v_scale = a.kv.v_scale ? a.kv.v_scale[kvh] : 1.f;
  const int64_t unit = (int64_t)b * gridDim.x + blockIdx.x;
  const int quads = D / 4;
  // [splits][R][D], then [splits][R][2] (room for a full block's rows in every unit)
  float* part = a.partials + unit * a.splits * min(rows_wg, group) * (D + 4);
  auto store = [&](int r, int d, v4f x, float f) {
    T* to = (T*)a.out + b * a.out_row + (int64_t)(kvh * group + row0 + r) * a.out_head + d;
    *(v2u*)to = v2u{pack2<T>(x[0] * f, x[1] * f), pack2<T>(x[2] * f, x[3] * f)};
  };
  auto store_lse = [&](int r, float M, float L) {
    a.lse[(int64_t)b * a.q_heads + kvh * group + row0 + r] = L == 0.f ? -inf : (M - kLift<T> + __builtin_amdgcn_logf(L)) * kLn2;
  };
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(part, 0, a.splits * R * (D + 4) * 4, 0x00020000);
  constexpr int kDevice = 16;   // device-scope cache policy (sc1): through the XCD's L2
  for (int x = threadIdx.x; x < R * quads; x += 64 * kWaves) {
    const int r = x / quads, d = (x - r * quads) * 4, tile = r >> 4;
    float M = -inf;
    for (int k = 0; k < nkw; ++k) M = fmaxf(M, stat[(tile + k * a.row_waves) * 16 + (r & 15)][0]);
    const float Mb = base_of(M);
    v4f o{0.f, 0.f, 0.f, 0.f};
    float L = 0.f;
    for (int k = 0; k < nkw; ++k) {
      const int w = (tile + k * a.row_waves) * 16 + (r & 15);
      const float f = __builtin_amdgcn_exp2f(stat[w][0] - Mb);
      L += stat[w][1] * f;
      o += *(const v4f*)(red + w * RS + d) * f;
    }
    if (too_long) L = nan;
    if (ns == 1) {
      store(r, d, o, L == 0.f ? 0.f : v_scale / L);
      if (a.lse && d == 0) store_lse(r, M, L);
    } else {
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4u, o), rs, ((split * R + r) * D + d) * 4, 0, kDevice);
      if (d == 0)
        __builtin_amdgcn_raw_buffer_store_b64(v2u{__builtin_bit_cast(uint32_t, M), __builtin_bit_cast(uint32_t, L)}, rs,
                                              (a.splits * R * D + (split * R + r) * 2) * 4, 0, kDevice);
    }
  }
  if (ns == 1 || a.join_apart) return;
  // The sequence's splits join in the workgroup that arrives last, in split order: partials move through device-coherent
  // accesses alone; every store is complete before the arrival count.  All of a value's loads are in flight at once.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) flag = __hip_atomic_fetch_add(a.counters + unit, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (flag != ns - 1) return;
  asm volatile("" ::: "memory");
  if (threadIdx.x == 0) __hip_atomic_store(a.counters + unit, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);   // next launch
  for (int x = threadIdx.x; x < R * quads; x += 64 * kWaves) {
    const int r = x / quads, d = (x - r * quads) * 4;
    v2u st[kJoinSplits];
    v4u y[kJoinSplits];
#pragma unroll
    for (int s = 0; s < kJoinSplits; ++s)
      if (s < ns) {
        st[s] = __builtin_amdgcn_raw_buffer_load_b64(rs, (a.splits * R * D + (s * R + r) * 2) * 4, 0, kDevice);
        y[s] = __builtin_amdgcn_raw_buffer_load_b128(rs, ((s * R + r) * D + d) * 4, 0, kDevice);
      }
    Joined j;
#pragma unroll
    for (int s = 0; s < kJoinSplits; ++s)
      if (s < ns) j.add(st[s], y[s]);
    store(r, d, j.o, j.l == 0.f ? 0.f : v_scale / j.l);
    if (a.lse && d == 0) store_lse(r, j.m, j.l);
  }
}

// The join of more splits than one workgroup takes at once: a workgroup for each query head, its threads over the splits and
// the dims.  (One workgroup per sequence and key head took 16 us for 64 splits of 5 heads, 39 for 128 of 16.)  96 splits of 40 heads: 6.1 us,
// of which a launch that waits for another takes about half.
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void attention_join_kernel(AttnArgs a) {
  __shared__ __align__(16) float sums[THREADS][4];
  __shared__ float stat[THREADS][2];
  const int b = blockIdx.y, h = blockIdx.x, group = a.q_heads / a.kv.heads, kvh = h / group, D = a.kv.dim;
  const int rows_wg = 16 * a.row_waves, rb = h % group / rows_wg, r = h % group - rb * rows_wg, R = min(rows_wg, group - rb * rows_wg);
  const int len0 = max(0, a.lengths[b]), len = len0 > a.max_length ? 0 : len0;
  const int first = a.window > 0 ? max(0, len - a.window) : 0, start = first & ~(kTile - 1);
  const int ns = splits_of(start, len, a.chunk);
  if (ns == 1) return;   // written already
  const int64_t unit = ((int64_t)b * a.kv.heads + kvh) * a.row_blocks + rb;
  const float* part = a.partials + unit * a.splits * min(rows_wg, group) * (D + 4);
  const float* part_stat = part + (int64_t)a.splits * R * D;
  const int quads = D / 4, lanes = THREADS / quads, own = threadIdx.x / quads, d = (threadIdx.x - own * quads) * 4;
  Joined j;
  if (own < lanes) {
    constexpr int kBatch = 8;
    for (int s0 = own; s0 < ns; s0 += kBatch * lanes) {
      v2u st[kBatch];
      v4u y[kBatch];
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int s = min(s0 + k * lanes, ns - 1);
        st[k] = *(const v2u*)(part_stat + (s * R + r) * 2);
        y[k] = *(const v4u*)(part + (s * R + r) * D + d);
      }
#pragma unroll
      for (int k = 0; k < kBatch; ++k)
        if (s0 + k * lanes < ns) j.add(st[k], y[k]);
    }
  }
  *(v4f*)sums[threadIdx.x] = j.o;
  stat[threadIdx.x][0] = j.m;
  stat[threadIdx.x][1] = j.l;
  __syncthreads();
  if (own > 0) return;
  Joined all;
  for (int k = 0; k < lanes; ++k) {
    const int x = k * quads + threadIdx.x;
    all.add(*(const v2u*)stat[x], *(const v4u*)sums[x]);
  }
  const float f = all.l == 0.f ? 0.f : (a.kv.v_scale ? a.kv.v_scale[kvh] : 1.f) / all.l;
  T* to = (T*)a.out + b * a.out_row + h * a.out_head + d;
  *(v2u*)to = v2u{pack2<T>(all.o[0] * f, all.o[1] * f), pack2<T>(all.o[2] * f, all.o[3] * f)};
  if (a.lse && threadIdx.x == 0)
    a.lse[(int64_t)b * a.q_heads + h] = all.l == 0.f ? -__builtin_huge_valf() : (all.m - kLift<T> + __builtin_amdgcn_logf(all.l)) * kLn2;
}

// How a call is cut: workgroups over the query heads of a key head, and splits of `chunk` keys.
struct Cut { int row_waves, row_blocks, splits, chunk; };

// About as many workgroups as stay resident, of 256 keys at least (32 x 4000 tokens in bf16: 3 a CU 69.9 us, 4 62.4, 6 66.3,
// 8 64.2; 64 x 3000 of 256 dims in fp8: 3 a CU 50.2, 4 58.3, 5 55.6; 8 x 2000 in splits of 128 keys or more 16.5, of 256 13.6; of 32
// heads that share one of keys, whose waves see more of a split each, 8 x 4000 13.3 and 15.6, of 128 heads 4 x 4000 17.7 and 22.9).
// The splits' partial sums lie in the workspace: as many splits as it holds, one (which needs none) in any.
Cut cut_of(int batch, int q_heads, int kv_heads, int dim, int size, int max_length, int window, int64_t workspace_bytes) {
  const int group = q_heads / kv_heads, tiles = (group + 15) / 16;
  Cut c;
  c.row_waves = tiles >= 3 ? 4 : tiles;
  c.row_blocks = (tiles + c.row_waves - 1) / c.row_waves;
  // keys a sequence can have, from a multiple of the step
  const int64_t span = std::min<int64_t>(max_length, window > 0 ? (int64_t)window + kTile - 1 : max_length);
  const int64_t units = (int64_t)batch * kv_heads * c.row_blocks, wanted = (size == 1 ? 3LL : 4LL) * device_cus();
  const int64_t least = (c.row_waves == 1 ? 2 * kWaves : 4) * kTile;   // keys of the shortest split
  int64_t splits = std::max<int64_t>(1, std::min((wanted + units - 1) / std::max<int64_t>(1, units), (span + least - 1) / least));
  splits = std::min<int64_t>(splits, kMostSplits);
  const int64_t each = units * std::min(16 * c.row_waves, group) * (dim + 4) * 4;   // bytes of one split of all units
  if (units > GQK_CTR_WORDS || workspace_bytes < GQK_CTR_BYTES) splits = 1;
  else if (each > 0) splits = std::max<int64_t>(1, std::min(splits, (workspace_bytes - GQK_CTR_BYTES) / each));
  c.chunk = (int)std::max<int64_t>(kTile, ((span + splits - 1) / splits + kTile - 1) / kTile * kTile);
  c.splits = (int)std::max<int64_t>(1, (span + c.chunk - 1) / c.chunk);
  return c;
}

// The general form takes any head dim up to DP and any page size; whole heads (FULL), pages of a multiple of 8 tokens (P8)
// and pages that are one run of memory (TIGHT) have fewer addresses to compute, the last one for each step.  Bound by memory like them:
// 32 x 4000 of 80 dims 45.8 us (4.5 TB/s), of 192 dims 106 us (4.6); of 128 dims in pages of 7 tokens 63.9, of 16 61.8.
template <typename T, typename C, int DP>
void launch(const AttnArgs& a, dim3 grid, bool full, hipStream_t st) {
  const bool p8 = a.kv.page_size % 8 == 0, tight = a.kv.k_token == DP && a.kv.v_token == DP;
  if (full && p8 && tight) attention_kernel<T, C, DP, true, true, true><<<grid, 64 * kWaves, 0, st>>>(a);
  else if (full && p8) attention_kernel<T, C, DP, true, true, false><<<grid, 64 * kWaves, 0, st>>>(a);
  else if (p8) attention_kernel<T, C, DP, false, true, false><<<grid, 64 * kWaves, 0, st>>>(a);
  else attention_kernel<T, C, DP, false, false, false><<<grid, 64 * kWaves, 0, st>>>(a);
}

template <typename T, typename C>
void launch(const AttnArgs& a, dim3 grid, hipStream_t st) {
  const int D = a.kv.dim;
  bool full = D == 64 || D == 128 || D == 256;
  if (sizeof(C) == 1)   // 16-byte loads of 8-bit keys
    full = full && !(((uintptr_t)a.kv.k | (uint64_t)a.kv.k_page | (uint64_t)a.kv.k_token | (uint64_t)a.kv.k_head) & 15);
  if (D <= 64) launch<T, C, 64>(a, grid, full, st);
  else if (D <= 128) launch<T, C, 128>(a, grid, full, st);
  else launch<T, C, 256>(a, grid, full, st);
}

}  // namespace
}  // namespace gqk

using namespace gqk;

extern "C" {

int64_t gqk_paged_attention_workspace_bytes(int batch, int q_heads, int kv_heads, int dim, int max_length, int window) {
  if (batch < 0 || kv_heads < 1 || q_heads < kv_heads || q_heads % kv_heads || dim < 8 || dim > 256 || dim % 8 ||
      max_length < 0 || max_length > GQK_MAX_KEYS || window < 0)
    return decode_fail(GQK_ERR_SHAPE, "paged_attention: %d sequences, %d / %d heads of %d, max_length %d, window %d", batch,
                       q_heads, kv_heads, dim, max_length, window);
  // of either size of pages: the larger
  const Cut c = cut_of(batch, q_heads, kv_heads, dim, 2, max_length, window, INT64_MAX);
  const int64_t rows = std::min(16 * c.row_waves, q_heads / kv_heads), units = (int64_t)batch * kv_heads * c.row_blocks;
  return c.splits > 1 ? GQK_CTR_BYTES + units * rows * c.splits * (dim + 4) * 4 : 0;
}

int gqk_paged_attention(const void* q, int64_t q_row, int64_t q_head, int dtype, int batch, int q_heads,
                        const gqk_pages* pages, const int32_t* table, int64_t table_row, int table_width,
                        const int32_t* lengths, int max_length, int window, float scale, void* out, int64_t out_row,
                        int64_t out_head, float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
  if (dtype != GQK_DTYPE_BF16 && dtype != GQK_DTYPE_F16) return decode_fail(GQK_ERR_ARG, "paged_attention: dtype %d", dtype);
  if (const int rc = check_pages("paged_attention", pages, dtype)) return rc;
  if (batch < 0 || batch > 65535 || q_heads < 1 || q_heads % pages->heads)
    return decode_fail(GQK_ERR_SHAPE, "paged_attention: %d sequences of %d query heads over %d", batch, q_heads, pages->heads);
  if (window < 0 || max_length < 0 || max_length > GQK_MAX_KEYS || table_width < 0 ||
      (int64_t)max_length > (int64_t)table_width * pages->page_size)
    return decode_fail(GQK_ERR_SHAPE, "paged_attention: window %d, lengths up to %d in %d pages of %d tokens", window, max_length,
                       table_width, pages->page_size);
  if (batch == 0) return GQK_OK;
  if (!q || !out || !lengths || (!table && max_length > 0)) return decode_fail(GQK_ERR_ARG, "paged_attention: null pointer");
  if (((uintptr_t)q | (uintptr_t)out) & 15 || (q_row | q_head | out_row | out_head) & 7)
    return decode_fail(GQK_ERR_SHAPE, "paged_attention: q and out are 16-byte aligned with strides that are multiples of 8");
  const Cut c = cut_of(batch, q_heads, pages->heads, pages->dim, pages->dtype == GQK_DTYPE_FP8 ? 1 : 2, max_length, window,
                       workspace ? workspace_bytes : 0);
  if (c.splits > 1 && (uintptr_t)workspace & 255)
    return decode_fail(GQK_ERR_SHAPE, "paged_attention: workspace is not 256-byte aligned");
  AttnArgs a{};
  a.q = q; a.q_row = q_row; a.q_head = q_head; a.kv = *pages; a.table = table; a.table_row = table_row; a.lengths = lengths;
  a.out = out; a.out_row = out_row; a.out_head = out_head; a.lse = lse; a.q_heads = q_heads; a.max_length = max_length;
  a.window = window; a.scale = scale * kLog2e; a.row_waves = c.row_waves; a.row_blocks = c.row_blocks; a.chunk = c.chunk;
  a.splits = c.splits;
  a.counters = (int*)workspace;
  a.partials = workspace ? (float*)((char*)workspace + GQK_CTR_BYTES) : nullptr;
  // key / page_size for keys below 2^31: 2^(31 + bits) / page_size rounded up fits 32 bits, its excess times a key stays
  // below 2^(31 + bits)
  int bits = 0;
  while (((int64_t)1 << bits) < pages->page_size) ++bits;
  a.shift = bits;
  a.magic = (uint32_t)((((uint64_t)1 << (31 + bits)) + pages->page_size - 1) / pages->page_size);
  // one workgroup joins up to 16 splits, of heads that its threads go over twice at most (in a launch of their own and in it: 32 heads
  // of 128 dims over one, 8 x 4000, 15.7 us and 21.3; 16 heads, two rounds, 16 x 2000, 17.9 and 16.6)
  a.join_apart = c.splits > kJoinSplits ||
                 (c.splits > 1 && std::min(16 * c.row_waves, q_heads / pages->heads) * (pages->dim / 4) > 2 * 64 * kWaves);
  const dim3 grid(pages->heads * c.row_blocks, batch, c.splits);
  const hipStream_t st = (hipStream_t)stream;
  const bool bf = dtype == GQK_DTYPE_BF16;
  if (pages->dtype == GQK_DTYPE_FP8) {
    if (bf) launch<bf16_t, fp8_t>(a, grid, st);
    else launch<f16_t, fp8_t>(a, grid, st);
  } else if (bf) {
    launch<bf16_t, bf16_t>(a, grid, st);
  } else {
    launch<f16_t, f16_t>(a, grid, st);
  }
  if (a.join_apart) {
    const dim3 all(q_heads, batch);
    if (c.splits > 128) {   // more threads cost more to bring together (us of 256 and 512: 256 splits 22.7 and 21.1, 16 13.2 and 14.0)
      if (bf) attention_join_kernel<bf16_t, 512><<<all, 512, 0, st>>>(a);
      else attention_join_kernel<f16_t, 512><<<all, 512, 0, st>>>(a);
    } else {
      if (bf) attention_join_kernel<bf16_t, 256><<<all, 256, 0, st>>>(a);
      else attention_join_kernel<f16_t, 256><<<all, 256, 0, st>>>(a);
    }
  }
  return decode_launched("paged_attention");
}

}  // extern "C"
