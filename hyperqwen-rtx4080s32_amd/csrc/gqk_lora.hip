// gqk_lora.hip - low-rank adapters of many requests beside a shared projection.
//
//   out[m, n] = y[m, n] + s_i sum_r B_i[n, r] h[m, p(n), r],   h[m, p, r] = sum_k A_i[p, r, k] x[m, k]
//
// with i = ids[m] the row's adapter (negative: out = y) and p(n) the part (q, k, v; gate, up) that
// column n belongs to.  h is kept in 32 bits in the workspace, after its counter region.
#include <algorithm>
#include "gqk_decode.h"

namespace gqk {
namespace {

typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

constexpr int kParts = 8;
constexpr int kDownWaves = 8, kUpWaves = 4;
constexpr int kBlock = 64;       // rows whose adapters a workgroup sorts out: one per lane
constexpr int kRankTiles = 4;    // 16-rank tiles of a workgroup of the first kernel
constexpr int kHPad = 68;        // row stride of its sums in LDS
constexpr int kNone = -1, kBad = -2;

struct LoraArgs {
  const void *y, *x, *a, *b;
  void* out;
  int64_t y_row, x_row, out_row, K, N;
  const void* ids;
  const float* scales;
  float* h;                  // [splits][M][parts * rank]
  int M, slots, parts, rank, wide_ids;
  int splits, chunks;        // splits of K; chunks of 64 ranks
  int columns;               // of a workgroup of the second kernel
  int wide_y;                // y and out are 16-byte aligned in every row
  int64_t ends[kParts];      // one past each part's last column
};

__device__ __forceinline__ v4f mfma(v4u a, v4u b, v4f c, bf16_t) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}
__device__ __forceinline__ v4f mfma(v4u a, v4u b, v4f c, f16_t) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

// Rows of one block that go with one adapter (or with none, kNone, or a bad id, kBad).
struct Unit {
  int adapter, count;
  const int* row;   // their numbers within the block
};

// Unit u (of up to `most` rows) of the block's rows: adapters in the order of their first row, each one's rows in order.
// A lane holds one row's id; a ballot finds the rows that share it, whose numbers go to LDS in order, a list for each
// wave.  False: the block has fewer units.  All waves find the same.
__device__ __forceinline__ bool find_unit(const LoraArgs& a, int64_t row0, int u, int most, int* lists, Unit& out) {
  const int lane = threadIdx.x & 63;
  const int64_t m = row0 + lane;
  int id = kNone;
  if (m < a.M) {
    const int64_t i = index_at(a.ids, a.wide_ids, m);
    id = i < 0 ? kNone : i >= a.slots ? kBad : (int)i;
  }
  uint64_t left = __ballot(m < a.M);
  while (left) {
    const int who = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
    const uint64_t same = __ballot(id == who) & left;
    const int count = __popcll(same), units = (count + most - 1) / most;
    if (u < units) {
      out.adapter = who;
      out.count = min(count - u * most, most);
      const int place = __builtin_amdgcn_mbcnt_hi((uint32_t)(same >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)same, 0)) - u * most;
      int* mine = lists + (threadIdx.x >> 6) * kBlock;
      if ((same >> lane & 1) && place >= 0 && place < out.count) mine[place] = lane;
      __builtin_amdgcn_wave_barrier();
      out.row = mine;
      return true;
    }
    u -= units;
    left &= ~same;
  }
  return false;
}

// 16 bytes at a byte offset from a base that the whole wave shares; zeros past `bytes`
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void* p, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (int)min(bytes, (int64_t)0x7ffffff0), 0x00020000);
}
constexpr uint32_t kOutside = 0x80000000u;   // an offset past every buffer
__device__ __forceinline__ v4u load16(__amdgpu_buffer_rsrc_t rs, uint32_t offset, uint32_t shared) {
  return __builtin_amdgcn_raw_buffer_load_b128(rs, offset, shared, 0);
}

// h = A x of one unit's rows, 64 ranks, one split of K: the ranks are the matrix instruction's rows and the batch
// rows its columns, both operands straight from global memory (8 values along K per lane).  The waves split the split's
// steps among themselves and join in LDS, in order.  A step is 64 values of K, so that a wave reads whole 128-byte lines
// of every row.
template <typename T, int TT>
__global__ __launch_bounds__(64 * kDownWaves, 2) void lora_down_kernel(LoraArgs a) {
  constexpr int kDepth = 2;   // steps in flight
  __shared__ __align__(16) float red[kDownWaves][16][kHPad];
  __shared__ int lists[kDownWaves * kBlock];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
  const int chunk = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
  const int64_t row0 = (int64_t)blockIdx.z * kBlock;
  const int PR = a.parts * a.rank, rank0 = chunk * 16 * kRankTiles, tiles = min(kRankTiles, (PR - rank0 + 15) / 16);
  const int all = (int)((a.K + 63) / 64), s0 = (int)((int64_t)all * split / a.splits), s1 = (int)((int64_t)all * (split + 1) / a.splits);
  const int K = (int)a.K, tail = K % 64;
  for (int u = blockIdx.y;; u += gridDim.y) {
    Unit unit;
    if (!find_unit(a, row0, u, 16 * TT, lists, unit)) return;
    if (unit.adapter < 0) continue;
    const int rows = (unit.count + 15) / 16;   // tiles of rows
    const T* A = (const T*)a.a + ((int64_t)unit.adapter * PR + rank0) * a.K;
    const T* X = (const T*)a.x + row0 * a.x_row;
    const __amdgpu_buffer_rsrc_t ra = buffer_of(A, (int64_t)min(16 * kRankTiles, PR - rank0) * a.K * 2);
    const __amdgpu_buffer_rsrc_t rx = buffer_of(X, ((int64_t)kBlock * a.x_row) * 2);
    uint32_t ao[kRankTiles], xo[TT];
#pragma unroll
    for (int t = 0; t < kRankTiles; ++t) ao[t] = min(t * 16 + n, PR - rank0 - 1) * (uint32_t)K * 2 + g * 16;
#pragma unroll
    for (int t = 0; t < TT; ++t) xo[t] = unit.row[min(t * 16 + n, unit.count - 1)] * (uint32_t)a.x_row * 2 + g * 16;
    v4f acc[kRankTiles][TT];
#pragma unroll
    for (int r = 0; r < kRankTiles; ++r)
#pragma unroll
      for (int t = 0; t < TT; ++t) acc[r][t] = v4f{0.f, 0.f, 0.f, 0.f};
    v4u av[kDepth][2][kRankTiles], xv[kDepth][2][TT];
    auto load = [&](int d, int s) {
      const uint32_t at = s * 128;
      const bool whole = tail == 0 || s + 1 < all;   // K may end inside the last step
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const bool in = whole || k * 32 + g * 8 < tail;
#pragma unroll
        for (int t = 0; t < TT; ++t)
          if (t < rows) xv[d][k][t] = load16(rx, in ? xo[t] + k * 64 : kOutside, at);
#pragma unroll
        for (int t = 0; t < kRankTiles; ++t)
          if (t < tiles) av[d][k][t] = load16(ra, in ? ao[t] + k * 64 : kOutside, at);
      }
    };
    const int steps = s1 - s0 > wave ? (s1 - s0 - wave + kDownWaves - 1) / kDownWaves : 0, first = s0 + wave;
#pragma unroll
    for (int d = 0; d < kDepth; ++d)
      if (d < steps) load(d, first + d * kDownWaves);
    for (int i = 0; i < steps; i += kDepth)
#pragma unroll
      for (int d = 0; d < kDepth; ++d)
        if (i + d < steps) {
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int r = 0; r < kRankTiles; ++r)
              if (r < tiles)
#pragma unroll
                for (int t = 0; t < TT; ++t)
                  if (t < rows) acc[r][t] = mfma(av[d][k][r], xv[d][k][t], acc[r][t], T{});
          if (i + d + kDepth < steps) load(d, first + (i + d + kDepth) * kDownWaves);
        }
    // lane (n, g) holds ranks 16 r + 4 g .. + 3 of column n
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      if (t >= rows) break;
      __syncthreads();
#pragma unroll
      for (int r = 0; r < kRankTiles; ++r)
        if (r < tiles) *(v4f*)&red[wave][n][r * 16 + g * 4] = acc[r][t];
      __syncthreads();
      const int row = threadIdx.x >> 5, c = (threadIdx.x & 31) * 2;   // 16 rows, 2 ranks a thread
      if (t * 16 + row < unit.count && rank0 + c < PR) {
        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kDownWaves; ++w) {
          sum.x += red[w][row][c];
          sum.y += red[w][row][c + 1];
        }
        *(float2*)(a.h + ((int64_t)split * a.M + row0 + unit.row[t * 16 + row]) * PR + rank0 + c) = sum;
      }
    }
  }
}

// out = y + s B h of one unit's rows and `columns` columns of one part.  The ranks that h has in 32 bits go into the
// product as two values of T each, h = hi + lo, in one instruction: 16 ranks of hi and the same 16 of lo against B's 16
// ranks twice (rounding h to T alone would put 2^-9 of the update, for bf16, on top of the output's own rounding; the second
// half of the instruction would be idle).  fp16 takes h over a power of two near its row's largest, to stay in range.
// B and y of a wave's first columns are on their way while h is gathered, those of the next while these are computed.
template <typename T, int TT>
__global__ __launch_bounds__(64 * kUpWaves, 2) void lora_up_kernel(LoraArgs a) {
  constexpr bool kF16 = __is_same(T, f16_t);
  constexpr int kSteps = 4;                               // 16-rank steps of B that are loaded ahead
  constexpr int kRowThreads = 64 * kUpWaves / (16 * TT);  // threads that gather one row of h
  constexpr int kOctets = 32 / kRowThreads;               // octets of ranks of one of them, at most
  extern __shared__ __align__(16) char lds[];             // h: [16 TT rows][hi, lo][ranks + 8]
  __shared__ float factor[TT * 16];
  __shared__ int lists[kUpWaves * kBlock];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
  const int64_t row0 = (int64_t)blockIdx.z * kBlock;
  const int PR = a.parts * a.rank, steps = (a.rank + 15) / 16, hrow = steps * 16 + 8;
  T* const hs = (T*)lds;
  // the part and its columns
  int part = 0, block = blockIdx.x;
  int64_t begin = 0;
  for (;;) {
    const int blocks = (int)((a.ends[part] - begin + a.columns - 1) / a.columns);
    if (block < blocks) break;
    block -= blocks;
    begin = a.ends[part++];
  }
  const int64_t c_begin = begin + (int64_t)block * a.columns;
  const int width = (int)min(a.ends[part] - c_begin, (int64_t)a.columns);
  for (int u = blockIdx.y;; u += gridDim.y) {
    Unit unit;
    if (!find_unit(a, row0, u, 16 * TT, lists, unit)) return;
    const bool some = unit.adapter >= 0;
    if (unit.adapter == kNone && a.out == a.y) continue;
    const int rows = (unit.count + 15) / 16;
    const __amdgpu_buffer_rsrc_t rb = buffer_of(
        (const T*)a.b + ((int64_t)max(unit.adapter, 0) * a.N + c_begin) * a.rank, some ? (int64_t)width * a.rank * 2 : 0);
    const T* y[TT];
    T* out[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      const int64_t m = row0 + unit.row[min(t * 16 + n, unit.count - 1)];
      y[t] = (const T*)a.y + m * a.y_row + c_begin + g * 8;
      out[t] = (T*)a.out + m * a.out_row + c_begin + g * 8;
    }
    // 32 columns at a time: as rows of two 16-row tiles dealt so that a lane gets 8 in a row of its batch row
    v4u bv[2][kSteps][2], yv[2][TT];
    auto load_b = [&](v4u (&to)[kSteps][2], int c0, int k0) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const uint32_t at = min(c0 + (n >> 2) * 8 + c * 4 + (n & 3), width - 1) * (uint32_t)a.rank * 2 + (g & 1) * 16;
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
          if (k0 + k < steps) to[k][c] = load16(rb, (k0 + k) * 16 + (g & 1) * 8 < a.rank ? at + k * 32 : kOutside, k0 * 32);
      }
    };
    auto load = [&](int buf, int c0) {
      if (some) load_b(bv[buf], c0, 0);
      if (a.wide_y)
#pragma unroll
        for (int t = 0; t < TT; ++t)
          if (t * 16 + n < unit.count && c0 + g * 8 + 8 <= width) yv[buf][t] = *(const v4u*)(y[t] + c0);
    };
    float f[TT];
    auto finish = [&](int buf, int c0) {
      v4f acc[2][TT];
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int t = 0; t < TT; ++t) acc[c][t] = v4f{0.f, 0.f, 0.f, 0.f};
      if (some)
        for (int k0 = 0; k0 < steps; k0 += kSteps) {
          if (k0 > 0) load_b(bv[buf], c0, k0);
#pragma unroll
          for (int k = 0; k < kSteps; ++k)
            if (k0 + k < steps)
#pragma unroll
              for (int t = 0; t < TT; ++t)
                if (t < rows) {
                  const v4u hv = *(const v4u*)(hs + ((t * 16 + n) * 2 + (g >> 1)) * hrow + (k0 + k) * 16 + (g & 1) * 8);
#pragma unroll
                  for (int c = 0; c < 2; ++c) acc[c][t] = mfma(bv[buf][k][c], hv, acc[c][t], T{});
                }
        }
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        if (t * 16 + n >= unit.count) continue;
        auto value = [&](float base, int e) {
          return some ? base + acc[e >> 2][t][e & 3] * f[t] : unit.adapter == kNone ? base : __builtin_nanf("");
        };
        if (a.wide_y && c0 + g * 8 + 8 <= width) {
          T v[8];
          __builtin_memcpy(v, &yv[buf][t], 16);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = (T)value((float)v[e], e);
          __builtin_memcpy(__builtin_assume_aligned(out[t] + c0, 16), v, 16);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (c0 + g * 8 + e < width) out[t][c0 + e] = (T)value((float)y[t][c0 + e], e);
        }
      }
    };
    constexpr int hop = 32 * kUpWaves;
    int c0 = wave * 32;
    if (c0 < width) load(0, c0);
    if (some) {
      __syncthreads();   // the last unit's h has been read
      const int r = threadIdx.x / kRowThreads, c = threadIdx.x % kRowThreads;
      const int64_t m = row0 + unit.row[min(r, unit.count - 1)];
      float v[kOctets][8], top = 0.f;
#pragma unroll
      for (int q = 0; q < kOctets; ++q) {
        const int rank = (q * kRowThreads + c) * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[q][e] = 0.f;
        if (rank < a.rank && r < rows * 16) {
          const float* from = a.h + m * PR + part * a.rank + rank;
          const int64_t hop_h = (int64_t)a.M * PR;
          for (int sp = 0; sp < a.splits; sp += 4) {
            v4f lo[4], hi[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const v4f* p = (const v4f*)(from + min(sp + j, a.splits - 1) * hop_h);
              lo[j] = p[0];
              hi[j] = p[1];
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (sp + j < a.splits)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  v[q][e] += lo[j][e];
                  v[q][4 + e] += hi[j][e];
                }
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[q][e]));
      }
      float down = 1.f, up = 1.f;
      if constexpr (kF16) {
        for (int o = kRowThreads / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
        if (top > 0.f && top < __builtin_huge_valf()) {
          const int e = min(max(ilogbf(top), -100), 100);
          down = ldexpf(1.f, -e);
          up = ldexpf(1.f, e);
        }
      }
      if (c == 0) factor[r] = (a.scales ? a.scales[unit.adapter] : 1.f) * up;
#pragma unroll
      for (int q = 0; q < kOctets; ++q) {
        const int rank = (q * kRowThreads + c) * 8;
        if (rank < steps * 16 && r < rows * 16) {
          T hi[8], lo[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float x = v[q][e] * down;
            hi[e] = (T)x;
            const float back = (float)hi[e];
            lo[e] = fabsf(back) < __builtin_huge_valf() ? (T)(x - back) : (T)0.f;   // inf stays, without inf - inf
          }
          __builtin_memcpy(hs + (r * 2) * hrow + rank, hi, 16);
          __builtin_memcpy(hs + (r * 2 + 1) * hrow + rank, lo, 16);
        }
      }
      __syncthreads();
    }
#pragma unroll
    for (int t = 0; t < TT; ++t) f[t] = some && t < rows ? factor[t * 16 + n] : 0.f;
    for (; c0 < width; c0 += 2 * hop) {
      if (c0 + hop < width) load(1, c0 + hop);
      finish(0, c0);
      if (c0 + hop >= width) break;
      if (c0 + 2 * hop < width) load(0, c0 + 2 * hop);
      finish(1, c0 + hop);
    }
  }
}

// How a call is cut.  Down: splits of K so that the launch has about 512 workgroups, each wave at least two steps.
// Rows of a block that share an adapter go 16 to a workgroup up to kBlock rows in all, 64 above.
struct Cut { int splits, chunks, blocks; };

Cut cut_of(int M, int64_t K, int parts, int rank) {
  Cut c;
  c.chunks = (parts * rank + 16 * kRankTiles - 1) / (16 * kRankTiles);
  c.blocks = (M + kBlock - 1) / kBlock;
  const int64_t wgs = (int64_t)c.chunks * (M <= kBlock ? std::min(M, 16) : c.blocks);
  const int64_t steps = (K + 63) / 64;
  c.splits = (int)std::max<int64_t>(1, std::min<int64_t>({512 / wgs, steps / kDownWaves, 16}));
  return c;
}

template <typename T, int TT>
void launch(const LoraArgs& g, const Cut& c, hipStream_t st) {
  // units of a block: its adapters, none, bad ids, and what does not fit one unit; the kernels step on over more
  const int units = TT == 1 ? std::min(g.M, std::min(g.slots, kBlock) + 2 + kBlock / 16) : 2;
  int64_t blocks = 0, begin = 0;
  for (int p = 0; p < g.parts; ++p) {
    blocks += (g.ends[p] - begin + g.columns - 1) / g.columns;
    begin = g.ends[p];
  }
  if (g.slots > 0) lora_down_kernel<T, TT><<<dim3(c.splits * c.chunks, units, c.blocks), 64 * kDownWaves, 0, st>>>(g);
  const size_t lds = (size_t)16 * TT * 2 * ((g.rank + 15) / 16 * 16 + 8) * sizeof(T);
  lora_up_kernel<T, TT><<<dim3((unsigned)blocks, units, c.blocks), 64 * kUpWaves, lds, st>>>(g);
}

}  // namespace
}  // namespace gqk

using namespace gqk;

extern "C" {

int64_t gqk_lora_workspace_bytes(int M, int64_t K, int parts, int rank) {
  if (M < 0 || K < 0 || parts < 1 || parts > kParts || rank < 8 || rank > 256 || rank % 8)
    return decode_fail(GQK_ERR_SHAPE, "lora: %d rows of %lld, %d parts (at most %d), rank %d (a multiple of 8 in 8..256)", M,
                       (long long)K, parts, kParts, rank);
  return M == 0 ? GQK_CTR_BYTES : GQK_CTR_BYTES + (int64_t)cut_of(M, K, parts, rank).splits * M * parts * rank * 4;
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
  if (K > GQK_LORA_MAX_K || x_row > GQK_LORA_MAX_K)
    return decode_fail(GQK_ERR_SHAPE, "lora_add: K %lld or x's row stride %lld above %d", (long long)K, (long long)x_row, GQK_LORA_MAX_K);
  if (((uintptr_t)x | (uintptr_t)a | (uintptr_t)b) & 15 || x_row & 7)
    return decode_fail(GQK_ERR_SHAPE, "lora_add: x, a and b are 16-byte aligned, x's row stride a multiple of 8");
  if (!workspace || workspace_bytes < need || (uintptr_t)workspace & 255)
    return decode_fail(GQK_ERR_SHAPE, "lora_add: workspace %lld bytes < %lld (or not 256-byte aligned)", (long long)workspace_bytes,
                       (long long)need);
  g.y = y; g.x = x; g.a = a; g.b = b; g.out = out; g.y_row = y_row; g.x_row = x_row; g.out_row = out_row; g.K = K;
  g.ids = ids; g.wide_ids = ids_64; g.scales = scales; g.h = (float*)((char*)workspace + GQK_CTR_BYTES);
  g.M = M; g.slots = slots; g.parts = parts; g.rank = rank;
  const Cut c = cut_of(M, K, parts, rank);
  if (c.blocks > 65535) return decode_fail(GQK_ERR_SHAPE, "lora_add: %d rows", M);
  g.splits = c.splits; g.chunks = c.chunks;
  g.wide_y = !(((uintptr_t)y | (uintptr_t)out) & 15) && !((y_row | out_row) & 7);
  for (int p = 0; p + 1 < parts; ++p) g.wide_y &= g.ends[p] % 8 == 0;
  // columns of a workgroup of the second kernel: 512, fewer where the launch would have too few of them
  const int64_t groups = M <= kBlock ? std::min(M, 16) : c.blocks;
  g.columns = 512;
  while (g.columns > 128 && groups * (g.N / g.columns) < 512) g.columns /= 2;
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == GQK_DTYPE_BF16) {
    if (M <= kBlock) launch<bf16_t, 1>(g, c, st);
    else launch<bf16_t, 4>(g, c, st);
  } else {
    if (M <= kBlock) launch<f16_t, 1>(g, c, st);
    else launch<f16_t, 4>(g, c, st);
  }
  return decode_launched("lora_add");
}

}  // extern "C"
