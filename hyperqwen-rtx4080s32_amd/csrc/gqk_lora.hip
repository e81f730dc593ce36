// gqk_lora.hip - low-rank adapters of many requests beside a shared projection.
//
//   out[m, n] = y[m, n] + s_i sum_r B_i[n, r] h[m, p(n), r],   h[m, p, r] = sum_k A_i[p, r, k] x[m, k]
//
// with i = ids[m] the row's adapter (negative: out = y) and p(n) the part (q, k, v; gate, up) that
// column n belongs to.  h is kept in 32 bits in the workspace, after its counter region.
#include <algorithm>
#include <type_traits>
#include "gqk_decode.h"

namespace gqk {
namespace {

typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

constexpr int kParts = 8;
constexpr int kWaves = 4;
constexpr int kStage = 128;      // values of K that the first kernel takes at a time
constexpr int kList = 64;        // rows of a unit, at most
// A workgroup sorts out the adapters of a block of 64 Q rows, Q ids to a lane.  Batches of up to kSmall rows are one block (Q 1
// or 4), so that each adapter is read once for its rows wherever they are, in units of 16; longer ones (prompts, whose
// rows come in runs) go by 64 rows and units of up to 64.  Long batches whose rows come mixed are right but slow, as a block's units after the
// first wait for one another: to q, k and v of 5120 values, 32 adapters of rank 16, 256 rows 39 us, 257 158, 512 205, but 36 sorted by adapter.
constexpr int kSmall = 256;
constexpr int kRankTiles = 4;    // 16-rank tiles of a workgroup of the first kernel
constexpr int kRowColumns = 64 * kWaves;
constexpr int64_t kRowBytes = 1 << 18;   // of a part's A, that a workgroup of a row reads by itself
constexpr int kXcds = 8;         // workgroups go to them in turn
constexpr int kNone = -1, kBad = -2;

struct LoraArgs {
  const void *y, *x, *a, *b;
  void* out;
  int64_t y_row, x_row, out_row, K, N;
  const void* ids;
  const float* scales;
  float* h;                  // [splits][M][parts * rank]
  int M, slots, parts, rank, wide_ids;
  int splits, chunks, blocks;   // splits of K; chunks of 64 ranks; blocks of rows
  int finer;                 // parts of each split, for the units after a block's first
  int columns;               // of a workgroup of the second kernel
  int half_units;            // the second kernel takes long batches by 32 rows, not 64
  int wide_y;                // y and out are 16-byte aligned in every row
  int64_t ends[kParts];      // one past each part's last column
};

__device__ __forceinline__ v4f mfma(v4u a, v4u b, v4f c, bf16_t) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}
__device__ __forceinline__ v4f mfma(v4u a, v4u b, v4f c, f16_t) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

// x without what T has no bits for
__device__ __forceinline__ bf16_t toward_zero(float x, bf16_t) {
  return __builtin_bit_cast(bf16_t, (uint16_t)(__builtin_bit_cast(uint32_t, x) >> 16 | (x != x ? 0x40 : 0)));   // NaN stays
}
__device__ __forceinline__ f16_t toward_zero(float x, f16_t) { return (f16_t)__builtin_amdgcn_cvt_pkrtz(x, x)[0]; }
// what T still holds beside a value, and which adds nothing to it that shows (0 beside 0); fp16 values are below 2 here
__device__ __forceinline__ float least_beside(float x, bf16_t) { return fabsf(x) * 0x1p-20f; }
__device__ __forceinline__ float least_beside(float x, f16_t) { return fminf(fabsf(x) * 0x1p30f, 0x1p-24f); }

// Rows of one block that go with one adapter (or with none, kNone, or a bad id, kBad).
struct Unit {
  int adapter, count;
  const int* row;   // their numbers within the block
  bool lead;        // of the block's first row's adapter
};

// Unit u (of up to `most` rows) of a block of 64 Q rows: adapters in the order of their first row, each one's rows in
// order.  A lane holds the ids of Q rows; ballots find the rows that share one, whose numbers go to LDS in order, a list for
// each wave.  False: the block has fewer units.  All waves find the same.
template <int Q>
__device__ __forceinline__ bool find_unit(const LoraArgs& a, int64_t row0, int u, int most, int* lists, Unit& out) {
  const int lane = threadIdx.x & 63;
  int id[Q];
  uint64_t left[Q];
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    const int64_t m = row0 + q * 64 + lane;
    id[q] = kNone;
    if (m < a.M) {
      const int64_t i = index_at(a.ids, a.wide_ids, m);
      id[q] = i < 0 ? kNone : i >= a.slots ? kBad : (int)i;
    }
    left[q] = __ballot(m < a.M);
  }
#pragma unroll
  for (int f = 0; f < Q; ++f)   // the first row that is left lies in part f
    while (left[f]) {
      const int who = __builtin_amdgcn_readlane(id[f], __builtin_ctzll(left[f]));
      uint64_t same[Q];
      int count = 0;
#pragma unroll
      for (int q = f; q < Q; ++q) {
        same[q] = __ballot(id[q] == who) & left[q];
        count += __popcll(same[q]);
      }
      const int units = (count + most - 1) / most;
      if (u < units) {
        out.adapter = who;
        out.lead = who == __builtin_amdgcn_readlane(id[0], 0);
        out.count = min(count - u * most, most);
        int* mine = lists + (threadIdx.x >> 6) * kList;
        int before = -u * most;   // rows of the adapter in earlier parts, from the unit's first
#pragma unroll
        for (int q = f; q < Q; ++q) {
          const int place =
              before + __builtin_amdgcn_mbcnt_hi((uint32_t)(same[q] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)same[q], 0));
          if ((same[q] >> lane & 1) && place >= 0 && place < out.count) mine[place] = q * 64 + lane;
          before += __popcll(same[q]);
        }
        __builtin_amdgcn_wave_barrier();
        out.row = mine;
        return true;
      }
      u -= units;
#pragma unroll
      for (int q = f; q < Q; ++q) left[q] &= ~same[q];
    }
  return false;
}

// 16 bytes at a byte offset from a base that the whole wave shares; zeros past `bytes`
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void* p, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (int)min(bytes, (int64_t)0x7ffffff0), 0x00020000);
}
// An offset past every buffer, with what is added to it too: a row of x or A is below 2^23 bytes, columns below 2^12.
constexpr uint32_t kOutside = 0x80000000u;
constexpr int kOnce = 2;   // a load's cache policy: its lines leave the cache first
template <int POLICY = 0>
__device__ __forceinline__ v4u load16(__amdgpu_buffer_rsrc_t rs, uint32_t offset) {
  return __builtin_amdgcn_raw_buffer_load_b128(rs, offset, 0, POLICY);
}

// h = A x of one unit's rows, 64 ranks, one split of K.  Rows of x and of A are far apart, and a lane of a matrix operand
// holds 16 bytes of one: loaded like that nothing coalesces (62 L1 accesses a load counted).  So 256 bytes of each row at a
// time come in as rows, 16 lanes to one, go through LDS with their 16-byte pieces swapped by the row's number (16 rows'
// pieces of one k-step in different banks), and are read as operands: ranks as the instruction's rows, batch rows as its
// columns.  Loads run kDepth stages ahead in registers; two LDS buffers, one barrier a stage.  A wave takes one 16-row tile and all
// ranks (TT = 4), or all 16 rows and one 16-rank tile (TT = 1).  x goes by once and leaves the caches first, so that A, which every
// block of rows reads again, stays (4096 rows of 17408 values 82.4 -> 78.1 us, both launches).
//
// 4096 rows of 17408 values, rank 64: 35 us, 4.1 TB/s of x, near what a copy reaches (4.75).  Without any load it takes
// 21: LDS, the barriers and the issue of each stage, beside which the loads go on (loads 4 stages ahead cost 1.4 us more, two workgroups a CU 2.6, blocks of
// 128 rows 9; eight waves with half of each stage change nothing).  48 rows of 5120, 12 adapters of rank 32: 6.6 us, a launch, ids, one trip to memory,
// partial sums out.
template <typename T, int TT, int Q>
__global__ __launch_bounds__(64 * kWaves, 2) void lora_down_kernel(LoraArgs a) {
  constexpr int kDepth = TT == 1 ? 4 : 2;
  constexpr int kRows = 16 * TT, kAcc = TT == 1 ? 1 : kRankTiles;
  __shared__ __align__(16) char buf[2][(kRows + 16 * kRankTiles) * 256];
  __shared__ int lists[kWaves * kList];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
  const int chunk = blockIdx.x / a.splits;
  // Long batches: a block's first unit by splits, which give every CU a workgroup; the later ones (a second prompt begins inside of
  // the block) by parts of them, as each shares a CU with another and would otherwise end last (us for one to four
  // parts, 4096 rows of 17408 values of three adapters: 70.9, 68.5, 67.7, 66.5, both launches).
  const bool later = TT > 1 && blockIdx.z > 0;
  const int splits = later ? a.splits * a.finer : a.splits;
  const int split = later ? blockIdx.x % a.splits * a.finer + blockIdx.z - 1 : blockIdx.x % a.splits;
  constexpr int kBlock = 64 * Q;
  const int64_t row0 = (int64_t)blockIdx.y * kBlock;
  const int PR = a.parts * a.rank, rank0 = chunk * 16 * kRankTiles, tiles = min(kRankTiles, (PR - rank0 + 15) / 16);
  const int all = (int)((a.K + kStage - 1) / kStage);
  const int s0 = (int)((int64_t)all * split / splits), stages = (int)((int64_t)all * (split + 1) / splits) - s0;
  const int K = (int)a.K, row = threadIdx.x >> 4, piece = threadIdx.x & 15;
  const int step = TT == 1 ? gridDim.z : later ? 1 : 1 << 20;
  for (int u = TT == 1 ? blockIdx.z : later;; u += step) {
    Unit unit;
    if (!find_unit<Q>(a, row0, u, kRows, lists, unit)) return;
    if (unit.adapter < 0) continue;
    const int rows = (unit.count + 15) / 16;   // tiles of rows
    const __amdgpu_buffer_rsrc_t ra = buffer_of((const T*)a.a + ((int64_t)unit.adapter * PR + rank0) * a.K,
                                                (int64_t)min(16 * kRankTiles, PR - rank0) * a.K * 2);
    const __amdgpu_buffer_rsrc_t rx = buffer_of((const T*)a.x + row0 * a.x_row, (int64_t)kBlock * a.x_row * 2);
    uint32_t ao[kRankTiles], xo[TT];
    // ranks and rows that are not there are offsets past the buffers: zeros, no branch
#pragma unroll
    for (int t = 0; t < kRankTiles; ++t)
      ao[t] = t * 16 + row < PR - rank0 ? (t * 16 + row) * (uint32_t)K * 2 + piece * 16 : kOutside;
#pragma unroll
    for (int t = 0; t < TT; ++t)
      xo[t] = t * 16 + row < unit.count ? unit.row[t * 16 + row] * (uint32_t)a.x_row * 2 + piece * 16 : kOutside;
    v4u av[kDepth][kRankTiles], xv[kDepth][TT];
    auto load = [&](int d, int s) {
      const bool in = s < s0 + stages && s * kStage + piece * 8 < K;   // K may end inside the last stage
#pragma unroll
      for (int t = 0; t < TT; ++t) xv[d][t] = load16<kOnce>(rx, in ? xo[t] + s * (2 * kStage) : kOutside);
#pragma unroll
      for (int t = 0; t < kRankTiles; ++t) av[d][t] = load16(ra, in ? ao[t] + s * (2 * kStage) : kOutside);
    };
    v4f acc[kAcc];
#pragma unroll
    for (int r = 0; r < kAcc; ++r) acc[r] = v4f{0.f, 0.f, 0.f, 0.f};
    const bool busy = wave < (TT == 1 ? tiles : rows);
#pragma unroll
    for (int d = 0; d < kDepth; ++d) load(d, s0 + d);
    __syncthreads();   // the last unit's stages have been read
    auto stage = [&](int d, int s) {
      char* const to = buf[d & 1];   // kDepth is even
      char* const at = to + row * 256 + (piece ^ row) * 16;
#pragma unroll
      for (int t = 0; t < TT; ++t) *(v4u*)(at + t * 4096) = xv[d][t];
#pragma unroll
      for (int t = 0; t < kRankTiles; ++t) *(v4u*)(at + (TT + t) * 4096) = av[d][t];
      load(d, s + kDepth);
      __syncthreads();
      if (busy)
#pragma unroll
        for (int k = 0; k < kStage / 32; ++k) {
          const char* from = to + n * 256 + ((k * 4 + g) ^ n) * 16;
          const v4u xop = *(const v4u*)(from + (TT == 1 ? 0 : wave) * 4096);
          if constexpr (TT == 1) {
            acc[0] = mfma(*(const v4u*)(from + (TT + wave) * 4096), xop, acc[0], T{});
          } else {
            // of tiles that the chunk does not have too: zeros cost less than the copies that a branch around each
            // instruction takes (64 moves a product counted)
#pragma unroll
            for (int r = 0; r < kRankTiles; ++r) acc[r] = mfma(*(const v4u*)(from + (TT + r) * 4096), xop, acc[r], T{});
          }
        }
    };
    // whole rounds of kDepth without a branch: the loads of the next stages stay on their way through a wait
    int i = 0;
    for (; i + kDepth <= stages; i += kDepth)
#pragma unroll
      for (int d = 0; d < kDepth; ++d) stage(d, s0 + i + d);
#pragma unroll
    for (int d = 0; d < kDepth - 1; ++d)
      if (i + d < stages) stage(d, s0 + i + d);
    // lane (n, g) holds ranks 4 g .. + 3 of a tile for row n
    const int r_at = (TT == 1 ? 0 : wave) * 16 + n;
    if (busy && r_at < unit.count) {
      float* to = a.h + ((int64_t)split * a.M + row0 + unit.row[r_at]) * PR;
#pragma unroll
      for (int r = 0; r < kAcc; ++r) {
        const int rank = rank0 + (TT == 1 ? wave : r) * 16 + g * 4;
        if ((TT == 1 || r < tiles) && rank < PR) *(v4f*)(to + rank) = acc[r];
      }
    }
  }
}

// out = y + s B h of one unit's rows and `columns` columns of one part.  The ranks that h has in 32 bits go into the
// product as two values of T each, h = hi + lo, in one instruction: 16 ranks of hi and the same 16 of lo against B's 16
// ranks twice (rounding h to T alone would put up to 2^-8 of the update, for bf16, on top of the output's own rounding; the second
// half of the instruction would be idle).  hi is cut off, not rounded, so that both have h's sign, which costs lo a bit: what is left of h's
// error is 2^-16 for bf16, 2^-22 for fp16.  fp16 takes h over a power of two near its row's largest, to stay in range.
//
// A wave takes 64 columns at a time by itself: their rows of B come in as one run of memory (EACH 16-byte pieces of
// a column, 8 EACH ranks at a time) and turn into operands in the wave's LDS, and the update goes back through the same LDS to
// meet y in whole lines (128 bytes of a row to 8 lanes).  B and y are on their way while h is gathered.  What lies outside of
// the columns or ranks is an offset past the buffer: zeros, no branch.
//
// Blocks of rows are dealt to the XCDs in turn, with all of a block's workgroups, which gather the same partial sums of h, on
// one XCD and near in time (dealt by columns: 4096 rows of 17408 values 83.9 -> 81.9 us, 8192 of 5120 to three parts 93.0 -> 85.7,
// both launches).
//
// 4096 rows of 5120 columns, rank 64: 32 us for 84 MB of y and out; 18 us of it go by at memory's rate, the first 9 to 14 are the
// launch, the ids and h on their way.  48 rows of 34816 columns, 12 adapters of rank 32: 14.4 us, of which B, y and out (33 MB) take 7 at a copy's
// rate; before them go the ids, the ballots and the gather of h, and each wave then has four strips of 64 columns in turn, one on its way.
template <typename T, int TT, int Q, int EACH>
__global__ __launch_bounds__(64 * kWaves, 2) void lora_up_kernel(LoraArgs a) {
  constexpr bool kF16 = __is_same(T, f16_t);
  constexpr int kRows = 16 * TT;
  constexpr int kRowThreads = 64 * kWaves / kRows;  // threads that gather one row of h
  constexpr int kRanks = 8 * EACH;                  // of a pass over B
  constexpr int kBRow = 2 * kRanks + 16;            // LDS bytes of a column
  constexpr int kDRow = 68;                         // LDS floats of a row's update
  constexpr int kStrip = 64 * kBRow > 16 * kDRow * 4 ? 64 * kBRow : 16 * kDRow * 4;
  extern __shared__ __align__(16) char lds[];       // h: [hi, lo][rows][ranks + 8]
  __shared__ __align__(16) char strip[kWaves][kStrip];   // B, then the update, of a wave's columns
  __shared__ float factor[kRows];
  __shared__ int lists[kWaves * kList];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
  constexpr int kBlock = 64 * Q;
  const int near = min(a.blocks, kXcds);
  const int64_t row0 = ((int64_t)blockIdx.z * near + blockIdx.x % near) * kBlock;
  if (row0 >= a.M) return;
  const int rank = a.rank, PR = a.parts * rank, padded = (rank + kRanks - 1) / kRanks * kRanks, hrow = padded + 8;
  T* const hs = (T*)lds;
  char* const mine = strip[wave];
  // the part and its columns
  int part = 0, block = blockIdx.x / near;
  int64_t begin = 0;
  for (;;) {
    const int blocks = (int)((a.ends[part] - begin + a.columns - 1) / a.columns);
    if (block < blocks) break;
    block -= blocks;
    begin = a.ends[part++];
  }
  const int64_t c_begin = begin + (int64_t)block * a.columns;
  const int width = (int)min(a.ends[part] - c_begin, (int64_t)a.columns);
  const T* const ybase = (const T*)a.y + row0 * a.y_row + c_begin;
  T* const obase = (T*)a.out + row0 * a.out_row + c_begin;
  for (int u = blockIdx.y;; u += gridDim.y) {
    Unit unit;
    if (!find_unit<Q>(a, row0, u, kRows, lists, unit)) return;
    if (unit.adapter < 0) {   // rows as they are, or NaN
      if (unit.adapter == kNone && a.out == a.y) continue;
      for (int x = threadIdx.x; x < unit.count * width; x += 64 * kWaves) {
        const int r = x / width, c = x - r * width;
        const int64_t m = unit.row[r];
        obase[m * a.out_row + c] = unit.adapter == kNone ? ybase[m * a.y_row + c] : (T)__builtin_nanf("");
      }
      continue;
    }
    const int rows = (unit.count + 15) / 16, splits = unit.lead ? a.splits : a.splits * a.finer;
    const __amdgpu_buffer_rsrc_t rb = buffer_of((const T*)a.b + ((int64_t)unit.adapter * a.N + c_begin) * rank, (int64_t)width * rank * 2);
    const __amdgpu_buffer_rsrc_t ry = buffer_of(ybase, kBlock * a.y_row * 2), ro = buffer_of(obase, kBlock * a.out_row * 2);
    // lane's place in y: rows t * 16 + i * 8 + lane / 8, columns (lane % 8) * 8 .. + 7 of the wave's
    const int c8 = (lane & 7) * 8;
    uint32_t yo[TT][2], oo[TT][2];
#pragma unroll
    for (int t = 0; t < TT; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = t * 16 + i * 8 + (lane >> 3);
        const uint32_t at = unit.row[min(r, unit.count - 1)];
        yo[t][i] = r < unit.count ? (at * (uint32_t)a.y_row + c8) * 2 : kOutside;
        oo[t][i] = r < unit.count ? (at * (uint32_t)a.out_row + c8) * 2 : kOutside;
      }
    v4u bv[EACH], yv[TT][2];
    auto load_b = [&](int c0, int k0) {
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const int col = i * (64 / EACH) + lane / EACH, r = k0 + lane % EACH * 8;
        bv[i] = load16(rb, c0 + col < width && r < rank ? ((c0 + col) * (uint32_t)rank + r) * 2 : kOutside);
      }
    };
    auto load_y = [&](int c0) {
#pragma unroll
      for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) yv[t][i] = load16(ry, c0 + c8 < width ? yo[t][i] + c0 * 2 : kOutside);
    };
    constexpr int hop = 64 * kWaves;
    int c0 = wave * 64;
    load_b(c0, 0);
    if (a.wide_y) load_y(c0);
    {
      __syncthreads();   // the last unit's h has been read
      const int r = threadIdx.x / kRowThreads, c = threadIdx.x % kRowThreads;
      const int64_t m = row0 + unit.row[min(r, unit.count - 1)];
      const float* const from = a.h + m * PR + part * rank;
      const int octets = (padded / 8 + kRowThreads - 1) / kRowThreads;   // of this thread
      auto gather = [&](int at, int sp0, int by, float (&v)[8]) {   // splits sp0, sp0 + by, .. of eight ranks, added in order
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.f;
        if (at >= rank || r >= rows * 16) return;
        constexpr int kBatch = 4;
        for (int sp = sp0; sp < splits; sp += kBatch * by) {
          v4f lo[kBatch], hi[kBatch];
#pragma unroll
          for (int j = 0; j < kBatch; ++j) {
            const v4f* p = (const v4f*)(from + (int64_t)min(sp + j * by, splits - 1) * a.M * PR + at);
            lo[j] = p[0];
            hi[j] = p[1];
          }
#pragma unroll
          for (int j = 0; j < kBatch; ++j)
            if (sp + j * by < splits)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                v[e] += lo[j][e];
                v[4 + e] += hi[j][e];
              }
        }
      };
      float down = 1.f, up = 1.f, top = 0.f;
      auto seen = [&](const float (&v)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[e]) < __builtin_huge_valf() ? fabsf(v[e]) : 0.f);
      };
      auto fit = [&]() {   // a power of two near the row's largest finite one
        if constexpr (kF16) {
          for (int o = kRowThreads / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
          if (top > 0.f) {
            const int e = min(max(ilogbf(top), -100), 100);
            down = ldexpf(1.f, -e);
            up = ldexpf(1.f, e);
          }
        }
      };
      auto put = [&](int at, const float (&v)[8]) {
        if (at >= padded) return;
        T hi[8], lo[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = v[e] * down;
          hi[e] = toward_zero(x, T{});
          const float back = (float)hi[e];
          // of x's sign and not 0 where x is not: an infinite weight times both is one infinity, and so is a weight times infinite ones
          const float rest = fabsf(back) < __builtin_huge_valf() ? x - back : back;
          lo[e] = (T)copysignf(fmaxf(fabsf(rest), least_beside(back, T{})), x);
        }
        __builtin_memcpy(hs + r * hrow + at, hi, 16);
        __builtin_memcpy(hs + (kRows + r) * hrow + at, lo, 16);
      };
      auto at = [&](int q) { return (q * kRowThreads + c) * 8; };
      constexpr int kGroups = kRowThreads / EACH;   // threads of a row that share eight ranks' splits
      if (kGroups > 1 && padded == kRanks) {
        float v[8];
        gather(c % EACH * 8, c / EACH, kGroups, v);
#pragma unroll
        for (int o = EACH; o < kRowThreads; o *= 2)
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] += __shfl_xor(v[e], o);
        seen(v);
        fit();
        if (c < EACH) put(c * 8, v);
      } else if (octets <= 2) {
        float v[2][8];
        gather(at(0), 0, 1, v[0]);
        gather(at(1), 0, 1, v[1]);
        seen(v[0]);
        seen(v[1]);
        fit();
        put(at(0), v[0]);
        put(at(1), v[1]);
      } else {   // more than registers hold: fp16 gathers twice
        float v[8];
        if constexpr (kF16)
          for (int q = 0; q < octets; ++q) {
            gather(at(q), 0, 1, v);
            seen(v);
          }
        fit();
        for (int q = 0; q < octets; ++q) {
          gather(at(q), 0, 1, v);
          put(at(q), v);
        }
      }
      if (c == 0) factor[r] = (a.scales ? a.scales[unit.adapter] : 1.f) * up;
      __syncthreads();
    }
    for (; c0 < width; c0 += hop) {
      v4f acc[4][TT];
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int t = 0; t < TT; ++t) acc[c][t] = v4f{0.f, 0.f, 0.f, 0.f};
      for (int k0 = 0; k0 < padded; k0 += kRanks) {
#pragma unroll
        for (int i = 0; i < EACH; ++i)
          *(v4u*)(mine + (i * (64 / EACH) + lane / EACH) * kBRow + lane % EACH * 16) = bv[i];
        const bool next = k0 + kRanks >= padded;
        load_b(next ? c0 + hop : c0, next ? 0 : k0 + kRanks);
#pragma unroll
        for (int k = 0; k < EACH / 2; ++k) {
          v4u bop[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) bop[c] = *(const v4u*)(mine + (c * 16 + n) * kBRow + k * 32 + (g & 1) * 16);
#pragma unroll
          for (int t = 0; t < TT; ++t) {   // of tiles that the unit does not have too, as above
            const v4u hv = *(const v4u*)(hs + ((g >> 1) * kRows + t * 16 + n) * hrow + k0 + k * 16 + (g & 1) * 8);
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[c][t] = mfma(bop[c], hv, acc[c][t], T{});
          }
        }
      }
      // lane (n, g) holds columns 16 c + 4 g .. + 3 of row n; through LDS to 8 columns of rows lane / 8 and 8 + lane / 8
      float* const turn = (float*)mine;
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        const float f = factor[t * 16 + n];
#pragma unroll
        for (int c = 0; c < 4; ++c) *(v4f*)(turn + n * kDRow + c * 16 + g * 4) = acc[c][t] * f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float* d = turn + (i * 8 + (lane >> 3)) * kDRow + c8;
          if (a.wide_y) {
            const v4f d0 = *(const v4f*)d, d1 = *(const v4f*)(d + 4);
            T v[8];
            v4u w;
            __builtin_memcpy(v, &yv[t][i], 16);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = (T)((float)v[e] + (e < 4 ? d0[e & 3] : d1[e & 3]));
            __builtin_memcpy(&w, v, 16);
            __builtin_amdgcn_raw_buffer_store_b128(w, ro, c0 + c8 < width ? oo[t][i] + c0 * 2 : kOutside, 0, 0);
          } else {
            const int r = t * 16 + i * 8 + (lane >> 3);
            const int64_t m = unit.row[min(r, unit.count - 1)];
            const T* from = ybase + m * a.y_row + c0 + c8;
            T* to = obase + m * a.out_row + c0 + c8;
            if (r < unit.count && c0 + c8 + 8 <= width) {
              T v[8];
              __builtin_memcpy(v, from, 16);
#pragma unroll
              for (int e = 0; e < 8; ++e) v[e] = (T)((float)v[e] + d[e]);
              __builtin_memcpy(to, v, 16);
            } else if (r < unit.count) {
              for (int e = 0; c0 + c8 + e < width; ++e) to[e] = (T)((float)from[e] + d[e]);
            }
          }
        }
      }
      if (a.wide_y) load_y(c0 + hop);
    }
  }
}

// A row by itself, in one launch: a workgroup takes 256 columns of one part and works out h of that part.  A wave takes RW
// ranks: each lane 8 values of K at a time of every rank's row and of x (whole runs of 1 KiB), products and sums in 32
// bits, the 64 lanes' sums through LDS in fours.  Then a thread has a column: B's row of it, read at the start, times h in 32
// bits.  A is read by every workgroup of its part, from the caches, which is cheap while a launch leaves CUs idle anyway; it saves
// the second launch and its wait for the first.  One row of 5120 values to q, k and v, rank 16: 7.2 us (two launches 9.4), of which
// a launch takes 2 and 164 KiB of A through one CU 3.
template <typename T, int RW>
__global__ __launch_bounds__(64 * kWaves, 2) void lora_row_kernel(LoraArgs a) {
  constexpr int kDepth = 40 / RW;
  constexpr int kRun = 512;   // values of K that a wave takes at a time
  __shared__ __align__(16) float sums[RW * kWaves][4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t m = blockIdx.y, id = index_at(a.ids, a.wide_ids, m);
  const int rank = a.rank, K = (int)a.K;
  int part = 0, block = blockIdx.x;
  int64_t begin = 0;
  for (;;) {
    const int blocks = (int)((a.ends[part] - begin + kRowColumns - 1) / kRowColumns);
    if (block < blocks) break;
    block -= blocks;
    begin = a.ends[part++];
  }
  const int64_t c_begin = begin + (int64_t)block * kRowColumns;
  const int width = (int)min(a.ends[part] - c_begin, (int64_t)kRowColumns), n = threadIdx.x;
  T* const out = (T*)a.out + m * a.out_row + c_begin + n;
  const float old = n < width ? to_f(((const T*)a.y)[m * a.y_row + c_begin + n]) : 0.f;
  if (id < 0 || id >= a.slots) {   // the row as it is, or NaN
    if (n < width && !(id < 0 && a.out == a.y)) *out = id < 0 ? (T)old : (T)__builtin_nanf("");
    return;
  }
  const __amdgpu_buffer_rsrc_t rx = buffer_of((const T*)a.x + m * a.x_row, (int64_t)K * 2);
  const __amdgpu_buffer_rsrc_t ra = buffer_of((const T*)a.a + (id * a.parts + part) * rank * K, (int64_t)rank * K * 2);
  const __amdgpu_buffer_rsrc_t rb = buffer_of((const T*)a.b + (id * a.N + c_begin) * rank, (int64_t)width * rank * 2);
  uint32_t ao[RW];
#pragma unroll
  for (int r = 0; r < RW; ++r) ao[r] = wave * RW + r < rank ? ((wave * RW + r) * (uint32_t)K + lane * 8) * 2 : kOutside;
  v4u av[kDepth][RW], xv[kDepth];
  auto load = [&](int d, int j) {
    const bool in = j * kRun + lane * 8 < K;   // K may end inside the last run
    xv[d] = load16(rx, in ? (j * kRun + lane * 8) * 2 : kOutside);
#pragma unroll
    for (int r = 0; r < RW; ++r) av[d][r] = load16(ra, in ? ao[r] + j * (2 * kRun) : kOutside);
  };
#pragma unroll
  for (int d = 0; d < kDepth; ++d) load(d, d);
  v4u bv[RW / 2];
#pragma unroll
  for (int i = 0; i < RW / 2; ++i) bv[i] = load16(rb, n < width && i * 8 < rank ? (n * (uint32_t)rank + i * 8) * 2 : kOutside);
  const float scale = a.scales ? a.scales[id] : 1.f;
  float acc[RW];
#pragma unroll
  for (int r = 0; r < RW; ++r) acc[r] = 0.f;
  for (int j = 0; j * kRun < K; j += kDepth)   // past K: zeros
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      T xs[8];
      __builtin_memcpy(xs, &xv[d], 16);
#pragma unroll
      for (int r = 0; r < RW; ++r) {
        T as[8];
        __builtin_memcpy(as, &av[d][r], 16);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[r] += to_f(as[e]) * to_f(xs[e]);
      }
      load(d, j + d + kDepth);
    }
#pragma unroll
  for (int r = 0; r < RW; ++r) {
    const float s = lane_sum<16>(acc[r]);
    if ((lane & 15) == 0) sums[wave * RW + r][lane >> 4] = s;
  }
  __syncthreads();
  float update = 0.f;
#pragma unroll
  for (int i = 0; i < RW / 2; ++i) {
    T bs[8];
    __builtin_memcpy(bs, &bv[i], 16);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (i * 8 < rank) {
        const v4f h = *(const v4f*)sums[i * 8 + e];
        update += to_f(bs[e]) * ((h[0] + h[1]) + (h[2] + h[3]));
      }
  }
  if (n < width) *out = (T)(old + scale * update);
}

// How a call is cut.  K is split so that the first launch has about a workgroup a CU, each at least two stages
// (4096 rows of 17408 values: 512 workgroups 69.2 us, 256 66.6, both launches: the second reads fewer partial sums).
struct Cut { int splits, chunks, blocks, finer; };

Cut cut_of(int M, int64_t K, int parts, int rank) {
  Cut c;
  c.chunks = (parts * rank + 16 * kRankTiles - 1) / (16 * kRankTiles);
  c.blocks = M <= kSmall ? 1 : (M + 63) / 64;
  const int64_t wgs = (int64_t)c.chunks * (M <= kSmall ? std::min(M, 16) : c.blocks);
  const int64_t stages = (K + kStage - 1) / kStage;
  c.splits = (int)std::max<int64_t>(1, std::min<int64_t>({256 / wgs, stages / 2, 16}));
  // partial sums that the second kernel adds: at most 16
  c.finer = M <= kSmall || c.splits == 1 ? 1 : (int)std::max<int64_t>(1, std::min<int64_t>({4, 16 / c.splits, stages / (2 * c.splits)}));
  return c;
}

// The same with at most as many partial sums of h as the workspace holds; false: not even one.
bool fit(Cut& c, int64_t bytes, int64_t h_bytes) {
  const int64_t most = (bytes - GQK_CTR_BYTES) / h_bytes;
  if (bytes < GQK_CTR_BYTES || most < 1) return false;
  c.splits = (int)std::min<int64_t>(c.splits, most);
  c.finer = (int)std::min<int64_t>(c.finer, most / c.splits);
  return true;
}

// Workgroups of `columns` columns over all parts.
int64_t column_blocks(const LoraArgs& g, int columns) {
  int64_t blocks = 0, begin = 0;
  for (int p = 0; p < g.parts; ++p) {
    blocks += (g.ends[p] - begin + columns - 1) / columns;
    begin = g.ends[p];
  }
  return blocks;
}

template <typename T>
void launch_rows(const LoraArgs& g, hipStream_t st) {
  const dim3 grid((unsigned)column_blocks(g, kRowColumns), g.M);
  if (g.rank <= 16) lora_row_kernel<T, 4><<<grid, 64 * kWaves, 0, st>>>(g);
  else lora_row_kernel<T, 8><<<grid, 64 * kWaves, 0, st>>>(g);
}

template <typename T, int TT, int Q>
void launch(const LoraArgs& g, const Cut& c, hipStream_t st) {
  // units of a block: its adapters, none, bad ids, and what does not fit one unit; the kernels step on over more
  const int units = TT == 1 ? std::min(g.M, std::min(g.slots, kSmall) + 2 + g.M / 16) : 2;
  const int64_t blocks = column_blocks(g, g.columns);
  const int near = std::min(c.blocks, kXcds);
  // units last: workgroups go to the XCDs in turn, and with units before blocks the second ones, mostly empty, fell on the
  // same XCDs every time (4096 rows of 17408 values 78.1 -> 66.6 us, both launches)
  if (g.slots > 0) lora_down_kernel<T, TT, Q><<<dim3(c.splits * c.chunks, c.blocks, TT == 1 ? units : 1 + c.finer), 64 * kWaves, 0, st>>>(g);
  auto up = [&](auto each, auto tiles) {
    constexpr int kEach = decltype(each)::value, kRanks = 8 * kEach, UT = decltype(tiles)::value;
    const size_t lds = (size_t)16 * UT * 2 * ((g.rank + kRanks - 1) / kRanks * kRanks + 8) * sizeof(T);
    lora_up_kernel<T, UT, Q, kEach><<<dim3((unsigned)(blocks * near), TT == 1 ? units : 1 + 4 / UT, (c.blocks + near - 1) / near),
                                      64 * kWaves, lds, st>>>(g);
  };
  auto by_rank = [&](auto tiles) {
    if (g.rank <= 16) up(std::integral_constant<int, 2>{}, tiles);
    else if (g.rank <= 32) up(std::integral_constant<int, 4>{}, tiles);
    else up(std::integral_constant<int, 8>{}, tiles);
  };
  if constexpr (TT == 1) {
    by_rank(std::integral_constant<int, 1>{});
  } else {
    if (g.half_units) by_rank(std::integral_constant<int, 2>{});
    else by_rank(std::integral_constant<int, 4>{});
  }
}

}  // namespace
}  // namespace gqk

using namespace gqk;

extern "C" {

int64_t gqk_lora_workspace_bytes(int M, int64_t K, int parts, int rank) {
  if (M < 0 || K < 0 || parts < 1 || parts > kParts || rank < 8 || rank > 256 || rank % 8)
    return decode_fail(GQK_ERR_SHAPE, "lora: %d rows of %lld, %d parts (at most %d), rank %d (a multiple of 8 in 8..256)", M,
                       (long long)K, parts, kParts, rank);
  if (M == 0) return GQK_CTR_BYTES;
  const Cut c = cut_of(M, K, parts, rank);
  return GQK_CTR_BYTES + (int64_t)c.splits * c.finer * M * parts * rank * 4;
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
  Cut c = cut_of(M, K, parts, rank);
  const int64_t h_bytes = (int64_t)M * parts * rank * 4;
  if (!workspace || !fit(c, workspace_bytes, h_bytes) || (uintptr_t)workspace & 255)
    return decode_fail(GQK_ERR_SHAPE, "lora_add: workspace %lld bytes < %lld (or not 256-byte aligned)", (long long)workspace_bytes,
                       (long long)(GQK_CTR_BYTES + h_bytes));
  g.y = y; g.x = x; g.a = a; g.b = b; g.out = out; g.y_row = y_row; g.x_row = x_row; g.out_row = out_row; g.K = K;
  g.ids = ids; g.wide_ids = ids_64; g.scales = scales; g.h = (float*)((char*)workspace + GQK_CTR_BYTES);
  g.M = M; g.slots = slots; g.parts = parts; g.rank = rank;
  if (M > GQK_LORA_MAX_ROWS) return decode_fail(GQK_ERR_SHAPE, "lora_add: %d rows, more than %d", M, GQK_LORA_MAX_ROWS);
  g.splits = c.splits; g.finer = c.finer; g.chunks = c.chunks; g.blocks = c.blocks;
  // whole 16-byte pieces in every row, and rows that 32-bit offsets reach
  g.wide_y = !(((uintptr_t)y | (uintptr_t)out) & 15) && !((y_row | out_row) & 7) && y_row < (1 << 22) && out_row < (1 << 22);
  for (int p = 0; p < parts; ++p) g.wide_y &= g.ends[p] % 8 == 0;
  // columns of a workgroup of the second kernel, which gathers h once for them: 64 for each wave, more where the launch
  // has workgroups enough
  // Units of 32 rows where 64 would leave too few workgroups for the chip (us for 64 and 32: 5120 columns of rank 64, 512 rows
  // 27.8 and 22.6, 1024 rows 38.9 and 31.7, 4096 rows 78.2 and 79.9; 34816 columns, 300 rows 39.4 and 29.9, 512 rows 28.0 and 30.0).
  g.half_units = M > kSmall && c.blocks * (g.N / 256) <= 1024;
  const int64_t groups = M <= kSmall ? std::min(M, 16) : c.blocks;
  g.columns = 64 * kWaves;
  while (g.columns < 1024 && groups * (g.N / g.columns) > 256) g.columns *= 2;
  const hipStream_t st = (hipStream_t)stream;
  // Rows by themselves, in one launch, while a workgroup for each 256 columns of each row finds a CU of its own and A is short (us
  // of two launches and of this: 8 rows of 5120 to 5120 columns, rank 16, 160 workgroups 10.6 and 7.0; to q, k and v, 224 workgroups 10.9
  // and 8.7, 16 rows 12.5 and 12.1, 24 rows 12.8 and 17.6; one row of 8192 (256 KiB of A) 9.6 and 9.1, of 17408 10.6 and 13.4).
  // They read x while others write out, which must lie apart.
  const uintptr_t x0 = (uintptr_t)x, x1 = x0 + ((M - 1) * x_row + K) * 2, o0 = (uintptr_t)out, o1 = o0 + ((M - 1) * out_row + g.N) * 2;
  const bool apart = x1 <= o0 || o1 <= x0;
  if (apart && rank <= 32 && (int64_t)rank * K * 2 <= kRowBytes && M * column_blocks(g, kRowColumns) <= device_cus()) {
    if (dtype == GQK_DTYPE_BF16) launch_rows<bf16_t>(g, st);
    else launch_rows<f16_t>(g, st);
  } else if (dtype == GQK_DTYPE_BF16) {
    if (M <= 64) launch<bf16_t, 1, 1>(g, c, st);
    else if (M <= kSmall) launch<bf16_t, 1, kSmall / 64>(g, c, st);
    else launch<bf16_t, 4, 1>(g, c, st);
  } else {
    if (M <= 64) launch<f16_t, 1, 1>(g, c, st);
    else if (M <= kSmall) launch<f16_t, 1, kSmall / 64>(g, c, st);
    else launch<f16_t, 4, 1>(g, c, st);
  }
  return decode_launched("lora_add");
}

}  // extern "C"
