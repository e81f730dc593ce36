// gqk_tree.hip - attention of several new tokens per sequence over a paged key-value cache: the tokens of a drafted tree, of a
// chain, or of a chunk of a prompt.
//
//   o_i = sum_j exp(scale q_i.k_j - m_i) v_j / sum_j exp(scale q_i.k_j - m_i),   m_i = max_j scale q_i.k_j
//
// over the keys j that new token i sees: those before the new ones, and of the new ones' those that its mask names (without a
// mask: its own and the earlier ones'); with a window the last `window` of them.  No key: zeros.
#include <algorithm>
#include "gqk_attend.h"

namespace gqk {
namespace {

typedef float v16f __attribute__((ext_vector_type(16)));
typedef short v4s __attribute__((ext_vector_type(4)));

constexpr int kMostSplits = 256;
constexpr int kMostGroups = 0xffffff;   // workgroups of 256 threads in a launch, whose threads are counted in 32 bits
constexpr int kStep = 64;   // keys of a step

struct TreeArgs {
  const void* q;
  int64_t q_row, q_head;
  gqk_pages kv;
  const int32_t* table;
  int64_t table_row;
  const int32_t *lengths, *starts, *mask;
  void* out;
  int64_t out_row, out_head;
  float* lse;
  float* partials;
  int tokens, batch, q_heads, words, max_length, max_tokens, window;
  float scale;          // of a score, in units of log 2, not negative: the queries take its sign
  uint32_t sign;
  int chunk, splits;    // keys of a split, and the most splits of a row tile
  int slots;            // places for row tiles
  bool once;            // a sequence has one: nobody else reads its keys, which leave the caches first
  uint32_t magic;       // key / page_size = 2 key magic >> 32 >> shift, exact below 2^31
  int shift;
};

__device__ __forceinline__ v16f mfma32(v4u a, v4u b, v16f c, bf16_t) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}
__device__ __forceinline__ v16f mfma32(v4u a, v4u b, v16f c, f16_t) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

// the larger of lane and lane ^ 32
__device__ __forceinline__ float over_halves(float x) {
  float y = x;
  asm("" : "+v"(y));   // (of the same value twice the compiler keeps one half)
  const auto both = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, y), false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)both[0]), __builtin_bit_cast(float, (uint32_t)both[1]));
}

// 16 bytes of every lane from base + own to LDS, the lanes' side by side from `to` on, while the wave goes on: it waits for vmcnt itself before
// anyone reads them.  (Of the builtin the compiler waits for all of these loads before the next read of LDS, whichever it reads: 680 us for a chunk of
// 4096 tokens behind 4096 where this took 593.)
// ONCE: they leave the caches first (64 sequences of up to 4000 keys, 655 MB: 153 -> 146 us).
template <bool ONCE>
__device__ __forceinline__ void load_to_lds(uint64_t base, uint32_t own, uint32_t to) {
  const v4u from{(uint32_t)base, (uint32_t)(base >> 32) & 0xffffu, 0xFFFFFFFFu, 0x00020000u};
#ifdef __HIP_DEVICE_COMPILE__
  if constexpr (ONCE) asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen nt lds" ::"v"(own), "s"(from), "s"(to) : "memory", "m0");
  else asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(own), "s"(from), "s"(to) : "memory", "m0");
#endif
}

// The same from an address of each lane.
template <bool ONCE>
__device__ __forceinline__ void load_lanes_to_lds(const void* from, uint32_t to) {
#ifdef __HIP_DEVICE_COMPILE__
  if constexpr (ONCE) asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off nt" ::"v"(from), "s"(to) : "memory", "m0");
  else asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(to) : "memory", "m0");
#endif
}

// A row tile: `rows` (token, query head) pairs of one sequence and key head, tokens outermost, from row row0 of the sequence's on.
struct Tile {
  int b, start, tokens;   // the sequence, its first row of q, its new tokens
  int row0, rows;
  int context, length;    // keys before the new tokens', and with them
  int begin, end;         // the keys that its rows can see lie in [begin, end); begin is a multiple of 32
  bool bad;               // lengths or a mask that cannot be: NaN
};

// The tile at place `slot`.  Sequence b's tiles take the places from starts[b] group / ROWS + b on, which are enough for them, so that
// a launch knows its size without reading the lengths.  False: the place has none.
template <int ROWS> __device__ __forceinline__ bool tile_at(const TreeArgs& a, int slot, int lane, Tile& t) {
  const int group = a.q_heads / a.kv.heads;
  auto place = [&](int b) { return (int64_t)max(0, a.starts[b]) * group / ROWS + b; };
  int lo = 0, n = a.batch;   // the last sequence whose first place is not behind: 64 candidates a step
  while (n > 1) {
    const int stride = (n + 63) / 64, b = lo + lane * stride;
    const bool before = lane * stride < n && place(b) <= slot;
    const int at = max(0, __popcll(__ballot(before)) - 1);
    lo += at * stride;
    n = min(stride, n - at * stride);
  }
  t.b = lo;
  t.start = a.starts[lo];
  const int stop = a.starts[lo + 1];
  if (t.start < 0 || stop > a.tokens || stop <= t.start) return false;
  t.tokens = stop - t.start;
  const int64_t own = slot - place(lo), all = (int64_t)t.tokens * group;
  if (own < 0 || own * ROWS >= all) return false;
  t.row0 = (int)(own * ROWS);
  t.rows = (int)min((int64_t)ROWS, all - t.row0);
  const int len = a.lengths[lo];
  t.bad = len < t.tokens || len > a.max_length || t.tokens > a.max_tokens || (a.mask && (int64_t)a.words * 32 < t.tokens);
  t.length = t.bad ? t.tokens : len;
  t.context = t.length - t.tokens;
  const int first = t.row0 / group, last = (t.row0 + t.rows - 1) / group;
  const int sees = a.mask ? t.context : t.context + first + 1;   // the least keys of a row (a mask may name none of the new ones)
  t.begin = (a.window > 0 ? max(0, sees - a.window) : 0) & ~31;
  t.end = t.bad ? 0 : a.mask ? t.length : t.context + last + 1;
  if (t.bad) t.begin = 0;
  return true;
}

// The first key that a row sees under the window, and its mask.
struct Row {
  int token, first;
  const int32_t* mask;
};
__device__ __forceinline__ Row row_of(const TreeArgs& a, const Tile& t, int row) {
  Row r{row / (a.q_heads / a.kv.heads), 0, nullptr};
  if (a.mask) r.mask = a.mask + (int64_t)(t.start + r.token) * a.words;
  if (a.window > 0 && !t.bad) {
    if (!a.mask) {
      r.first = max(0, t.context + r.token + 1 - a.window);
    } else {   // of the new tokens' keys that it sees, the last ones first
      int left = a.window;
      for (int w = (t.tokens - 1) >> 5; w >= 0 && left > 0; --w) {
        uint32_t bits = r.mask[w];
        if (w == (t.tokens - 1) >> 5 && t.tokens & 31) bits &= (1u << (t.tokens & 31)) - 1;
        const int c = __popc(bits);
        if (c < left) { left -= c; continue; }
        for (int over = c - left; over > 0; --over) bits &= bits - 1;   // the lowest of them are too far back
        r.first = t.context + w * 32 + __ffs(bits) - 1;
        left = 0;
      }
      if (left > 0) r.first = t.context > 0 || left < a.window ? max(0, t.context - left) : t.length - 1;   // (the last: it sees none at all)
    }
  }
  return r;
}

// Which of the keys base .. base + 31 a row sees.
__device__ __forceinline__ uint32_t seen_of(const TreeArgs& a, const Tile& t, const Row& r, int base) {
  auto below = [](int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1; };   // the first n
  uint32_t seen = below((a.mask ? t.length : t.context + r.token + 1) - base);
  if (a.mask && base + 32 > t.context) {
    const int at = base - t.context;
    uint32_t bits;
    if (at >= 0) {
      const int w = at >> 5, s = at & 31;
      bits = w < a.words ? (uint32_t)r.mask[w] >> s : 0u;
      if (s && w + 1 < a.words) bits |= (uint32_t)r.mask[w + 1] << (32 - s);
    } else {
      bits = (uint32_t)r.mask[0] << -at | below(-at);
    }
    seen &= bits;
  }
  return seen & ~below(r.first - base);
}

// Where 16-byte chunk c of a key lies in its row of LDS: a wave that reads one chunk of 32 keys, or two 16-dim runs of eight, finds them in
// different banks.
template <int DP> __device__ __forceinline__ int place_of(int key, int c) {
  return DP == 64 ? c ^ ((key >> 1 & 1) << 2 | (key >> 2 & 3)) : c ^ ((key & 3) << 2 | (key >> 2 & 3));
}

// A workgroup takes one row tile of one key head and one split of its keys.  Its four waves are 4 / KW groups of 32 rows by KW
// groups of 32 or 64 keys of each step; keys and values of a step of KT keys go through LDS, the next step's on their way
// meanwhile, so that a page's row is read once by the workgroup, in whole lines, whatever its type and layout.
//
// Both products run on 32 x 32 x 16 matrix instructions with the keys (then the dims) as the rows and the tile's rows as the
// columns: S^T = K Q^T, lane l has row l % 32's scores of keys 8 (i / 4) + 4 (l / 32) + i % 4 of 32, and as O^T += V^T P^T may take the
// keys in any order, these are its operand as they are; V's operand comes transposed out of LDS in the same order.  Only the
// maximum crosses lanes.
//
// Scores, statistics and sums are in 32 bits; the weights become T for the second product, as in the attention of single tokens, because the matrix
// instructions of 32-bit operands run at a sixteenth of the rate (error against 64 bits 2.1e-3 in bf16 and 2.5e-4 in fp16, of which the result's own rounding
// is 1.7e-3 and 2.1e-4).
//
// What bounds it (bf16, 40 heads over 8 of 128 dims).  Chunks of prompts, the matrix instructions and what the vector units do between them: 4096
// tokens behind 4096, 516 GFLOP, 524 to 552 us from one card to another, 930 to 980 TFLOP/s.  Trees, memory: 32 of up to 16 tokens behind up to 4000, 337 MB, 84 us, 4.0 TB/s, where loads
// without the products take as long (partial sums of two splits move another 43 MB); 64 of 4, 655 MB, 136 us, 4.8 TB/s.  8-bit pages are widened on
// the way to LDS, in every workgroup that reads them: four trees of up to 61 tokens behind 32768, 197 MB, 93 GFLOP, 158 us.  Workgroups of eight
// waves and 256 rows were slower (581 us for the chunk, when this took 540), and so were three steps on their way (584), steps of 32 keys
// (640), halves of steps with a wait each (no faster for trees, 573 for the chunk), and the next step's scores
// among a step's exponentials (540 where this took 517).  Shares of equal steps, dealt over the tiles from
// what the lengths are, gave 172 us for the four trees and 107 for the windows of cut_of, and 16 for the smallest call in place of 11.
//
// RUNS: pages hold whole runs of the keys of one round of loads: a run's page is one number for the whole workgroup, and a chunk's place
// in it the thread's own, so that nothing is computed per chunk (32 trees in pages of 16 tokens 84 us, of 7 137).  FULL: heads have all DP dims; else
// those behind the last stay the zeros that LDS begins with (80 dims 85 us, addressed chunk by chunk 132).  16-bit pages go to LDS directly
// (by way of registers: 197 and, of 7 tokens, 232).
template <typename T, typename C, int DP, int KW, bool RUNS, bool FULL>
__global__ __launch_bounds__(256, DP == 256 ? 1 : 2) void tree_kernel(TreeArgs a) {
  constexpr bool F8 = sizeof(C) == 1, DIRECT = !F8;
  constexpr int KT = kStep;
  constexpr int RW = 4 / KW, ROWS = 32 * RW;
  constexpr int NM = DP / 16, ND = DP / 32, CPK = DP / 8;
  constexpr int RL = 16, NR = KT / RL / 4;       // keys of a run, runs of a wave's share of a step
  constexpr int NI = RL * CPK / 64, KPI = 64 / CPK;   // loads of a run, keys of a load
  constexpr int KB = KT / 32 / KW;               // 32-key blocks of a wave
  constexpr int TB = KT * DP * 2;                // bytes of a step's keys, or values
  constexpr int RS = DP + 4;                     // row stride of the sums
  constexpr int LDS = std::max(4 * TB, 4 * 32 * RS * 4);
  __shared__ __align__(1024) char lds[LDS];      // (addresses are made by xor: rows begin at multiples of their size)
  __shared__ float stat[4 * 32][2];
  __shared__ uint32_t odd[3][KT / 32];           // of three steps: keys with a value that is not finite
  __shared__ int wrong, lows[4];
  typedef __attribute__((address_space(3))) char* Lds;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kvh = blockIdx.x % a.kv.heads, slot = a.slots - 1 - (int)(blockIdx.x / a.kv.heads), split = blockIdx.y;
  Tile t;
  if (!tile_at<ROWS>(a, slot, lane, t)) return;
  const int ns = splits_of(t.begin, t.end, a.chunk);
  if (split >= ns) return;
  const int group = a.q_heads / a.kv.heads, D = FULL ? DP : a.kv.dim;
  const int k_begin = t.begin + split * a.chunk, k_end = t.end > k_begin ? k_begin + min(a.chunk, t.end - k_begin) : k_begin;
  const int steps = (k_end - k_begin + KT - 1) / KT;
  const float inf = __builtin_huge_valf(), nan = __builtin_nanf("");
  const int kw = wave % KW, rw = wave / KW, n = lane & 31, hh = lane >> 5;
  const int own = rw * 32 + n;                   // of the tile's rows
  const bool live = own < t.rows;
  const Row row = row_of(a, t, t.row0 + (live ? own : 0));
  // The first key that any of the rows sees: what lies behind all windows is not looked up, as a server may have given up its pages.
  int low = a.window > 0 ? max(0, t.context + t.row0 / group + 1 - a.window) : 0;
  if (a.mask && a.window > 0) {
    low = row.first;
    for (int o = 16; o > 0; o >>= 1) low = min(low, __shfl_xor(low, o));
    if (lane == 0) lows[wave] = low;
  }
  // scores of zero are those of queries of zero: a key that is not seen has -inf, which no factor may make NaN
  const float factor = a.scale * (a.kv.k_scale ? fabsf(a.kv.k_scale[kvh]) : 1.f), scale = factor == 0.f ? 1.f : factor;
  const uint32_t sign = a.sign ^ (a.kv.k_scale && a.kv.k_scale[kvh] < 0.f ? 0x80008000u : 0u);

  v4u q[NM];
  {
    const int head = kvh * group + (t.row0 + (live ? own : 0)) % group;
    const T* qp = (const T*)a.q + (int64_t)(t.start + row.token) * a.q_row + head * a.q_head;
#pragma unroll
    for (int i = 0; i < NM; ++i) {
      const int d = i * 16 + hh * 8;
      q[i] = d < D ? *(const v4u*)(qp + d) : v4u{0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < 4; ++w) q[i][w] = live && d < D && factor != 0.f ? q[i][w] ^ sign : 0u;
    }
  }

  v16f acc[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) acc[d] = v16f{};
  float m = -inf, l = 0.f;
  uint32_t top_page = 0;
  if (tid < KT / 32) odd[0][tid] = odd[1][tid] = odd[2][tid] = 0;
  if (tid == 0) wrong = 0;
  if (DIRECT && !FULL && D < DP)   // dims that no load brings
    for (int x = tid * 16; x < 4 * TB; x += 256 * 16) *(v4u*)(lds + x) = v4u{0, 0, 0, 0};
  __syncthreads();
  if (a.mask && a.window > 0) low = min(min(lows[0], lows[1]), min(lows[2], lows[3]));
  low = __builtin_amdgcn_readfirstlane(low);

  // A step's keys come as runs of sixteen, NR to a wave; a load brings KPI keys of one, each lane 16 bytes of LDS: at place lane % CPK of
  // its key's row, where one chunk of dims lies (place_of is its own inverse).
  const int ps = a.kv.page_size, key0 = wave * NR * RL;
  auto key_of = [&](int r, int j) { return key0 + r * RL + j * KPI + lane / CPK; };   // of the step
  auto dims_of = [&](int j) { return place_of<DP>(j * KPI + lane / CPK, lane % CPK) * 8; };
  auto at_of = [&](int r, int j) { return (key0 + r * RL) * DP * 2 + j * 1024; };     // of lane 0's bytes
  typedef const __attribute__((address_space(4))) int32_t* Uniform;
  const int32_t* table = a.table + (int64_t)t.b * a.table_row;
  const C* const kb = (const C*)a.kv.k + kvh * a.kv.k_head;
  const C* const vb = (const C*)a.kv.v + kvh * a.kv.v_head;
  auto page_of = [&](int key) { return (int)(__umulhi(2u * (uint32_t)key, a.magic) >> a.shift); };
  struct Raw { uint32_t w[F8 ? 2 : 4]; };
  constexpr int HELD = DIRECT ? 1 : NR * NI;
  Raw kr[HELD], vr[HELD];
  const uint32_t lds_at = (uint32_t)(uintptr_t)(Lds)lds;
  constexpr int PAGES = RUNS ? NR : NR * NI;
  int page[PAGES], place[PAGES];   // of the step that is fetched next: pages, and places in them
  const int last = max(0, k_end - 1);
  auto look = [&](int base) {      // a key behind the last is read as the last one's page, one before the first as the first one's, and not used
#pragma unroll
    for (int i = 0; i < PAGES; ++i) {
      const int key = max(min(base + (RUNS ? key0 + i * RL : key_of(i / NI, i % NI)), RUNS ? last & ~(RL - 1) : last), RUNS ? low & ~(RL - 1) : low);
      const int at = page_of(key);
      if constexpr (RUNS) page[i] = ((Uniform)table)[at];
      else page[i] = table[at];
      place[i] = key - at * ps;
    }
  };
  // The chunks of a step's keys and values: on their way to LDS (DIRECT) or to registers.
  const uint32_t k_page = (uint32_t)a.kv.k_page * sizeof(C), v_page = (uint32_t)a.kv.v_page * sizeof(C);
  const uint32_t k_tok = (uint32_t)a.kv.k_token * sizeof(C), v_tok = (uint32_t)a.kv.v_token * sizeof(C);
  uint32_t k_own[RUNS ? NI : 1], v_own[RUNS ? NI : 1];   // a lane's bytes of a run, from its first key's
  if constexpr (RUNS)
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      k_own[j] = (j * KPI + lane / CPK) * k_tok + dims_of(j) * (uint32_t)sizeof(C);
      v_own[j] = (j * KPI + lane / CPK) * v_tok + dims_of(j) * (uint32_t)sizeof(C);
    }
  auto fetch = [&](int buf) {
#pragma unroll
    for (int i = 0; i < PAGES; ++i) {
      const bool out = (uint32_t)page[i] >= (uint32_t)a.kv.pages;   // a page outside of the cache is not read
      top_page = max(top_page, (uint32_t)page[i]);
      const uint32_t p = out ? 0 : page[i];
      if constexpr (RUNS) {
        const char* const kp = (const char*)kb + ((uint64_t)p * k_page + (uint32_t)place[i] * k_tok);
        const char* const vp = (const char*)vb + ((uint64_t)p * v_page + (uint32_t)place[i] * v_tok);
        auto load = [&]<bool ONCE>() {
#pragma unroll
          for (int j = 0; j < NI; ++j) {
            const uint32_t to = lds_at + buf * 2 * TB + at_of(i, j);
            if (!FULL && dims_of(j) >= D) continue;   // (a lane that does not load does not write to LDS)
            load_to_lds<ONCE>((uint64_t)kp, k_own[j], to);
            load_to_lds<ONCE>((uint64_t)vp, v_own[j], to + TB);
          }
        };
        if constexpr (DIRECT) {
          if (a.once) load.template operator()<true>();
          else load.template operator()<false>();
        } else {
#pragma unroll
          for (int j = 0; j < NI; ++j) {
            kr[i * NI + j] = vr[i * NI + j] = Raw{};
            if (!FULL && dims_of(j) >= D) continue;
            __builtin_memcpy(&kr[i * NI + j], __builtin_assume_aligned(kp + k_own[j], sizeof(Raw)), sizeof(Raw));
            __builtin_memcpy(&vr[i * NI + j], __builtin_assume_aligned(vp + v_own[j], sizeof(Raw)), sizeof(Raw));
          }
        }
      } else {
        Raw k{}, v{};
        const int d = dims_of(i % NI);
        if (d < D) {
          const C* const kp = kb + (int64_t)p * a.kv.k_page + (int64_t)place[i] * a.kv.k_token + d;
          const C* const vp = vb + (int64_t)p * a.kv.v_page + (int64_t)place[i] * a.kv.v_token + d;
          if constexpr (DIRECT) {
            const uint32_t to = lds_at + buf * 2 * TB + at_of(i / NI, i % NI);
            if (a.once) {
              load_lanes_to_lds<true>(kp, to);
              load_lanes_to_lds<true>(vp, to + TB);
            } else {
              load_lanes_to_lds<false>(kp, to);
              load_lanes_to_lds<false>(vp, to + TB);
            }
          } else {
            __builtin_memcpy(&k, __builtin_assume_aligned(kp, sizeof(Raw)), sizeof(Raw));
            __builtin_memcpy(&v, __builtin_assume_aligned(vp, sizeof(Raw)), sizeof(Raw));
          }
        }
        if constexpr (!DIRECT) {
          kr[i] = k;
          vr[i] = v;
        }
      }
    }
  };
  auto wide = [&](const Raw& r) {
    if constexpr (F8) return widen8<T>(r.w[0], r.w[1]);
    else return v4u{r.w[0], r.w[1], r.w[2], r.w[3]};
  };
  // rows of the tile that see all keys below `whole`, and none that the window takes
  const int whole = a.mask ? t.context : t.context + t.row0 / group + 1;
  const int open = a.window > 0 ? t.end - a.window : 0;   // from here on the window takes nothing (a row sees at most the keys up to end)
  auto mixed = [&](int base, int keys) { return base + keys > whole || base < open; };
  // A weight of 0 does not silence a value that is not finite: where some rows see a key and some do not, such values are put aside.
  auto put_aside = [&](v4u& v, int key, int third) {
    constexpr uint32_t e = __is_same(T, f16_t) ? 0x7c00u : 0x7f80u;
    bool any = false;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const bool lo = (v[w] & e) == e, hi = (v[w] >> 16 & e) == e;
      any |= lo | hi;
      v[w] &= (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
    }
    if (any) atomicOr(&odd[third][key >> 5], 1u << (key & 31));
    return any;
  };
  auto stage = [&](int base, int buf, int third) {
    const bool some = mixed(base, KT);
    if (DIRECT && !some) return;   // what has come stays as it is (the last key is in none but a mixed step)
#pragma unroll
    for (int i = 0; i < NR * NI; ++i) {
      const int key = key_of(i / NI, i % NI);
      v4u* const to = (v4u*)(lds + buf * 2 * TB + at_of(i / NI, i % NI) + lane * 16);
      v4u *const k = to, *const v = (v4u*)((char*)to + TB);
      v4u x = v4u{0, 0, 0, 0};
      if constexpr (DIRECT) {
        if (base + key >= k_end) *k = *v = x;   // behind the last key: whatever there was
        else if (x = *v, put_aside(x, key, third)) *v = x;
      } else {
        if (some) {
          const bool there = base + key < k_end;
          *k = there ? wide(kr[i]) : x;
          x = there ? wide(vr[i]) : x;
          put_aside(x, key, third);
          *v = x;
        } else {
          *k = wide(kr[i]);
          *v = wide(vr[i]);
        }
      }
    }
  };

  // A wave's operands in LDS: of keys, chunk 2 i + hh of key n is at (n's row, chunk hh) ^ 32 i; of values a lane reads four dims of key r4 of
  // a group of four, and has four keys of dim lane % 16 after the transposition: chunk 4 d + .. of the row at ^ 64 d, the group eight keys on at ^ 32.
  const int r4 = (lane & 15) >> 2;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(Lds)lds + kw * KB * 32 * DP * 2;
  const uint32_t k_at = lds0 + n * DP * 2 + place_of<DP>(n, hh) * 16;
  const uint32_t v_at = lds0 + TB + (4 * hh + r4) * DP * 2 + place_of<DP>(4 * hh + r4, (lane >> 4 & 1) * 2 + ((lane & 3) >> 1)) * 16 + (lane & 1) * 8;

  if (steps > 0) {
    look(k_begin);
    fetch(0);
    if constexpr (!DIRECT) stage(k_begin, 0, 0);
    look(k_begin + KT);
  }
  if constexpr (!DIRECT) __syncthreads();
  int third = 0;
  for (int s = 0; s < steps; ++s) {
    const int base = k_begin + s * KT, buf = s & 1, third_next = third == 2 ? 0 : third + 1, third_free = third_next == 2 ? 0 : third_next + 1;
    const bool more = s + 1 < steps;
    if constexpr (DIRECT) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      stage(base, buf, third);
      __syncthreads();
    }
    if (more) {
      fetch(buf ^ 1);
      look(base + 2 * KT);
    }
    if (mixed(base - KT, KT) && tid < KT / 32) odd[third_free][tid] = 0;   // the last step's: written again two steps from now at the earliest
    const int first = base + kw * KB * 32;
    if (first < k_end) {
      uint32_t ka = k_at + buf * 2 * TB, va = v_at + buf * 2 * TB;
      asm volatile("" : "+v"(ka), "+v"(va));   // their variants are made anew in each step, not kept
      typedef const __attribute__((address_space(3))) char* From;
      auto keys = [&](int i, int b) { return *(const __attribute__((address_space(3))) v4u*)((From)(uintptr_t)(ka ^ (i * 32)) + b * 32 * DP * 2); };
      auto values = [&](int b, int x) {   // of dims 32 (x / 2) on and sixteen keys
        typedef __attribute__((address_space(3))) v4s* Four;
        const uint32_t at = va ^ (x >> 1) * 64;
        const int rows = (b * 32 + 16 * (x & 1)) * DP * 2;
        const v2u lo = __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Four)((From)(uintptr_t)at + rows)));
        const v2u hi = __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Four)((From)(uintptr_t)(at ^ 32) + rows + 8 * DP * 2)));
        return v4u{lo.x, lo.y, hi.x, hi.y};
      };
      v16f sc[KB];
#pragma unroll
      for (int b = 0; b < KB; ++b) sc[b] = v16f{};
#pragma unroll
      for (int i = 0; i < NM; ++i)
#pragma unroll
        for (int b = 0; b < KB; ++b) sc[b] = mfma32(keys(i, b), q[i], sc[b], T{});
      v4u vf[2 * ND];
#pragma unroll
      for (int x = 0; x < 2 * ND; ++x) vf[x] = values(0, x);
      // six reads ahead of the products (of the compiler two: 592 -> 577 us for a chunk of 4096 tokens behind 4096)
      __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);
#pragma unroll
      for (int i = 0; i < NM * KB - 6; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
#pragma unroll
      for (int i = 0; i < 6; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
      }
      if (mixed(first, 32 * KB)) {
#pragma unroll
        for (int b = 0; b < KB; ++b) {
          const uint32_t mine = seen_of(a, t, row, first + b * 32) >> (4 * hh);
#pragma unroll
          for (int i = 0; i < 16; ++i) sc[b][i] = mine >> ((i & 3) + 8 * (i >> 2)) & 1 ? sc[b][i] : -inf;
        }
      }
      // (a median with infinity is the larger; of fmaxf the compiler makes two instructions for a product's result)
      float top = -inf;
#pragma unroll
      for (int b = 0; b < KB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = __builtin_amdgcn_fmed3f(top, sc[b][i], inf);
      top = over_halves(top) * scale;
      const float mn = fmaxf(m, top), mb = base_of(mn);
      if (__any(mn != m)) {   // rarely, once the first keys were seen
        const float f = __builtin_amdgcn_exp2f(m - mb);
        l *= f;
#pragma unroll
        for (int d = 0; d < ND; ++d) acc[d] *= f;
      }
      m = mn;
      if (mixed(base, KT)) {   // (the step, as where they were put aside: this wave's keys may be seen by all rows)
        // the values that were put aside reach the rows that see them: as they are, whatever their weight
#pragma unroll 1
        for (int b = 0; b < KB; ++b)
#pragma unroll 1
          for (uint32_t rest = __builtin_amdgcn_readfirstlane(odd[third][kw * KB + b]); rest; rest &= rest - 1) {
            const int bit = __ffs(rest) - 1, key = first + b * 32 + bit, at = page_of(key);
            const int from_page = table[at];
            if ((uint32_t)from_page >= (uint32_t)a.kv.pages) continue;   // what was put aside is another page's, and the result NaN anyway
            const bool sees = seen_of(a, t, row, first + b * 32) >> bit & 1;
            const C* from = vb + from_page * a.kv.v_page + (int64_t)(key - at * ps) * a.kv.v_token;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const int dim = d * 32 + 8 * j + 4 * hh;
                if (!sees || dim >= D) continue;
                C x[4];
                __builtin_memcpy(x, __builtin_assume_aligned(from + dim, 4 * sizeof(C)), 4 * sizeof(C));
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float y = to_f(x[e]);
                  acc[d][4 * j + e] += y - y == 0.f ? 0.f : y;
                }
              }
          }
      }
      const float pb = kLift<T> - mb;
#pragma unroll
      for (int b = 0; b < KB; ++b) {
        v4u pt[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float p[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            p[i] = __builtin_amdgcn_exp2f(sc[b][8 * k + i] * scale + pb);
            l += p[i];
          }
          pt[k] = v4u{pack2<T>(p[0], p[1]), pack2<T>(p[2], p[3]), pack2<T>(p[4], p[5]), pack2<T>(p[6], p[7])};
        }
#pragma unroll
        for (int y = 0; y < 2 * ND; ++y) {   // all dims of sixteen keys, then of the others: no product waits for the one before
          const int x = (y % ND) * 2 + y / ND;
          acc[x >> 1] = mfma32(vf[x], pt[x & 1], acc[x >> 1], T{});
          if (b + 1 < KB) vf[x] = values(b + 1, x);
        }
      }
    }
    if constexpr (!DIRECT) {
      if (more) stage(base + KT, buf ^ 1, third_next);
      __syncthreads();
    }
    third = third_next;
  }
  if constexpr (DIRECT) __syncthreads();
  l += __shfl_xor(l, 32);
  if (top_page >= (uint32_t)a.kv.pages) wrong = 1;

  // the waves' sums, joined: lane (n, hh) holds dims 32 d + 8 j + 4 hh + e of row n in acc[d][4 j + e]
  float* const red = (float*)lds;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *(v4f*)(red + (wave * 32 + n) * RS + d * 32 + j * 8 + hh * 4) = v4f{acc[d][4 * j], acc[d][4 * j + 1], acc[d][4 * j + 2], acc[d][4 * j + 3]};
  if (hh == 0) {
    stat[wave * 32 + n][0] = m;
    stat[wave * 32 + n][1] = l;
  }
  __syncthreads();
  const bool lost = wrong || t.bad;
  const float v_scale = a.kv.v_scale ? a.kv.v_scale[kvh] : 1.f;
  const int quads = D / 4;
  float* const part = a.partials + ((int64_t)slot * a.kv.heads + kvh) * a.splits * ROWS * (D + 4);   // [splits][ROWS][D], then [splits][ROWS][2]
  for (int x = tid; x < t.rows * quads; x += 256) {
    const int r = x / quads, d = (x - r * quads) * 4, w0 = (r >> 5) * KW;
    float M = -inf, L = 0.f;
#pragma unroll
    for (int k = 0; k < KW; ++k) M = fmaxf(M, stat[(w0 + k) * 32 + (r & 31)][0]);
    const float Mb = base_of(M);
    v4f o{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < KW; ++k) {
      const int w = (w0 + k) * 32 + (r & 31);
      const float f = __builtin_amdgcn_exp2f(stat[w][0] - Mb);
      L += stat[w][1] * f;
      o += *(const v4f*)(red + w * RS + d) * f;
    }
    if (lost) L = nan;
    if (ns > 1) {
      *(v4f*)(part + ((int64_t)split * ROWS + r) * D + d) = o;
      if (d == 0) {
        float* st = part + (int64_t)a.splits * ROWS * D + ((int64_t)split * ROWS + r) * 2;
        st[0] = M;
        st[1] = L;
      }
      continue;
    }
    const int token = (t.row0 + r) / group, head = kvh * group + (t.row0 + r) % group;
    const float f = L == 0.f ? 0.f : v_scale / L;
    T* to = (T*)a.out + (int64_t)(t.start + token) * a.out_row + head * a.out_head + d;
    *(v2u*)to = v2u{pack2<T>(o[0] * f, o[1] * f), pack2<T>(o[2] * f, o[3] * f)};
    if (a.lse && d == 0)
      a.lse[(int64_t)(t.start + token) * a.q_heads + head] = L == 0.f ? -inf : (M - kLift<T> + __builtin_amdgcn_logf(L)) * kLn2;
  }
}

// The join of a row tile's splits, in their order: a workgroup for eight rows of it, or for 32 where those would be more than stay resident, as
// each looks its tile up first (43 MB of two splits of 32 sequences: 10.7 -> 6.9 us).  Two splits are read without the six that are not there.
template <typename T, int ROWS, int kRows>
__global__ __launch_bounds__(256) void tree_join_kernel(TreeArgs a) {
  const int tid = threadIdx.x, parts = ROWS / kRows, D = a.kv.dim, quads = D / 4, group = a.q_heads / a.kv.heads;
  const int kvh = blockIdx.x % a.kv.heads, rest = blockIdx.x / a.kv.heads, slot = rest / parts, r0 = (rest - slot * parts) * kRows;
  Tile t;
  if (!tile_at<ROWS>(a, slot, tid & 63, t)) return;
  const int ns = splits_of(t.begin, t.end, a.chunk);
  if (ns == 1) return;   // written already
  const float* part = a.partials + ((int64_t)slot * a.kv.heads + kvh) * a.splits * ROWS * (D + 4);
  const float* stat = part + (int64_t)a.splits * ROWS * D;
  for (int x = tid; x < kRows * quads; x += 256) {
    const int r = r0 + x / quads, d = x % quads * 4;
    if (r >= t.rows) continue;
    Joined j;
    auto take = [&]<int N>(int s0) {   // so many at once
      v2u st[N];
      v4u y[N];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int64_t s = min(s0 + k, ns - 1);
        st[k] = *(const v2u*)(stat + (s * ROWS + r) * 2);
        y[k] = *(const v4u*)(part + (s * ROWS + r) * D + d);
      }
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (s0 + k < ns) j.add(st[k], y[k]);
    };
    if (ns == 2) take.template operator()<2>(0);
    else
      for (int s0 = 0; s0 < ns; s0 += 8) take.template operator()<8>(s0);
    const int token = (t.row0 + r) / group, head = kvh * group + (t.row0 + r) % group;
    const float f = j.l == 0.f ? 0.f : (a.kv.v_scale ? a.kv.v_scale[kvh] : 1.f) / j.l;
    T* to = (T*)a.out + (int64_t)(t.start + token) * a.out_row + head * a.out_head + d;
    *(v2u*)to = v2u{pack2<T>(j.o[0] * f, j.o[1] * f), pack2<T>(j.o[2] * f, j.o[3] * f)};
    if (a.lse && d == 0)
      a.lse[(int64_t)(t.start + token) * a.q_heads + head] = j.l == 0.f ? -__builtin_huge_valf() : (j.m - kLift<T> + __builtin_amdgcn_logf(j.l)) * kLn2;
  }
}

// How a call is cut: waves that share a row's keys, rows of a tile, places for tiles, splits of `chunk` keys.
struct Cut { int key_waves, rows, slots, splits, chunk; };

// Up to 64 rows of a sequence are a tile of 64, in which two waves share the keys (16 sequences of up to 8000 8-bit keys and 8 tokens of 5 heads: 68 us, in
// tiles of 128 rows 86; 64 of up to 4000 and 4 tokens 136 and 162; tiles of 32 rows with four waves to the keys, 128 a step: 146).
//
// Where the tiles that a batch is likely to have are fewer than the workgroups that stay resident, their keys are split, into as many
// splits as still stay all at once: a few more would run on their own at the end (24 sequences of a window of 4096 keys, heads of 256 dims: 2
// splits 85.6 us, 3 111, 4 94; one of 100000 keys: 64 splits 89 us, 128 109; 16 of up to 8000 8-bit keys: 4 splits 68, 5 83).  Tiles of prompts see
// different lengths, so that a tenth more than stay do not run on their own (320 and 512 tokens of two prompts behind 5000 and 8000: 2 splits 171 us, none 211).
Cut cut_of(int tokens, int batch, int q_heads, int kv_heads, int dim, int max_tokens, int max_length, int window, int64_t workspace_bytes) {
  const int group = q_heads / kv_heads;
  const int64_t most = (int64_t)std::min(tokens, max_tokens) * group;   // rows of a sequence
  Cut c;
  c.key_waves = most <= 64 ? 2 : 1;
  c.rows = 32 * 4 / c.key_waves;
  const int64_t slots = (int64_t)tokens * group / c.rows + batch;
  c.slots = (int)slots;
  // keys that a row tile can see, from a multiple of 32
  const int64_t sees = std::min<int64_t>((int64_t)std::min(tokens, max_tokens), c.rows / group + 1);
  const int64_t span = std::min<int64_t>(max_length, window > 0 ? (int64_t)window + sees + std::min(tokens, max_tokens) + 31 : max_length);
  const int64_t units = slots * kv_heads;
  const int64_t stay = (int64_t)device_cus() * (dim <= 128 ? 2 : 1);   // workgroups, by their LDS
  const bool one = most <= c.rows;
  const int64_t tiles = std::max<int64_t>(1, one ? std::min(batch, tokens) : (int64_t)tokens * group / c.rows + batch / 2) * kv_heads;
  int64_t splits = std::max<int64_t>(1, std::min((one ? stay : stay + stay / 10) / tiles, (span + kStep - 1) / kStep));
  splits = std::min<int64_t>(splits, kMostSplits);
  const int64_t each = units * c.rows * (dim + 4) * 4;   // bytes of one split of all units
  if (workspace_bytes < GQK_CTR_BYTES || units * (c.rows / 32) > kMostGroups) splits = 1;   // (the join has a workgroup for 32 rows at least)
  else splits = std::max<int64_t>(1, std::min(splits, (workspace_bytes - GQK_CTR_BYTES) / std::max<int64_t>(1, each)));
  c.chunk = (int)std::min<int64_t>(0x7fffff80, std::max<int64_t>(kStep, ((span + splits - 1) / splits + kStep - 1) / kStep * kStep));
  c.splits = (int)std::max<int64_t>(1, (span + c.chunk - 1) / c.chunk);
  return c;
}

template <typename T, typename C, int DP, bool RUNS, bool FULL>
void launch(const TreeArgs& a, const Cut& c, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)c.slots * a.kv.heads), c.splits);
  if (c.key_waves == 2) tree_kernel<T, C, DP, 2, RUNS, FULL><<<grid, 256, 0, st>>>(a);
  else tree_kernel<T, C, DP, 1, RUNS, FULL><<<grid, 256, 0, st>>>(a);
}

template <typename T, typename C, int DP>
void launch(const TreeArgs& a, const Cut& c, hipStream_t st) {
  const int64_t page_bytes = (int64_t)a.kv.page_size * std::max(a.kv.k_token, a.kv.v_token) * (int64_t)sizeof(C);   // from its first key to the next's
  if (a.kv.page_size % 16 || page_bytes > 0x7fffffff) launch<T, C, DP, false, false>(a, c, st);
  else if (a.kv.dim == DP) launch<T, C, DP, true, true>(a, c, st);
  else launch<T, C, DP, true, false>(a, c, st);
}

template <typename T, typename C>
void launch(const TreeArgs& a, const Cut& c, hipStream_t st) {
  if (a.kv.dim <= 64) launch<T, C, 64>(a, c, st);
  else if (a.kv.dim <= 128) launch<T, C, 128>(a, c, st);
  else launch<T, C, 256>(a, c, st);
}

template <typename T, int ROWS>
void join(const TreeArgs& a, const Cut& c, hipStream_t st) {
  const int64_t eights = (int64_t)c.slots * a.kv.heads * (ROWS / 8);   // (at most 4 kMostGroups, by the count of splits)
  if (eights > 8 * device_cus()) tree_join_kernel<T, ROWS, 32><<<dim3((unsigned)(eights / 4)), 256, 0, st>>>(a);
  else tree_join_kernel<T, ROWS, 8><<<dim3((unsigned)eights), 256, 0, st>>>(a);
}

}  // namespace
}  // namespace gqk

using namespace gqk;

extern "C" {

int64_t gqk_tree_attention_workspace_bytes(int tokens, int batch, int q_heads, int kv_heads, int dim, int max_tokens, int max_length,
                                           int window) {
  if (tokens < 0 || tokens > GQK_MAX_TOKENS || batch < 0 || batch > 65535 || kv_heads < 1 || q_heads < kv_heads || q_heads % kv_heads ||
      q_heads / kv_heads > GQK_MAX_GROUP || dim < 8 || dim > 256 || dim % 8 || max_tokens < 0 || max_length < 0 || max_length > GQK_MAX_KEYS || window < 0)
    return decode_fail(GQK_ERR_SHAPE, "tree_attention: %d tokens of %d sequences, %d / %d heads of %d, max_tokens %d, max_length %d, window %d",
                       tokens, batch, q_heads, kv_heads, dim, max_tokens, max_length, window);
  if (tokens == 0 || batch == 0) return 0;
  const Cut c = cut_of(tokens, batch, q_heads, kv_heads, dim, max_tokens, max_length, window, INT64_MAX);
  return c.splits > 1 ? GQK_CTR_BYTES + (int64_t)c.slots * kv_heads * c.rows * c.splits * (dim + 4) * 4 : 0;
}

int gqk_tree_attention(const void* q, int64_t q_row, int64_t q_head, int dtype, int tokens, int batch, int q_heads,
                       const gqk_pages* pages, const int32_t* table, int64_t table_row, int table_width, const int32_t* lengths,
                       const int32_t* starts, const int32_t* mask, int mask_words, int max_length, int max_tokens, int window, float scale,
                       void* out, int64_t out_row, int64_t out_head, float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "tree_attention";
  if (dtype != GQK_DTYPE_BF16 && dtype != GQK_DTYPE_F16) return decode_fail(GQK_ERR_ARG, "%s: dtype %d", what, dtype);
  if (const int rc = check_pages(what, pages, dtype)) return rc;
  if (tokens < 0 || tokens > GQK_MAX_TOKENS || batch < 0 || batch > 65535 || q_heads < 1 || q_heads % pages->heads ||
      q_heads / pages->heads > GQK_MAX_GROUP)
    return decode_fail(GQK_ERR_SHAPE, "%s: %d tokens of %d sequences, %d query heads over %d", what, tokens, batch, q_heads, pages->heads);
  if (window < 0 || max_tokens < 0 || max_length < 0 || max_length > GQK_MAX_KEYS || table_width < 0 ||
      (int64_t)max_length > (int64_t)table_width * pages->page_size)
    return decode_fail(GQK_ERR_SHAPE, "%s: window %d, up to %d tokens, lengths up to %d in %d pages of %d tokens", what, window, max_tokens,
                       max_length, table_width, pages->page_size);
  if (mask && mask_words < 1) return decode_fail(GQK_ERR_SHAPE, "%s: a mask of %d words", what, mask_words);
  if (tokens == 0 || batch == 0) return GQK_OK;
  if (!q || !out || !lengths || !starts || (!table && max_length > 0)) return decode_fail(GQK_ERR_ARG, "%s: null pointer", what);
  if (((uintptr_t)q | (uintptr_t)out) & 15 || (q_row | q_head | out_row | out_head) & 7)
    return decode_fail(GQK_ERR_SHAPE, "%s: q and out are 16-byte aligned with strides that are multiples of 8", what);
  const Cut c = cut_of(tokens, batch, q_heads, pages->heads, pages->dim, max_tokens, max_length, window, workspace ? workspace_bytes : 0);
  if ((uintptr_t)workspace & 255) return decode_fail(GQK_ERR_SHAPE, "%s: workspace is not 256-byte aligned", what);
  if ((int64_t)c.slots * pages->heads > kMostGroups)
    return decode_fail(GQK_ERR_SHAPE, "%s: %d tokens of %d sequences, %d heads over %d are more than a launch takes", what, tokens, batch, q_heads,
                       pages->heads);
  TreeArgs a{};
  a.q = q; a.q_row = q_row; a.q_head = q_head; a.kv = *pages; a.table = table; a.table_row = table_row; a.lengths = lengths; a.starts = starts;
  a.mask = mask; a.words = mask_words; a.out = out; a.out_row = out_row; a.out_head = out_head; a.lse = lse; a.tokens = tokens; a.batch = batch;
  a.q_heads = q_heads; a.max_length = max_length; a.max_tokens = max_tokens; a.window = window; a.scale = fabsf(scale) * kLog2e; a.sign = scale < 0.f ? 0x80008000u : 0u;
  a.chunk = c.chunk; a.splits = c.splits; a.slots = c.slots; a.once = (int64_t)std::min(tokens, max_tokens) * (q_heads / pages->heads) <= c.rows;
  a.partials = workspace ? (float*)((char*)workspace + GQK_CTR_BYTES) : nullptr;
  const PageDivisor by = page_divisor(pages->page_size);
  a.magic = by.magic;
  a.shift = by.shift;
  const hipStream_t st = (hipStream_t)stream;
  const bool bf = dtype == GQK_DTYPE_BF16;
  if (pages->dtype == GQK_DTYPE_FP8) {
    if (bf) launch<bf16_t, fp8_t>(a, c, st);
    else launch<f16_t, fp8_t>(a, c, st);
  } else if (bf) {
    launch<bf16_t, bf16_t>(a, c, st);
  } else {
    launch<f16_t, f16_t>(a, c, st);
  }
  if (c.splits > 1) {
    if (bf) c.rows == 64 ? join<bf16_t, 64>(a, c, st) : join<bf16_t, 128>(a, c, st);
    else c.rows == 64 ? join<f16_t, 64>(a, c, st) : join<f16_t, 128>(a, c, st);
  }
  return decode_launched(what);
}

}  // extern "C"
