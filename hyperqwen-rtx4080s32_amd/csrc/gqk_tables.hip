// gqk_tables.hip - what a step of many sequences needs to know of its tokens, built on the GPU from the sequences' lengths.
//
// Sequence b brings n_b = counts[b] new tokens behind lengths[b] keys; its tokens are the rows start_b = n_0 + .. + n_(b-1) on.  Token i
// of it: place p = lengths[b] + i in the cache, slot = page * page_size + p % page_size with the page of its list that holds p; its
// position is lengths[b] plus the number of its ancestors among the new tokens (a chain: i), and a tree's mask has the bits of those
// ancestors and its own.
#include <algorithm>
#include "gqk_decode.h"

namespace gqk {
namespace {

struct TablesArgs {
  const int32_t* lists;
  int64_t list_row;
  const void* requests;
  const int32_t *lengths, *counts, *parents;
  int32_t *table, *totals, *starts, *sequences, *positions, *mask;
  int64_t* slots;
  int wide_requests, lists_n, width, batch, tokens, page_size, tree, words;
};

constexpr int kThreads = 256;

// Sequence blockIdx.x, a part (blockIdx.y) of its table's columns and of its tokens; the sequence after the last is the rows without one.
// Everything is in the trips to memory that follow one another: counts, the list, (the tree's parents,) the stores.  A workgroup adds up
// the counts before its own by itself, which needs no second launch.  32 trees of up to 16 tokens, tables of 256 pages: 4.8 us; 512 chunks of up to
// 63, tables of 2048 (4.2 MB written): 5.3.  A call takes the host 10, half of it the seven or eight tensors that it returns.
__global__ __launch_bounds__(kThreads) void tables_kernel(TablesArgs a) {
  __shared__ int64_t sums[kThreads / 64];
  __shared__ int32_t parent[GQK_MAX_TREE];
  const int b = blockIdx.x, tid = threadIdx.x;
  const bool none = b == a.batch;
  const int len = none ? 0 : a.lengths[b], n0 = none ? 0 : a.counts[b];
  const int64_t request = none ? -1 : index_at(a.requests, a.wide_requests, b);
  int64_t before = 0;
  for (int i = tid; i < b; i += kThreads) before += max(0, a.counts[i]);
  for (int o = 32; o > 0; o >>= 1) before += __shfl_xor(before, o);
  if ((tid & 63) == 0) sums[tid >> 6] = before;
  __syncthreads();
  before = 0;
#pragma unroll
  for (int k = 0; k < kThreads / 64; ++k) before += sums[k];
  const int part = blockIdx.y * kThreads + tid, step = gridDim.y * kThreads;
  const int start = (int)min(before, (int64_t)a.tokens);
  if (none) {   // the rows behind the last token
    if (b == 0 && part == 0) a.starts[0] = 0;
    for (int t = start + part; t < a.tokens; t += step) {
      a.sequences[t] = -1;
      a.positions[t] = 0;
      a.slots[t] = -1;
      for (int w = 0; w < a.words; ++w) a.mask[(int64_t)t * a.words + w] = 0;
    }
    return;
  }
  const int n = max(0, n0), end = (int)min(before + n, (int64_t)a.tokens);
  const int64_t total = (int64_t)len + n, room = min((int64_t)a.width * a.page_size, (int64_t)GQK_MAX_KEYS);
  const bool empty = request < 0 && n == 0;   // a row of the batch without a sequence
  const bool sound = request >= 0 && request < a.lists_n && len >= 0 && n0 >= 0 && total <= room && before + n <= a.tokens &&
                     (a.tree == 0 || n <= a.tree);
  if (part == 0) {
    a.totals[b] = empty ? 0 : sound ? (int)total : 0x7fffffff;   // above any bound on the lengths: the attention's result is NaN
    a.starts[b + 1] = end;
    if (b == 0) a.starts[0] = 0;
  }
  const int32_t* list = a.lists + (sound ? request * a.list_row : 0);
  const int pages = sound ? (int)((total + a.page_size - 1) / a.page_size) : 0;
  for (int j = part; j < a.width; j += step) a.table[(int64_t)b * a.width + j] = j < pages ? list[j] : -1;
  if (a.tree && sound) {
    for (int i = tid; i < n; i += kThreads) parent[i] = a.parents[start + i];
    __syncthreads();
  }
  for (int i = part; i < end - start; i += step) {
    const int t = start + i;
    int64_t slot = -1;
    int position = -1;
    if (sound) {
      const int place = len + i, page = place / a.page_size, at = list[page];
      slot = at < 0 ? -1 : (int64_t)at * a.page_size + (place - page * a.page_size);
      position = place;
    }
    if (a.tree) {
      // From the token to its oldest ancestor the numbers fall, so that each word of the row is complete when the walk leaves it.
      int32_t* row = a.mask + (int64_t)t * a.words;
      bool good = sound;
      int depth = 0, word = a.words - 1;
      uint32_t bits = 0;
      for (int p = i; good;) {
        for (; word > (p >> 5); --word, bits = 0) row[word] = (int)bits;
        bits |= 1u << (p & 31);
        const int up = parent[p];
        good = up >= -1 && up < p;   // a parent comes before its child
        if (up < 0) break;
        ++depth;
        p = up;
      }
      for (; word >= 0; --word, bits = 0) row[word] = (int)bits;
      if (!good)
        for (int w = 0; w < a.words; ++w) row[w] = 0;
      position = good ? len + depth : -1;
    }
    a.sequences[t] = b;
    a.positions[t] = position;
    a.slots[t] = slot;
  }
}

}  // namespace
}  // namespace gqk

using namespace gqk;

extern "C" int gqk_step_tables(const int32_t* lists, int64_t list_row, int lists_n, int width, const void* requests, int requests_64,
                               const int32_t* lengths, const int32_t* counts, int batch, int tokens, int page_size,
                               const int32_t* parents, int tree, int32_t* table, int32_t* totals, int32_t* starts, int32_t* sequences,
                               int32_t* positions, int64_t* slots, int32_t* mask, void* stream) {
  const char* what = "step_tables";
  if (lists_n < 0 || width < 0 || batch < 0 || batch > 65535 || tokens < 0 || page_size < 1)
    return decode_fail(GQK_ERR_SHAPE, "%s: %d lists of %d pages of %d tokens, %d sequences (at most 65535), %d tokens", what, lists_n, width,
                       page_size, batch, tokens);
  if (tree < 0 || tree > GQK_MAX_TREE || (tree == 0 && parents) || (tree > 0 && tokens > 0 && !parents))
    return decode_fail(GQK_ERR_SHAPE, "%s: trees of up to %d tokens (at most %d, with parents)", what, tree, GQK_MAX_TREE);
  if (lists_n > 1 && list_row < width) return decode_fail(GQK_ERR_SHAPE, "%s: lists of %d pages overlap", what, width);
  if (!starts || (batch > 0 && (!requests || !lengths || !counts || !totals)) || (batch > 0 && width > 0 && (!table || (lists_n > 0 && !lists))) ||
      (tokens > 0 && (!sequences || !positions || !slots || (tree && !mask))))
    return decode_fail(GQK_ERR_ARG, "%s: null pointer", what);
  TablesArgs a{};
  a.lists = lists; a.list_row = list_row; a.lists_n = lists_n; a.width = width; a.requests = requests; a.wide_requests = requests_64;
  a.lengths = lengths; a.counts = counts; a.batch = batch; a.tokens = tokens; a.page_size = page_size; a.parents = parents; a.tree = tree;
  a.words = (tree + 31) / 32; a.table = table; a.totals = totals; a.starts = starts; a.sequences = sequences; a.positions = positions;
  a.slots = slots; a.mask = mask;
  // a thousand columns or tokens to a workgroup while that leaves no more than a thousand workgroups
  const int parts = std::max(1, std::min((std::max(width, tokens) + 1023) / 1024, 1024 / (batch + 1)));
  tables_kernel<<<dim3(batch + 1, parts), kThreads, 0, (hipStream_t)stream>>>(a);
  return decode_launched(what);
}
