// gqk_pages.hip - copies of a cache's pages: in every plane (each layer's keys and values), page
// src[i] to page dst[i], one launch for each 448 pairs (and each 32768 planes).
#include <new>
#include <vector>
#include "gqk_decode.h"

namespace gqk {
namespace {

// Pairs travel in the kernel's arguments (at most 4 KiB of them): no upload, nothing to keep alive.
constexpr int kPairs = 448;
struct CopyArgs {
  char* base;
  int64_t plane, page, bytes;
  int32_t src[kPairs], dst[kPairs];
};

typedef uint32_t v4u __attribute__((ext_vector_type(4)));

// A workgroup copies one page of one plane; nothing is computed, memory bounds it.  Lines on their way through leave the
// caches first (400 pages of 16 KiB in 128 planes: 325 -> 306 us, 5.5 TB/s read and written together).
template <typename W>
__global__ __launch_bounds__(256) void copy_kernel(CopyArgs a) {
  const W* from = (const W*)(a.base + blockIdx.y * a.plane + a.src[blockIdx.x] * a.page);
  W* to = (W*)(a.base + blockIdx.y * a.plane + a.dst[blockIdx.x] * a.page);
  for (int64_t i = threadIdx.x; i < a.bytes / (int64_t)sizeof(W); i += 256)
    __builtin_nontemporal_store(__builtin_nontemporal_load(from + i), to + i);
}

}  // namespace
}  // namespace gqk

using namespace gqk;

extern "C" int gqk_copy_pages(void* base, int64_t planes, int64_t plane_stride, int64_t pages, int64_t page_stride,
                              int64_t page_bytes, const int32_t* src, const int32_t* dst, int64_t n, void* stream) {
  const char* what = "copy_pages";
  if (planes < 0 || pages < 0 || pages > 0x7fffffff || page_bytes < 0 || n < 0 || page_stride < page_bytes || plane_stride < 0)
    return decode_fail(GQK_ERR_SHAPE, "%s: %lld planes of %lld pages of %lld bytes (stride %lld), %lld pairs", what,
                       (long long)planes, (long long)pages, (long long)page_bytes, (long long)page_stride, (long long)n);
  if (n == 0) return GQK_OK;
  if (!src || !dst) return decode_fail(GQK_ERR_ARG, "%s: null pointer", what);
  try {
    std::vector<uint8_t> seen((size_t)pages, 0);   // 1: written, 2: read
    for (int64_t i = 0; i < n; ++i) {
      if (src[i] < 0 || src[i] >= pages || dst[i] < 0 || dst[i] >= pages)
        return decode_fail(GQK_ERR_SHAPE, "%s: pair %lld (%d to %d) is outside of %lld pages", what, (long long)i, src[i], dst[i],
                           (long long)pages);
      if (seen[dst[i]] & 1) return decode_fail(GQK_ERR_ARG, "%s: page %d is written twice", what, dst[i]);
      seen[dst[i]] |= 1;
      seen[src[i]] |= 2;
    }
    for (int64_t i = 0; i < n; ++i)
      if (seen[dst[i]] == 3) return decode_fail(GQK_ERR_ARG, "%s: page %d is both read and written", what, dst[i]);
  } catch (const std::bad_alloc&) {
    return decode_fail(GQK_ERR_ARG, "%s: no host memory to check %lld pairs", what, (long long)n);
  }
  if (planes == 0 || page_bytes == 0) return GQK_OK;
  if (!base) return decode_fail(GQK_ERR_ARG, "%s: null pointer", what);
  const hipStream_t st = (hipStream_t)stream;
  const uint64_t bits = (uintptr_t)base | (uint64_t)page_stride | (uint64_t)plane_stride | (uint64_t)page_bytes;
  CopyArgs a{};
  a.plane = plane_stride; a.page = page_stride; a.bytes = page_bytes;
  for (int64_t p0 = 0; p0 < planes; p0 += 32768) {
    a.base = (char*)base + p0 * plane_stride;
    for (int64_t i0 = 0; i0 < n; i0 += kPairs) {
      const int c = (int)(n - i0 < kPairs ? n - i0 : kPairs);
      for (int i = 0; i < c; ++i) a.src[i] = src[i0 + i], a.dst[i] = dst[i0 + i];
      const dim3 grid(c, (unsigned)(planes - p0 < 32768 ? planes - p0 : 32768));
      if (!(bits & 15)) copy_kernel<v4u><<<grid, 256, 0, st>>>(a);
      else if (!(bits & 3)) copy_kernel<uint32_t><<<grid, 256, 0, st>>>(a);
      else copy_kernel<uint8_t><<<grid, 256, 0, st>>>(a);
    }
  }
  return decode_launched(what);
}
