// Block copies inside a paged cache pool: what forking a request (its last,
// partly filled block gets an own copy) and compacting a pool (live blocks move
// into free ones further down) need on the device.
//
// A pool is `planes` equal arrays of num_blocks pages (a layer's K or V each), a
// page one contiguous run; the 8-bit pool's block scales are a second set of
// planes and move in the same launch.  Pure copy, bound by HBM: 2 * n * planes *
// page bytes.  One CTA copies one page of one plane, four 16-byte loads a thread
// in flight: 600 pages of 32 KB in 24 planes take 152 us = 6.2 TB/s (95 % of a plain
// copy), 64 of 16 KB in 64 planes 24.4 us = 5.5 TB/s.  The pairs ride in the kernel's parameters, so a call needs no
// device list, no copy of one and no synchronisation.
#include <stdlib.h>

#include "abi_util.h"
#include "common.cuh"

namespace muk {

constexpr int kPairs = 256;          // pairs per launch (2 KB of parameters)
constexpr int kCopyThreads = 256;

struct PagePairs {
  int32_t src[kPairs], dst[kPairs];
};

__global__ void __launch_bounds__(kCopyThreads)
    copy_pages_kernel(uint8_t* pool, int64_t plane_stride, int64_t page_bytes, uint8_t* scales,
                      int64_t scale_plane_stride, int scale_bytes,
                      const __grid_constant__ PagePairs pairs) {
  // programmatic dependent launch: let the next kernel launch once every CTA
  // of this one runs, and wait for the previous kernel before touching memory
  grid_dep_launch();
  grid_dep_wait();
  const int64_t s = pairs.src[blockIdx.x], d = pairs.dst[blockIdx.x];
  const int plane = blockIdx.y;
  uint8_t* base = pool + (int64_t)plane * plane_stride;
  const uint4* from = reinterpret_cast<const uint4*>(base + s * page_bytes);
  uint4* to = reinterpret_cast<uint4*>(base + d * page_bytes);
  const int64_t units = page_bytes / 16;
  for (int64_t i = threadIdx.x; i < units; i += 4 * blockDim.x) {
    uint4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i + u * blockDim.x < units) v[u] = __ldcs(from + i + u * blockDim.x);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i + u * blockDim.x < units) __stcs(to + i + u * blockDim.x, v[u]);
  }
  if (scales != nullptr) {
    uint8_t* sb = scales + (int64_t)plane * scale_plane_stride;
    for (int i = threadIdx.x; i < scale_bytes / 4; i += blockDim.x)
      reinterpret_cast<uint32_t*>(sb + d * scale_bytes)[i] =
          reinterpret_cast<const uint32_t*>(sb + s * scale_bytes)[i];
  }
}

}  // namespace muk

using namespace muk;

extern "C" int muk_copy_pages(void* pool, int64_t plane_stride, int num_planes, int64_t page_bytes,
                              void* scales, int64_t scale_plane_stride, int scale_bytes,
                              int num_blocks, const int32_t* src, const int32_t* dst, int n,
                              void* stream) {
  if (n <= 0) return MUK_OK;
  MUK_REQUIRE(pool && src && dst, "muk_copy_pages: null pointer");
  MUK_REQUIRE(num_planes > 0 && num_planes <= 65535 && num_blocks > 0,
              "muk_copy_pages: %d planes of %d blocks", num_planes, num_blocks);
  MUK_REQUIRE(page_bytes > 0 && page_bytes % 16 == 0 && plane_stride % 16 == 0 &&
                  MUK_ALIGNED16(pool) && plane_stride / page_bytes >= num_blocks,
              "muk_copy_pages: pages and planes must be multiples of 16 bytes (page %lld, plane "
              "%lld)",
              (long long)page_bytes, (long long)plane_stride);
  MUK_REQUIRE(scales == nullptr ||
                  (scale_bytes > 0 && scale_bytes % 4 == 0 && scale_plane_stride % 4 == 0 &&
                   (reinterpret_cast<uintptr_t>(scales) & 3u) == 0 &&
                   scale_plane_stride / scale_bytes >= num_blocks),
              "muk_copy_pages: block scales of %d bytes, plane %lld", scale_bytes,
              (long long)scale_plane_stride);
  // The copies run in any order: no page may be written twice, or read and
  // written.  1 = read, 2 = written.
  uint8_t* seen = static_cast<uint8_t*>(calloc((size_t)num_blocks, 1));
  if (seen == nullptr) {
    set_last_error("muk_copy_pages: out of host memory");
    return MUK_ERR_INVALID_ARG;
  }
  const char* bad = nullptr;
  int at = 0;
  for (int i = 0; i < n && bad == nullptr; ++i) {
    at = i;
    if (src[i] < 0 || src[i] >= num_blocks || dst[i] < 0 || dst[i] >= num_blocks) {
      bad = "a block id is out of range";
    } else if (seen[dst[i]] != 0 || src[i] == dst[i]) {
      bad = "a destination is named twice, or is a source too";
    } else if (seen[src[i]] == 2) {
      bad = "a source is a destination too";
    } else {
      seen[src[i]] = 1;
      seen[dst[i]] = 2;
    }
  }
  free(seen);
  MUK_REQUIRE(bad == nullptr, "muk_copy_pages: %s (pair %d)", bad, at);
  const int64_t units = page_bytes / 16;
  const int threads = units >= kCopyThreads ? kCopyThreads : (int)((units + 31) / 32 * 32);
  for (int i = 0; i < n; i += kPairs) {
    PagePairs p;
    const int m = n - i < kPairs ? n - i : kPairs;
    for (int j = 0; j < kPairs; ++j) {
      p.src[j] = src[i + (j < m ? j : 0)];
      p.dst[j] = dst[i + (j < m ? j : 0)];
    }
    launch_pdl(copy_pages_kernel, dim3(m, num_planes), dim3(threads), 0, as_stream(stream),
               static_cast<uint8_t*>(pool), plane_stride, page_bytes, static_cast<uint8_t*>(scales),
               scale_plane_stride, scale_bytes, p);
    MUK_TRY(check_launch("muk_copy_pages"));
  }
  return MUK_OK;
}
