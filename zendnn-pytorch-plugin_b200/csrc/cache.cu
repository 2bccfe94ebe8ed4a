// Pages of a paged cache copied, in every layer's cache by one launch: cache[dst[i]] = cache[src[i]].
//
// Bound by memory: every byte of the pages is read once and written once.
#include "tc05.cuh"

namespace zt {

namespace {

constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 4;   // vectors in flight per thread
constexpr int kMaxCaches = 64;   // caches per launch; they travel in the launch's parameters

struct CopyParams {
  struct {
    char *base;
    int64_t stride, bytes;   // page to page, and of a page
  } cache[kMaxCaches];
  const void *src, *dst;
  int index64, num_pages;
  int *status;
};

// blockIdx.x: chunk of a page, y: pair, z: cache.  V: the vector that bases, strides and page sizes are multiples of.
template <typename V>
__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(const __grid_constant__ CopyParams p, int64_t first_pair) {
  grid_launch_dependents();
  grid_dependency_wait();
  const int64_t pair = first_pair + blockIdx.y;
  const int64_t src = p.index64 ? reinterpret_cast<const int64_t *>(p.src)[pair] : reinterpret_cast<const int32_t *>(p.src)[pair];
  const int64_t dst = p.index64 ? reinterpret_cast<const int64_t *>(p.dst)[pair] : reinterpret_cast<const int32_t *>(p.dst)[pair];
  if (src < 0 || dst < 0) return;
  if (src >= p.num_pages || dst >= p.num_pages) {
    if (threadIdx.x == 0) tc::report_timeout(p.status, kStatusBadIndex);
    return;
  }
  const auto &c = p.cache[blockIdx.z];
  const V *from = reinterpret_cast<const V *>(c.base + src * c.stride);
  V *to = reinterpret_cast<V *>(c.base + dst * c.stride);
  const int64_t n = c.bytes / (int64_t)sizeof(V);
  const int64_t i = (int64_t)blockIdx.x * (kCopyThreads * kCopyUnroll) + threadIdx.x;
  V x[kCopyUnroll];
#pragma unroll
  for (int u = 0; u < kCopyUnroll; ++u)
    if (i + u * kCopyThreads < n) x[u] = from[i + u * kCopyThreads];
#pragma unroll
  for (int u = 0; u < kCopyUnroll; ++u)
    if (i + u * kCopyThreads < n) to[i + u * kCopyThreads] = x[u];
}

}  // namespace
}  // namespace zt

using namespace zt;

extern "C" int zt_cache_copy_pages(const zt_cache_copy_args_t *a, void *stream) {
  ZT_REQUIRE(a != nullptr, ZT_INVALID_ARGUMENT, "zt_cache_copy_pages: null argument block");
  ZT_REQUIRE(a->n_caches >= 0 && a->n_pairs >= 0 && a->num_pages >= 0, ZT_INVALID_ARGUMENT, "zt_cache_copy_pages: negative size");
  if (a->n_caches == 0 || a->n_pairs == 0) return ZT_SUCCESS;
  ZT_REQUIRE(a->caches && a->page_stride_bytes && a->page_bytes && a->src && a->dst, ZT_INVALID_ARGUMENT,
             "zt_cache_copy_pages: null pointer");
  int *status = device_status_ptr();
  ZT_REQUIRE(status != nullptr, ZT_CUDA_ERROR, "zt_cache_copy_pages: no device status word");
  for (int i = 0; i < a->n_caches; ++i) {
    ZT_REQUIRE(a->caches[i] && a->page_bytes[i] >= 0 && a->page_stride_bytes[i] >= a->page_bytes[i], ZT_INVALID_ARGUMENT,
               "zt_cache_copy_pages: cache %d: pages of %lld bytes need a pointer and a stride of at least that (%lld)", i,
               (long long)a->page_bytes[i], (long long)a->page_stride_bytes[i]);
    ZT_REQUIRE(a->page_bytes[i] <= ((int64_t)1 << 40), ZT_INVALID_ARGUMENT, "zt_cache_copy_pages: pages of %lld bytes",
               (long long)a->page_bytes[i]);
  }
  cudaStream_t st = (cudaStream_t)stream;
  for (int c0 = 0; c0 < a->n_caches; c0 += kMaxCaches) {
    const int n = a->n_caches - c0 < kMaxCaches ? a->n_caches - c0 : kMaxCaches;
    CopyParams p{};
    uintptr_t bits = 0;
    int64_t most = 0;
    for (int i = 0; i < n; ++i) {
      p.cache[i] = {(char *)a->caches[c0 + i], a->page_stride_bytes[c0 + i], a->page_bytes[c0 + i]};
      bits |= (uintptr_t)p.cache[i].base | (uintptr_t)p.cache[i].stride | (uintptr_t)p.cache[i].bytes;
      if (p.cache[i].bytes > most) most = p.cache[i].bytes;
    }
    if (most == 0) continue;
    p.src = a->src, p.dst = a->dst, p.index64 = a->index_64, p.num_pages = a->num_pages, p.status = status;
    const int64_t chunk = (int64_t)kCopyThreads * kCopyUnroll * (bits % 16 == 0 ? 16 : 1);
    const int64_t chunks = ceil_div(most, chunk);
    ZT_REQUIRE(chunks < ((int64_t)1 << 31), ZT_UNSUPPORTED, "zt_cache_copy_pages: pages of %lld bytes are too large", (long long)most);
    for (int64_t first = 0; first < a->n_pairs; first += 65535) {
      const int64_t pairs = a->n_pairs - first < 65535 ? a->n_pairs - first : 65535;
      const dim3 grid((unsigned)chunks, (unsigned)pairs, (unsigned)n);
      if (bits % 16 == 0)
        ZT_CUDA_OK(launch_overlapped(copy_pages_kernel<uint4>, grid, dim3(kCopyThreads), (size_t)0, st, p, first));
      else
        ZT_CUDA_OK(launch_overlapped(copy_pages_kernel<uint8_t>, grid, dim3(kCopyThreads), (size_t)0, st, p, first));
      const int rc = launch_status("copy_pages_kernel");
      if (rc != ZT_SUCCESS) return rc;
    }
  }
  return ZT_SUCCESS;
}
