// Copies of cache pages: for every pool and every pair (src, dst), page dst becomes page src. One launch serves all layers
// (keys and values, or 4-bit pages): forking a sequence copies one page in each of dozens of pools, a few KB a piece.
//
// Pairs are independent: no dst is another pair's src or dst. A pair with a page number outside the pool is left out.
#include "host_common.h"
#include "launch_behind.cuh"
#include "ptx.cuh"

namespace icb {

constexpr int kPageCopyPools = 96;        // pools of one launch (kernel parameters hold 4 KB)
constexpr int kPageCopyThreads = 128;
constexpr int kPageCopyDepth = 5;         // accesses in flight per thread

struct PagePool {
  uint8_t* base;
  long long layer_bytes;                  // distance of the layers of a stacked pool
  long long page_bytes;
  long long first_item;                   // where this pool's work items start
  int layers, num_pages;
};
struct PageCopyArgs {
  PagePool pool[kPageCopyPools];
  const int* src;
  const int* dst;
  int pools, pairs;
};

// A page is cut into the fewest equal stretches that a block moves with all its loads in flight. Equal: 4-bit pages of 18 KB and
// the like would leave a short last stretch (448 pairs of 18 KB in 32 layers, from 64 pages: 58 us, now 50.3, 0.92 of the copy
// bandwidth). Blocks that take neighbouring VECs across pages' borders need two divisions per access and wait for them (76 us).
// 128 threads of 5 accesses: 8 KB pages, 448 pairs in 56 pools, 40.8 us; 256 of 4 45.5, 128 of 16 53.6.
__host__ __device__ inline long long page_stretches(long long n) {
  return (n + kPageCopyThreads * kPageCopyDepth - 1) / (kPageCopyThreads * kPageCopyDepth);
}

template <typename VEC>
__global__ void __launch_bounds__(kPageCopyThreads) page_copy_kernel(const __grid_constant__ PageCopyArgs a) {
  wait_for_previous();
  const uint32_t item = blockIdx.x;
  int p = 0;
  while (p + 1 < a.pools && item >= a.pool[p + 1].first_item) ++p;
  const PagePool& pool = a.pool[p];
  const uint32_t n = (uint32_t)(pool.page_bytes / (long long)sizeof(VEC)), stretches = (uint32_t)page_stretches(n);
  const uint32_t local = item - (uint32_t)pool.first_item, unit = local / stretches, each = (n + stretches - 1) / stretches;
  const uint32_t layer = unit / a.pairs, pair = unit - layer * a.pairs;
  const int s = a.src[pair], d = a.dst[pair];
  if (s < 0 || d < 0 || s >= pool.num_pages || d >= pool.num_pages) return;
  const VEC* from = reinterpret_cast<const VEC*>(pool.base + layer * pool.layer_bytes + s * pool.page_bytes);
  VEC* to = reinterpret_cast<VEC*>(pool.base + layer * pool.layer_bytes + d * pool.page_bytes);
  const uint32_t at = (local - unit * stretches) * each + threadIdx.x, end = min(n, at - threadIdx.x + each);
  VEC x[kPageCopyDepth];
#pragma unroll
  for (int i = 0; i < kPageCopyDepth; ++i)
    if (at + i * kPageCopyThreads < end) x[i] = from[at + i * kPageCopyThreads];
#pragma unroll
  for (int i = 0; i < kPageCopyDepth; ++i)
    if (at + i * kPageCopyThreads < end) to[at + i * kPageCopyThreads] = x[i];
}

template <typename VEC>
static int launch_page_copy(PageCopyArgs& a, cudaStream_t st) {
  long long items = 0;
  for (int p = 0; p < a.pools; ++p) {
    const long long n = a.pool[p].page_bytes / (long long)sizeof(VEC);
    if (n > 0x7fffffffLL) return -2;
    a.pool[p].first_item = items;
    items += page_stretches(n) * a.pool[p].layers * a.pairs;
  }
  if (items <= 0) return 0;
  if (items > 0x7fffffffLL) return -3;
  return launch_behind("page_copy", page_copy_kernel<VEC>, (unsigned)items, kPageCopyThreads, 0, st, a);
}

}  // namespace icb

using namespace icb;

// pools: host array of n records {address, layers, bytes between layers, pages, bytes of a page}; src, dst: device int32
// [pairs].
ICB_API int icb_copy_pages(const long long* pools, int n, const int* src, const int* dst, int pairs, void* stream) {
  if (pairs <= 0 || n <= 0) return 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  for (int lo = 0; lo < n; lo += kPageCopyPools) {
    PageCopyArgs a;
    a.pools = n - lo < kPageCopyPools ? n - lo : kPageCopyPools;
    a.pairs = pairs;
    a.src = src;
    a.dst = dst;
    long long align = 0;
    for (int p = 0; p < a.pools; ++p) {
      const long long* rec = pools + 5 * (lo + p);
      if (rec[1] < 0 || rec[3] < 0 || rec[4] < 0 || rec[1] > 0x7fffffffLL || rec[3] > 0x7fffffffLL) return -2;
      a.pool[p] = PagePool{reinterpret_cast<uint8_t*>(rec[0]), rec[2], rec[4], 0, (int)rec[1], (int)rec[3]};
      align |= rec[0] | rec[2] | rec[4];
    }
    const int rc = align % 16 == 0 ? launch_page_copy<uint4>(a, st)
                   : align % 4 == 0 ? launch_page_copy<uint32_t>(a, st)
                                    : launch_page_copy<uint8_t>(a, st);
    if (rc != 0) return rc;
  }
  return 0;
}
