// Copies of pages inside a paged cache: the first `rows` token rows of page src become those of page dst, in every cache
// tensor (keys and values of every layer), in one launch.  Rows of dst behind them are left as they are.
//
// The pairs are host data of one step, so they travel as the kernel's parameter: nothing is staged, nothing has to outlive the
// call, and a captured graph holds them.  Bound by memory traffic (each row read and written once); work items are
// (pair, tensor, 32 KiB of the rows), and every thread has eight 16-byte loads in flight before its first store.

#include <cuda_runtime.h>
#include <stdint.h>

namespace b200 {

struct CacheTensor {
  char* base;
  long long page_bytes;        // between pages
  long long head_bytes;        // between heads of a page (rows of a head follow one another)
  int heads;
  int row_vecs;                // 16-byte vectors of a token row of a head
};

struct PagePair {
  int src, dst, rows;
};

template <int N>
struct PagePairs {
  PagePair p[N];
};

static constexpr int kCopyThreads = 256, kCopyDepth = 8;
static constexpr int kCopyVecs = kCopyThreads * kCopyDepth;

template <int N>
__global__ void __launch_bounds__(kCopyThreads)
cache_copy_kernel(const CacheTensor* __restrict__ tensors, int num_tensors, int num_pairs, int page, int chunks,
                  const __grid_constant__ PagePairs<N> pairs) {
  const long long total = static_cast<long long>(num_pairs) * num_tensors * chunks;
  for (long long item = blockIdx.x; item < total; item += gridDim.x) {
    const int chunk = static_cast<int>(item % chunks);
    const long long rest = item / chunks;
    const CacheTensor t = tensors[rest % num_tensors];
    const PagePair pr = pairs.p[rest / num_tensors];
    int heads = t.heads, per = pr.rows * t.row_vecs;             // vectors of a head
    if (pr.rows == page && t.head_bytes == static_cast<long long>(per) * 16) {
      per *= heads;                                              // a whole page in one piece
      heads = 1;
    }
    const int all = heads * per, first = chunk * kCopyVecs + threadIdx.x;
    if (chunk * kCopyVecs >= all) continue;
    const char* src = t.base + pr.src * t.page_bytes;
    char* dst = t.base + pr.dst * t.page_bytes;
    uint4 v[kCopyDepth];
    long long at[kCopyDepth];
#pragma unroll
    for (int u = 0; u < kCopyDepth; ++u) {
      const int i = first + u * kCopyThreads;
      const int h = i / per;
      at[u] = h * t.head_bytes + static_cast<long long>(i - h * per) * 16;
      if (i < all) v[u] = *reinterpret_cast<const uint4*>(src + at[u]);
    }
#pragma unroll
    for (int u = 0; u < kCopyDepth; ++u)
      if (first + u * kCopyThreads < all) *reinterpret_cast<uint4*>(dst + at[u]) = v[u];
  }
}

template <int N>
static int launch_copy(const CacheTensor* tensors, int num_tensors, const PagePair* pairs, int num_pairs, int page, int chunks,
                       int sms, cudaStream_t stream) {
  PagePairs<N> arg;
  for (int i = 0; i < num_pairs; ++i) arg.p[i] = pairs[i];
  const long long total = static_cast<long long>(num_pairs) * num_tensors * chunks, cap = 8LL * sms;
  cache_copy_kernel<N><<<static_cast<int>(total < cap ? total : cap), kCopyThreads, 0, stream>>>(tensors, num_tensors, num_pairs,
                                                                                                page, chunks, arg);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

}  // namespace b200

// tensors: device array of descriptors; pairs: num_pairs x (src, dst, rows) on the host, checked by the caller.
// max_vecs: most 16-byte vectors of a page of any tensor.
extern "C" int b200_cache_copy(const void* tensors, int num_tensors, const int* pairs, int num_pairs, int page, int max_vecs,
                               int sms, cudaStream_t stream) {
  using namespace b200;
  if (num_pairs <= 0 || num_tensors <= 0) return 0;
  const auto* ts = static_cast<const CacheTensor*>(tensors);
  const auto* pp = reinterpret_cast<const PagePair*>(pairs);
  const int chunks = (max_vecs + kCopyVecs - 1) / kCopyVecs;
  for (int i = 0; i < num_pairs;) {
    const int n = num_pairs - i < 2048 ? num_pairs - i : 2048;
    const int rc = n <= 16 ? launch_copy<16>(ts, num_tensors, pp + i, n, page, chunks, sms, stream)
                 : n <= 256 ? launch_copy<256>(ts, num_tensors, pp + i, n, page, chunks, sms, stream)
                            : launch_copy<2048>(ts, num_tensors, pp + i, n, page, chunks, sms, stream);
    if (rc != 0) return rc;
    i += n;
  }
  return 0;
}
