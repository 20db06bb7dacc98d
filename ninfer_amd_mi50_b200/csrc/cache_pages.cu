// Rows and pages of the cache copied within it, for all of a group's layers in one launch: the rows of the path that was
// kept of a tree moved up behind what its request held, and pages copied for a request that is forked.
//
// A page is `planes` runs (keys and values of every key head; one for rows of any width) of page_size rows of row_bytes.
// Both kernels only move bytes: what bounds them is memory, and for few rows a trip to it.  160 pages of 28 layers, 587 MB, are
// copied in 179 us (6.5 TB/s read and written), a page of 24 layers in 5.3; the rows kept of one request and 24 layers move in
// 4.5 us, of 64 requests in 7.5.
#include "common.cuh"

namespace nf {
namespace {

constexpr int kThreads = 256;
constexpr int kMoves = 128;               // rows of a request looked up at a time

__device__ int g_pages_error = 0;

struct PageShape {
  unsigned char* base;
  long long layer_bytes;                  // from one layer's pages to the next one's
  int layers, num_pages, planes, page_size, row_bytes;
};

// Row lengths[s] + 1 + j takes the place of row lengths[s] + path[s][j], j < accepted[s].  path rises, so path[j] > j, and
// a thread that takes its piece of the rows in that order reads each before it is written; pieces of one row are one
// thread's throughout.
template <typename P>
__global__ void __launch_bounds__(kThreads)
compact_cache_kernel(PageShape c, const int* __restrict__ block_table, int bt_width, const int* __restrict__ lengths,
                     const int* __restrict__ path, const int* __restrict__ accepted, int most) {
  __shared__ long long from[kMoves], to[kMoves];
  __shared__ int moves, wrong;
  const int s = blockIdx.x, n = accepted[s], len = lengths[s];
  if (threadIdx.x == 0) wrong = n < 0 || n > most || len < 0;
  __syncthreads();
  const int* p = path + (size_t)s * most;
  for (int j = threadIdx.x; j < min(n, most); j += kThreads)
    if (p[j] <= j || (j > 0 && p[j] <= p[j - 1])) wrong = 1;
  __syncthreads();
  if (wrong) {                                             // a path that makes no sense moves nothing
    if (blockIdx.y == 0 && threadIdx.x == 0) atomicCAS(&g_pages_error, 0, 1 + s);
    return;
  }
  const int pieces = c.row_bytes / (int)sizeof(P);
  const long long page_bytes = (long long)c.planes * c.page_size * c.row_bytes;
  const long long all = (long long)c.layers * c.planes * pieces;
  for (int j0 = 0; j0 < n; j0 += kMoves) {
    __syncthreads();
    if (threadIdx.x == 0) moves = 0;
    if (threadIdx.x < 32) {
      // (warp 0 lists the rows that move, in order)
      int count = 0;
      for (int j = j0 + threadIdx.x; j - (int)threadIdx.x < min(n, j0 + kMoves); j += 32) {
        bool go = false;
        long long a = 0, b = 0;
        if (j < min(n, j0 + kMoves) && p[j] != j + 1) {
          const long long src = (long long)len + p[j], dst = (long long)len + 1 + j;
          const long long lp = src / c.page_size, lq = dst / c.page_size;
          const int page = lp < bt_width ? block_table[(size_t)s * bt_width + lp] : -1;
          const int onto = lq < bt_width ? block_table[(size_t)s * bt_width + lq] : -1;
          go = page >= 0 && page < c.num_pages && onto >= 0 && onto < c.num_pages;
          if (!go) atomicCAS(&g_pages_error, 0, 1 + s);
          a = page * page_bytes + src % c.page_size * c.row_bytes;
          b = onto * page_bytes + dst % c.page_size * c.row_bytes;
        }
        const unsigned who = __ballot_sync(0xffffffffu, go);
        if (go) {
          const int at = count + __popc(who & ((1u << threadIdx.x) - 1));
          from[at] = a, to[at] = b;
        }
        count += __popc(who);
      }
      if (threadIdx.x == 0) moves = count;
    }
    __syncthreads();
    const int m = moves;
    for (long long i = blockIdx.y * (long long)kThreads + threadIdx.x; i < all; i += (long long)gridDim.y * kThreads) {
      const long long plane = i / pieces;
      unsigned char* at = c.base + plane / c.planes * c.layer_bytes + plane % c.planes * c.page_size * c.row_bytes + i % pieces * (long long)sizeof(P);
      for (int j = 0; j < m; ++j) *reinterpret_cast<P*>(at + to[j]) = *reinterpret_cast<const P*>(at + from[j]);
    }
  }
}

// Page dst[i] takes page src[i]'s first rows[i] rows (all, where rows is null).
template <typename P>
__global__ void __launch_bounds__(kThreads)
copy_pages_kernel(PageShape c, const int* __restrict__ src, const int* __restrict__ dst, const int* __restrict__ rows) {
  const int i = blockIdx.x, a = src[i], b = dst[i], n = rows ? rows[i] : c.page_size;
  if (a < 0 || a >= c.num_pages || b < 0 || b >= c.num_pages || n < 0 || n > c.page_size) {
    if (blockIdx.y == 0 && blockIdx.z == 0 && threadIdx.x == 0) atomicCAS(&g_pages_error, 0, 1 + i);
    return;
  }
  if (a == b) return;
  const long long plane_bytes = (long long)c.page_size * c.row_bytes, page_bytes = c.planes * plane_bytes;
  // runs of bytes that lie together: the page, or the filled part of every plane
  const int runs = n == c.page_size ? 1 : c.planes;
  const long long run = (n == c.page_size ? page_bytes : (long long)n * c.row_bytes) / (int)sizeof(P), all = run * runs;
  for (int layer = blockIdx.z; layer < c.layers; layer += gridDim.z) {
    const unsigned char* from = c.base + layer * c.layer_bytes + a * page_bytes;
    unsigned char* to = c.base + layer * c.layer_bytes + b * page_bytes;
    for (long long k = blockIdx.y * (long long)kThreads + threadIdx.x; k < all; k += (long long)gridDim.y * kThreads) {
      const long long at = runs == 1 ? k * (long long)sizeof(P) : k / run * plane_bytes + k % run * (long long)sizeof(P);
      *reinterpret_cast<P*>(to + at) = *reinterpret_cast<const P*>(from + at);
    }
  }
}

template <typename F> int by_piece(const PageShape& c, F f) {
  const uintptr_t u = (uintptr_t)c.base | (uintptr_t)c.row_bytes | (uintptr_t)c.layer_bytes;
  if (u % 16 == 0) return f(uint4());
  if (u % 4 == 0) return f(unsigned());
  return f((unsigned short)0);
}

int check_shape(const PageShape& c) {
  NF_REQUIRE(c.base && c.layers > 0 && c.num_pages > 0 && c.planes > 0 && c.page_size > 0 && c.row_bytes > 0 && c.row_bytes % 2 == 0 &&
                 (uintptr_t)c.base % 2 == 0 && c.layer_bytes % 2 == 0,
             "cache pages: bad sizes layers=%d pages=%d planes=%d page=%d row=%d", c.layers, c.num_pages, c.planes, c.page_size, c.row_bytes);
  return 0;
}

}  // namespace
}  // namespace nf

using namespace nf;

// block_table int32 [S, bt_width]; lengths, accepted int32 [S]; path int32 [S, most], rising.
extern "C" int nf_compact_cache(void* pages, long long layer_bytes, int layers, int num_pages, int planes, int page_size, int row_bytes,
                                const int* block_table, int bt_width, const int* lengths, const int* path, const int* accepted, int S,
                                int most, cudaStream_t stream) {
  if (S == 0 || most == 0) return 0;
  const PageShape c = {(unsigned char*)pages, layer_bytes, layers, num_pages, planes, page_size, row_bytes};
  if (int rc = check_shape(c)) return rc;
  NF_REQUIRE(S > 0 && most > 0 && bt_width > 0, "compact cache: bad sizes S=%d most=%d", S, most);
  return by_piece(c, [&](auto p) {
    using P = decltype(p);
    const long long all = (long long)layers * planes * (row_bytes / (int)sizeof(P));
    const dim3 grid(S, (unsigned)((all + kThreads - 1) / kThreads < 1024 ? (all + kThreads - 1) / kThreads : 1024));
    compact_cache_kernel<P><<<grid, kThreads, 0, stream>>>(c, block_table, bt_width, lengths, path, accepted, most);
    return check_launch("compact_cache");
  });
}

// src, dst int32 [n], rows int32 [n] or null.
extern "C" int nf_copy_pages(void* pages, long long layer_bytes, int layers, int num_pages, int planes, int page_size, int row_bytes,
                             const int* src, const int* dst, const int* rows, int n, cudaStream_t stream) {
  if (n == 0) return 0;
  const PageShape c = {(unsigned char*)pages, layer_bytes, layers, num_pages, planes, page_size, row_bytes};
  if (int rc = check_shape(c)) return rc;
  NF_REQUIRE(n > 0, "copy pages: bad number of pages %d", n);
  return by_piece(c, [&](auto p) {
    using P = decltype(p);
    const long long all = (long long)planes * page_size * row_bytes / (int)sizeof(P);
    const long long x = (all + kThreads * 8 - 1) / (kThreads * 8);
    const dim3 grid(n, (unsigned)(x < 64 ? x : 64), layers < 65535 ? layers : 65535);
    copy_pages_kernel<P><<<grid, kThreads, 0, stream>>>(c, src, dst, rows);
    return check_launch("copy_pages");
  });
}

// 0, or 1 + a request or an entry that did not fit a call since the last time.  Synchronises.
extern "C" int nf_cache_pages_status() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_pages_error, sizeof(int)) != cudaSuccess) return -1;
  if (v) cudaMemcpyToSymbol(g_pages_error, &zero, sizeof(int));
  return v;
}
