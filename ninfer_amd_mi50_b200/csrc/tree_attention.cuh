// What the kernels of tree attention share: a request's rows and keys, which of them a row sees, and the host's side of
// shared memory beyond 48 KB.
#pragma once

#include <algorithm>
#include <atomic>

#include "common.cuh"

namespace nf {

constexpr int kTreeRows = 16;     // (node, query head) pairs of a CTA on CUDA cores

struct TreeArgs {
  const int *block_table, *lengths, *row0, *mask;
  float *ws_acc, *ws_ml;          // [shares][T][Hq][D], [shares][T][Hq][2]
  long long* ws_line;             // the tensor-core form's own: see tree_attention_tc.cu
  long long q_stride;
  int bt_width, words, S, T, Hq, Hkv, D, page_size, num_pages, max_context, chunk, shares;
  int whole_written;              // a request with one share has its result from the first kernel
  float scale;
  unsigned inverse_heads;         // 2^32 / (Hq / Hkv), rounded up: see node_of
};

// Pair p's node, p / (Hq / Hkv).  The inverse is at most 1 too large, which at p below 2^20 (256 nodes of 4,095 heads) stays
// below 2^-12 of a node, less than a pair's part; one query head a key head has no inverse in 32 bits.
__device__ __forceinline__ int node_of(const TreeArgs& a, int p) { return a.inverse_heads ? (int)__umulhi((unsigned)p, a.inverse_heads) : p; }

struct TreeRequest {
  int row0, nodes, len, keys;     // its rows, the keys it held, these and its nodes'
  bool bad;
};

// What the tensors say of request s, brought into the bounds that the call gave.
__device__ __forceinline__ TreeRequest tree_request(const TreeArgs& a, int s) {
  TreeRequest r;
  const int begin = a.row0[s], end = a.row0[s + 1], len = a.lengths[s];
  r.row0 = min(max(begin, 0), a.T);
  r.nodes = min(min(max(end, r.row0), a.T) - r.row0, 32 * a.words);
  r.len = min(max(len, 0), a.max_context);
  r.keys = min(r.len + r.nodes, a.max_context);      // (both below 2^30: see the call)
  r.bad = begin < 0 || end < begin || end > a.T || end - begin > 32 * a.words || len < 0 || len > a.max_context - r.nodes;
  return r;
}

// Whether node i of the request sees key j < r.keys.
__device__ __forceinline__ bool tree_sees(const TreeArgs& a, const TreeRequest& r, int i, int j) {
  const int k = j - r.len;
  return k < 0 || (a.mask[(size_t)(r.row0 + i) * a.words + (k >> 5)] >> (k & 31) & 1);
}

// The tensor-core form (tree_attention_tc.cu).
bool tree_tc_fits(int D, int page_size, long long page_rows);
int tree_tc_ctas(int S, int T, int Hq, int Hkv, int words, int max_context);
long long tree_tc_workspace(int ctas, int S, int D);
int launch_tree_tc(TreeArgs a, int ctas, float* ws, const void* qkv, const void* pages, void* out, cudaStream_t stream);
// The form for few pairs (tree_attention_mma.cu).
int tree_mma_chunk(int S, int T, int Hq, int Hkv, int max_context);
int launch_tree_mma(const TreeArgs& a, const void* qkv, const void* pages, void* out, cudaStream_t stream);

// Lets KERNEL have `bytes` of dynamic shared memory, asked for once a device (the question takes the host as long as a launch).
template <auto KERNEL>
inline int allow_smem(size_t bytes) {
  static std::atomic<size_t> had[64];
  if (bytes <= 48 * 1024) return 0;
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  const bool known = e == cudaSuccess && device >= 0 && device < 64;
  if (known && had[device].load(std::memory_order_relaxed) >= bytes) return 0;
  if (e == cudaSuccess) e = cudaFuncSetAttribute((const void*)KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e != cudaSuccess) (void)cudaGetLastError();
  NF_REQUIRE(e == cudaSuccess, "cannot have %zu bytes of shared memory: %s", bytes, cudaGetErrorString(e));
  if (known) had[device].store(bytes, std::memory_order_relaxed);
  return 0;
}

}  // namespace nf
