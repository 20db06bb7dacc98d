// Attention of trees of drafted tokens over the paged cache, on CUDA cores in float32: float32 tensors, and bfloat16 ones
// of head sizes that the tensor-core form does not take.
//
// Request s holds len keys (lengths[s]) and brings n = row0[s + 1] - row0[s] nodes, whose keys and values lie in its pages
// behind those, node i's at position len + i.  Row row0[s] + i sees every key j < len, and key len + k where bit k of its
// mask is set:
//
//   out[t, h] = sum_j softmax_j(scale q[t, h] . k[j, g]) v[j, g],   g = h / (Hq / Hkv);   0 where a row sees no key
//
// All nodes of a request read the same keys, so a CTA takes 16 (node, query head) pairs of one key head and a share of
// `chunk` keys.  Shares begin at multiples of `chunk`; each leaves an unnormalised sum with its maximum and its
// weights' sum, and a second kernel adds a row's shares up in ascending order (with one share the first kernel writes
// the result).  Scores, weights and sums are float32.
#include "tree_attention.cuh"

namespace nf {

__device__ int g_tree_error = 0;

namespace {

constexpr int kThreads = 128;
constexpr int kTile = 32;        // keys at a time: one a lane

// Warp w keeps pairs 4 w .. 4 w + 3 of the CTA's 16; a lane has one key's scores, then every 32nd column of the values.
template <typename T, int NC>
__global__ void __launch_bounds__(kThreads)
tree_attention_rows_kernel(TreeArgs a, const T* __restrict__ qkv, const T* __restrict__ pages, T* __restrict__ out) {
  extern __shared__ __align__(16) float smem[];
  const int D = a.D, G = a.Hq / a.Hkv, KS = D + 4;           // (rows of keys 4 floats apart: 16-byte reads of 8 lanes meet no bank twice)
  float* Qs = smem;                                          // [16][D]
  float* Ks = Qs + kTreeRows * D;                            // [32][KS]
  float* Vs = Ks + kTile * KS;                               // [32][D]
  float* Ps = Vs + kTile * D;                                // [4 warps][32 keys][4 pairs]
  __shared__ int key_page[kTile];
  const int s = blockIdx.y / a.Hkv, g = blockIdx.y % a.Hkv;
  const TreeRequest r = tree_request(a, s);
  const int pair0 = blockIdx.z * kTreeRows, pairs = r.nodes * G;
  const int first = blockIdx.x * a.chunk, last = min(first + a.chunk, r.keys);
  if (blockIdx.x == 0 && blockIdx.z == 0 && g == 0 && threadIdx.x == 0 && r.bad) atomicCAS(&g_tree_error, 0, 1 + s);
  if (pair0 >= pairs || (first >= last && (first > 0 || a.shares > 1))) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < kTreeRows * D; i += kThreads) {
    const int p = pair0 + i / D;
    Qs[i] = p < pairs ? to_float(qkv[(size_t)(r.row0 + p / G) * a.q_stride + (size_t)(g * G + p % G) * D + i % D]) : 0.f;
  }
  const size_t head = (size_t)a.page_size * D, page_stride = 2 * (size_t)a.Hkv * head;
  float acc[4][NC], m[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY, l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) acc[i][c] = 0.f;
  }
  const float scale2 = a.scale * 1.4426950408889634f;
  for (int k0 = first; k0 < last; k0 += kTile) {
    __syncthreads();                                         // the tile before has been read
    if (threadIdx.x < kTile) {
      const int j = k0 + threadIdx.x;
      int page = -1;
      if (j < last) {
        const int lp = j / a.page_size;
        page = lp < a.bt_width ? a.block_table[(size_t)s * a.bt_width + lp] : -1;
        if (page < 0 || page >= a.num_pages) {
          page = -1;
          atomicCAS(&g_tree_error, 0, 1 + s);
        }
      }
      key_page[threadIdx.x] = page;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kTile * D / 4; i += kThreads) {
      const int k = i / (D / 4), d = i % (D / 4) * 4, page = key_page[k];
      float kv[2][4] = {};
      if (page >= 0) {
        const T* p = pages + (size_t)page * page_stride + (size_t)g * head + (size_t)((k0 + k) % a.page_size) * D + d;
        load4(p, kv[0]);
        load4(p + (size_t)a.Hkv * head, kv[1]);
      }
      store4(Ks + k * KS + d, kv[0]);
      store4(Vs + k * D + d, kv[1]);
    }
    __syncthreads();
    float x[4] = {};
    for (int d = 0; d < D; d += 4) {
      const float4 k = *reinterpret_cast<const float4*>(Ks + lane * KS + d);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 q = *reinterpret_cast<const float4*>(Qs + (4 * warp + i) * D + d);
        x[i] = fmaf(q.x, k.x, fmaf(q.y, k.y, fmaf(q.z, k.z, fmaf(q.w, k.w, x[i]))));
      }
    }
    const int j = k0 + lane;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int p = pair0 + 4 * warp + i;
      const bool seen = p < pairs && key_page[lane] >= 0 && tree_sees(a, r, p / G, j);
      const float v = seen ? x[i] * scale2 : -INFINITY, top = fmaxf(m[i], warp_max(v));
      const float base = top == -INFINITY ? 0.f : top, keep = exp2f(m[i] - base);
      const float w = exp2f(v - base);
      l[i] = l[i] * keep + w;                                // (a lane's own part)
      m[i] = top;
#pragma unroll
      for (int c = 0; c < NC; ++c) acc[i][c] *= keep;
      Ps[(warp * kTile + lane) * 4 + i] = w;
    }
    __syncwarp();
    for (int k = 0; k < kTile; ++k) {
      const float4 w = *reinterpret_cast<const float4*>(Ps + (warp * kTile + k) * 4);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int d = lane + 32 * c;
        // (a value that no pair of the warp sees may be no number: its weight of nothing must not turn the sum into none)
        const float v = d < D ? Vs[k * D + d] : 0.f;
        acc[0][c] += w.x ? w.x * v : 0.f;
        acc[1][c] += w.y ? w.y * v : 0.f;
        acc[2][c] += w.z ? w.z * v : 0.f;
        acc[3][c] += w.w ? w.w * v : 0.f;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int p = pair0 + 4 * warp + i;
    const float sum = warp_sum(l[i]);
    if (p >= pairs) continue;
    const size_t row = (size_t)(r.row0 + p / G) * a.Hq + g * G + p % G;
    if (a.shares == 1) {
#pragma unroll
      for (int c = 0; c < NC; ++c)
        if (lane + 32 * c < D) out[row * D + lane + 32 * c] = from_float<T>(sum > 0.f ? acc[i][c] / sum : (sum == 0.f ? 0.f : sum));
    } else {
      const size_t at = (size_t)blockIdx.x * a.T * a.Hq + row;
#pragma unroll
      for (int c = 0; c < NC; ++c)
        if (lane + 32 * c < D) a.ws_acc[at * D + lane + 32 * c] = acc[i][c];
      if (lane == 0) reinterpret_cast<float2*>(a.ws_ml)[at] = make_float2(m[i], sum);
    }
  }
}

// One warp a (row, query head): its request's shares in ascending order.
template <typename T>
__global__ void __launch_bounds__(128)
tree_attention_merge_kernel(TreeArgs a, T* __restrict__ out) {
  const int at = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  chain_wait(a.ws_acc, a.ws_ml, a.lengths, a.row0);
  if (at >= a.T * a.Hq) return;
  const int t = at / a.Hq;
  int lo = 0, hi = a.S;                                      // the last request that begins at or before the row
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (a.row0[mid] <= t) lo = mid; else hi = mid;
  }
  const TreeRequest r = tree_request(a, lo);
  if (t < r.row0 || t >= r.row0 + r.nodes) return;           // a row behind the last request's
  const int shares = (r.keys + a.chunk - 1) / a.chunk;
  if (shares == 1 && a.whole_written) return;
  const size_t step = (size_t)a.T * a.Hq;
  const float2* ml = reinterpret_cast<const float2*>(a.ws_ml) + at;
  float m = -INFINITY;
  for (int c = lane; c < shares; c += 32) m = fmaxf(m, ml[c * step].x);
  const float top = warp_max(m), base = top == -INFINITY ? 0.f : top;
  float l = 0.f, sum[8] = {};
  for (int c0 = 0; c0 < shares; c0 += 32) {
    float w = 0.f;                                           // of share c0 + lane
    if (c0 + lane < shares) {
      const float2 v = ml[(c0 + lane) * step];
      w = exp2f(v.x - base);
      l += w * v.y;
    }
    const int n = min(32, shares - c0);
#pragma unroll 4
    for (int c = 0; c < n; ++c) {
      const float wc = __shfl_sync(0xffffffffu, w, c);
      const float* acc = a.ws_acc + ((c0 + c) * step + at) * a.D;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (128 * i + 4 * lane < a.D) {
          const float4 v = *reinterpret_cast<const float4*>(acc + 128 * i + 4 * lane);
          if (wc) sum[4 * i] += wc * v.x, sum[4 * i + 1] += wc * v.y, sum[4 * i + 2] += wc * v.z, sum[4 * i + 3] += wc * v.w;
        }
    }
  }
  l = warp_sum(l);
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int d = 128 * i + 4 * lane + k;
      if (d < a.D) out[(size_t)at * a.D + d] = from_float<T>(l > 0.f ? sum[4 * i + k] / l : (l == 0.f ? 0.f : l));
    }
}

template <typename T, int NC>
int launch_rows(const TreeArgs& a, const void* qkv, const void* pages, void* out, cudaStream_t stream) {
  const size_t smem = ((size_t)kTreeRows * a.D + kTile * (2 * a.D + 4) + 4 * kTile * 4) * sizeof(float);
  if (int rc = allow_smem((const void*)tree_attention_rows_kernel<T, NC>, smem)) return rc;
  const int pairs = (int)min(32ll * a.words, (long long)a.T) * (a.Hq / a.Hkv);
  const dim3 grid(a.shares, a.S * a.Hkv, (pairs + kTreeRows - 1) / kTreeRows);
  NF_REQUIRE(grid.y <= 65535 && grid.z <= 65535, "tree attention: %d requests with %d key heads are too many", a.S, a.Hkv);
  tree_attention_rows_kernel<T, NC><<<grid, kThreads, smem, stream>>>(a, (const T*)qkv, (const T*)pages, (T*)out);
  return check_launch("tree_attention_rows");
}

template <typename T>
int launch_merge(const TreeArgs& a, void* out, cudaStream_t stream) {
  if (a.shares == 1) return 0;
  launch_chained(tree_attention_merge_kernel<T>, dim3((a.T * a.Hq + 3) / 4), dim3(128), 0, stream, a, (T*)out);
  return check_launch("tree_attention_merge");
}

template <typename T>
int launch_rows_of(const TreeArgs& a, const void* qkv, const void* pages, void* out, cudaStream_t stream) {
  if (a.D <= 64) return launch_rows<T, 2>(a, qkv, pages, out, stream);
  if (a.D <= 128) return launch_rows<T, 4>(a, qkv, pages, out, stream);
  return launch_rows<T, 8>(a, qkv, pages, out, stream);
}

}  // namespace
}  // namespace nf

using namespace nf;

// Whether the tensor-core form takes these sizes: bfloat16, heads of 64 or 128, whole pages a block of 128 keys, queries on
// 16-byte boundaries.
extern "C" int nf_tree_attention_tensor(int dtype, int Hkv, int D, int page_size, long long num_pages, const void* qkv, long long q_stride) {
  return dtype == kBF16 && tree_tc_fits(D, page_size, num_pages * 2 * Hkv * page_size) && (uintptr_t)qkv % 16 == 0 && q_stride % 8 == 0;
}

// Keys a share takes, for calls of these sizes; the workspace is a float for every (share, row, query head, D + 2).
extern "C" int nf_tree_attention_chunk(int S, int T, int Hq, int Hkv, int words, int max_context, int tensor) {
  if (tensor) return tree_tc_chunk(S, T, Hq, Hkv, words, max_context);
  // shares enough that a few hundred CTAs are under way, of 64 keys at least
  const long long pairs = std::min(32ll * words, (long long)T) * (Hq / Hkv);
  const long long ctas = (long long)S * Hkv * ((pairs + kTreeRows - 1) / kTreeRows);
  const long long shares = std::max(1ll, (148 * 4 + ctas - 1) / ctas);
  const long long chunk = ((max_context + shares - 1) / shares + 63) / 64 * 64;
  return (int)std::max(64ll, std::min(chunk, 1ll << 20));
}

// qkv [T, q_stride] with the queries in its first Hq * D columns; pages [num_pages, 2, Hkv, page_size, D]; block_table int32
// [S, bt_width]; lengths int32 [S], row0 int32 [S + 1], mask int32 [T, words]; out [T, Hq * D]: rows that no request has
// stay as they are.  max_context: no request has more keys, its nodes' among them.  ws: see nf_tree_attention_chunk; none
// where one share takes all keys.
extern "C" int nf_tree_attention(const void* qkv, long long q_stride, const void* pages, const int* block_table, int bt_width,
                                 const int* lengths, const int* row0, const int* mask, int words, void* out, float* ws, int S, int T,
                                 int Hq, int Hkv, int D, int page_size, int num_pages, int max_context, int chunk, int tensor, float scale,
                                 int dtype, cudaStream_t stream) {
  if (S == 0 || T == 0) return 0;
  NF_REQUIRE(S > 0 && T > 0 && Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && D > 0 && D % 16 == 0 && D <= 256 && page_size > 0 && num_pages > 0 &&
                 bt_width > 0 && words > 0 && max_context > 0 && chunk > 0 && q_stride >= (long long)Hq * D && (long long)T * Hq < (1ll << 31),
             "tree attention: bad sizes S=%d T=%d Hq=%d Hkv=%d D=%d page=%d", S, T, Hq, Hkv, D, page_size);
  NF_REQUIRE(dtype == kF32 || dtype == kBF16, "tree attention: unknown type %d", dtype);
  NF_REQUIRE((uintptr_t)pages % 16 == 0, "tree attention: pages must be 16-byte aligned");
  const int shares = (max_context + chunk - 1) / chunk;
  NF_REQUIRE(shares == 1 || ws, "tree attention: %d shares of keys want a workspace", shares);
  float* ws_ml = ws ? ws + (size_t)shares * T * Hq * D : nullptr;
  TreeArgs a = {block_table, lengths, row0, mask, ws, ws_ml, q_stride, bt_width, words, S, T, Hq, Hkv, D, page_size, num_pages, max_context,
                chunk, shares, tensor, scale};
  if (tensor) {
    NF_REQUIRE(nf_tree_attention_tensor(dtype, Hkv, D, page_size, num_pages, qkv, q_stride) && chunk % 128 == 0 && (uintptr_t)out % 16 == 0,
               "tree attention: sizes the tensor-core form does not take (D=%d page=%d)", D, page_size);
    if (int rc = launch_tree_tc(a, qkv, pages, out, stream)) return rc;
  } else if (int rc = dtype == kF32 ? launch_rows_of<float>(a, qkv, pages, out, stream) : launch_rows_of<__nv_bfloat16>(a, qkv, pages, out, stream)) {
    return rc;
  }
  return dtype == kF32 ? launch_merge<float>(a, out, stream) : launch_merge<__nv_bfloat16>(a, out, stream);
}

// 0, or 1 + a request of which lengths, rows or pages did not fit a call since the last time.  Synchronises.
extern "C" int nf_tree_attention_status() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_tree_error, sizeof(int)) != cudaSuccess) return -1;
  if (v) cudaMemcpyToSymbol(g_tree_error, &zero, sizeof(int));
  return v;
}
