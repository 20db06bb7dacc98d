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
// the result).  Scores, weights and sums are float32.  What bounds it is multiply-adds out of shared memory: 2 requests of 12
// nodes behind 1,000 keys, 16 heads of 128, float32: 32 us in a replayed graph, 4 of which the reading of keys and values would
// take.  bfloat16, 27 nodes behind 4,097 keys, 16 query and 4 key heads of 96: 58 us; of 256: 194 (of 128, by mma.sync: 15.5).
#include "tree_attention.cuh"

namespace nf {

__device__ int g_tree_error = 0;

namespace {

constexpr int kThreads = 128;
constexpr int kTile = 32;        // keys at a time: one a lane

// Warp w keeps pairs 4 w .. 4 w + 3 of the CTA's 16; a lane has one key's scores, then every 32nd column of the values.
// Float32 tiles come by asynchronous copies, the next one while one is worked on; bfloat16 ones pass through registers.
template <typename T, int NC>
__global__ void __launch_bounds__(kThreads)
tree_attention_rows_kernel(TreeArgs a, const T* __restrict__ qkv, const T* __restrict__ pages, T* __restrict__ out) {
  constexpr bool ASYNC = sizeof(T) == 4;
  extern __shared__ __align__(16) float smem[];
  const int D = a.D, G = a.Hq / a.Hkv, KS = D + 4;           // (rows of keys 4 floats apart: 16-byte reads of 8 lanes meet no bank twice)
  const int tile = kTile * (KS + D);
  float* Qs = smem;                                          // [16][D]
  float* Ps = Qs + kTreeRows * D;                            // [4 warps][32 keys][4 pairs]
  float* KV = Ps + 4 * kTile * 4;                            // [ASYNC ? 2 : 1 tiles][keys [32][KS], values [32][D]]
  const int of = blockIdx.x / a.shares, share = blockIdx.x % a.shares, s = of / a.Hkv, g = of % a.Hkv;
  const TreeRequest r = tree_request(a, s);
  const int pair0 = blockIdx.z * kTreeRows, pairs = r.nodes * G;
  const int first = share * a.chunk, last = min(first + a.chunk, r.keys);
  if (share == 0 && blockIdx.z == 0 && g == 0 && threadIdx.x == 0 && r.bad) atomicCAS(&g_tree_error, 0, 1 + s);
  if (pair0 >= pairs || (first >= last && (first > 0 || a.shares > 1))) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D4 = D / 4;
  const size_t head = (size_t)a.page_size * D, page_stride = 2 * (size_t)a.Hkv * head;
  // where key `lane` of a tile lies in the pool; -1 for none
  auto source = [&](int k0) -> long long {
    const int j = k0 + lane;
    if (j >= last) return -1;
    const int lp = j / a.page_size, page = lp < a.bt_width ? a.block_table[(size_t)s * a.bt_width + lp] : -1;
    if (page < 0 || page >= a.num_pages) {
      atomicCAS(&g_tree_error, 0, 1 + s);
      return -1;
    }
    return (long long)(page * page_stride + g * head + (size_t)(j - lp * a.page_size) * D);
  };
  auto fetch = [&](float* to, long long mine) {
#pragma unroll 4
    for (int i0 = 0; i0 < kTile * D4; i0 += kThreads) {      // (D is a multiple of 16: all threads have as many pieces)
      const int i = i0 + threadIdx.x, k = i / D4, d = (i - k * D4) * 4;
      const long long from = __shfl_sync(0xffffffffu, mine, k);
      float *tk = to + k * KS + d, *tv = to + kTile * KS + k * D + d;
      const T* p = pages + (from < 0 ? 0 : from + d);
      if constexpr (ASYNC) {
        cp16_or_zeros(tk, (const float*)p, from >= 0);
        cp16_or_zeros(tv, (const float*)(p + (from < 0 ? 0 : (size_t)a.Hkv * head)), from >= 0);
      } else {
        float kv[2][4] = {};
        if (from >= 0) {
          load4(p, kv[0]);
          load4(p + (size_t)a.Hkv * head, kv[1]);
        }
        store4(tk, kv[0]);
        store4(tv, kv[1]);
      }
    }
  };
  long long mine = source(first);
  if constexpr (ASYNC) {
    fetch(KV, mine);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  for (int i = threadIdx.x; i < kTreeRows * D; i += kThreads) {
    const int row = i / D, p = pair0 + row;
    Qs[i] = p < pairs ? to_float(qkv[(size_t)(r.row0 + p / G) * a.q_stride + (size_t)(g * G + p % G) * D + i - row * D]) : 0.f;
  }
  float acc[4][NC], m[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY, l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) acc[i][c] = 0.f;
  }
  const float scale2 = a.scale * 1.4426950408889634f;
  int turn = 0;
  for (int k0 = first; k0 < last; k0 += kTile, turn ^= 1) {
    const long long here = mine;
    mine = source(k0 + kTile);
    float* Ks = KV + (ASYNC ? turn * tile : 0);
    if constexpr (ASYNC) {
      if (k0 + kTile < last) fetch(KV + (turn ^ 1) * tile, mine);            // (that place has been read: see the end of the loop)
      asm volatile("cp.async.commit_group;" ::: "memory");
      asm volatile("cp.async.wait_group 1;" ::: "memory");
    } else {
      fetch(Ks, here);
    }
    __syncthreads();
    const float* Vs = Ks + kTile * KS;
    float x[4] = {};
#pragma unroll 4
    for (int d = 0; d < D; d += 4) {
      const float4 k = *reinterpret_cast<const float4*>(Ks + lane * KS + d);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 q = *reinterpret_cast<const float4*>(Qs + (4 * warp + i) * D + d);
        x[i] = fmaf(q.x, k.x, fmaf(q.y, k.y, fmaf(q.z, k.z, fmaf(q.w, k.w, x[i]))));
      }
    }
    const int j = k0 + lane;
    float v[4], top[4], w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int p = pair0 + 4 * warp + i;
      v[i] = p < pairs && here >= 0 && tree_sees(a, r, p / G, j) ? x[i] * scale2 : -INFINITY;
      top[i] = v[i];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
      for (int i = 0; i < 4; ++i) top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float up = fmaxf(m[i], top[i]), base = up == -INFINITY ? 0.f : up, keep = exp2f(m[i] - base);
      w[i] = exp2f(v[i] - base);
      l[i] = l[i] * keep + w[i];                             // (a lane's own part)
      m[i] = up;
#pragma unroll
      for (int c = 0; c < NC; ++c) acc[i][c] *= keep;
    }
    *reinterpret_cast<float4*>(Ps + (warp * kTile + lane) * 4) = make_float4(w[0], w[1], w[2], w[3]);
    __syncwarp();
    if (k0 + kTile <= r.len) {
#pragma unroll 4
      for (int k = 0; k < kTile; ++k) {
        const float4 w = *reinterpret_cast<const float4*>(Ps + (warp * kTile + k) * 4);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const int d = lane + 32 * c;
          const float v = d < D ? Vs[k * D + d] : 0.f;
          acc[0][c] = fmaf(w.x, v, acc[0][c]), acc[1][c] = fmaf(w.y, v, acc[1][c]), acc[2][c] = fmaf(w.z, v, acc[2][c]), acc[3][c] = fmaf(w.w, v, acc[3][c]);
        }
      }
    } else {
      for (int k = 0; k < kTile; ++k) {
        const float4 w = *reinterpret_cast<const float4*>(Ps + (warp * kTile + k) * 4);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const int d = lane + 32 * c;
          // (a value that a pair does not see may be no number: its weight of nothing must not turn the sum into none)
          const float v = d < D ? Vs[k * D + d] : 0.f;
          acc[0][c] += w.x ? w.x * v : 0.f;
          acc[1][c] += w.y ? w.y * v : 0.f;
          acc[2][c] += w.z ? w.z * v : 0.f;
          acc[3][c] += w.w ? w.w * v : 0.f;
        }
      }
    }
    __syncthreads();                                         // the tile has been read
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
      const size_t at = (size_t)share * a.T * a.Hq + row;
#pragma unroll
      for (int c = 0; c < NC; ++c)
        if (lane + 32 * c < D) a.ws_acc[at * D + lane + 32 * c] = acc[i][c];
      if (lane == 0) reinterpret_cast<float2*>(a.ws_ml)[at] = make_float2(m[i], sum);
    }
  }
}

// Adds up a row's shares in ascending order: WARPS warps a (row, query head), warp w shares w, w + WARPS, ..., whose sums
// then come together.  What a share that the row has not would hold is fetched beside the others and left out: how many it
// has is known only when the request's numbers have come.
template <typename T, int WARPS>
__global__ void __launch_bounds__(128)
tree_attention_merge_kernel(TreeArgs a, T* __restrict__ out) {
  constexpr int AT_ONCE = 8;
  __shared__ float part[WARPS > 1 ? 4 : 1][256 + 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, at = WARPS > 1 ? blockIdx.x : blockIdx.x * 4 + warp;
  const int t = at / a.Hq;
  chain_wait(a.ws_acc, a.ws_ml, a.lengths, a.row0);
  if (at >= a.T * a.Hq) return;                              // (one warp a row: the others go on)
  const int own = WARPS > 1 ? warp : 0, most = (a.shares - own + WARPS - 1) / WARPS;       // shares that this warp looks at
  const size_t step = (size_t)a.T * a.Hq;
  const float2* ml = reinterpret_cast<const float2*>(a.ws_ml) + at;
  auto fetch = [&](int c0, float4 (*v)[2]) {
#pragma unroll
    for (int c = 0; c < AT_ONCE; ++c)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (c0 + c < most && 128 * i + 4 * lane < a.D)
          v[c][i] = *reinterpret_cast<const float4*>(a.ws_acc + ((size_t)(own + WARPS * (c0 + c)) * step + at) * a.D + 128 * i + 4 * lane);
  };
  float4 v[AT_ONCE][2];
  fetch(0, v);
  float2 first = lane < a.shares ? ml[lane * step] : make_float2(-INFINITY, 0.f);          // of all shares, up to 32
  int s = 0;                                                 // the last request that begins at or before the row
  for (int s0 = 1; s0 < a.S; s0 += 32) s += __popc(__ballot_sync(0xffffffffu, s0 + lane < a.S && a.row0[s0 + lane] <= t));
  const TreeRequest r = tree_request(a, s);
  if (t < r.row0 || t >= r.row0 + r.nodes) return;           // a row behind the last request's
  const int shares = (r.keys + a.chunk - 1) / a.chunk;
  if (shares == 1 && a.whole_written) return;
  float m = lane < shares ? first.x : -INFINITY;
  for (int c = 32 + lane; c < shares; c += 32) m = fmaxf(m, ml[c * step].x);
  const float top = warp_max(m), base = top == -INFINITY ? 0.f : top;
  const int n = (shares - own + WARPS - 1) / WARPS;
  float l = 0.f, sum[8] = {};
  for (int c0 = 0; c0 < n; c0 += AT_ONCE) {
    if (c0) fetch(c0, v);
#pragma unroll
    for (int c = 0; c < AT_ONCE; ++c) {
      if (c0 + c >= n) break;
      const int share = own + WARPS * (c0 + c);
      float2 x;
      if (share < 32) x = make_float2(__shfl_sync(0xffffffffu, first.x, share), __shfl_sync(0xffffffffu, first.y, share));
      else x = ml[share * step];
      const float w = exp2f(x.x - base);
      l += w * x.y;
      if (w)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          sum[4 * i] += w * v[c][i].x, sum[4 * i + 1] += w * v[c][i].y, sum[4 * i + 2] += w * v[c][i].z, sum[4 * i + 3] += w * v[c][i].w;
    }
  }
  if constexpr (WARPS > 1) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (128 * i + 4 * lane + k < a.D) part[warp][128 * i + 4 * lane + k] = sum[4 * i + k];
    if (lane == 0) part[warp][256] = l;
    __syncthreads();
    l = (part[0][256] + part[1][256]) + (part[2][256] + part[3][256]);
    for (int d = threadIdx.x; d < a.D; d += 128) {
      const float x = (part[0][d] + part[1][d]) + (part[2][d] + part[3][d]);
      out[(size_t)at * a.D + d] = from_float<T>(l > 0.f ? x / l : (l == 0.f ? 0.f : l));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (128 * i + 4 * lane < a.D) out[(size_t)at * a.D + 128 * i + 4 * lane + k] = from_float<T>(l > 0.f ? sum[4 * i + k] / l : (l == 0.f ? 0.f : l));
  }
}

template <typename T, int NC>
int launch_rows(const TreeArgs& a, const void* qkv, const void* pages, void* out, cudaStream_t stream) {
  const size_t smem = ((size_t)kTreeRows * a.D + 4 * kTile * 4 + (sizeof(T) == 4 ? 2 : 1) * kTile * (2 * a.D + 4)) * sizeof(float);
  if (int rc = allow_smem<tree_attention_rows_kernel<T, NC>>(smem)) return rc;
  const int pairs = (int)min(32ll * a.words, (long long)a.T) * (a.Hq / a.Hkv);
  const long long x = (long long)a.S * a.Hkv * a.shares;
  NF_REQUIRE(x < (1ll << 31), "tree attention: %d requests with %d key heads are too many", a.S, a.Hkv);
  const dim3 grid((unsigned)x, 1, (pairs + kTreeRows - 1) / kTreeRows);
  NF_REQUIRE(grid.y <= 65535 && grid.z <= 65535, "tree attention: %d requests with %d key heads are too many", a.S, a.Hkv);
  tree_attention_rows_kernel<T, NC><<<grid, kThreads, smem, stream>>>(a, (const T*)qkv, (const T*)pages, (T*)out);
  return check_launch("tree_attention_rows");
}

template <typename T>
int launch_merge(const TreeArgs& a, void* out, cudaStream_t stream) {
  if (a.shares == 1) return 0;
  // a warp a row takes eight shares in one trip to memory
  if (a.shares <= 8) launch_chained(tree_attention_merge_kernel<T, 1>, dim3((a.T * a.Hq + 3) / 4), dim3(128), 0, stream, a, (T*)out);
  else launch_chained(tree_attention_merge_kernel<T, 4>, dim3(a.T * a.Hq), dim3(128), 0, stream, a, (T*)out);
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

static bool form_takes(int form, int dtype, int Hkv, int D, int page_size, long long num_pages, bool aligned) {
  if (form == 0) return true;
  return dtype == kBF16 && (D == 64 || D == 128) && aligned && page_size % 16 == 0 && num_pages * 2 * Hkv * page_size < (1ll << 31) &&
         (form == 2 || (form == 1 && tree_tc_fits(D, page_size, num_pages * 2 * Hkv * page_size)));
}

// How a call of these sizes is served: 4 times the keys of a share (of form 1: the CTAs), plus the form: 0 CUDA cores; 1
// tcgen05, 2 mma.sync, both for bfloat16, heads of 64 or 128, pages of a multiple of 16 rows, and queries and results on
// 16-byte boundaries.  Up to 32 pairs a request and key head on average, or where all is little, mma.sync, which is then the
// faster (replayed graphs): 8 requests of up to 32 nodes, 16 key heads, behind 8,192 keys 76 to 80 us and 77 to 83 with tcgen05;
// 32 of 8 nodes, 4 query heads a key head, behind 2,000 47.5 and 53.6; one of 27 nodes, 7 query heads, behind 4,097 16.7 and
// 22.5.  Beyond, the other where pages are 16, 32, 64 or 128 rows: 4 requests of up to 64 nodes, 16 key heads, behind 30,000 144
// and 317; 16 of them, 7 query heads, behind 16,384 224 and 849.  Other pages go by mma.sync with any number of pairs, which reads the cache
// again for each 32 (8 requests of up to 64 nodes, 7 query heads, behind 8,192: pages of 96 rows 269, of 64, on tcgen05, 74);
// what that form does not take either, to CUDA cores (8 of 32, 4 query heads of 96: 729; of 128, on tcgen05, 34).
// `form` from 0 on asks for one; it counts where it takes the sizes.
extern "C" long long nf_tree_attention_plan(int form, int dtype, int S, int T, int Hq, int Hkv, int D, int page_size, long long num_pages, int words,
                                            int max_context, int aligned) {
  const bool asked = form >= 0 && form_takes(form, dtype, Hkv, D, page_size, num_pages, aligned);
  if (!asked) {
    form = form_takes(1, dtype, Hkv, D, page_size, num_pages, aligned) ? 1 : (form_takes(2, dtype, Hkv, D, page_size, num_pages, aligned) ? 2 : 0);
    const long long pairs = ((long long)T * (Hq / Hkv) + S - 1) / S;                 // of a request and key head, on average
    if (form == 1 && (pairs <= 32 || (pairs + 31) / 32 * S * Hkv * ((max_context + 63) / 64) <= 148 * 16)) form = 2;
  }
  if (form == 1) return 4ll * tree_tc_ctas(S, T, Hq, Hkv, words, max_context) + 1;
  if (form == 2) return 4ll * tree_mma_chunk(S, T, Hq, Hkv, max_context) + 2;
  // shares enough that a few hundred CTAs are under way, of 64 keys at least
  const long long pairs = std::min(32ll * words, (long long)T) * (Hq / Hkv);
  const long long ctas = (long long)S * Hkv * ((pairs + kTreeRows - 1) / kTreeRows);
  const long long shares = std::max(1ll, (148 * 4 + ctas - 1) / ctas);
  const long long chunk = ((max_context + shares - 1) / shares + 63) / 64 * 64;
  return 4ll * std::max(64ll, std::min(chunk, 1ll << 20));
}

// Floats of workspace that a call with this plan wants.
extern "C" long long nf_tree_attention_workspace(long long plan, int S, int T, int Hq, int D, int max_context) {
  if ((plan & 3) == 1) return tree_tc_workspace((int)(plan >> 2), S, D);
  const long long shares = (max_context + (plan >> 2) - 1) / (plan >> 2);
  return shares > 1 ? shares * T * Hq * (D + 2) : 0;
}

// A call's operands, 8 bytes each: a caller that packs them at once spares the host a conversion for every argument.
struct TreeCall {
  const void* qkv;
  long long q_stride;
  const void* pages;
  const int* block_table;
  long long bt_width;
  const int *lengths, *row0, *mask;
  long long words;
  void* out;
  float* ws;
  long long S, T, Hq, Hkv, D, page_size, num_pages, max_context, plan;
  double scale;
  long long dtype;
  cudaStream_t stream;
};

// qkv [T, q_stride] with the queries in its first Hq * D columns; pages [num_pages, 2, Hkv, page_size, D]; block_table int32
// [S, bt_width]; lengths int32 [S], row0 int32 [S + 1], mask int32 [T, words]; out [T, Hq * D]: rows that no request has
// stay as they are.  max_context: no request has more keys, its nodes' among them.  plan, ws: see nf_tree_attention_plan
// and nf_tree_attention_workspace.
extern "C" int nf_tree_attention(const TreeCall* call) {
  const TreeCall& c = *call;
  const void *qkv = c.qkv, *pages = c.pages;
  void* out = c.out;
  const long long q_stride = c.q_stride, plan = c.plan;
  const int *block_table = c.block_table, *lengths = c.lengths, *row0 = c.row0, *mask = c.mask;
  float* ws = c.ws;
  const int bt_width = (int)c.bt_width, words = (int)c.words, S = (int)c.S, T = (int)c.T, Hq = (int)c.Hq, Hkv = (int)c.Hkv, D = (int)c.D,
            page_size = (int)c.page_size, num_pages = (int)c.num_pages, max_context = (int)c.max_context, dtype = (int)c.dtype;
  const float scale = (float)c.scale;
  cudaStream_t stream = c.stream;
  if (S == 0 || T == 0) return 0;
  const int form = (int)(plan & 3), chunk = (int)(plan >> 2);
  NF_REQUIRE(S > 0 && T > 0 && Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && D > 0 && D % 16 == 0 && D <= 256 && page_size > 0 && num_pages > 0 &&
                 bt_width > 0 && words > 0 && max_context > 0 && chunk > 0 && q_stride >= (long long)Hq * D && (long long)T * Hq < (1ll << 31),
             "tree attention: bad sizes S=%d T=%d Hq=%d Hkv=%d D=%d page=%d", S, T, Hq, Hkv, D, page_size);
  NF_REQUIRE(dtype == kF32 || dtype == kBF16, "tree attention: unknown type %d", dtype);
  NF_REQUIRE((uintptr_t)pages % 16 == 0, "tree attention: pages must be 16-byte aligned");
  const int shares = form == 1 ? 1 : (max_context + chunk - 1) / chunk;
  NF_REQUIRE(form == 1 ? chunk <= 148 && (chunk == 1 || ws) : shares == 1 || ws, "tree attention: shares of keys want a workspace");
  float* ws_ml = ws ? ws + (size_t)shares * T * Hq * D : nullptr;
  const int G = Hq / Hkv;
  NF_REQUIRE(G < 4096, "tree attention: %d query heads a key head are too many", G);
  TreeArgs a = {block_table, lengths, row0, mask, ws, ws_ml, nullptr, q_stride, bt_width, words, S, T, Hq, Hkv, D, page_size, num_pages, max_context,
                chunk, shares, form != 0, scale, G == 1 ? 0u : (unsigned)(((1ull << 32) + G - 1) / G)};
  if (form) {
    const bool aligned = (uintptr_t)qkv % 16 == 0 && q_stride % 8 == 0 && (uintptr_t)out % 16 == 0;
    NF_REQUIRE(form_takes(form, dtype, Hkv, D, page_size, num_pages, aligned) && (form == 1 || chunk % 128 == 0),
               "tree attention: sizes that form %d does not take (D=%d page=%d)", form, D, page_size);
    if (form == 1) return launch_tree_tc(a, chunk, ws, qkv, pages, out, stream);
    if (int rc = launch_tree_mma(a, qkv, pages, out, stream)) return rc;
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
