// Attention of trees of drafted tokens in bfloat16 where a key head's (node, query head) pairs are few
// (tree_attention.cu says what is computed): what counts is then reading keys and values, and how soon.
//
// A CTA takes 16 or 32 pairs of a (request, key head) and a share of the keys, 64 at a time: the first of its four warps
// asks for them by TMA, page by page (128-byte swizzle), two stages ahead in a ring of three; each warp takes 16 of the 64
// keys.  (A fifth warp for the copies would leave the others 168 registers, too few beside 32 rows of sums.)  A warp's step is the
// usual flash step: S = Q K^T and O += P V by ``mma.sync.m16n8k16`` with the pairs as the 16 rows, a reference maximum that
// is raised only when a score passes it by 8 in the exponent, weights rounded to bfloat16 in between (2^-8 of one at most,
// as independent from key to key as the rounding of the result, so that the result is 1.4 times as far from the 64-bit one
// as its own rounding puts it; their sum is of the unrounded ones).  With 16 pairs a CTA a weight goes into the second
// product as two numbers, its rounding and what that left, which costs 5 % there; with 32 it would be 10 %.  At the end the
// sums of the four warps are put together in shared memory.
//
// The tensor cores' newer form (tree_attention_tc.cu) wants 128 rows at once and a chain of copies, products and softmax a
// block of 128 keys; with few pairs most of that is waiting.
//
// What bounds it: a warp's step is a chain of ldmatrix, products, exponentials and products, 0.85 us with 32 pairs, and two CTAs
// an SM hide some of each other's.  8 requests of up to 32 nodes behind up to 8,192 keys, 16 key heads: 76 us in a replayed
// graph, 5.2 TB/s while the first kernel runs (80 % of what a copy reaches); one of 27 nodes behind 4,097, 28 query heads: 16.7 us.
// A word a stage says which of its boxes have a page (1 to 2 % of this; found out once by all threads it was as much).
#include "tcgen05.cuh"
#include "tree_attention.cuh"

namespace nf {
namespace {

constexpr int kGroups = 4;              // 16 keys each
constexpr int kStageKeys = 16 * kGroups;
constexpr int kStages = 3;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRaise = 8.f;
constexpr int kThreads = 32 * kGroups;

__device__ int g_tree_mma_wait = 0;
__device__ int g_tree_mma_error = 0;

__device__ __forceinline__ void ldsm4(unsigned* r, unsigned at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldsm4t(unsigned* r, unsigned at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void mma(float* c, const unsigned* a, unsigned b0, unsigned b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ unsigned pack(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const unsigned*>(&v);
}

__device__ __forceinline__ unsigned pack_two(float x, float y, unsigned& rest) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
  rest = pack(x - __low2float(v), y - __high2float(v));
  return *reinterpret_cast<const unsigned*>(&v);
}

struct __align__(8) Ring {
  unsigned long long full[kStages], empty[kStages];
  unsigned here[kStages];               // bit i: the stage's i-th box has a page; in the place of others lies what lay there before
  int stop;
};

template <int D> constexpr int stage_bytes() { return 2 * kStageKeys * D * 2; }
// the ring, at the end the warps' sums [4][rows][4 lanes][D / 4 + 4] in its place; queries; maxima and sums; barriers
template <int D, int MT> constexpr size_t smem_bytes() {
  const size_t ring = (size_t)kStages * stage_bytes<D>(), sums = (size_t)kGroups * 16 * MT * (D + 16) * 4;
  return 1024 + (ring > sums ? ring : sums) + 16 * MT * D * 2 + kGroups * 16 * MT * sizeof(float2) + sizeof(Ring);
}

// MT times 16 pairs; warp w takes the keys 16 w .. of every stage.
template <int D, int MT>
__global__ void __launch_bounds__(kThreads, 2)
tree_attention_mma_kernel(const __grid_constant__ CUtensorMap map_kv, const __grid_constant__ TreeArgs a, int box_rows, int page_shift,
                          const __nv_bfloat16* __restrict__ qkv, __nv_bfloat16* __restrict__ out) {
  constexpr int ROWS = 16 * MT, PIECES = D / 8, ATOMS = D / 64, SB = stage_bytes<D>(), OL = D / 4 + 4, OS = 4 * OL, PARTS = MT == 1 ? 2 : 1, AB = kStageKeys * 128;     // AB: 64 numbers of the stage's keys
  constexpr size_t kRing = (size_t)kStages * SB, kSums = (size_t)kGroups * ROWS * OS * 4;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + (-smem_u32(smem_raw) & 1023u);          // (an offset, so that what lies here is known to be shared memory)
  unsigned char* Qs = smem + (kRing > kSums ? kRing : kSums);
  float2* stat = reinterpret_cast<float2*>(Qs + ROWS * D * 2);
  Ring* ring = reinterpret_cast<Ring*>(stat + kGroups * ROWS);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int s = blockIdx.x / a.Hkv, g = blockIdx.x % a.Hkv, G = a.Hq / a.Hkv;
  const int first = blockIdx.y * a.chunk;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&ring->full[i], 1);
      mbar_init(&ring->empty[i], kGroups);
    }
    ring->stop = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  chain_wait(qkv);
  const int* bt = a.block_table + (size_t)s * a.bt_width;
  // the first pages, on their way beside the request's numbers: lane i that of the i-th box
  int page = -1;
  const auto look_up = [&](int key) {
    const int lp = page_shift >= 0 ? key >> page_shift : key / a.page_size;
    return lp < a.bt_width ? bt[lp] : -1;
  };
  if (warp == 0 && (long long)first + box_rows * lane < a.max_context) page = look_up(first + box_rows * lane);
  const TreeRequest r = tree_request(a, s);
  if (r.bad && blockIdx.y == 0 && blockIdx.z == 0 && g == 0 && threadIdx.x == 0) atomicCAS(&g_tree_mma_error, 0, 1 + s);
  const int pair0 = blockIdx.z * ROWS, pairs = r.nodes * G;
  const int last = min(first + a.chunk, r.keys);
  if (pair0 >= pairs || first >= last) return;
  const int steps = (last - first + kStageKeys - 1) / kStageKeys;
  volatile int* stop = &ring->stop;
  // a stage's keys and values, by the first warp: 32 boxes are looked up at a time, lane i the i-th
  const int per = kStageKeys / box_rows, serves = 32 / per;                // boxes a stage, stages that a look-up serves
  auto fetch = [&](int i) -> bool {
    const int st = i % kStages, key0 = first + kStageKeys * i, from = i % serves * per;
    if (i % serves == 0 && i > 0) {
      const int key = key0 + box_rows * lane;
      page = key < last ? look_up(key) : -1;
    }
    const int at = (lane - from) * box_rows;
    const bool wanted = lane >= from && lane < from + per && key0 + at < last, there = wanted && page >= 0 && page < a.num_pages;
    if (wanted && !there) atomicCAS(&g_tree_mma_error, 0, 1 + s);
    const unsigned boxes = __ballot_sync(0xffffffffu, there);
    if (!__all_sync(0xffffffffu, mbar_wait(&ring->empty[st], ((i / kStages) & 1) ^ 1, stop, 1, &g_tree_mma_wait))) return false;
    if (elect_one()) {
      ((volatile Ring*)ring)->here[st] = boxes >> from;
      mbar_expect_tx(&ring->full[st], (unsigned)__popc(boxes) * 2 * box_rows * D * 2);
    }
    __syncwarp();
    if (there) {                                             // each lane its box of keys and of values
      const int in_page = page_shift >= 0 ? (key0 + at) & (a.page_size - 1) : (key0 + at) % a.page_size;
      const int y = (page * 2 * a.Hkv + g) * a.page_size + in_page;
      unsigned char* to = smem + (size_t)st * SB + at * 128;
#pragma unroll
      for (int x = 0; x < ATOMS; ++x) {
        tma_load_2d(to + x * AB, &map_kv, 64 * x, y, &ring->full[st]);
        tma_load_2d(to + SB / 2 + x * AB, &map_kv, 64 * x, y + a.Hkv * a.page_size, &ring->full[st]);
      }
    }
    __syncwarp();
    return true;
  };
  int issued = 0;
  if (warp == 0)                                             // (the barriers are this thread's own to begin with: thread 0 made them)
    for (; issued < min(steps, kStages - 1); ++issued) {
      __syncwarp();
      fetch(issued);
    }
  {                                                          // queries: [row][D], a row's 16-byte pieces exchanged by its number
    constexpr int EACH = ROWS * PIECES / kThreads, PER = PIECES / EACH;    // pieces a thread, threads a row
    const int row = threadIdx.x / PER, c0 = threadIdx.x % PER, p = pair0 + row, node = node_of(a, p);
    const uint4* q = reinterpret_cast<const uint4*>(qkv + (size_t)(p < pairs ? r.row0 + node : 0) * a.q_stride + (size_t)(g * G + p - node * G) * D);
    uint4 v[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) v[i] = p < pairs ? q[c0 + PER * i] : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < EACH; ++i) *reinterpret_cast<uint4*>(Qs + row * D * 2 + (((c0 + PER * i) ^ (row & 7)) << 4)) = v[i];
  }
  __syncthreads();
  float o[MT][D / 8][4], m_run[MT][2], l_run[MT][2];
  const int group = warp, quad = lane >> 2, t4 = lane & 3;
  {
    const float sc2 = a.scale * kLog2e;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      m_run[m][0] = m_run[m][1] = -INFINITY, l_run[m][0] = l_run[m][1] = 0.f;
#pragma unroll
      for (int n = 0; n < D / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[m][n][i] = 0.f;
    }
    // where this lane's row of the matrices lies that an ldmatrix fetches side by side: 4 places in an atom's row, pieces
    // exchanged.  Keys: rows of 8 keys, then 8 more numbers; values: 8 more keys, then rows of 8 numbers; queries: 16 rows,
    // then 8 more numbers.
    const int lr = (lane & 7) + ((lane >> 4) << 3), lc = (lane >> 3) & 1, vr = (lane & 7) + (((lane >> 3) & 1) << 3), vc = lane >> 4;
    unsigned key_at[4], value_at[4], query_at[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      key_at[k] = smem_u32(smem) + (16 * group + lr) * 128 + (((2 * k + lc) ^ (lr & 7)) << 4);
      value_at[k] = smem_u32(smem) + SB / 2 + (16 * group + vr) * 128 + (((2 * k + vc) ^ (vr & 7)) << 4);
      query_at[k] = smem_u32(Qs) + (lane & 15) * D * 2 + (((2 * k + vc) ^ (lane & 7)) << 4);
    }
    const unsigned own_box = 1u << 16 * group / box_rows;    // of a stage, the one that the warp's 16 keys lie in
    unsigned stage = 0;
    int st = 0;
    unsigned parity = 0;
    for (int i = 0; i < steps; ++i) {
      const int k0 = first + kStageKeys * i + 16 * group;
      if (warp == 0 && issued < steps) {
        if (!fetch(issued)) break;
        ++issued;
      }
      if (!__all_sync(0xffffffffu, mbar_wait(&ring->full[st], parity, stop, 2, &g_tree_mma_wait))) break;
      if (k0 < last) {
        const bool gone = !(((volatile Ring*)ring)->here[st] & own_box);     // keys without a page: no row sees them
        float c[MT][2][4] = {};
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          unsigned b[4];
          ldsm4(b, key_at[k & 3] + stage + (k >> 2) * AB);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            unsigned q[4];
            ldsm4(q, query_at[k & 3] + 16 * m * D * 2 + (k >> 2) * 128);
            mma(c[m][0], q, b[0], b[1]);
            mma(c[m][1], q, b[2], b[3]);
          }
        }
        if (k0 + 16 > r.len || gone) {                       // (else keys that every row sees)
          const int from = k0 - r.len;                       // the tree's node at the tile's first key
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int p = pair0 + 16 * m + quad + 8 * h;
              unsigned seen = 0;                             // bit i: key k0 + i
              if (p < pairs && !gone) {
                const int* words = a.mask + (size_t)(r.row0 + node_of(a, p)) * a.words;
                const int w = from >> 5;                     // (-1 for keys that the request held)
                const unsigned lo = w < 0 ? ~0u : (unsigned)words[w], hi = w + 1 < a.words ? (unsigned)words[w + 1] : 0u;
                seen = __funnelshift_r(lo, hi, from & 31);
                if (last - k0 < 16) seen &= (1u << (last - k0)) - 1;
              }
#pragma unroll
              for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int x = 0; x < 2; ++x)
                  if (!(seen >> (8 * n + 2 * t4 + x) & 1)) c[m][n][2 * h + x] = -INFINITY;
            }
          // values behind the last key, or without a page: whatever lies there would be multiplied by a weight of nothing
          for (int e = lane; e < 16 * PIECES; e += 32)
            if (k0 + e / PIECES >= last || gone)
              *reinterpret_cast<uint4*>(smem + stage + SB / 2 + (e % PIECES >> 3) * AB + (16 * group + e / PIECES) * 128 + (e & 7) * 16) = make_uint4(0, 0, 0, 0);
          if (gone) fence_async_smem();                      // (a later stage's copy may take their place)
          __syncwarp();
        }
        float top[MT][2];
        bool raise = false;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h) top[m][h] = fmaxf(fmaxf(c[m][0][2 * h], c[m][0][2 * h + 1]), fmaxf(c[m][1][2 * h], c[m][1][2 * h + 1]));
#pragma unroll
        for (int x = 1; x < 4; x *= 2)
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) top[m][h] = fmaxf(top[m][h], __shfl_xor_sync(0xffffffffu, top[m][h], x));
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h) raise |= top[m][h] * sc2 > m_run[m][h] + kRaise;     // (nothing so far: -inf, which any score passes)
        if (__any_sync(0xffffffffu, raise)) {                // seldom: for the first keys, as a rule, when there is nothing to rescale
          float keep[MT][2];
          bool more = false;
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float up = fmaxf(top[m][h] * sc2, m_run[m][h]);
              more |= l_run[m][h] != 0.f;
              keep[m][h] = up == -INFINITY ? 1.f : ex2(m_run[m][h] - up);
              m_run[m][h] = up;
            }
          if (__any_sync(0xffffffffu, more)) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                l_run[m][h] *= keep[m][h];
#pragma unroll
                for (int n = 0; n < D / 8; ++n) o[m][n][2 * h] *= keep[m][h], o[m][n][2 * h + 1] *= keep[m][h];
              }
          }
        }
        unsigned w[MT][4], rest[MT][4];                      // PARTS == 2: the weights as two bfloat16 numbers, their rounding and what it left
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float base = m_run[m][h] == -INFINITY ? 0.f : m_run[m][h];
            const float w0 = ex2(fmaf(c[m][0][2 * h], sc2, -base)), w1 = ex2(fmaf(c[m][0][2 * h + 1], sc2, -base));
            const float w2 = ex2(fmaf(c[m][1][2 * h], sc2, -base)), w3 = ex2(fmaf(c[m][1][2 * h + 1], sc2, -base));
            l_run[m][h] += (w0 + w1) + (w2 + w3);
            w[m][h] = pack_two(w0, w1, rest[m][h]);
            w[m][2 + h] = pack_two(w2, w3, rest[m][2 + h]);
          }
#pragma unroll
        for (int n = 0; n < D / 16; ++n) {
          unsigned b[4];
          ldsm4t(b, value_at[n & 3] + stage + (n >> 2) * AB);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            mma(o[m][2 * n], w[m], b[0], b[1]);
            mma(o[m][2 * n + 1], w[m], b[2], b[3]);
            if (PARTS == 2) {
              mma(o[m][2 * n], rest[m], b[0], b[1]);
              mma(o[m][2 * n + 1], rest[m], b[2], b[3]);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&ring->empty[st]);
      stage += SB;
      if (++st == kStages) st = 0, stage = 0, parity ^= 1;
    }
    // all copies have landed before the CTA may end, or its memory serve the sums (bounded, where something went wrong)
    if (warp == 0)
      for (int i = max(0, issued - kStages); i < issued; ++i)
        for (unsigned n = 0; n < (1u << 20); ++n)
          if (mbar_try(&ring->full[i % kStages], (i / kStages) & 1)) break;
  }
  // the four warps' sums of a row, one beside the other: each lane's numbers together, so that they go in few instructions
  // (what a CTA runs once costs it the fetch of its code, some 14 cycles an instruction)
  float* sums = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float l = l_run[m][h];
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      if (t4 == 0) stat[group * ROWS + 16 * m + quad + 8 * h] = make_float2(m_run[m][h], l);
    }
  __syncthreads();                                           // all have done with the ring
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const unsigned to = smem_u32(smem) + 4 * ((group * ROWS + 16 * m + quad + 8 * h) * OS + t4 * OL);
#pragma unroll
      for (int n = 0; n < D / 8; n += 2)
        asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to + 8 * n), "f"(o[m][n][2 * h]), "f"(o[m][n][2 * h + 1]), "f"(o[m][n + 1][2 * h]),
                     "f"(o[m][n + 1][2 * h + 1]) : "memory");
    }
  __syncthreads();
  const bool whole = r.keys <= a.chunk;
  constexpr int LANES = D / 4;                               // of a row, four numbers each: two of 16 j + 2 t, two of 8 further on
  const int ot = threadIdx.x % LANES / (LANES / 4), oj = threadIdx.x % (LANES / 4);
#pragma unroll 1
  for (int row = threadIdx.x / LANES; row < ROWS; row += kThreads / LANES) {
    const int p = pair0 + row, d = 16 * oj + 2 * ot;
    if (p >= pairs) break;
    float2 st[kGroups];
    float4 v[kGroups];
#pragma unroll
    for (int w = 0; w < kGroups; ++w) {
      st[w] = stat[w * ROWS + row];
      v[w] = *reinterpret_cast<const float4*>(sums + ((size_t)w * ROWS + row) * OS + ot * OL + 4 * oj);
    }
    const float top = fmaxf(fmaxf(st[0].x, st[1].x), fmaxf(st[2].x, st[3].x)), base = top == -INFINITY ? 0.f : top;
    float l = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kGroups; ++w) {
      const float f = ex2(st[w].x - base);
      l = fmaf(f, st[w].y, l);
      x.x = fmaf(f, v[w].x, x.x), x.y = fmaf(f, v[w].y, x.y), x.z = fmaf(f, v[w].z, x.z), x.w = fmaf(f, v[w].w, x.w);
    }
    const int node = node_of(a, p);
    const size_t to = (size_t)(r.row0 + node) * a.Hq + g * G + p - node * G;
    if (whole) {
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
      *reinterpret_cast<unsigned*>(out + to * D + d) = pack(x.x * inv, x.y * inv);
      *reinterpret_cast<unsigned*>(out + to * D + d + 8) = pack(x.z * inv, x.w * inv);
    } else {
      const size_t ws = (size_t)blockIdx.y * a.T * a.Hq + to;
      *reinterpret_cast<float2*>(a.ws_acc + ws * D + d) = make_float2(x.x, x.y);
      *reinterpret_cast<float2*>(a.ws_acc + ws * D + d + 8) = make_float2(x.z, x.w);
      if (d == 0) reinterpret_cast<float2*>(a.ws_ml)[ws] = make_float2(top, l);
    }
  }
}

template <int D, int MT>
int launch_mma(const CUtensorMap& map, const TreeArgs& a, int box_rows, const void* qkv, void* out, cudaStream_t stream) {
  constexpr size_t smem = smem_bytes<D, MT>();
  if (int rc = allow_smem<tree_attention_mma_kernel<D, MT>>(smem)) return rc;
  const long long pairs = std::min(32ll * a.words, (long long)a.T) * (a.Hq / a.Hkv);
  const long long x = (long long)a.S * a.Hkv, z = (pairs + 16 * MT - 1) / (16 * MT);
  NF_REQUIRE(x < (1ll << 31) && a.shares <= 65535 && z <= 65535, "tree attention: %d requests with %d key heads are too many", a.S, a.Hkv);
  launch_chained(tree_attention_mma_kernel<D, MT>, dim3((unsigned)x, a.shares, (unsigned)z), dim3(kThreads), smem, stream, map, a, box_rows,
                 a.page_size & (a.page_size - 1) ? -1 : __builtin_ctz(a.page_size), (const __nv_bfloat16*)qkv, (__nv_bfloat16*)out);
  return check_launch("tree_attention_mma");
}

}  // namespace

// Pairs a CTA takes: 16 where a request has no more on average.
int tree_mma_rows(int S, int T, int Hq, int Hkv) { return (long long)T * (Hq / Hkv) <= 16ll * S ? 16 : 32; }

int tree_mma_chunk(int S, int T, int Hq, int Hkv, int max_context) {
  const long long pairs = ((long long)T * (Hq / Hkv) + S - 1) / S, rows = tree_mma_rows(S, T, Hq, Hkv);
  const long long ctas = (pairs + rows - 1) / rows * S * Hkv;
  const auto keys = [&](long long shares) { return ((max_context + shares - 1) / shares + 127) / 128 * 128; };
  // as many shares as have room at once, of 384 keys at least: with fewer what a CTA does once is the most of it (one row
  // of 16 heads behind 8,192 keys in shares of 256, 512 and 1,024 keys: 23.5, 17.7 and 23.2 us).  Long shares in some more,
  // since requests are not of one length (8 requests of 32 nodes behind up to 8,192 keys in 2, 5 and 8 shares: 99, 89, 96)
  long long chunk = keys(std::max(1ll, 296 / ctas));
  if (chunk > 2048) chunk = keys(std::max(1ll, (5 * 148 + ctas - 1) / ctas));
  return (int)std::max(384ll, chunk);
}

int launch_tree_mma(const TreeArgs& a, const void* qkv, const void* pages, void* out, cudaStream_t stream) {
  const bool few = tree_mma_rows(a.S, a.T, a.Hq, a.Hkv) == 16;
  const int box_rows = a.page_size % 64 == 0 ? 64 : (a.page_size % 32 == 0 ? 32 : 16);
  CUtensorMap map;
  if (int rc = make_map(&map, pages, (long long)a.num_pages * 2 * a.Hkv * a.page_size, a.D, box_rows)) return rc;
  if (a.D == 64) return few ? launch_mma<64, 1>(map, a, box_rows, qkv, out, stream) : launch_mma<64, 2>(map, a, box_rows, qkv, out, stream);
  return few ? launch_mma<128, 1>(map, a, box_rows, qkv, out, stream) : launch_mma<128, 2>(map, a, box_rows, qkv, out, stream);
}

}  // namespace nf

using namespace nf;

// 0, or the code of the first wait that ran out since the last time (1 producer, 2 consumers), or 100 + a request (from 1 on)
// whose lengths, rows or pages did not fit.  Synchronises.
extern "C" int nf_tree_attention_mma_status() {
  int v = 0, w = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_tree_mma_wait, sizeof(int)) != cudaSuccess) return -1;
  if (cudaMemcpyFromSymbol(&w, g_tree_mma_error, sizeof(int)) != cudaSuccess) return -1;
  if (v) cudaMemcpyToSymbol(g_tree_mma_wait, &zero, sizeof(int));
  if (w) cudaMemcpyToSymbol(g_tree_mma_error, &zero, sizeof(int));
  return v ? v : (w ? 100 + w : 0);
}
