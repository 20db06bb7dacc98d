// Low-rank adapters of a step's rows beside a shared projection, bfloat16, on the 5th-generation tensor cores:
//
//   y[t, f] = sum_k x[t, k] W[f, k] + sum_r h[t, slice(f) R + r] B[a, f, r],   h[t, j] = s[a] sum_k x[t, k] A[a, j, k],   a = ids[t]
//
// Two launches.  The first computes h (here, or a warp a number in adapter.cu where the rows are few); the second is the
// shared product, whose accumulators take the adapters' part before they are rounded, once, to bfloat16.  The second may
// begin while the first runs (it is launched chained): it needs h only when its own sum over k is done.
//
// `adapter_wide_kernel`, many rows: a persistent CTA an SM, tiles of 128 rows x up to 256 features, k in steps of 64 through a
// ring of TMA stages, two accumulators in tensor memory so that a tile's epilogue runs under the next tile's products.  Behind
// the last step over k a tile takes one step more for each adapter that occurs among its 128 rows: rows of h of that adapter,
// zeros for the others, times the adapter's rows of B.  h enters as two bfloat16 numbers, the nearest and what it leaves
// (2^-17 of h is lost), both against the same rows of B: the adapters' part is then as good as the float32 sum it is added to.
// Tiles never reach over the end of a slice, so a tile needs one slice's columns of h.
//
// `adapter_rows_kernel`, few rows: the time is that of reading W once.  W is the 128-row operand, the rows of x the other; the
// CTAs of a cluster share a tile of 128 features and split k; their sums meet through distributed shared memory, each CTA
// adding up the rows it owns, in the order of the CTAs, and adding the adapters' part: a thread a feature, whose row of B it
// reads from memory once for each row of x with another adapter than the one before.
#define NF_CHAIN_CLASS 0x40
#include "tcgen05.cuh"

namespace nf {
namespace {

constexpr int kAdM = 128, kAdK = 64;                 // rows of a tile, k of a step
constexpr int kAdTile = kAdM * kAdK * 2;             // bytes of 128 rows of one step
constexpr int kAdMaxStages = 12;
constexpr int kNone = 0x7fffffff;

__device__ int g_adapter_tc_error = 0;               // code of the first wait that was given up on
__device__ int g_adapter_tc_index = 0;               // 1 + a row whose adapter lies outside the pool

// A wait of a whole warp: all of its lanes go on, or none does.
__device__ __forceinline__ bool warp_wait(void* bar, unsigned parity, volatile int* stop, int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, stop, code, &g_adapter_tc_error));
}

struct TcSlices {
  int n;
  int end[8];
};

// bf16 x bf16 -> f32, both operands K-major, 128 rows, n columns
__device__ __forceinline__ unsigned ad_instr_desc(int n) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((unsigned)(n >> 3) << 17) | ((unsigned)(kAdM >> 4) << 24);
}

// The adapters that occur among a tile's rows, in ascending order: each lane holds four rows' ids (-1: none), the next one
// is the smallest above the last.
struct TileIds {
  int v[4];
  __device__ __forceinline__ void load(const int* ids, int row0, int rows, int n) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = row0 + lane + 32 * i;
      const int a = t < rows ? ids[t] : -1;
      v[i] = a >= 0 && a < n ? a : -1;
    }
  }
  __device__ __forceinline__ int next(int last) const {
    int m = kNone;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = v[i] > last ? min(m, v[i]) : m;
    return __reduce_min_sync(0xffffffffu, m);
  }
};

// ---- h: the adapters' first product ---------------------------------------------------------------------------------------

struct __align__(8) ShrinkBars {
  unsigned long long full[kAdMaxStages], empty[kAdMaxStages], acc_full[2], acc_empty[2];
  unsigned tmem_base;
  int stop;
};

// D[j, t] = sum over this CTA's part of k of A[a, j, k] x[t, k], for the adapters a of a tile of up to 128 rows: every
// gridDim.z-th of those that occur.  Parts of k are left beside one another in h [parts, rows, SR], for whoever reads them to add.
// 192 threads: producer, MMA, four epilogue warps.  grid: (parts of k, row tiles * tiles of 128 j, adapters in turn).
__global__ void __launch_bounds__(192, 1)
adapter_shrink_tc_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_x, const float* __restrict__ scale,
                         const int* __restrict__ ids, float* __restrict__ h, int rows, int K, int SR, int n, int row_tiles, int NT,
                         int a_box, int stages) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  ShrinkBars* bars = reinterpret_cast<ShrinkBars*>(smem);
  unsigned char* stage0 = smem + 1024;
  const int stage_bytes = kAdTile + NT * 128;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* stop = &bars->stop;
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) { mbar_init(&bars->full[s], 1); mbar_init(&bars->empty[s], 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(&bars->acc_full[b], 1); mbar_init(&bars->acc_empty[b], 4); }
    bars->stop = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars->tmem_base)), "r"(256) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const unsigned tmem = bars->tmem_base;
  chain_wait(ids, scale);
  chain_release_late();               // the product behind this may begin: what came before is complete
  const int tile = blockIdx.y % row_tiles, jt = blockIdx.y / row_tiles;
  const int row0 = tile * kAdM, j0 = jt * kAdM;
  const int steps = (K + kAdK - 1) / kAdK;
  const int k_first = (int)((long long)blockIdx.x * steps / gridDim.x), k_last = (int)((long long)(blockIdx.x + 1) * steps / gridDim.x);
  TileIds tids;
  tids.load(ids, row0, rows, n);

  if (warp == 0) {
    int it = 0, turn = 0, issued = 0;
    bool ok = true;
    for (int a = tids.next(-1); a != kNone && ok; a = tids.next(a), ++turn) {
      if (turn % (int)gridDim.z != (int)blockIdx.z) continue;
      if (lane == 0) {
        for (int ks = k_first; ks < k_last; ++ks, ++it) {
          const int s = it % stages;
          if (!mbar_wait(&bars->empty[s], ((it / stages) & 1) ^ 1, stop, 1, &g_adapter_tc_error)) { ok = false; break; }
          unsigned char* st = stage0 + (size_t)s * stage_bytes;
          mbar_expect_tx(&bars->full[s], a_box * 128 + NT * 128);
          tma_load_2d(st, &map_a, ks * kAdK, a * SR + j0, &bars->full[s]);
          tma_load_2d(st + kAdTile, &map_x, ks * kAdK, row0, &bars->full[s]);
          issued = it + 1;
        }
      }
      ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
    }
    if (!ok && lane == 0) {
      for (int j = max(0, issued - stages); j < issued; ++j)
        for (unsigned i = 0; i < (1u << 20); ++i)
          if (mbar_try(&bars->full[j % stages], (j / stages) & 1)) break;
    }
  } else if (warp == 1) {
    int it = 0, turn = 0, done = 0;
    bool ok = true;
    const unsigned idesc = ad_instr_desc(NT);
    for (int a = tids.next(-1); a != kNone && ok; a = tids.next(a), ++turn) {
      if (turn % (int)gridDim.z != (int)blockIdx.z) continue;
      if (lane == 0) {
        const int ab = done & 1;
        if (!mbar_wait(&bars->acc_empty[ab], ((done >> 1) & 1) ^ 1, stop, 2, &g_adapter_tc_error)) ok = false;
        tc_fence_after();
        for (int ks = k_first; ks < k_last && ok; ++ks, ++it) {
          const int s = it % stages;
          if (!mbar_wait(&bars->full[s], (it / stages) & 1, stop, 3, &g_adapter_tc_error)) { ok = false; break; }
          tc_fence_after();
          unsigned char* st = stage0 + (size_t)s * stage_bytes;
          const unsigned long long da = smem_desc(st), db = smem_desc(st + kAdTile);
#pragma unroll
          for (int kk = 0; kk < kAdK / 16; ++kk) tc_mma(tmem + ab * 128, da + 2 * kk, db + 2 * kk, idesc, ks > k_first || kk > 0 ? 1u : 0u);
          tc_commit(&bars->empty[s]);
        }
        if (ok) tc_commit(&bars->acc_full[ab]);
      }
      ++done;
      ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
    }
  } else {
    const int quad = warp & 3, j = j0 + quad * 32 + lane;
    int turn = 0, done = 0;
    float* part = h + (size_t)blockIdx.x * rows * SR;
    for (int a = tids.next(-1); a != kNone; a = tids.next(a), ++turn) {
      if (turn % (int)gridDim.z != (int)blockIdx.z) continue;
      const int ab = done & 1;
      if (!warp_wait(&bars->acc_full[ab], (done >> 1) & 1, stop, 4)) break;
      tc_fence_after();
      const float sc = scale[a];
      const unsigned at = tmem + ab * 128 + ((unsigned)(quad * 32) << 16);
#pragma unroll 1
      for (int q = 0; q * 32 < NT; ++q) {
        const int id = q == 0 ? tids.v[0] : q == 1 ? tids.v[1] : q == 2 ? tids.v[2] : tids.v[3];
        const unsigned mine = __ballot_sync(0xffffffffu, id == a);      // this tile's rows 32 q .. 32 q + 31 with adapter a
        if (!mine) continue;
        unsigned v[32];
        if (q * 32 + 32 <= NT) tc_ld32(at + q * 32, v);
        else tc_ld16(at + q * 32, v);                  // (NT is a multiple of 16)
        tc_wait_ld();
        if (j < SR) {
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if (mine & (1u << c)) part[(size_t)(row0 + q * 32 + c) * SR + j] = __uint_as_float(v[c]) * sc;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->acc_empty[ab]);
      ++done;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256) : "memory");
  }
}

// ---- many rows -------------------------------------------------------------------------------------------------------------

struct __align__(8) WideBars {
  unsigned long long full[kAdMaxStages], empty[kAdMaxStages], acc_full[2], acc_empty[2], h_full, h_empty;
  unsigned tmem_base;
  int stop;
};

constexpr int kWideEpilogueWarps = 8;
constexpr int kWideThreads = 32 * (2 + 4 + kWideEpilogueWarps);
constexpr int kWideHead = 1024, kWideH = 2 * kAdTile;      // barriers; the two parts of a tile's rows of h
constexpr int kWideSmem = 225 * 1024;

struct WideTile {
  int row0, f0, width, slice;
};
// Tile i: features vary fastest, so that the CTAs that run together share rows of x and go through W side by side.
__device__ __forceinline__ WideTile wide_tile(int i, int f_tiles, int BN, const TcSlices& sl) {
  WideTile w;
  const int m = i / f_tiles;
  int f = i - m * f_tiles, begin = 0;
  w.row0 = m * kAdM;
  w.slice = 0;
  for (int s = 0;; ++s) {
    const int tiles = (sl.end[s] - begin + BN - 1) / BN;
    if (f < tiles || s + 1 >= sl.n) {
      w.slice = s;
      w.f0 = begin + f * BN;
      w.width = min(BN, sl.end[s] - w.f0);
      return w;
    }
    f -= tiles;
    begin = sl.end[s];
  }
}

// Warps: 0 producer, 1 MMA and tensor memory, 2..5 rows of h (a thread a row), 6..13 epilogue.
__global__ void __launch_bounds__(kWideThreads, 1)
adapter_wide_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_b,
                    const int* __restrict__ ids, const float* __restrict__ h, int parts, __nv_bfloat16* __restrict__ y, int rows, int N, int K,
                    int R, int n, const __grid_constant__ TcSlices slices, int f_tiles, int n_tiles, int BN, int stages) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  WideBars* bars = reinterpret_cast<WideBars*>(smem);
  unsigned char* h_tile = smem + kWideHead;
  unsigned char* stage0 = h_tile + kWideH;
  const int stage_bytes = kAdTile + BN * 128;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* stop = &bars->stop;
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) { mbar_init(&bars->full[s], 1); mbar_init(&bars->empty[s], 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(&bars->acc_full[b], 1); mbar_init(&bars->acc_empty[b], kWideEpilogueWarps); }
    mbar_init(&bars->h_full, 4);
    mbar_init(&bars->h_empty, 1);
    bars->stop = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars->tmem_base)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const unsigned tmem = bars->tmem_base;
  const int steps = (K + kAdK - 1) / kAdK;
  const int r_steps = (R + kAdK - 1) / kAdK;          // steps of up to 64 ranks an adapter
  const int r_here = min(R, kAdK);                    // ranks of one such step (R is 16, 32, 64 or 128)
  TileIds tids;

  if (warp == 0) {
    // ---- producer: x and W (the kernel before the first launch wrote x: complete, see chain_release_late there) ----------
    int it = 0, issued = 0;
    bool ok = true;
    for (int i = blockIdx.x; i < n_tiles && ok; i += gridDim.x) {
      const WideTile w = wide_tile(i, f_tiles, BN, slices);
      tids.load(ids, w.row0, rows, n);
      if (lane == 0) {
        for (int ks = 0; ks < steps; ++ks, ++it) {
          const int s = it % stages;
          if (!mbar_wait(&bars->empty[s], ((it / stages) & 1) ^ 1, stop, 1, &g_adapter_tc_error)) { ok = false; break; }
          unsigned char* st = stage0 + (size_t)s * stage_bytes;
          mbar_expect_tx(&bars->full[s], stage_bytes);
          tma_load_2d(st, &map_x, ks * kAdK, w.row0, &bars->full[s]);
          tma_load_2d(st + kAdTile, &map_w, ks * kAdK, w.f0, &bars->full[s]);
          issued = it + 1;
        }
      }
      for (int a = tids.next(-1); a != kNone; a = tids.next(a)) {
        if (lane == 0 && ok) {
          for (int rs = 0; rs < r_steps; ++rs, ++it) {
            const int s = it % stages;
            if (!mbar_wait(&bars->empty[s], ((it / stages) & 1) ^ 1, stop, 1, &g_adapter_tc_error)) { ok = false; break; }
            unsigned char* st = stage0 + (size_t)s * stage_bytes;
            mbar_expect_tx(&bars->full[s], BN * 128);
            tma_load_2d(st + kAdTile, &map_b, rs * kAdK, a * N + w.f0, &bars->full[s]);
            issued = it + 1;
          }
        }
      }
      ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
    }
    if (!ok && lane == 0) {
      for (int j = max(0, issued - stages); j < issued; ++j)
        for (unsigned i = 0; i < (1u << 20); ++i)
          if (mbar_try(&bars->full[j % stages], (j / stages) & 1)) break;
    }
  } else if (warp == 1) {
    // ---- MMA ----------------------------------------------------------------------------------------------------------------
    int it = 0, done = 0, ht = 0;
    bool ok = true;
    const unsigned idesc = ad_instr_desc(BN);
    for (int i = blockIdx.x; i < n_tiles && ok; i += gridDim.x, ++done) {
      const WideTile w = wide_tile(i, f_tiles, BN, slices);
      tids.load(ids, w.row0, rows, n);
      const int ab = done & 1;
      const unsigned acc = tmem + ab * 256;
      if (lane == 0) {
        if (!mbar_wait(&bars->acc_empty[ab], ((done >> 1) & 1) ^ 1, stop, 2, &g_adapter_tc_error)) ok = false;
        tc_fence_after();
        for (int ks = 0; ks < steps && ok; ++ks, ++it) {
          const int s = it % stages;
          if (!mbar_wait(&bars->full[s], (it / stages) & 1, stop, 3, &g_adapter_tc_error)) { ok = false; break; }
          tc_fence_after();
          unsigned char* st = stage0 + (size_t)s * stage_bytes;
          const unsigned long long da = smem_desc(st), db = smem_desc(st + kAdTile);
#pragma unroll
          for (int kk = 0; kk < kAdK / 16; ++kk) tc_mma(acc, da + 2 * kk, db + 2 * kk, idesc, ks > 0 || kk > 0 ? 1u : 0u);
          tc_commit(&bars->empty[s]);
        }
      }
      for (int a = tids.next(-1); a != kNone; a = tids.next(a)) {
        if (lane == 0 && ok) {
          for (int rs = 0; rs < r_steps; ++rs, ++it, ++ht) {
            const int s = it % stages;
            if (!mbar_wait(&bars->h_full, ht & 1, stop, 5, &g_adapter_tc_error) ||
                !mbar_wait(&bars->full[s], (it / stages) & 1, stop, 3, &g_adapter_tc_error)) { ok = false; break; }
            tc_fence_after();
            const unsigned long long hi = smem_desc(h_tile), lo = smem_desc(h_tile + kAdTile);
            const unsigned long long db = smem_desc(stage0 + (size_t)s * stage_bytes + kAdTile);
            for (int kk = 0; kk < r_here / 16; ++kk) {
              tc_mma(acc, hi + 2 * kk, db + 2 * kk, idesc, 1u);
              tc_mma(acc, lo + 2 * kk, db + 2 * kk, idesc, 1u);
            }
            tc_commit(&bars->empty[s]);
            tc_commit(&bars->h_empty);
          }
        }
      }
      if (lane == 0 && ok) tc_commit(&bars->acc_full[ab]);
      ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
    }
  } else if (warp < 6) {
    // ---- rows of h: this thread's row of the tile, in the operand's swizzled image --------------------------------------------
    chain_wait(h);
    const int r = (warp - 2) * 32 + lane, SR = slices.n * R;
    int ht = 0;
    bool ok = true;
    for (int i = blockIdx.x; i < n_tiles && ok; i += gridDim.x) {
      const WideTile w = wide_tile(i, f_tiles, BN, slices);
      tids.load(ids, w.row0, rows, n);
      const int t = w.row0 + r;
      const int own = t < rows ? ids[t] : -1;
      if (w.f0 == 0 && own >= n) atomicCAS(&g_adapter_tc_index, 0, t + 1);
      for (int a = tids.next(-1); a != kNone && ok; a = tids.next(a)) {
        for (int rs = 0; rs < r_steps; ++rs, ++ht) {
          if (!warp_wait(&bars->h_empty, (ht & 1) ^ 1, stop, 6)) { ok = false; break; }
          const float* src = h + (size_t)t * SR + w.slice * R + rs * kAdK;
          for (int j = 0; j < r_here / 8; ++j) {
            uint4 hi = make_uint4(0, 0, 0, 0), lo = hi;
            if (own == a) {
              float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
              for (int p = 0; p < parts; ++p) {
                float u[8];
                load8(src + (size_t)p * rows * SR + 8 * j, u);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] += u[e];
              }
              __nv_bfloat162 a2[4], b2[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                a2[e] = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
                const float2 back = __bfloat1622float2(a2[e]);
                // (of an infinity nothing is left)
                b2[e] = __floats2bfloat162_rn(isinf(back.x) ? 0.f : v[2 * e] - back.x, isinf(back.y) ? 0.f : v[2 * e + 1] - back.y);
              }
              hi = *reinterpret_cast<uint4*>(a2);
              lo = *reinterpret_cast<uint4*>(b2);
            }
            const int at = r * 128 + ((j ^ (r & 7)) << 4);
            *reinterpret_cast<uint4*>(h_tile + at) = hi;
            *reinterpret_cast<uint4*>(h_tile + kAdTile + at) = lo;
          }
          fence_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars->h_full);
        }
      }
    }
  } else {
    // ---- epilogue: tensor-memory lanes 32 * (warp % 4) .. + 31, every other run of 32 columns --------------------------------
    const int quad = warp & 3, half = (warp - 6) >> 2;
    int done = 0;
    for (int i = blockIdx.x; i < n_tiles; i += gridDim.x, ++done) {
      const WideTile w = wide_tile(i, f_tiles, BN, slices);
      const int ab = done & 1;
      if (!warp_wait(&bars->acc_full[ab], (done >> 1) & 1, stop, 4)) break;
      tc_fence_after();
      const int t = w.row0 + quad * 32 + lane;
      __nv_bfloat16* out = y + (size_t)t * N + w.f0;
      const bool whole = N % 8 == 0 && w.f0 % 8 == 0;
      for (int c0 = half * 32; c0 < BN; c0 += 64) {
        unsigned v[32];
        if (c0 < w.width) {
          tc_ld32(tmem + ab * 256 + ((unsigned)(quad * 32) << 16) + c0, v);
          tc_wait_ld();
        }
        if (c0 + 64 >= BN) {                      // the last this warp reads of the accumulator
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars->acc_empty[ab]);
        }
        if (c0 >= w.width || t >= rows) continue;
        if (whole && c0 + 32 <= w.width) {
#pragma unroll
          for (int c = 0; c < 32; c += 8) {
            __nv_bfloat162 o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = __floats2bfloat162_rn(__uint_as_float(v[c + 2 * e]), __uint_as_float(v[c + 2 * e + 1]));
            *reinterpret_cast<uint4*>(out + c0 + c) = *reinterpret_cast<uint4*>(o);
          }
        } else {
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if (c0 + c < w.width) out[c0 + c] = __float2bfloat16_rn(__uint_as_float(v[c]));
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// ---- few rows ----------------------------------------------------------------------------------------------------------------

constexpr int kRowsMost = 64;              // rows that adapter_rows_kernel takes

struct __align__(8) RowsBars {
  unsigned long long full[kAdMaxStages], empty[kAdMaxStages], acc_full;
  unsigned tmem_base;
  int stop;
};

__device__ __forceinline__ unsigned cluster_addr(unsigned local, int rank) {
  unsigned remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
  return remote;
}

// grid: (members of the cluster, feature tiles).  192 threads: producer, MMA, four epilogue warps (a thread a feature).
__global__ void __launch_bounds__(192)
adapter_rows_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const int* __restrict__ ids,
                    const float* __restrict__ h, int parts, const __nv_bfloat16* __restrict__ B, __nv_bfloat16* __restrict__ y, int rows,
                    int N, int K, int R, int n, const __grid_constant__ TcSlices slices, int NT, int stages) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  RowsBars* bars = reinterpret_cast<RowsBars*>(smem);
  unsigned char* stage0 = smem + 1024;
  const int stage_bytes = kAdTile + NT * 128;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int members = gridDim.x, member = blockIdx.x;          // the cluster is the grid's first dimension
  volatile int* stop = &bars->stop;
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) { mbar_init(&bars->full[s], 1); mbar_init(&bars->empty[s], 1); }
    mbar_init(&bars->acc_full, 1);
    bars->stop = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars->tmem_base)), "r"(64) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const unsigned tmem = bars->tmem_base;
  const WideTile w = wide_tile(blockIdx.y, gridDim.y, kAdM, slices);
  const int steps = (K + kAdK - 1) / kAdK;
  const int k_first = (int)((long long)member * steps / members), k_last = (int)((long long)(member + 1) * steps / members);
  float* sums = reinterpret_cast<float*>(stage0);              // [NT][128], in the stages once they are read
  bool fine = true;

  if (warp == 0) {
    if (lane == 0) {
      int issued = 0;
      for (int it = 0; it < k_last - k_first; ++it) {
        const int s = it % stages;
        if (!mbar_wait(&bars->empty[s], ((it / stages) & 1) ^ 1, stop, 11, &g_adapter_tc_error)) { fine = false; break; }
        unsigned char* st = stage0 + (size_t)s * stage_bytes;
        mbar_expect_tx(&bars->full[s], stage_bytes);
        tma_load_2d(st, &map_w, (k_first + it) * kAdK, w.f0, &bars->full[s]);
        tma_load_2d(st + kAdTile, &map_x, (k_first + it) * kAdK, 0, &bars->full[s]);
        issued = it + 1;
      }
      if (!fine)
        for (int j = max(0, issued - stages); j < issued; ++j)
          for (unsigned i = 0; i < (1u << 20); ++i)
            if (mbar_try(&bars->full[j % stages], (j / stages) & 1)) break;
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      const unsigned idesc = ad_instr_desc(NT);
      for (int it = 0; it < k_last - k_first; ++it) {
        const int s = it % stages;
        if (!mbar_wait(&bars->full[s], (it / stages) & 1, stop, 13, &g_adapter_tc_error)) { fine = false; break; }
        tc_fence_after();
        unsigned char* st = stage0 + (size_t)s * stage_bytes;
        const unsigned long long dw = smem_desc(st), dx = smem_desc(st + kAdTile);
#pragma unroll
        for (int kk = 0; kk < kAdK / 16; ++kk) tc_mma(tmem, dw + 2 * kk, dx + 2 * kk, idesc, it > 0 || kk > 0 ? 1u : 0u);
        tc_commit(&bars->empty[s]);
      }
      if (fine) tc_commit(&bars->acc_full);
    }
    __syncwarp();
  } else {
    const int quad = warp & 3;
    if (warp_wait(&bars->acc_full, 0, stop, 14)) {
      tc_fence_after();
      for (int c0 = 0; c0 < NT; c0 += 16) {
        unsigned v[16];
        tc_ld16(tmem + ((unsigned)(quad * 32) << 16) + c0, v);
        tc_wait_ld();
#pragma unroll
        for (int c = 0; c < 16; ++c) sums[(c0 + c) * kAdM + quad * 32 + lane] = __uint_as_float(v[c]);
      }
    }
    tc_fence_before();
  }
  // the members' sums are all there
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (warp >= 2) {
    const int d = (warp & 3) * 32 + lane, f = w.f0 + d, SR = slices.n * R;
    const int t_first = (int)((long long)member * rows / members), t_last = (int)((long long)(member + 1) * rows / members);
    const unsigned local = smem_u32(sums + d);
    chain_wait(h);
    for (int t = t_first; t < t_last; ++t) {
      float sum = 0.f;
      for (int m = 0; m < members; ++m) {
        float v;
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr(local + t * kAdM * 4, m)) : "memory");
        sum += v;
      }
      const int a = ids[t];
      if (a >= n && blockIdx.y == 0 && d == 0) atomicCAS(&g_adapter_tc_index, 0, t + 1);
      if (a >= 0 && a < n && d < w.width) {
        const __nv_bfloat16* b = B + ((size_t)a * N + f) * R;
        const float* hr = h + (size_t)t * SR + w.slice * R;
        for (int j = 0; j < R; j += 8) {
          float bv[8], hv[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
          load8(b + j, bv);
          for (int p = 0; p < parts; ++p) {
            float u[8];
            load8(hr + (size_t)p * rows * SR + j, u);
#pragma unroll
            for (int e = 0; e < 8; ++e) hv[e] += u[e];
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) sum = fmaf(hv[e], bv[e], sum);
        }
      }
      if (d < w.width) y[(size_t)t * N + f] = __float2bfloat16_rn(sum);
    }
  }
  // nobody reads another's shared memory any more
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(64) : "memory");
  }
}

// ---- host ----------------------------------------------------------------------------------------------------------------------

int sm_count() {
  static int n = 0;
  if (!n) {
    int dev = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (n <= 0) n = 1;
  }
  return n;
}

int feature_tiles(const TcSlices& s, int width) {
  int tiles = 0, begin = 0;
  for (int i = 0; i < s.n; ++i) {
    tiles += (s.end[i] - begin + width - 1) / width;
    begin = s.end[i];
  }
  return tiles;
}

template <typename F>
int room_for(F* kernel, size_t smem) {
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  NF_REQUIRE(e == cudaSuccess, "adapter_linear: cannot have %zu bytes of shared memory: %s", smem, cudaGetErrorString(e));
  return 0;
}

}  // namespace

int adapter_shrink_simt(const void* x, const void* A, const float* scale, const int* ids, float* h, int rows, int K, int SR, int n,
                        cudaStream_t stream);

}  // namespace nf

using namespace nf;

// Parts of k that the first product of `rows` rows is cut into: h takes parts * rows * n_slices * R floats.
extern "C" int nf_adapter_parts(int rows, int K) {
  const int tiles = (rows + kAdM - 1) / kAdM, steps = (K + kAdK - 1) / kAdK;
  if (rows <= 16) return 1;
  int p = 1;
  while (p < 8 && 2 * p * tiles <= sm_count() && steps >= 4 * p) p *= 2;
  return p;
}

// y = x W^T + the adapters' part (see the head of this file): x [rows, K], W [N, K], A [n, n_slices * R, K], B [n, N, R], y
// [rows, N] bfloat16; scale float32 [n]; ids [rows], -1 for none; h float32 [nf_adapter_parts(rows, K), rows, n_slices * R].  ends: the
// n_slices features (host memory) at which the slices end, the last N.  K a multiple of 8, R 16, 32, 64 or 128, bases
// 16-byte aligned.
extern "C" int nf_adapter_linear(const void* x, const void* W, const void* A, const void* B, const float* scale, const int* ids, float* h,
                                 void* y, int rows, int N, int K, int R, int n, int n_slices, const int* ends, cudaStream_t stream) {
  if (rows == 0 || N == 0) return 0;
  NF_REQUIRE(rows > 0 && N > 0 && K > 0 && n > 0, "adapter_linear: bad sizes rows=%d N=%d K=%d n=%d", rows, N, K, n);
  NF_REQUIRE(K % 8 == 0, "adapter_linear: K=%d must be a multiple of 8", K);
  NF_REQUIRE(R == 16 || R == 32 || R == 64 || R == 128, "adapter_linear: rank %d is not 16, 32, 64 or 128", R);
  NF_REQUIRE(n_slices >= 1 && n_slices <= 8, "adapter_linear: %d slices, 1 to 8", n_slices);
  NF_REQUIRE((long long)n * N < (1ll << 31) && (long long)n * n_slices * R < (1ll << 31), "adapter_linear: %d adapters of %d features are too many", n, N);
  NF_REQUIRE((uintptr_t)x % 16 == 0 && (uintptr_t)W % 16 == 0 && (uintptr_t)A % 16 == 0 && (uintptr_t)B % 16 == 0 && (uintptr_t)h % 16 == 0 &&
             (uintptr_t)y % 16 == 0, "adapter_linear: operands must be 16-byte aligned");
  TcSlices sl{n_slices, {}};
  for (int i = 0; i < n_slices; ++i) {
    sl.end[i] = ends[i];
    NF_REQUIRE(ends[i] > (i ? ends[i - 1] : 0), "adapter_linear: slice %d ends at %d", i, ends[i]);
  }
  NF_REQUIRE(ends[n_slices - 1] == N, "adapter_linear: the slices end at %d of %d features", ends[n_slices - 1], N);
  const int SR = n_slices * R, parts = nf_adapter_parts(rows, K), steps = (K + kAdK - 1) / kAdK;

  // ---- h
  if (rows <= 16) {
    if (int rc = adapter_shrink_simt(x, A, scale, ids, h, rows, K, SR, n, stream)) return rc;
  } else {
    const int tiles = (rows + kAdM - 1) / kAdM, j_tiles = (SR + kAdM - 1) / kAdM;
    const int NT = rows >= kAdM ? kAdM : (rows + 15) & ~15, a_box = SR < kAdM ? SR : kAdM;
    CUtensorMap ma, mx;
    if (int rc = make_map(&ma, A, (long long)n * SR, K, a_box)) return rc;
    if (int rc = make_map(&mx, x, rows, K, NT)) return rc;
    const int stage = kAdTile + NT * 128, stages = 6;
    const size_t smem = 2048 + (size_t)stages * stage;
    static int asked = room_for(adapter_shrink_tc_kernel, 2048 + 6 * (size_t)(2 * kAdTile));
    if (asked) return asked;
    int turns = sm_count() / (parts * tiles * j_tiles);          // CTAs that take a tile's adapters in turn
    const int most = n < NT ? n : NT;
    turns = turns < 1 ? 1 : turns > most ? most : turns;
    launch_chained(adapter_shrink_tc_kernel, dim3(parts, tiles * j_tiles, turns), dim3(192), smem, stream, ma, mx, scale, ids, h, rows, K, SR,
                   n, tiles, NT, a_box, stages);
    if (int rc = check_launch("adapter_shrink")) return rc;
  }

  // ---- the shared product and the adapters' part
  CUtensorMap mx, mw;
  if (rows <= kRowsMost) {
    const int NT = (rows + 15) & ~15, tiles = feature_tiles(sl, kAdM);
    int members = 1;
    while (members < 8 && 2 * members * tiles <= 2 * sm_count() && steps >= 4 * members) members *= 2;
    if (int rc = make_map(&mw, W, N, K, kAdM)) return rc;
    if (int rc = make_map(&mx, x, rows, K, NT)) return rc;
    const int stage = kAdTile + NT * 128, here = (steps + members - 1) / members;
    int stages = (104 * 1024) / stage;
    stages = stages > here ? here : stages;
    const int least = (NT * kAdM * 4 + stage - 1) / stage;       // the sums take the stages' place
    stages = stages < least ? least : stages;
    const size_t smem = 2048 + (size_t)stages * stage;
    static int asked = room_for(adapter_rows_kernel, 108 * 1024);
    if (asked) return asked;
    NF_REQUIRE(tiles <= 65535, "adapter_linear: %d features are too many", N);
    launch_chained_cluster(adapter_rows_kernel, dim3(members, tiles), dim3(192), smem, stream, members, mw, mx, ids, (const float*)h, parts,
                           (const __nv_bfloat16*)B, (__nv_bfloat16*)y, rows, N, K, R, n, sl, NT, stages);
    return check_launch("adapter_rows");
  }
  // The width of a tile: the one whose rounds of tiles take the least, a round's time being that of its widest operand.
  const int m_tiles = (rows + kAdM - 1) / kAdM;
  int BN = 256;
  long long best = -1;
  for (int c = 256; c >= 64; c -= 32) {
    const long long tiles = (long long)m_tiles * feature_tiles(sl, c);
    const long long cost = ((tiles + sm_count() - 1) / sm_count()) * (c > 112 ? c : 112);
    if (best < 0 || cost < best) { best = cost; BN = c; }
  }
  CUtensorMap mb;
  if (int rc = make_map(&mx, x, rows, K, kAdM)) return rc;
  if (int rc = make_map(&mw, W, N, K, BN)) return rc;
  if (int rc = make_map(&mb, B, (long long)n * N, R, BN)) return rc;
  const int f_tiles = feature_tiles(sl, BN);
  const long long n_tiles = (long long)f_tiles * m_tiles;
  NF_REQUIRE(n_tiles < (1ll << 31), "adapter_linear: %d rows of %d features are too many", rows, N);
  int stages = (kWideSmem - kWideHead - kWideH) / (kAdTile + BN * 128);
  stages = stages > kAdMaxStages ? kAdMaxStages : stages;
  static int asked = room_for(adapter_wide_kernel, kWideSmem + 1024);
  if (asked) return asked;
  const int grid = n_tiles < sm_count() ? (int)n_tiles : sm_count();
  launch_chained(adapter_wide_kernel, dim3(grid), dim3(kWideThreads), (size_t)kWideSmem + 1024, stream, mx, mw, mb, ids, (const float*)h, parts,
                 (__nv_bfloat16*)y, rows, N, K, R, n, sl, f_tiles, (int)n_tiles, BN, stages);
  return check_launch("adapter_wide");
}

// 0, or the code of the first wait that one of these kernels gave up on since the last call (1 to 6 the wide form and the
// first product, 11 to 14 the form for few rows); 100 + 1 + a row whose adapter lay outside the pool.  Synchronises.
extern "C" int nf_adapter_tc_status() {
  int v[2] = {0, 0}, zero = 0;
  if (cudaMemcpyFromSymbol(&v[0], g_adapter_tc_error, sizeof(int)) != cudaSuccess) return -1;
  if (cudaMemcpyFromSymbol(&v[1], g_adapter_tc_index, sizeof(int)) != cudaSuccess) return -1;
  if (v[0]) cudaMemcpyToSymbol(g_adapter_tc_error, &zero, sizeof(int));
  if (v[1]) cudaMemcpyToSymbol(g_adapter_tc_index, &zero, sizeof(int));
  return v[0] ? v[0] : (v[1] ? 100 + v[1] : 0);
}
