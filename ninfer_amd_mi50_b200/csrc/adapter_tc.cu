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
// the last step over k a tile takes a step or a few more for each adapter that occurs among its rows: rows of h of that adapter,
// zeros for the others, times the adapter's rows of B.  The kernel that makes h lays it out so, a block of 128 rows for every
// adapter of a row tile, and these steps go through the ring like all others.  h enters as two bfloat16 numbers, the nearest and
// what it leaves (2^-17 of h is lost), both against the same rows of B: the adapters' part is then as good as the float32 sum it is
// added to.  Tiles never reach over the end of a slice, so a tile needs one slice's columns of h.
//
// `adapter_rows_kernel`, few rows: the time is that of reading W once.  W is the 128-row operand, the rows of x the other; the
// CTAs of a cluster share a tile of 128 features and split k; their sums meet through distributed shared memory, each CTA
// adding up the rows it owns, in the order of the CTAs.  The adapters' part is added there, a thread a feature, whose row of B it
// reads from memory once for each row of x with another adapter than the one before; or, where that is much (many rows or ranks),
// it is a few more steps of the product, as in the wide kernel, an adapter's steps taken by one CTA of the cluster.
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

// bf16 x bf16 -> f32, both operands K-major, m rows, n columns
__device__ __forceinline__ unsigned ad_instr_desc(int n, int m) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((unsigned)(n >> 3) << 17) | ((unsigned)(m >> 4) << 24);
}

__device__ __forceinline__ unsigned cluster_addr(unsigned local, int rank) {
  unsigned remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
  return remote;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// One CTA, or the two of a cluster that work on one tile.  Barriers that the products' issuer waits for are those of the even CTA.
template <int CTAS>
__device__ __forceinline__ void tc_alloc(unsigned* base, unsigned cols) {
  if (CTAS == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(base)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(base)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
}
template <int CTAS>
__device__ __forceinline__ void tc_dealloc(unsigned base, unsigned cols) {
  if (CTAS == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols) : "memory");
  else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols) : "memory");
}
template <int CTAS>
__device__ __forceinline__ void tma_load(void* dst, const CUtensorMap* map, int x, int y, void* bar) {
  if (CTAS == 2) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
        ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(cluster_addr(smem_u32(bar), 0)) : "memory");
  } else {
    tma_load_2d(dst, map, x, y, bar);
  }
}
template <int CTAS>
__device__ __forceinline__ void mma(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc, unsigned accumulate) {
  if (CTAS == 2) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
  } else {
    tc_mma(d, a, b, idesc, accumulate);
  }
}
template <int CTAS>
__device__ __forceinline__ void commit(void* bar) {
  if (CTAS == 2) {
    const unsigned short both = 3;
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"(both) : "memory");
  } else {
    tc_commit(bar);
  }
}
template <int CTAS>
__device__ __forceinline__ void arrive_leader(void* bar) {
  if (CTAS == 2) asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr(smem_u32(bar), 0)) : "memory");
  else mbar_arrive(bar);
}
// warp_wait for arrivals that may come from the other CTA of the cluster.
__device__ __forceinline__ bool warp_wait_cluster(void* bar, unsigned parity, volatile int* stop, int code) {
  for (unsigned i = 0; i < kPollLimit; ++i) {
    unsigned ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    if (__all_sync(0xffffffffu, ok)) return true;
    if ((i & 1023u) == 1023u && __any_sync(0xffffffffu, *stop)) return false;
  }
  *stop = 1;
  atomicCAS(&g_adapter_tc_error, 0, code);
  return false;
}

// The adapters that occur among a tile's rows, in ascending order: each lane holds four rows' ids (-1: none), the next one
// is the smallest above the last.
template <int CTAS>
struct TileIds {
  int v[4 * CTAS];
  __device__ __forceinline__ void load(const int* ids, int row0, int rows, int n) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < 4 * CTAS; ++i) {
      const int t = row0 + lane + 32 * i;
      const int a = t < rows ? ids[t] : -1;
      v[i] = a >= 0 && a < n ? a : -1;
    }
  }
  // Leaves the adapters that are `turn` modulo `turns`.
  __device__ __forceinline__ void keep(int turn, int turns) {
#pragma unroll
    for (int i = 0; i < 4 * CTAS; ++i) v[i] = v[i] >= 0 && v[i] % turns == turn ? v[i] : -1;
  }
  __device__ __forceinline__ int next(int last) const {
    int m = kNone;
#pragma unroll
    for (int i = 0; i < 4 * CTAS; ++i) m = v[i] > last ? min(m, v[i]) : m;
    return __reduce_min_sync(0xffffffffu, m);
  }
};

// The stage of a ring and the parity of its present use, step after step (no division by the number of stages).
struct Ring {
  int s = 0;
  unsigned phase = 0;
  __device__ __forceinline__ void next(int stages) {
    if (++s == stages) { s = 0; phase ^= 1; }
  }
};

// ---- h: the adapters' first product ---------------------------------------------------------------------------------------

struct __align__(8) ShrinkBars {
  unsigned long long full[kAdMaxStages], empty[kAdMaxStages], acc_full, acc_empty;
  unsigned tmem_base;
  int stop;
  int id[kAdM];                         // the rows' adapters, -1: none
  unsigned char first[kAdM], place[kAdM];      // whether a row is the first with its adapter; that adapter's place among the tile's
};

// CTAs of a cluster wait for one another, and an allocation of tensor memory waits for the SM's other CTAs: whatever of these
// kernels may meet on an SM, from several streams too, has to find its columns at once.  One CTA of this kernel (256 columns, more
// than half of the shared memory) beside those of adapter_rows_kernel (64 each, that split k 36 KB each; of more than 64 rows 128, and nearly
// all of the shared memory) do; the wide kernel, and all others that take all columns, leave no shared memory for either.
constexpr size_t kShrinkSmemLeast = 118 * 1024, kShrinkSmemMost = 204 * 1024;
constexpr int kShrinkCols = 256;        // columns of an accumulator: numbers of h of all adapters of a pass

// 8 numbers of h as the nearest bfloat16 and what that leaves.
__device__ __forceinline__ void split_h(const float* v, uint4& hi, uint4& lo) {
  __nv_bfloat162 a[4], b[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    a[e] = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
    const float2 back = __bfloat1622float2(a[e]);
    // (of an infinity nothing is left)
    b[e] = __floats2bfloat162_rn(isinf(back.x) ? 0.f : v[2 * e] - back.x, isinf(back.y) ? 0.f : v[2 * e + 1] - back.y);
  }
  hi = *reinterpret_cast<uint4*>(a);
  lo = *reinterpret_cast<uint4*>(b);
}

// D[t, (adapter, j)] over a tile of up to 128 rows: x is the 128-row operand, the rows of A of up to `group` of the adapters
// that occur in the tile the other, so that x is read once for all of them.  The CTAs of a cluster split k; each sends every row's
// own numbers to the member that owns the row, which adds them up in the members' order, scales and writes them.
// gridDim.z CTAs take the adapters of a tile in turn, by their number.  What is written: `places` 0, a row's numbers as they are, [rows,
// SR] float32; otherwise blocks of 128 rows, [row tile][place of the adapter among the tile's, `places` of them][slice][128][2 R]
// bfloat16, R numbers rounded and R of what that leaves, zeros in the rows of other adapters.
// 192 threads: producer, MMA, four epilogue warps (a thread a row).  grid: (members, row tiles * j tiles, adapters in turn).
// What bounds it: not its bytes (2048 rows of 2048, eight adapters of rank 16: 8.8 MB, 1.4 us; 12 under the profiler) but a CTA's chain:
// tensor memory, the first loads, a step every 0.3 us, the cluster's two barriers.  So k is split as far as clusters run at once, and a
// tile's adapters are taken in groups, with x read once for a group.
__global__ void __launch_bounds__(192, 1)
adapter_shrink_tc_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_x, const float* __restrict__ scale,
                         const int* __restrict__ ids, float* __restrict__ h, int rows, int K, int SR, int n, int row_tiles, int x_box, int JW,
                         int group, int stages, int places, int R) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  ShrinkBars* bars = reinterpret_cast<ShrinkBars*>(smem);
  unsigned char* stage0 = smem + 1024;
  const int stage_bytes = kAdTile + group * JW * 128;
  float* sums = reinterpret_cast<float*>(stage0 + (size_t)stages * stage_bytes);      // [members][share of rows][JW + 4], written by all members
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int members = gridDim.x, member = blockIdx.x, share = kAdM / members;          // (a power of two up to 8)
  const int JP = JW + 4;              // numbers between two rows of sums: threads store rows side by side, no bank twice
  volatile int* stop = &bars->stop;
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");      // this member is there
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) { mbar_init(&bars->full[s], 1); mbar_init(&bars->empty[s], 1); }
    mbar_init(&bars->acc_full, 1);
    mbar_init(&bars->acc_empty, 4);
    bars->stop = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncwarp();
  if (warp == 1) tc_alloc<1>(&bars->tmem_base, kShrinkCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const unsigned tmem = bars->tmem_base;
  chain_wait(ids, scale);
  chain_release_late();
  const int tile = blockIdx.y % row_tiles, jt = blockIdx.y / row_tiles;
  const int row0 = tile * kAdM, j0 = jt * JW, jn = min(JW, SR - j0);
  const int steps = (K + kAdK - 1) / kAdK;
  const int k_first = (int)((long long)member * steps / members), k_last = (int)((long long)(member + 1) * steps / members);
  TileIds<1> tids;
  tids.load(ids, row0, rows, n);
  tids.keep(blockIdx.z, gridDim.z);
  // the next group of adapters: lane g holds the g-th; returns how many
  int last = -1;
  auto next_group = [&](int& mine) {
    int count = 0;
    while (count < group) {
      const int a = tids.next(last);
      if (a == kNone) break;
      if (lane == count) mine = a;
      last = a;
      ++count;
    }
    return count;
  };

  if (warp == 0) {
    int issued = 0, mine = 0;
    bool ok = true;
    Ring ring;
    for (;;) {
      const int count = next_group(mine);
      if (!count || !ok) break;
      for (int ks = k_first; ks < k_last; ++ks, ring.next(stages), ++issued) {
        const int s = ring.s;
        if (!warp_wait(&bars->empty[s], ring.phase ^ 1, stop, 1)) { ok = false; break; }
        unsigned char* st = stage0 + (size_t)s * stage_bytes;
        if (lane == 0) {
          mbar_expect_tx(&bars->full[s], x_box * 128 + count * JW * 128);
          tma_load_2d(st, &map_x, ks * kAdK, row0, &bars->full[s]);
        }
        __syncwarp();
        if (lane < count) tma_load_2d(st + kAdTile + lane * JW * 128, &map_a, ks * kAdK, mine * SR + j0, &bars->full[s]);
      }
    }
    if (!ok && lane == 0) {
      for (int j = max(0, issued - stages); j < issued; ++j)
        for (unsigned i = 0; i < (1u << 20); ++i)
          if (mbar_try(&bars->full[j % stages], (j / stages) & 1)) break;
    }
    __syncwarp();
  } else if (warp == 1) {
    int done = 0, mine = 0;
    bool ok = true;
    Ring ring;
    for (;;) {
      const int count = next_group(mine);
      if (!count || !ok) break;
      const unsigned idesc = ad_instr_desc(count * JW, kAdM);
      if (!warp_wait(&bars->acc_empty, (done & 1) ^ 1, stop, 2)) break;
      tc_fence_after();
      for (int ks = k_first; ks < k_last; ++ks) {
        if (!warp_wait(&bars->full[ring.s], ring.phase, stop, 3)) { ok = false; break; }
        tc_fence_after();
        unsigned char* st = stage0 + (size_t)ring.s * stage_bytes;
        const unsigned long long dx = smem_desc(st), da = smem_desc(st + kAdTile);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < kAdK / 16; ++kk) tc_mma(tmem, dx + 2 * kk, da + 2 * kk, idesc, ks > k_first || kk > 0 ? 1u : 0u);
          tc_commit(&bars->empty[ring.s]);
          if (ks + 1 == k_last) tc_commit(&bars->acc_full);
        }
        __syncwarp();
        ring.next(stages);
      }
      ++done;
    }
  } else {
    const int quad = warp & 3, r = quad * 32 + lane, t = row0 + r;
    int own = t < rows ? ids[t] : -1;
    if (own >= n) {
      if (member == 0 && jt == 0 && blockIdx.z == 0) atomicCAS(&g_adapter_tc_index, 0, t + 1);
      own = -1;
    }
    bars->id[r] = own = max(own, -1);
    if (places) {
      // the place of the row's adapter among the tile's in ascending order: how many first rows of smaller ones there are
      asm volatile("bar.sync 1, 128;" ::: "memory");
      int earlier = 0;
      for (int o = 0; o < r; ++o) earlier |= bars->id[o] == own;
      bars->first[r] = own >= 0 && !earlier;
      asm volatile("bar.sync 1, 128;" ::: "memory");
      int place = 0;
      for (int o = 0; o < kAdM; ++o) place += bars->first[o] && bars->id[o] < own;
      bars->place[r] = (unsigned char)place;
    }
    int done = 0, mine = 0;
    const unsigned to = cluster_addr(smem_u32(sums + ((size_t)member * share + r % share) * JP), r / share);
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");      // every member is there: its shared memory may be written
    for (;;) {
      const int count = next_group(mine);
      if (!count) break;
      if (!warp_wait(&bars->acc_full, done & 1, stop, 4)) break;
      tc_fence_after();
      for (int g = 0; g < count; ++g) {
        const int a = __shfl_sync(0xffffffffu, mine, g);       // (every lane, before any condition on its own row)
        const bool is = own == a;          // (a is none of the marks for no adapter)
        if (!__any_sync(0xffffffffu, is)) continue;
        const unsigned at = tmem + g * JW + ((unsigned)(quad * 32) << 16);
        for (int c = 0; c < jn; c += 16) {
          unsigned v[16];
          tc_ld16(at + c, v);
          tc_wait_ld();
          if (is) {
#pragma unroll
            for (int e = 0; e < 16; e += 4)
              asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + (c + e) * 4), "r"(v[e]), "r"(v[e + 1]), "r"(v[e + 2]),
                           "r"(v[e + 3]) : "memory");
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->acc_empty);
      ++done;
    }
  }
  __syncwarp();
  if (warp < 2) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  cluster_barrier();                  // every member's part is there
  const int pieces = jn >> 3;
  auto numbers = [&](int rl, int j, float* v) {                // 8 numbers of this member's row rl, from j on
    const float sc = scale[bars->id[member * share + rl]];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
    for (int m = 0; m < members; ++m) {
      float u[8];
      load8(sums + ((size_t)m * share + rl) * JP + j, u);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += u[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= sc;
  };
  if (!places) {
    for (int i = threadIdx.x; i < share * pieces; i += blockDim.x) {
      const int rl = i / pieces, j = (i - rl * pieces) * 8, id = bars->id[member * share + rl];
      if (id < 0 || id % (int)gridDim.z != (int)blockIdx.z) continue;
      float v[8];
      numbers(rl, j, v);
      float* to = h + (size_t)(row0 + member * share + rl) * SR + j0 + j;
      store4(to, v);
      store4(to + 4, v + 4);
    }
  } else {
    for (int a = tids.next(-1); a != kNone; a = tids.next(a)) {
      int place = -1;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (tids.v[i] == a) place = bars->place[lane + 32 * i];
      place = __reduce_max_sync(0xffffffffu, place);
      __nv_bfloat16* block = reinterpret_cast<__nv_bfloat16*>(h) + ((size_t)tile * places + place) * kAdM * 2 * SR;
      for (int i = threadIdx.x; i < share * pieces; i += blockDim.x) {
        const int rl = i / pieces, j = j0 + (i - rl * pieces) * 8, r = member * share + rl, slice = j / R;
        uint4 hi = make_uint4(0, 0, 0, 0), lo = hi;
        if (bars->id[r] == a) {
          float v[8];
          numbers(rl, j - j0, v);
          split_h(v, hi, lo);
        }
        __nv_bfloat16* to = block + ((size_t)slice * kAdM + r) * 2 * R + (j - slice * R);
        *reinterpret_cast<uint4*>(to) = hi;
        *reinterpret_cast<uint4*>(to + R) = lo;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tc_dealloc<1>(tmem, kShrinkCols);
  }
}

// ---- many rows -------------------------------------------------------------------------------------------------------------

struct __align__(8) WideBars {
  unsigned long long full[kAdMaxStages], empty[kAdMaxStages], acc_full[2], acc_empty[2];
  unsigned tmem_base;
  int stop;
};

constexpr int kWideEpilogueWarps = 8;
constexpr int kWideThreads = 32 * (2 + kWideEpilogueWarps);
constexpr int kWideHead = 1024;                            // barriers
constexpr int kTurnRow = 80, kTurnBytes = 32 * kTurnRow;                 // a warp's 32 x 32 results, rows 80 bytes apart (no bank twice)
constexpr int kWideSmem = 225 * 1024;

struct WideTile {
  int row0, f0, width, slice;
};
// Tile i: features vary fastest, so that the CTAs that run together share rows of x and go through W side by side.
__device__ __forceinline__ WideTile wide_tile(int i, int f_tiles, int tile_rows, int BN, const TcSlices& sl) {
  WideTile w;
  const int m = i / f_tiles;
  int f = i - m * f_tiles, begin = 0;
  w.row0 = m * tile_rows;
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

// The tile a CTA (or pair) takes after `i`: rounds of as many tiles as there are CTAs, the first dealt forwards, the others backwards.
// The engine puts decoded rows first, so a step's first tiles have the most adapters, and the CTAs with those get none of the last,
// shorter round.
__device__ __forceinline__ int next_tile(int i, int first, int stride) { return i < stride ? 2 * stride - 1 - first : i + stride; }

// CTAS 1: a CTA a tile of 128 rows x BN features.  CTAS 2: two CTAs of a cluster a tile of 256 x BN; each holds its own 128 rows of x
// and half of the features' rows of W, and the even one issues products over both (`cta_group::2`): half of W's bytes a CTA.
// Warps: 0 producer, 1 MMA and tensor memory, 2..9 epilogue.  map_h: h as the first product lays it out, `places` blocks a row tile.
// TY: the type of y, bfloat16, or float32 for a caller that has more to do with the sums.
// What bounds it: the tensor cores (73 % busy under the profiler at 2048 rows of 2048 x 6144) and the operands' way into shared memory,
// which at 256 x 256 a pair takes as long as the products: 512 cycles a step, 600 to 700 measured.  8192 rows of 3584 x 4608 take 194 us
// with h, 1.4 PFLOP/s; the library's product without adapters 172.
template <int CTAS, typename TY>
__global__ void __launch_bounds__(kWideThreads, 1)
adapter_wide_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_b,
                    const __grid_constant__ CUtensorMap map_h, const int* __restrict__ ids, TY* __restrict__ y, int rows, int N, int K,
                    int R, int n, int places, const __grid_constant__ TcSlices slices, int f_tiles, int n_tiles, int BN, int stages) {
  extern __shared__ unsigned char smem_raw[];      // [barriers | stages | results on their way]
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  WideBars* bars = reinterpret_cast<WideBars*>(smem);
  unsigned char* stage0 = smem + kWideHead;
  const int w_bytes = BN / CTAS * 128, stage_bytes = kAdTile + w_bytes;
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = CTAS == 2 ? (int)(blockIdx.x & 1) : 0, first = blockIdx.x / CTAS, stride = gridDim.x / CTAS;
  volatile int* stop = &bars->stop;
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) { mbar_init(&bars->full[s], 1); mbar_init(&bars->empty[s], 1); }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bars->acc_full[b], 1);
      mbar_init(&bars->acc_empty[b], kWideEpilogueWarps * CTAS);
    }
    bars->stop = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncwarp();
  if (warp == 1) tc_alloc<CTAS>(&bars->tmem_base, 512);
  tc_fence_before();
  if (CTAS == 2) cluster_barrier();
  __syncthreads();
  tc_fence_after();
  const unsigned tmem = bars->tmem_base;
  const int steps = (K + kAdK - 1) / kAdK;
  // An adapter's steps: up to 32 ranks one, with both parts of h beside one another; beyond, 64 numbers of a part each.
  const int r_steps = (R + kAdK - 1) / kAdK, h_steps = R <= 32 ? 1 : 2 * r_steps;
  TileIds<CTAS> tids;

  if (warp == 0) {
    // ---- producer: x and W (what wrote x is complete, see chain_release_late in the kernels that make h), then h and B ----
    int issued = 0;
    bool ok = true, waited = false;
    Ring ring;
    auto step = [&](const CUtensorMap* mx, int kx, int x_row, const CUtensorMap* mw, int kw, int w_row) {
      if (!warp_wait(&bars->empty[ring.s], ring.phase ^ 1, stop, 1)) { ok = false; return; }
      unsigned char* st = stage0 + (size_t)ring.s * stage_bytes;
      if (elect_one()) {
        if (rank == 0) mbar_expect_tx(&bars->full[ring.s], CTAS * stage_bytes);
        tma_load<CTAS>(st, mx, kx, x_row, &bars->full[ring.s]);
        tma_load<CTAS>(st + kAdTile, mw, kw, w_row, &bars->full[ring.s]);
      }
      __syncwarp();
      ++issued;
      ring.next(stages);
    };
    for (int i = first; i < n_tiles && ok; i = next_tile(i, first, stride)) {
      const WideTile w = wide_tile(i, f_tiles, kAdM * CTAS, BN, slices);
      tids.load(ids, w.row0, rows, n);
      const int x_row = w.row0 + rank * kAdM, w_row = w.f0 + rank * (BN / CTAS);
      for (int ks = 0; ks < steps && ok; ++ks) step(&map_x, ks * kAdK, x_row, &map_w, ks * kAdK, w_row);
      if (!waited) { chain_wait(); waited = true; }
      int place = 0;                            // of the adapter among this CTA's own rows
      for (int a = tids.next(-1); a != kNone && ok; a = tids.next(a)) {
        bool here = false;
#pragma unroll
        for (int v = 0; v < 4; ++v) here |= (rank ? tids.v[4 * (CTAS - 1) + v] : tids.v[v]) == a;
        here = __any_sync(0xffffffffu, here);
        // (the other CTA's alone: rows behind the last block, which read as zeros)
        const int h_row = here ? ((x_row / kAdM * places + place) * slices.n + w.slice) * kAdM : (rows + kAdM - 1) / kAdM * places * slices.n * kAdM;
        for (int e = 0; e < h_steps && ok; ++e) step(&map_h, e * kAdK, h_row, &map_b, e % r_steps * kAdK, a * N + w_row);
        place += here;
      }
    }
    if (!waited) chain_wait();
    // copies still on their way land in this CTA's shared memory (the even CTA's barriers count both CTAs' bytes)
    if (!ok && lane == 0 && rank == 0) {
      for (int j = max(0, issued - stages); j < issued; ++j)
        for (unsigned i = 0; i < (1u << 20); ++i)
          if (mbar_try(&bars->full[j % stages], (j / stages) & 1)) break;
    }
    __syncwarp();
  } else if (warp == 1 && rank == 0) {
    // ---- MMA ----------------------------------------------------------------------------------------------------------------
    int done = 0;
    bool ok = true;
    Ring ring;
    const unsigned idesc = ad_instr_desc(BN, kAdM * CTAS);
    for (int i = first; i < n_tiles && ok; i = next_tile(i, first, stride), ++done) {
      const WideTile w = wide_tile(i, f_tiles, kAdM * CTAS, BN, slices);
      tids.load(ids, w.row0, rows, n);
      const int ab = done & 1;
      const unsigned acc = tmem + ab * 256;
      if (!warp_wait_cluster(&bars->acc_empty[ab], ((done >> 1) & 1) ^ 1, stop, 2)) break;
      tc_fence_after();
      for (int ks = 0; ks < steps; ++ks, ring.next(stages)) {
        if (!warp_wait(&bars->full[ring.s], ring.phase, stop, 3)) { ok = false; break; }
        tc_fence_after();
        unsigned char* st = stage0 + (size_t)ring.s * stage_bytes;
        const unsigned long long da = smem_desc(st), db = smem_desc(st + kAdTile);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < kAdK / 16; ++kk) mma<CTAS>(acc, da + 2 * kk, db + 2 * kk, idesc, ks > 0 || kk > 0 ? 1u : 0u);
          commit<CTAS>(&bars->empty[ring.s]);
        }
        __syncwarp();
      }
      for (int a = tids.next(-1); a != kNone && ok; a = tids.next(a)) {
        for (int e = 0; e < h_steps; ++e, ring.next(stages)) {
          if (!warp_wait(&bars->full[ring.s], ring.phase, stop, 3)) { ok = false; break; }
          tc_fence_after();
          unsigned char* st = stage0 + (size_t)ring.s * stage_bytes;
          const unsigned long long dh = smem_desc(st), db = smem_desc(st + kAdTile);
          const int n_kk = min(R, kAdK) / 16;
          if (elect_one()) {
            for (int kk = 0; kk < n_kk; ++kk) {
              mma<CTAS>(acc, dh + 2 * kk, db + 2 * kk, idesc, 1u);
              if (R <= 32) mma<CTAS>(acc, dh + 2 * (n_kk + kk), db + 2 * kk, idesc, 1u);
            }
            commit<CTAS>(&bars->empty[ring.s]);
          }
          __syncwarp();
        }
      }
      if (ok && elect_one()) commit<CTAS>(&bars->acc_full[ab]);
      __syncwarp();
    }
  } else if (warp >= 2) {
    // ---- epilogue: tensor-memory lanes 32 * (warp % 4) .. + 31, every other run of 32 columns --------------------------------
    const int quad = warp & 3, half = (warp - 2) >> 2;
    int done = 0;
    for (int i = first; i < n_tiles; i = next_tile(i, first, stride), ++done) {
      const WideTile w = wide_tile(i, f_tiles, kAdM * CTAS, BN, slices);
      const int ab = done & 1;
      if (!warp_wait(&bars->acc_full[ab], (done >> 1) & 1, stop, 4)) break;
      tc_fence_after();
      const int t0 = w.row0 + rank * kAdM + quad * 32, count = min(32, rows - t0);
      constexpr int P = 16 / (int)sizeof(TY);              // numbers of a 16-byte piece
      const bool whole = N % P == 0 && w.f0 % P == 0 && w.width % P == 0;
      unsigned char* turned = stage0 + (size_t)stages * stage_bytes + (warp - 2) * kTurnBytes;
      for (int c0 = half * 32; c0 < BN; c0 += 64) {
        unsigned v[32];
        if (c0 < w.width) {
          tc_ld32(tmem + ab * 256 + ((unsigned)(quad * 32) << 16) + c0, v);
          tc_wait_ld();
        }
        if (c0 + 64 >= BN) {                      // the last this warp reads of the accumulator
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_leader<CTAS>(&bars->acc_empty[ab]);
        }
        if (c0 >= w.width) continue;
        if constexpr (P == 4) {
          // A lane's 32 sums are a whole line of its row: stored from here.
          if (lane < count) {
            float* to = y + (size_t)(t0 + lane) * N + w.f0 + c0;
#pragma unroll
            for (int c = 0; c < 32; c += 4) {
              if (whole) {
                if (c0 + c < w.width) *reinterpret_cast<uint4*>(to + c) = make_uint4(v[c], v[c + 1], v[c + 2], v[c + 3]);
              } else {
#pragma unroll
                for (int e = c; e < c + 4; ++e)
                  if (c0 + e < w.width) to[e] = __uint_as_float(v[e]);
              }
            }
          }
          __syncwarp();
        } else {
          // A lane has 64 bytes of a row of its own: stored from there, every store of a warp goes to 32 lines.  The results change hands
          // in shared memory, and a store covers 64 bytes of eight rows (5537 rows of 824 x 7392 93 -> 78 us), or, where rows of y are not
          // 16-byte pieces, of one.
          __syncwarp();
#pragma unroll
          for (int c = 0; c < 32; c += 8) {
            __nv_bfloat162 o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = __floats2bfloat162_rn(__uint_as_float(v[c + 2 * e]), __uint_as_float(v[c + 2 * e + 1]));
            *reinterpret_cast<uint4*>(turned + lane * kTurnRow + 2 * c) = *reinterpret_cast<uint4*>(o);
          }
          __syncwarp();
          if (whole) {
            const int c = c0 + 8 * (lane & 3);
            __nv_bfloat16* to = y + (size_t)t0 * N + w.f0 + c;
            if (c < w.width) {                      // (whole: widths are multiples of 8)
#pragma unroll
              for (int r = lane >> 2; r < 32; r += 8)
                if (r < count) *reinterpret_cast<uint4*>(to + (size_t)r * N) = *reinterpret_cast<const uint4*>(turned + r * kTurnRow + 16 * (lane & 3));
            }
          } else if (c0 + lane < w.width) {
            unsigned short* to = reinterpret_cast<unsigned short*>(y) + (size_t)t0 * N + w.f0 + c0 + lane;
#pragma unroll 8
            for (int r = 0; r < count; ++r) to[(size_t)r * N] = *reinterpret_cast<const unsigned short*>(turned + r * kTurnRow + 2 * lane);
          }
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  if (CTAS == 2) cluster_barrier();       // the even CTA's products read the odd one's shared memory
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tc_dealloc<CTAS>(tmem, 512);
  }
}

// ---- few rows ----------------------------------------------------------------------------------------------------------------

constexpr int kRowsMost = 64;              // rows that adapter_rows_kernel takes whatever the other sizes
constexpr int kStagedLeast = 128, kBlocksAbove = 512;      // numbers of h of a member's rows and a slice: see RowsForm

struct __align__(8) RowsBars {
  unsigned long long full[kAdMaxStages], empty[kAdMaxStages], acc_full;
  unsigned tmem_base;
  int stop;
};

// grid: (members of the cluster, feature tiles).  320 threads: producer, MMA, eight epilogue warps (two threads a feature, rows of
// x in turn).
constexpr int kRowsThreads = 320;
enum RowsForm { kRowsPlain, kRowsStaged, kRowsBlocks };
constexpr int kRowsAtOnce = 4;             // rows of x whose rows of B a thread has under way

// The adapters' part, by FORM.  kRowsPlain: added up by a thread a feature, which reads its row of B while W is read, and h.
// kRowsStaged: a member fetches h of its rows at once, into the stages, which nothing uses any more by then; read where it is used, every
// row and 16 ranks are a trip to L2 in turn (64 rows of 2048 x 9216 and rank 16 21.1 us instead of 22.5; a single row 8.1 instead of 7.1).
// kRowsBlocks: steps of the product, h in the blocks of the wide kernel, rows of B brought into L2 while W is read.  64 rows of 2048 x
// 3584, 24 adapters: rank 16 18.3 us instead of 12.2, the products, their sums and their way to the owners now come behind h; rank 64 23.1
// instead of 36.1, rank 128 35.6 instead of 62.8.
// What bounds it: one row of 2048 x 2048 takes 7.5 us, its 8.4 MB 1.3: launch, the first loads, the members' sums, h and the rows of y,
// one after the other.  64 rows of 3584 x 3584 with 48 adapters of rank 32 take 19.6 us, their 43 MB 6.7: h is there after 12, W's sums
// by then, and the adapters' part takes 4.
template <RowsForm FORM, typename TY>
__global__ void __launch_bounds__(kRowsThreads, 2)
adapter_rows_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_b,
                    const __grid_constant__ CUtensorMap map_h, const int* __restrict__ ids, const float* __restrict__ h,
                    const __nv_bfloat16* __restrict__ B, TY* __restrict__ y, int rows, int N, int K, int R, int n,
                    const __grid_constant__ TcSlices slices, int NT, int stages) {
  constexpr bool STAGED = FORM == kRowsStaged, BLOCKS = FORM == kRowsBlocks;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  RowsBars* bars = reinterpret_cast<RowsBars*>(smem);
  unsigned char* stage0 = smem + 1024;
  const int stage_bytes = kAdTile + NT * 128;
  float* sums = reinterpret_cast<float*>(stage0 + (size_t)stages * stage_bytes);      // [members][share of rows][128], written by all members
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int members = gridDim.x, member = blockIdx.x;          // the cluster is the grid's first dimension
  const int share = (rows + members - 1) / members;            // rows of x that a member adds up: [member * share, ...)
  volatile int* stop = &bars->stop;
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");      // this member is there
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) { mbar_init(&bars->full[s], 1); mbar_init(&bars->empty[s], 1); }
    mbar_init(&bars->acc_full, 1);
    bars->stop = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncwarp();
  const unsigned columns = NT > 64 ? 128 : 64;
  if (warp == 1) tc_alloc<1>(&bars->tmem_base, columns);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const unsigned tmem = bars->tmem_base;
  const WideTile w = wide_tile(blockIdx.y, gridDim.y, kAdM, kAdM, slices);
  const int steps = (K + kAdK - 1) / kAdK;
  const int k_first = (int)((long long)member * steps / members), k_last = (int)((long long)(member + 1) * steps / members);
  const int quad = warp & 3, turn = warp >= 6 ? 1 : 0;         // (epilogue warps)
  const int d = quad * 32 + lane, f = w.f0 + d;
  const int t_first = member * share, t_last = min(rows, t_first + share);

  // a thread's rows of x: t_first + turn, + 2, ...; their adapters and rows of B
  int a[kRowsAtOnce];
  uint4 raw[kRowsAtOnce][2];
  auto ask = [&](int t0) {
#pragma unroll
    for (int i = 0; i < kRowsAtOnce; ++i) {
      const int t = t0 + 2 * i;
      a[i] = t < t_last ? ids[t] : -1;
    }
#pragma unroll
    for (int i = 0; i < kRowsAtOnce; ++i) {
      if (a[i] >= n && blockIdx.y == 0 && d == 0) atomicCAS(&g_adapter_tc_index, 0, t0 + 2 * i + 1);
      if (a[i] >= n || d >= w.width) a[i] = -1;
      if (a[i] >= 0) {
        const uint4* b = reinterpret_cast<const uint4*>(B + ((size_t)a[i] * N + f) * R);
        raw[i][0] = b[0];
        raw[i][1] = b[1];
      }
    }
  };

  // BLOCKS: this member's adapters, those whose place among the rows' is the member's modulo the members; an adapter's steps as in the
  // wide kernel
  const int r_steps = (R + kAdK - 1) / kAdK, h_steps = R <= 32 ? 1 : 2 * r_steps;
  TileIds<1> tids;
  if (BLOCKS && warp < 3) tids.load(ids, 0, rows, n);
  auto own_adapters = [&](auto each) {         // each(adapter, place) until it says no
    int place = 0;
    for (int a = tids.next(-1); a != kNone; a = tids.next(a), ++place)
      if (place % members == member && !each(a, place)) break;
  };

  if (warp == 0) {
    Ring ring;
    int issued = 0;
    const int count = k_last - k_first;
    auto step = [&](const CUtensorMap* mw, int kw, int w_row, const CUtensorMap* mx, int kx, int x_row) {
      if (!warp_wait(&bars->empty[ring.s], ring.phase ^ 1, stop, 11)) return false;
      unsigned char* st = stage0 + (size_t)ring.s * stage_bytes;
      if (elect_one()) {
        mbar_expect_tx(&bars->full[ring.s], stage_bytes);
        tma_load_2d(st, mw, kw, w_row, &bars->full[ring.s]);
        tma_load_2d(st + kAdTile, mx, kx, x_row, &bars->full[ring.s]);
      }
      __syncwarp();
      ++issued;
      ring.next(stages);
      return true;
    };
    bool ok = true;
    for (int it = 0; it < count && ok; ++it) ok = step(&map_w, (k_first + it) * kAdK, w.f0, &map_x, (k_first + it) * kAdK, 0);
    if (BLOCKS) {
      chain_wait();
      if (ok)
        own_adapters([&](int a, int place) {
          for (int e = 0; e < h_steps && ok; ++e)
            ok = step(&map_b, e % r_steps * kAdK, a * N + w.f0, &map_h, e * kAdK, (place * slices.n + w.slice) * kAdM);
          return ok;
        });
    }
    if (!ok)
      for (int j = max(0, issued - stages); j < issued; ++j)
        for (unsigned i = 0; i < (1u << 20); ++i)
          if (mbar_try(&bars->full[j % stages], (j / stages) & 1)) break;
    __syncwarp();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  } else if (warp == 1) {
    Ring ring;
    const unsigned idesc = ad_instr_desc(NT, kAdM);
    const int count = k_last - k_first;
    bool ok = true;
    for (int it = 0; it < count; ++it, ring.next(stages)) {
      if (!warp_wait(&bars->full[ring.s], ring.phase, stop, 13)) { ok = false; break; }
      tc_fence_after();
      unsigned char* st = stage0 + (size_t)ring.s * stage_bytes;
      const unsigned long long dw = smem_desc(st), dx = smem_desc(st + kAdTile);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < kAdK / 16; ++kk) tc_mma(tmem, dw + 2 * kk, dx + 2 * kk, idesc, it > 0 || kk > 0 ? 1u : 0u);
        tc_commit(&bars->empty[ring.s]);
        if (!BLOCKS && it + 1 == count) tc_commit(&bars->acc_full);
      }
      __syncwarp();
    }
    if (BLOCKS && ok) {
      const int n_kk = min(R, kAdK) / 16;
      own_adapters([&](int, int) {
        for (int e = 0; e < h_steps; ++e, ring.next(stages)) {
          if (!warp_wait(&bars->full[ring.s], ring.phase, stop, 13)) return ok = false;
          tc_fence_after();
          unsigned char* st = stage0 + (size_t)ring.s * stage_bytes;
          const unsigned long long db = smem_desc(st), dh = smem_desc(st + kAdTile);
          if (elect_one()) {
            for (int kk = 0; kk < n_kk; ++kk) {
              tc_mma(tmem, db + 2 * kk, dh + 2 * kk, idesc, 1u);
              if (R <= 32) tc_mma(tmem, db + 2 * kk, dh + 2 * (n_kk + kk), idesc, 1u);
            }
            tc_commit(&bars->empty[ring.s]);
          }
          __syncwarp();
        }
        return true;
      });
      if (ok && elect_one()) tc_commit(&bars->acc_full);
      __syncwarp();
    }
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  } else {
    if (BLOCKS) {
      // rows of B into L2 while W is read: the steps that fetch them wait for h
      if (warp == 2)
        own_adapters([&](int a, int) {
          if (lane == 0)
            asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(B + ((size_t)a * N + w.f0) * R), "r"(w.width * R * 2) : "memory");
          return true;
        });
    } else {
      ask(t_first + turn);
    }
    __syncwarp();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");      // every member is there: its shared memory may be written
    if (warp_wait(&bars->acc_full, 0, stop, 14)) {
      tc_fence_after();
      // this CTA's sums go to the members that own the rows
      for (int c0 = 16 * turn; c0 < NT; c0 += 32) {
        unsigned v[16];
        tc_ld16(tmem + ((unsigned)(quad * 32) << 16) + c0, v);
        tc_wait_ld();
        int to = c0 / share, tl = c0 - to * share;
        const unsigned mine = smem_u32(sums + (size_t)member * share * kAdM + d);
        unsigned at = cluster_addr(mine, min(to, members - 1));
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          if (c0 + c < rows) asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(at + tl * kAdM * 4), "r"(v[c]) : "memory");
          if (++tl == share) { tl = 0; ++to; at = cluster_addr(mine, min(to, members - 1)); }
        }
      }
    }
    tc_fence_before();
  }
  __syncwarp();
  cluster_barrier();                   // all sums are there, and nothing of tensor memory is still to be read
  if (warp == 1) {
    tc_fence_after();
    tc_dealloc<1>(tmem, columns);
  }
  if (warp >= 2) {
    const int SR = slices.n * R;
    float* hs = reinterpret_cast<float*>(stage0);
    float sum[kRowsAtOnce];
    auto add_up = [&](int t0) {          // the members' sums, in their order
#pragma unroll
      for (int i = 0; i < kRowsAtOnce; ++i) {
        const int tl = min(t0 + 2 * i, t_last - 1) - t_first;
        sum[i] = 0.f;
        for (int m = 0; m < members; ++m) sum[i] += sums[((size_t)m * share + tl) * kAdM + d];
      }
    };
    if (BLOCKS) {
      for (int t0 = t_first + turn; t0 < t_last; t0 += 2 * kRowsAtOnce) {
        add_up(t0);
#pragma unroll
        for (int i = 0; i < kRowsAtOnce; ++i)
          if (t0 + 2 * i < t_last && d < w.width) y[(size_t)(t0 + 2 * i) * N + f] = from_float<TY>(sum[i]);
      }
      return;
    }
    if (STAGED && t_first < t_last) add_up(t_first + turn);
    chain_wait(h);
    if (STAGED) {
      const int pieces = R >> 2;
      for (int i = threadIdx.x - 64; i < (t_last - t_first) * pieces; i += kRowsThreads - 64) {
        const int tl = i / pieces;
        float v[4];
        load4(h + (size_t)(t_first + tl) * SR + w.slice * R + 4 * (i - tl * pieces), v);
        store4(hs + 4 * i, v);
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
    }
    for (int t0 = t_first + turn; t0 < t_last; t0 += 2 * kRowsAtOnce) {
      if (t0 != t_first + turn) ask(t0);
      if (!STAGED || t0 != t_first + turn) add_up(t0);
      for (int j = 0; j < R; j += 16) {
        if (j > 0) {
#pragma unroll
          for (int i = 0; i < kRowsAtOnce; ++i)
            if (a[i] >= 0) {
              const uint4* b = reinterpret_cast<const uint4*>(B + ((size_t)a[i] * N + f) * R + j);
              raw[i][0] = b[0];
              raw[i][1] = b[1];
            }
        }
#pragma unroll
        for (int i = 0; i < kRowsAtOnce; ++i)
          if (a[i] >= 0) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float bv[8], hv[8];
              unpack8(raw[i][c], bv);
              if (STAGED) load8(hs + (t0 + 2 * i - t_first) * R + j + 8 * c, hv);
              else load8(h + (size_t)(t0 + 2 * i) * SR + w.slice * R + j + 8 * c, hv);
#pragma unroll
              for (int e = 0; e < 8; ++e) sum[i] = fmaf(hv[e], bv[e], sum[i]);
            }
          }
      }
#pragma unroll
      for (int i = 0; i < kRowsAtOnce; ++i)
        if (t0 + 2 * i < t_last && d < w.width) y[(size_t)(t0 + 2 * i) * N + f] = from_float<TY>(sum[i]);
    }
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
  // An SM that runs one kernel with a part of its memory as shared memory takes no CTA of the next one that needs more.
  cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
  return 0;
}

// Clusters of `members` (1, 2, 4 or 8) CTAs that run at once.  A cluster lies within a part of the device, whose SMs are no multiple of
// 4 or 8 (of a CTA that fills an SM 74 clusters of two, 33 of four, 15 of eight), and clusters beyond that begin when others end.
template <typename F>
int clusters_at_once(F* kernel, int threads, size_t smem, int members) {
  static int known[4] = {};
  int& n = known[members == 8 ? 3 : members >> 1];
  if (!n) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(members);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = members;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) n = 1;
  }
  return n;
}

}  // namespace

int adapter_shrink_simt(const void* x, const void* A, const float* scale, const int* ids, float* h, int rows, int K, int SR, int n,
                        cudaStream_t stream);

}  // namespace nf

using namespace nf;

// Blocks of 128 rows of h that a row tile may need: the adapters that may occur in it.
static int adapter_places(int rows, int n) {
  const int most = rows < kAdM ? rows : kAdM;
  return n < most ? n : most;
}

// Rows that one pass serves: all, unless h would take more than kScratchBytes (many adapters, many ranks, many rows).
constexpr long long kScratchBytes = 256ll << 20;
static int rows_a_pass(int rows, int SR, int n) {
  if (rows <= kRowsMost) return rows;
  const long long tile = (long long)adapter_places(rows, n) * kAdM * SR * 4;
  long long pairs = kScratchBytes / (2 * tile);
  if (pairs < 1) pairs = 1;
  return 2 * kAdM * pairs < rows ? (int)(2 * kAdM * pairs) : rows;
}

// Floats of scratch that nf_adapter_linear needs for `rows` rows, SR numbers of h a row, a pool of n adapters.
extern "C" long long nf_adapter_scratch(int rows, int SR, int n) {
  if (rows <= 16) return (long long)rows * SR;
  return (long long)((rows_a_pass(rows, SR, n) + kAdM - 1) / kAdM) * adapter_places(rows, n) * kAdM * SR;
}

// One pass; the rows that an error names are counted from its first.
template <typename TY>
static int adapter_pass(const void* x, const void* W, const void* A, const void* B, const float* scale, const int* ids, float* h, TY* y, int rows,
                        int N, int K, int R, int n, const TcSlices& sl, cudaStream_t stream) {
  const int SR = sl.n * R, steps = (K + kAdK - 1) / kAdK, n_slices = sl.n;
  const int row_tiles = (rows + kAdM - 1) / kAdM, places = adapter_places(rows, n);

  // ---- which kernel the product is, and how it is split
  const int NT = (rows + 15) & ~15, f_tiles128 = feature_tiles(sl, kAdM);
  int parts = 1, share = rows;              // members of a cluster of adapter_rows_kernel, rows of x that each adds up
  bool blocks = false;
  if (rows <= kAdM) {
    // As many members as have all clusters begin at once: two CTAs an SM, one where the first product runs (of more than 64 rows one, and
    // none); clusters of 4 and 8 leave SMs over (8 rows of 2048 x 4608: 8 members, of whose 36 clusters some came late, 12.5 us, 4 members
    // 9.7; 64 rows 19.0 and 14.9).
    const int slots = (rows > kRowsMost ? 1 : 2) * sm_count() - (rows > 16 ? sm_count() / 24 * 8 : 0);
    const auto fit = [&](int m) { return m * f_tiles128 <= (m == 2 && rows <= kRowsMost ? 2 * sm_count() : slots - 8 * (m - 1)); };
    while (parts < 8 && steps >= 4 * parts && fit(2 * parts)) parts *= 2;
    share = (rows + parts - 1) / parts;
    // (between them: a thread's numbers of h, of all the rows that it adds up; of more than 64 rows the other way is the wide kernel, which
    // splits no k: 100 rows of 3584 x 3584 and rank 16 24 us instead of 36, of 3584 x 7168, where no two members have room, 44 instead of 37)
    blocks = rows > 16 && (rows > kRowsMost ? parts > 1 : share * R > kBlocksAbove);
  }

  // The wide kernel's tile: the one whose rounds take the least, a round's time being that of the products or of the operands' way into
  // shared memory (64 bytes a cycle), whichever is the longer; below 128 features only where they leave the first product its SMs (200 rows
  // of 2048 x 5632: tiles of 64 32 us, of 128 27).
  int BN = 256, ctas = 2, wide_grid = sm_count();
  long long least = -1;
  for (int g = 2; g >= 1; --g) {
    const int m_tiles = (rows + kAdM * g - 1) / (kAdM * g), at_once = sm_count() / g;
    for (int c = 256; c >= 64; c -= 32) {
      const long long tiles = (long long)m_tiles * feature_tiles(sl, c);
      const int loads = (kAdTile + c / g * 128) / 64, step = 2 * c > loads ? 2 * c : loads;
      const long long cost = ((tiles + at_once - 1) / at_once) * step;
      if (c < 128 && 4 * tiles * g > sm_count()) break;
      if (least < 0 || cost < least) {
        least = cost;
        BN = c;
        ctas = g;
        wide_grid = tiles < at_once ? (int)tiles * g : at_once * g;
      }
    }
  }

  // ---- h
  // Few rows: a warp a number.  K 2048, N 3584, 24 adapters of rank 16, the whole call that way and on tensor cores: 17 rows 8.2 and 9.6 us,
  // 24 rows 8.4 and 10.0, 32 rows 10.2 and 9.6, 64 rows 13.4 and 12.0; K 3584, 48 adapters of rank 32: 17 rows 15.0 and 14.6, 24 rows 15.6 and
  // 16.8, 32 rows 16.3 and 17.0, 64 rows 21.6 and 19.7; K 2048, N 6144, 16 adapters of rank 16: 17 rows 11.8 and 12.8, 64 rows 16.3 and 17.0.
  if (rows <= 16) {
    if (int rc = adapter_shrink_simt(x, A, scale, ids, h, rows, K, SR, n, stream)) return rc;
  } else {
    static int asked = room_for(adapter_shrink_tc_kernel, kShrinkSmemMost);
    if (asked) return asked;
    const int JW = SR < kAdM ? SR : kAdM, j_tiles = (SR + JW - 1) / JW, tiles = row_tiles * j_tiles;
    const int most = n < kAdM ? (n < rows ? n : rows) : (rows < kAdM ? rows : kAdM);      // adapters that a tile's rows may have
    // How many members split k, and how many CTAs take a tile's adapters in turn: the least time by a simple account in cycles of what a CTA
    // and a group of adapters cost however short, of a step's bytes and of rounds of clusters, for tiles with as many adapters as may be and
    // for tiles with two (1024 rows of 2048 x 4608, 24 adapters of rank 16 among all rows: 8 members, 2 in turn 57 us, 4 and 4 38).  Behind
    // few rows comes a product that streams W: two SMs of five are enough for what it would otherwise wait for (64 rows of 3584 x 3584, 48
    // adapters of rank 32: 19.7 us, on all of them 25.3).
    const bool few = rows <= kRowsMost;
    const int cols = few || blocks ? kShrinkCols : kShrinkCols / 2;
    struct Split {
      int members, turns;
      long long cost;
    };
    const auto split = [&](int sms) {
      Split best{1, 1, -1};
      for (int m = 1; m <= 8 && (m == 1 || steps >= 2 * m); m *= 2) {
        const int at_once = clusters_at_once(adapter_shrink_tc_kernel, 192, kShrinkSmemMost, m) * sms / sm_count();
        if (at_once < 1) continue;
        const int z_most = at_once / tiles < 1 ? 1 : at_once / tiles > most ? most : at_once / tiles;
        for (int z = 1; z <= z_most; ++z) {
          const auto time = [&](int adapters) {
            const int each = (adapters + z - 1) / z, group = cols / JW < each ? cols / JW : each;
            return 6000 + (each + group - 1) / group * (2000 + (steps + m - 1) / m * (kAdTile + group * JW * 128) / 48);
          };
          const long long cost = (long long)((tiles * z + at_once - 1) / at_once) * (time(most) + time(most < 2 ? most : 2));
          if (best.cost < 0 || cost < best.cost) best = {m, z, cost};
        }
      }
      return best;
    };
    const int least_room = sm_count() * 2 / 5;
    Split plan = split(few ? least_room : blocks ? sm_count() - parts * f_tiles128 : sm_count());
    // A wide kernel that needs few SMs runs beside the first product where that is not much longer for it (512 rows of 2048 x 2048 34 -> 26 us).
    if (!few && !blocks && 4 * wide_grid <= 3 * sm_count()) {
      const Split beside = split(sm_count() - wide_grid > least_room ? sm_count() - wide_grid : least_room);
      if (4 * beside.cost <= 5 * plan.cost) plan = beside;
    }
    const int members = plan.members, turns = plan.turns;
    const int each = (most + turns - 1) / turns, group = cols / JW < each ? cols / JW : each;
    const int x_box = rows >= kAdM ? kAdM : (rows + 7) & ~7;
    CUtensorMap ma, mx;
    if (int rc = make_map(&ma, A, (long long)n * SR, K, JW)) return rc;
    if (int rc = make_map(&mx, x, rows, K, x_box)) return rc;
    const int stage = kAdTile + group * JW * 128, sums = kAdM * (JW + 4) * 4;
    int stages = ((few ? (int)kShrinkSmemLeast - 2048 : 200 * 1024) - sums) / stage;
    stages = stages > 8 ? 8 : stages < 2 ? 2 : stages;
    size_t smem = 2048 + (size_t)stages * stage + sums;
    smem = smem < kShrinkSmemLeast ? kShrinkSmemLeast : smem;
    NF_REQUIRE(tiles <= 65535, "adapter_linear: %d rows are too many", rows);
    launch_chained_cluster(adapter_shrink_tc_kernel, dim3(members, tiles, turns), dim3(192), smem, stream, members, ma, mx, scale,
                           ids, h, rows, K, SR, n, row_tiles, x_box, JW, group, stages, few && !blocks ? 0 : places, R);
    if (int rc = check_launch("adapter_shrink")) return rc;
  }

  // ---- the shared product and the adapters' part
  CUtensorMap mx, mw, mb, mh;
  if (rows <= kRowsMost || blocks) {
    if (int rc = make_map(&mw, W, N, K, kAdM)) return rc;
    if (int rc = make_map(&mx, x, rows, K, NT)) return rc;
    const int stage = kAdTile + NT * 128, here = (steps + parts - 1) / parts, sums = parts * share * kAdM * 4;
    int stages = ((NT > 64 ? 200 : 104) * 1024 - sums) / stage;
    if (!blocks) {
      stages = stages > here ? here : stages;
      while (stages * stage < share * R * 4) ++stages;      // (h of a member's rows takes their place)
    }
    stages = stages > kAdMaxStages ? kAdMaxStages : stages;
    const size_t smem = 2048 + (size_t)stages * stage + sums;
    static int asked = room_for(adapter_rows_kernel<kRowsPlain, TY>, 108 * 1024), asked_staged = room_for(adapter_rows_kernel<kRowsStaged, TY>, 108 * 1024),
               asked_blocks = room_for(adapter_rows_kernel<kRowsBlocks, TY>, 204 * 1024);
    if (asked || asked_staged || asked_blocks) return 1;
    NF_REQUIRE(f_tiles128 <= 65535, "adapter_linear: %d features are too many", N);
    mb = mh = mw;
    if (blocks) {
      if (int rc = make_map(&mb, B, (long long)n * N, R, kAdM)) return rc;
      if (int rc = make_map(&mh, h, (long long)places * n_slices * kAdM, 2 * R, NT)) return rc;
    }
    const auto kernel = blocks ? adapter_rows_kernel<kRowsBlocks, TY>
                               : share * R >= kStagedLeast ? adapter_rows_kernel<kRowsStaged, TY> : adapter_rows_kernel<kRowsPlain, TY>;
    launch_chained_cluster(kernel, dim3(parts, f_tiles128), dim3(kRowsThreads), smem, stream, parts, mw, mx, mb, mh, ids, (const float*)h,
                           (const __nv_bfloat16*)B, y, rows, N, K, R, n, sl, NT, stages);
    return check_launch("adapter_rows");
  }
  if (int rc = make_map(&mx, x, rows, K, kAdM)) return rc;
  if (int rc = make_map(&mw, W, N, K, BN / ctas)) return rc;
  if (int rc = make_map(&mb, B, (long long)n * N, R, BN / ctas)) return rc;
  if (int rc = make_map(&mh, h, (long long)row_tiles * places * n_slices * kAdM, 2 * R, kAdM)) return rc;
  const int f_tiles = feature_tiles(sl, BN);
  const long long n_tiles = (long long)f_tiles * ((rows + kAdM * ctas - 1) / (kAdM * ctas));
  NF_REQUIRE(n_tiles < (1ll << 30), "adapter_linear: %d rows of %d features are too many", rows, N);
  int stages = (kWideSmem - kWideHead - kWideEpilogueWarps * kTurnBytes) / (kAdTile + BN / ctas * 128);
  stages = stages > kAdMaxStages ? kAdMaxStages : stages;
  static int asked1 = room_for(adapter_wide_kernel<1, TY>, kWideSmem + 1024), asked2 = room_for(adapter_wide_kernel<2, TY>, kWideSmem + 1024);
  if (asked1 || asked2) return 1;
  const int at_once = sm_count() / ctas, grid = ctas * (n_tiles < at_once ? (int)n_tiles : at_once);
  if (ctas == 2)
    launch_chained_cluster(adapter_wide_kernel<2, TY>, dim3(grid), dim3(kWideThreads), (size_t)kWideSmem + 1024, stream, 2, mx, mw, mb, mh, ids,
                           y, rows, N, K, R, n, places, sl, f_tiles, (int)n_tiles, BN, stages);
  else
    launch_chained(adapter_wide_kernel<1, TY>, dim3(grid), dim3(kWideThreads), (size_t)kWideSmem + 1024, stream, mx, mw, mb, mh, ids,
                   y, rows, N, K, R, n, places, sl, f_tiles, (int)n_tiles, BN, stages);
  return check_launch("adapter_wide");
}

// y = x W^T + the adapters' part (see the head of this file): x [rows, K], W [N, K], A [n, n_slices * R, K], B [n, N, R], y
// [rows, N] bfloat16 (y float32 where y_dtype says so); scale float32 [n]; ids [rows], -1 for none; h: scratch of nf_adapter_scratch(rows, n_slices * R, n)
// floats.  ends: the n_slices features (host memory) at which the slices end, the last N.  K a multiple of 8, R 16, 32, 64
// or 128, bases 16-byte aligned.
extern "C" int nf_adapter_linear(const void* x, const void* W, const void* A, const void* B, const float* scale, const int* ids, float* h,
                                 void* y, int rows, int N, int K, int R, int n, int n_slices, const int* ends, int y_dtype, cudaStream_t stream) {
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
  const int pass = rows_a_pass(rows, n_slices * R, n);
  for (int t = 0; t < rows; t += pass) {
    const int now = rows - t < pass ? rows - t : pass;
    const auto pass_to = [&](auto* to) {
      return adapter_pass((const __nv_bfloat16*)x + (size_t)t * K, W, A, B, scale, ids + t, h, to + (size_t)t * N, now, N, K, R, n, sl, stream);
    };
    if (int rc = y_dtype == kF32 ? pass_to((float*)y) : pass_to((__nv_bfloat16*)y)) return rc;
  }
  return 0;
}

// 0, or the code of the first wait that one of these kernels gave up on since the last call (1 to 4 the wide form and the
// first product, 11 to 14 the form for few rows); 100 + 1 + a row whose adapter lay outside the pool.  Synchronises.
extern "C" int nf_adapter_tc_status() {
  int v[2] = {0, 0}, zero = 0;
  if (cudaMemcpyFromSymbol(&v[0], g_adapter_tc_error, sizeof(int)) != cudaSuccess) return -1;
  if (cudaMemcpyFromSymbol(&v[1], g_adapter_tc_index, sizeof(int)) != cudaSuccess) return -1;
  if (v[0]) cudaMemcpyToSymbol(g_adapter_tc_error, &zero, sizeof(int));
  if (v[1]) cudaMemcpyToSymbol(g_adapter_tc_index, &zero, sizeof(int));
  return v[0] ? v[0] : (v[1] ? 100 + v[1] : 0);
}
