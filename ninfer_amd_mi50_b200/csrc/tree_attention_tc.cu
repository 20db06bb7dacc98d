// Attention of trees of drafted tokens in bfloat16 on the 5th-generation tensor cores (tree_attention.cu says what is
// computed).  All (node, query head) pairs of a key head read the same keys, so they are the rows of one product, 128 a
// tile.  A CTA a SM walks its items, each some keys of a request's key head and one or two tiles of pairs; the copies for an
// item are on their way while the one before it is worked off.
//
//   warps 0, 2   producers of keys and of values: TMA copies (128-byte swizzle), page by page through the block table, in
//                blocks of 128 keys, into rings
//   warp 1       issuer of ``tcgen05.mma``: S = Q K^T (128 x 128) and O += P V, with P out of tensor memory
//   warps 4-11   two softmax groups, a thread a row: the queries of the item to come, then 64 scores at a time, a reference
//                maximum that is raised only when a score passes it by 8 in the exponent (O's row, and the weights of the
//                step's first half, are then rescaled), weights 2^(s - m) rounded to bfloat16 in the place of the scores
//
// Each group has an S and an O of its own in tensor memory (128 columns each, all 512).  With two tiles of pairs a group
// takes one of them and both read each block of keys; with one tile they take every other block, and their sums are put
// together at the end.  Either way one group's exponentials run under the other's products.  The products are issued by
// one thread and run in its order, PV(A), QK(A), PV(B), QK(B): the scores of a step are there only when the sums of the step
// before are, and P, which lies where S did, and O need no signs of their own.
//
// Only blocks that reach behind the keys that the request held are masked, and those that lack a page: there a thread shifts
// its row's mask so that bit i says whether its i-th score counts.  Keys behind the last node or without a page are masked and
// their values set to zero, since whatever lies there would be multiplied by a weight of nothing.
//
// The weights are rounded to bfloat16 for the second product (an error of 2^-8 of a weight at most, as independent from
// key to key as the rounding of the result), a second time where the step's second half makes them less than 2^-8 of the
// largest; their sum is of the unrounded ones.  Scores, maxima, sums and O are float32.
//
// What bounds it: 128 x 128 scores take a group some 3,700 cycles, of which the exponentials of both groups are 2,050 on their
// own pipe and the products 2,060, one behind the other (the first waits for the scores, the second for the weights).  At this
// rate the GPU draws its 1,000 W and runs at 1.7 instead of 1.97 GHz, so that what shortens the chain gains less than it
// saves.  16 requests as below: 224 us in a replayed graph, 0.63 PFLOP/s of what the formula asks for, a quarter of the rows being padding.
//
// Every wait is bounded: the one that runs out records a code in `g_tree_tc_error` and sets `stop`, upon which the other
// waits run out too, the CTA's warps leave, wait (bounded) for copies in flight, and free tensor memory.
#include "tcgen05.cuh"
#include "tree_attention.cuh"

namespace nf {
namespace {

constexpr int kRows = 128;       // pairs of a CTA (MMA M)
constexpr int kKeys = 128;       // keys per block
constexpr int kThreads = 384;
constexpr int kMostRequests = 512;    // of a launch: their numbers lie in shared memory
constexpr int kAtom = 128 * 128; // bytes of a swizzle atom column: 128 rows x 64 bf16
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRaise = 8.f;

__device__ int g_tree_tc_error = 0;
__device__ int g_tree_tc_index = 0;

struct __align__(8) Barriers {
  unsigned long long q_full, q_empty, k_full[4], k_empty[4], v_full[4], v_empty[4], s_full[2], p_full[2], o_final[2], o_read;
  unsigned tmem_base;
  // Of the last blocks of keys, bit i: the i-th page is missing, and in its place lies what lay there before.  A word is read
  // until the block's weights are there, by when the producer is at most STAGES + 1 blocks ahead: twice as many words as stages
  unsigned lacking[8];
  int stop, quit[2];
};

struct Requests {
  long long start[kMostRequests + 1];   // where each request's work begins on the line
  long long quota;                      // of a CTA
  int row0[kMostRequests], nodes[kMostRequests], len[kMostRequests], keys[kMostRequests];
};

// Descriptor of an MN-major operand with 128-byte swizzle: 64 contiguous MN elements a row, rows = k, the next 64 MN
// elements `lbo` bytes further.
__device__ __forceinline__ unsigned long long smem_desc_mn(const void* p, unsigned lbo) {
  unsigned long long d = 0;
  d |= (unsigned long long)((smem_u32(p) & 0x3FFFFu) >> 4);
  d |= (unsigned long long)(lbo >> 4) << 16;
  d |= (unsigned long long)(1024 >> 4) << 32;
  d |= (unsigned long long)1 << 46;
  d |= (unsigned long long)2 << 61;
  return d;
}
// bf16 x bf16 -> f32, M = 128, N = n; b_mn: the B operand is MN-major.
__device__ __forceinline__ unsigned mma_desc(int n, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn ? (1u << 16) : 0u) | ((unsigned)(n >> 3) << 17) | ((unsigned)(kRows >> 4) << 24);
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float x, float y, float z) {
  float v;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(v) : "f"(x), "f"(y), "f"(z));
  return v;
}

// Two float32 in one register pair, which this architecture multiplies and adds at once.
__device__ __forceinline__ unsigned long long pair_of(float x, float y) {
  unsigned long long v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y));
  return v;
}
__device__ __forceinline__ void halves(unsigned long long v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ unsigned long long fma2(unsigned long long x, unsigned long long y, unsigned long long z) {
  unsigned long long v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(x), "l"(y), "l"(z));
  return v;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long x, unsigned long long y) {
  unsigned long long v;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(x), "l"(y));
  return v;
}

// Scores that are not seen become -inf: their weight is exactly zero.
__device__ __forceinline__ void hide(unsigned* u, unsigned seen) {
#pragma unroll
  for (int i = 0; i < 32; ++i)
    if (!(seen >> i & 1)) u[i] = 0xff800000u;
}

// A bounded wait of a whole warp: all its lanes go on, or none.
__device__ __forceinline__ bool warp_wait(void* bar, unsigned parity, volatile int* stop, int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, stop, code, &g_tree_tc_error));
}

// The work of a launch lies on a line: request after request, their key heads, their units of two tiles of pairs and at the
// end, where one tile is left, of one; a unit's length is kAround, for what comes before and behind its blocks, and kTwo or
// kOne for each block of keys (in hundreds of cycles, as measured with heads of 128; with heads of 64 they are no measure of
// time, and only say how the line is shared).  Each CTA takes as much of the line: the end of a unit that another began, units
// as a whole, and the beginning of one.  (Replayed graphs: 16 requests of 32 to 64 nodes behind 8,192 to 16,384 keys, 28 query
// heads of 128: 224 us, and 241 with shares of one length dealt to CTAs, the longest first; one of 100 nodes behind 65,536 keys
// 132 and 140; four of up to 64 behind 30,000, 16 key heads 144 and 161.  The first with heads of 64: 174.)  Block b of a unit
// that begins at `o` is the CTA's within whose part o + kAround + b * kTwo lies.
constexpr int kTwo = 37, kOne = 22, kAround = 120;
constexpr int kLeast = 4 * kOne;          // of a CTA's part: 256 keys and more

__host__ __device__ __forceinline__ int two_tiles(int pairs) { return (pairs + kRows - 1) / (2 * kRows); }       // units of two tiles
__device__ __forceinline__ int blocks_of(int keys) { return (keys + kKeys - 1) / kKeys; }
// The units of a request's key head, and their length on the line.
struct Units {
  int twos, all, blocks;
  __device__ __forceinline__ Units(int pairs, int keys) : twos(two_tiles(pairs)), blocks(blocks_of(keys)) { all = twos + (pairs > twos * 2 * kRows); }
  __device__ __forceinline__ int block(int u) const { return u < twos ? kTwo : kOne; }
  __device__ __forceinline__ int length(int u) const { return kAround + block(u) * blocks; }      // (below 2^30 / 128 * 37)
  __device__ __forceinline__ long long head() const { return (long long)twos * length(0) + (all > twos ? length(twos) : 0); }
};

// What a CTA works on at a time: blocks of keys of a unit, of (request s, key head g), and `tiles` (1 or 2) tiles of pairs.
struct Item {
  int s, g, unit, pair0, pairs, tiles, first, last, blocks, row0, len, keys;
  bool begins, whole;                   // has the unit's first block; all of them
  long long at;                         // where the unit `unit` begins, which is the one after this item's
  __device__ __forceinline__ int steps(int group) const { return tiles == 2 ? blocks : (blocks + 1 - group) >> 1; }
  __device__ __forceinline__ int block(int group, int step) const { return tiles == 2 ? step : 2 * step + group; }
};
// The beginning of the CTA's part.
__device__ __forceinline__ void first_item(const TreeArgs& a, const Requests& q, Item& t) {
  const long long begin = blockIdx.x * q.quota;
  int lo = 0, hi = a.S;                 // the last request that begins at or before it
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (q.start[mid] <= begin) lo = mid; else hi = mid;
  }
  const long long head = Units(q.nodes[lo] * (a.Hq / a.Hkv), q.keys[lo]).head();
  t.s = lo, t.g = t.unit = 0, t.at = q.start[lo];
  while (t.g < a.Hkv - 1 && t.at + head <= begin) ++t.g, t.at += head;
}
// The next item; false behind the CTA's last.
__device__ __forceinline__ bool next_item(const TreeArgs& a, const Requests& q, Item& t) {
  const long long begin = blockIdx.x * q.quota, end = begin + q.quota;
  while (t.s < a.S && t.at < end) {
    t.pairs = q.nodes[t.s] * (a.Hq / a.Hkv), t.keys = q.keys[t.s];
    const Units units(t.pairs, t.keys);
    if (t.unit >= units.all) {
      t.unit = 0;
      if (units.all == 0 || ++t.g == a.Hkv) t.g = 0, ++t.s;
      continue;
    }
    const int each = units.block(t.unit), length = each * units.blocks;
    const long long o = t.at + kAround;
    t.tiles = t.unit < units.twos ? 2 : 1, t.pair0 = t.unit * 2 * kRows;
    ++t.unit, t.at = o + length;
    const int from = (int)min(max(begin - o, 0ll), (long long)length), to = (int)min(max(end - o, 0ll), (long long)length);
    const int b0 = (from + each - 1) / each, b1 = (to + each - 1) / each;
    if (b0 >= b1) continue;
    t.row0 = q.row0[t.s], t.len = q.len[t.s];
    t.begins = b0 == 0, t.whole = t.begins && b1 == units.blocks;
    t.first = b0 * kKeys, t.last = min(b1 * kKeys, t.keys), t.blocks = b1 - b0;
    return true;
  }
  return false;
}

// Bits of the 64 keys of a block's half that have a page.
__device__ __forceinline__ unsigned long long paged64(unsigned lacking, int half, int page_size) {
  unsigned long long v = ~0ull;
#pragma unroll
  for (int i = 0; i < 64; i += 16)
    if (lacking >> (64 * half + i) / page_size & 1) v &= ~(0xffffull << i);
  return v;
}

// Bits of the 64 keys from `key0` on that row `row` of the request sees.
__device__ __forceinline__ unsigned long long seen64(const TreeArgs& a, const Item& t, int row, int key0) {
  const int k0 = key0 - t.len, left = t.keys - key0;
  if (left <= 0) return 0ull;
  const unsigned long long real = left >= 64 ? ~0ull : (1ull << left) - 1;
  if (k0 <= -64) return real;
  const int* m = a.mask + (size_t)row * a.words;
  auto word = [&](int w) { return w < a.words ? (unsigned long long)(unsigned)m[w] : 0ull; };
  unsigned long long v;
  if (k0 < 0) v = ((word(0) | word(1) << 32) << -k0) | ((1ull << -k0) - 1);
  else {
    const int w = k0 >> 5, sh = k0 & 31;
    v = (word(w) | word(w + 1) << 32) >> sh;
    if (sh) v |= word(w + 2) << (64 - sh);
  }
  return v & real;
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
tree_attention_tc_kernel(const __grid_constant__ CUtensorMap map_kv, const __grid_constant__ TreeArgs a, const __nv_bfloat16* __restrict__ qkv,
                         __nv_bfloat16* __restrict__ out) {
  constexpr int ATOMS = D / 64, KB = ATOMS * kAtom;          // bytes of a tile of queries, and of a block of keys or values
  constexpr int STAGES = D == 64 ? 4 : 2;
  constexpr int PIECES = D / 8;                              // 16-byte pieces of a query
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + (-smem_u32(smem_raw) & 1023u);          // (an offset, so that what lies here is known to be shared memory)
  unsigned char* Qs = smem;                                  // [2 tiles]
  unsigned char* KV = Qs + 2 * KB;                           // [stages][keys, values]
  Barriers* bars = reinterpret_cast<Barriers*>(KV + 2 * STAGES * KB);
  float2* s_stat = reinterpret_cast<float2*>(bars + 1);      // [2 item parities][2 groups][128 rows] (maximum, sum)
  Requests& reqs = *reinterpret_cast<Requests*>(s_stat + 4 * kRows);
  volatile int* stop = &bars->stop;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = a.Hq / a.Hkv;

  if (threadIdx.x == 0) {
    mbar_init(&bars->q_full, 8);
    mbar_init(&bars->q_empty, 1);
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&bars->k_full[i], 1);
      mbar_init(&bars->k_empty[i], 1);
      mbar_init(&bars->v_full[i], 1);
      mbar_init(&bars->v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->s_full[i], 1);
      mbar_init(&bars->p_full[i], 4);
      mbar_init(&bars->o_final[i], 1);
    }
    mbar_init(&bars->o_read, 8);
    bars->stop = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars->tmem_base)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  chain_wait(qkv);                       // (barriers and tensor memory are this SM's own; everything below was written by earlier kernels)
  for (int s = threadIdx.x; s < a.S; s += kThreads) {
    const TreeRequest r = tree_request(a, s);
    if (r.bad && blockIdx.x == 0) atomicCAS(&g_tree_tc_index, 0, 1 + s);
    reqs.row0[s] = r.row0, reqs.nodes[s] = r.nodes, reqs.len[s] = r.len, reqs.keys[s] = r.keys;
    reqs.start[s + 1] = a.Hkv * Units(r.nodes * G, r.keys).head();
  }
  __syncthreads();
  if (warp == 0) {                       // running sums
    long long sum = 0;
    if (lane == 0) reqs.start[0] = 0;
    for (int s0 = 0; s0 < a.S; s0 += 32) {
      long long v = s0 + lane < a.S ? reqs.start[s0 + lane + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      v += sum;
      if (s0 + lane < a.S) reqs.start[s0 + lane + 1] = v;
      sum = __shfl_sync(0xffffffffu, v, 31);
    }
    if (lane == 0) reqs.quota = max((long long)kLeast, (sum + gridDim.x - 1) / gridDim.x);
  }
  __syncthreads();
  if (blockIdx.x == 0 && gridDim.x > 1) {          // for the kernel that adds shares up
    for (int s = threadIdx.x; s < a.S; s += kThreads) a.ws_line[1 + s] = reqs.start[s];
    if (threadIdx.x == 0) a.ws_line[0] = reqs.quota;
  }
  Item t;
  first_item(a, reqs, t);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const unsigned tmem = bars->tmem_base;                     // S of group g at columns 128 g, O at 256 + 128 g

  if (warp < 4) {
    if (warp == 0 || warp == 2) {
      // ---- producers -------------------------------------------------------------------------------------------------
      const int kv = warp >> 1, per = kKeys / a.page_size;                // pages a block spans (at most 8)
      bool ok = true;
      int gb = 0, issued = -1;
      while (ok && next_item(a, reqs, t)) {
        const int* bt = a.block_table + (size_t)t.s * a.bt_width;
        for (int blk = 0; blk < t.blocks; ++blk, ++gb) {
          const int st = gb % STAGES;
          // lane i looks up the block's i-th page
          const int j = t.first + blk * kKeys + lane * a.page_size;
          int page = -1;
          if (lane < per && j < t.last) {
            const int lp = j / a.page_size;
            page = lp < a.bt_width ? bt[lp] : -1;
            if (page < 0 || page >= a.num_pages) {
              page = -1;
              atomicCAS(&g_tree_tc_index, 0, 1 + t.s);
            }
          }
          const unsigned there = __ballot_sync(0xffffffffu, page >= 0), wanted = __ballot_sync(0xffffffffu, lane < per && j < t.last);
          unsigned char* to = KV + (2 * st + kv) * KB;
          void* full = kv ? &bars->v_full[st] : &bars->k_full[st];
          void* empty = kv ? &bars->v_empty[st] : &bars->k_empty[st];
          if (!warp_wait(empty, ((gb / STAGES) & 1) ^ 1, stop, 2)) { ok = false; break; }
          if (elect_one()) {
            if (kv == 0) ((volatile unsigned*)bars->lacking)[gb % (2 * STAGES)] = wanted & ~there;
            mbar_expect_tx(full, (unsigned)__popc(there) * a.page_size * D * 2);
          }
          __syncwarp();
          for (int i = 0; i < per; ++i) {
            const int y = ((__shfl_sync(0xffffffffu, page, i) * 2 + kv) * a.Hkv + t.g) * a.page_size;
            if ((there >> i & 1) && elect_one())
              for (int x = 0; x < ATOMS; ++x) tma_load_2d(to + x * kAtom + i * a.page_size * 128, &map_kv, 64 * x, y, full);
          }
          issued = gb;
        }
      }
      if (!ok && lane == 0)                                  // copies asked for still land in this CTA's shared memory
        for (int b = max(0, issued - STAGES + 1); b <= issued; ++b) {
          void* full = kv ? &bars->v_full[b % STAGES] : &bars->k_full[b % STAGES];
          for (unsigned i = 0; i < (1u << 20); ++i)
            if (mbar_try(full, (b / STAGES) & 1)) break;
        }
    } else if (warp == 1) {
      // ---- products --------------------------------------------------------------------------------------------------------
      const unsigned desc_qk = mma_desc(kKeys, false), desc_pv = mma_desc(D, true);
      int gb = 0, gi = 0, done[2] = {0, 0};                  // blocks and items before this one, steps of each group
      bool ok = true;
      for (; ok && next_item(a, reqs, t); ++gi) {
        const bool two = t.tiles == 2;
        const int n0 = t.steps(0), n1 = t.steps(1);
        int to_come = n0 + n1;                               // products of queries and keys
        // (one lane waits, issues and waits again: the tensor cores take a product only when they can begin it, so that what
        // lies between two of them is time that they stand still)
        auto wait = [&](void* bar, unsigned parity, int code) { return mbar_wait(bar, parity, stop, code, &g_tree_tc_error); };
        // S = Q K^T of a group's step
        auto scores = [&](int group, int b, int left) -> bool {
          const int st = b % STAGES;
          const unsigned long long dq = smem_desc(Qs + (two ? group * KB : 0)), dk = smem_desc(KV + 2 * st * KB);
          if (!wait(&bars->k_full[st], (b / STAGES) & 1, 4)) return false;
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {              // (an atom on: 16,384 bytes, of which a descriptor counts sixteenths)
            const int off = (kk >> 2) * (kAtom / 16) + 2 * (kk & 3);
            tc_mma(tmem + group * kKeys, dq + off, dk + off, desc_qk, kk > 0 ? 1u : 0u);
          }
          tc_commit(&bars->s_full[group]);
          if (!two || group == 1) tc_commit(&bars->k_empty[st]);
          if (left == 0) tc_commit(&bars->q_empty);
          return true;
        };
        bool all = true;
        if (elect_one()) {
          all = wait(&bars->q_full, gi & 1, 3) && scores(0, gb + t.block(0, 0), to_come - 1) && (n1 == 0 || scores(1, gb + t.block(1, 0), to_come - 2));
        }
        ok = __all_sync(0xffffffffu, all);
        to_come -= 1 + (n1 > 0);
        for (int step = 0; ok && step < n0; ++step)
#pragma unroll 1
          for (int group = 0; ok && group < 2; ++group) {
            const int n = group ? n1 : n0;
            if (step >= n) continue;
            const int b = gb + t.block(group, step), st = b % STAGES;
            if (step + 1 < n) --to_come;
            all = true;
            if (elect_one()) {
              all = (step > 0 || gi == 0 || wait(&bars->o_read, (gi - 1) & 1, 7)) && wait(&bars->v_full[st], (b / STAGES) & 1, 5) &&
                    wait(&bars->p_full[group], (done[group] + step) & 1, 6);
              if (all) {
                tc_fence_after();
                const unsigned long long dv = smem_desc_mn(KV + (2 * st + 1) * KB, kAtom);
#pragma unroll
                for (int kk = 0; kk < kKeys / 16; ++kk)      // (16 keys on: 2,048 bytes)
                  tc_mma_ts(tmem + (2 + group) * kKeys, tmem + group * kKeys + 8 * kk, dv + 128 * kk, desc_pv, (step > 0 || kk > 0) ? 1u : 0u);
                if (!two || group == 1) tc_commit(&bars->v_empty[st]);
                if (step == n - 1) tc_commit(&bars->o_final[group]);
                if (step + 1 < n) all = scores(group, gb + t.block(group, step + 1), to_come);
              }
            }
            ok = __all_sync(0xffffffffu, all);
          }
        if (ok && n1 == 0 && elect_one()) tc_commit(&bars->o_final[1]);
        __syncwarp();
        gb += t.blocks, done[0] += n0, done[1] += n1;
      }
    }
  } else {
    // ---- softmax -----------------------------------------------------------------------------------------------------------
    const int group = (warp >> 2) - 1, quad = warp & 3, row = quad * 32 + lane;
    const unsigned lane_addr = (unsigned)(quad * 32) << 16;
    const unsigned tmem_s = tmem + lane_addr + group * kKeys, tmem_o = tmem + lane_addr + (2 + group) * kKeys;
    const float sc2 = a.scale * kLog2e;
    int gb = 0, gi = 0, done = 0;
    // An item's queries as the swizzled image has them: a warp takes 32 rows of its group's tile, or with one tile 16, and
    // the lanes of a row its 16-byte pieces side by side
    auto load_queries = [&](const Item& t) {
      constexpr int AT_ONCE = 32 / PIECES;                   // rows
      const bool two = t.tiles == 2;
      const int c = lane % PIECES, n = two ? 32 : 16, r0 = (two ? quad * 32 : (4 * group + quad) * 16) + lane / PIECES;
      unsigned char* tile = Qs + (two ? group * KB : 0) + (c >> 3) * kAtom;
      const int p0 = t.pair0 + (two ? group * kRows : 0);
      const __nv_bfloat16* q = qkv + (size_t)t.row0 * a.q_stride + (size_t)t.g * G * D + 8 * c;
#pragma unroll 1
      for (int h = 0; h < n; h += 8 * AT_ONCE) {
        uint4 v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int p = p0 + r0 + h + i * AT_ONCE, node = node_of(a, p);
          v[i] = p < t.pairs && h + i * AT_ONCE < n ? *reinterpret_cast<const uint4*>(q + (size_t)node * a.q_stride + (size_t)(p - node * G) * D) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int row = r0 + h + i * AT_ONCE;
          if (h + i * AT_ONCE < n) *reinterpret_cast<uint4*>(tile + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = v[i];
        }
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->q_full);
    };
    Item next = t;
    bool more = next_item(a, reqs, next);
    if (more) load_queries(next);
    for (; more; ++gi) {
      t = next;
      const int tile0 = t.pair0 + (t.tiles == 2 ? group * kRows : 0), p = tile0 + row;
      const bool real = p < t.pairs, idle = tile0 + quad * 32 >= t.pairs;      // idle: none of the warp's rows is anybody's
      const int in_tree = node_of(a, p), node = real ? t.row0 + in_tree : 0, head = t.g * G + p - in_tree * G, n = t.steps(group);
      float m_ref = 0.f, l_run = 0.f;
      bool have = false, ok = true;
      for (int step = 0; ok && step < n; ++step, ++done) {
        const int blk = t.block(group, step), kb = t.first + blk * kKeys;
        if (!warp_wait(&bars->s_full[group], done & 1, stop, 8)) { ok = false; break; }
        tc_fence_after();
        const unsigned lacking = ((volatile unsigned*)bars->lacking)[(gb + blk) % (2 * STAGES)];
        if (!idle) {
          // 64 scores at a time, of which the weights follow at once; a later 64 that raise the reference take the earlier ones'
          // weights along
#pragma unroll 1
          for (int h = 0; h < 2; ++h) {
            unsigned u[64];
            tc_ld32(tmem_s + 64 * h, u);
            tc_ld32(tmem_s + 64 * h + 32, u + 32);
            tc_wait_ld();
            if (kb + 64 * h + 64 > t.len || lacking) {       // (else keys that every row sees)
              unsigned long long seen = real ? seen64(a, t, node, kb + 64 * h) : 0ull;
              if (lacking) seen &= paged64(lacking, h, a.page_size);
              hide(u, (unsigned)seen);
              hide(u + 32, (unsigned)(seen >> 32));
            }
            float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int i = 0; i < 64; i += 2) m4[(i >> 1) & 3] = max3(m4[(i >> 1) & 3], __uint_as_float(u[i]), __uint_as_float(u[i + 1]));
            const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * sc2;
            float alpha = 1.f;
            bool raise = false;
            if (!have) {
              have = mx != -INFINITY;
              m_ref = have ? mx : 0.f;
            } else if (mx > m_ref + kRaise) {
              raise = true;
              alpha = exp2f(m_ref - mx);
              m_ref = mx;
            }
            if (__any_sync(0xffffffffu, raise)) {
              l_run *= alpha;
              // O: the product of the step before has run, as its scores came first.  At an item's first step there is none of it
              // yet, and the other group may still be reading what O holds of the item before: only the issuer waits for that
#pragma unroll 1
              for (int c = 0; c < (step ? D / 32 : 0); ++c) {
                unsigned o[32];
                tc_ld32(tmem_o + 32 * c, o);
                tc_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                tc_st32(tmem_o + 32 * c, o);
              }
              if (h) {
                unsigned o[32];
                tc_wait_st();
                tc_ld32(tmem_s, o);
                tc_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                  const __nv_bfloat162 v = *reinterpret_cast<const __nv_bfloat162*>(&o[i]);
                  const __nv_bfloat162 w = __floats2bfloat162_rn(__low2float(v) * alpha, __high2float(v) * alpha);
                  o[i] = *reinterpret_cast<const unsigned*>(&w);
                }
                tc_st32(tmem_s, o);
              }
            }
            const unsigned long long sc = pair_of(sc2, sc2), low = pair_of(-m_ref, -m_ref);
            unsigned long long sum[2] = {0ull, 0ull};        // (two pairs of 0.f)
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              float x, y;
              halves(fma2(pair_of(__uint_as_float(u[2 * i]), __uint_as_float(u[2 * i + 1])), sc, low), x, y);
              x = ex2(x), y = ex2(y);
              sum[i & 1] = add2(sum[i & 1], pair_of(x, y));
              const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
              u[i] = *reinterpret_cast<const unsigned*>(&v);
            }
            tc_st32(tmem_s + 32 * h, u);                     // (over scores that have been read)
            float s0, s1;
            halves(add2(sum[0], sum[1]), s0, s1);
            l_run += s0 + s1;
          }
          tc_wait_st();
        }
        if ((t.last - kb < kKeys || lacking) && (t.tiles == 1 || group == 0)) {      // nothing behind the request's last key, or without a page
          const int b = gb + blk, st = b % STAGES;
          if (!warp_wait(&bars->v_full[st], (b / STAGES) & 1, stop, 9)) { ok = false; break; }
          unsigned char* v = KV + (2 * st + 1) * KB;
          for (int i = (lacking ? 0 : (t.last - kb) * 8) + row; i < kKeys * 8; i += 128)
            if (kb + i / 8 >= t.last || lacking >> i / 8 / a.page_size & 1)
#pragma unroll
              for (int x = 0; x < ATOMS; ++x) reinterpret_cast<uint4*>(v + x * kAtom)[i] = make_uint4(0, 0, 0, 0);
          fence_async_smem();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->p_full[group]);
      }
      // the next item's queries, once this one's last scores are there: on their way while its last values are added up
      more = next_item(a, reqs, next);
      if (more && ok) {
        ok = warp_wait(&bars->q_empty, gi & 1, stop, 1);
        if (ok) load_queries(next);
      }
      // ---- the item's rows -----------------------------------------------------------------------------------------------
      float2* stat = s_stat + (gi & 1) * 2 * kRows;
      stat[group * kRows + row] = make_float2(have ? m_ref : -INFINITY, l_run);
      // whether all leave is one thread's word, so that none waits at this barrier alone
      if (threadIdx.x == 128) bars->quit[gi & 1] = *stop;
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (((volatile int*)bars->quit)[gi & 1]) break;
      ok = ok && warp_wait(&bars->o_final[0], gi & 1, stop, 10) && warp_wait(&bars->o_final[1], gi & 1, stop, 10);
      tc_fence_after();
      if (ok && !idle) {
        // two tiles: each group its own O; one: both groups' O, half of the columns each
        const bool two = t.tiles == 2, other = !two && t.steps(1) > 0;
        const float2 mine = stat[(two ? group : 0) * kRows + row], further = other ? stat[kRows + row] : make_float2(-INFINITY, 0.f);
        const float top = fmaxf(mine.x, further.x), base = top == -INFINITY ? 0.f : top;
        float w0 = exp2f(mine.x - base), w1 = exp2f(further.x - base);
        const float l = mine.y * w0 + further.y * w1, inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
        // (a share's numbers lie [D / 4][row of the unit][4]: the rows of a warp's lanes side by side)
        const size_t place = (size_t)node * a.Hq + head, slot = 2 * blockIdx.x + t.begins, at = p - t.pair0;
        const bool whole = t.whole;
        if (whole) w0 *= inv, w1 *= inv;
        const unsigned o0 = tmem + lane_addr + (2 + (two ? group : 0)) * kKeys, o1 = tmem + lane_addr + 3 * kKeys;
        const int c0 = two ? 0 : group * (D / 2), cn = two ? D : c0 + D / 2;
#pragma unroll 1
        for (int c = c0; c < cn; c += 32) {
          unsigned o[32], x[32];
          tc_ld32(o0 + c, o);
          if (other) tc_ld32(o1 + c, x);
          tc_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            float v = __uint_as_float(o[i]) * w0;
            if (other) v = fmaf(__uint_as_float(x[i]), w1, v);
            o[i] = __float_as_uint(v);
          }
          if (!real) continue;
          if (!whole) {
            uint4* to = reinterpret_cast<uint4*>(a.ws_acc) + (slot * (D / 4) + c / 4) * (2 * kRows) + at;
#pragma unroll
            for (int i = 0; i < 8; ++i) to[i * 2 * kRows] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
          } else {
            uint4* to = reinterpret_cast<uint4*>(out + place * D + c);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              unsigned w[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const __nv_bfloat162 v = __floats2bfloat162_rn(__uint_as_float(o[8 * i + 2 * k]), __uint_as_float(o[8 * i + 2 * k + 1]));
                w[k] = *reinterpret_cast<const unsigned*>(&v);
              }
              to[i] = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        }
        if (real && !whole && (two || group == 0)) reinterpret_cast<float2*>(a.ws_ml)[slot * 2 * kRows + at] = make_float2(top, l);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->o_read);
      gb += t.blocks;
    }
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// The CTA within whose part `at` lies.
__device__ __forceinline__ int part_of(long long at, long long quota) {
  return (at | quota) >> 32 ? (int)(at / quota) : (int)((unsigned)at / (unsigned)quota);
}

// Adds up the shares of units that more CTAs than one worked on, in ascending order: a CTA takes 32 pairs of a key head, a lane
// a pair, and each of its eight warps an eighth of the numbers; they come together in shared memory, out of which rows are
// written whole.
__global__ void __launch_bounds__(256)
tree_attention_merge_units_kernel(TreeArgs a, __nv_bfloat16* __restrict__ out) {
  constexpr int AT_ONCE = 4;
  __shared__ __align__(16) float turned[32][128 + 4];
  __shared__ int row_of[32];                                 // each pair's (row, query head) in the result; -1 for none
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = blockIdx.y, G = a.Hq / a.Hkv, each = a.D / 32;
  const int pair = blockIdx.x * 32 + lane, t = pair / G;
  chain_wait(a.ws_acc, a.ws_ml, a.ws_line, a.lengths, a.row0);
  int lo = 0, hi = a.S;                                      // the last request that begins at or before the pair's row
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (a.row0[mid] <= t) lo = mid; else hi = mid;
  }
  const TreeRequest r = tree_request(a, lo);
  int shares = 0, cta = 0, row = 0;
  if (pair < (long long)a.T * G && t >= r.row0 && t < r.row0 + r.nodes) {
    const Units units(r.nodes * G, r.keys);
    const int p = pair - r.row0 * G, u = p / (2 * kRows);
    const long long at = a.ws_line[1 + lo] + g * units.head() + (long long)u * units.length(0) + kAround, quota = a.ws_line[0];
    row = p - u * 2 * kRows;
    cta = part_of(at, quota);
    shares = part_of(at + (long long)units.block(u) * (units.blocks - 1), quota) - cta + 1;
  }
  const bool mine = shares > 1;                              // (one share: its result is there already)
  const auto slot = [&](int c) { return (size_t)(2 * (cta + c) + (c == 0)); };
  const float2* ml = reinterpret_cast<const float2*>(a.ws_ml) + row;
  float top = -INFINITY;
  for (int c = 0; c < (mine ? shares : 0); ++c) top = fmaxf(top, ml[slot(c) * 2 * kRows].x);
  const float base = top == -INFINITY ? 0.f : top;
  float l = 0.f;
  float4 sum[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) sum[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  const float4* acc = reinterpret_cast<const float4*>(a.ws_acc) + warp * each * 2 * kRows + row;
#pragma unroll 1
  for (int c0 = 0; c0 < (mine ? shares : 0); c0 += AT_ONCE) {
    float4 v[AT_ONCE][4];
    float2 x[AT_ONCE];
#pragma unroll
    for (int c = 0; c < AT_ONCE; ++c) {
      const bool there = c0 + c < shares;
      x[c] = there ? ml[slot(c0 + c) * 2 * kRows] : make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (there && i < each) v[c][i] = acc[(slot(c0 + c) * (a.D / 4) + i) * 2 * kRows];
    }
#pragma unroll
    for (int c = 0; c < AT_ONCE; ++c) {
      const float w = exp2f(x[c].x - base);
      l += w * x[c].y;
      if (w != 0.f && c0 + c < shares)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < each) sum[i].x += w * v[c][i].x, sum[i].y += w * v[c][i].y, sum[i].z += w * v[c][i].z, sum[i].w += w * v[c][i].w;
    }
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < each) *reinterpret_cast<float4*>(&turned[lane][4 * (warp * each + i)]) = make_float4(sum[i].x * inv, sum[i].y * inv, sum[i].z * inv, sum[i].w * inv);
  if (warp == 0) row_of[lane] = mine ? t * a.Hq + g * G + pair - t * G : -1;
  __syncthreads();
  for (int e = threadIdx.x; e < 32 * (a.D / 4); e += 256) {
    const int row = e / (a.D / 4), d = e % (a.D / 4) * 4;
    if (row_of[row] >= 0) store4(out + (size_t)row_of[row] * a.D + d, &turned[row][d]);
  }
}

template <int D>
int launch_tc(const CUtensorMap& map, TreeArgs a, int ctas, const void* qkv, void* out, cudaStream_t stream) {
  const size_t smem = 1024 + (size_t)(2 + 2 * (D == 64 ? 4 : 2)) * (D / 64) * kAtom + sizeof(Barriers) + 4 * kRows * sizeof(float2) + sizeof(Requests);
  static_assert(sizeof(Barriers) % 8 == 0, "float2 follow");
  if (int rc = allow_smem<tree_attention_tc_kernel<D>>(smem)) return rc;
  const int S = a.S, G = a.Hq / a.Hkv;
  const dim3 merges((unsigned)(((long long)a.T * G + 31) / 32), a.Hkv);
  for (int s0 = 0; s0 < S; s0 += kMostRequests) {
    a.S = std::min(kMostRequests, S - s0);
    launch_chained(tree_attention_tc_kernel<D>, dim3(ctas), dim3(kThreads), smem, stream, map, a, (const __nv_bfloat16*)qkv, (__nv_bfloat16*)out);
    if (int rc = check_launch("tree_attention_tc")) return rc;
    if (ctas > 1) {
      launch_chained(tree_attention_merge_units_kernel, merges, dim3(256), 0, stream, a, (__nv_bfloat16*)out);
      if (int rc = check_launch("tree_attention_merge_units")) return rc;
    }
    a.lengths += a.S, a.row0 += a.S, a.block_table += (size_t)a.S * a.bt_width;
  }
  return 0;
}

}  // namespace

bool tree_tc_fits(int D, int page_size, long long page_rows) {
  return (D == 64 || D == 128) && (page_size == 16 || page_size == 32 || page_size == 64 || page_size == 128) && page_rows < (1ll << 31);
}

// CTAs: as many as there are SMs, or as there may be parts of kLeast.
int tree_tc_ctas(int S, int T, int Hq, int Hkv, int words, int max_context) {
  const long long pairs = std::min(32ll * words, (long long)T) * (Hq / Hkv), units = (pairs + 2 * kRows - 1) / (2 * kRows) * S * Hkv;
  return (int)std::min(148ll, units == 1 && max_context <= 2 * kKeys ? 1 : units * ((max_context + 255ll) / 256 + 2));
}

// Floats: two shares a CTA, the line's parts as 64-bit numbers.
long long tree_tc_workspace(int ctas, int S, int D) { return ctas > 1 ? 2ll * ctas * 2 * kRows * (D + 2) + 2 * (S + 1) : 0; }

int launch_tree_tc(TreeArgs a, int ctas, float* ws, const void* qkv, const void* pages, void* out, cudaStream_t stream) {
  CUtensorMap map;
  if (int rc = make_map(&map, pages, (long long)a.num_pages * 2 * a.Hkv * a.page_size, a.D, a.page_size)) return rc;
  a.ws_acc = ws, a.ws_ml = ws + 2ll * ctas * 2 * kRows * a.D;
  a.ws_line = (long long*)(a.ws_ml + 2ll * ctas * 2 * kRows * 2);
  return a.D == 64 ? launch_tc<64>(map, a, ctas, qkv, out, stream) : launch_tc<128>(map, a, ctas, qkv, out, stream);
}

}  // namespace nf

using namespace nf;

// 0, or the code of the first wait that ran out since the last time (2 producers, 3-7 issuer, 8-11 softmax), or 100 + a
// request (from 1 on) whose lengths, rows or pages did not fit.  Synchronises.
extern "C" int nf_tree_attention_tc_status() {
  int v = 0, w = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_tree_tc_error, sizeof(int)) != cudaSuccess) return -1;
  if (cudaMemcpyFromSymbol(&w, g_tree_tc_index, sizeof(int)) != cudaSuccess) return -1;
  if (v) cudaMemcpyToSymbol(g_tree_tc_error, &zero, sizeof(int));
  if (w) cudaMemcpyToSymbol(g_tree_tc_index, &zero, sizeof(int));
  return v ? v : (w ? 100 + w : 0);
}
