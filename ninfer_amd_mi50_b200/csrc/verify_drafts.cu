// Which drafted tokens stand: a walk down every request's tree, against the model's probabilities and given random numbers.
//
// Rows row0[s] .. row0[s + 1] - 1 are the nodes of request s; node 0 is its root, the newest token that it had, and parent
// numbers are below a node's own.  p[v] is the model's distribution behind node v, q[c] the one that node c's token x_c was
// drawn from (where no draft is given, x_c stands for itself: q[c] is 1 at x_c).  From v = 0, r = p[v], z = 1:
//
//   for v's children c in ascending order:   u_c z q[c][x_c] < r[x_c]:  c is accepted, v = c and start again from its r
//                                            else r = max(r - z q[c], 0), z = sum r   (no draft: r[x_c] = 0, z -= r[x_c])
//   when no child is left: the next token is the lowest i with r[0] + .. + r[i] > u_root (r[0] + .. + r[V - 1])
//
// so that the tokens are distributed as the model's own.  Where r is zero throughout (only by rounding), the next token is
// drawn from p[v].  Everything is in 64 bits: r's sums over the vocabulary decide between neighbouring tokens.
//
// A child's test needs three numbers, so those of all nodes are fetched at once and the walk goes over shared memory; what
// takes time is the vocabulary's row at the walk's end, and one for a rejection of a drafted token.  A cluster of CTAs
// takes a request: each walks by itself (the same numbers, the same steps) and reads its part of such rows, a warp a run of
// neighbouring numbers; the runs' sums change hands in shared memory.  The drawn token is then in one CTA's part, in one
// warp's run, which the CTA reads once more.  (151,936 tokens: a chain of 5 takes 8.9 us, 8 trees of up to 32 14.0, 64 chains of 6
// drawn tokens 26.5, when the rows that are read come at 3.0 TB/s.  One CTA a request took 30 to 178.)
//
// What a rejection of a drawn token leaves is not kept: each pass over the vocabulary reads the target's row and those of all
// siblings rejected so far, so that k of them cost some k^2 / 2 rows (1, 7 and 30 refused siblings of one node: 10, 110 and
// 1,570 us; 8 trees of up to 32 nodes, drawn from a draft model near the target: 64 us).
#include "common.cuh"

namespace nf {
namespace {

constexpr int kThreads = 512;
constexpr int kNodes = 1024;            // most nodes of a request
constexpr int kWarps = kThreads / 32;
constexpr int kCtas = 8;                // of a cluster

__device__ int g_verify_error = 0;

struct VerifyArgs {
  const float *probs, *draft, *draws;
  const int *tokens, *parents, *row0;
  int *accepted, *path, *said;
  long long probs_ld, draft_ld;
  int T, V, most, run;                  // run: numbers of a warp, a multiple of 128
};

struct Shared {
  int token[kNodes], parent[kNodes];
  float ask[kNodes], have[kNodes];      // u_c q[c][x_c] is ask * draw; have: p[parent][x_c]
  float draw[kNodes];
  int rejected[kNodes];                 // at the present node
  double mass[kNodes];                  // z when it was rejected
  double run[kWarps], total[2][kCtas];  // total: of a pass and of the next in turn, as a CTA may have gone on while another still reads
  double z;
  int node, next, accepted, n_rejected, todo, summed, first, last;
};

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_meet() { cluster_arrive(), cluster_wait(); }
__device__ __forceinline__ unsigned cluster_rank() {
  unsigned r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void put_cluster_f64(double* local, unsigned cta, double v) {
  unsigned remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"((unsigned)__cvta_generic_to_shared(local)), "r"(cta));
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(remote), "d"(v) : "memory");
}
// A probability: what is no positive number counts as none.
__device__ __forceinline__ double mass_of(float p) { return p > 0.f ? (double)p : 0.0; }

// Four neighbouring numbers of a row, of which the first `n` are in it: at once where the row allows it.
__device__ __forceinline__ float4 four(const float* p, int n, bool vec) {
  if (vec && n >= 4) return *reinterpret_cast<const float4*>(p);
  return make_float4(n > 0 ? p[0] : 0.f, n > 1 ? p[1] : 0.f, n > 2 ? p[2] : 0.f, n > 3 ? p[3] : 0.f);
}
// What is left of p[v] at tokens i .. i + 3 after the node's rejections: `p` are its numbers there, `q` those of the first
// rejected draft, `n` tokens are in the vocabulary.
__device__ __forceinline__ void left_at(const VerifyArgs& a, const Shared& sh, int row0, int n_rejected, int i, int n, bool vec, float4 p, float4 q,
                                        double* r) {
  r[0] = mass_of(p.x), r[1] = mass_of(p.y), r[2] = mass_of(p.z), r[3] = mass_of(p.w);
  for (int k = 0; k < n_rejected; ++k) {
    const int c = sh.rejected[k];
    if (a.draft) {
      if (k) q = four(a.draft + (size_t)(row0 + c) * a.draft_ld + i, n, vec);
      const double z = sh.mass[k];
      r[0] = fmax(r[0] - z * mass_of(q.x), 0.0), r[1] = fmax(r[1] - z * mass_of(q.y), 0.0);
      r[2] = fmax(r[2] - z * mass_of(q.z), 0.0), r[3] = fmax(r[3] - z * mass_of(q.w), 0.0);
    } else {
      const int x = sh.token[c] - i;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (x == j) r[j] = 0.0;
    }
  }
}
__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The sum of what is left: every warp's run, and all CTAs' sums in `total`.
__device__ double sum_left(const VerifyArgs& a, Shared& sh, double* total, int row0, int n_rejected, bool vec) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int begin = (cluster_rank() * kWarps + warp) * a.run, end = min(begin + a.run, a.V);
  constexpr int AT_ONCE = 5;            // (a run of 152,000 numbers' is 1,280: two trips to memory)
  const float* p = a.probs + (size_t)(row0 + sh.node) * a.probs_ld;
  const float* q = a.draft && n_rejected ? a.draft + (size_t)(row0 + sh.rejected[0]) * a.draft_ld : nullptr;
  double sum = 0.0;
  for (int i0 = begin + 4 * lane; i0 < end; i0 += 128 * AT_ONCE) {
    float4 x[AT_ONCE], y[AT_ONCE];
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      const int i = i0 + 128 * u;
      x[u] = four(p + i, end - i, vec);
      y[u] = q ? four(q + i, end - i, vec) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      const int i = i0 + 128 * u;
      double r[4];
      left_at(a, sh, row0, i < end ? n_rejected : 0, i, end - i, vec, x[u], y[u], r);
      sum += (r[0] + r[1]) + (r[2] + r[3]);
    }
  }
  sum = warp_sum_f64(sum);
  if (lane == 0) sh.run[warp] = sum;
  __syncthreads();
  if (warp == 0) {                      // (the runs in their order; each CTA's sum goes to all)
    double part = 0.0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) part += sh.run[w];
    if (lane < kCtas) put_cluster_f64(&total[cluster_rank()], lane, part);
  }
  cluster_meet();
  double all = 0.0;
#pragma unroll
  for (int c = 0; c < kCtas; ++c) all += total[c];
  return all;
}

// The lowest token whose running sum passes `draw` times the whole, written to `*to` by the CTA that has it; -1 where
// nothing is left, or something infinite.  Called by all threads of all CTAs after sum_left.  Where rounding keeps the sums of a stretch from what
// they were as parts, the last token that has anything is taken.
__device__ void draw_token(const VerifyArgs& a, Shared& sh, const double* total, int row0, int n_rejected, bool vec, double all, double draw, int* to) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const double bound = draw * all;
  double run = 0.0, before = 0.0;
  int mine = -1;
  for (int c = 0; c < kCtas; ++c) {
    const double t = total[c];
    if (t > 0.0) {
      mine = c, before = run;
      if (run + t > bound) break;
    }
    run += t;
  }
  if (mine < 0 || all == INFINITY) {
    if (cluster_rank() == 0 && threadIdx.x == 0) *to = -1;
    return;
  }
  if ((unsigned)mine != cluster_rank()) return;
  run = before;
  mine = -1;
  for (int w = 0; w < kWarps; ++w) {
    const double t = sh.run[w];
    if (t > 0.0) {
      mine = w, before = run;
      if (run + t > bound) break;
    }
    run += t;
  }
  // that warp's run, four numbers a thread of the whole CTA
  const int begin = (cluster_rank() * kWarps + mine) * a.run, end = min(begin + a.run, a.V);
  const float* p = a.probs + (size_t)(row0 + sh.node) * a.probs_ld;
  const float* q = a.draft && n_rejected ? a.draft + (size_t)(row0 + sh.rejected[0]) * a.draft_ld : nullptr;
  if (threadIdx.x == 0) sh.first = 0x7fffffff, sh.last = -1;
  for (int i0 = begin; i0 < end; i0 += 4 * kThreads) {
    const int i = i0 + 4 * threadIdx.x;
    double r[4] = {0.0, 0.0, 0.0, 0.0};
    if (i < end)
      left_at(a, sh, row0, n_rejected, i, end - i, vec, four(p + i, end - i, vec), q ? four(q + i, end - i, vec) : make_float4(0.f, 0.f, 0.f, 0.f), r);
    const double sum = (r[0] + r[1]) + (r[2] + r[3]);
    double upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    __syncthreads();                                       // (all have read sh.run, and the sums of the stretch before)
    if (lane == 31) sh.run[warp] = upto;
    __syncthreads();
    double at = before;
    for (int w = 0; w < warp; ++w) at += sh.run[w];
    if (sum > 0.0) {
      int last = -1, found = -1;
      double x = at + (upto - sum);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x += r[j];
        if (r[j] > 0.0) {
          last = i + j;
          if (found < 0 && x > bound) found = i + j;
        }
      }
      if (found < 0 && at + upto > bound) found = last;
      if (found >= 0) atomicMin(&sh.first, found);
      atomicMax(&sh.last, last);
    }
    for (int w = 0; w < kWarps; ++w) before += sh.run[w];
  }
  __syncthreads();
  if (threadIdx.x == 0) *to = sh.first != 0x7fffffff ? sh.first : sh.last;
}

__global__ void __launch_bounds__(kThreads) verify_drafts_kernel(VerifyArgs a) {
  extern __shared__ __align__(16) unsigned char raw[];
  Shared& sh = *reinterpret_cast<Shared*>(raw);
  cluster_arrive();                                        // (to be there before another CTA writes to this one)
  const unsigned rank = cluster_rank();
  const int s = blockIdx.x / kCtas;
  const int begin0 = a.row0[s], end0 = a.row0[s + 1];
  const int row0 = min(max(begin0, 0), a.T), n = min(min(max(end0, row0), a.T) - row0, kNodes);
  bool bad = begin0 < 0 || end0 <= begin0 || end0 > a.T || end0 - begin0 > kNodes;
  int* path = a.path + (size_t)s * a.most;
  int* said = a.said + (size_t)s * (a.most + 1);
  if (rank == 0) {
    for (int i = threadIdx.x; i < a.most; i += kThreads) path[i] = -1;
    for (int i = threadIdx.x; i < a.most + 1; i += kThreads) said[i] = -1;
  }
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int row = row0 + i, token = a.tokens[row], parent = a.parents[row];
    const bool fits = i == 0 || (token >= 0 && token < a.V && parent >= 0 && parent < i);
    bad |= !fits;
    sh.token[i] = token;
    sh.parent[i] = fits && i > 0 ? parent : -1;            // (a node that does not fit is nobody's child)
    sh.draw[i] = a.draws[row];
    sh.ask[i] = a.draft && fits && i > 0 ? a.draft[(size_t)row * a.draft_ld + token] : 1.f;
    sh.have[i] = fits && i > 0 ? a.probs[(size_t)(row0 + parent) * a.probs_ld + token] : 0.f;
  }
  if (bad && rank == 0) atomicCAS(&g_verify_error, 0, 1 + s);
  if (threadIdx.x == 0) sh.node = 0, sh.next = 1, sh.accepted = 0, sh.n_rejected = 0, sh.z = 1.0, sh.summed = 0;
  __syncthreads();
  cluster_wait();
  if (n == 0) {                                            // (no root: the whole cluster leaves)
    if (rank == 0 && threadIdx.x == 0) a.accepted[s] = 0;
    return;
  }
  // rows that can be read four numbers at a time
  const bool vec = ((uintptr_t)a.probs | (uintptr_t)a.draft) % 16 == 0 && (a.probs_ld | a.draft_ld) % 4 == 0;
  double all = 0.0;
  int pass = 0;
  for (;;) {
    if (threadIdx.x == 0) {
      int v = sh.node, i = sh.next, k = sh.n_rejected, got = sh.accepted, summed = sh.summed;
      double z = sh.z;
      bool wait = false;                                   // for the sum of what a rejection has left
      for (; i < n && got < a.most && !wait; ++i) {
        if (sh.parent[i] != v) continue;
        const int x = sh.token[i];
        double have = mass_of(sh.have[i]);
        for (int j = 0; j < k; ++j) {
          const int c = sh.rejected[j];
          if (a.draft) have = fmax(have - sh.mass[j] * mass_of(a.draft[(size_t)(row0 + c) * a.draft_ld + x]), 0.0);
          else if (sh.token[c] == x) have = 0.0;
        }
        if ((double)sh.draw[i] * z * mass_of(sh.ask[i]) < have) {
          if (rank == 0) path[got] = i, said[got] = x;
          ++got;
          v = i, k = 0, z = 1.0;
        } else {
          sh.rejected[k] = i, sh.mass[k] = z, ++k;
          if (a.draft) wait = true;
          else z -= have;
        }
        summed = 0;
      }
      sh.node = v, sh.next = i, sh.n_rejected = k, sh.accepted = got, sh.z = z, sh.todo = wait, sh.summed = summed;
    }
    __syncthreads();
    if (!sh.todo) break;
    pass ^= 1;
    all = sum_left(a, sh, sh.total[pass], row0, sh.n_rejected, vec);
    if (threadIdx.x == 0) sh.z = all, sh.summed = 1;
  }
  int k = sh.n_rejected;
  if (!sh.summed) pass ^= 1, all = sum_left(a, sh, sh.total[pass], row0, k, vec);      // (where the last thing was a rejection its sums serve the draw)
  if (!(all > 0.0) && k > 0) k = 0, pass ^= 1, all = sum_left(a, sh, sh.total[pass], row0, 0, vec);
  if ((!(all > 0.0) || all == INFINITY) && rank == 0 && threadIdx.x == 0) atomicCAS(&g_verify_error, 0, 1 + s);
  draw_token(a, sh, sh.total[pass], row0, k, vec, all, (double)sh.draw[0], said + sh.accepted);
  if (rank == 0 && threadIdx.x == 0) a.accepted[s] = sh.accepted;
  cluster_meet();                                          // (no CTA leaves while another may still write to it)
}

}  // namespace
}  // namespace nf

using namespace nf;

extern "C" int nf_verify_most_nodes() { return kNodes; }

// probs float32 [T, V] with rows probs_ld apart; draft the same or null; tokens, parents int32 [T]; row0 int32 [S + 1];
// draws float32 [T].  accepted int32 [S], path int32 [S, most], said int32 [S, most + 1].
extern "C" int nf_verify_drafts(const float* probs, long long probs_ld, const float* draft, long long draft_ld, const int* tokens,
                                const int* parents, const int* row0, const float* draws, int* accepted, int* path, int* said, int S, int T,
                                int V, int most, cudaStream_t stream) {
  if (S == 0) return 0;
  NF_REQUIRE(S > 0 && S <= (1 << 20) && T > 0 && V > 0 && V <= (1 << 30) && most > 0 && probs_ld >= V && (!draft || draft_ld >= V),
             "verify drafts: bad sizes S=%d T=%d V=%d most=%d", S, T, V, most);
  const int run = ((V + kCtas * kWarps - 1) / (kCtas * kWarps) + 127) / 128 * 128;
  VerifyArgs a = {probs, draft, draws, tokens, parents, row0, accepted, path, said, probs_ld, draft_ld, T, V, most, run};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(S * kCtas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sizeof(Shared);
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = kCtas;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  static_assert(sizeof(Shared) <= 48 * 1024, "the walk's numbers fit the shared memory that needs no asking");
  const cudaError_t e = cudaLaunchKernelEx(&cfg, verify_drafts_kernel, a);
  if (e != cudaSuccess) note_launch_error(e);
  return check_launch("verify_drafts");
}

// 0, or 1 + a request whose tree, tokens or probabilities made no sense since the last time.  Synchronises.
extern "C" int nf_verify_drafts_status() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_verify_error, sizeof(int)) != cudaSuccess) return -1;
  if (v) cudaMemcpyToSymbol(g_verify_error, &zero, sizeof(int));
  return v;
}
