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
// takes a request: each walks by itself (the same numbers, the same steps), reads its part of such rows, and the parts'
// sums change hands in shared memory.  A part is summed in segments of 1,024 numbers, so that the drawn token is searched
// for in one of them.
#include "common.cuh"

namespace nf {
namespace {

constexpr int kThreads = 512;
constexpr int kNodes = 1024;            // most nodes of a request
constexpr int kSegment = 1024;          // numbers a warp sums up
constexpr int kMaxSegments = 1024;      // of a CTA

__device__ int g_verify_error = 0;

struct VerifyArgs {
  const float *probs, *draft, *draws;
  const int *tokens, *parents, *row0;
  int *accepted, *path, *said;
  long long probs_ld, draft_ld;
  int T, V, most, part;                 // part: numbers of a CTA, a multiple of kSegment
};

struct Shared {
  int token[kNodes], parent[kNodes];
  float ask[kNodes], have[kNodes];      // u_c q[c][x_c] is ask * draw; have: p[parent][x_c]
  float draw[kNodes];
  int rejected[kNodes];                 // at the present node
  double mass[kNodes];                  // z when it was rejected
  double segment[kMaxSegments], total[16];
  double z;
  int node, next, accepted, n_rejected, todo;
};

__device__ __forceinline__ void cluster_meet() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ unsigned cluster_rank() {
  unsigned r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ unsigned cluster_size() {
  unsigned r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void put_cluster_f64(double* local, unsigned cta, double v) {
  unsigned remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"((unsigned)__cvta_generic_to_shared(local)), "r"(cta));
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(remote), "d"(v) : "memory");
}
// A probability: what is no positive number counts as none.
__device__ __forceinline__ double mass_of(float p) { return p > 0.f ? (double)p : 0.0; }

// What is left of p[v] at token i after the node's rejections.
__device__ __forceinline__ double left_at(const VerifyArgs& a, const Shared& sh, int row0, int n_rejected, int i) {
  double r = mass_of(a.probs[(size_t)(row0 + sh.node) * a.probs_ld + i]);
  for (int k = 0; k < n_rejected; ++k) {
    const int c = sh.rejected[k];
    if (a.draft) r = fmax(r - sh.mass[k] * mass_of(a.draft[(size_t)(row0 + c) * a.draft_ld + i]), 0.0);
    else if (sh.token[c] == i) r = 0.0;
  }
  return r;
}

// The sum of what is left: every CTA's segments, and all CTAs' sums in `total`.
__device__ double sum_left(const VerifyArgs& a, Shared& sh, int row0, int n_rejected, int begin, int end) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n_seg = (end - begin + kSegment - 1) / kSegment;
  for (int g = warp; g < n_seg; g += kThreads / 32) {
    const int lo = begin + g * kSegment, hi = min(lo + kSegment, end);
    double sum = 0.0;
    for (int i = lo + lane; i < hi; i += 32) sum += left_at(a, sh, row0, n_rejected, i);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) sh.segment[g] = sum;
  }
  cluster_meet();                       // (also: the sums of the time before have been read by all)
  if (warp == 0) {
    double sum = 0.0;
    if (lane == 0)
      for (int g = 0; g < n_seg; ++g) sum += sh.segment[g];
    sum = __shfl_sync(0xffffffffu, sum, 0);
    if ((unsigned)lane < cluster_size()) put_cluster_f64(&sh.total[cluster_rank()], lane, sum);
  }
  cluster_meet();
  double all = 0.0;
  for (unsigned c = 0; c < cluster_size(); ++c) all += sh.total[c];
  return all;
}

// The lowest token whose running sum passes `draw` times the whole, by the warp that has it; -1 where nothing is left.
// Called by all threads of all CTAs after sum_left; one thread of the cluster writes `*to`.
__device__ void draw_token(const VerifyArgs& a, const Shared& sh, int row0, int n_rejected, int begin, int end, double all, double draw, int* to) {
  if (threadIdx.x >= 32) return;
  const int lane = threadIdx.x;
  const double bound = draw * all;
  // the CTA, then the segment, where the running sum passes the bound; else the last that has anything
  double run = 0.0, before = 0.0;
  int cta = -1;
  for (unsigned c = 0; c < cluster_size(); ++c) {
    if (sh.total[c] > 0.0) {
      cta = c, before = run;
      if (run + sh.total[c] > bound) break;
    }
    run += sh.total[c];
  }
  if (cta < 0) {
    if (cluster_rank() == 0 && lane == 0) *to = -1;
    return;
  }
  if ((unsigned)cta != cluster_rank()) return;
  run = before;
  int seg = -1;
  const int n_seg = (end - begin + kSegment - 1) / kSegment;
  for (int g = 0; g < n_seg; ++g) {
    if (sh.segment[g] > 0.0) {
      seg = g, before = run;
      if (run + sh.segment[g] > bound) break;
    }
    run += sh.segment[g];
  }
  const int lo = begin + seg * kSegment, hi = min(lo + kSegment, end);
  int last = -1;
  run = before;
  for (int i0 = lo; i0 < hi; i0 += 32) {
    const int i = i0 + lane;
    const double r = i < hi ? left_at(a, sh, row0, n_rejected, i) : 0.0;
    double upto = r;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const unsigned some = __ballot_sync(0xffffffffu, r > 0.0), past = __ballot_sync(0xffffffffu, r > 0.0 && run + upto > bound);
    if (past) {
      if (lane == 0) *to = i0 + __ffs(past) - 1;
      return;
    }
    if (some) last = i0 + 31 - __clz(some);
    run += __shfl_sync(0xffffffffu, upto, 31);
  }
  if (lane == 0) *to = last;
}

__global__ void __launch_bounds__(kThreads) verify_drafts_kernel(VerifyArgs a) {
  extern __shared__ __align__(16) unsigned char raw[];
  Shared& sh = *reinterpret_cast<Shared*>(raw);
  const unsigned rank = cluster_rank();
  const int s = blockIdx.x / cluster_size();
  const int begin0 = a.row0[s], end0 = a.row0[s + 1];
  const int row0 = min(max(begin0, 0), a.T), n = min(min(max(end0, row0), a.T) - row0, kNodes);
  bool bad = begin0 < 0 || end0 <= begin0 || end0 > a.T || end0 - begin0 > kNodes;
  const int begin = min((int)rank * a.part, a.V), end = min(begin + a.part, a.V);
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
  if (threadIdx.x == 0) sh.node = 0, sh.next = 1, sh.accepted = 0, sh.n_rejected = 0, sh.z = 1.0;
  __syncthreads();
  if (n == 0) {                                            // (no root: the whole cluster leaves)
    if (rank == 0 && threadIdx.x == 0) a.accepted[s] = 0;
    return;
  }
  double all = 0.0;
  bool summed = false;
  for (;;) {
    if (threadIdx.x == 0) {
      int v = sh.node, i = sh.next, k = sh.n_rejected, got = sh.accepted;
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
        if ((double)sh.draw[i] * z * (double)sh.ask[i] < have) {
          if (rank == 0) path[got] = i, said[got] = x;
          ++got;
          v = i, k = 0, z = 1.0;
        } else {
          sh.rejected[k] = i, sh.mass[k] = z, ++k;
          if (a.draft) wait = true;
          else z -= have;
        }
      }
      sh.node = v, sh.next = i, sh.n_rejected = k, sh.accepted = got, sh.z = z, sh.todo = wait;
    }
    __syncthreads();
    summed = sh.todo;
    if (!summed) break;
    all = sum_left(a, sh, row0, sh.n_rejected, begin, end);
    if (threadIdx.x == 0) sh.z = all;
    if (sh.next >= n) break;                               // (nothing else to ask: the sums serve the draw)
    __syncthreads();
  }
  int k = sh.n_rejected;
  if (!summed) all = sum_left(a, sh, row0, k, begin, end);
  if (!(all > 0.0) && k > 0) k = 0, all = sum_left(a, sh, row0, 0, begin, end);
  if (!(all > 0.0) && rank == 0 && threadIdx.x == 0) atomicCAS(&g_verify_error, 0, 1 + s);
  draw_token(a, sh, row0, k, begin, end, all, (double)sh.draw[0], said + sh.accepted);
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
  NF_REQUIRE(S > 0 && S <= (1 << 20) && T > 0 && V > 0 && most > 0 && probs_ld >= V && (!draft || draft_ld >= V),
             "verify drafts: bad sizes S=%d T=%d V=%d most=%d", S, T, V, most);
  const int ctas = 8;
  const int part = ((V + ctas - 1) / ctas + kSegment - 1) / kSegment * kSegment;
  NF_REQUIRE(part / kSegment <= kMaxSegments, "verify drafts: a vocabulary of %d is too large", V);
  VerifyArgs a = {probs, draft, draws, tokens, parents, row0, accepted, path, said, probs_ld, draft_ld, T, V, most, part};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(S * ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sizeof(Shared);
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ctas;
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
