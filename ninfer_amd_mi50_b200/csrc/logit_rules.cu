// Penalties for repeated tokens, biases and masks on a step's logits, from a log of every request's tokens that stays on
// the device.  For row r of a request with tokens [0, length), the generated ones from `start` on, c and g the times that
// token i occurs in all of them and in the generated ones:
//
//   v = l[i];  v = v > 0 ? v / p^c : v p^c;  v = v - f g - q [g > 0] + bias(i);  out = allowed(i) ? v : -inf
//
// (p: repetition, as nf_repetition_penalty applies it, once for every occurrence; f frequency, q presence).  A token that
// the mask leaves out is -inf whatever its logit was, NaN included; a mask that allows nothing leaves a row of -inf.
//
// The log holds tokens, not counts: a table of counts for every slot and token would be read whole at every step, as many
// bytes as the logits.  A CTA takes a piece of the vocabulary of one row, counts the log's tokens that lie in it in shared
// memory (integer additions: the order of the log's reading does not show), and walks its logits once.
#include "common.cuh"

namespace nf {

// set by a row whose slot, length or start does not fit the log, or whose mask or biases do not fit theirs: 1 + the row; read by
// nf_rules_index_status
__device__ int g_rules_error = 0;

struct RuleArgs {
  const float* logits;
  float* out;
  int* history;                  // [slots, capacity]
  const int *slots, *lengths, *starts, *tokens;   // [rows]; tokens: the last of each row, to be written to its log, or null
  const float* penalties;        // [rows, 3]: repetition, frequency, presence
  const int *bias_offsets, *bias_ids;             // [rows + 1], or null
  const float* bias_values;
  const unsigned* mask;          // [mask_rows, words], or null
  const int* mask_index;         // [rows]: row of `mask`, negative for none
  int V, ld_in, ld_out, n_slots, capacity, n_bias, mask_rows, words;
};

template <int V> struct Int { static constexpr int value = V; };

constexpr int kSharedLog = 16384;      // tokens of a log from which a cluster shares it out

// Occurrences of one token: in the prompt, and among the generated ones.  A log of up to 65,535 tokens has both in one word.
template <bool WORD> struct Counts;
template <> struct Counts<true> {
  static constexpr int kWords = 1;
  __device__ static void add(unsigned* n, int, unsigned d, bool made) { atomicAdd(n + d, made ? 0x10000u : 1u); }
  __device__ static uint4 any(const unsigned* n, int, int d) { return *reinterpret_cast<const uint4*>(n + d); }
  __device__ static void clear(unsigned* n, int, int d) { n[d] = 0; }
  __device__ static void get(const unsigned* n, int, int d, unsigned& all, unsigned& made) {
    made = n[d] >> 16;
    all = (n[d] & 0xffffu) + made;
  }
};
template <> struct Counts<false> {
  static constexpr int kWords = 2;
  __device__ static void add(unsigned* n, int C, unsigned d, bool made) { atomicAdd(n + d + (made ? C : 0), 1u); }
  __device__ static uint4 any(const unsigned* n, int C, int d) {
    const uint4 u = *reinterpret_cast<const uint4*>(n + d), v = *reinterpret_cast<const uint4*>(n + C + d);
    return make_uint4(u.x | v.x, u.y | v.y, u.z | v.z, u.w | v.w);
  }
  __device__ static void clear(unsigned* n, int C, int d) { n[d] = n[C + d] = 0; }
  __device__ static void get(const unsigned* n, int C, int d, unsigned& all, unsigned& made) {
    made = n[C + d];
    all = n[d] + made;
  }
};

// What tokens [lo, lo + span) of the vocabulary have of a row's log: the places [from, end) of it, those from `start` on
// generated.  (Additions whose results nobody waits for: with the first occurrence of a token noticed by what its addition returns,
// long logs took 1.7 times as long.)
template <int THREADS, bool WORD>
struct PieceLog {
  static constexpr int U = 4;   // runs of four tokens a thread has under way
  unsigned* counts;             // [kWords][plane]
  int plane, lo, span;
  const int4* quads;
  int from, start, end;
  __device__ __forceinline__ void one(int t, bool made) {
    const unsigned d = (unsigned)t - (unsigned)lo;
    if (d < (unsigned)span) Counts<WORD>::add(counts, plane, d, made);
  }
  __device__ __forceinline__ void ask(int q0, int4* t) const {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (4 * (q0 + u * THREADS) < end) t[u] = quads[q0 + u * THREADS];
  }
  __device__ __forceinline__ void take(int q0, const int4* t) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int p = 4 * (q0 + u * THREADS);
      if (p >= end) break;
      const int n[4] = {t[u].x, t[u].y, t[u].z, t[u].w};
      if (p >= from && p + 4 <= end) {
#pragma unroll
        for (int e = 0; e < 4; ++e) one(n[e], p + e >= start);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (p + e >= from && p + e < end) one(n[e], p + e >= start);
      }
    }
  }
};

// A CTA takes a piece of WALK * PIECES * 4 * THREADS tokens of one row, counted from the last 16-byte boundary at or before the
// row's start.  It copies the piece's logits under the mask, WALK steps of PIECES runs of four a thread, and then does what is left to
// do at the biased tokens and at those that occur in the log, one thread each.  (Done where the logits are copied, the powers and
// quotients of the few tokens that occur held up nearly every warp: 204 instructions a run of four, 256 rows of 151936 99 us.)
// What bounds it: 256 rows of 151936 take 64 us, of which the copy alone, as it runs without rules, 49 (6.3 TB/s), 64 rows 22.3 of which the
// copy 13.7 (16.6 under masks); the rest is a CTA's chain from a row's numbers to its log to the counts to the list.  So everything that does not wait for anything is asked for first,
// the log's loads are under way while the logits are copied, a walked piece's logits are brought into L2 meanwhile, and a walked
// piece leaves room for three CTAs on an SM (two: a tenth longer).  One row of 151936 and a short log 2.9 us: the chain and the launch.
// SPLIT: CTAs of a cluster, with a piece each.  A long log is shared out: each CTA counts a part of it for all SPLIT pieces, and adds up what
// the others have for its own.
template <int THREADS, int PIECES, int WALK, bool WORD, int SPLIT>
__global__ void __launch_bounds__(THREADS, WALK > 1 ? 3 : 2)
logit_rules_kernel(RuleArgs a) {
  constexpr int STEP = THREADS * 4 * PIECES, C = STEP * WALK, CC = C * SPLIT;      // tokens of a piece, tokens that are counted
  extern __shared__ __align__(16) unsigned rule_smem[];   // [counts of CC tokens | list]
  __shared__ int listed;
  __shared__ unsigned mask[C / 32 + 2];                   // the piece's words of the row's mask
  chain_wait();
  const int r = blockIdx.y, tid = threadIdx.x;
  const float* row = a.logits + (size_t)r * a.ld_in;
  float* out = a.out + (size_t)r * a.ld_out;
  const bool in_place = a.logits == a.out;
  const int pad = (int)(((uintptr_t)row >> 2) & 3);
  const int lo = (int)blockIdx.x * C - pad;   // the token of the piece's place 0
  const int member = SPLIT > 1 ? (int)blockIdx.x % SPLIT : 0, own = member * C;      // own: where the piece's counts begin
  const bool pairs = (((uintptr_t)out >> 2) & 3) == (unsigned)pad;       // runs of four are aligned on both sides

  // everything that does not wait for anything is asked for first
  const int slot = a.slots[r], m = a.mask ? a.mask_index[r] : -1, last_token = a.tokens ? a.tokens[r] : 0;
  int len = a.lengths[r], start = a.starts[r];
  const float rep = a.penalties[3 * r], freq = a.penalties[3 * r + 1], pres = a.penalties[3 * r + 2];
  int b0 = 0, b1 = 0;
  if (a.bias_offsets) { b0 = a.bias_offsets[r]; b1 = a.bias_offsets[r + 1]; }
  float v[PIECES][4];
  auto fetch = [&](int w) {
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      const int i0 = lo + w * STEP + 4 * (tid + p * THREADS);
      if (i0 >= 0 && i0 + 4 <= a.V) {
        load4(row + i0, v[p]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[p][e] = i0 + e >= 0 && i0 + e < a.V ? row[i0 + e] : 0.f;
      }
    }
  };
  if (!in_place) {
    if (WALK > 1 && tid == 0) {                            // the later steps' logits into L2 (whole 16-byte runs of this row)
      const int first = lo + STEP, count = (min(lo + C, a.V) - first) & ~3;
      if (count > 0) asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(row + first), "r"(count * 4));
    }
    fetch(0);
  }
  const bool generated = freq != 0.f || pres != 0.f || rep != 1.f;
  const bool fits = slot >= 0 && slot < a.n_slots && len >= (a.tokens ? 1 : 0) && len <= a.capacity;
  if (tid == 0 && (!fits || start < 0 || start > len || (a.mask && m >= a.mask_rows) || b0 < 0 || b0 > b1 || b1 > a.n_bias))
    atomicCAS(&g_rules_error, 0, r + 1);
  if (!fits) len = 0;
  // (places of the log and of the lists are walked in steps beyond them: none of these may begin near the end of an int)
  start = min(max(start, 0), len);
  b1 = min(max(b1, 0), a.n_bias);
  b0 = min(max(b0, 0), b1);
  int* log = a.history + (size_t)(fits ? slot : 0) * a.capacity;
  // earlier tokens count for the repetition penalty only; the log holds all but the last of the row where that comes with the call
  const int from = rep != 1.f ? 0 : start, end = generated ? (a.tokens ? len - 1 : len) : 0;
  const bool shared = SPLIT > 1 && end - from >= kSharedLog;      // (the members of a cluster have the same row)
  PieceLog<THREADS, WORD> piece{rule_smem + (shared ? 0 : own), CC, shared ? lo - own : lo, shared ? CC : C,
                                reinterpret_cast<const int4*>(log), from, start, end};
  unsigned* counts = rule_smem + own;                      // of this CTA's piece
  unsigned short* list = reinterpret_cast<unsigned short*>(rule_smem + Counts<WORD>::kWords * CC);      // [C] places that occur, in any order
  constexpr int RUN = PieceLog<THREADS, WORD>::U * THREADS;
  const int q_first = (from >> 2) + (shared ? member * RUN : 0) + tid, q_step = shared ? SPLIT * RUN : RUN;
  int4 held[PieceLog<THREADS, WORD>::U];
  piece.ask(q_first, held);
  const unsigned* bits = m >= 0 && m < a.mask_rows ? a.mask + (size_t)m * a.words : nullptr;
  const int first = max(lo, 0), last = min(lo + C, a.V);    // this piece's tokens
  const int word0 = first >> 5, words = ((last + 31) >> 5) - word0;
  if (bits)
    for (int i = tid; i < words; i += THREADS) mask[i] = bits[word0 + i];
  int bias_id = -1;                                        // this thread's entry; those beyond as many as threads are read later
  float bias = 0.f;
  if (b0 + tid < b1) {
    bias_id = a.bias_ids[b0 + tid];
    bias = a.bias_values[b0 + tid];
  }
  if (generated)
#pragma unroll
    for (int w = 0; w < Counts<WORD>::kWords; ++w)
      for (int i = tid; i < piece.span / 4; i += THREADS) reinterpret_cast<uint4*>(piece.counts + w * CC)[i] = make_uint4(0, 0, 0, 0);
  if (tid == 0) listed = 0;
  __syncthreads();

  // the piece's logits under the mask
  // (whole and aligned on both sides, with nothing to look after: 256 rows 63.9 us, by the other way 68.0, where the copy's instructions show)
  if (!in_place && pairs && lo >= 0 && lo + C <= a.V) {
#pragma unroll 1
    for (int w = 0; w < WALK; ++w) {
      if (w > 0) {
#pragma unroll
        for (int p = 0; p < PIECES; ++p) load4(row + lo + w * STEP + 4 * (tid + p * THREADS), v[p]);
      }
#pragma unroll
      for (int p = 0; p < PIECES; ++p) {
        const int i0 = lo + w * STEP + 4 * (tid + p * THREADS);
        if (bits) {
          const int word = (i0 >> 5) - word0;
          const unsigned on = __funnelshift_r(mask[word], mask[word + 1], i0);      // (by i0 modulo 32)
#pragma unroll
          for (int e = 0; e < 4; ++e) v[p][e] = on & (1u << e) ? v[p][e] : -INFINITY;
        }
        store4(out + i0, v[p]);
      }
    }
  } else {
#pragma unroll 1
    for (int w = 0; w < WALK; ++w) {
      if (lo + w * STEP >= a.V) break;
      if (in_place && !bits) break;                           // nothing changes but at single tokens
      if (w > 0 && !in_place) fetch(w);
#pragma unroll
      for (int p = 0; p < PIECES; ++p) {
        const int i0 = lo + w * STEP + 4 * (tid + p * THREADS);
        if (i0 + 4 <= 0 || i0 >= a.V) continue;
        const bool inside = i0 >= 0 && i0 + 4 <= a.V;
        unsigned on = 0xfu;                                   // tokens that the mask allows
        if (bits) {
          const int from = max(i0, 0), word = (from >> 5) - word0, sh = from & 31;
          unsigned x = mask[word] >> sh;
          if (sh > 28 && word + 1 < words) x |= mask[word + 1] << (32 - sh);
          on &= x << (from - i0);
        }
        if (in_place) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!(on & (1u << e)) && i0 + e >= 0 && i0 + e < a.V) out[i0 + e] = -INFINITY;
          continue;
        }
        if (on != 0xfu) {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[p][e] = on & (1u << e) ? v[p][e] : -INFINITY;
        }
        if (pairs && inside) {
          store4(out + i0, v[p]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (i0 + e >= 0 && i0 + e < a.V) out[i0 + e] = v[p][e];
        }
      }
    }
  }
  // (not before: it would hold up the copy for a trip to memory; in place, before anything but the mask has changed it)
  float biased = bias_id >= first && bias_id < last ? row[bias_id] : 0.f;
  // the log
  if (generated) {
    piece.take(q_first, held);
    for (int q = q_first + q_step; 4 * q < end; q += q_step) {
      piece.ask(q, held);
      piece.take(q, held);
    }
  }
  if (a.tokens && tid == 0 && len > 0) {
    if (generated && (member == 0 || !shared) && len - 1 >= from) piece.one(last_token, len - 1 >= start);
    if (blockIdx.x == 0) log[len - 1] = last_token;
  }

  // the rules of one token that the mask allows, from its logit
  auto rules = [&](float x, unsigned c, unsigned g) {
    if (c && rep != 1.f && x != 0.f && !isinf(x)) {        // (0 and the infinities stay what they are, whatever p^c is)
      const float times = powf(rep, (float)c);
      x = x > 0.f ? x / times : x * times;
    }
    return g ? x - (float)g * freq - pres : x;
  };
  auto allowed = [&](int i) { return !bits || (mask[(i >> 5) - word0] >> (i & 31)) & 1u; };
  if (shared) {
    asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
    for (int i = tid; i < Counts<WORD>::kWords * C / 4; i += THREADS) {
      unsigned* n = counts + i / (C / 4) * CC + i % (C / 4) * 4;      // (which only this thread reads here, and nobody elsewhere)
      uint4 sum = make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int m = 0; m < SPLIT; ++m) {
        unsigned at;
        uint4 v;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((unsigned)__cvta_generic_to_shared(n)), "r"(m));
        asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
        sum = make_uint4(sum.x + v.x, sum.y + v.y, sum.z + v.z, sum.w + v.w);
      }
      *reinterpret_cast<uint4*>(n) = sum;
    }
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");      // this thread reads the others' counts no more
  }
  __syncthreads();                                          // the counts are complete, the piece is written
  // biased tokens: all of their rules, and they are off the list of the others
  if (b0 < b1) {
    for (int i = b0 + tid; i < b1; i += THREADS) {
      if (i >= b0 + THREADS) {
        bias_id = a.bias_ids[i];
        bias = a.bias_values[i];
        if (bias_id >= first && bias_id < last) biased = row[bias_id];
      }
      if (bias_id < first || bias_id >= last || !allowed(bias_id)) continue;
      unsigned c = 0, g = 0;
      if (generated) {
        Counts<WORD>::get(counts, CC, bias_id - lo, c, g);
        Counts<WORD>::clear(counts, CC, bias_id - lo);
      }
      out[bias_id] = rules(biased, c, g) + bias;
    }
    __syncthreads();
  }
  // the other tokens that occur
  if (!generated) return;
  for (int d = 4 * tid; d < C; d += 4 * THREADS) {
    const uint4 n = Counts<WORD>::any(counts, CC, d);
    if (n.x | n.y | n.z | n.w) {
      int at = atomicAdd(&listed, (n.x != 0) + (n.y != 0) + (n.z != 0) + (n.w != 0));
      if (n.x) list[at++] = (unsigned short)d;
      if (n.y) list[at++] = (unsigned short)(d + 1);
      if (n.z) list[at++] = (unsigned short)(d + 2);
      if (n.w) list[at++] = (unsigned short)(d + 3);
    }
  }
  __syncthreads();
  for (int k = tid; k < listed; k += THREADS) {
    const int d = list[k], i = lo + d;
    if (i < 0 || i >= a.V || !allowed(i)) continue;
    unsigned c, g;
    Counts<WORD>::get(counts, CC, d, c, g);
    out[i] = rules(row[i], c, g);
  }
  if (shared) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");      // nobody reads this CTA's counts any more
}

// A thread an entry: 64 entries are a launch and two trips to memory in turn, 2 us; no entry is read twice, nothing to tile.
__global__ void __launch_bounds__(256)
append_history_kernel(int* __restrict__ history, const int* __restrict__ slots, const int* __restrict__ positions,
                      const int* __restrict__ tokens, int n, int n_slots, int capacity) {
  chain_wait();
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const int s = slots[i], p = positions[i];
  if (s < 0 || s >= n_slots || p < 0 || p >= capacity) {
    if (s >= 0) atomicCAS(&g_rules_error, 0, i + 1);       // a negative slot: a row of no request
    return;
  }
  history[(size_t)s * capacity + p] = tokens[i];
}

}  // namespace nf

using namespace nf;

// history[slots[i], positions[i]] = tokens[i]; entries with a negative slot are left out.
extern "C" int nf_append_history(int* history, const int* slots, const int* positions, const int* tokens, int n, int n_slots,
                                 int capacity, cudaStream_t stream) {
  if (n == 0) return 0;
  NF_REQUIRE(n > 0 && n_slots > 0 && capacity > 0, "append_history: bad sizes n=%d slots=%d capacity=%d", n, n_slots, capacity);
  launch_chained(append_history_kernel, dim3((n + 255) / 256), dim3(256), 0, stream, history, slots, positions, tokens, n, n_slots, capacity);
  return check_launch("append_history");
}

// out[r] from logits[r] (rows ld_in and ld_out floats apart; out may be logits).  tokens: the last token of every row, written
// to its log's place lengths[r] - 1 and counted with it, or null (the log holds it already).  bias: ids and values of row r at
// [bias_offsets[r], bias_offsets[r + 1]), each id once a row, or null.  mask: bit i & 31 of word i >> 5 of row
// mask_index[r] is set where token i is allowed.  capacity: a multiple of 4, up to 2^30; history 16-byte aligned.
extern "C" int nf_logit_rules(const float* logits, float* out, int* history, const int* slots, const int* lengths, const int* starts,
                              const int* tokens, const float* penalties, const int* bias_offsets, const int* bias_ids,
                              const float* bias_values, int n_bias, const unsigned* mask, const int* mask_index, int mask_rows,
                              int rows, int V, int ld_in, int ld_out, int n_slots, int capacity, cudaStream_t stream) {
  if (rows == 0) return 0;
  NF_REQUIRE(rows > 0 && rows <= 65535 && V > 0 && V <= (1 << 30), "logit_rules: bad sizes rows=%d V=%d", rows, V);
  NF_REQUIRE(ld_in >= V && ld_out >= V, "logit_rules: rows %d and %d apart for %d logits", ld_in, ld_out, V);
  NF_REQUIRE(n_slots > 0 && capacity > 0 && capacity % 4 == 0 && capacity <= (1 << 30) && (uintptr_t)history % 16 == 0,
             "logit_rules: a log of %d slots with %d tokens (a multiple of 4, up to 2^30), 16-byte aligned", n_slots, capacity);
  NF_REQUIRE(n_bias >= 0 && n_bias <= (1 << 30), "logit_rules: %d biases", n_bias);
  const RuleArgs a{logits, out, history, slots, lengths, starts, tokens, penalties, bias_offsets, bias_ids, bias_values, mask,
                   mask_index, V, ld_in, ld_out, n_slots, capacity, n_bias, mask_rows, (V + 31) / 32};
  // A piece of the vocabulary costs a reading of the log, a table to clear and to look through: the largest that still make several
  // CTAs a SM.  Rows of 151936 with logs of up to 4,000 tokens, us in pieces of 16384, 8192 and 4096: 16 rows 9.8 (4096) and 8.3
  // (8192), 32 rows 14.3, 13.3 and 17.5, 64 rows 27.0, 25.4 and 39.1 (logs of up to 8,192), 96 and 128 rows the same in the first two.
  // Few rows whose logs may be long: pieces of 2048 in clusters of four, which share out a log of kSharedLog tokens and more (alone and in
  // clusters, us: 5 rows of 32003 and logs of 131,072 tokens 17.5 and 10.6, one of 151936 20.6 and 10.5, with a log of 2,000 3.2 and 3.4).
  // More rows read their logs faster in pieces of 4096 and 8192 (16 rows of 151936 and logs of 131,072 tokens 29, in clusters 39).
  // (The lengths are on the device: what the host knows of the logs, for this and for the counts' words, is how long they may become.)
  const auto ctas = [&](int piece) { return (long long)rows * ((V + 3 + piece - 1) / piece); };
  const bool word = capacity < 65536;
  const auto run = [&](auto threads, auto pieces, auto walk, auto packed, auto split) {
    constexpr int T = decltype(threads)::value, P = decltype(pieces)::value, L = decltype(walk)::value, S = decltype(split)::value;
    constexpr int C = T * 4 * P * L, CC = C * S;
    constexpr bool W = decltype(packed)::value;
    constexpr int most = 4 * Counts<W>::kWords * CC + 2 * C;
    const int bytes = 4 * Counts<W>::kWords * CC + 2 * (C < capacity ? C : capacity);      // (the list has a place for every token of a log)
    if (most > 40 * 1024) {
      static const cudaError_t asked = cudaFuncSetAttribute(logit_rules_kernel<T, P, L, W, S>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
      if (asked != cudaSuccess) note_launch_error(asked);
    }
    const dim3 grid((V + 3 + CC - 1) / CC * S, rows);
    if (S > 1) launch_chained_cluster(logit_rules_kernel<T, P, L, W, S>, grid, dim3(T), (size_t)bytes, stream, S, a);
    else launch_chained(logit_rules_kernel<T, P, L, W, S>, grid, dim3(T), (size_t)bytes, stream, a);
  };
  const Int<512> threads;
  if (ctas(16384) >= 6 * 148) {
    if (word) run(threads, Int<2>{}, Int<4>{}, Int<1>{}, Int<1>{}); else run(threads, Int<2>{}, Int<2>{}, Int<0>{}, Int<1>{});
  } else if (ctas(8192) >= 2 * 148) {
    if (word) run(threads, Int<2>{}, Int<2>{}, Int<1>{}, Int<1>{}); else run(threads, Int<2>{}, Int<2>{}, Int<0>{}, Int<1>{});
  } else if (ctas(4096) >= 2 * 148) {
    if (word) run(threads, Int<2>{}, Int<1>{}, Int<1>{}, Int<1>{}); else run(threads, Int<2>{}, Int<1>{}, Int<0>{}, Int<1>{});
  } else {
    if (word) run(threads, Int<1>{}, Int<1>{}, Int<1>{}, Int<1>{}); else run(threads, Int<1>{}, Int<1>{}, Int<0>{}, Int<4>{});
  }
  return check_launch("logit_rules");
}

// 0, or 1 + a row (or an appended entry) whose slot, length, start, mask or biases did not fit since the last call.  Synchronises.
extern "C" int nf_rules_index_status() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_rules_error, sizeof(int)) != cudaSuccess) return -1;
  if (v) cudaMemcpyToSymbol(g_rules_error, &zero, sizeof(int));
  return v;
}
