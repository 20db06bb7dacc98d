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

// set by a row whose slot, length or start does not fit the log: 1 + the row; read by nf_rules_index_status
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

constexpr int kRuleThreads = 256;

// PIECES: runs of four logits a thread; a CTA's piece of the vocabulary is kRuleThreads * 4 * PIECES of them, counted from the
// last 16-byte boundary at or before the row's start.
template <int PIECES>
__global__ void __launch_bounds__(kRuleThreads)
logit_rules_kernel(RuleArgs a) {
  constexpr int C = kRuleThreads * 4 * PIECES;
  extern __shared__ __align__(16) unsigned rule_smem[];
  unsigned* all = rule_smem;                  // [C] occurrences anywhere
  unsigned* made = all + C;                   // [C] among the generated ones
  float* add = reinterpret_cast<float*>(made + C);   // [C] biases (where there are any)
  chain_wait();
  const int r = blockIdx.y, tid = threadIdx.x;
  const float* row = a.logits + (size_t)r * a.ld_in;
  float* out = a.out + (size_t)r * a.ld_out;
  const int pad = (int)(((uintptr_t)row >> 2) & 3);
  const int lo = (int)blockIdx.x * C - pad;   // the token of place 0
  const bool pairs = (((uintptr_t)out >> 2) & 3) == (unsigned)pad;       // runs of four are aligned on both sides

  float v[PIECES][4];
#pragma unroll
  for (int p = 0; p < PIECES; ++p) {
    const int i = lo + 4 * (tid + p * kRuleThreads);
    if (i >= 0 && i + 4 <= a.V) {
      load4(row + i, v[p]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[p][e] = i + e >= 0 && i + e < a.V ? row[i + e] : 0.f;
    }
  }
  for (int i = tid; i < 2 * C / 4; i += kRuleThreads) reinterpret_cast<uint4*>(all)[i] = make_uint4(0, 0, 0, 0);
  const bool biased = a.bias_offsets != nullptr;
  if (biased)
    for (int i = tid; i < C / 4; i += kRuleThreads) reinterpret_cast<float4*>(add)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  __syncthreads();

  // ---- the log's tokens that lie in this piece
  const float rep = a.penalties[3 * r], freq = a.penalties[3 * r + 1], pres = a.penalties[3 * r + 2];
  const int slot = a.slots[r];
  int len = a.lengths[r], start = a.starts[r];
  const bool fits = slot >= 0 && slot < a.n_slots && len >= (a.tokens ? 1 : 0) && len <= a.capacity;
  if (!fits || start < 0) {
    if (tid == 0) atomicCAS(&g_rules_error, 0, r + 1);
    start = max(start, 0);
    if (!fits) len = 0;
  }
  if (len > 0) {
    int* log = a.history + (size_t)slot * a.capacity;
    int from = rep != 1.f ? 0 : start;                 // earlier tokens count for the repetition penalty only
    if (rep == 1.f && freq == 0.f && pres == 0.f) from = len;
    const int end = a.tokens ? len - 1 : len;
    for (int i = (from & ~3) + 4 * tid; i < end; i += 4 * kRuleThreads) {
      const int4 t4 = *reinterpret_cast<const int4*>(log + i);
      const int t[4] = {t4.x, t4.y, t4.z, t4.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const unsigned d = (unsigned)(t[e] - lo);
        if (i + e >= from && i + e < end && d < (unsigned)C) {
          atomicAdd(&all[d], 1u);
          if (i + e >= start) atomicAdd(&made[d], 1u);
        }
      }
    }
    if (a.tokens && tid == 0) {
      const int t = a.tokens[r];
      const unsigned d = (unsigned)(t - lo);
      if (len - 1 >= from && d < (unsigned)C) {
        atomicAdd(&all[d], 1u);
        if (len - 1 >= start) atomicAdd(&made[d], 1u);
      }
      if (blockIdx.x == 0) log[len - 1] = t;
    }
  }
  if (biased) {
    const int b0 = max(a.bias_offsets[r], 0), b1 = min(a.bias_offsets[r + 1], a.n_bias);
    for (int i = b0 + tid; i < b1; i += kRuleThreads) {
      const unsigned d = (unsigned)(a.bias_ids[i] - lo);
      if (d < (unsigned)C) atomicAdd(&add[d], a.bias_values[i]);
    }
  }
  const int m = a.mask ? a.mask_index[r] : -1;
  if (a.mask && m >= a.mask_rows && tid == 0) atomicCAS(&g_rules_error, 0, r + 1);
  const unsigned* bits = a.mask && m >= 0 && m < a.mask_rows ? a.mask + (size_t)m * a.words : nullptr;
  __syncthreads();

#pragma unroll
  for (int p = 0; p < PIECES; ++p) {
    const int d0 = 4 * (tid + p * kRuleThreads), i0 = lo + d0;
    if (i0 + 4 <= 0 || i0 >= a.V) continue;
    const uint4 c4 = *reinterpret_cast<const uint4*>(all + d0), g4 = *reinterpret_cast<const uint4*>(made + d0);
    const unsigned c[4] = {c4.x, c4.y, c4.z, c4.w}, g[4] = {g4.x, g4.y, g4.z, g4.w};
    float b[4] = {0.f, 0.f, 0.f, 0.f};
    if (biased) load4(add + d0, b);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = i0 + e;
      if (i < 0 || i >= a.V) continue;
      float x = v[p][e];
      if (c[e] && rep != 1.f && x != 0.f && !isinf(x)) {       // (0 and the infinities stay what they are, whatever p^c is)
        const float times = powf(rep, (float)c[e]);
        x = x > 0.f ? x / times : x * times;
      }
      if (g[e]) x = x - (float)g[e] * freq - pres;
      if (biased) x += b[e];
      if (bits && !((bits[i >> 5] >> (i & 31)) & 1u)) x = -INFINITY;
      v[p][e] = x;
    }
    if (pairs && i0 >= 0 && i0 + 4 <= a.V) {
      store4(out + i0, v[p]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i0 + e >= 0 && i0 + e < a.V) out[i0 + e] = v[p][e];
    }
  }
}

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
// mask_index[r] is set where token i is allowed.  capacity: a multiple of 4; history 16-byte aligned.
extern "C" int nf_logit_rules(const float* logits, float* out, int* history, const int* slots, const int* lengths, const int* starts,
                              const int* tokens, const float* penalties, const int* bias_offsets, const int* bias_ids,
                              const float* bias_values, int n_bias, const unsigned* mask, const int* mask_index, int mask_rows,
                              int rows, int V, int ld_in, int ld_out, int n_slots, int capacity, cudaStream_t stream) {
  if (rows == 0) return 0;
  NF_REQUIRE(rows > 0 && rows <= 65535 && V > 0 && V <= (1 << 30), "logit_rules: bad sizes rows=%d V=%d", rows, V);
  NF_REQUIRE(ld_in >= V && ld_out >= V, "logit_rules: rows %d and %d apart for %d logits", ld_in, ld_out, V);
  NF_REQUIRE(n_slots > 0 && capacity > 0 && capacity % 4 == 0 && (uintptr_t)history % 16 == 0,
             "logit_rules: a log of %d slots with %d tokens (a multiple of 4), 16-byte aligned", n_slots, capacity);
  const RuleArgs a{logits, out, history, slots, lengths, starts, tokens, penalties, bias_offsets, bias_ids, bias_values, mask,
                   mask_index, V, ld_in, ld_out, n_slots, capacity, n_bias, mask_rows, (V + 31) / 32};
  constexpr int P = 2, C = kRuleThreads * 4 * P;
  const size_t smem = (size_t)C * 4 * (bias_offsets ? 3 : 2);
  launch_chained(logit_rules_kernel<P>, dim3((V + 3 + C - 1) / C, rows), dim3(kRuleThreads), smem, stream, a);
  return check_launch("logit_rules");
}

// 0, or 1 + a row (or an appended entry) whose slot, length, start or mask did not fit since the last call.  Synchronises.
extern "C" int nf_rules_index_status() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_rules_error, sizeof(int)) != cudaSuccess) return -1;
  if (v) cudaMemcpyToSymbol(g_rules_error, &zero, sizeof(int));
  return v;
}
