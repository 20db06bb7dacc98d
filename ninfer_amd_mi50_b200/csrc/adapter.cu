// Low-rank adapters of a step's rows beside a shared projection, on CUDA cores: the float32 form, and bfloat16 products
// whose rows are not 16-byte pieces.
//
//   y[t, f] = z[t, f] + sum_r h[t, slice(f) R + r] B[a, f, r],   h[t, j] = s[a] sum_k x[t, k] A[a, j, k],   a = ids[t]
//
// z is the shared product in float32.  A row without an adapter (ids -1) keeps it.  All sums are float32.
//
// What bounds it: a row's adapter is S R K + N R numbers that have to be read once; few rows are a matter of latency.  The
// first kernel gives a warp one number of h.  The second gives a thread one feature and 8 rows, whose B row stays in registers
// as long as the rows' adapter does not change: within a request every row has the same.  Few float32 rows are served by
// `adapter_rows_f32_kernel` instead, which computes the shared product itself.
#include "common.cuh"

namespace nf {

__device__ int g_adapter_error = 0;     // 1 + the first row whose adapter lay outside the pool; read by nf_adapter_index_status

// The adapter of row t: -1 for none, and for one that does not exist.
__device__ __forceinline__ int adapter_of(const int* ids, int t, int n) {
  const int a = ids[t];
  if (a >= n) atomicCAS(&g_adapter_error, 0, t + 1);
  return a >= 0 && a < n ? a : -1;
}

template <typename T> struct Piece;      // numbers of a 16-byte piece
template <> struct Piece<float> { static constexpr int n = 4; };
template <> struct Piece<__nv_bfloat16> { static constexpr int n = 8; };
__device__ __forceinline__ void load_piece(const float* p, float* v) { load4(p, v); }
__device__ __forceinline__ void load_piece(const __nv_bfloat16* p, float* v) { load8(p, v); }
__device__ __forceinline__ void piece_floats(const uint4& raw, float (&v)[8]) { unpack8(raw, v); }
__device__ __forceinline__ void piece_floats(const uint4& raw, float (&v)[4]) {
  v[0] = __uint_as_float(raw.x); v[1] = __uint_as_float(raw.y); v[2] = __uint_as_float(raw.z); v[3] = __uint_as_float(raw.w);
}

constexpr int kShrinkWarps = 8;

// h[t, j], JW numbers a warp.  Four pieces of each row of A and of x a lane are under way at a time: with one, a row of 2,048 numbers
// is eight trips to memory in turn.  Two numbers a warp where there are many: what these CTAs hold of the SMs' registers, the product
// behind them, which has begun by then, has to wait for.  16 rows of 2048 and rank 16: 4.9 us under the profiler, launch and two trips to
// memory; 512 rows 7.0 in float32, x and A from L2 by then (17 in bfloat16 of 2044, number by number).
template <typename T, int JW>
__global__ void __launch_bounds__(32 * kShrinkWarps)
adapter_shrink_kernel(const T* __restrict__ x, const T* __restrict__ A, const float* __restrict__ scale, const int* __restrict__ ids,
                      float* __restrict__ h, int K, int SR, int n, int whole) {
  chain_wait(x, A, scale, ids);
  chain_release_late();                  // a product launched behind this may begin: what came before is complete
  const int t = blockIdx.x, j = (blockIdx.y * kShrinkWarps + (threadIdx.x >> 5)) * JW, lane = threadIdx.x & 31;
  const int a = adapter_of(ids, t, n);
  if (a < 0 || j >= SR) return;          // (SR is a multiple of 16)
  constexpr int P = Piece<T>::n, U = 4;
  const T* xr = x + (size_t)t * K;
  const T* row = A + ((size_t)a * SR + j) * K;
  float sum[JW];
#pragma unroll
  for (int q = 0; q < JW; ++q) sum[q] = 0.f;
  if (whole) {
    for (int k0 = lane * P; k0 < K; k0 += U * 32 * P) {
      uint4 u[U][JW], v[U];
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (k0 + i * 32 * P < K) {
          v[i] = *reinterpret_cast<const uint4*>(xr + k0 + i * 32 * P);
#pragma unroll
          for (int q = 0; q < JW; ++q) u[i][q] = *reinterpret_cast<const uint4*>(row + (size_t)q * K + k0 + i * 32 * P);
        }
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (k0 + i * 32 * P < K) {
          float xv[P], av[P];
          piece_floats(v[i], xv);
#pragma unroll
          for (int q = 0; q < JW; ++q) {
            piece_floats(u[i][q], av);
#pragma unroll
            for (int e = 0; e < P; ++e) sum[q] = fmaf(av[e], xv[e], sum[q]);
          }
        }
    }
  } else {
    for (int k = lane; k < K; k += 32)
#pragma unroll
      for (int q = 0; q < JW; ++q) sum[q] = fmaf(to_float(row[(size_t)q * K + k]), to_float(xr[k]), sum[q]);
  }
#pragma unroll
  for (int q = 0; q < JW; ++q) {
    const float v = warp_sum(sum[q]);
    if (lane == 0) h[(size_t)t * SR + j + q] = v * scale[a];
  }
}

template <typename T>
static void launch_shrink(const void* x, const void* A, const float* scale, const int* ids, float* h, int rows, int K, int SR, int n,
                          cudaStream_t stream) {
  const int whole = (K * (int)sizeof(T)) % 16 == 0;
  const bool two = (long long)rows * SR >= 16 * kShrinkWarps;
  const int at_once = kShrinkWarps * (two ? 2 : 1);
  launch_chained(two ? adapter_shrink_kernel<T, 2> : adapter_shrink_kernel<T, 1>, dim3(rows, (SR + at_once - 1) / at_once),
                 dim3(32 * kShrinkWarps), 0, stream, (const T*)x, (const T*)A, scale, ids, h, K, SR, n, whole);
}

// The bfloat16 form alone, for adapter_tc.cu.
int adapter_shrink_simt(const void* x, const void* A, const float* scale, const int* ids, float* h, int rows, int K, int SR, int n,
                        cudaStream_t stream) {
  launch_shrink<__nv_bfloat16>(x, A, scale, ids, h, rows, K, SR, n, stream);
  return check_launch("adapter_shrink");
}

struct AdapterSlices {                    // features below end[s] belong to slice s
  int n;
  int end[8];
};

constexpr int kExpandRows = 8;

// R numbers a feature; rank in pieces of 16 numbers so that a feature's row stays in registers.  What bounds it: z in and y out, 512 rows
// of 2048 in float32 8.4 MB, 1.3 us; 16 under the profiler, since 512 CTAs wait for one trip to memory after the other (ids, z, B, h).
// It serves what is not worth more: float32 beyond 64 rows, where the product before it takes 142, and rows that TMA cannot fetch.
template <typename T, typename TY>
__global__ void __launch_bounds__(256)
adapter_expand_kernel(const float* __restrict__ z, const float* __restrict__ h, const T* __restrict__ B, const int* __restrict__ ids,
                      TY* __restrict__ y, int rows, int N, int R, int SR, int n, AdapterSlices slices) {
  chain_wait(z, h, B, ids);
  const int f = blockIdx.x * blockDim.x + threadIdx.x, t0 = blockIdx.y * kExpandRows;
  if (f >= N) return;
  int s = 0;
  while (s + 1 < slices.n && f >= slices.end[s]) ++s;
  float sum[kExpandRows];
  int own[kExpandRows];
#pragma unroll
  for (int i = 0; i < kExpandRows; ++i) {
    const int t = t0 + i;
    own[i] = t < rows ? adapter_of(ids, t, n) : -1;
    sum[i] = t < rows ? z[(size_t)t * N + f] : 0.f;
  }
  for (int r0 = 0; r0 < R; r0 += 16) {
    float b[16];
    int held = -1;
#pragma unroll
    for (int i = 0; i < kExpandRows; ++i) {
      if (own[i] < 0) continue;
      if (own[i] != held) {
        held = own[i];
        const T* row = B + ((size_t)held * N + f) * R + r0;
#pragma unroll
        for (int c = 0; c < 16; c += Piece<T>::n) load_piece(row + c, b + c);
      }
      const float* hr = h + (size_t)(t0 + i) * SR + s * R + r0;
#pragma unroll
      for (int c = 0; c < 16; ++c) sum[i] = fmaf(hr[c], b[c], sum[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < kExpandRows; ++i)
    if (t0 + i < rows) y[(size_t)(t0 + i) * N + f] = from_float<TY>(sum[i]);
}

// ---- few float32 rows: the shared product with the adapters' part in its epilogue ----------------------------------------------

// What bounds it: reading W once (2048 x 2048: 16.8 MB, 2.6 us; 16 rows 11 to 14 with h, 135 as library products and gathers), and beyond a
// few rows x, which every CTA reads for its four features.  A CTA takes four features and RB rows of x; its eight warps take k in
// turn, 128 numbers a step, so that the SMs have enough of W under way; a lane multiplies its four numbers of each of the four rows
// of W with those of the RB rows of x, which come out of L1.  The lanes' sums are added while they are dealt out (2 RB - 2 shuffles
// instead of five for every sum), the warps' in their order.  Sums of K / 256 terms a lane, then of few: less is lost than in one
// chain over k.
constexpr int kF32Warps = 8, kF32Features = 4;

// The sums of C numbers a lane over the warp, dealt out: halves change hands until each lane has C / 32 of them, or 32 / C lanes the
// same one.  `base`: the first of the lane's.
template <int C, int O>
__device__ __forceinline__ void deal_sums(float* sum, int lane, int& base) {
  if constexpr (O > 0) {
    if constexpr (C > 1) {
      const bool high = lane & O;
#pragma unroll
      for (int i = 0; i < C / 2; ++i) {
        const float give = high ? sum[i] : sum[i + C / 2], keep = high ? sum[i + C / 2] : sum[i];
        sum[i] = keep + __shfl_xor_sync(0xffffffffu, give, O);
      }
      base += high ? C / 2 : 0;
      deal_sums<C / 2, O / 2>(sum, lane, base);
    } else {
      sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], O);
      deal_sums<1, O / 2>(sum, lane, base);
    }
  }
}

template <int RB>
__global__ void __launch_bounds__(32 * kF32Warps, RB == 4 ? 3 : 2)
adapter_rows_f32_kernel(const float* __restrict__ x, const float* __restrict__ W, const float* __restrict__ h, const float* __restrict__ B,
                        const int* __restrict__ ids, float* __restrict__ y, int rows, int N, int K, int R, int SR, int n,
                        const __grid_constant__ AdapterSlices slices) {
  constexpr int NV = RB * kF32Features;              // sums of a CTA: [row][feature]
  __shared__ float part[kF32Warps][NV];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int f0 = blockIdx.x * kF32Features, t0 = blockIdx.y * RB;
  const float* wr[kF32Features];
#pragma unroll
  for (int i = 0; i < kF32Features; ++i) wr[i] = W + (size_t)min(f0 + i, N - 1) * K;
  const float* x0 = x + (size_t)t0 * K;
  const int t_most = min(RB, rows - t0) - 1;         // (rows beyond are computed as the last one, and not written)
  float sum[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) sum[i] = 0.f;
  // (x is complete: the kernel before this one waited for what wrote it, and let this one begin)
  constexpr int STEP = 128 * kF32Warps;
  for (int k0 = warp * 128 + lane * 4; k0 < K; k0 += 2 * STEP) {
    float w[2][kF32Features][4];
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (k0 + u * STEP < K) {
#pragma unroll
        for (int i = 0; i < kF32Features; ++i) load4(wr[i] + k0 + u * STEP, w[u][i]);
      }
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (k0 + u * STEP < K) {
#pragma unroll
        for (int r = 0; r < RB; ++r) {
          float v[4];
          load4(x0 + (size_t)min(r, t_most) * K + k0 + u * STEP, v);
#pragma unroll
          for (int i = 0; i < kF32Features; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[r * kF32Features + i] = fmaf(w[u][i][e], v[e], sum[r * kF32Features + i]);
        }
      }
  }
  int base = 0;
  deal_sums<NV, 16>(sum, lane, base);
  constexpr int LEFT = NV >= 32 ? NV / 32 : 1;
#pragma unroll
  for (int i = 0; i < LEFT; ++i) part[warp][base + i] = sum[i];      // (two lanes that share a sum write the same)
  __syncthreads();
  chain_wait(h);
  // four threads a sum, a quarter of the ranks each
  const int q = threadIdx.x & 3;
  for (int i = threadIdx.x >> 2; i < NV; i += 8 * kF32Warps) {      // (NV is a multiple of the eight sums of a warp)
    const int t = t0 + i / kF32Features, f = f0 + i % kF32Features;
    const bool live = t < rows && f < N;
    float add = 0.f;
    if (live) {
      const int a = blockIdx.x == 0 && q == 0 && i % kF32Features == 0 ? adapter_of(ids, t, n) : (ids[t] < n ? ids[t] : -1);
      if (a >= 0) {
        int s = 0;
        while (s + 1 < slices.n && f >= slices.end[s]) ++s;
        const float* b = B + ((size_t)a * N + f) * R;
        const float* hr = h + (size_t)t * SR + s * R;
        for (int r = 4 * q; r < R; r += 16) {
          float u[4], v[4];
          load4(b + r, u);
          load4(hr + r, v);
#pragma unroll
          for (int e = 0; e < 4; ++e) add = fmaf(u[e], v[e], add);
        }
      }
    }
    add += __shfl_xor_sync(0xffffffffu, add, 1);
    add += __shfl_xor_sync(0xffffffffu, add, 2);
    if (live && q == 0) {
      float z = part[0][i];
#pragma unroll
      for (int w = 1; w < kF32Warps; ++w) z += part[w][i];
      y[(size_t)t * N + f] = z + add;
    }
  }
}

template <int RB>
static void launch_rows_f32(const void* x, const void* W, const void* A, const void* B, const float* scale, const int* ids, float* h, void* y,
                            int rows, int N, int K, int R, int n, const AdapterSlices& slices, cudaStream_t stream) {
  const int SR = slices.n * R;
  launch_shrink<float>(x, A, scale, ids, h, rows, K, SR, n, stream);
  launch_chained(adapter_rows_f32_kernel<RB>, dim3((N + kF32Features - 1) / kF32Features, (rows + RB - 1) / RB), dim3(32 * kF32Warps), 0, stream,
                 (const float*)x, (const float*)W, (const float*)h, (const float*)B, ids, (float*)y, rows, N, K, R, SR, n, slices);
}

template <typename T, typename TY>
static int launch_adapter(const void* x, const void* A, const void* B, const float* scale, const int* ids, const float* z, float* h,
                          void* y, int rows, int N, int K, int R, int n, const AdapterSlices& slices, cudaStream_t stream) {
  const int SR = slices.n * R;
  launch_shrink<T>(x, A, scale, ids, h, rows, K, SR, n, stream);
  launch_chained(adapter_expand_kernel<T, TY>, dim3((N + 255) / 256, (rows + kExpandRows - 1) / kExpandRows), dim3(256), 0, stream, z,
                 (const float*)h, (const T*)B, ids, (TY*)y, rows, N, R, SR, n, slices);
  return check_launch("adapter_add");
}

}  // namespace nf

using namespace nf;

// y = x W^T + the adapters' part in float32, for few rows: x [rows, K], W [N, K], A [n, n_slices * R, K], B [n, N, R], y [rows, N],
// h scratch [rows, n_slices * R]; ends as below.  K a multiple of 4, R of 16, bases 16-byte aligned.
extern "C" int nf_adapter_rows_f32(const void* x, const void* W, const void* A, const void* B, const float* scale, const int* ids, float* h,
                                   void* y, int rows, int N, int K, int R, int n, int n_slices, const int* ends, cudaStream_t stream) {
  if (rows == 0 || N == 0) return 0;
  NF_REQUIRE(rows > 0 && N > 0 && K > 0 && n > 0, "adapter_rows_f32: bad sizes rows=%d N=%d K=%d n=%d", rows, N, K, n);
  NF_REQUIRE(K % 4 == 0 && R > 0 && R % 16 == 0, "adapter_rows_f32: K=%d must be a multiple of 4, rank %d of 16", K, R);
  NF_REQUIRE(n_slices >= 1 && n_slices <= 8, "adapter_rows_f32: %d slices, 1 to 8", n_slices);
  NF_REQUIRE(rows <= 65535, "adapter_rows_f32: %d rows, at most 65535", rows);
  NF_REQUIRE((uintptr_t)x % 16 == 0 && (uintptr_t)W % 16 == 0 && (uintptr_t)A % 16 == 0 && (uintptr_t)B % 16 == 0 && (uintptr_t)h % 16 == 0,
             "adapter_rows_f32: operands must be 16-byte aligned");
  AdapterSlices s{n_slices, {}};
  for (int i = 0; i < n_slices; ++i) s.end[i] = ends[i];
  NF_REQUIRE(s.end[n_slices - 1] == N, "adapter_rows_f32: the slices end at %d of %d features", s.end[n_slices - 1], N);
  if (rows <= 4) launch_rows_f32<4>(x, W, A, B, scale, ids, h, y, rows, N, K, R, n, s, stream);
  else if (rows <= 8) launch_rows_f32<8>(x, W, A, B, scale, ids, h, y, rows, N, K, R, n, s, stream);
  else launch_rows_f32<16>(x, W, A, B, scale, ids, h, y, rows, N, K, R, n, s, stream);
  return check_launch("adapter_rows_f32");
}

// y = z + the adapters' part (see the head of this file).  z float32 [rows, N], h float32 scratch [rows, n_slices * R]; x, A
// [n, n_slices * R, K], B [n, N, R] of `dtype`, y of `y_dtype` (the same, or float32); ends: the n_slices features (host memory) at which the slices end, the
// last N.  R: a multiple of 16.  All bases 16-byte aligned.
extern "C" int nf_adapter_add(const void* x, const void* A, const void* B, const float* scale, const int* ids, const float* z,
                              float* h, void* y, int rows, int N, int K, int R, int n, int n_slices, const int* ends, int dtype,
                              int y_dtype, cudaStream_t stream) {
  if (rows == 0 || N == 0) return 0;
  NF_REQUIRE(rows > 0 && N > 0 && K > 0 && n > 0, "adapter_add: bad sizes rows=%d N=%d K=%d n=%d", rows, N, K, n);
  NF_REQUIRE(R > 0 && R % 16 == 0, "adapter_add: rank %d must be a multiple of 16", R);
  NF_REQUIRE(n_slices >= 1 && n_slices <= 8, "adapter_add: %d slices, 1 to 8", n_slices);
  NF_REQUIRE(rows <= 65535 * kExpandRows, "adapter_add: %d rows, at most %d", rows, 65535 * kExpandRows);
  NF_REQUIRE((uintptr_t)x % 16 == 0 && (uintptr_t)A % 16 == 0 && (uintptr_t)B % 16 == 0 && (uintptr_t)h % 16 == 0,
             "adapter_add: operands must be 16-byte aligned");
  AdapterSlices s{n_slices, {}};
  for (int i = 0; i < n_slices; ++i) s.end[i] = ends[i];
  NF_REQUIRE(s.end[n_slices - 1] == N, "adapter_add: the slices end at %d of %d features", s.end[n_slices - 1], N);
  NF_REQUIRE(y_dtype == dtype || y_dtype == kF32, "adapter_add: the result is float32 or of the operands' type");
  if (dtype == kBF16 && y_dtype == kBF16)
    return launch_adapter<__nv_bfloat16, __nv_bfloat16>(x, A, B, scale, ids, z, h, y, rows, N, K, R, n, s, stream);
  if (dtype == kBF16) return launch_adapter<__nv_bfloat16, float>(x, A, B, scale, ids, z, h, y, rows, N, K, R, n, s, stream);
  return launch_adapter<float, float>(x, A, B, scale, ids, z, h, y, rows, N, K, R, n, s, stream);
}

// 0, or 1 + a row whose adapter lay outside the pool since the last call (it was served without one).  Synchronises.
extern "C" int nf_adapter_index_status() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_adapter_error, sizeof(int)) != cudaSuccess) return -1;
  if (v) cudaMemcpyToSymbol(g_adapter_error, &zero, sizeof(int));
  return v;
}
