// Low-rank adapters of a step's rows beside a shared projection, on CUDA cores: the float32 form, and bfloat16 products
// whose rows are not 16-byte pieces.
//
//   y[t, f] = z[t, f] + sum_r h[t, slice(f) R + r] B[a, f, r],   h[t, j] = s[a] sum_k x[t, k] A[a, j, k],   a = ids[t]
//
// z is the shared product in float32.  A row without an adapter (ids -1) keeps it.  All sums are float32.
//
// What bounds it: a row's adapter is S R K + N R numbers that have to be read once; few rows are a matter of latency.  The
// first kernel gives a warp one number of h: K numbers of one row of A in 16-byte loads, the row of x in shared memory.
// The second gives a thread one feature and 8 rows, whose B row stays in registers as long as the rows' adapter does not
// change: within a request every row has the same.
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

constexpr int kShrinkWarps = 8;
constexpr int kShrinkK = 4096;           // numbers of a row of x that lie in shared memory at a time

// h[t, j0 .. j0 + 16 * warps) of one row
template <typename T>
__global__ void __launch_bounds__(32 * kShrinkWarps)
adapter_shrink_kernel(const T* __restrict__ x, const T* __restrict__ A, const float* __restrict__ scale, const int* __restrict__ ids,
                      float* __restrict__ h, int K, int SR, int n, int whole) {
  __shared__ float xs[kShrinkK];
  chain_wait(x, A, scale, ids);
  chain_release_late();                  // a product launched behind this may begin: what came before is complete
  const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int a = adapter_of(ids, t, n);
  if (a < 0) return;
  constexpr int P = Piece<T>::n;
  const T* At = A + (size_t)a * SR * K;
  for (int j0 = blockIdx.y * 2 * kShrinkWarps; j0 < SR; j0 += gridDim.y * 2 * kShrinkWarps) {
    const int j = j0 + 2 * warp;                       // this warp's two numbers
    float sum[2] = {0.f, 0.f};
    for (int k0 = 0; k0 < K; k0 += kShrinkK) {
      const int kn = min(kShrinkK, K - k0);
      __syncthreads();
      for (int k = threadIdx.x; k < kn; k += blockDim.x) xs[k] = to_float(x[(size_t)t * K + k0 + k]);
      __syncthreads();
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        if (j + q >= SR) break;
        const T* row = At + (size_t)(j + q) * K + k0;
        if (whole) {
          for (int k = lane * P; k < kn; k += 32 * P) {
            float v[P];
            load_piece(row + k, v);
#pragma unroll
            for (int i = 0; i < P; ++i) sum[q] = fmaf(v[i], xs[k + i], sum[q]);
          }
        } else {
          for (int k = lane; k < kn; k += 32) sum[q] = fmaf(to_float(row[k]), xs[k], sum[q]);
        }
      }
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const float v = warp_sum(sum[q]);
      if (lane == 0 && j + q < SR) h[(size_t)t * SR + j + q] = v * scale[a];
    }
  }
}

template <typename T>
static void launch_shrink(const void* x, const void* A, const float* scale, const int* ids, float* h, int rows, int K, int SR, int n,
                          cudaStream_t stream) {
  const int whole = (K * (int)sizeof(T)) % 16 == 0;
  launch_chained(adapter_shrink_kernel<T>, dim3(rows, (SR + 2 * kShrinkWarps - 1) / (2 * kShrinkWarps)), dim3(32 * kShrinkWarps), 0, stream,
                 (const T*)x, (const T*)A, scale, ids, h, K, SR, n, whole);
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

// R numbers a feature; rank in pieces of 16 numbers so that a feature's row stays in registers
template <typename T>
__global__ void __launch_bounds__(256)
adapter_expand_kernel(const float* __restrict__ z, const float* __restrict__ h, const T* __restrict__ B, const int* __restrict__ ids,
                      T* __restrict__ y, int rows, int N, int R, int SR, int n, AdapterSlices slices) {
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
    if (t0 + i < rows) y[(size_t)(t0 + i) * N + f] = from_float<T>(sum[i]);
}

template <typename T>
static int launch_adapter(const void* x, const void* A, const void* B, const float* scale, const int* ids, const float* z, float* h,
                          void* y, int rows, int N, int K, int R, int n, const AdapterSlices& slices, cudaStream_t stream) {
  const int SR = slices.n * R;
  launch_shrink<T>(x, A, scale, ids, h, rows, K, SR, n, stream);
  launch_chained(adapter_expand_kernel<T>, dim3((N + 255) / 256, (rows + kExpandRows - 1) / kExpandRows), dim3(256), 0, stream, z,
                 (const float*)h, (const T*)B, ids, (T*)y, rows, N, R, SR, n, slices);
  return check_launch("adapter_add");
}

}  // namespace nf

using namespace nf;

// y = z + the adapters' part (see the head of this file).  z float32 [rows, N], h float32 scratch [rows, n_slices * R]; x, A
// [n, n_slices * R, K], B [n, N, R] and y of `dtype`; ends: the n_slices features (host memory) at which the slices end, the
// last N.  R: a multiple of 16.  All bases 16-byte aligned.
extern "C" int nf_adapter_add(const void* x, const void* A, const void* B, const float* scale, const int* ids, const float* z,
                              float* h, void* y, int rows, int N, int K, int R, int n, int n_slices, const int* ends, int dtype,
                              cudaStream_t stream) {
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
  if (dtype == kBF16) return launch_adapter<__nv_bfloat16>(x, A, B, scale, ids, z, h, y, rows, N, K, R, n, s, stream);
  return launch_adapter<float>(x, A, B, scale, ids, z, h, y, rows, N, K, R, n, s, stream);
}

// 0, or 1 + a row whose adapter lay outside the pool since the last call (it was served without one).  Synchronises.
extern "C" int nf_adapter_index_status() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_adapter_error, sizeof(int)) != cudaSuccess) return -1;
  if (v) cudaMemcpyToSymbol(g_adapter_error, &zero, sizeof(int));
  return v;
}
