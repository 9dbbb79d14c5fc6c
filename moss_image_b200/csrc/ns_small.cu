// Orthogonalised update of matrices with a short side of at most 64 (adapter factors).
//
// With R = X X^T, a step X <- (a I + b R + c R R) X =: P X turns R into P R P, so the whole iteration
// stays on the r x r square: Q <- P Q, R <- P R P, and the result is Q X. X is read twice (once
// for R, whose trace is the squared Frobenius norm, once for Q X) however many steps there are,
// instead of three times a step. All of it is f32: R's small eigenvalues, which grow by (a^2) a step,
// need its precision, and Q X is rounded once.
//
// Three launches: partial R over column ranges, the iteration (one CTA per matrix), Q X.
#include <algorithm>
#include <mutex>

#include "ns_args.cuh"

namespace moss {
namespace ns {
namespace {

constexpr int kThreads = 256;
constexpr int kCols = 64;  // columns of X in shared memory at a time

// kCols columns of X from column c0, as xs[column][row]; zero past r and c.
template <int kSide>
__device__ __forceinline__ void load_columns(const Small& s, int64_t b, int c0, float (*xs)[kSide + 4]) {
  const int64_t base = b * s.r * s.c;
  if (s.tall) {  // G [c][r]: columns of X are rows of G
    for (int i = threadIdx.x; i < kCols * kSide; i += kThreads) {
      const int row = i % kSide, col = i / kSide;
      const bool in = row < s.r && c0 + col < s.c;
      xs[col][row] = in ? load_as_float(s.g, s.dtype, base + static_cast<int64_t>(c0 + col) * s.r + row) : 0.0f;
    }
  } else {
    for (int i = threadIdx.x; i < kCols * kSide; i += kThreads) {
      const int col = i % kCols, row = i / kCols;
      const bool in = row < s.r && c0 + col < s.c;
      xs[col][row] = in ? load_as_float(s.g, s.dtype, base + static_cast<int64_t>(row) * s.c + c0 + col) : 0.0f;
    }
  }
}

// Partial X X^T over this CTA's column range. A thread sums a 4 x 4 piece over every kSlices-th column.
template <int kSide>
__global__ void __launch_bounds__(kThreads) small_gram_kernel(const Small s) {
  constexpr int kPieces = (kSide / 4) * (kSide / 4);
  constexpr int kSlices = kThreads / kPieces;
  __shared__ __align__(16) float xs[kCols][kSide + 4];
  __shared__ float join[kSlices > 1 ? kThreads * 16 : 1];
  const int64_t b = blockIdx.y;
  const int ranges = (s.c + kCols - 1) / kCols;
  const int first = static_cast<int>(static_cast<int64_t>(blockIdx.x) * ranges / s.chunks);
  const int last = static_cast<int>(static_cast<int64_t>(blockIdx.x + 1) * ranges / s.chunks);
  const int piece = threadIdx.x % kPieces, slice = threadIdx.x / kPieces;
  const int i0 = piece / (kSide / 4) * 4, j0 = piece % (kSide / 4) * 4;
  float acc[4][4] = {};
  for (int t = first; t < last; ++t) {
    __syncthreads();
    load_columns<kSide>(s, b, t * kCols, xs);
    __syncthreads();
#pragma unroll 4
    for (int k = slice; k < kCols; k += kSlices) {
      const float4 u = *reinterpret_cast<const float4*>(&xs[k][i0]);
      const float4 v = *reinterpret_cast<const float4*>(&xs[k][j0]);
      const float x[4] = {u.x, u.y, u.z, u.w}, y[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(x[i], y[j], acc[i][j]);
    }
  }
  float* out = s.partial + (b * s.chunks + blockIdx.x) * kSide * kSide;
  if constexpr (kSlices > 1) {
#pragma unroll
    for (int e = 0; e < 16; ++e) join[threadIdx.x * 16 + e] = acc[e / 4][e % 4];
    __syncthreads();
    for (int e = threadIdx.x; e < kPieces * 16; e += kThreads) {
      float v = 0.0f;
      for (int k = 0; k < kSlices; ++k) v += join[k * kPieces * 16 + e];
      const int p = e / 16;
      out[(p / (kSide / 4) * 4 + (e % 16) / 4) * kSide + p % (kSide / 4) * 4 + e % 4] = v;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<float4*>(out + (i0 + i) * kSide + j0) = make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
  }
}

// z = x^T y, kSide x kSide in shared memory (x^T = x for the symmetric P).
template <int kSide>
__device__ __forceinline__ void multiply(const float (*x)[kSide + 4], const float (*y)[kSide + 4],
                                         float (&z)[kSide * kSide / kThreads]) {
  constexpr int kT = kSide == 64 ? 4 : kSide == 32 ? 2 : 1;
  const int i0 = threadIdx.x / (kSide / kT) * kT, j0 = threadIdx.x % (kSide / kT) * kT;
#pragma unroll
  for (int e = 0; e < kT * kT; ++e) z[e] = 0.0f;
#pragma unroll 8
  for (int k = 0; k < kSide; ++k) {
    float u[kT], v[kT];
#pragma unroll
    for (int e = 0; e < kT; ++e) {
      u[e] = x[k][i0 + e];
      v[e] = y[k][j0 + e];
    }
#pragma unroll
    for (int i = 0; i < kT; ++i)
#pragma unroll
      for (int j = 0; j < kT; ++j) z[i * kT + j] = fmaf(u[i], v[j], z[i * kT + j]);
  }
}

template <int kSide>
__global__ void __launch_bounds__(kThreads) small_iterate_kernel(const Small s) {
  constexpr int kT = kSide == 64 ? 4 : kSide == 32 ? 2 : 1;
  using Row = float[kSide + 4];
  extern __shared__ __align__(16) float smem[];
  Row* R = reinterpret_cast<Row*>(smem);
  Row* P = R + kSide;
  Row* Q = P + kSide;
  Row* T = Q + kSide;
  const int64_t b = blockIdx.x;
  const int i0 = threadIdx.x / (kSide / kT) * kT, j0 = threadIdx.x % (kSide / kT) * kT;
  const float* partial = s.partial + b * s.chunks * kSide * kSide;
  for (int e = threadIdx.x; e < kSide * kSide; e += kThreads) {
    float v = 0.0f;
    for (int k = 0; k < s.chunks; ++k) v += partial[static_cast<int64_t>(k) * kSide * kSide + e];
    R[e / kSide][e % kSide] = v;
  }
  __syncthreads();
  float trace = 0.0f;
  for (int i = 0; i < s.r; ++i) trace += R[i][i];
  const float norm = sqrtf(trace);
  // NaN stays NaN: every entry then is
  const float inv = 1.0f / (norm < s.eps ? s.eps : norm);
  __syncthreads();
  for (int e = threadIdx.x; e < kSide * kSide; e += kThreads) {
    const int i = e / kSide, j = e % kSide;
    R[i][j] = R[i][j] * inv * inv;
    Q[i][j] = i == j ? inv : 0.0f;
  }
  float z[kSide * kSide / kThreads];
  auto put = [&](Row* to) {
#pragma unroll
    for (int i = 0; i < kT; ++i)
#pragma unroll
      for (int j = 0; j < kT; ++j) to[i0 + i][j0 + j] = z[i * kT + j];
  };
  auto put_transposed = [&](Row* to) {
#pragma unroll
    for (int i = 0; i < kT; ++i)
#pragma unroll
      for (int j = 0; j < kT; ++j) to[j0 + j][i0 + i] = z[i * kT + j];
  };
  for (int step = 0; step < s.steps; ++step) {
    const float ca = s.coefficients[3 * step], cb = s.coefficients[3 * step + 1], cc = s.coefficients[3 * step + 2];
    __syncthreads();
    multiply<kSide>(R, R, z);
#pragma unroll
    for (int i = 0; i < kT; ++i)
#pragma unroll
      for (int j = 0; j < kT; ++j)
        z[i * kT + j] = (i0 + i == j0 + j ? ca : 0.0f) + cb * R[i0 + i][j0 + j] + cc * z[i * kT + j];
    put(P);
    __syncthreads();
    multiply<kSide>(P, Q, z);
    __syncthreads();
    put(Q);
    if (step + 1 == s.steps) break;
    // (P R) P in this order: R P P is the same only without rounding, and its error would not shrink
    // with R's small eigenvalues
    multiply<kSide>(P, R, z);
    put_transposed(T);
    __syncthreads();
    multiply<kSide>(T, P, z);
    put(R);
  }
  __syncthreads();
  float* q = s.q + b * kSide * kSide;  // Q^T
  for (int e = threadIdx.x; e < kSide * kSide; e += kThreads) q[e] = Q[e % kSide][e / kSide];
}

// out = Q X for kCols columns.
template <int kSide>
__global__ void __launch_bounds__(kThreads) small_apply_kernel(const Small s) {
  __shared__ __align__(16) float xs[kCols][kSide + 4];
  __shared__ __align__(16) float q[kSide][kSide + 4];  // Q^T
  const int64_t b = blockIdx.y;
  for (int e = threadIdx.x; e < kSide * kSide; e += kThreads) q[e / kSide][e % kSide] = s.q[b * kSide * kSide + e];
  const int c0 = blockIdx.x * kCols;
  load_columns<kSide>(s, b, c0, xs);
  __syncthreads();
  // a thread: 4 columns x kSide / 16 rows
  constexpr int kRows = kSide / 16;
  const int j0 = threadIdx.x % 16 * 4, i0 = threadIdx.x / 16 * kRows;
  float acc[kRows][4] = {};
#pragma unroll 4
  for (int k = 0; k < kSide; ++k) {
    float x[4], w[kRows];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = xs[j0 + j][k];
#pragma unroll
    for (int i = 0; i < kRows; ++i) w[i] = q[k][i0 + i];
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(w[i], x[j], acc[i][j]);
  }
  __nv_bfloat16* out = s.out + b * s.r * s.c;
#pragma unroll
  for (int i = 0; i < kRows; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = i0 + i, col = c0 + j0 + j;
      if (row >= s.r || col >= s.c) continue;
      out[s.tall ? static_cast<int64_t>(col) * s.r + row : static_cast<int64_t>(row) * s.c + col] =
          __float2bfloat16_rn(acc[i][j]);
    }
}

template <int kSide>
int launch_typed(const Small& s, cudaStream_t stream) {
  constexpr int kIterateBytes = 4 * kSide * (kSide + 4) * 4;
  static std::once_flag once;
  static cudaError_t attr_err = cudaSuccess;
  std::call_once(once, [] {
    attr_err = cudaFuncSetAttribute(small_iterate_kernel<kSide>, cudaFuncAttributeMaxDynamicSharedMemorySize, kIterateBytes);
  });
  MOSS_CUDA_TRY(attr_err);
  const unsigned batch = static_cast<unsigned>(s.batch);
  small_gram_kernel<kSide><<<dim3(s.chunks, batch), kThreads, 0, stream>>>(s);
  MOSS_CUDA_TRY(cudaGetLastError());
  small_iterate_kernel<kSide><<<batch, kThreads, kIterateBytes, stream>>>(s);
  MOSS_CUDA_TRY(cudaGetLastError());
  small_apply_kernel<kSide><<<dim3((s.c + kCols - 1) / kCols, batch), kThreads, 0, stream>>>(s);
  return check_cuda(cudaGetLastError(), "small_apply_kernel");
}

}  // namespace

int small_side(int r) { return r <= 16 ? 16 : r <= 32 ? 32 : 64; }

int small_chunks(int64_t batch, int c, int sms) {
  const int64_t ranges = (c + kCols - 1) / kCols;
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(ranges, 4LL * sms / std::max<int64_t>(1, batch))));
}

int launch_small(const Small& s, cudaStream_t stream) {
  switch (small_side(s.r)) {
    case 16: return launch_typed<16>(s, stream);
    case 32: return launch_typed<32>(s, stream);
    default: return launch_typed<64>(s, stream);
  }
}

}  // namespace ns
}  // namespace moss
