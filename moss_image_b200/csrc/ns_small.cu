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
// Columns of X in shared memory at a time: 32 KB of f32, rows 16 bytes past a multiple of 128 apart, so
// that 16-byte reads of neighbouring rows meet in different banks.
template <int kSide>
constexpr int kCols = 8192 / kSide;
template <int kSide>
constexpr int kPitch = kCols<kSide> + 4;

template <int kKind>
__device__ __forceinline__ float4 load4(const void* g, int64_t at) {
  if constexpr (kKind == kF32) {
    return __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(g) + at));
  } else {
    const uint2 w = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(g) + at));
    if constexpr (kKind == kBF16) {
      return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                         __uint_as_float(w.y & 0xffff0000u));
    } else {
      const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x));
      const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
      return make_float4(a.x, a.y, b.x, b.y);
    }
  }
}

// kCols columns of X from column c0, as xs[row][column]; zero past r and c. s.wide: groups of four values of
// a row of G are aligned and whole.
template <int kSide, int kKind>
__device__ __forceinline__ void load_columns(const Small& s, int64_t b, int c0, float* xs) {
  constexpr int kC = kCols<kSide>, kP = kPitch<kSide>;
  const int64_t base = b * s.r * s.c;
  if (!s.tall) {
#pragma unroll 8
    for (int i = threadIdx.x; i < kSide * kC / 4; i += kThreads) {
      const int row = i / (kC / 4), col = i % (kC / 4) * 4;
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      const int left = s.c - c0 - col;
      if (row < s.r && left > 0) {
        const int64_t at = base + static_cast<int64_t>(row) * s.c + c0 + col;
        if (s.wide) {
          v = load4<kKind>(s.g, at);
        } else {
          v.x = load_as_float(s.g, kKind, at);
          if (left > 1) v.y = load_as_float(s.g, kKind, at + 1);
          if (left > 2) v.z = load_as_float(s.g, kKind, at + 2);
          if (left > 3) v.w = load_as_float(s.g, kKind, at + 3);
        }
      }
      *reinterpret_cast<float4*>(xs + row * kP + col) = v;
    }
  } else {  // G [c][r]: four values of a row of G are four rows of one column of X
#pragma unroll 8
    for (int i = threadIdx.x; i < kSide * kC / 4; i += kThreads) {
      const int col = i % kC, row = i / kC * 4;
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      const int left = s.r - row;
      if (c0 + col < s.c && left > 0) {
        const int64_t at = base + static_cast<int64_t>(c0 + col) * s.r + row;
        if (s.wide) {
          v = load4<kKind>(s.g, at);
        } else {
          v.x = load_as_float(s.g, kKind, at);
          if (left > 1) v.y = load_as_float(s.g, kKind, at + 1);
          if (left > 2) v.z = load_as_float(s.g, kKind, at + 2);
          if (left > 3) v.w = load_as_float(s.g, kKind, at + 3);
        }
      }
      xs[row * kP + col] = v.x;
      xs[(row + 1) * kP + col] = v.y;
      xs[(row + 2) * kP + col] = v.z;
      xs[(row + 3) * kP + col] = v.w;
    }
  }
}

// Partial X X^T over this CTA's column range, upper half. With T = side / 8, piece (t, u), t <= u, is the
// 8 x 8 products of rows t, t + T, .. with rows u, u + T, ..; a thread sums one piece over every kSlices-th
// group of four columns. 64 multiply-adds for 16 values read is what keeps shared memory from
// being the bound (4 x 4 pieces took 53 us for 144 x 32 x 3072).
template <int kSide, int kKind>
__global__ void __launch_bounds__(kThreads, 2) small_gram_kernel(const Small s) {
  constexpr int kT = kSide / 8;
  constexpr int kPieces = kT * (kT + 1) / 2;
  constexpr int kSlices = kThreads / kPieces;
  constexpr int kC = kCols<kSide>, kP = kPitch<kSide>;
  extern __shared__ __align__(16) float xs[];
  const int64_t b = blockIdx.y;
  const int ranges = (s.c + kC - 1) / kC;
  const int first = static_cast<int>(static_cast<int64_t>(blockIdx.x) * ranges / s.chunks);
  const int last = static_cast<int>(static_cast<int64_t>(blockIdx.x + 1) * ranges / s.chunks);
  const int piece = threadIdx.x % kPieces, slice = threadIdx.x / kPieces;
  int u = 0;
  while ((u + 1) * (u + 2) / 2 <= piece) ++u;
  const int t = piece - u * (u + 1) / 2;
  float acc[8][8] = {};
  for (int range = first; range < last; ++range) {
    __syncthreads();
    load_columns<kSide, kKind>(s, b, range * kC, xs);
    __syncthreads();
    if (slice < kSlices) {
      for (int k = slice * 4; k < kC; k += kSlices * 4) {
        float4 x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = *reinterpret_cast<const float4*>(xs + (t + kT * i) * kP + k);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float4 y = *reinterpret_cast<const float4*>(xs + (u + kT * j) * kP + k);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            acc[i][j] = fmaf(x[i].x, y.x, acc[i][j]);
            acc[i][j] = fmaf(x[i].y, y.y, acc[i][j]);
            acc[i][j] = fmaf(x[i].z, y.z, acc[i][j]);
            acc[i][j] = fmaf(x[i].w, y.w, acc[i][j]);
          }
        }
      }
    }
  }
  // the slices' sums, in slice order, eight values of each piece at a time
  float* out = s.partial + (b * s.chunks + blockIdx.x) * kSide * kSide;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    __syncthreads();
    if (slice < kSlices) {
#pragma unroll
      for (int j = 0; j < 8; ++j) xs[(slice * kPieces + piece) * 9 + j] = acc[i][j];
    }
    __syncthreads();
    for (int e = threadIdx.x; e < kPieces * 8; e += kThreads) {
      const int p = e >> 3, j = e & 7;
      float v = 0.0f;
      for (int k = 0; k < kSlices; ++k) v += xs[(k * kPieces + p) * 9 + j];
      int pu = 0;
      while ((pu + 1) * (pu + 2) / 2 <= p) ++pu;
      const int row = p - pu * (pu + 1) / 2 + kT * i, col = pu + kT * j;
      out[row * kSide + col] = v;
      out[col * kSide + row] = v;
    }
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

// out = Q X for kCols columns. A warp takes 8 rows of 128 columns, 4 columns a lane: Q is read by the whole
// warp at once, X once for 8 rows.
template <int kSide, int kKind>
__global__ void __launch_bounds__(kThreads, 3) small_apply_kernel(const Small s) {
  constexpr int kC = kCols<kSide>, kP = kPitch<kSide>;
  extern __shared__ __align__(16) float xs[];
  float* q = xs + kSide * kP;  // Q^T, dense
  const int64_t b = blockIdx.y;
  const int c0 = blockIdx.x * kC;
  load_columns<kSide, kKind>(s, b, c0, xs);
  for (int e = threadIdx.x; e < kSide * kSide; e += kThreads) q[e] = s.q[b * kSide * kSide + e];
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int i0 = warp % (kSide / 8) * 8, j0 = warp / (kSide / 8) * 128 + lane * 4;
  float acc[8][4] = {};
#pragma unroll 8
  for (int k = 0; k < kSide; ++k) {
    const float4 x = *reinterpret_cast<const float4*>(xs + k * kP + j0);
    const float4 lo = *reinterpret_cast<const float4*>(q + k * kSide + i0);
    const float4 hi = *reinterpret_cast<const float4*>(q + k * kSide + i0 + 4);
    const float w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      acc[i][0] = fmaf(w[i], x.x, acc[i][0]);
      acc[i][1] = fmaf(w[i], x.y, acc[i][1]);
      acc[i][2] = fmaf(w[i], x.z, acc[i][2]);
      acc[i][3] = fmaf(w[i], x.w, acc[i][3]);
    }
  }
  __nv_bfloat16* out = s.out + b * s.r * s.c;
  const int col0 = c0 + j0;
  if (!s.tall) {
    const bool whole = s.out_wide && col0 + 4 <= s.c;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i0 + i >= s.r) break;
      __nv_bfloat16* dst = out + static_cast<int64_t>(i0 + i) * s.c + col0;
      if (whole) {
        const __nv_bfloat162 p0 = __floats2bfloat162_rn(acc[i][0], acc[i][1]);
        const __nv_bfloat162 p1 = __floats2bfloat162_rn(acc[i][2], acc[i][3]);
        *reinterpret_cast<uint2*>(dst) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&p0), *reinterpret_cast<const uint32_t*>(&p1));
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (col0 + j < s.c) dst[j] = __float2bfloat16_rn(acc[i][j]);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (col0 + j >= s.c) break;
      __nv_bfloat16* dst = out + static_cast<int64_t>(col0 + j) * s.r + i0;
      if (s.out_wide && i0 + 8 <= s.r) {
        uint32_t p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const __nv_bfloat162 h = __floats2bfloat162_rn(acc[2 * i][j], acc[2 * i + 1][j]);
          p[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        *reinterpret_cast<uint4*>(dst) = make_uint4(p[0], p[1], p[2], p[3]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i0 + i < s.r) dst[i] = __float2bfloat16_rn(acc[i][j]);
      }
    }
  }
}

template <int kSide, int kKind>
int launch_typed(const Small& s, cudaStream_t stream) {
  constexpr int kIterateBytes = 4 * kSide * (kSide + 4) * 4;
  constexpr int kTileBytes = kSide * kPitch<kSide> * 4;
  constexpr int kApplyBytes = kTileBytes + kSide * kSide * 4;
  static_assert(kThreads * 9 * 4 <= kTileBytes, "the slices' sums fit the tile");
  static std::once_flag once;
  static cudaError_t attr_err = cudaSuccess;
  std::call_once(once, [] {
    attr_err = cudaFuncSetAttribute(small_iterate_kernel<kSide>, cudaFuncAttributeMaxDynamicSharedMemorySize, kIterateBytes);
    if (attr_err == cudaSuccess)
      attr_err = cudaFuncSetAttribute(small_apply_kernel<kSide, kKind>, cudaFuncAttributeMaxDynamicSharedMemorySize, kApplyBytes);
  });
  MOSS_CUDA_TRY(attr_err);
  const unsigned batch = static_cast<unsigned>(s.batch);
  small_gram_kernel<kSide, kKind><<<dim3(s.chunks, batch), kThreads, kTileBytes, stream>>>(s);
  MOSS_CUDA_TRY(cudaGetLastError());
  small_iterate_kernel<kSide><<<batch, kThreads, kIterateBytes, stream>>>(s);
  MOSS_CUDA_TRY(cudaGetLastError());
  small_apply_kernel<kSide, kKind><<<dim3((s.c + kCols<kSide> - 1) / kCols<kSide>, batch), kThreads, kApplyBytes, stream>>>(s);
  return check_cuda(cudaGetLastError(), "small_apply_kernel");
}
template <int kSide>
int launch_side(const Small& s, cudaStream_t stream) {
  if (s.dtype == kBF16) return launch_typed<kSide, kBF16>(s, stream);
  if (s.dtype == kF16) return launch_typed<kSide, kF16>(s, stream);
  return launch_typed<kSide, kF32>(s, stream);
}

}  // namespace

int small_side(int r) { return r <= 16 ? 16 : r <= 32 ? 32 : 64; }

// Column ranges per matrix: enough CTAs for the GPU (two a multiprocessor), no more than there are tiles.
int small_chunks(int64_t batch, int r, int c, int sms) {
  const int cols = 8192 / small_side(r);
  const int64_t ranges = (c + cols - 1) / cols;
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(ranges, 4LL * sms / std::max<int64_t>(1, batch))));
}

int launch_small(const Small& s, cudaStream_t stream) {
  switch (small_side(s.r)) {
    case 16: return launch_side<16>(s, stream);
    case 32: return launch_side<32>(s, stream);
    default: return launch_side<64>(s, stream);
  }
}

}  // namespace ns
}  // namespace moss
