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
// Columns of X in shared memory at a time: 16 KB of f32 (Gram) or 32 KB (apply). Rows lie 16 bytes past a
// multiple of 128 apart, so that 16-byte reads of neighbouring rows meet in different banks.
template <int kSide>
constexpr int kGramCols = 4096 / kSide;
template <int kSide>
constexpr int kApplyCols = 8192 / kSide;

template <int kKind>
struct Raw4 {  // four neighbouring values of G as they are stored
  uint32_t w[kKind == kF32 ? 4 : 2];
};
template <int kKind>
__device__ __forceinline__ Raw4<kKind> load_raw4(const Small& s, int64_t at, int left) {
  Raw4<kKind> r{};
  if (left <= 0) return r;
  if (s.wide) {
    if constexpr (kKind == kF32) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(static_cast<const float*>(s.g) + at));
      r.w[0] = v.x;
      r.w[1] = v.y;
      r.w[2] = v.z;
      r.w[3] = v.w;
    } else {
      const uint2 v = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(s.g) + at));
      r.w[0] = v.x;
      r.w[1] = v.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i >= left) break;
      if constexpr (kKind == kF32)
        r.w[i] = __ldg(static_cast<const uint32_t*>(s.g) + at + i);
      else
        r.w[i / 2] |= static_cast<uint32_t>(__ldg(static_cast<const uint16_t*>(s.g) + at + i)) << (16 * (i & 1));
    }
  }
  return r;
}
template <int kKind>
__device__ __forceinline__ float4 to_float4(const Raw4<kKind>& r) {
  if constexpr (kKind == kF32) {
    return make_float4(__uint_as_float(r.w[0]), __uint_as_float(r.w[1]), __uint_as_float(r.w[2]), __uint_as_float(r.w[3]));
  } else if constexpr (kKind == kBF16) {
    return make_float4(__uint_as_float(r.w[0] << 16), __uint_as_float(r.w[0] & 0xffff0000u), __uint_as_float(r.w[1] << 16),
                       __uint_as_float(r.w[1] & 0xffff0000u));
  } else {
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&r.w[0]));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&r.w[1]));
    return make_float4(a.x, a.y, b.x, b.y);
  }
}

// kC columns of X from column c0 on their way to shared memory: fetch() starts the loads (zero past r and c),
// put() writes xs[row][column]. Between the two the CTA works on the tile before.
template <int kSide, int kC, int kKind>
struct Tile {
  static constexpr int kPitch = kC + 4;
  static constexpr int kLoads = kSide * kC / 4 / kThreads;
  Raw4<kKind> raw[kLoads];
  __device__ __forceinline__ void fetch(const Small& s, int64_t b, int c0) {
    const int64_t base = b * s.r * s.c;
#pragma unroll
    for (int l = 0; l < kLoads; ++l) {
      const int i = threadIdx.x + l * kThreads;
      if (!s.tall) {
        const int row = i / (kC / 4), col = c0 + i % (kC / 4) * 4;
        raw[l] = load_raw4<kKind>(s, base + static_cast<int64_t>(row) * s.c + col, row < s.r ? s.c - col : 0);
      } else {  // G [c][r]: four values of a row of G are four rows of one column of X
        const int col = c0 + i % kC, row = i / kC * 4;
        raw[l] = load_raw4<kKind>(s, base + static_cast<int64_t>(col) * s.r + row, col < s.c ? s.r - row : 0);
      }
    }
  }
  __device__ __forceinline__ void put(bool tall, float* xs) const {
#pragma unroll
    for (int l = 0; l < kLoads; ++l) {
      const int i = threadIdx.x + l * kThreads;
      const float4 v = to_float4<kKind>(raw[l]);
      if (!tall) {
        *reinterpret_cast<float4*>(xs + i / (kC / 4) * kPitch + i % (kC / 4) * 4) = v;
      } else {
        float* to = xs + i / kC * 4 * kPitch + i % kC;
        to[0] = v.x;
        to[kPitch] = v.y;
        to[2 * kPitch] = v.z;
        to[3 * kPitch] = v.w;
      }
    }
  }
};

// Partial X X^T over this CTA's column range, upper half. With T = side / 8, piece (t, u), t <= u, is the
// 8 x 8 products of rows t, t + T, .. with rows u, u + T, ..; a thread sums one piece over every kSlices-th
// group of four columns. 64 multiply-adds for 16 values read is what keeps shared memory from
// being the bound (4 x 4 pieces took 53 us for 144 x 32 x 3072).
template <int kSide, int kKind>
__global__ void __launch_bounds__(kThreads, 2) small_gram_kernel(const Small s) {
  constexpr int kT = kSide / 8;
  constexpr int kPieces = kT * (kT + 1) / 2;
  constexpr int kSlices = kThreads / kPieces;
  constexpr int kC = kGramCols<kSide>;
  using T = Tile<kSide, kC, kKind>;
  constexpr int kP = T::kPitch;
  __shared__ __align__(16) float xs[kSide * kP > kThreads * 9 ? kSide * kP : kThreads * 9];
  const int64_t b = blockIdx.y;
  const int ranges = (s.c + kC - 1) / kC;
  const int first = static_cast<int>(static_cast<int64_t>(blockIdx.x) * ranges / s.chunks);
  const int last = static_cast<int>(static_cast<int64_t>(blockIdx.x + 1) * ranges / s.chunks);
  const int piece = threadIdx.x % kPieces, slice = threadIdx.x / kPieces;
  int u = 0;
  while ((u + 1) * (u + 2) / 2 <= piece) ++u;
  const int t = piece - u * (u + 1) / 2;
  float acc[8][8] = {};
  T next;
  if (first < last) next.fetch(s, b, first * kC);
  for (int range = first; range < last; ++range) {
    __syncthreads();
    next.put(s.tall, xs);
    __syncthreads();
    if (range + 1 < last) next.fetch(s, b, (range + 1) * kC);
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
  pdl_trigger();
}

// z = x^T y for a 4 x 4 piece, kSide x kSide in shared memory (x^T = x for the symmetric P).
template <int kSide>
__device__ __forceinline__ void multiply(const float (*x)[kSide + 4], const float (*y)[kSide + 4], int i0, int j0,
                                         float (&z)[4][4]) {
#pragma unroll
  for (int e = 0; e < 16; ++e) z[e / 4][e % 4] = 0.0f;
#pragma unroll 8
  for (int k = 0; k < kSide; ++k) {
    const float4 u = *reinterpret_cast<const float4*>(&x[k][i0]);
    const float4 v = *reinterpret_cast<const float4*>(&y[k][j0]);
    const float p[4] = {u.x, u.y, u.z, u.w}, q[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) z[i][j] = fmaf(p[i], q[j], z[i][j]);
  }
}

// The iteration of one matrix. Half of the threads carry R (three products a step, one after another), the
// other half Q, whose product only needs the step's P.
template <int kSide>
constexpr int kIterateThreads = 2 * (kSide / 4) * (kSide / 4);

template <int kSide>
__global__ void __launch_bounds__(kIterateThreads<kSide>) small_iterate_kernel(const Small s) {
  constexpr int kPieces = (kSide / 4) * (kSide / 4);
  using Row = float[kSide + 4];
  extern __shared__ __align__(16) float smem[];
  Row* R = reinterpret_cast<Row*>(smem);
  Row* P = R + kSide;
  Row* Q = P + kSide;
  Row* T = Q + kSide;
  const int64_t b = blockIdx.x;
  const bool carries_r = threadIdx.x < kPieces;
  const int piece = threadIdx.x % kPieces;
  const int i0 = piece / (kSide / 4) * 4, j0 = piece % (kSide / 4) * 4;
  pdl_wait();
  pdl_trigger();
  const float* partial = s.partial + b * s.chunks * kSide * kSide;
  for (int e = threadIdx.x * 4; e < kSide * kSide; e += kIterateThreads<kSide> * 4) {
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int k = 0; k < s.chunks; ++k) {
      const float4 w = *reinterpret_cast<const float4*>(partial + static_cast<int64_t>(k) * kSide * kSide + e);
      v.x += w.x;
      v.y += w.y;
      v.z += w.z;
      v.w += w.w;
    }
    *reinterpret_cast<float4*>(&R[e / kSide][e % kSide]) = v;
  }
  __syncthreads();
  float trace = 0.0f;
  for (int i = 0; i < s.r; ++i) trace += R[i][i];
  const float norm = sqrtf(trace);
  const float inv = 1.0f / (norm < s.eps ? s.eps : norm);  // NaN stays NaN: every entry then is
  __syncthreads();
  float z[4][4];
  auto put = [&](Row* to, bool transposed) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<float4*>(&to[(transposed ? j0 : i0) + i][transposed ? i0 : j0]) =
          transposed ? make_float4(z[0][i], z[1][i], z[2][i], z[3][i]) : make_float4(z[i][0], z[i][1], z[i][2], z[i][3]);
  };
  if (carries_r) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) R[i0 + i][j0 + j] = R[i0 + i][j0 + j] * inv * inv;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) Q[i0 + i][j0 + j] = i0 + i == j0 + j ? inv : 0.0f;
  }
  for (int step = 0; step < s.steps; ++step) {
    const float ca = s.coefficients[3 * step], cb = s.coefficients[3 * step + 1], cc = s.coefficients[3 * step + 2];
    const bool last = step + 1 == s.steps;
    __syncthreads();
    if (carries_r) {
      multiply<kSide>(R, R, i0, j0, z);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          z[i][j] = (i0 + i == j0 + j ? ca : 0.0f) + cb * R[i0 + i][j0 + j] + cc * z[i][j];
      put(P, false);
    }
    __syncthreads();
    if (!carries_r) {
      multiply<kSide>(P, Q, i0, j0, z);
    } else if (!last) {
      // (P R) P in this order: R P P is the same only without rounding, and its error would not shrink
      // with R's small eigenvalues
      multiply<kSide>(P, R, i0, j0, z);
      put(T, true);
    }
    __syncthreads();
    if (!carries_r) {
      put(Q, false);
    } else if (!last) {
      multiply<kSide>(T, P, i0, j0, z);
      put(R, false);
    }
  }
  __syncthreads();
  float* q = s.q + b * kSide * kSide;  // Q^T
  for (int e = threadIdx.x; e < kSide * kSide; e += kIterateThreads<kSide>) q[e] = Q[e % kSide][e / kSide];
}

// out = Q X over this CTA's column range. A warp takes 8 rows of 128 columns, 4 columns a lane: Q is read by
// the whole warp at once, X once for 8 rows.
template <int kSide, int kKind>
__global__ void __launch_bounds__(kThreads, 2) small_apply_kernel(const Small s) {
  constexpr int kC = kApplyCols<kSide>;
  using T = Tile<kSide, kC, kKind>;
  constexpr int kP = T::kPitch;
  extern __shared__ __align__(16) float xs[];
  float* q = xs + kSide * kP;  // Q^T, dense
  const int64_t b = blockIdx.y;
  const int ranges = (s.c + kC - 1) / kC;
  const int first = static_cast<int>(static_cast<int64_t>(blockIdx.x) * ranges / gridDim.x);
  const int last = static_cast<int>(static_cast<int64_t>(blockIdx.x + 1) * ranges / gridDim.x);
  T next;
  if (first < last) next.fetch(s, b, first * kC);  // G is the caller's: no kernel of this call writes it
  pdl_wait();
  for (int e = threadIdx.x; e < kSide * kSide; e += kThreads) q[e] = s.q[b * kSide * kSide + e];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int i0 = warp % (kSide / 8) * 8, j0 = warp / (kSide / 8) * 128 + lane * 4;
  for (int range = first; range < last; ++range) {
  __syncthreads();
  next.put(s.tall, xs);
  __syncthreads();
  if (range + 1 < last) next.fetch(s, b, (range + 1) * kC);
  const int c0 = range * kC;
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
}

template <int kSide, int kKind>
int launch_typed(const Small& s, cudaStream_t stream) {
  constexpr int kIterateBytes = 4 * kSide * (kSide + 4) * 4;
  constexpr int kApplyBytes = kSide * Tile<kSide, kApplyCols<kSide>, kKind>::kPitch * 4 + kSide * kSide * 4;
  static std::once_flag once;
  static cudaError_t attr_err = cudaSuccess;
  std::call_once(once, [] {
    attr_err = cudaFuncSetAttribute(small_iterate_kernel<kSide>, cudaFuncAttributeMaxDynamicSharedMemorySize, kIterateBytes);
    if (attr_err == cudaSuccess)
      attr_err = cudaFuncSetAttribute(small_apply_kernel<kSide, kKind>, cudaFuncAttributeMaxDynamicSharedMemorySize, kApplyBytes);
  });
  MOSS_CUDA_TRY(attr_err);
  const unsigned batch = static_cast<unsigned>(s.batch);
  small_gram_kernel<kSide, kKind><<<dim3(s.chunks, batch), kThreads, 0, stream>>>(s);
  MOSS_CUDA_TRY(cudaGetLastError());
  const int rc = launch_dependent("small_iterate_kernel", small_iterate_kernel<kSide>, dim3(batch),
                                  dim3(kIterateThreads<kSide>), kIterateBytes, stream, s);
  if (rc != MOSS_OK) return rc;
  const int tiles = (s.c + kApplyCols<kSide> - 1) / kApplyCols<kSide>;
  return launch_dependent("small_apply_kernel", small_apply_kernel<kSide, kKind>, dim3(std::min(tiles, s.chunks), batch),
                          dim3(kThreads), kApplyBytes, stream, s);
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
  const int cols = 4096 / small_side(r);
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
