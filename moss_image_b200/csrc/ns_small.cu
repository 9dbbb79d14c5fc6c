// Orthogonalised update of matrices with a short side of at most 64 (adapter factors).
//
// With R = X X^T, a step X <- (a I + b R + c R R) X =: P X turns R into P R P, so the whole iteration
// stays on the r x r square: Q <- P Q, R <- P R P, and the result is Q X. X is read twice (once
// for R, whose trace is the squared Frobenius norm, once for Q X) however many steps there are,
// instead of three times a step. R's small eigenvalues, which grow by a^2 a step, need f32's
// precision: the iteration is f32, and the two products with X run on the tensor cores
// (mma.sync m16n8k16) with each f32 operand as the sum of two float16 numbers, scaled by powers of two,
// hi hi + hi lo + lo hi with f32 sums. What that leaves out is 2^-22 of a product. (tcgen05's 128-row
// tiles would be three quarters empty here, and these kernels are bound by HBM and latency.)
//
// Three launches: partial R over column ranges, the iteration (one CTA per matrix), Q X. 144 x 32 x 3072 f32:
// 54 us, of which the first takes 19 (57 MB), the second 11 and the third 20; all three are bound by latency,
// at two CTAs a multiprocessor with one tile in registers while another is worked on.
#include <algorithm>

#include "ns_args.cuh"

namespace moss {
namespace ns {
namespace {

constexpr int kThreads = 256;
// Columns of X in shared memory at a time: 8192 values, as two float16 tiles whose rows lie 16 bytes past a
// multiple of 128 apart, so that the eight rows of an ldmatrix meet in different banks.
template <int kSide>
constexpr int kCols = 8192 / kSide;
template <int kSide>
constexpr int kPitch = kCols<kSide> + 8;
template <int kSide>
constexpr int kTileHalves = kSide * kPitch<kSide>;  // of one of the two tiles

template <int kKind>
struct Raw4 {  // four neighbouring values of G as they are stored
  uint32_t w[kKind == kF32 ? 4 : 2];
};
template <int kKind>
__device__ __forceinline__ Raw4<kKind> load_whole4(const void* g, int64_t at) {
  Raw4<kKind> r;
  if constexpr (kKind == kF32) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(static_cast<const float*>(g) + at));
    r.w[0] = v.x;
    r.w[1] = v.y;
    r.w[2] = v.z;
    r.w[3] = v.w;
  } else {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(g) + at));
    r.w[0] = v.x;
    r.w[1] = v.y;
  }
  return r;
}
template <int kKind>
__device__ __forceinline__ Raw4<kKind> load_raw4(const Small& s, int64_t at, int left) {
  Raw4<kKind> r{};
  if (left <= 0) return r;
  if (s.wide) {
    r = load_whole4<kKind>(s.g, at);
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

// p with v in [2^(p + 10), 2^(p + 11)): v 2^-p is about 1024. At most 117, and not below -127, where 2^-p is still
// normal: what is smaller, f32's subnormals included, is then below 2 and on a grid of 2^-22, which float16 holds.
constexpr int kLeastScale = -127;
__device__ __forceinline__ int scale_of(float v) {
  return min(117, max(kLeastScale, static_cast<int>((__float_as_uint(v) >> 23) & 0xffu) - 127 - 10));
}
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(a, b);
  const float2 back = __half22float2(h);
  const __half2 l = __floats2half2_rn(a - back.x, b - back.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}

// kCols columns of X from column c0 on their way to shared memory: fetch() starts the loads (zero past r and
// c), put() writes xs[row][column] as hi + lo. Between the two the CTA works on the tile before.
template <int kSide, int kKind>
struct Tile {
  static constexpr int kC = kCols<kSide>;
  static constexpr int kLoads = kSide * kC / 4 / kThreads;
  Raw4<kKind> raw[kLoads];
  __device__ __forceinline__ void fetch(const Small& s, int64_t b, int c0) {
    const int64_t base = b * s.r * s.c;
    if (s.wide && s.r == kSide && c0 + kC <= s.c) {  // a whole tile: one address, constant steps
      if (!s.tall) {
        const int64_t at = base + static_cast<int64_t>(threadIdx.x / (kC / 4)) * s.c + c0 + threadIdx.x % (kC / 4) * 4;
        const int64_t step = static_cast<int64_t>(kThreads / (kC / 4)) * s.c;
#pragma unroll
        for (int l = 0; l < kLoads; ++l) raw[l] = load_whole4<kKind>(s.g, at + l * step);
      } else {
        constexpr int kSweeps = kC > kThreads ? kC / kThreads : 1;  // of the CTA over a group of four rows
        const int col = threadIdx.x % kC, row = threadIdx.x / kC * 4;
        const int64_t at = base + static_cast<int64_t>(c0 + col) * kSide + row;
#pragma unroll
        for (int l = 0; l < kLoads; ++l)
          raw[l] = load_whole4<kKind>(s.g, at + (l % kSweeps) * kThreads * kSide +
                                               l / kSweeps * (kC < kThreads ? 4 * (kThreads / kC) : 4));
      }
      return;
    }
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
  __device__ __forceinline__ float amax() const {
    float m = 0.0f;
#pragma unroll
    for (int l = 0; l < kLoads; ++l) {
      const float4 v = to_float4<kKind>(raw[l]);
      m = max_nan(m, max_nan(max_nan(fabsf(v.x), fabsf(v.y)), max_nan(fabsf(v.z), fabsf(v.w))));
    }
    return m;
  }
  __device__ __forceinline__ void put(bool tall, float scale, __half* hi, __half* lo) const {
    constexpr int kP = kPitch<kSide>;
#pragma unroll
    for (int l = 0; l < kLoads; ++l) {
      const int i = threadIdx.x + l * kThreads;
      const float4 v = to_float4<kKind>(raw[l]);
      uint2 h, q;
      split2(v.x * scale, v.y * scale, h.x, q.x);
      split2(v.z * scale, v.w * scale, h.y, q.y);
      if (!tall) {
        const int at = i / (kC / 4) * kP + i % (kC / 4) * 4;
        *reinterpret_cast<uint2*>(hi + at) = h;
        *reinterpret_cast<uint2*>(lo + at) = q;
      } else {
        const int at = i / kC * 4 * kP + i % kC;
        const __half2 h0 = *reinterpret_cast<const __half2*>(&h.x), h1 = *reinterpret_cast<const __half2*>(&h.y);
        const __half2 q0 = *reinterpret_cast<const __half2*>(&q.x), q1 = *reinterpret_cast<const __half2*>(&q.y);
        hi[at] = __low2half(h0);
        hi[at + kP] = __high2half(h0);
        hi[at + 2 * kP] = __low2half(h1);
        hi[at + 3 * kP] = __high2half(h1);
        lo[at] = __low2half(q0);
        lo[at + kP] = __high2half(q0);
        lo[at + 2 * kP] = __low2half(q1);
        lo[at + 3 * kP] = __high2half(q1);
      }
    }
  }
};

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Lane addresses within a 16 x 16 block of halves at (row, column) of a tile. A operand and, by .trans, a B
// operand that lies [reduction][column]: rows by lane % 16, column halves by lane / 16.
__device__ __forceinline__ uint32_t block_rows(uint32_t tile, int pitch, int row, int col, int lane) {
  return tile + 2 * ((row + (lane & 15)) * pitch + col + (lane >> 4) * 8);
}
// A B operand that lies [column][reduction]: two 8-column tiles, each two 8-wide reduction halves.
__device__ __forceinline__ uint32_t block_columns(uint32_t tile, int pitch, int row, int col, int lane) {
  return tile + 2 * ((row + (lane >> 4) * 8 + (lane & 7)) * pitch + col + ((lane >> 3) & 1) * 8);
}

// Partial X X^T over this CTA's column range: hi hi^T + hi lo^T + (hi lo^T)^T. A warp holds one block of at
// most 32 x 32 of both products, over every kSplits-th 16 columns. X is scaled by the largest value met so
// far; when a tile brings a larger one, the sums are scaled down with it (powers of two, exact). They leave
// scaled, with their exponent beside them: the squares of f32's values have twice its range.
template <int kSide, int kKind>
__global__ void __launch_bounds__(kThreads, 2) small_gram_kernel(const Small s) {
  constexpr int kC = kCols<kSide>, kP = kPitch<kSide>;
  constexpr int kBlk = kSide < 32 ? kSide : 32;
  constexpr int kBlocks = kSide / kBlk;  // per side
  constexpr int kSplits = kThreads / 32 / (kBlocks * kBlocks);
  constexpr int kMT = kBlk / 16, kNT = kBlk / 8;
  __shared__ __align__(16) __half tiles[2 * kTileHalves<kSide>];
  __shared__ float warp_max[kThreads / 32];
  static_assert(sizeof(tiles) >= kSplits * kSide * (kSide + 1) * 4, "the joined sums fit the tiles");
  const int64_t b = blockIdx.y;
  const int ranges = (s.c + kC - 1) / kC;
  const int first = static_cast<int>(static_cast<int64_t>(blockIdx.x) * ranges / s.chunks);
  const int last = static_cast<int>(static_cast<int64_t>(blockIdx.x + 1) * ranges / s.chunks);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = warp % kSplits, block = warp / kSplits;
  const int i0 = block / kBlocks * kBlk, j0 = block % kBlocks * kBlk;
  __half* hi = tiles;
  __half* lo = tiles + kTileHalves<kSide>;
  const uint32_t hi_addr = smem_u32(hi), lo_addr = smem_u32(lo);
  float hh[kMT][kNT][4] = {}, hl[kMT][kNT][4] = {};
  int p = kLeastScale;  // X is held times 2^-p
  Tile<kSide, kKind> next;
  if (first < last) next.fetch(s, b, first * kC);
  for (int range = first; range < last; ++range) {
    float amax = next.amax();
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, d));
    if (lane == 0) warp_max[warp] = amax;
    __syncthreads();  // the maxima are there, and the tiles free
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) amax = max_nan(amax, warp_max[w]);
    const int q = scale_of(amax);
    if (q > p) {
      const float down = pow2(max(-126, 2 * (p - q)));
#pragma unroll
      for (int i = 0; i < kMT; ++i)
#pragma unroll
        for (int j = 0; j < kNT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            hh[i][j][e] *= down;
            hl[i][j][e] *= down;
          }
      p = q;
    }
    next.put(s.tall, pow2(-p), hi, lo);
    __syncthreads();
    if (range + 1 < last) next.fetch(s, b, (range + 1) * kC);
#pragma unroll
    for (int k = split * 16; k < kC; k += kSplits * 16) {
      uint32_t a[kMT][4];
#pragma unroll
      for (int i = 0; i < kMT; ++i) ldmatrix4(block_rows(hi_addr, kP, i0 + i * 16, k, lane), a[i]);
#pragma unroll
      for (int j = 0; j < kNT / 2; ++j) {
        uint32_t bh[4], bl[4];
        ldmatrix4(block_columns(hi_addr, kP, j0 + j * 16, k, lane), bh);
        ldmatrix4(block_columns(lo_addr, kP, j0 + j * 16, k, lane), bl);
#pragma unroll
        for (int i = 0; i < kMT; ++i) {
          mma16816(hh[i][2 * j], a[i], bh[0], bh[1]);
          mma16816(hh[i][2 * j + 1], a[i], bh[2], bh[3]);
          mma16816(hl[i][2 * j], a[i], bl[0], bl[1]);
          mma16816(hl[i][2 * j + 1], a[i], bl[2], bl[3]);
        }
      }
    }
  }
  // The warps' sums, always in the same order: the first half of the splits each to a region of its own, the
  // second half on top of them, then the regions.
  constexpr int kRegions = kSplits / 2;
  using Row = float[kSide + 1];
  Row* regions = reinterpret_cast<Row*>(tiles);  // [region][hh, hl][kSide]
  Row* sum = regions + split % kRegions * 2 * kSide;
  Row* cross = sum + kSide;
#pragma unroll
  for (int turn = 0; turn < 2; ++turn) {
    __syncthreads();
    if (split / kRegions != turn) continue;
#pragma unroll
    for (int i = 0; i < kMT; ++i)
#pragma unroll
      for (int j = 0; j < kNT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = i0 + i * 16 + (lane >> 2) + (e >> 1) * 8, col = j0 + j * 8 + (lane & 3) * 2 + (e & 1);
          sum[row][col] = (turn > 0 ? sum[row][col] : 0.0f) + hh[i][j][e];
          cross[row][col] = (turn > 0 ? cross[row][col] : 0.0f) + hl[i][j][e];
        }
  }
  __syncthreads();
  float* out = s.partial + (b * s.chunks + blockIdx.x) * kSide * kSide;
  if (threadIdx.x == 0) s.exponents[b * s.chunks + blockIdx.x] = p;
  for (int e = threadIdx.x; e < kSide * kSide; e += kThreads) {
    const int row = e / kSide, col = e % kSide;
    float same = 0.0f, across = 0.0f;
#pragma unroll
    for (int k = 0; k < kRegions; ++k) {
      const Row* part = regions + k * 2 * kSide;
      same += part[row][col];
      across += part[kSide + row][col] + part[kSide + col][row];
    }
    out[e] = same + across;
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
  // X, R and the norm are held in units of 2^xp of the matrix's largest value from here on. The exponents come with
  // the sums: a pass over them before would be one more wait for L2.
  const int* exponents = s.exponents + b * s.chunks;
  int xp = kLeastScale;
  for (int e = threadIdx.x * 4; e < kSide * kSide; e += kIterateThreads<kSide> * 4) {
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    xp = kLeastScale;
#pragma unroll 4
    for (int k = 0; k < s.chunks; ++k) {
      const float4 w = *reinterpret_cast<const float4*>(partial + static_cast<int64_t>(k) * kSide * kSide + e);
      const int p = exponents[k], top = max(xp, p);
      const float mine = pow2(max(-126, 2 * (xp - top))), its = pow2(max(-126, 2 * (p - top)));  // one of them is 1
      v.x = fmaf(w.x, its, v.x * mine);
      v.y = fmaf(w.y, its, v.y * mine);
      v.z = fmaf(w.z, its, v.z * mine);
      v.w = fmaf(w.w, its, v.w * mine);
      xp = top;
    }
    *reinterpret_cast<float4*>(&R[e / kSide][e % kSide]) = v;
  }
  __syncthreads();
  float trace = 0.0f;
  for (int i = 0; i < s.r; ++i) trace += R[i][i];
  const float norm = sqrtf(trace);
  // eps in the same units; what passes f32's range (a tiny matrix against an eps above 1) is left for the result
  const int eps_exp = s.eps_exponent - xp;
  const float eps = s.eps_fraction * pow2(min(126, max(-126, eps_exp)));
  const float inv = 1.0f / (norm < eps ? eps : norm);  // NaN stays NaN: every entry then is
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
      for (int j = 0; j < 4; ++j) Q[i0 + i][j0 + j] = i0 + i == j0 + j ? 1.0f : 0.0f;
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
  // Q as hi + lo, times 2^-qp, and what the product with X, times 2^-xp, has to be multiplied by.
  __shared__ float warp_max[kIterateThreads<kSide> / 32];
  float amax = 0.0f;
  for (int e = threadIdx.x; e < kSide * kSide; e += kIterateThreads<kSide>)
    amax = max_nan(amax, fabsf(Q[e / kSide][e % kSide]));
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, d));
  if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = amax;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kIterateThreads<kSide> / 32; ++w) amax = max_nan(amax, warp_max[w]);
  const int qp = max(-126, scale_of(amax));  // its own power of two is normal as well
  const float down = pow2(-qp);
  __half* hi = s.q + b * 2 * kSide * kSide;
  __half* lo = hi + kSide * kSide;
  for (int e = threadIdx.x * 2; e < kSide * kSide; e += kIterateThreads<kSide> * 2) {
    uint32_t h, l;
    split2(Q[e / kSide][e % kSide] * down, Q[e / kSide][e % kSide + 1] * down, h, l);
    *reinterpret_cast<uint32_t*>(hi + e) = h;
    *reinterpret_cast<uint32_t*>(lo + e) = l;
  }
  if (threadIdx.x == 0) {
    s.factors[2 * b] = pow2(-xp);
    s.factors[2 * b + 1] = inv * pow2(qp) * (norm < eps ? pow2(-min(126, max(0, eps_exp - 126))) : 1.0f);
  }
}

// out = Q X over this CTA's column range: hi hi + hi lo + lo hi. A warp takes an eighth of a tile's columns, all rows.
template <int kSide, int kKind>
__global__ void __launch_bounds__(kThreads, 2) small_apply_kernel(const Small s) {
  constexpr int kC = kCols<kSide>, kP = kPitch<kSide>, kQP = kSide + 8;
  constexpr int kMT = kSide / 16, kNT = kC / 64;  // 16-row and 8-column tiles of a warp
  extern __shared__ __align__(16) __half smem_halves[];
  __half* hi = smem_halves;
  __half* lo = hi + kTileHalves<kSide>;
  __half* qh = lo + kTileHalves<kSide>;
  __half* ql = qh + kSide * kQP;
  __nv_bfloat16* staged = reinterpret_cast<__nv_bfloat16*>(smem_halves);  // over the tiles, once they are used
  constexpr int kWidePitch = kC + 8, kTallPitch = kSide + 8;
  static_assert(kC * kTallPitch <= 2 * kTileHalves<kSide>, "the turned outputs fit the tiles");
  const int64_t b = blockIdx.y;
  const int ranges = (s.c + kC - 1) / kC;
  const int first = static_cast<int>(static_cast<int64_t>(blockIdx.x) * ranges / gridDim.x);
  const int last = static_cast<int>(static_cast<int64_t>(blockIdx.x + 1) * ranges / gridDim.x);
  Tile<kSide, kKind> next;
  if (first < last) next.fetch(s, b, first * kC);  // G is the caller's: no kernel of this call writes it
  pdl_wait();
  for (int e = threadIdx.x * 8; e < 2 * kSide * kSide; e += kThreads * 8) {
    const int part = e / (kSide * kSide), at = e % (kSide * kSide);
    *reinterpret_cast<uint4*>((part ? ql : qh) + at / kSide * kQP + at % kSide) =
        *reinterpret_cast<const uint4*>(s.q + b * 2 * kSide * kSide + e);
  }
  const float x_scale = s.factors[2 * b], factor = s.factors[2 * b + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t hi_addr = smem_u32(hi), lo_addr = smem_u32(lo), qh_addr = smem_u32(qh), ql_addr = smem_u32(ql);
  __nv_bfloat16* out = s.out + b * s.r * s.c;
  for (int range = first; range < last; ++range) {
    __syncthreads();
    next.put(s.tall, x_scale, hi, lo);
    __syncthreads();
    if (range + 1 < last) next.fetch(s, b, (range + 1) * kC);
    const int c0 = range * kC;
    float acc[kMT][kNT][4] = {};
#pragma unroll
    for (int k = 0; k < kSide; k += 16) {
      uint32_t ah[kMT][4], al[kMT][4];
#pragma unroll
      for (int i = 0; i < kMT; ++i) {
        ldmatrix4(block_rows(qh_addr, kQP, i * 16, k, lane), ah[i]);
        ldmatrix4(block_rows(ql_addr, kQP, i * 16, k, lane), al[i]);
      }
#pragma unroll
      for (int j = 0; j < kNT / 2; ++j) {
        uint32_t bh[4], bl[4];
        const int col = warp * kNT * 8 + j * 16;
        ldmatrix4_trans(block_rows(hi_addr, kP, k, col, lane), bh);
        ldmatrix4_trans(block_rows(lo_addr, kP, k, col, lane), bl);
#pragma unroll
        for (int i = 0; i < kMT; ++i) {
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            mma16816(acc[i][2 * j + t], al[i], bh[2 * t], bh[2 * t + 1]);
            mma16816(acc[i][2 * j + t], ah[i], bl[2 * t], bl[2 * t + 1]);
            mma16816(acc[i][2 * j + t], ah[i], bh[2 * t], bh[2 * t + 1]);
          }
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kMT; ++i)
#pragma unroll
      for (int j = 0; j < kNT; ++j)
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const int row = i * 16 + (lane >> 2) + (e >> 1) * 8, col = warp * kNT * 8 + j * 8 + (lane & 3) * 2;
          const __nv_bfloat162 v = __floats2bfloat162_rn(acc[i][j][e] * factor, acc[i][j][e + 1] * factor);
          if (!s.tall) {
            *reinterpret_cast<__nv_bfloat162*>(staged + row * kWidePitch + col) = v;
          } else {
            staged[col * kTallPitch + row] = __low2bfloat16(v);
            staged[(col + 1) * kTallPitch + row] = __high2bfloat16(v);
          }
        }
    __syncthreads();
    // whole rows of the result: of kC columns, or (tall) of r values
    const int rows = s.tall ? min(kC, s.c - c0) : s.r, width = s.tall ? s.r : min(kC, s.c - c0);
    const int64_t pitch = s.tall ? s.r : s.c;
    __nv_bfloat16* to = out + (s.tall ? static_cast<int64_t>(c0) * s.r : c0);
    const int from_pitch = s.tall ? kTallPitch : kWidePitch;
    if (s.out_wide) {
      const int per_row = width / 8;
      for (int e = threadIdx.x; e < rows * per_row; e += kThreads) {
        const int row = e / per_row, col = e % per_row * 8;
        *reinterpret_cast<uint4*>(to + row * pitch + col) = *reinterpret_cast<const uint4*>(staged + row * from_pitch + col);
      }
    } else {
      for (int e = threadIdx.x; e < rows * width; e += kThreads) {
        const int row = e / width, col = e % width;
        to[row * pitch + col] = staged[row * from_pitch + col];
      }
    }
  }
}

template <int kSide, int kKind>
int launch_typed(const Small& s, cudaStream_t stream) {
  constexpr int kIterateBytes = 4 * kSide * (kSide + 4) * 4;
  constexpr int kApplyBytes = 2 * (2 * kTileHalves<kSide> + 2 * kSide * (kSide + 8));
  static DeviceSetup setup;
  int rc = setup("small_iterate_kernel", nullptr, [](int*) {
    const cudaError_t e =
        cudaFuncSetAttribute(small_iterate_kernel<kSide>, cudaFuncAttributeMaxDynamicSharedMemorySize, kIterateBytes);
    if (e != cudaSuccess) return e;
    return cudaFuncSetAttribute(small_apply_kernel<kSide, kKind>, cudaFuncAttributeMaxDynamicSharedMemorySize, kApplyBytes);
  });
  if (rc != MOSS_OK) return rc;
  const unsigned batch = static_cast<unsigned>(s.batch);
  small_gram_kernel<kSide, kKind><<<dim3(s.chunks, batch), kThreads, 0, stream>>>(s);
  MOSS_CUDA_TRY(cudaGetLastError());
  rc = launch_dependent("small_iterate_kernel", small_iterate_kernel<kSide>, dim3(batch),
                                  dim3(kIterateThreads<kSide>), kIterateBytes, stream, s);
  if (rc != MOSS_OK) return rc;
  const int tiles = (s.c + kCols<kSide> - 1) / kCols<kSide>;
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

// Column ranges per matrix: one round of the GPU (two CTAs a multiprocessor; two rounds took 25 us for the Gram
// pass of 144 x 32 x 3072 instead of 20), no more than there are tiles.
int small_chunks(int64_t batch, int r, int c, int sms) {
  const int cols = 8192 / small_side(r);
  const int64_t ranges = (c + cols - 1) / cols;
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(ranges, 2LL * sms / std::max<int64_t>(1, batch))));
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
