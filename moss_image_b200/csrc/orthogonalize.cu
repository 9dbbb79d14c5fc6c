// The orthogonalised update (moss_orthogonalize): X = G / max(|G|, eps), then steps of
//   A = X X^T,  X <- a X + (b A + c A A) X,
// an odd polynomial of the singular values that drives them towards 1 (Newton-Schulz). The Gram
// matrix is taken on the shorter side; a tall G is iterated as its transpose.
//
// Precision. The iteration multiplies what is small in X by a (3.4 for the usual coefficients) every
// step, rounding noise included, so 16 bits are not all alike here. Operands are float16: its 11 bits
// cost no more on the tensor cores than bfloat16's 8, and its range is met by powers of two, X times
// about sqrt(c) (entries near 1) and A, B times `gain`. X itself is held as two float16 numbers,
// hi + lo: products read hi, the a X term reads both, so that hi's rounding enters only through
// (b A + c A A), which is small in the directions that still have to grow. lo is dropped for the last steps, two at
// most, whose product of growths (kLateGrowth) leaves hi's rounding below bfloat16's. With the usual coefficients the
// result is within 1.4 times its own rounding to bfloat16 of float64's, momentum with a few directions 80 times
// stronger than the rest included; bfloat16 operands are 5 to 100 times further off. Tested in tests/test_gpu_muon.py.
#include <algorithm>
#include <cmath>
#include <cstring>

#include "ns_args.cuh"

namespace moss {
namespace ns {

int sm_count() { return device_sm_count(); }

constexpr int kThreads = 256;
constexpr int kNormParts = 512;       // at most, per matrix
constexpr int kPartValues = 16384;    // values per part where there are fewer

// Sums of squares over equal ranges of a matrix, in f64 (neither overflow nor a loss in long sums).
template <int kKind>
__global__ void __launch_bounds__(kThreads) sum_squares_kernel(const void* __restrict__ g, int64_t size, bool wide,
                                                               double* __restrict__ parts) {
  const int64_t base = static_cast<int64_t>(blockIdx.y) * size;
  const int64_t chunks = (size + 7) / 8;
  const int64_t first = chunks * blockIdx.x / gridDim.x, last = chunks * (blockIdx.x + 1) / gridDim.x;
  double sum = 0.0;
#pragma unroll 4
  for (int64_t i = first + threadIdx.x; i < last; i += kThreads) {
    float v[8];
    load8<kKind>(g, base + i * 8, size - i * 8, wide, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += static_cast<double>(v[j]) * v[j];
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  __shared__ double warps[kThreads / 32];
  if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kThreads / 32; ++w) sum += warps[w];
    parts[static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x] = sum;
  }
  pdl_trigger();
}

// unit / max(|G|, eps) from the parts, the same in every warp: as the product of a power of two and a factor near unit,
// since the norm of float32 values, or what divides by it, may be past float32. A matrix whose norm is so far below eps
// that the steps only multiply it (by `growth` at most) is held larger by 1 / shift, or float16 would lose it.
struct Scale {
  float power, factor, shift;
};
__device__ __forceinline__ Scale scale_of(const double* parts, int num_parts, float eps, float unit, double growth) {
  double sum = 0.0;
  for (int p = threadIdx.x & 31; p < num_parts; p += 32) sum += parts[p];
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  const double norm = sqrt(sum);
  auto exponent_of = [](double v) { return static_cast<int>((__double2hiint(v) >> 20) & 0x7ff) - 1023; };
  const int held = norm < eps ? min(126, max(0, exponent_of(eps) - exponent_of(norm * growth) - 1)) : 0;
  const float shift = pow2(-held);
  const double divisor = (norm < eps ? eps : norm) * shift;  // NaN stays NaN
  const int exponent = exponent_of(divisor);
  const int p = min(126, max(-126, exponent));
  // an infinity in G makes the norm one: the matrix is NaN
  const float rest = exponent > 1000 ? __int_as_float(0x7fffffff)
                                     : static_cast<float>(divisor * __hiloint2double((1023 - p) << 20, 0));
  return {pow2(-p), unit / rest, shift};
}

__device__ __forceinline__ void split8(const float (&v)[8], Scale scale, uint4& hi, uint4& lo) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = v[2 * i] * scale.power * scale.factor, b = v[2 * i + 1] * scale.power * scale.factor;
    const __half2 p = __floats2half2_rn(a, b);
    const float2 back = __half22float2(p);
    const __half2 q = __floats2half2_rn(a - back.x, b - back.y);
    h[i] = *reinterpret_cast<const uint32_t*>(&p);
    l[i] = *reinterpret_cast<const uint32_t*>(&q);
  }
  hi = make_uint4(h[0], h[1], h[2], h[3]);
  lo = make_uint4(l[0], l[1], l[2], l[3]);
}

// hi + lo = G * unit / max(|G|, eps), its columns padded with zeros to cp. A CTA: kNormRows rows of 512 columns.
constexpr int kNormRows = 16;
template <int kKind>
__global__ void __launch_bounds__(kThreads) normalize_kernel(const void* __restrict__ g, int r, int c, int cp, bool wide,
                                                             const double* __restrict__ parts, int num_parts,
                                                             float eps, float unit, double growth,
                                                             __half* __restrict__ hi, __half* __restrict__ lo,
                                                             float* __restrict__ shifts) {
  pdl_wait();
  const int64_t b = blockIdx.z;
  const Scale scale = scale_of(parts + b * num_parts, num_parts, eps, unit, growth);
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) shifts[b] = scale.shift;
  const int j = blockIdx.x * 512 + (threadIdx.x & 63) * 8;
  const int i0 = blockIdx.y * kNormRows + (threadIdx.x >> 6);
  pdl_trigger();
  if (j >= cp) return;
  float v[kNormRows / 4][8];
#pragma unroll
  for (int k = 0; k < kNormRows / 4; ++k) {
    const int i = i0 + 4 * k;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[k][e] = 0.0f;
    if (i < r && j < c) load8<kKind>(g, (b * r + i) * c + j, c - j, wide, v[k]);
  }
#pragma unroll
  for (int k = 0; k < kNormRows / 4; ++k) {
    uint4 h, l;
    split8(v[k], scale, h, l);
    if (i0 + 4 * k >= r) continue;
    const int64_t at = (b * r + i0 + 4 * k) * cp + j;
    *reinterpret_cast<uint4*>(hi + at) = h;
    *reinterpret_cast<uint4*>(lo + at) = l;
  }
}

// The same for a tall G [c][r]: 64 x 64 tiles turned through shared memory, so that both sides move whole rows.
template <int kKind>
__global__ void __launch_bounds__(kThreads) normalize_tall_kernel(const void* __restrict__ g, int r, int c, int cp, bool wide,
                                                                  const double* __restrict__ parts,
                                                                  int num_parts, float eps, float unit, double growth,
                                                                  __half* __restrict__ hi, __half* __restrict__ lo,
                                                                  float* __restrict__ shifts) {
  __shared__ float tile[64][65];
  pdl_wait();
  const int64_t b = blockIdx.z;
  const Scale scale = scale_of(parts + b * num_parts, num_parts, eps, unit, growth);
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) shifts[b] = scale.shift;
  pdl_trigger();
  const int i0 = blockIdx.y * 64, j0 = blockIdx.x * 64;
  const int e = (threadIdx.x & 7) * 8, w = threadIdx.x >> 3;
#pragma unroll
  for (int k = w; k < 64; k += kThreads / 8) {  // rows of G
    float v[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = 0.0f;
    if (j0 + k < c && i0 + e < r) load8<kKind>(g, (b * c + j0 + k) * r + i0 + e, r - i0 - e, wide, v);
#pragma unroll
    for (int q = 0; q < 8; ++q) tile[e + q][k] = v[q];
  }
  __syncthreads();
#pragma unroll
  for (int k = w; k < 64; k += kThreads / 8) {
    if (i0 + k >= r) continue;
    float v[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = tile[k][e + q];
    uint4 h, l;
    split8(v, scale, h, l);
    const int64_t at = (b * r + i0 + k) * cp + j0 + e;
    *reinterpret_cast<uint4*>(hi + at) = h;
    *reinterpret_cast<uint4*>(lo + at) = l;
  }
}

// Norms and the padded, scaled operands.
template <int kKind>
static int launch_normalize(const void* g, int64_t batch, int r, int c, int cp, bool tall, float eps, float unit,
                            double growth, double* parts, int num_parts, __half* hi, __half* lo, float* shifts,
                            cudaStream_t stream) {
  const int64_t size = static_cast<int64_t>(r) * c;
  const bool aligned = reinterpret_cast<uintptr_t>(g) % 16 == 0;
  const unsigned z = static_cast<unsigned>(batch);
  sum_squares_kernel<kKind><<<dim3(num_parts, z), kThreads, 0, stream>>>(g, size, aligned && size % 8 == 0, parts);
  MOSS_CUDA_TRY(cudaGetLastError());
  const bool wide = aligned && (tall ? r : c) % 8 == 0;
  if (tall)
    return launch_dependent("normalize_tall_kernel", normalize_tall_kernel<kKind>, dim3(cp / 64, (r + 63) / 64, z), dim3(kThreads),
                            0, stream, g, r, c, cp, wide, parts, num_parts, eps, unit, growth, hi, lo, shifts);
  return launch_dependent("normalize_kernel", normalize_kernel<kKind>, dim3((cp + 511) / 512, (r + kNormRows - 1) / kNormRows, z),
                          dim3(kThreads), 0, stream, g, r, c, cp, wide, parts, num_parts, eps, unit, growth, hi, lo, shifts);
}

struct Layout {
  int r, c, sp, cp, side, chunks;
  bool tall, small;
  size_t x[2], low[2], a, b, parts, shifts, partial, exponents, q, factors, total;
};

static Layout layout_of(int64_t batch, int64_t rows, int64_t cols) {
  Layout l{};
  l.tall = rows > cols;
  l.r = static_cast<int>(std::min(rows, cols));
  l.c = static_cast<int>(std::max(rows, cols));
  l.small = l.r <= kSmallSide;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 1023) / 1024 * 1024;
    return here;
  };
  if (l.small) {
    l.side = small_side(l.r);
    l.chunks = small_chunks(batch, l.r, l.c, sm_count());
    const size_t square = static_cast<size_t>(l.side) * l.side * 4 * batch;
    l.partial = take(square * l.chunks);
    l.exponents = take(static_cast<size_t>(batch) * l.chunks * 4);
    l.q = take(square);
    l.factors = take(static_cast<size_t>(batch) * 8);
  } else {
    l.sp = (l.r + 63) / 64 * 64;
    l.cp = (l.c + 127) / 128 * 128;
    const size_t wide = static_cast<size_t>(batch) * l.r * l.cp * 2, square = static_cast<size_t>(batch) * l.r * l.sp * 2;
    for (int i = 0; i < 2; ++i) {
      l.x[i] = take(wide);
      l.low[i] = take(wide);
    }
    l.a = take(square);
    l.b = take(square);
    l.parts = take(static_cast<size_t>(batch) * kNormParts * 8);
    l.shifts = take(static_cast<size_t>(batch) * 4);
  }
  l.total = at;
  return l;
}

// A step p changes a rounding error of X by at most the largest slope |p'| over the singular values. Steps without lo:
// their slopes' product is at most this, which the last two with the usual coefficients reach (4.9 each at the upper end of
// the range; 3.4 at 0).
constexpr double kLateGrowth = 25.0;

// Over s in [0, top]: largest |p(s)| = |s (a + b s^2 + c s^4)|, largest |p'(s)|, and largest |b s^2 + c s^4|.
static void bounds_of(const float* k, double top, double* value, double* slope, double* square) {
  const double a = k[0], b = k[1], c = k[2];
  auto p = [&](double s) { return std::fabs(s * (a + s * s * (b + c * s * s))); };
  auto m = [&](double l) { return std::fabs(l * (b + c * l)); };
  auto d = [&](double l) { return std::fabs(a + l * (3.0 * b + 5.0 * c * l)); };  // l = s^2
  *slope = std::max(d(0.0), d(top * top));
  if (c != 0.0) {
    const double l = -3.0 * b / (10.0 * c);
    if (l > 0.0 && l < top * top) *slope = std::max(*slope, d(l));
  }
  *value = p(top);
  const double disc = 9.0 * b * b - 20.0 * a * c;  // p' = a + 3 b l + 5 c l^2, l = s^2
  if (c != 0.0 && disc >= 0.0) {
    for (const double sign : {-1.0, 1.0}) {
      const double l = (-3.0 * b + sign * std::sqrt(disc)) / (10.0 * c);
      if (l > 0.0 && l < top * top) *value = std::max(*value, p(std::sqrt(l)));
    }
  } else if (c == 0.0 && b != 0.0) {
    const double l = -a / (3.0 * b);
    if (l > 0.0 && l < top * top) *value = std::max(*value, p(std::sqrt(l)));
  }
  *square = m(top * top);
  if (c != 0.0) {
    const double l = -b / (2.0 * c);
    if (l > 0.0 && l < top * top) *square = std::max(*square, m(l));
  }
}

static int check_shape(int64_t batch, int64_t rows, int64_t cols) {
  if (batch < 0 || rows < 0 || cols < 0) return fail(MOSS_ERR_INVALID_ARGUMENT, "negative orthogonalize shape");
  if (batch > 65535) return fail(MOSS_ERR_INVALID_ARGUMENT, "at most 65535 matrices in one call");
  if (rows > (1 << 20) || cols > (1 << 20)) return fail(MOSS_ERR_INVALID_ARGUMENT, "orthogonalize dimension too large");
  if (batch * ((std::min(rows, cols) + 127) / 128 * 128) > INT32_MAX)
    return fail(MOSS_ERR_INVALID_ARGUMENT, "too many rows to orthogonalize in one call");
  return MOSS_OK;
}

static int run(const void* g, int dtype, int64_t batch, int64_t rows, int64_t cols, int steps, const float* coefficients,
               float eps, __nv_bfloat16* out, void* workspace, size_t workspace_bytes, int* status, cudaStream_t stream) {
  if (!is_float_kind(dtype)) return fail(MOSS_ERR_UNSUPPORTED, "unsupported dtype code %d", dtype);
  int rc = check_shape(batch, rows, cols);
  if (rc != MOSS_OK) return rc;
  if (steps < 1 || steps > kMaxSteps || coefficients == nullptr)
    return fail(MOSS_ERR_INVALID_ARGUMENT, "orthogonalize takes 1 to %d steps with three coefficients each", kMaxSteps);
  if (!(eps > 0.0f) || !std::isfinite(eps)) return fail(MOSS_ERR_INVALID_ARGUMENT, "eps must be positive and finite");
  // singular values start in [0, 1]: where each step can take them bounds X, A and B
  double top = 1.001, most = 1.0, widest = 1.0, slopes[kMaxSteps];
  for (int i = 0; i < steps; ++i) {
    const float* k = coefficients + 3 * i;
    if (!std::isfinite(k[0]) || !std::isfinite(k[1]) || !std::isfinite(k[2]))
      return fail(MOSS_ERR_INVALID_ARGUMENT, "the coefficients must be finite");
    double value, square;
    bounds_of(k, top, &value, &slopes[i], &square);
    most = std::max({most, top * top, square});
    widest = std::max(widest, top);
    top = 1.02 * value;
  }
  widest = std::max(widest, top);
  if (!(widest <= 32.0) || !(most <= 4096.0))
    return fail(MOSS_ERR_INVALID_ARGUMENT, "the coefficients let singular values grow past 32");
  if (batch == 0 || rows == 0 || cols == 0) return clear_ok();
  if (g == nullptr || out == nullptr) return fail(MOSS_ERR_INVALID_ARGUMENT, "null matrix pointer");
  const Layout l = layout_of(batch, rows, cols);
  if (workspace == nullptr || workspace_bytes < l.total || reinterpret_cast<uintptr_t>(workspace) % 256 != 0)
    return fail(MOSS_ERR_INVALID_ARGUMENT, "orthogonalize needs %zu bytes of 256-byte aligned workspace", l.total);
  uint8_t* ws = static_cast<uint8_t*>(workspace);

  if (l.small) {
    Small s{};
    s.g = g;
    s.dtype = dtype;
    s.batch = batch;
    s.r = l.r;
    s.c = l.c;
    s.tall = l.tall;
    s.steps = steps;
    const int64_t inner = l.tall ? l.r : l.c;
    s.wide = inner % 4 == 0 && reinterpret_cast<uintptr_t>(g) % 16 == 0;
    s.out_wide = inner % 8 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
    std::memcpy(s.coefficients, coefficients, sizeof(float) * 3 * steps);
    s.eps_fraction = std::frexp(eps, &s.eps_exponent);
    s.out = out;
    s.chunks = l.chunks;
    s.partial = reinterpret_cast<float*>(ws + l.partial);
    s.exponents = reinterpret_cast<int*>(ws + l.exponents);
    s.q = reinterpret_cast<__half*>(ws + l.q);
    s.factors = reinterpret_cast<float*>(ws + l.factors);
    rc = launch_small(s, stream);
    return rc == MOSS_OK ? clear_ok() : rc;
  }

  rc = bind_context();
  if (rc != MOSS_OK) return rc;
  // powers of two: X in units of 1 / unit (entries near 1), A and B in units of 1 / gain (below 2^14)
  const float unit = std::exp2(std::round(0.5 * std::log2(static_cast<double>(l.c))));
  const float gain = std::exp2(std::floor(14.0 - std::log2(most)));
  double growth = 1.0, product = 1.0;  // of what is too small for the steps' squares to matter
  for (int i = 0; i < steps; ++i) growth = std::max(growth, product *= std::fabs(static_cast<double>(coefficients[3 * i])));
  double* parts = reinterpret_cast<double*>(ws + l.parts);
  float* shifts = reinterpret_cast<float*>(ws + l.shifts);
  const int64_t size = rows * cols;
  const int num_parts = static_cast<int>(std::max<int64_t>(
      1, std::min<int64_t>({(size + kPartValues - 1) / kPartValues, kNormParts, 8LL * sm_count() / batch + 1})));
  __half* x[2] = {reinterpret_cast<__half*>(ws + l.x[0]), reinterpret_cast<__half*>(ws + l.x[1])};
  __half* low[2] = {reinterpret_cast<__half*>(ws + l.low[0]), reinterpret_cast<__half*>(ws + l.low[1])};
  __half* ga = reinterpret_cast<__half*>(ws + l.a);
  __half* gb = reinterpret_cast<__half*>(ws + l.b);
  if (dtype == kBF16)
    rc = launch_normalize<kBF16>(g, batch, l.r, l.c, l.cp, l.tall, eps, unit, growth, parts, num_parts, x[0], low[0], shifts,
                                 stream);
  else if (dtype == kF16)
    rc = launch_normalize<kF16>(g, batch, l.r, l.c, l.cp, l.tall, eps, unit, growth, parts, num_parts, x[0], low[0], shifts,
                                 stream);
  else
    rc = launch_normalize<kF32>(g, batch, l.r, l.c, l.cp, l.tall, eps, unit, growth, parts, num_parts, x[0], low[0], shifts,
                                 stream);
  if (rc != MOSS_OK) return rc;
  int with_low = steps;  // steps whose a X term reads lo
  for (double late = 1.0; with_low > std::max(1, steps - 2) && (late *= slopes[with_low - 1]) <= kLateGrowth;) --with_low;
  for (int i = 0; i < steps; ++i) {
    const float* k = coefficients + 3 * i;
    Args a{};
    a.r = l.r;
    a.c = l.c;
    a.sp = l.sp;
    a.cp = l.cp;
    a.batch = static_cast<int>(batch);
    a.tall = l.tall;
    a.shifts = shifts;
    a.status = StatusSink{status, status_mirror_for_current_device()};
    const __half* xi = x[i & 1];
    a.alpha = gain / (unit * unit);
    a.out_hi = ga;
    rc = launch_gemm(kGram, xi, xi, a, stream);
    if (rc != MOSS_OK) return rc;
    a.alpha = k[2] / gain;
    a.beta = k[1];
    a.add_hi = ga;
    a.out_hi = gb;
    rc = launch_gemm(kSquare, ga, ga, a, stream);
    if (rc != MOSS_OK) return rc;
    const bool last = i + 1 == steps;
    const float to_unit = last ? 1.0f / unit : 1.0f;  // exact: a power of two
    a.alpha = to_unit / gain;
    a.beta = k[0] * to_unit;
    a.add_hi = xi;
    a.add_lo = i < with_low ? low[i & 1] : nullptr;
    a.out_hi = x[(i + 1) & 1];
    a.out_lo = i + 1 < with_low ? low[(i + 1) & 1] : nullptr;
    a.result = last ? out : nullptr;
    rc = launch_gemm(kUpdate, gb, xi, a, stream);
    if (rc != MOSS_OK) return rc;
  }
  return clear_ok();
}

}  // namespace ns
}  // namespace moss

using namespace moss;

extern "C" int moss_orthogonalize_workspace_bytes(int64_t batch, int64_t rows, int64_t cols, size_t* bytes) {
  if (bytes == nullptr) return fail(MOSS_ERR_INVALID_ARGUMENT, "null bytes pointer");
  *bytes = 0;
  const int rc = ns::check_shape(batch, rows, cols);
  if (rc != MOSS_OK) return rc;
  if (batch == 0 || rows == 0 || cols == 0) return clear_ok();
  *bytes = ns::layout_of(batch, rows, cols).total;
  return clear_ok();
}

extern "C" int moss_orthogonalize(const void* g, int g_dtype, int64_t batch, int64_t rows, int64_t cols, int steps,
                                  const float* coefficients, float eps, void* out, void* workspace,
                                  size_t workspace_bytes, int* status, moss_stream_t stream) {
  return ns::run(g, g_dtype, batch, rows, cols, steps, coefficients, eps, static_cast<__nv_bfloat16*>(out), workspace,
                 workspace_bytes, status, reinterpret_cast<cudaStream_t>(stream));
}
