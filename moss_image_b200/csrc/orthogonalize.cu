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
// (b A + c A A), which is small in the directions that still have to grow. The last two steps
// grow nothing and drop lo. Against float64 the result is within 1.4 times its own rounding to bfloat16,
// momentum with a few directions 80 times stronger than the rest included; bfloat16 operands are
// 5 to 100 times further off. Tested in tests/test_gpu_muon.py.
#include <algorithm>
#include <cmath>
#include <cstring>

#include "ns_args.cuh"

namespace moss {
namespace ns {

int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 148;
  return n;
}

constexpr int kThreads = 256;
constexpr int kNormParts = 64;

// Sums of squares over equal ranges of a matrix, in f64 (neither overflow nor a loss in long sums).
__global__ void __launch_bounds__(kThreads) sum_squares_kernel(const void* __restrict__ g, int dtype, int64_t size,
                                                               double* __restrict__ parts) {
  const int64_t base = static_cast<int64_t>(blockIdx.y) * size;
  const int64_t first = size * blockIdx.x / gridDim.x, last = size * (blockIdx.x + 1) / gridDim.x;
  double sum = 0.0;
  for (int64_t i = first + threadIdx.x; i < last; i += kThreads) {
    const double v = load_as_float(g, dtype, base + i);
    sum += v * v;
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
}

// hi + lo = G * unit / max(|G|, eps), padded with zeros to [rp][cp]; 32 x 32 tiles through shared memory
// when G is tall (so that both sides are read and written by rows).
__global__ void __launch_bounds__(kThreads) normalize_kernel(const void* __restrict__ g, int dtype, int r, int c, int rp,
                                                             int cp, int tall, const double* __restrict__ parts,
                                                             int num_parts, float eps, float unit, __half* __restrict__ hi,
                                                             __half* __restrict__ lo) {
  __shared__ float tile[32][33];
  const int64_t b = blockIdx.z;
  double sum = 0.0;
  for (int p = 0; p < num_parts; ++p) sum += parts[b * num_parts + p];
  const float norm = static_cast<float>(sqrt(sum));
  const float scale = unit / (norm < eps ? eps : norm);  // NaN stays NaN
  const int i0 = blockIdx.y * 32, j0 = blockIdx.x * 32;
  const int64_t base = b * r * c;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  for (int k = w; k < 32; k += kThreads / 32) {
    const int i = tall ? i0 + lane : i0 + k, j = tall ? j0 + k : j0 + lane;
    float v = 0.0f;
    if (i < r && j < c)
      v = load_as_float(g, dtype, base + (tall ? static_cast<int64_t>(j) * r + i : static_cast<int64_t>(i) * c + j));
    tile[tall ? lane : k][tall ? k : lane] = v * scale;
  }
  __syncthreads();
  for (int k = w; k < 32; k += kThreads / 32) {
    const float v = tile[k][lane];
    const __half h = __float2half_rn(v);
    const int64_t at = (b * rp + i0 + k) * cp + j0 + lane;
    hi[at] = h;
    lo[at] = __float2half_rn(v - __half2float(h));
  }
}

struct Layout {
  int r, c, rp, cp, side, chunks;
  bool tall, small;
  size_t x[2], low[2], a, b, parts, partial, q, total;
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
    l.chunks = small_chunks(batch, l.c, sm_count());
    const size_t square = static_cast<size_t>(l.side) * l.side * 4 * batch;
    l.partial = take(square * l.chunks);
    l.q = take(square);
  } else {
    l.rp = (l.r + 127) / 128 * 128;
    l.cp = (l.c + 127) / 128 * 128;
    const size_t wide = static_cast<size_t>(batch) * l.rp * l.cp * 2, square = static_cast<size_t>(batch) * l.rp * l.rp * 2;
    for (int i = 0; i < 2; ++i) {
      l.x[i] = take(wide);
      l.low[i] = take(wide);
    }
    l.a = take(square);
    l.b = take(square);
    l.parts = take(static_cast<size_t>(batch) * kNormParts * 8);
  }
  l.total = at;
  return l;
}

// Largest |s (a + b s^2 + c s^4)| over [0, top], and largest |b l + c l^2| over l = s^2 of the same range.
static void bounds_of(const float* k, double top, double* value, double* square) {
  const double a = k[0], b = k[1], c = k[2];
  auto p = [&](double s) { return std::fabs(s * (a + s * s * (b + c * s * s))); };
  auto m = [&](double l) { return std::fabs(l * (b + c * l)); };
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
  double top = 1.001, most = 1.0, widest = 1.0;
  for (int i = 0; i < steps; ++i) {
    const float* k = coefficients + 3 * i;
    if (!std::isfinite(k[0]) || !std::isfinite(k[1]) || !std::isfinite(k[2]))
      return fail(MOSS_ERR_INVALID_ARGUMENT, "the coefficients must be finite");
    double value, square;
    bounds_of(k, top, &value, &square);
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
    std::memcpy(s.coefficients, coefficients, sizeof(float) * 3 * steps);
    s.eps = eps;
    s.out = out;
    s.chunks = l.chunks;
    s.partial = reinterpret_cast<float*>(ws + l.partial);
    s.q = reinterpret_cast<float*>(ws + l.q);
    rc = launch_small(s, stream);
    return rc == MOSS_OK ? clear_ok() : rc;
  }

  rc = bind_context();
  if (rc != MOSS_OK) return rc;
  // powers of two: X in units of 1 / unit (entries near 1), A and B in units of 1 / gain (below 2^14)
  const float unit = std::exp2(std::round(0.5 * std::log2(static_cast<double>(l.c))));
  const float gain = std::exp2(std::floor(14.0 - std::log2(most)));
  double* parts = reinterpret_cast<double*>(ws + l.parts);
  const int64_t size = rows * cols;
  const int num_parts = static_cast<int>(std::min<int64_t>(kNormParts, (size + 4095) / 4096));
  sum_squares_kernel<<<dim3(num_parts, static_cast<unsigned>(batch)), kThreads, 0, stream>>>(g, dtype, size, parts);
  MOSS_CUDA_TRY(cudaGetLastError());
  __half* x[2] = {reinterpret_cast<__half*>(ws + l.x[0]), reinterpret_cast<__half*>(ws + l.x[1])};
  __half* low[2] = {reinterpret_cast<__half*>(ws + l.low[0]), reinterpret_cast<__half*>(ws + l.low[1])};
  __half* ga = reinterpret_cast<__half*>(ws + l.a);
  __half* gb = reinterpret_cast<__half*>(ws + l.b);
  normalize_kernel<<<dim3(l.cp / 32, l.rp / 32, static_cast<unsigned>(batch)), kThreads, 0, stream>>>(
      g, dtype, l.r, l.c, l.rp, l.cp, l.tall, parts, num_parts, eps, unit, x[0], low[0]);
  MOSS_CUDA_TRY(cudaGetLastError());
  const int with_low = std::max(1, steps - 2);  // steps whose a X term reads lo
  for (int i = 0; i < steps; ++i) {
    const float* k = coefficients + 3 * i;
    Args a{};
    a.r = l.r;
    a.c = l.c;
    a.rp = l.rp;
    a.cp = l.cp;
    a.batch = static_cast<int>(batch);
    a.tall = l.tall;
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
