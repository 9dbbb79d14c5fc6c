// Block quantisers of the fp8 linear.
//
// Rows (activations, gradients): one scale for each row and 128 columns, the least power of two
// 2^p with max|x| <= 448 * 2^p. Dividing by a power of two is exact, so a code is the one correct
// rounding of x / 2^p (ties to even) whichever way the division is done, and a block keeps the
// format's full relative precision: fp8 is a floating-point type, so only the range matters.
// Weights: one f32 scale max|w| / 448 for each 128 x 128 block, as fp8 checkpoints store them.
//
// Both are bound by HBM: 2 bytes read and 1 written per value. A half-warp holds one row's 128
// columns (16 bytes a lane), so the maximum is four shuffles away and the values are read once.
#include <algorithm>

#include "fp8_args.cuh"
#include "fp8_codes.cuh"

namespace moss {
namespace fp8 {

constexpr int kThreads = 256;
constexpr int kRowsPerCta = kThreads / 16;
// Column blocks per half-warp, loaded together as they are stored: 128 bytes a thread in flight. With
// half of that, unpacked on arrival, the kernel reached 3.8 TB/s instead of 6.3 (9216 x 12288 bf16).
template <int kKind>
constexpr int kBatch = kKind == kF32 ? 4 : 8;

// Codes and scale of the half-warp's 128 columns of one row, 8 a lane.
__device__ __forceinline__ void emit_block(const float (&v)[8], float amax, int64_t row, int block, int kb, int sub,
                                           uint8_t* codes, float* scale, int64_t row_pitch) {
  float block_scale;
  const uint2 q = block_codes(v, amax, block_scale);
  *reinterpret_cast<uint2*>(codes + (row * kb + block) * kBlock + sub * 8) = q;
  if (sub == 0) scale[block * row_pitch + row] = block_scale;
}

// kWide: rows on 16-byte boundaries and whole 8-value chunks (k a multiple of 8).
template <int kKind, bool kWide>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const void* __restrict__ x, int64_t m, int64_t k, int kb,
                                                                 uint8_t* __restrict__ codes, float* __restrict__ scale,
                                                                 int64_t row_pitch) {
  pdl_trigger();
  // neighbouring CTAs walk along the rows: DRAM pages are read whole
  constexpr int kB = kBatch<kKind>;
  const int groups = (kb + kB - 1) / kB;
  const int64_t row = static_cast<int64_t>(blockIdx.x / groups) * kRowsPerCta + (threadIdx.x >> 4);
  const int sub = threadIdx.x & 15;
  const int first = static_cast<int>(blockIdx.x % groups) * kB;
  if constexpr (kWide) {
    Raw<kKind> raw[kB];
#pragma unroll
    for (int i = 0; i < kB; ++i) {
      const int64_t c0 = static_cast<int64_t>(first + i) * kBlock + sub * 8;
      raw[i] = row < m && c0 < k ? load_raw<kKind>(x, row * k + c0) : Raw<kKind>{};
    }
#pragma unroll
    for (int i = 0; i < kB; ++i) {
      const float amax = half_warp_max(max_nan(kAmaxFloor, amax_of<kKind>(raw[i])));
      if (row >= m || first + i >= kb) continue;
      float v[8];
      values_of<kKind>(raw[i], v);
      emit_block(v, amax, row, first + i, kb, sub, codes, scale, row_pitch);
    }
  } else {
    for (int i = 0; i < kB; ++i) {
      float v[8];
      float amax = kAmaxFloor;
      if (row < m && first + i < kb) {
        const int64_t c0 = static_cast<int64_t>(first + i) * kBlock + sub * 8;
        load8<kKind>(x, row * k + c0, k - c0, false, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = max_nan(amax, fabsf(v[j]));
      }
      amax = half_warp_max(amax);
      if (row < m && first + i < kb) emit_block(v, amax, row, first + i, kb, sub, codes, scale, row_pitch);
    }
  }
}

template <int kKind>
static int launch_rows_of(const void* x, int64_t m, int64_t k, uint8_t* codes, float* scale, int64_t row_pitch,
                          cudaStream_t stream) {
  const int kb = static_cast<int>((k + kBlock - 1) / kBlock);
  const int64_t ctas = (m + kRowsPerCta - 1) / kRowsPerCta * ((kb + kBatch<kKind> - 1) / kBatch<kKind>);
  if (ctas > INT32_MAX) return fail(MOSS_ERR_INVALID_ARGUMENT, "too many rows to quantise in one call");
  if (reinterpret_cast<uintptr_t>(x) % 16 == 0 && k % 8 == 0)
    quantize_rows_kernel<kKind, true><<<static_cast<unsigned>(ctas), kThreads, 0, stream>>>(x, m, k, kb, codes, scale, row_pitch);
  else
    quantize_rows_kernel<kKind, false><<<static_cast<unsigned>(ctas), kThreads, 0, stream>>>(x, m, k, kb, codes, scale, row_pitch);
  return check_cuda(cudaGetLastError(), "quantize_rows_kernel");
}

int launch_quantize_rows(const void* x, int dtype, int64_t m, int64_t k, uint8_t* codes, float* scale,
                         int64_t row_pitch, cudaStream_t stream) {
  if (dtype == kBF16) return launch_rows_of<kBF16>(x, m, k, codes, scale, row_pitch, stream);
  if (dtype == kF16) return launch_rows_of<kF16>(x, m, k, codes, scale, row_pitch, stream);
  return launch_rows_of<kF32>(x, m, k, codes, scale, row_pitch, stream);
}

// One CTA per 128 x 128 weight block: 16 rows at a time, 8 sweeps held in registers. Once per weight: 12288 x 3072 bf16
// 76 us (1.5 TB/s; a true division for every value).
template <int kKind>
__global__ void __launch_bounds__(kThreads) quantize_weight_kernel(const void* __restrict__ w, int64_t n, int64_t k,
                                                                   bool wide, uint8_t* __restrict__ codes, int64_t ld,
                                                                   float* __restrict__ scale, int* status) {
  constexpr int kSweeps = kBlock / kRowsPerCta;
  __shared__ float warp_max[kThreads / 32];
  const int64_t row0 = static_cast<int64_t>(blockIdx.y) * kBlock + (threadIdx.x >> 4);
  const int64_t c0 = static_cast<int64_t>(blockIdx.x) * kBlock + (threadIdx.x & 15) * 8;
  float v[kSweeps][8];
  float amax = kAmaxFloor;
#pragma unroll
  for (int i = 0; i < kSweeps; ++i) {
    const int64_t row = row0 + i * kRowsPerCta;
    if (row < n) {
      load8<kKind>(w, row * k + c0, k - c0, wide && c0 + 8 <= k, v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) amax = max_nan(amax, fabsf(v[i][j]));
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, d));
  if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = amax;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) amax = max_nan(amax, warp_max[i]);
  const float s = __fdiv_rn(amax, 448.0f);
  if (threadIdx.x == 0) {
    scale[static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x] = s;
    if (!(amax < __uint_as_float(0x7f800000u))) report_status(status, MOSS_STATUS_NONFINITE_WEIGHT);
  }
#pragma unroll
  for (int i = 0; i < kSweeps; ++i) {
    const int64_t row = row0 + i * kRowsPerCta;
    if (row >= n) continue;
    uint32_t q[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
      q[h] = codes4(__fdiv_rn(v[i][4 * h], s), __fdiv_rn(v[i][4 * h + 1], s), __fdiv_rn(v[i][4 * h + 2], s),
                    __fdiv_rn(v[i][4 * h + 3], s));
    // rows of codes are a multiple of 16 bytes long: whole words up to that, zero past k
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (c0 + 4 * h < ld) *reinterpret_cast<uint32_t*>(codes + row * ld + c0 + 4 * h) = q[h];
  }
}

}  // namespace fp8
}  // namespace moss

using namespace moss;

extern "C" int moss_fp8_quantize_rows(const void* x, int x_dtype, int64_t m, int64_t k, uint8_t* codes, float* scale,
                                      int64_t row_pitch, moss_stream_t stream) {
  if (!is_float_kind(x_dtype)) return fail(MOSS_ERR_UNSUPPORTED, "unsupported dtype code %d", x_dtype);
  if (m < 0 || k < 0 || m > INT32_MAX || k > (1 << 22)) return fail(MOSS_ERR_INVALID_ARGUMENT, "bad quantiser shape");
  if (row_pitch < m) return fail(MOSS_ERR_INVALID_ARGUMENT, "row_pitch is less than the row count");
  if (m == 0 || k == 0) return clear_ok();
  if (x == nullptr || codes == nullptr || scale == nullptr) return fail(MOSS_ERR_INVALID_ARGUMENT, "null pointer");
  if (reinterpret_cast<uintptr_t>(codes) % 16 != 0) return fail(MOSS_ERR_INVALID_ARGUMENT, "codes must be 16-byte aligned");
  const int rc = fp8::launch_quantize_rows(x, x_dtype, m, k, codes, scale, row_pitch, reinterpret_cast<cudaStream_t>(stream));
  return rc == MOSS_OK ? clear_ok() : rc;
}

extern "C" int moss_fp8_quantize_weight(const void* w, int w_dtype, int64_t n, int64_t k, uint8_t* codes, int64_t ld,
                                        float* scale, int* status, moss_stream_t stream) {
  if (!is_float_kind(w_dtype)) return fail(MOSS_ERR_UNSUPPORTED, "unsupported dtype code %d", w_dtype);
  if (n < 0 || k < 0 || n > (1 << 22) || k > INT32_MAX - 256) return fail(MOSS_ERR_INVALID_ARGUMENT, "bad quantiser shape");
  if (ld % 16 != 0 || ld < k || ld >= k + 16)
    return fail(MOSS_ERR_INVALID_ARGUMENT, "the code pitch must be k rounded up to a multiple of 16");
  if (n == 0 || k == 0) return clear_ok();
  if (w == nullptr || codes == nullptr || scale == nullptr) return fail(MOSS_ERR_INVALID_ARGUMENT, "null pointer");
  if (reinterpret_cast<uintptr_t>(codes) % 16 != 0) return fail(MOSS_ERR_INVALID_ARGUMENT, "codes must be 16-byte aligned");
  const bool wide = reinterpret_cast<uintptr_t>(w) % 16 == 0 && (k * dtype_size(w_dtype)) % 16 == 0;
  const dim3 grid(static_cast<unsigned>((k + fp8::kBlock - 1) / fp8::kBlock),
                  static_cast<unsigned>((n + fp8::kBlock - 1) / fp8::kBlock));
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (w_dtype == MOSS_DTYPE_BF16)
    fp8::quantize_weight_kernel<kBF16><<<grid, fp8::kThreads, 0, s>>>(w, n, k, wide, codes, ld, scale, status);
  else if (w_dtype == MOSS_DTYPE_F16)
    fp8::quantize_weight_kernel<kF16><<<grid, fp8::kThreads, 0, s>>>(w, n, k, wide, codes, ld, scale, status);
  else
    fp8::quantize_weight_kernel<kF32><<<grid, fp8::kThreads, 0, s>>>(w, n, k, wide, codes, ld, scale, status);
  MOSS_CUDA_TRY(cudaGetLastError());
  return clear_ok();
}
