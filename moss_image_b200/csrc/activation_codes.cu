// Activations as 8-bit codes: encode, decode, and the weight gradient's plan and joins.
//
// Encode and decode are bound by HBM (2 + 33/32 bytes a 16-bit value each): 16 values a thread, as one
// 32-byte load and one 16-byte store, two threads to a block. Rows that 32-byte accesses cannot take (a width that is no
// multiple of 16, an unaligned view) go lane by lane, a block to a warp. 9216 x 3072 bf16, both: 29 us, 5.9 TB/s;
// 1003 x 1090 f16 lane by lane: 5 us each.
#include <algorithm>
#include <cstring>

#include "codes_args.cuh"

namespace moss {
namespace codes {
namespace {

constexpr int kThreads = 256;

// The exponent byte of a block with the largest magnitude `amax` (NaN where the block has one).
__device__ __forceinline__ int block_power(float amax, int cap, bool& finite) {
  const uint32_t bits = __float_as_uint(amax) & 0x7fffffffu;
  finite = bits < 0x7f800000u;
  // amax = f * 2^(e - 126) with f in [1/2, 1): one more where f > 127/128
  const int p = static_cast<int>(bits >> 23) - 126 - 7 + ((bits & 0x7fffffu) > 0x7e0000u ? 1 : 0);
  return max(-126, min(cap, p));
}

// round to nearest even and clamp: the low byte of 1.5 * 2^23 + v is the code (|v| <= 128 before the clamp)
__device__ __forceinline__ uint32_t code_of(float v, float inverse) {
  const float q = fminf(fmaxf(v * inverse, -static_cast<float>(kCodeMax)), static_cast<float>(kCodeMax));
  return __float_as_uint(q + 12582912.0f);
}
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return prmt(prmt(a, b, 0x0040u), prmt(c, d, 0x0040u), 0x5410u);
}

// 16 consecutive values, 32-byte aligned.
template <int K>
__device__ __forceinline__ void load16(const void* p, int64_t i, float (&f)[16]) {
  const char* at = static_cast<const char*>(p) + i * (K == kF32 ? 4 : 2);
#pragma unroll
  for (int h = 0; h < (K == kF32 ? 2 : 1); ++h) {
    uint32_t w[8];
    asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                 : "l"(at + 32 * h));
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (K == kF32) {
        f[8 * h + j] = __uint_as_float(w[j]);
      } else if constexpr (K == kBF16) {
        f[2 * j] = __uint_as_float(w[j] << 16);
        f[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
      } else {
        const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
        f[2 * j] = t.x;
        f[2 * j + 1] = t.y;
      }
    }
  }
}

template <int K>
__global__ void __launch_bounds__(kThreads) encode_wide_kernel(const void* __restrict__ x, uint32_t units, uint32_t chunks,
                                                               int cap, int8_t* codes, uint8_t* exponents) {
  const uint32_t unit = blockIdx.x * kThreads + threadIdx.x;
  const uint32_t row = unit / chunks, chunk = unit - row * chunks;
  const bool live = unit < units;
  float f[16], amax = 0.0f;
  if (live) {
    load16<K>(x, static_cast<int64_t>(unit) * 16, f);
#pragma unroll
    for (int j = 0; j < 16; ++j) amax = max_nan(amax, fabsf(f[j]));
  }
  // the block's other half: a row of an odd number of halves ends without one, and a partner of another row is not asked
  const uint32_t partner = chunk ^ 1u;
  const int lane = threadIdx.x & 31;
  const int from = (chunk & 1u) != 0 ? lane - 1 : lane + 1;
  const float theirs = __shfl_sync(0xffffffffu, amax, from & 31);
  // (an odd number of halves a row puts some pairs across two warps: those read the other half themselves)
  if (!live) return;
  if (partner < chunks) {
    if (from >= 0 && from < 32) {
      amax = max_nan(amax, theirs);
    } else {
      float g[16];
      load16<K>(x, (static_cast<int64_t>(row) * chunks + partner) * 16, g);
#pragma unroll
      for (int j = 0; j < 16; ++j) amax = max_nan(amax, fabsf(g[j]));
    }
  }
  bool finite;
  const int p = block_power(amax, cap, finite);
  const float inverse = pow2(-p);
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    w[j] = finite ? pack4(code_of(f[4 * j], inverse), code_of(f[4 * j + 1], inverse), code_of(f[4 * j + 2], inverse),
                          code_of(f[4 * j + 3], inverse))
                  : 0u;
  *reinterpret_cast<uint4*>(codes + static_cast<int64_t>(unit) * 16) = make_uint4(w[0], w[1], w[2], w[3]);
  if ((chunk & 1u) == 0) exponents[static_cast<int64_t>(row) * ((chunks + 1) / 2) + chunk / 2] = static_cast<uint8_t>(finite ? p + 127 : 255);
}

// A warp takes kEach blocks at a time, a lane a column; codes from the row's end to its pitch are zero.
constexpr int kEach = 4;
template <int K>
__global__ void __launch_bounds__(kThreads) encode_lane_kernel(const void* __restrict__ x, uint32_t units, int64_t cols,
                                                               uint32_t blocks, int cap, int8_t* codes, int64_t ld,
                                                               uint8_t* exponents) {
  const int lane = threadIdx.x & 31;
  const uint32_t first = (blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * kEach;
  float v[kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const uint32_t unit = first + e, at = unit / blocks;
    const int64_t row = at, c = (unit - at * blocks) * kBlock + lane;
    v[e] = unit < units && c < cols ? load_as_float(x, K, row * cols + c) : 0.0f;
  }
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const uint32_t unit = first + e, at = unit / blocks;
    const int64_t row = at, c = (unit - at * blocks) * kBlock + lane;
    if (unit >= units) break;
    float amax = fabsf(v[e]);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, off));
    bool finite;
    const int p = block_power(amax, cap, finite);
    if (c < ld) codes[row * ld + c] = finite ? static_cast<int8_t>(code_of(v[e], pow2(-p)) & 0xffu) : int8_t{0};
    if (lane == 0) exponents[unit] = static_cast<uint8_t>(finite ? p + 127 : 255);
  }
}

__device__ __forceinline__ float scale_of(uint8_t exponent) { return __uint_as_float(static_cast<uint32_t>(exponent) << 23); }
// Byte k of w as a signed value: 2^23 + 128 + code, less the 2^23 + 128.
template <int k>
__device__ __forceinline__ float code_value(uint32_t w) {
  return __uint_as_float(prmt(w ^ 0x80808080u, 0x4b000000u, 0x7440u | k)) - 8388736.0f;
}

template <int K>
__global__ void __launch_bounds__(kThreads) decode_wide_kernel(const int8_t* __restrict__ codes, int64_t ld,
                                                               const uint8_t* __restrict__ exponents, uint32_t units,
                                                               uint32_t chunks, void* out, int64_t out_ld) {
  const uint32_t unit = blockIdx.x * kThreads + threadIdx.x;
  if (unit >= units) return;
  const uint32_t row = unit / chunks, chunk = unit - row * chunks;
  const uint4 u = __ldg(reinterpret_cast<const uint4*>(codes + static_cast<int64_t>(row) * ld + chunk * 16));
  const float s = scale_of(__ldg(exponents + static_cast<int64_t>(row) * ((chunks + 1) / 2) + chunk / 2));
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  float f[16];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    f[4 * j] = code_value<0>(w[j]) * s;
    f[4 * j + 1] = code_value<1>(w[j]) * s;
    f[4 * j + 2] = code_value<2>(w[j]) * s;
    f[4 * j + 3] = code_value<3>(w[j]) * s;
  }
  char* to = static_cast<char*>(out) + (static_cast<int64_t>(row) * out_ld + chunk * 16) * (K == kF32 ? 4 : 2);
  uint32_t o[8];
  if constexpr (K == kF32) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = __float_as_uint(f[8 * h + j]);
      gemm::stg256(to + 32 * h, o);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = gemm::pack2_kind<K>(f[2 * j], f[2 * j + 1]);
    gemm::stg256(to, o);
  }
}

template <int K>
__global__ void __launch_bounds__(kThreads) decode_lane_kernel(const int8_t* __restrict__ codes, int64_t ld,
                                                               const uint8_t* __restrict__ exponents, uint32_t units,
                                                               int64_t cols, uint32_t blocks, void* out, int64_t out_ld) {
  const int lane = threadIdx.x & 31;
  const uint32_t first = (blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * kEach;
  float v[kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const uint32_t unit = first + e, at = unit / blocks;
    const int64_t row = at, c = (unit - at * blocks) * kBlock + lane;
    v[e] = unit < units && c < cols ? static_cast<float>(codes[row * ld + c]) * scale_of(__ldg(exponents + unit)) : 0.0f;
  }
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const uint32_t unit = first + e, at = unit / blocks;
    const int64_t row = at, c = (unit - at * blocks) * kBlock + lane;
    if (unit < units && c < cols) store_from_float(out, K, row * out_ld + c, v[e]);
  }
}

// Rows of 16-bit values to rows of a pitch that tensor maps take.
__global__ void __launch_bounds__(kThreads) copy_rows_kernel(const uint16_t* __restrict__ from, int64_t rows, int64_t cols,
                                                             uint16_t* to, int64_t ld) {
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    for (int64_t c = threadIdx.x; c < cols; c += kThreads) to[row * ld + c] = __ldg(from + row * cols + c);
  }
}

// out = sum over the splits, in split order, rounded once.
__global__ void __launch_bounds__(kThreads) join_kernel(const Args a) {
  pdl_wait();
  const int64_t total = static_cast<int64_t>(a.N) * a.K, step = a.part_rows * a.part_cols;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int64_t n = i / a.K, k = i - n * a.K;
    const float* src = a.partial + n * a.part_cols + k;
    float v = 0.0f;
#pragma unroll 8
    for (int s = 0; s < a.splits; ++s) v += __ldg(src + s * step);
    store_from_float(a.out, a.out_kind, i, v);
  }
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
bool aligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

int check_rows(int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 0) return fail(MOSS_ERR_INVALID_ARGUMENT, "negative shape of coded activations");
  // (blocks and halves of blocks are counted in 32 bits)
  if (cols > INT32_MAX - 256 || (cols > 0 && rows > ((int64_t{1} << 32) - 4096) / ceil_div(cols, 16)))
    return fail(MOSS_ERR_INVALID_ARGUMENT, "coded activations of %lld x %lld values are too large",
                static_cast<long long>(rows), static_cast<long long>(cols));
  return MOSS_OK;
}

int check_codes(const void* codes, int64_t ld, int64_t cols, const void* exponents) {
  if (codes == nullptr || exponents == nullptr) return fail(MOSS_ERR_INVALID_ARGUMENT, "null codes or exponents pointer");
  if (ld < cols || ld % 16 != 0 || !aligned(codes, 16))
    return fail(MOSS_ERR_INVALID_ARGUMENT, "codes need 16-byte aligned rows (pitch %lld for %lld columns)",
                static_cast<long long>(ld), static_cast<long long>(cols));
  return MOSS_OK;
}

int encode(const void* x, int kind, int64_t rows, int64_t cols, int8_t* codes, int64_t ld, uint8_t* exponents, cudaStream_t stream) {
  const int cap = kind == kF16 ? 9 : 121;
  if (cols % 16 == 0 && ld == cols && aligned(x, 32)) {
    const uint32_t chunks = static_cast<uint32_t>(cols / 16), units = static_cast<uint32_t>(rows * chunks);
    const unsigned grid = static_cast<unsigned>(ceil_div(rows * chunks, kThreads));
    if (kind == kF16)
      encode_wide_kernel<kF16><<<grid, kThreads, 0, stream>>>(x, units, chunks, cap, codes, exponents);
    else if (kind == kBF16)
      encode_wide_kernel<kBF16><<<grid, kThreads, 0, stream>>>(x, units, chunks, cap, codes, exponents);
    else
      encode_wide_kernel<kF32><<<grid, kThreads, 0, stream>>>(x, units, chunks, cap, codes, exponents);
  } else {
    const uint32_t blocks = static_cast<uint32_t>(ceil_div(cols, kBlock));
    const uint32_t units = static_cast<uint32_t>(rows * blocks);
    const int64_t grid = ceil_div(rows * blocks, kThreads / 32 * kEach);
    if (kind == kF16)
      encode_lane_kernel<kF16><<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(x, units, cols, blocks, cap, codes, ld, exponents);
    else if (kind == kBF16)
      encode_lane_kernel<kBF16><<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(x, units, cols, blocks, cap, codes, ld, exponents);
    else
      encode_lane_kernel<kF32><<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(x, units, cols, blocks, cap, codes, ld, exponents);
  }
  return check_cuda(cudaGetLastError(), "encode kernel");
}

template <int K>
int decode_typed(const int8_t* codes, int64_t ld, const uint8_t* exponents, int64_t rows, int64_t cols, void* out,
                 int64_t out_ld, cudaStream_t stream) {
  if (cols % 16 == 0 && out_ld % 16 == 0 && aligned(out, 32)) {
    const uint32_t chunks = static_cast<uint32_t>(cols / 16), units = static_cast<uint32_t>(rows * chunks);
    decode_wide_kernel<K><<<static_cast<unsigned>(ceil_div(rows * chunks, kThreads)), kThreads, 0, stream>>>(
        codes, ld, exponents, units, chunks, out, out_ld);
  } else {
    const uint32_t blocks = static_cast<uint32_t>(ceil_div(cols, kBlock));
    const int64_t grid = ceil_div(rows * blocks, kThreads / 32 * kEach);
    decode_lane_kernel<K><<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(codes, ld, exponents, static_cast<uint32_t>(rows * blocks),
                                                                                cols, blocks, out, out_ld);
  }
  return check_cuda(cudaGetLastError(), "decode kernel");
}

// How a gradient is computed. Few features: the codes are read once and decoded in registers (codes_rows.cu). More:
// the rows are decoded into the workspace (12 of 145 us at 9216 x 3072 -> 3072), and a GEMM reads them by TMA. Decoding
// tiles between TMA and the MMAs would save that copy, but send each operand through shared memory twice more beside
// the MMAs' own reads, which take half of its cycles.
struct Plan {
  bool few = false, pair = false;
  int tiles_m = 1, tiles_n = 1, splits = 1, per_split = 0;
};
Plan make_plan(int64_t m, int64_t n, int64_t k, int sms) {
  Plan p;
  if (n <= kFewFeatures) {
    p.few = true;
    p.tiles_n = static_cast<int>(ceil_div(k, kRowsColumns));
    // one CTA a multiprocessor; 64 rows a split at least, kRowsMost at most
    const int64_t wanted = std::max<int64_t>(1, sms / std::max(1, p.tiles_n));
    int64_t rows = std::max<int64_t>(ceil_div(m, wanted), 64);
    rows = std::min<int64_t>(ceil_div(rows, 16) * 16, kRowsMost);
    p.per_split = static_cast<int>(rows);
    p.splits = static_cast<int>(ceil_div(m, rows));
    return p;
  }
  const int64_t steps = ceil_div(m, kStep);
  const int64_t pair_tiles = ceil_div(n, 256) * ceil_div(k, 256), single_tiles = ceil_div(n, 128) * ceil_div(k, 128);
  // relative cost of a round: a pair tile has four times the products of a single one in 1.5 times the step's time (single
  // tiles are bound by what a multiprocessor reads). Pair and single tiles, us, 9216 rows: 3072 x 3072 121 and 161, 1024 x 3072
  // 60 and 82, 2000 x 2000 68 and 114; 1536 x 1536 48 and 42, 768 x 768 24 and 22.
  const int64_t pair_cost = ceil_div(pair_tiles, std::max(1, sms / 2)) * 20;
  const int64_t single_cost = ceil_div(single_tiles, sms) * 13;
  p.pair = pair_cost <= single_cost;
  p.tiles_m = static_cast<int>(ceil_div(n, p.pair ? 256 : 128));
  p.tiles_n = static_cast<int>(ceil_div(k, p.pair ? 256 : 128));
  const int64_t tiles = static_cast<int64_t>(p.tiles_m) * p.tiles_n;
  // the reduction is cut where tiles leave at least half of the GPU idle, four steps or more a split
  const int64_t slots = p.pair ? sms / 2 : sms;
  const int64_t splits = std::max<int64_t>(1, std::min<int64_t>(slots / tiles, steps / 4));
  p.per_split = static_cast<int>(ceil_div(steps, splits));
  p.splits = static_cast<int>(ceil_div(steps, p.per_split));
  return p;
}

// Workspace: decoded rows, partials, copied gradient rows; each 256-byte aligned. The last are needed for gradients that TMA
// cannot read in place alone, so their room comes last.
struct Layout {
  int64_t x_ld, y_ld, part_rows, part_cols;
  size_t partial, y, total;
};
Layout layout_of(int64_t m, int64_t n, int64_t k, const Plan& p) {
  Layout l{};
  auto up = [](size_t v) { return (v + 255) / 256 * 256; };
  l.x_ld = ceil_div(k, 16) * 16;
  l.y_ld = ceil_div(n, 8) * 8;
  l.partial = p.few ? 0 : up(static_cast<size_t>(m) * l.x_ld * 2);
  if (p.splits > 1) {
    l.part_rows = p.few ? n : static_cast<int64_t>(p.tiles_m) * (p.pair ? 256 : 128);
    l.part_cols = p.few ? static_cast<int64_t>(p.tiles_n) * kRowsColumns : static_cast<int64_t>(p.tiles_n) * (p.pair ? 256 : 128);
  }
  l.y = l.partial + (p.splits > 1 ? up(static_cast<size_t>(p.splits) * l.part_rows * l.part_cols * 4) : 0);
  l.total = l.y + (p.few ? 0 : up(static_cast<size_t>(m) * l.y_ld * 2));
  return l;
}

int check_gradient(int64_t m, int64_t n, int64_t k) {
  if (m < 0 || n < 0 || k < 0) return fail(MOSS_ERR_INVALID_ARGUMENT, "negative shape of a coded gradient");
  if (m > INT32_MAX - 4096 || n > (1 << 22) || k > (1 << 22))
    return fail(MOSS_ERR_INVALID_ARGUMENT, "coded gradient dimension too large");
  return check_rows(m, k);
}

int gradient(const void* dy, int dtype, int64_t m, int64_t n, const int8_t* codes, int64_t ld, const uint8_t* exponents,
             int64_t k, void* dw, int dw_dtype, void* workspace, size_t workspace_bytes, int* status, cudaStream_t stream) {
  if (dtype != kF16 && dtype != kBF16) return fail(MOSS_ERR_UNSUPPORTED, "coded gradients are computed from 16-bit gradients");
  if (!is_float_kind(dw_dtype)) return fail(MOSS_ERR_UNSUPPORTED, "unsupported dtype code");
  int rc = check_gradient(m, n, k);
  if (rc != MOSS_OK) return rc;
  if (n == 0 || k == 0) return clear_ok();
  if (dw == nullptr) return fail(MOSS_ERR_INVALID_ARGUMENT, "null output pointer");
  if (m == 0) {
    MOSS_CUDA_TRY(cudaMemsetAsync(dw, 0, static_cast<size_t>(n) * k * dtype_size(dw_dtype), stream));
    return clear_ok();
  }
  if (dy == nullptr) return fail(MOSS_ERR_INVALID_ARGUMENT, "null gradient pointer");
  rc = check_codes(codes, ld, k, exponents);
  if (rc != MOSS_OK) return rc;
  const Plan plan = make_plan(m, n, k, device_sm_count());
  const Layout l = layout_of(m, n, k, plan);
  const bool in_place = n % 8 == 0 && aligned(dy, 16);
  const size_t needed = in_place ? l.y : l.total;
  if (needed > 0 && (workspace == nullptr || workspace_bytes < needed || !aligned(workspace, 256)))
    return fail(MOSS_ERR_INVALID_ARGUMENT, "the coded gradient needs %zu bytes of 256-byte aligned workspace", needed);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  Args a{};
  a.M = static_cast<int>(m);
  a.N = static_cast<int>(n);
  a.K = static_cast<int>(k);
  a.dy = dy;
  a.codes = codes;
  a.ld = ld;
  a.exponents = exponents;
  a.out = dw;
  a.out_kind = dw_dtype;
  a.partial = reinterpret_cast<float*>(ws + l.partial);
  a.part_rows = l.part_rows;
  a.part_cols = l.part_cols;
  a.splits = plan.splits;
  a.per_split = plan.per_split;
  a.tiles_m = plan.tiles_m;
  a.tiles_n = plan.tiles_n;
  // row tiles per rasterisation group: at most one round of the grid, so that a group's operands stay in L2
  const int slots = plan.pair ? std::max(1, device_sm_count() / 2) : device_sm_count();
  a.group_m = plan.tiles_n < slots ? std::max(1, std::min(gemm::kGroupM, slots / plan.tiles_n)) : gemm::kGroupM;
  a.status = StatusSink{status, status_mirror_for_current_device()};
  if (plan.few) {
    rc = launch_rows(dtype, a, stream);
  } else {
    rc = launch_decode(codes, ld, exponents, m, k, ws, l.x_ld, dtype, stream);
    if (rc != MOSS_OK) return rc;
    const void* rows = dy;
    if (!in_place) {
      copy_rows_kernel<<<static_cast<unsigned>(std::min<int64_t>(m, 8LL * device_sm_count())), kThreads, 0, stream>>>(
          static_cast<const uint16_t*>(dy), m, n, reinterpret_cast<uint16_t*>(ws + l.y), l.y_ld);
      MOSS_CUDA_TRY(cudaGetLastError());
      rows = ws + l.y;
    }
    rc = bind_context();
    if (rc != MOSS_OK) return rc;
    CUtensorMap ty, tx;
    const CUtensorMapDataType type = dtype == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    if (!gemm::make_map(&ty, type, 2, rows, n, m, static_cast<uint64_t>(l.y_ld) * 2, 64, kStep, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !gemm::make_map(&tx, type, 2, ws, k, m, static_cast<uint64_t>(l.x_ld) * 2, 64, kStep, CU_TENSOR_MAP_SWIZZLE_128B))
      return fail(MOSS_ERR_CUDA, "the driver refused a tensor map of the coded gradient");
    rc = launch_gemm(plan.pair, dtype, ty, tx, a, stream);
  }
  if (rc != MOSS_OK) return rc;
  if (plan.splits > 1) {
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>(ceil_div(n * k, kThreads), 8LL * device_sm_count()));
    rc = launch_dependent("join_kernel", join_kernel, dim3(grid), dim3(kThreads), 0, stream, a);
    if (rc != MOSS_OK) return rc;
  }
  return clear_ok();
}

}  // namespace

int launch_decode(const int8_t* codes, int64_t ld, const uint8_t* exponents, int64_t rows, int64_t cols, void* out,
                  int64_t out_ld, int kind, cudaStream_t stream) {
  if (kind == kF16) return decode_typed<kF16>(codes, ld, exponents, rows, cols, out, out_ld, stream);
  if (kind == kBF16) return decode_typed<kBF16>(codes, ld, exponents, rows, cols, out, out_ld, stream);
  return decode_typed<kF32>(codes, ld, exponents, rows, cols, out, out_ld, stream);
}

}  // namespace codes
}  // namespace moss

using namespace moss;

extern "C" int moss_codes_encode(const void* x, int dtype, int64_t rows, int64_t cols, int8_t* codes, int64_t ld,
                                 uint8_t* exponents, moss_stream_t stream) {
  if (!is_float_kind(dtype)) return fail(MOSS_ERR_UNSUPPORTED, "unsupported dtype code");
  int rc = codes::check_rows(rows, cols);
  if (rc != MOSS_OK) return rc;
  if (rows == 0 || cols == 0) return clear_ok();
  if (x == nullptr) return fail(MOSS_ERR_INVALID_ARGUMENT, "null input pointer");
  rc = codes::check_codes(codes, ld, cols, exponents);
  if (rc == MOSS_OK && ld != codes::ceil_div(cols, 16) * 16)
    rc = fail(MOSS_ERR_INVALID_ARGUMENT, "the encoder writes rows of the least pitch, %lld columns rounded up to 16", static_cast<long long>(cols));
  if (rc == MOSS_OK) rc = codes::encode(x, dtype, rows, cols, codes, ld, exponents, reinterpret_cast<cudaStream_t>(stream));
  return rc != MOSS_OK ? rc : clear_ok();
}

extern "C" int moss_codes_decode(const int8_t* codes, int64_t ld, const uint8_t* exponents, int64_t rows, int64_t cols,
                                 void* out, int dtype, moss_stream_t stream) {
  if (!is_float_kind(dtype)) return fail(MOSS_ERR_UNSUPPORTED, "unsupported dtype code");
  int rc = codes::check_rows(rows, cols);
  if (rc != MOSS_OK) return rc;
  if (rows == 0 || cols == 0) return clear_ok();
  if (out == nullptr) return fail(MOSS_ERR_INVALID_ARGUMENT, "null output pointer");
  rc = codes::check_codes(codes, ld, cols, exponents);
  if (rc == MOSS_OK) rc = codes::launch_decode(codes, ld, exponents, rows, cols, out, cols, dtype, reinterpret_cast<cudaStream_t>(stream));
  return rc != MOSS_OK ? rc : clear_ok();
}

extern "C" int moss_coded_gradient_workspace_bytes(int64_t rows, int64_t n, int64_t cols, size_t* bytes) {
  if (bytes == nullptr) return fail(MOSS_ERR_INVALID_ARGUMENT, "null bytes pointer");
  *bytes = 0;
  const int rc = codes::check_gradient(rows, n, cols);
  if (rc != MOSS_OK) return rc;
  if (rows == 0 || n == 0 || cols == 0) return clear_ok();
  *bytes = codes::layout_of(rows, n, cols, codes::make_plan(rows, n, cols, device_sm_count())).total;
  return clear_ok();
}

extern "C" int moss_coded_gradient(const void* dy, int dtype, int64_t rows, int64_t n, const int8_t* codes, int64_t ld,
                                   const uint8_t* exponents, int64_t cols, void* dw, int dw_dtype, void* workspace,
                                   size_t workspace_bytes, int* status, moss_stream_t stream) {
  return codes::gradient(dy, dtype, rows, n, codes, ld, exponents, cols, dw, dw_dtype, workspace, workspace_bytes, status,
                         reinterpret_cast<cudaStream_t>(stream));
}
