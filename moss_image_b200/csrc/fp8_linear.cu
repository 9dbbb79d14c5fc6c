// Entry points of the block-scaled fp8 linear: plan, workspace layout, quantise, multiply, join.
#include <algorithm>
#include <cstring>

#include "fp8_args.cuh"

namespace moss {
namespace fp8 {

int sm_count() { return device_sm_count(); }

static int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Rows up to 64 stream the weight (fp8_rows.cu). Above that, pair tiles when their rounds over the
// GPU's pairs take no longer than those of single tiles; a single tile's block costs a quarter of
// a pair tile's products at the same rate, but reads twice the shared memory for them.
Plan make_plan(int64_t m, int64_t nc, int64_t kr, int sms) {
  Plan p;
  const int64_t kb = ceil_div(kr, kBlock);
  int64_t slots;  // work units that run at once
  if (m <= 64) {
    p.kind = Plan::kRows;
    p.tn = m <= 16 ? 16 : m <= 32 ? 32 : 64;
    p.tiles_m = 1;
    p.tiles_n = static_cast<int>(ceil_div(nc, 128));
    // two CTAs a multiprocessor; tiles that already reach three quarters of them are not split (2 rows x 3072 ->
    // 18432: 14.9 us in one piece, 13.9 in two and 2.5 to join them)
    slots = 4LL * p.tiles_n > 3LL * sms ? 0 : 2LL * sms;
  } else {
    const int64_t pair_tiles = ceil_div(m, 256) * ceil_div(nc, 256);
    const int64_t single_tiles = ceil_div(m, 128) * ceil_div(nc, 128);
    const int64_t pair_cost = ceil_div(pair_tiles, std::max(1, sms / 2)) * 512;
    const int64_t single_cost = ceil_div(single_tiles, sms) * 340;
    p.kind = pair_cost <= single_cost ? Plan::kPair : Plan::kSingle;
    const int64_t side = p.kind == Plan::kPair ? 256 : 128;
    p.tiles_m = static_cast<int>(ceil_div(m, side));
    p.tiles_n = static_cast<int>(ceil_div(nc, side));
    slots = p.kind == Plan::kPair ? 0 : sms;  // pair tiles fill the GPU by the rule above
  }
  // Split the reduction when the tiles leave at least half of the slots idle, four blocks or more a split.
  const int64_t tiles = static_cast<int64_t>(p.tiles_m) * p.tiles_n;
  const int64_t splits = std::max<int64_t>(1, std::min<int64_t>(slots / std::max<int64_t>(1, tiles), kb / 4));
  p.kb_per_split = static_cast<int>(ceil_div(kb, splits));
  p.splits = static_cast<int>(ceil_div(kb, p.kb_per_split));
  return p;
}

// Workspace: codes of the rows, their scales, the split partials; each 256-byte aligned.
struct Layout {
  int64_t row_pitch;
  size_t codes, scale, partial, total;
};
static Layout layout_of(int64_t m, int64_t nc, int64_t kr, const Plan& p) {
  Layout l{};
  auto up = [](size_t v) { return (v + 255) / 256 * 256; };
  const int64_t kb = ceil_div(kr, kBlock);
  l.row_pitch = ceil_div(m, 128) * 128;
  l.codes = 0;
  const bool codes = m > kRowsQuantised;
  l.scale = codes ? up(static_cast<size_t>(m) * kb * kBlock) : 0;
  l.partial = l.scale + (codes ? up(static_cast<size_t>(kb) * l.row_pitch * 4) : 0);
  if (p.splits > 1) {
    const size_t values = p.kind == Plan::kRows ? static_cast<size_t>(m) * nc
                                                : static_cast<size_t>(p.tiles_m) * p.tiles_n * 128 * 128;
    l.total = l.partial + up(values * p.splits * 4);
  } else {
    l.total = l.partial;
  }
  return l;
}

// out = sum over the splits, in split order, plus the bias in f32, rounded once.
__global__ void __launch_bounds__(256) join_splits_kernel(const float* __restrict__ partial, int splits, int64_t total,
                                                          int nc, const void* bias, int bias_kind, void* out, int out_kind) {
  pdl_wait();
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * 256) {
    float v = 0.0f;
    for (int s = 0; s < splits; ++s) v += __ldg(partial + s * total + i);
    if (bias != nullptr) v += load_as_float(bias, bias_kind, i % nc);
    store_from_float(out, out_kind, i, v);
  }
}

// The same for partials by tiles, [split][tile][128 columns][128 rows]: 32 x 32 outputs a CTA, turned
// through shared memory so that both sides are read and written in rows of 32.
__global__ void __launch_bounds__(256) join_tiles_kernel(const float* __restrict__ partial, int splits, int m, int nc,
                                                         int tiles_m, int tiles_n, int group_m, const void* bias,
                                                         int bias_kind, void* out, int out_kind) {
  __shared__ float turned[32][33];
  pdl_wait();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int m_blk, n_blk;
  gemm::tile_coords(blockIdx.x, tiles_m, tiles_n, m_blk, n_blk, group_m);
  const int r0 = static_cast<int>(blockIdx.y) / 4 * 32, c0 = static_cast<int>(blockIdx.y) % 4 * 32;
  if (m_blk * 128 + r0 >= m || n_blk * 128 + c0 >= nc) return;
  const int64_t step = static_cast<int64_t>(tiles_m) * tiles_n * 128 * 128;
  const float* src = partial + (static_cast<int64_t>(blockIdx.x) * 128 + c0) * 128 + r0 + lane;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = w + 8 * i;
    float v = 0.0f;
    for (int s = 0; s < splits; ++s) v += __ldg(src + s * step + c * 128);
    turned[c][lane] = v;
  }
  __syncthreads();
  const int col = n_blk * 128 + c0 + lane;
  if (col >= nc) return;
  const float b = bias != nullptr ? load_as_float(bias, bias_kind, col) : 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = m_blk * 128 + r0 + w + 8 * i;
    if (row < m) store_from_float(out, out_kind, static_cast<int64_t>(row) * nc + col, turned[lane][w + 8 * i] + b);
  }
}

__global__ void __launch_bounds__(256) fill_bias_rows_kernel(int64_t total, int nc, const void* bias, int bias_kind,
                                                             void* out, int out_kind) {
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * 256)
    store_from_float(out, out_kind, i, bias != nullptr ? load_as_float(bias, bias_kind, i % nc) : 0.0f);
}

static int check_shape(int64_t m, int64_t n, int64_t k) {
  if (m < 0 || n < 0 || k < 0) return fail(MOSS_ERR_INVALID_ARGUMENT, "negative fp8 linear shape");
  if (m > INT32_MAX - 256 || n > (1 << 22) || k > (1 << 22)) return fail(MOSS_ERR_INVALID_ARGUMENT, "fp8 linear dimension too large");
  return MOSS_OK;
}

static int run(bool dx, const void* x, int x_dtype, int64_t m, int64_t n, int64_t k, const uint8_t* codes, int64_t ld,
               const float* scale, const void* bias, int bias_dtype, void* out, int out_dtype, void* workspace,
               size_t workspace_bytes, int* status, cudaStream_t stream) {
  if (!is_float_kind(x_dtype) || !is_float_kind(out_dtype)) return fail(MOSS_ERR_UNSUPPORTED, "unsupported dtype code");
  if (bias != nullptr && !is_float_kind(bias_dtype)) return fail(MOSS_ERR_UNSUPPORTED, "unsupported bias dtype code");
  int rc = check_shape(m, n, k);
  if (rc != MOSS_OK) return rc;
  const int64_t kr = dx ? n : k, nc = dx ? k : n;
  if (m == 0 || nc == 0) return clear_ok();
  if (out == nullptr) return fail(MOSS_ERR_INVALID_ARGUMENT, "null output pointer");
  if (kr == 0) {
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>(ceil_div(m * nc, 256), 4096));
    fill_bias_rows_kernel<<<grid, 256, 0, stream>>>(m * nc, static_cast<int>(nc), bias, bias_dtype, out, out_dtype);
    MOSS_CUDA_TRY(cudaGetLastError());
    return clear_ok();
  }
  if (x == nullptr || codes == nullptr || scale == nullptr) return fail(MOSS_ERR_INVALID_ARGUMENT, "null input, weight or scale pointer");
  if (ld < k || ld % 16 != 0 || reinterpret_cast<uintptr_t>(codes) % 16 != 0)
    return fail(MOSS_ERR_INVALID_ARGUMENT, "weight codes need 16-byte aligned rows (pitch %lld for %lld columns)",
                static_cast<long long>(ld), static_cast<long long>(k));
  const Plan plan = make_plan(m, nc, kr, sm_count());
  const Layout l = layout_of(m, nc, kr, plan);
  if (l.total > 0 &&
      (workspace == nullptr || workspace_bytes < l.total || reinterpret_cast<uintptr_t>(workspace) % 256 != 0))
    return fail(MOSS_ERR_INVALID_ARGUMENT, "the fp8 linear needs %zu bytes of 256-byte aligned workspace", l.total);
  uint8_t* ws = static_cast<uint8_t*>(workspace);

  Args a{};
  a.M = static_cast<int>(m);
  a.Nc = static_cast<int>(nc);
  a.kb = static_cast<int>(ceil_div(kr, kBlock));
  a.x = x;
  a.x_kind = x_dtype;
  a.x_cols = kr;
  a.x_wide = kr % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
  a.row_scale = reinterpret_cast<float*>(ws + l.scale);
  a.row_pitch = l.row_pitch;
  a.w_scale = scale;
  const int k_blocks = static_cast<int>(ceil_div(k, kBlock));
  a.ws_col = dx ? 1 : k_blocks;
  a.ws_red = dx ? k_blocks : 1;
  a.col_blocks = static_cast<int>(ceil_div(nc, kBlock));
  a.bias = bias;
  a.bias_kind = bias_dtype;
  a.out = out;
  a.out_kind = out_dtype;
  a.partial = reinterpret_cast<float*>(ws + l.partial);
  a.splits = plan.splits;
  a.kb_per_split = plan.kb_per_split;
  a.tiles_m = plan.tiles_m;
  a.tiles_n = plan.tiles_n;
  // row tiles per rasterisation group: at most one round of the grid, so that a group's rows stay in L2
  const int slots = plan.kind == Plan::kPair ? std::max(1, sm_count() / 2) : sm_count();
  a.group_m = plan.tiles_n < slots ? std::max(1, std::min(gemm::kGroupM, slots / plan.tiles_n)) : gemm::kGroupM;
  a.status = StatusSink{status, status_mirror_for_current_device()};

  rc = bind_context();
  if (rc != MOSS_OK) return rc;
  CUtensorMap ta, tw, to;
  memset(&to, 0, sizeof(to));
  memset(&ta, 0, sizeof(ta));
  memset(&tw, 0, sizeof(tw));
  const uint32_t rows_box = plan.kind == Plan::kRows ? plan.tn : 128;
  const bool quantises = m <= kRowsQuantised;
  if ((!quantises && !gemm::make_map(&ta, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, ws + l.codes, static_cast<uint64_t>(a.kb) * kBlock, m,
                      static_cast<uint64_t>(a.kb) * kBlock, kBlock, rows_box, CU_TENSOR_MAP_SWIZZLE_128B)) ||
      !gemm::make_map(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, codes, k, n, ld, kBlock, 128, CU_TENSOR_MAP_SWIZZLE_128B))
    return fail(MOSS_ERR_CUDA, "the driver refused a tensor map of the fp8 linear");
  if (plan.kind != Plan::kRows && out_dtype != kF32)
    a.tma_out = gemm::make_map(&to, out_dtype == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                               2, out, nc, m, static_cast<uint64_t>(nc) * 2, 64, 128, CU_TENSOR_MAP_SWIZZLE_128B);
  if (!quantises) {
    rc = launch_quantize_rows(x, x_dtype, m, kr, ws + l.codes, reinterpret_cast<float*>(ws + l.scale), l.row_pitch, stream);
    if (rc != MOSS_OK) return rc;
  }
  rc = plan.kind == Plan::kRows ? launch_rows(dx, plan, ta, tw, a, stream) : launch_gemm(dx, plan, ta, tw, to, a, stream);
  if (rc != MOSS_OK) return rc;
  if (plan.splits > 1 && plan.kind != Plan::kRows) {
    rc = launch_dependent("join_tiles_kernel", join_tiles_kernel, dim3(static_cast<unsigned>(plan.tiles_m * plan.tiles_n), 16),
                          dim3(256), 0, stream, a.partial, plan.splits, a.M, a.Nc, plan.tiles_m, plan.tiles_n, a.group_m,
                          bias, bias_dtype, out, out_dtype);
  } else if (plan.splits > 1) {
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>(ceil_div(m * nc, 256), 8LL * sm_count()));
    rc = launch_dependent("join_splits_kernel", join_splits_kernel, dim3(grid), dim3(256), 0, stream, a.partial, plan.splits,
                          m * nc, a.Nc, bias, bias_dtype, out, out_dtype);
  }
  if (rc != MOSS_OK) return rc;
  return clear_ok();
}

}  // namespace fp8
}  // namespace moss

using namespace moss;

extern "C" int moss_fp8_linear_workspace_bytes(int64_t m, int64_t n_out, int64_t k_red, size_t* bytes) {
  if (bytes == nullptr) return fail(MOSS_ERR_INVALID_ARGUMENT, "null bytes pointer");
  *bytes = 0;
  const int rc = fp8::check_shape(m, n_out, k_red);
  if (rc != MOSS_OK) return rc;
  if (m == 0 || n_out == 0 || k_red == 0) return clear_ok();
  *bytes = fp8::layout_of(m, n_out, k_red, fp8::make_plan(m, n_out, k_red, fp8::sm_count())).total;
  return clear_ok();
}

extern "C" int moss_fp8_linear_fwd(const void* x, int x_dtype, int64_t m, int64_t k, const uint8_t* codes, int64_t ld,
                                   const float* scale, int64_t n, const void* bias, int bias_dtype, void* y,
                                   int y_dtype, void* workspace, size_t workspace_bytes, int* status,
                                   moss_stream_t stream) {
  return fp8::run(false, x, x_dtype, m, n, k, codes, ld, scale, bias, bias_dtype, y, y_dtype, workspace,
                  workspace_bytes, status, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int moss_fp8_linear_dx(const void* dy, int dy_dtype, int64_t m, int64_t n, const uint8_t* codes, int64_t ld,
                                  const float* scale, int64_t k, void* dx, int dx_dtype, void* workspace,
                                  size_t workspace_bytes, int* status, moss_stream_t stream) {
  return fp8::run(true, dy, dy_dtype, m, n, k, codes, ld, scale, nullptr, 0, dx, dx_dtype, workspace, workspace_bytes,
                  status, reinterpret_cast<cudaStream_t>(stream));
}
