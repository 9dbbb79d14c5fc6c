// Entry points of the attention to another sequence: checks, plan, tensor maps, joins.
#include <algorithm>
#include <cmath>
#include <cstring>

#include "cross_args.cuh"

namespace moss {
namespace cross {
namespace {

constexpr int kThreads = 256;
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// The splits' outputs weighted by their sums: out = sum_s 2^(L_s - L) O_s, in split order. A thread takes 8 values.
__global__ void __launch_bounds__(kThreads) join_forward_kernel(const Args a, int kind, int64_t vectors) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= vectors) return;
  const int each = a.head_dim / 8;
  const int64_t at = i / each, row = at / a.q_heads;
  const int head = static_cast<int>(at - row * a.q_heads);
  const float* lse = a.partial_lse + head * a.q_rows + row;
  const int64_t lse_step = a.q_heads * a.q_rows, step = a.q_rows * a.q_heads * a.head_dim;
  float top = -INFINITY;
  for (int s = 0; s < a.splits; ++s) top = max_nan(top, __ldg(lse + s * lse_step));
  float sum = 0.0f, v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
  if (top != -INFINITY) {
    for (int s = 0; s < a.splits; ++s) {
      const float w = exp2f(__ldg(lse + s * lse_step) - top);
      sum += w;
      float o[8];
      load8<kF32>(a.partial + s * step, i * 8, 8, true, o);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = fmaf(w, o[j], v[j]);
    }
    const float inverse = 1.0f / sum;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= inverse;
  }
  uint4 w;
  if (kind == kBF16)
    w = make_uint4(gemm::pack2_kind<kBF16>(v[0], v[1]), gemm::pack2_kind<kBF16>(v[2], v[3]),
                   gemm::pack2_kind<kBF16>(v[4], v[5]), gemm::pack2_kind<kBF16>(v[6], v[7]));
  else
    w = make_uint4(gemm::pack2_kind<kF16>(v[0], v[1]), gemm::pack2_kind<kF16>(v[2], v[3]),
                   gemm::pack2_kind<kF16>(v[4], v[5]), gemm::pack2_kind<kF16>(v[6], v[7]));
  *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + i * 8) = w;
  if (a.lse != nullptr && i == at * each) a.lse[head * a.q_rows + row] = top == -INFINITY ? INFINITY : top + log2f(sum);
}

// The splits' sums in split order, rounded once. A thread takes 8 values.
__global__ void __launch_bounds__(kThreads) join_sums_kernel(const float* __restrict__ partial, int splits, int64_t vectors,
                                                             void* out, int kind) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= vectors) return;
  float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    float o[8];
    load8<kF32>(partial, (s * vectors + i) * 8, 8, true, o);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += o[j];
  }
  uint4 w;
  if (kind == kBF16)
    w = make_uint4(gemm::pack2_kind<kBF16>(v[0], v[1]), gemm::pack2_kind<kBF16>(v[2], v[3]),
                   gemm::pack2_kind<kBF16>(v[4], v[5]), gemm::pack2_kind<kBF16>(v[6], v[7]));
  else
    w = make_uint4(gemm::pack2_kind<kF16>(v[0], v[1]), gemm::pack2_kind<kF16>(v[2], v[3]),
                   gemm::pack2_kind<kF16>(v[4], v[5]), gemm::pack2_kind<kF16>(v[6], v[7]));
  *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + i * 8) = w;
}
int join_sums(const float* partial, int splits, int64_t values, void* out, int kind, cudaStream_t stream) {
  const int64_t vectors = values / 8;
  join_sums_kernel<<<static_cast<unsigned>(ceil_div(vectors, kThreads)), kThreads, 0, stream>>>(partial, splits, vectors, out, kind);
  return check_cuda(cudaGetLastError(), "join_sums_kernel");
}

// The same for the split units of dk and dv, a CTA for each quarter of a unit and tensor.
__global__ void __launch_bounds__(kThreads) join_tail_kernel(const Args a, int kind) {
  const int of = a.whole + static_cast<int>(blockIdx.x), head = of / a.tiles;
  int seq, tile;
  if (!find_tile<true>(a, kTile, of - head * a.tiles, seq, tile)) return;
  const Sequence s = sequence_of(a, seq);
  const int rows = min(kTile, s.kn - tile * kTile), each = a.head_dim / 8;
  const int64_t unit = static_cast<int64_t>(kTile) * a.head_dim, step = a.tail * unit;
  const float* from = a.partial + static_cast<int64_t>(blockIdx.y) * a.splits * step + blockIdx.x * unit;
  uint16_t* const to = static_cast<uint16_t*>(blockIdx.y == 0 ? a.dv : a.dk);
  const int quarter = kTile / 4 * each;
  for (int i = blockIdx.z * quarter + threadIdx.x; i < min(rows * each, static_cast<int>(blockIdx.z + 1) * quarter); i += kThreads) {
    float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int p = 0; p < a.splits; ++p) {
      float o[8];
      load8<kF32>(from + p * step, i * 8, 8, true, o);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += o[j];
    }
    uint4 w;
    if (kind == kBF16)
      w = make_uint4(gemm::pack2_kind<kBF16>(v[0], v[1]), gemm::pack2_kind<kBF16>(v[2], v[3]),
                     gemm::pack2_kind<kBF16>(v[4], v[5]), gemm::pack2_kind<kBF16>(v[6], v[7]));
    else
      w = make_uint4(gemm::pack2_kind<kF16>(v[0], v[1]), gemm::pack2_kind<kF16>(v[2], v[3]),
                     gemm::pack2_kind<kF16>(v[4], v[5]), gemm::pack2_kind<kF16>(v[6], v[7]));
    const int row = i / each, c = i - row * each;
    *reinterpret_cast<uint4*>(to + ((s.k_row + tile * kTile + row) * a.k_heads + head) * a.head_dim + c * 8) = w;
  }
}

// Exponents of the greatest |V|^2 that each sequence's keys have, by key head: 16 lanes a row of a head.
__global__ void __launch_bounds__(kThreads) value_sizes_kernel(const Args a, const uint16_t* __restrict__ v, int64_t v_batch,
                                                               int64_t v_token, int64_t v_head) {
  const int64_t at = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / 16, row = at / a.k_heads;
  const int head = static_cast<int>(at - row * a.k_heads), part = threadIdx.x & 15;
  int seq = -1;
  const uint16_t* from = v;
  if (row < a.k_rows) {
    if (a.k_offsets == nullptr) {
      seq = static_cast<int>(row / a.tk);
      const int64_t key = row - static_cast<int64_t>(seq) * a.tk;
      if (a.mask != nullptr && __ldg(a.mask + seq * a.mask_ld + key) == 0) seq = -1;
      from += seq * v_batch + key * v_token;
    } else {
      int low = 0, high = a.batch;  // the first boundary behind the row is that of `low`
      while (low < high) {
        const int mid = (low + high) / 2;
        if (clamped(a.k_offsets, mid + 1, a.tk) > row)
          high = mid;
        else
          low = mid + 1;
      }
      if (low < a.batch) seq = low;  // (nobody looks at rows behind the last sequence)
      from += row * v_token;
    }
  }
  float sum = 0.0f;
  if (seq >= 0 && 8 * part < a.head_dim) {
    float x[8];
    load8<kF16>(from + head * v_head, 8 * part, 8, true, x);
#pragma unroll
    for (int j = 0; j < 8; ++j) sum = fmaf(x[j], x[j], sum);
  }
#pragma unroll
  for (int d = 8; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  if (seq >= 0 && part == 0) raise_to(a.sizes + static_cast<int64_t>(seq) * a.k_heads + head, exponent_of(fabsf(sum)));
}

struct Problem {
  int64_t batch, tq, tk, q_heads, k_heads, head_dim;
  bool packed;
  int64_t q_rows() const { return packed ? tq : batch * tq; }
  int64_t k_rows() const { return packed ? tk : batch * tk; }
};

int check(const Problem& p) {
  if (p.batch < 0 || p.tq < 0 || p.tk < 0 || p.q_heads < 1 || p.k_heads < 1)
    return fail(MOSS_ERR_INVALID_ARGUMENT, "negative shape of a cross attention, or no heads");
  if (p.q_heads % p.k_heads != 0) return fail(MOSS_ERR_INVALID_ARGUMENT, "query heads must be a multiple of the key heads");
  if (p.head_dim < 8 || p.head_dim > 128 || p.head_dim % 8 != 0)
    return fail(MOSS_ERR_UNSUPPORTED, "head_dim must be a multiple of 8 up to 128, not %lld", static_cast<long long>(p.head_dim));
  const int64_t tiles = p.packed ? p.tq / kTile + p.tk / kTile + 2 * (p.batch + 2) : p.batch * (p.tq / kTile + p.tk / kTile + 2);
  if (p.tq > INT32_MAX - 4096 || p.tk > INT32_MAX - 4096 || p.batch > INT32_MAX - 4096 || tiles > (1 << 30) / p.q_heads)
    return fail(MOSS_ERR_INVALID_ARGUMENT, "cross attention too large");
  return MOSS_OK;
}

// Tiles of `rows` rows over all sequences, at most.
int64_t tiles_of(const Problem& p, int64_t tokens, int64_t rows) {
  return p.packed ? tokens / rows + p.batch + 1 : p.batch * ceil_div(tokens, rows);
}

// Splits of the keys: as many as bring the units (of `rows` queries) to one for each multiprocessor, two key tiles or more each.
int key_splits(const Problem& p, int64_t rows) {
  const int64_t units = std::max<int64_t>(1, p.q_heads * (p.packed ? ceil_div(p.tq, rows) : tiles_of(p, p.tq, rows)));
  const int64_t keys = ceil_div(p.packed ? ceil_div(p.tk, std::max<int64_t>(1, p.batch)) : p.tk, kTile);
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(device_sm_count() / units, keys / 2)));
}

size_t up(size_t v) { return (v + 255) / 256 * 256; }

struct ForwardLayout {
  size_t lse, total;
};
ForwardLayout forward_layout(const Problem& p, int splits) {
  ForwardLayout l{};
  if (splits <= 1) return l;
  l.lse = up(static_cast<size_t>(splits) * p.q_rows() * p.q_heads * p.head_dim * 4);
  l.total = l.lse + up(static_cast<size_t>(splits) * p.q_rows() * p.q_heads * 4);
  return l;
}

// How dk and dv are shared out: whole units (a key tile of one head) in full rounds over the multiprocessors, and the last
// ones split over their queries where that is shorter, in steps of a tile pair (1.2 us measured), with two more a unit for its
// start and end, and the partial sums' way through memory. (192 units of 32 steps: 44 of them split in three.)
struct KeyPlan {
  int64_t whole = 0, tail = 0;
  int splits = 1;
};
KeyPlan plan_keys(const Problem& p) {
  const int64_t sms = device_sm_count();
  const int64_t units = p.k_heads * tiles_of(p, p.tk, kTile);
  // (of packed keys a tile for each sequence at most is not there)
  const int64_t there = std::min(units, p.k_heads * (p.packed ? ceil_div(p.tk, kTile) + p.batch / 2 : units));
  const int64_t queries = p.packed ? ceil_div(p.tq, std::max<int64_t>(1, p.batch)) : p.tq;
  const int64_t steps = ceil_div(queries, kTile) * (p.q_heads / p.k_heads);
  KeyPlan plan;
  const int64_t rest = there % sms;
  double least = static_cast<double>(steps + 2);
  for (int64_t s = 2; s <= std::min<int64_t>(16, steps / 2) && rest > 0; ++s) {
    // written and read once in f32, at 4 TB/s, and a launch
    const double bytes = 16.0 * s * rest * kTile * p.head_dim;
    const double cost = static_cast<double>(ceil_div(rest * s, sms) * (ceil_div(steps, s) + 2)) + bytes / 4e12 / 1.2e-6 + 3.0;
    if (cost < least) {
      plan.splits = static_cast<int>(s);
      least = cost;
    }
  }
  // packed sequences differ in length, which only the device knows: more and smaller units even that out
  if (p.packed) plan.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(ceil_div(4 * sms, std::max<int64_t>(1, there)), steps / 4)));
  if (p.packed) plan.splits = std::min(plan.splits, 16);
  plan.tail = plan.splits == 1 ? 0 : there < sms || p.packed ? units : rest;
  plan.whole = units - plan.tail;
  return plan;
}

struct BackwardLayout {
  size_t dq, dkv, sizes, sizes_bytes, total;  // after the deltas
};
BackwardLayout backward_layout(const Problem& p, int dq_splits, const KeyPlan& keys) {
  BackwardLayout l{};
  l.dq = up(static_cast<size_t>(p.q_heads) * p.q_rows() * 4);
  l.dkv = l.dq + (dq_splits > 1 ? up(static_cast<size_t>(dq_splits) * p.q_rows() * p.q_heads * p.head_dim * 4) : 0);
  l.sizes = l.dkv + up(static_cast<size_t>(keys.tail) * keys.splits * 2 * kTile * p.head_dim * 4);
  l.sizes_bytes = 2 * static_cast<size_t>(p.batch + 1) * p.k_heads * sizeof(int);  // (rows behind the last sequence are one more)
  l.total = l.sizes + up(l.sizes_bytes);
  return l;
}

struct Strides {
  int64_t batch, token, head;
};

bool make_map(CUtensorMap* map, int kind, const void* p, const Problem& s, int64_t tokens, int64_t heads, Strides st) {
  const uint64_t dims[4] = {static_cast<uint64_t>(s.head_dim), static_cast<uint64_t>(tokens), static_cast<uint64_t>(heads),
                            static_cast<uint64_t>(s.packed ? 1 : s.batch)};
  // (a dimension of one entry may come with any stride)
  const uint64_t row = static_cast<uint64_t>(ceil_div(s.head_dim, 8) * 16);
  const uint64_t strides[3] = {tokens == 1 ? row : static_cast<uint64_t>(st.token) * 2, heads == 1 ? row : static_cast<uint64_t>(st.head) * 2,
                               dims[3] == 1 ? row : static_cast<uint64_t>(st.batch) * 2};
  const uint32_t box[4] = {64, kTile, 1, 1};
  return gemm::make_map_nd(map, kind == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, p, 4,
                           dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

Args args_of(const Problem& p, const int64_t* q_offsets, const int64_t* k_offsets, const uint8_t* mask, int64_t mask_ld,
             float scale, int* status) {
  Args a{};
  a.batch = static_cast<int>(p.batch);
  a.q_heads = static_cast<int>(p.q_heads);
  a.k_heads = static_cast<int>(p.k_heads);
  a.group = static_cast<int>(p.q_heads / p.k_heads);
  a.head_dim = static_cast<int>(p.head_dim);
  a.tq = static_cast<int>(p.tq);
  a.tk = static_cast<int>(p.tk);
  a.q_offsets = q_offsets;
  a.k_offsets = k_offsets;
  a.mask = mask;
  a.mask_ld = mask_ld;
  a.scale = scale;
  a.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  a.q_rows = p.q_rows();
  a.k_rows = p.k_rows();
  a.splits = 1;
  a.status = StatusSink{status, status_mirror_for_current_device()};
  return a;
}

int check_call(const Problem& p, int dtype, const int64_t* q_offsets, const int64_t* k_offsets, const uint8_t* mask, float scale) {
  if (dtype != kF16 && dtype != kBF16) return fail(MOSS_ERR_UNSUPPORTED, "cross attention takes f16 and bf16");
  if ((q_offsets == nullptr) != (k_offsets == nullptr)) return fail(MOSS_ERR_INVALID_ARGUMENT, "packed rows need both boundaries");
  if (q_offsets != nullptr && mask != nullptr) return fail(MOSS_ERR_UNSUPPORTED, "packed keys take no mask");
  if (!(scale > 0.0f) || !std::isfinite(scale)) return fail(MOSS_ERR_INVALID_ARGUMENT, "the scale must be positive and finite");
  return check(p);
}

int forward(const Problem& p, const void* q, Strides qs, const void* k, Strides ks, const void* v, Strides vs, int dtype,
            const int64_t* q_offsets, const int64_t* k_offsets, const uint8_t* mask, int64_t mask_ld, float scale, void* out,
            float* lse, void* workspace, size_t workspace_bytes, int* status, cudaStream_t stream) {
  int rc = check_call(p, dtype, q_offsets, k_offsets, mask, scale);
  if (rc != MOSS_OK) return rc;
  if (p.q_rows() == 0) return clear_ok();
  if (out == nullptr) return fail(MOSS_ERR_INVALID_ARGUMENT, "null output pointer");
  if (p.k_rows() == 0) {  // no keys at all (what the row sums are then, nothing reads)
    MOSS_CUDA_TRY(cudaMemsetAsync(out, 0, static_cast<size_t>(p.q_rows()) * p.q_heads * p.head_dim * 2, stream));
    return clear_ok();
  }
  if (q == nullptr || k == nullptr || v == nullptr) return fail(MOSS_ERR_INVALID_ARGUMENT, "null query, key or value pointer");
  Args a = args_of(p, q_offsets, k_offsets, mask, mask_ld, scale, status);
  a.splits = key_splits(p, 2 * kTile);
  const ForwardLayout l = forward_layout(p, a.splits);
  if (l.total > 0 && (workspace == nullptr || workspace_bytes < l.total || reinterpret_cast<uintptr_t>(workspace) % 256 != 0))
    return fail(MOSS_ERR_INVALID_ARGUMENT, "the cross attention needs %zu bytes of 256-byte aligned workspace", l.total);
  a.out = out;
  a.lse = lse;
  a.partial = static_cast<float*>(workspace);
  a.partial_lse = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + l.lse);
  a.tiles = static_cast<int>(tiles_of(p, p.tq, 2 * kTile));
  rc = bind_context();
  if (rc != MOSS_OK) return rc;
  Maps maps;
  const Strides dense{p.tq * p.q_heads * p.head_dim, p.q_heads * p.head_dim, p.head_dim};
  if (!make_map(&maps.o, dtype, out, p, p.tq, p.q_heads, dense) || !make_map(&maps.q, dtype, q, p, p.tq, p.q_heads, qs) ||
      !make_map(&maps.k, dtype, k, p, p.tk, p.k_heads, ks) || !make_map(&maps.v, dtype, v, p, p.tk, p.k_heads, vs))
    return fail(MOSS_ERR_INVALID_ARGUMENT, "queries, keys, values and outputs need 16-byte aligned rows of one stride");
  rc = launch_forward(dtype, maps, a, stream);
  if (rc != MOSS_OK) return rc;
  if (a.splits > 1) {
    const int64_t vectors = a.q_rows * a.q_heads * (a.head_dim / 8);
    join_forward_kernel<<<static_cast<unsigned>(ceil_div(vectors, kThreads)), kThreads, 0, stream>>>(a, dtype, vectors);
    MOSS_CUDA_TRY(cudaGetLastError());
  }
  return clear_ok();
}

int backward(const Problem& p, const void* grad, const void* q, Strides qs, const void* k, Strides ks, const void* v, Strides vs,
             int dtype, const int64_t* q_offsets, const int64_t* k_offsets, const uint8_t* mask, int64_t mask_ld, float scale,
             const void* out, const float* lse, void* dq, void* dk, void* dv, void* workspace, size_t workspace_bytes,
             int* status, cudaStream_t stream) {
  int rc = check_call(p, dtype, q_offsets, k_offsets, mask, scale);
  if (rc != MOSS_OK) return rc;
  if ((dk == nullptr) != (dv == nullptr)) return fail(MOSS_ERR_INVALID_ARGUMENT, "the gradients of keys and values come together");
  const size_t q_bytes = static_cast<size_t>(p.q_rows()) * p.q_heads * p.head_dim * 2;
  const size_t k_bytes = static_cast<size_t>(p.k_rows()) * p.k_heads * p.head_dim * 2;
  if (p.q_rows() > 0 && dq == nullptr) return fail(MOSS_ERR_INVALID_ARGUMENT, "null gradient pointer");
  if (p.q_rows() == 0 || p.k_rows() == 0) {  // nobody looks at anything
    if (q_bytes > 0) MOSS_CUDA_TRY(cudaMemsetAsync(dq, 0, q_bytes, stream));
    if (dk != nullptr && k_bytes > 0) {
      MOSS_CUDA_TRY(cudaMemsetAsync(dk, 0, k_bytes, stream));
      MOSS_CUDA_TRY(cudaMemsetAsync(dv, 0, k_bytes, stream));
    }
    return clear_ok();
  }
  if (grad == nullptr || q == nullptr || k == nullptr || v == nullptr || out == nullptr || lse == nullptr)
    return fail(MOSS_ERR_INVALID_ARGUMENT, "null input pointer");
  const int dq_splits = key_splits(p, kTile);
  const KeyPlan keys = plan_keys(p);
  const BackwardLayout l = backward_layout(p, dq_splits, keys);
  if (workspace == nullptr || workspace_bytes < l.total || reinterpret_cast<uintptr_t>(workspace) % 256 != 0)
    return fail(MOSS_ERR_INVALID_ARGUMENT, "the cross attention's gradients need %zu bytes of 256-byte aligned workspace", l.total);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  Args a = args_of(p, q_offsets, k_offsets, mask, mask_ld, scale, status);
  a.o = out;
  a.grad = grad;
  a.lse = const_cast<float*>(lse);
  a.delta = reinterpret_cast<float*>(ws);
  a.out = dq;
  a.partial = reinterpret_cast<float*>(ws + l.dq);
  a.splits = dq_splits;
  a.tiles = static_cast<int>(tiles_of(p, p.tq, kTile));
  rc = bind_context();
  if (rc != MOSS_OK) return rc;
  Maps maps;
  const Strides dense{p.tq * p.q_heads * p.head_dim, p.q_heads * p.head_dim, p.head_dim};
  if (!make_map(&maps.o, dtype, out, p, p.tq, p.q_heads, dense) || !make_map(&maps.grad, dtype, grad, p, p.tq, p.q_heads, dense) ||
      !make_map(&maps.q, dtype, q, p, p.tq, p.q_heads, qs) || !make_map(&maps.k, dtype, k, p, p.tk, p.k_heads, ks) ||
      !make_map(&maps.v, dtype, v, p, p.tk, p.k_heads, vs))
    return fail(MOSS_ERR_INVALID_ARGUMENT, "queries, keys, values, outputs and gradients need 16-byte aligned rows of one stride");
  if (dtype == kF16) {
    a.sizes = reinterpret_cast<int*>(ws + l.sizes);
    MOSS_CUDA_TRY(cudaMemsetAsync(a.sizes, 0, l.sizes_bytes, stream));
    const int64_t threads = p.k_rows() * p.k_heads * 16;
    value_sizes_kernel<<<static_cast<unsigned>(ceil_div(threads, kThreads)), kThreads, 0, stream>>>(
        a, static_cast<const uint16_t*>(v), vs.batch, vs.token, vs.head);
    MOSS_CUDA_TRY(cudaGetLastError());
  }
  rc = launch_dq(dtype, maps, a, stream);
  if (rc == MOSS_OK && dq_splits > 1) rc = join_sums(a.partial, dq_splits, static_cast<int64_t>(q_bytes / 2), dq, dtype, stream);
  if (rc != MOSS_OK || dk == nullptr) return rc != MOSS_OK ? rc : clear_ok();
  a.dk = dk;
  a.dv = dv;
  a.partial = reinterpret_cast<float*>(ws + l.dkv);
  a.splits = keys.splits;
  a.whole = static_cast<int>(keys.whole);
  a.tail = static_cast<int>(keys.tail);
  a.tiles = static_cast<int>(tiles_of(p, p.tk, kTile));
  rc = launch_dkv(dtype, maps, a, stream);
  if (rc == MOSS_OK && a.tail > 0) {
    join_tail_kernel<<<dim3(static_cast<unsigned>(a.tail), 2, 4), kThreads, 0, stream>>>(a, dtype);
    rc = check_cuda(cudaGetLastError(), "join_tail_kernel");
  }
  return rc != MOSS_OK ? rc : clear_ok();
}

}  // namespace
}  // namespace cross
}  // namespace moss

using namespace moss;

extern "C" int moss_cross_attention_workspace_bytes(int64_t batch, int64_t q_tokens, int64_t k_tokens, int64_t q_heads,
                                                    int64_t k_heads, int64_t head_dim, int packed, int backward,
                                                    size_t* bytes) {
  if (bytes == nullptr) return fail(MOSS_ERR_INVALID_ARGUMENT, "null bytes pointer");
  *bytes = 0;
  const cross::Problem p{batch, q_tokens, k_tokens, q_heads, k_heads, head_dim, packed != 0};
  const int rc = cross::check(p);
  if (rc != MOSS_OK) return rc;
  if (p.q_rows() == 0 || p.k_rows() == 0) return clear_ok();
  *bytes = backward != 0 ? cross::backward_layout(p, cross::key_splits(p, cross::kTile), cross::plan_keys(p)).total
                         : cross::forward_layout(p, cross::key_splits(p, 2 * cross::kTile)).total;
  return clear_ok();
}

extern "C" int moss_cross_attention_fwd(const void* q, int64_t q_batch, int64_t q_token, int64_t q_head, const void* k,
                                        int64_t k_batch, int64_t k_token, int64_t k_head, const void* v, int64_t v_batch,
                                        int64_t v_token, int64_t v_head, int dtype, int64_t batch, int64_t q_tokens,
                                        int64_t k_tokens, int64_t q_heads, int64_t k_heads, int64_t head_dim,
                                        const int64_t* q_offsets, const int64_t* k_offsets, const uint8_t* mask,
                                        int64_t mask_ld, float scale, void* out, float* lse, void* workspace,
                                        size_t workspace_bytes, int* status, moss_stream_t stream) {
  const cross::Problem p{batch, q_tokens, k_tokens, q_heads, k_heads, head_dim, q_offsets != nullptr};
  return cross::forward(p, q, {q_batch, q_token, q_head}, k, {k_batch, k_token, k_head}, v, {v_batch, v_token, v_head}, dtype,
                        q_offsets, k_offsets, mask, mask_ld, scale, out, lse, workspace, workspace_bytes, status,
                        reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int moss_cross_attention_bwd(const void* grad, const void* q, int64_t q_batch, int64_t q_token, int64_t q_head,
                                        const void* k, int64_t k_batch, int64_t k_token, int64_t k_head, const void* v,
                                        int64_t v_batch, int64_t v_token, int64_t v_head, int dtype, int64_t batch,
                                        int64_t q_tokens, int64_t k_tokens, int64_t q_heads, int64_t k_heads,
                                        int64_t head_dim, const int64_t* q_offsets, const int64_t* k_offsets,
                                        const uint8_t* mask, int64_t mask_ld, float scale, const void* out, const float* lse,
                                        void* dq, void* dk, void* dv, void* workspace, size_t workspace_bytes, int* status,
                                        moss_stream_t stream) {
  const cross::Problem p{batch, q_tokens, k_tokens, q_heads, k_heads, head_dim, q_offsets != nullptr};
  return cross::backward(p, grad, q, {q_batch, q_token, q_head}, k, {k_batch, k_token, k_head}, v, {v_batch, v_token, v_head},
                         dtype, q_offsets, k_offsets, mask, mask_ld, scale, out, lse, dq, dk, dv, workspace, workspace_bytes,
                         status, reinterpret_cast<cudaStream_t>(stream));
}
