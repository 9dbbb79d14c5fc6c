// Rotary positions of queries and keys (moss_rotary).
//
// Each head's first `rotary_dim` values are R / 2 pairs, (2 i, 2 i + 1) in the interleaved layout
// or (i, i + R / 2) in the half layout; pair i of a token is turned by that token's angle:
//   (a, b) -> (a cos - b sin, a sin + b cos),
// in f32, rounded once to the tensors' type. The other head_dim - rotary_dim values are copied.
// The gradient is the same map with -sin (`inverse`): the matrix of a turn is orthogonal.
//
// The bound is HBM traffic: q and k are read once and written once. One launch serves both, and a
// thread keeps its 16-byte slice of the token's cos / sin row in registers for kHeads heads,
// so the f32 table costs L1 traffic once per kHeads heads and DRAM traffic once per token.
// 9216 tokens x 48 heads x 128 bf16: 39.0 us, 0.89 of the copy rate (32768 tokens, or float32, 72 us: all of it). Where a
// part of the head is copied, the turning and the copying lanes of a warp wait for each other (12287 x 32 x 128 f16,
// 64 turned: 46.5 us for 31.2).
#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "common.cuh"
#include "errors.cuh"

namespace moss {
namespace rotary {

constexpr int kThreads = 128;  // small blocks: the last round of a grid leaves less idle (25% on 12287 x 32 heads)
constexpr int kHeads = 4;  // heads per thread: independent 16-byte loads in flight

// n / d for 0 <= n < 2^31 by a multiplication (Granlund and Montgomery, 1994).
struct Divisor {
  uint32_t d, mul;
  int shift;
};
static Divisor divisor(int d) {
  Divisor v;
  v.d = static_cast<uint32_t>(d);
  v.shift = 0;
  while ((1ll << v.shift) < d) ++v.shift;
  v.mul = static_cast<uint32_t>(((1ull << 32) * ((1ull << v.shift) - v.d)) / v.d + 1);
  return v;
}
__device__ __forceinline__ int quotient(int n, const Divisor& v) {
  return static_cast<int>((__umulhi(static_cast<uint32_t>(n), v.mul) + static_cast<uint32_t>(n)) >> v.shift);
}

struct Part {  // the queries or the keys
  const void* in;
  void* out;  // dense [batch, tokens, heads, head_dim]
  int64_t batch_stride, token_stride, head_stride;
  int heads, groups;  // groups of kHeads heads
};

struct Args {
  Part part[2];
  const float* cos;
  const float* sin;
  const int64_t* positions;  // row of the table for each token; null: the token's index
  int64_t position_stride;   // between batches (0: shared)
  int64_t table_rows;
  int rows, tokens;  // batch * tokens, tokens
  int head_dim, half;
  int chunks, turned;  // work items of one head: all, and those that hold pairs
  int items;           // work items of one token
  Divisor by_chunks, by_items, by_tokens;
  int rows_per_block;
  int inverse;
};

template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};

// To and from f32, pairs by packed conversions (one by one they are a third of the kernel's time).
template <typename T, int N>
__device__ __forceinline__ void widen(const Vec<T, N>& x, float (&f)[N]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = x.v[i];
  } else if constexpr (N == 1) {
    f[0] = static_cast<float>(x.v[0]);
  } else {
    using P = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const P p = reinterpret_cast<const P*>(x.v)[i];
      f[2 * i] = __low2float(p);
      f[2 * i + 1] = __high2float(p);
    }
  }
}
template <typename T, int N>
__device__ __forceinline__ void narrow(const float (&f)[N], Vec<T, N>& x) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < N; ++i) x.v[i] = f[i];
  } else if constexpr (N == 1) {
    if constexpr (std::is_same<T, __half>::value)
      x.v[0] = __float2half_rn(f[0]);
    else
      x.v[0] = __float2bfloat16_rn(f[0]);
  } else {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      if constexpr (std::is_same<T, __half>::value)
        reinterpret_cast<__half2*>(x.v)[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      else
        reinterpret_cast<__nv_bfloat162*>(x.v)[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    }
  }
}


// kVec values per access; a chunk of pairs covers kVec values (interleaved) or kVec values of
// each half (half layout).
template <typename T, int kVec, bool kInterleaved>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const Args args) {
  constexpr int kAngles = kInterleaved ? (kVec > 1 ? kVec / 2 : 1) : kVec;
  // one value per access cannot hold an interleaved pair: the two are then read one by one
  constexpr bool kSplitPair = kInterleaved && kVec == 1;
  const int row0 = static_cast<int>(blockIdx.x) * args.rows_per_block;
  const int rows_here = min(args.rows_per_block, args.rows - row0);
  for (int it = threadIdx.x; it < rows_here * args.items; it += kThreads) {
    const int r = quotient(it, args.by_items);
    const int w = it - r * args.items;
    const int row = row0 + r;
    const int b = quotient(row, args.by_tokens);
    const int s = row - b * args.tokens;
    const int g = quotient(w, args.by_chunks);
    const int c = w - g * args.chunks;
    const bool keys = g >= args.part[0].groups;
    const Part& p = args.part[keys ? 1 : 0];
    const int h0 = (keys ? g - args.part[0].groups : g) * kHeads;
    const int n = min(kHeads, p.heads - h0);
    const T* in = static_cast<const T*>(p.in) + b * p.batch_stride + s * p.token_stride + h0 * p.head_stride;
    T* out = static_cast<T*>(p.out) + (static_cast<int64_t>(row) * p.heads + h0) * args.head_dim;
    if (c >= args.turned) {  // values past rotary_dim: copied
      const int at = 2 * args.half + (c - args.turned) * kVec;
      Vec<T, kVec> v[kHeads];
#pragma unroll
      for (int j = 0; j < kHeads; ++j)
        if (j < n) v[j] = *reinterpret_cast<const Vec<T, kVec>*>(in + j * p.head_stride + at);
#pragma unroll
      for (int j = 0; j < kHeads; ++j)
        if (j < n) *reinterpret_cast<Vec<T, kVec>*>(out + j * args.head_dim + at) = v[j];
      continue;
    }
    const int first = (kSplitPair ? 2 : 1) * c * kVec;  // first value of the chunk
    const int second = kInterleaved ? first + 1 : first + args.half;
    const int angle = kInterleaved ? first / 2 : first;
    Vec<T, kVec> lo[kHeads], hi[kHeads];
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
      if (j >= n) continue;
      lo[j] = *reinterpret_cast<const Vec<T, kVec>*>(in + j * p.head_stride + first);
      if constexpr (!kInterleaved || kSplitPair)
        hi[j] = *reinterpret_cast<const Vec<T, kVec>*>(in + j * p.head_stride + second);
    }
    const int64_t place = args.positions != nullptr ? args.positions[b * args.position_stride + s] : s;
    Vec<float, kAngles> co, si;
    if (place >= 0 && place < args.table_rows) {
      co = *reinterpret_cast<const Vec<float, kAngles>*>(args.cos + place * args.half + angle);
      si = *reinterpret_cast<const Vec<float, kAngles>*>(args.sin + place * args.half + angle);
    } else {  // a position outside the table has no angle: its token reads NaN
#pragma unroll
      for (int i = 0; i < kAngles; ++i) co.v[i] = si.v[i] = __int_as_float(0x7fffffff);
    }
    if (args.inverse) {
#pragma unroll
      for (int i = 0; i < kAngles; ++i) si.v[i] = -si.v[i];
    }
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
      if (j >= n) continue;
      T* dst = out + j * args.head_dim;
      float x[kVec], y[kVec];
      widen(lo[j], x);
      if constexpr (kInterleaved && !kSplitPair) {
#pragma unroll
        for (int i = 0; i < kAngles; ++i) {
          y[2 * i] = x[2 * i] * co.v[i] - x[2 * i + 1] * si.v[i];
          y[2 * i + 1] = x[2 * i] * si.v[i] + x[2 * i + 1] * co.v[i];
        }
        narrow(y, lo[j]);
        *reinterpret_cast<Vec<T, kVec>*>(dst + first) = lo[j];
      } else {
        widen(hi[j], y);
#pragma unroll
        for (int i = 0; i < kAngles; ++i) {
          const float a = x[i], b2 = y[i];
          x[i] = a * co.v[i] - b2 * si.v[i];
          y[i] = a * si.v[i] + b2 * co.v[i];
        }
        narrow(x, lo[j]);
        narrow(y, hi[j]);
        *reinterpret_cast<Vec<T, kVec>*>(dst + first) = lo[j];
        *reinterpret_cast<Vec<T, kVec>*>(dst + second) = hi[j];
      }
    }
  }
}

template <typename T, int kVec>
static int launch(Args a, bool interleaved, int rotary_dim, cudaStream_t stream) {
  a.turned = interleaved ? (kVec == 1 ? a.half : rotary_dim / kVec) : a.half / kVec;
  a.chunks = a.turned + (a.head_dim - rotary_dim) / kVec;
  a.items = (a.part[0].groups + a.part[1].groups) * a.chunks;
  a.by_chunks = divisor(a.chunks);
  a.by_items = divisor(a.items);
  a.by_tokens = divisor(a.tokens);
  // about four work items per thread and block, fewer when that would leave SMs without a block
  const int64_t want = std::max<int64_t>(1, 4 * kThreads / a.items);
  a.rows_per_block = static_cast<int>(std::min<int64_t>(want, std::max<int64_t>(1, a.rows / 592)));
  const unsigned grid = static_cast<unsigned>((a.rows + a.rows_per_block - 1) / a.rows_per_block);
  if (interleaved)
    rotary_kernel<T, kVec, true><<<grid, kThreads, 0, stream>>>(a);
  else
    rotary_kernel<T, kVec, false><<<grid, kThreads, 0, stream>>>(a);
  return check_cuda(cudaGetLastError(), "rotary_kernel");
}

// The widest access that every address allows: `vec` values at a time.
static bool fits(const Args& a, int vec, int esize, int rotary_dim, bool interleaved) {
  const uintptr_t bytes = static_cast<uintptr_t>(vec) * esize;
  if (a.head_dim % vec != 0 || rotary_dim % vec != 0 || (!interleaved && a.half % vec != 0)) return false;
  const uintptr_t angles = (interleaved ? vec / 2 : vec) * sizeof(float);
  if (reinterpret_cast<uintptr_t>(a.cos) % angles != 0 || reinterpret_cast<uintptr_t>(a.sin) % angles != 0) return false;
  for (const Part& p : a.part) {
    if (p.heads == 0) continue;
    if (reinterpret_cast<uintptr_t>(p.in) % bytes != 0 || reinterpret_cast<uintptr_t>(p.out) % bytes != 0) return false;
    if (p.batch_stride % vec != 0 || p.token_stride % vec != 0 || p.head_stride % vec != 0) return false;
  }
  return true;
}

template <typename T>
static int dispatch(const Args& a, bool interleaved, int rotary_dim, cudaStream_t stream) {
  constexpr int kWidest = 16 / sizeof(T);
  if (fits(a, kWidest, sizeof(T), rotary_dim, interleaved)) return launch<T, kWidest>(a, interleaved, rotary_dim, stream);
  if constexpr (kWidest > 4) {  // 16-bit rows whose half is a multiple of 4 values only (head 80, 40 turned)
    if (fits(a, 4, sizeof(T), rotary_dim, interleaved)) return launch<T, 4>(a, interleaved, rotary_dim, stream);
  }
  return launch<T, 1>(a, interleaved, rotary_dim, stream);
}

}  // namespace rotary
}  // namespace moss

using namespace moss;

extern "C" int moss_rotary(const void* q, int64_t q_batch_stride, int64_t q_token_stride, int64_t q_head_stride,
                           int64_t q_heads, const void* k, int64_t k_batch_stride, int64_t k_token_stride,
                           int64_t k_head_stride, int64_t k_heads, int dtype, int64_t batch, int64_t tokens,
                           int64_t head_dim, const float* cos, const float* sin, int64_t table_rows, int64_t rotary_dim,
                           const int64_t* positions, int64_t position_stride, int interleaved, int inverse, void* q_out,
                           void* k_out, moss_stream_t stream) {
  if (!is_float_kind(dtype)) return fail(MOSS_ERR_UNSUPPORTED, "unsupported dtype code %d", dtype);
  if (batch < 0 || tokens < 0 || q_heads < 0 || k_heads < 0 || table_rows < 0)
    return fail(MOSS_ERR_INVALID_ARGUMENT, "negative rotary shape");
  if (head_dim < 1 || head_dim > 8192) return fail(MOSS_ERR_INVALID_ARGUMENT, "head_dim must be in [1, 8192]");
  if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 2 != 0)
    return fail(MOSS_ERR_INVALID_ARGUMENT, "rotary_dim must be even and at most head_dim");
  if (q_heads + k_heads > 65536 || (batch > 0 && tokens > INT32_MAX / batch))
    return fail(MOSS_ERR_INVALID_ARGUMENT, "too many heads or tokens");
  if (batch == 0 || tokens == 0 || q_heads + k_heads == 0) return clear_ok();
  if ((q_heads > 0 && (q == nullptr || q_out == nullptr)) || (k_heads > 0 && (k == nullptr || k_out == nullptr)))
    return fail(MOSS_ERR_INVALID_ARGUMENT, "null query or key pointer");
  if (rotary_dim > 0 && (cos == nullptr || sin == nullptr)) return fail(MOSS_ERR_INVALID_ARGUMENT, "null angle table");
  if (positions == nullptr && table_rows < tokens)
    return fail(MOSS_ERR_INVALID_ARGUMENT, "the angle table has %lld rows for %lld tokens",
                static_cast<long long>(table_rows), static_cast<long long>(tokens));
  rotary::Args a{};
  auto part = [](const void* in, void* out, int64_t bs, int64_t ts, int64_t hs, int64_t heads) {
    rotary::Part p{};
    p.in = in;
    p.out = out;
    p.batch_stride = bs;
    p.token_stride = ts;
    p.head_stride = hs;
    p.heads = static_cast<int>(heads);
    p.groups = static_cast<int>((heads + rotary::kHeads - 1) / rotary::kHeads);
    return p;
  };
  a.part[0] = part(q, q_out, q_batch_stride, q_token_stride, q_head_stride, q_heads);
  a.part[1] = part(k, k_out, k_batch_stride, k_token_stride, k_head_stride, k_heads);
  a.cos = cos;
  a.sin = sin;
  a.positions = positions;
  a.position_stride = position_stride;
  a.table_rows = table_rows;
  a.rows = static_cast<int>(batch * tokens);
  a.tokens = static_cast<int>(tokens);
  a.head_dim = static_cast<int>(head_dim);
  a.half = static_cast<int>(rotary_dim / 2);
  a.inverse = inverse != 0;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int rd = static_cast<int>(rotary_dim);
  int rc;
  if (dtype == MOSS_DTYPE_BF16)
    rc = rotary::dispatch<__nv_bfloat16>(a, interleaved != 0, rd, s);
  else if (dtype == MOSS_DTYPE_F16)
    rc = rotary::dispatch<__half>(a, interleaved != 0, rd, s);
  else
    rc = rotary::dispatch<float>(a, interleaved != 0, rd, s);
  return rc == MOSS_OK ? clear_ok() : rc;
}
