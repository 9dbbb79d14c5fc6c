// Layer norm over the last dimension, with gradients of the input, the gain and the offset:
//   mean = sum x / dim, rstd = 1 / sqrt(sum (x - mean)^2 / dim + eps), n = (x - mean) * rstd
//   y  = n * w + b                                            rounded once, to promote(x, w)
//   dx = rstd * (dn - sum(dn) / dim - n * sum(dn * n) / dim)  with dn = dy * w
//   dw = sum over rows of dy * n,   db = sum over rows of dy
// Everything between a load and a store is f32; the variance is summed from the centred values, so a mean
// far from zero costs it no digits (the mean has its own rounding, which is a part of the centred values).
//
// Bound by HBM where no gain is read (32768 x 3072 f32: 144 us, 0.85 of the copy rate), with one by shared memory as well, which
// it is read from as f32 (9216 x 3072 bf16: 32 us forward, 48 backward, 7 for the join). x and y (forward), x, dy and dx
// (backward) cross HBM once, because a row stays in the registers of
// its team of 8, 32, 128 or 512 threads from the load to the store. A thread owns the same columns in every row, so
// the gain and the offset are read once for each thread, and the weight gradients are summed in registers
// over all of a team's rows, then over the CTA's teams through shared memory; one row of f32 partials for
// each CTA is added in CTA order by a second kernel. No atomics: the sums do not depend on timing.
#include <algorithm>

#include "common.cuh"
#include "errors.cuh"

namespace moss {
namespace lnorm {
namespace {

constexpr int kThreads = 512;
constexpr int kMaxDim = 16384;  // 512 threads of 32 values

struct Args {
  const void* x;
  const void* w;
  const void* b;
  int g_kind;        // type of w and b
  const void* dy;
  float2* stats;     // mean and rstd of each row (forward writes, backward reads)
  void* out;         // y or dx
  float* partial;    // [CTAs][2][dim] sums of dy * n and of dy, or null
  int64_t rows;
  int dim;
  float eps;
};

// V values of kind K as they lie in memory.
template <int K, int V>
struct Raw {
  static constexpr int kBytes = V * (K == kF32 ? 4 : 2);
  static constexpr int kWords = kBytes < 4 ? 1 : kBytes / 4;
  uint32_t w[kWords];
};

template <int K, int V>
__device__ __forceinline__ Raw<K, V> load(const void* p, int64_t i) {
  Raw<K, V> r;
  const char* at = static_cast<const char*>(p) + i * (K == kF32 ? 4 : 2);
  if constexpr (Raw<K, V>::kBytes >= 16) {
#pragma unroll
    for (int c = 0; c < Raw<K, V>::kWords / 4; ++c) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(at) + c);
      r.w[4 * c] = u.x;
      r.w[4 * c + 1] = u.y;
      r.w[4 * c + 2] = u.z;
      r.w[4 * c + 3] = u.w;
    }
  } else if constexpr (Raw<K, V>::kBytes == 8) {
    const uint2 u = __ldg(reinterpret_cast<const uint2*>(at));
    r.w[0] = u.x;
    r.w[1] = u.y;
  } else if constexpr (Raw<K, V>::kBytes == 4) {
    r.w[0] = __ldg(reinterpret_cast<const uint32_t*>(at));
  } else {
    r.w[0] = __ldg(reinterpret_cast<const uint16_t*>(at));
  }
  return r;
}

template <int K, int V>
__device__ __forceinline__ void widen(const Raw<K, V>& r, float (&f)[V]) {
  if constexpr (K == kF32) {
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = __uint_as_float(r.w[j]);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const uint32_t h = j % 2 == 0 ? r.w[j / 2] & 0xffffu : r.w[j / 2] >> 16;
      f[j] = K == kBF16 ? __uint_as_float(h << 16) : __half2float(__ushort_as_half(static_cast<uint16_t>(h)));
    }
  }
}

template <int K>
__device__ __forceinline__ uint32_t round16(float v) {
  if constexpr (K == kBF16) return __bfloat16_as_ushort(__float2bfloat16_rn(v));
  return __half_as_ushort(__float2half_rn(v));
}
template <int K>
__device__ __forceinline__ uint32_t round16x2(float lo, float hi) {
  if constexpr (K == kBF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <int K, int V>
__device__ __forceinline__ void store(void* p, int64_t i, const float (&f)[V]) {
  char* at = static_cast<char*>(p) + i * (K == kF32 ? 4 : 2);
  if constexpr (K == kF32) {
    if constexpr (V == 8) {
      reinterpret_cast<float4*>(at)[0] = make_float4(f[0], f[1], f[2], f[3]);
      reinterpret_cast<float4*>(at)[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else if constexpr (V == 2) {
      *reinterpret_cast<float2*>(at) = make_float2(f[0], f[1]);
    } else {
      *reinterpret_cast<float*>(at) = f[0];
    }
  } else if constexpr (V == 8) {
    *reinterpret_cast<uint4*>(at) = make_uint4(round16x2<K>(f[0], f[1]), round16x2<K>(f[2], f[3]),
                                               round16x2<K>(f[4], f[5]), round16x2<K>(f[6], f[7]));
  } else if constexpr (V == 2) {
    *reinterpret_cast<uint32_t*>(at) = round16x2<K>(f[0], f[1]);
  } else {
    *reinterpret_cast<uint16_t*>(at) = static_cast<uint16_t>(round16<K>(f[0]));
  }
}

// Sums over a team of T threads, N of them at once; the same in every thread. Teams past a warp meet in shared
// memory behind a barrier of their own; the two slots take turns, so one barrier a sum is enough.
template <int T, int N>
__device__ __forceinline__ void team_sum(float (&v)[N], float (*red)[kThreads / 32][2], int& slot) {
#pragma unroll
  for (int off = (T < 32 ? T : 32) / 2; off > 0; off >>= 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], off);
  }
  if constexpr (T > 32) {
    const int warp = threadIdx.x >> 5, first = warp / (T / 32) * (T / 32);
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) red[slot][warp][i] = v[i];
    }
    asm volatile("bar.sync %0, %1;" ::"r"(1 + static_cast<int>(threadIdx.x) / T), "n"(T) : "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0.0f;
#pragma unroll
    for (int k = 0; k < T / 32; ++k) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += red[slot][first + k][i];
    }
    slot ^= 1;
  }
}

// The gain (or offset) as f32 in shared memory, for all rows of the CTA (in registers it makes the kernels spill).
__device__ __forceinline__ void stage_gain(float* to, const void* p, int kind, int dim, float absent) {
  if (p != nullptr && kind != kF32 && dim % 8 == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
    for (int i = threadIdx.x * 8; i < dim; i += kThreads * 8) {
      float v[8];
      if (kind == kBF16)
        load8<kBF16>(p, i, 8, true, v);
      else
        load8<kF16>(p, i, 8, true, v);
      *reinterpret_cast<float4*>(to + i) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(to + i + 4) = make_float4(v[4], v[5], v[6], v[7]);
    }
    return;
  }
  for (int i = threadIdx.x; i < dim; i += kThreads) to[i] = p == nullptr ? absent : load_as_float(p, kind, i);
}
template <int V>
__device__ __forceinline__ void gain_at(const float* held, int at, float (&g)[V]) {
  if constexpr (V == 8) {
    const float4 lo = *reinterpret_cast<const float4*>(held + at), hi = *reinterpret_cast<const float4*>(held + at + 4);
    g[0] = lo.x; g[1] = lo.y; g[2] = lo.z; g[3] = lo.w;
    g[4] = hi.x; g[5] = hi.y; g[6] = hi.z; g[7] = hi.w;
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) g[j] = held[at + j];
  }
}

// A thread's columns are those of its vectors thread + i * T of V values, for i < C.
//
// The next row is on its way while a team reduces and writes the one it holds.
template <int KX, int KY, int T, int V, int C>
__global__ void __launch_bounds__(kThreads) layernorm_fwd_kernel(const Args a) {
  extern __shared__ __align__(16) float gain[];  // w, then b, each padded to 4 values
  __shared__ float red[2][kThreads / 32][2];
  int slot = 0;
  const int thread = threadIdx.x % T;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (kThreads / T);
  const float inv_dim = 1.0f / static_cast<float>(a.dim);
  // few rows are spread over the CTAs first
  int64_t row = T < 32 ? static_cast<int64_t>(blockIdx.x) * (kThreads / T) + threadIdx.x / T
                       : blockIdx.x + static_cast<int64_t>(threadIdx.x / T) * gridDim.x;
  // a warp's teams take their shuffles together: rows past the end are computed on zeros and not stored
  const int64_t last = T < 32 ? (a.rows + 32 / T - 1) / (32 / T) * (32 / T) : a.rows;
  Raw<KX, V> next[C];
  auto fetch = [&](int64_t r) {
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int at = (thread + i * T) * V;
      if (r < a.rows && at < a.dim) next[i] = load<KX, V>(a.x, r * a.dim + at);
    }
  };
#pragma unroll
  for (int i = 0; i < C; ++i) {
#pragma unroll
    for (int k = 0; k < Raw<KX, V>::kWords; ++k) next[i].w[k] = 0;
  }
  fetch(row);
  float* const offset = gain + (a.dim + 3) / 4 * 4;
  const bool plain = a.w == nullptr && a.b == nullptr;
  if (!plain) stage_gain(gain, a.w, a.g_kind, a.dim, 1.0f);
  if (!plain) stage_gain(offset, a.b, a.g_kind, a.dim, 0.0f);
  __syncthreads();
  for (; row < last; row += step) {
    Raw<KX, V> held[C];
#pragma unroll
    for (int i = 0; i < C; ++i) held[i] = next[i];
    fetch(row + step);
    float sum[1] = {0.0f}, squares[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < C; ++i) {
      if ((thread + i * T) * V >= a.dim) continue;
      float f[V];
      widen<KX, V>(held[i], f);
#pragma unroll
      for (int j = 0; j < V; ++j) sum[0] += f[j];
    }
    team_sum<T, 1>(sum, red, slot);
    const float mean = sum[0] * inv_dim;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      if ((thread + i * T) * V >= a.dim) continue;
      float f[V];
      widen<KX, V>(held[i], f);
#pragma unroll
      for (int j = 0; j < V; ++j) squares[0] = fmaf(f[j] - mean, f[j] - mean, squares[0]);
    }
    team_sum<T, 1>(squares, red, slot);
    const float rstd = rsqrtf(fmaf(squares[0], inv_dim, a.eps));
    if (row >= a.rows) continue;
    if (a.stats != nullptr && thread == 0) a.stats[row] = make_float2(mean, rstd);
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int at = (thread + i * T) * V;
      if (at >= a.dim) continue;
      float f[V];
      widen<KX, V>(held[i], f);
      if (plain) {
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] = (f[j] - mean) * rstd;
      } else {
        float w[V], b[V];
        gain_at<V>(gain, at, w);
        gain_at<V>(offset, at, b);
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] = fmaf((f[j] - mean) * rstd, w[j], b[j]);
      }
      store<KY, V>(a.out, row * a.dim + at, f);
    }
  }
}

// A thread's own values of a row that is on its way, in shared memory: pieces of at most 16 bytes, a piece of the
// CTA's threads side by side. Written and read by the same thread, so no barrier is needed.
template <int K, int V, int C>
struct Staged {
  static constexpr int kBytes = Raw<K, V>::kBytes;
  static constexpr int kPiece = kBytes < 4 ? 4 : kBytes < 16 ? kBytes : 16;
  static constexpr int kPieces = kBytes <= 16 ? 1 : kBytes / 16;
  static constexpr uint32_t kRow = static_cast<uint32_t>(C) * kPieces * kThreads * kPiece;  // of all threads
  __device__ __forceinline__ static uint32_t at(int i, int piece) {
    return static_cast<uint32_t>(((i * kPieces + piece) * kThreads + threadIdx.x) * kPiece);
  }
  __device__ __forceinline__ static void copy(uint8_t* stage, int i, const void* p, int64_t from) {
    const char* src = static_cast<const char*>(p) + from * (K == kF32 ? 4 : 2);
#pragma unroll
    for (int c = 0; c < kPieces; ++c) {
      if constexpr (kBytes >= 16) {
        cp_async16(smem_u32(stage + at(i, c)), src + 16 * c);
      } else if constexpr (kBytes >= 4) {
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(stage + at(i, 0))), "l"(src), "n"(kBytes) : "memory");
      } else {  // two bytes: too few for an asynchronous copy
        *reinterpret_cast<uint16_t*>(stage + at(i, 0)) = __ldg(reinterpret_cast<const uint16_t*>(src));
      }
    }
  }
  __device__ __forceinline__ static void read(const uint8_t* stage, int i, float (&f)[V]) {
    Raw<K, V> r;
    if constexpr (kBytes >= 16) {
#pragma unroll
      for (int c = 0; c < kPieces; ++c) {
        const uint4 u = *reinterpret_cast<const uint4*>(stage + at(i, c));
        r.w[4 * c] = u.x;
        r.w[4 * c + 1] = u.y;
        r.w[4 * c + 2] = u.z;
        r.w[4 * c + 3] = u.w;
      }
    } else if constexpr (kBytes == 8) {
      const uint2 u = *reinterpret_cast<const uint2*>(stage + at(i, 0));
      r.w[0] = u.x;
      r.w[1] = u.y;
    } else if constexpr (kBytes == 4) {
      r.w[0] = *reinterpret_cast<const uint32_t*>(stage + at(i, 0));
    } else {
      r.w[0] = *reinterpret_cast<const uint16_t*>(stage + at(i, 0));
    }
    widen<K, V>(r, f);
  }
};
template <int KX, int KY, int V, int C>
constexpr uint32_t stage_bytes() { return Staged<KX, V, C>::kRow + Staged<KY, V, C>::kRow; }

// kGain: the sums for dw and db are wanted (up to 64 registers a thread, and a reduction at the end). The rows that a
// team takes next are on their way, `stages` at a time (9216 x 3072 bf16: 47 us, 50 without).
template <int KX, int KY, int T, int V, int C, bool kGain>
__global__ void __launch_bounds__(kThreads) layernorm_bwd_kernel(const Args a, int stages) {
  extern __shared__ __align__(16) float gain[];  // w, padded to 4 values; then the stages, and [2][dim] joined sums in their place
  uint8_t* const ring = reinterpret_cast<uint8_t*>(gain + (a.dim + 3) / 4 * 4);
  float* const joined = reinterpret_cast<float*>(ring);
  __shared__ float red[2][kThreads / 32][2];
  using SX = Staged<KX, V, C>;
  using SY = Staged<KY, V, C>;
  constexpr uint32_t kStage = stage_bytes<KX, KY, V, C>();
  int slot = 0;
  const int thread = threadIdx.x % T;
  const int team = threadIdx.x / T;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (kThreads / T);
  const float inv_dim = 1.0f / static_cast<float>(a.dim);
  const int64_t last = T < 32 ? (a.rows + 32 / T - 1) / (32 / T) * (32 / T) : a.rows;
  const int64_t first = T < 32 ? static_cast<int64_t>(blockIdx.x) * (kThreads / T) + team : blockIdx.x + static_cast<int64_t>(team) * gridDim.x;
  auto fetch = [&](int64_t row, int stage) {
    if (row < a.rows) {
      uint8_t* to = ring + stage * kStage;
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const int at = (thread + i * T) * V;
        if (at >= a.dim) continue;
        SX::copy(to, i, a.x, row * a.dim + at);
        SY::copy(to + SX::kRow, i, a.dy, row * a.dim + at);
      }
    }
    cp_async_commit();
  };
  // two groups are always under way, so that the wait's count is the same for any number of stages
  for (int k = 0; k < 2; ++k) {
    if (k < stages - 1)
      fetch(first + k * step, k);
    else
      cp_async_commit();
  }
  stage_gain(gain, a.w, a.g_kind, a.dim, 1.0f);
  __syncthreads();
  float dw[C][V], db[C][V];
#pragma unroll
  for (int i = 0; i < C; ++i) {
#pragma unroll
    for (int j = 0; j < V; ++j) dw[i][j] = db[i][j] = 0.0f;
  }
  int stage = 0;
  for (int64_t row = first; row < last; row += step) {
    const bool live = row < a.rows;
    const float2 stats = live ? __ldg(a.stats + row) : make_float2(0.0f, 0.0f);
    const int ahead = stage == 0 ? stages - 1 : stage - 1;  // the slot that the row before has left
    fetch(row + (stages - 1) * step, ahead);
    if (stages == 3)
      cp_async_wait<2>();
    else if (stages == 2)
      cp_async_wait<1>();
    else
      cp_async_wait<0>();
    const uint8_t* held = ring + stage * kStage;
    if (++stage == stages) stage = 0;
    float sums[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int at = (thread + i * T) * V;
      if (!live || at >= a.dim) continue;
      float x[V], d[V], w[V];
      SX::read(held, i, x);
      SY::read(held + SX::kRow, i, d);
      gain_at<V>(gain, at, w);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float n = (x[j] - stats.x) * stats.y, dn = d[j] * w[j];
        sums[0] += dn;
        sums[1] = fmaf(dn, n, sums[1]);
        if constexpr (kGain) {
          dw[i][j] = fmaf(d[j], n, dw[i][j]);
          db[i][j] += d[j];
        }
      }
    }
    team_sum<T, 2>(sums, red, slot);
    if (!live || a.out == nullptr) continue;
    const float s0 = sums[0] * inv_dim, s1 = sums[1] * inv_dim;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int at = (thread + i * T) * V;
      if (at >= a.dim) continue;
      float x[V], d[V], w[V];
      SX::read(held, i, x);
      SY::read(held + SX::kRow, i, d);
      gain_at<V>(gain, at, w);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float n = (x[j] - stats.x) * stats.y;
        x[j] = stats.y * (fmaf(d[j], w[j], -s0) - n * s1);
      }
      store<KX, V>(a.out, row * a.dim + at, x);
    }
  }
  cp_async_wait<0>();
  __syncthreads();
  if constexpr (kGain) {
    float* mine = a.partial + static_cast<int64_t>(blockIdx.x) * 2 * a.dim;
    if constexpr (T == kThreads) {
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const int at = (thread + i * T) * V;
        if (at >= a.dim) continue;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          mine[at + j] = dw[i][j];
          mine[a.dim + at + j] = db[i][j];
        }
      }
    } else {
      for (int t = 0; t < kThreads / T; ++t) {  // team by team, in their order
        __syncthreads();
        if (team != t) continue;
#pragma unroll
        for (int i = 0; i < C; ++i) {
          const int at = (thread + i * T) * V;
          if (at >= a.dim) continue;
#pragma unroll
          for (int j = 0; j < V; ++j) {
            joined[at + j] = dw[i][j] + (t > 0 ? joined[at + j] : 0.0f);
            joined[a.dim + at + j] = db[i][j] + (t > 0 ? joined[a.dim + at + j] : 0.0f);
          }
        }
      }
      __syncthreads();
      for (int c = threadIdx.x; c < 2 * a.dim; c += kThreads) mine[c] = joined[c];
    }
  }
}

// Columns of the partials added in CTA order: 32 columns a CTA, eight runs of the partials that are added last.
__global__ void __launch_bounds__(256) layernorm_join_kernel(const float* __restrict__ partial, int parts, int dim,
                                                             void* dw, void* db, int kind) {
  __shared__ float runs[8][32];
  pdl_wait();
  const int lane = threadIdx.x & 31, run = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  const int each = (parts + 7) / 8, first = run * each, end = min(parts, first + each);
  float v = 0.0f;
  if (c < 2 * dim) {
#pragma unroll 8
    for (int p = first; p < end; ++p) v += __ldg(partial + static_cast<int64_t>(p) * 2 * dim + c);
  }
  runs[run][lane] = v;
  __syncthreads();
  if (run != 0 || c >= 2 * dim) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) v += runs[k][lane];
  if (c < dim) {
    if (dw != nullptr) store_from_float(dw, kind, c, v);
  } else if (db != nullptr) {
    store_from_float(db, kind, c - dim, v);
  }
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Values of a vector: 8 where rows and pointers allow 16-byte accesses, else 2 or 1.
int vector_of(bool backward, int x_kind, int y_kind, const Args& a) {
  for (int v : {8, 2}) {
    auto at = [&](const void* p, int kind) { return reinterpret_cast<uintptr_t>(p) % std::min(16, v * dtype_size(kind)) == 0; };
    if (a.dim % v == 0 && at(a.x, x_kind) && (backward ? at(a.dy, y_kind) && at(a.out, x_kind) : at(a.out, y_kind))) return v;
  }
  return 1;
}

// Threads of a row's team: the fewest that hold it with 24 values each, or 16 in narrow vectors, whose values take a
// register each (more make the gradients' sums spill; a team of 512 holds up to 32).
int team_of(int64_t dim, int v) {
  if (v == 8 && dim <= 8 * 24) return 8;
  const int held = v == 8 ? 24 : 16;
  return dim <= 32 * held ? 32 : dim <= 128 * held ? 128 : 512;
}

// CTAs: each multiprocessor's resident ones (one of the backward pass: its partial sums are then few), no more than
// there are rows (teams of several rows a warp: than fill them).
int ctas_of(int64_t rows, int team, int per_sm) {
  const int64_t asked = team < 32 ? ceil_div(rows, kThreads / team) : rows;
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(asked, static_cast<int64_t>(per_sm) * device_sm_count())));
}

// most: the dynamic shared memory that the kernel is allowed, once for each device. (Asked for by call, it would be the last
// caller's: another thread's launch between a call's request and its launch could then be refused.)
template <typename F, typename... More>
int launch_kernel(const char* what, F* kern, DeviceSetup& setup, size_t most, int ctas, size_t smem, const Args& a, cudaStream_t stream,
                  More... more) {
  const int rc = setup(what, nullptr, [&](int*) {
    return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(most));
  });
  if (rc != MOSS_OK) return rc;
  kern<<<ctas, kThreads, smem, stream>>>(a, more...);
  return check_cuda(cudaGetLastError(), what);
}

template <int KX, int KY, int T, int V, int C>
int launch(bool backward, const Args& a, cudaStream_t stream) {
  const size_t gain = static_cast<size_t>(a.dim + 3) / 4 * 4 * sizeof(float);
  if (!backward) {
    static DeviceSetup setup;
    constexpr size_t kMost = 2 * sizeof(float) * ((std::min(T * V * C, kMaxDim) + 3) / 4 * 4);
    return launch_kernel("layernorm_fwd_kernel", layernorm_fwd_kernel<KX, KY, T, V, C>, setup, kMost, ctas_of(a.rows, T, 2), 2 * gain, a, stream);
  }
  // the stages that fit one CTA a multiprocessor: three, two (f32 rows), or one (f32 rows past 8192 values)
  constexpr size_t kStage = stage_bytes<KX, KY, V, C>(), kRoom = 226 * 1024;
  const int stages = static_cast<int>(std::max<size_t>(1, std::min<size_t>(3, (kRoom - gain) / kStage)));
  const size_t joined = a.partial == nullptr || T == kThreads ? 0 : 2 * sizeof(float) * a.dim;
  const size_t smem = gain + std::max(stages * kStage, joined);
  auto run = [&](auto kern, DeviceSetup& setup) {
    return launch_kernel("layernorm_bwd_kernel", kern, setup, kRoom, ctas_of(a.rows, T, 1), smem, a, stream, stages);
  };
  static DeviceSetup without, with_gain;
  return a.partial == nullptr ? run(layernorm_bwd_kernel<KX, KY, T, V, C, false>, without)
                              : run(layernorm_bwd_kernel<KX, KY, T, V, C, true>, with_gain);
}

template <int KX, int KY>
int launch_shape(bool backward, const Args& a, cudaStream_t stream) {
  const int v = vector_of(backward, KX, KY, a), team = team_of(a.dim, v);
  if (v == 8) {
    if (team == 8) return launch<KX, KY, 8, 8, 3>(backward, a, stream);
    if (team == 32) return launch<KX, KY, 32, 8, 3>(backward, a, stream);
    if (team == 128) return launch<KX, KY, 128, 8, 3>(backward, a, stream);
    return a.dim <= 512 * 24 ? launch<KX, KY, 512, 8, 3>(backward, a, stream) : launch<KX, KY, 512, 8, 4>(backward, a, stream);
  }
  if (v == 2) {
    if (team == 32) return launch<KX, KY, 32, 2, 8>(backward, a, stream);
    if (team == 128) return launch<KX, KY, 128, 2, 8>(backward, a, stream);
    return launch<KX, KY, 512, 2, 16>(backward, a, stream);
  }
  if (team == 32) return launch<KX, KY, 32, 1, 16>(backward, a, stream);
  if (team == 128) return launch<KX, KY, 128, 1, 16>(backward, a, stream);
  return launch<KX, KY, 512, 1, 32>(backward, a, stream);
}

int launch_typed(bool backward, int x_kind, int y_kind, const Args& a, cudaStream_t stream) {
  if (x_kind == kF16) return y_kind == kF16 ? launch_shape<kF16, kF16>(backward, a, stream) : launch_shape<kF16, kF32>(backward, a, stream);
  if (x_kind == kBF16) return y_kind == kBF16 ? launch_shape<kBF16, kBF16>(backward, a, stream) : launch_shape<kBF16, kF32>(backward, a, stream);
  return launch_shape<kF32, kF32>(backward, a, stream);
}

// The type of y: torch's promotion of x and the gain.
int result_kind(int x, int g, bool gain) { return !gain || x == g ? x : kF32; }

// Rows of partial sums that a backward pass may write: narrow vectors' teams are as large or larger, so as many or more.
int most_parts(int64_t rows, int64_t dim) { return ctas_of(rows, team_of(dim, 1), 1); }

int check(int64_t rows, int64_t dim, int x_dtype, int g_dtype, bool gain) {
  if (!is_float_kind(x_dtype) || (gain && !is_float_kind(g_dtype))) return fail(MOSS_ERR_UNSUPPORTED, "unsupported dtype code");
  if (rows < 0 || dim < 1) return fail(MOSS_ERR_INVALID_ARGUMENT, "layer norm needs rows >= 0 and a width of at least 1");
  if (dim > kMaxDim) return fail(MOSS_ERR_UNSUPPORTED, "layer norm holds rows of up to %d values, not %lld", kMaxDim, static_cast<long long>(dim));
  return MOSS_OK;
}

}  // namespace
}  // namespace lnorm
}  // namespace moss

using namespace moss;

extern "C" int moss_layernorm_fwd(const void* x, int x_dtype, int64_t rows, int64_t dim, const void* weight,
                                  const void* bias, int g_dtype, float eps, void* y, float* stats,
                                  moss_stream_t stream) {
  const bool gain = weight != nullptr || bias != nullptr;
  const int rc = lnorm::check(rows, dim, x_dtype, g_dtype, gain);
  if (rc != MOSS_OK) return rc;
  if (rows == 0) return clear_ok();
  if (x == nullptr || y == nullptr) return fail(MOSS_ERR_INVALID_ARGUMENT, "null input or output pointer");
  lnorm::Args a{};
  a.x = x;
  a.w = weight;
  a.b = bias;
  a.g_kind = g_dtype;
  a.stats = reinterpret_cast<float2*>(stats);
  a.out = y;
  a.rows = rows;
  a.dim = static_cast<int>(dim);
  a.eps = eps;
  const int done = lnorm::launch_typed(false, x_dtype, lnorm::result_kind(x_dtype, g_dtype, gain), a,
                                       reinterpret_cast<cudaStream_t>(stream));
  return done != MOSS_OK ? done : clear_ok();
}

extern "C" int moss_layernorm_bwd_workspace_bytes(int64_t rows, int64_t dim, size_t* bytes) {
  if (bytes == nullptr) return fail(MOSS_ERR_INVALID_ARGUMENT, "null bytes pointer");
  *bytes = 0;
  const int rc = lnorm::check(rows, dim, kF32, kF32, false);
  if (rc != MOSS_OK) return rc;
  *bytes = static_cast<size_t>(lnorm::most_parts(rows, dim)) * 2 * dim * sizeof(float);
  return clear_ok();
}

extern "C" int moss_layernorm_bwd(const void* dy, const void* x, int x_dtype, int64_t rows, int64_t dim,
                                  const void* weight, int g_dtype, const float* stats, int gain, void* dx, void* dw,
                                  void* db, void* workspace, size_t workspace_bytes, moss_stream_t stream) {
  int rc = lnorm::check(rows, dim, x_dtype, g_dtype, gain != 0);
  if (rc != MOSS_OK) return rc;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool sums = dw != nullptr || db != nullptr;
  if (sums && gain == 0) return fail(MOSS_ERR_INVALID_ARGUMENT, "gradients of a gain that the forward pass did not have");
  if (rows == 0) {
    if (dw != nullptr) MOSS_CUDA_TRY(cudaMemsetAsync(dw, 0, dim * dtype_size(g_dtype), s));
    if (db != nullptr) MOSS_CUDA_TRY(cudaMemsetAsync(db, 0, dim * dtype_size(g_dtype), s));
    return clear_ok();
  }
  if (dy == nullptr || x == nullptr || stats == nullptr) return fail(MOSS_ERR_INVALID_ARGUMENT, "null input pointer");
  const int parts = lnorm::most_parts(rows, dim);
  if (sums && (workspace == nullptr || workspace_bytes < static_cast<size_t>(parts) * 2 * dim * sizeof(float) ||
               reinterpret_cast<uintptr_t>(workspace) % 16 != 0))
    return fail(MOSS_ERR_INVALID_ARGUMENT, "the layer norm's gradients need %zu bytes of 16-byte aligned workspace",
                static_cast<size_t>(parts) * 2 * dim * sizeof(float));
  if (dx == nullptr && !sums) return clear_ok();
  lnorm::Args a{};
  a.x = x;
  a.w = weight;
  a.g_kind = g_dtype;
  a.dy = dy;
  a.stats = reinterpret_cast<float2*>(const_cast<float*>(stats));
  a.out = dx;
  a.partial = sums ? static_cast<float*>(workspace) : nullptr;
  a.rows = rows;
  a.dim = static_cast<int>(dim);
  rc = lnorm::launch_typed(true, x_dtype, lnorm::result_kind(x_dtype, g_dtype, gain != 0), a, s);
  if (rc != MOSS_OK) return rc;
  if (sums) {
    const int y_kind = lnorm::result_kind(x_dtype, g_dtype, gain != 0);
    const int written = lnorm::ctas_of(rows, lnorm::team_of(dim, lnorm::vector_of(true, x_dtype, y_kind, a)), 1);
    rc = launch_dependent("layernorm_join_kernel", lnorm::layernorm_join_kernel,
                          dim3(static_cast<unsigned>((2 * dim + 31) / 32)), dim3(256), 0, s, a.partial, written, a.dim, dw,
                          db, g_dtype);
    if (rc != MOSS_OK) return rc;
  }
  return clear_ok();
}
