// Weight gradients of few features (an adapter's first factor) from coded activations:
//   dW[n, k] = sum over rows m of dY[m, n] * code[m, k] * 2^p[m, k / 32],  n <= 32
//
// Bound by the codes, which cross HBM once: a CTA takes 128 columns and a run of rows, whose few values of dY it
// keeps in shared memory. Two times eight warps share the columns and the rows, 16 at a time: a lane loads 8 codes of
// each of four rows (the next two sixteens are on their way meanwhile), pairs them by rows, scales the pairs exactly
// and feeds them to warp-level MMAs as they lie, column j of every lane forming one 8-column operand, against dY
// read transposed from shared memory. The tensor work is small; the MMAs spare the CUDA cores the multiply-adds. The warps'
// sums are added in warp order, the splits' in split order. 9216 x 3072 -> 32: 19 us (the codes' way through HBM 4.4): 8 of
// them to issue 310 instructions for 1024 codes of a warp; the rest are two loads ahead of 16 warps, which do not cover their
// latency, and the eight rounds of sums at the end.
#include <algorithm>

#include "codes_args.cuh"

namespace moss {
namespace codes {
namespace {

constexpr int kThreads = 512;
constexpr int kRowWarps = 8;               // warps that share the rows of 64 columns
constexpr int kEach = kRowsColumns / 2 / 8;  // columns of one lane
static_assert(kThreads == 2 * kRowWarps * 32 && kEach == 8, "two column halves, eight codes a load");
constexpr int kPitch = 40;  // 16-bit values between rows of dY: eight rows of 16 bytes meet different banks
constexpr int kSumPitch = kRowsColumns + 8;  // a feature's sums: [16 operands][8 columns], eight features in different banks
constexpr uint32_t kSumBytes = kFewFeatures * kSumPitch * 4;

__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
template <int K>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (K == kBF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The scales of two rows as one pair of 16-bit values. f16 has no 2^p below -24 or above 15 although code * 2^p may be a value of
// it (or zero): there the scale is two factors, the second of which is 1 for p in [-14, 15]. The scale of a block with an
// infinity or NaN is an infinity.
struct Scales {
  uint32_t first, second;
};
template <int K>
__device__ __forceinline__ Scales scales_of(uint32_t e0, uint32_t e1) {
  Scales s;
  if constexpr (K == kBF16) {
    s.first = (e0 << 7) | (e1 << 23);
    s.second = 0;
  } else {
    auto half_pow2 = [](int p) {  // p in [-24, 15]; 16 reads as an infinity
      return p >= -14 ? static_cast<uint32_t>(p + 15) << 10 : 1u << (p + 24);
    };
    auto first = [&](uint32_t e) { return half_pow2(e == 255u ? 16 : max(-14, min(15, static_cast<int>(e) - 127))); };
    auto second = [&](uint32_t e) {
      const int p = static_cast<int>(e) - 127;
      return half_pow2(p > 15 ? min(15, p - 15) : max(-24, min(0, p + 14)));
    };
    s.first = first(e0) | (first(e1) << 16);
    s.second = second(e0) | (second(e1) << 16);
  }
  return s;
}

// Codes c and c + 1 of two rows (words w0 and w1) as scaled pairs (row 0, row 1), for columns 2 h and 2 h + 1 of the word.
template <int K>
__device__ __forceinline__ void pairs_of(uint32_t w0, uint32_t w1, Scales s, uint32_t (&out)[4]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t both = prmt(w0, w1, h == 0 ? 0x5140u : 0x7362u);
    if constexpr (K == kBF16) {
      const __nv_bfloat162 f = *reinterpret_cast<const __nv_bfloat162*>(&s.first);
      gemm::dequant_word_bf16(both, f, out[2 * h], out[2 * h + 1]);
    } else {
      const __half2 f = *reinterpret_cast<const __half2*>(&s.first), g = *reinterpret_cast<const __half2*>(&s.second);
      gemm::dequant_word_f16(both, f, out[2 * h], out[2 * h + 1]);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        __half2 v = *reinterpret_cast<__half2*>(&out[2 * h + i]);
        v = __hmul2(v, g);
        out[2 * h + i] = *reinterpret_cast<uint32_t*>(&v);
      }
    }
  }
}

// kTiles: 16-feature tiles of dW's rows.
template <int K, int kTiles>
__global__ void __launch_bounds__(kThreads, 1) codes_rows_kernel(const Args a) {
  extern __shared__ __align__(16) uint8_t smem[];
  float* const sums = reinterpret_cast<float*>(smem);                  // [32][kSumPitch]
  uint16_t* const dy = reinterpret_cast<uint16_t*>(smem + kSumBytes);  // [rows of the split, whole 16s][kPitch]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int row_warp = warp & (kRowWarps - 1), half = warp / kRowWarps;
  const int split = blockIdx.y, row0 = split * a.per_split;
  const int rows = min(a.per_split, a.M - row0);
  const int col = blockIdx.x * kRowsColumns + (half * 8 + g) * kEach;  // this lane's columns
  const bool wanted = col < a.K;                                       // (rows are padded to whole 16s)
  const int64_t blocks = (a.K + kBlock - 1) / kBlock;
  struct Held {
    uint2 codes[4];
    uint32_t exponent[4];
  };
  // rows 2 t, 2 t + 1, 2 t + 8 and 2 t + 9 of the 16 at `at`
  const int8_t* const code_from = a.codes + static_cast<int64_t>(row0) * a.ld + col;
  const uint8_t* const exponent_from = a.exponents + row0 * blocks + col / kBlock;
  auto fetch = [&](int at, Held& h) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = at + 2 * t + (i & 1) + (i >> 1) * 8;
      h.codes[i] = make_uint2(0, 0);
      h.exponent[i] = 127;
      if (wanted && r < rows) {
        asm volatile("ld.global.nc.L1::no_allocate.v2.b32 {%0, %1}, [%2];"
                     : "=r"(h.codes[i].x), "=r"(h.codes[i].y)
                     : "l"(code_from + r * a.ld));
        h.exponent[i] = __ldg(exponent_from + r * blocks);
      }
    }
  };
  Held next[2];
  fetch(row_warp * 16, next[0]);
  fetch((row_warp + kRowWarps) * 16, next[1]);
  // dY's rows, zero past the last row and feature
  const uint16_t* from = static_cast<const uint16_t*>(a.dy) + static_cast<int64_t>(row0) * a.N;
  const int whole = (rows + 15) / 16 * 16;
  if (a.N % 8 == 0 && (reinterpret_cast<uintptr_t>(from) & 15) == 0) {
    for (int i = threadIdx.x; i < whole * 4; i += kThreads) {
      const int r = i >> 2, c = (i & 3) * 8;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (r < rows && c < a.N) v = __ldg(reinterpret_cast<const uint4*>(from + static_cast<int64_t>(r) * a.N + c));
      *reinterpret_cast<uint4*>(dy + r * kPitch + c) = v;
    }
  } else {
    for (int i = threadIdx.x; i < whole * kFewFeatures; i += kThreads) {
      const int r = i / kFewFeatures, c = i % kFewFeatures;
      dy[r * kPitch + c] = r < rows && c < a.N ? __ldg(from + static_cast<int64_t>(r) * a.N + c) : uint16_t{0};
    }
  }
  __syncthreads();

  float acc[kTiles][kEach][4];
#pragma unroll
  for (int i = 0; i < kTiles; ++i) {
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][j][e] = 0.0f;
    }
  }
  // 8 x 8 matrices of dY by rows m, transposed on the way: (n 0-7, m 0-7), (n 8-15, m 0-7), (n 0-7, m 8-15), (n 8-15, m 8-15)
  const uint32_t dy_lane = smem_u32(dy) + (((lane >> 4) * 8 + (lane & 7)) * kPitch + ((lane >> 3) & 1) * 8) * 2;
  auto take = [&](int at, Held& slot) {
    const Held held = slot;
    fetch(at + 2 * kRowWarps * 16, slot);
    uint32_t left[kTiles][4];
#pragma unroll
    for (int i = 0; i < kTiles; ++i) ldmatrix_x4_trans(dy_lane + (at * kPitch + i * 16) * 2, left[i]);
    const Scales s0 = scales_of<K>(held.exponent[0], held.exponent[1]);
    const Scales s1 = scales_of<K>(held.exponent[2], held.exponent[3]);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      uint32_t b0[4], b1[4];
      pairs_of<K>(q == 0 ? held.codes[0].x : held.codes[0].y, q == 0 ? held.codes[1].x : held.codes[1].y, s0, b0);
      pairs_of<K>(q == 0 ? held.codes[2].x : held.codes[2].y, q == 0 ? held.codes[3].x : held.codes[3].y, s1, b1);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int i = 0; i < kTiles; ++i) mma_16816<K>(acc[i][4 * q + j], left[i], b0[j], b1[j]);
      }
    }
  };
  for (int at = row_warp * 16; at < rows; at += 2 * kRowWarps * 16) {
    take(at, next[0]);
    if (at + kRowWarps * 16 < rows) take(at + kRowWarps * 16, next[1]);
  }

  // acc[i][j]: features i * 16 + g and + 8, operand columns 2 t and 2 t + 1, which are columns (2 t) * 8 + j and + 8 of the half
  for (int v = 0; v < kRowWarps; ++v) {
    __syncthreads();
    if (row_warp != v) continue;
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float2* to = reinterpret_cast<float2*>(sums + (i * 16 + g + h * 8) * kSumPitch + (half * kEach + j) * 8 + 2 * t);
          const float2 had = v > 0 ? *to : make_float2(0.0f, 0.0f);
          *to = make_float2(acc[i][j][2 * h] + had.x, acc[i][j][2 * h + 1] + had.y);
        }
      }
    }
  }
  __syncthreads();
  const int cols = min(kRowsColumns, a.K - static_cast<int>(blockIdx.x) * kRowsColumns);
  for (int i = threadIdx.x; i < a.N * kRowsColumns; i += kThreads) {
    const int n = i / kRowsColumns, c = i % kRowsColumns;
    if (c >= cols) continue;
    const float v = sums[n * kSumPitch + (c / 64 * kEach + c % kEach) * 8 + c % 64 / kEach];
    if (a.splits > 1)
      a.partial[(split * a.part_rows + n) * a.part_cols + blockIdx.x * kRowsColumns + c] = v;
    else
      store_from_float(a.out, a.out_kind, static_cast<int64_t>(n) * a.K + blockIdx.x * kRowsColumns + c, v);
  }
}

template <int K, int kTiles>
int launch_typed(const Args& a, cudaStream_t stream) {
  auto kern = codes_rows_kernel<K, kTiles>;
  static DeviceSetup setup;
  constexpr int kMost = kSumBytes + kRowsMost * kPitch * 2;
  const int rc = setup("codes_rows_kernel", nullptr, [&](int*) {
    return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost);
  });
  if (rc != MOSS_OK) return rc;
  const size_t smem = kSumBytes + static_cast<size_t>(a.per_split) * kPitch * 2;
  kern<<<dim3(static_cast<unsigned>(a.tiles_n), static_cast<unsigned>(a.splits)), kThreads, smem, stream>>>(a);
  return check_cuda(cudaGetLastError(), "codes_rows_kernel");
}

}  // namespace

int launch_rows(int kind, const Args& a, cudaStream_t stream) {
  if (a.splits > 65535) return fail(MOSS_ERR_INVALID_ARGUMENT, "too many rows of coded activations");
  if (kind == kBF16) return a.N <= 16 ? launch_typed<kBF16, 1>(a, stream) : launch_typed<kBF16, 2>(a, stream);
  return a.N <= 16 ? launch_typed<kF16, 1>(a, stream) : launch_typed<kF16, 2>(a, stream);
}

}  // namespace codes
}  // namespace moss
