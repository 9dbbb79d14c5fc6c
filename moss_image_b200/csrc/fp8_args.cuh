// Shared declarations of the block-scaled fp8 linear (fp8_quantize.cu, fp8_gemm.cu, fp8_rows.cu).
//
// The product of one output value sums over blocks of 128 reduction indices:
//   y[m, c] = sum_kb  sA[kb, m] * sW[block of c, kb] * (sum over the block of codeA * codeW)
// with e4m3 codes. The inner sums run on the tensor cores (tcgen05.mma.kind::f8f6f4, f32 in
// TMEM); every block's sum is then scaled and added in f32 registers, because both scales
// change from block to block. sA is a power of two, so sA * sW is exact and a block costs one
// rounding.
#pragma once

#include "common.cuh"
#include "errors.cuh"
#include "gemm_args.cuh"

namespace moss {
namespace fp8 {

constexpr int kBlock = 128;  // reduction indices (= bytes) per block, and the weight block's side
// Blocks whose largest magnitude is below this keep the scale of this magnitude (codes near 0).
constexpr float kAmaxFloor = 7.888609052210118e-31f;  // 2^-100

struct Args {
  int M, Nc, kb;            // rows, output columns, reduction blocks
  const void* x;            // the rows themselves, for the kernel that quantises them
  int x_kind, x_wide;       // x_wide: 8 values at a time are aligned and whole
  int64_t x_cols;
  const float* row_scale;   // [kb][row_pitch]
  int64_t row_pitch;
  const float* w_scale;     // element (block of the column, reduction block) at cb * ws_col + kb * ws_red
  int ws_col, ws_red, col_blocks;
  const void* bias;         // forward only
  int bias_kind;
  void* out;                // [M, Nc] dense
  int out_kind;
  int tma_out;              // the output has a tensor map: 16-bit, rows and base on 16-byte boundaries
  // splits > 1: f32 partials, [split][M][Nc] (few rows) or [split][tile][128 columns][128 rows]
  float* partial;
  int splits, kb_per_split;
  int tiles_m, tiles_n, group_m;
  StatusSink status;
};

// The kernel a problem runs on.
struct Plan {
  enum Kind { kRows, kSingle, kPair } kind = kRows;
  int tn = 16;      // tokens per tile of the few-row kernel
  int tiles_m = 0, tiles_n = 0;
  int splits = 1, kb_per_split = 0;
};
constexpr int kRowsQuantised = 32;  // the few-row kernel quantises up to this many rows itself
Plan make_plan(int64_t m, int64_t nc, int64_t kr, int sms);

int sm_count();

// codes [m][kb * 128] (zero past k) and scale [kb][row_pitch] of the rows of x.
int launch_quantize_rows(const void* x, int dtype, int64_t m, int64_t k, uint8_t* codes, float* scale,
                         int64_t row_pitch, cudaStream_t stream);

int launch_gemm(bool dx, const Plan& plan, const CUtensorMap& ta, const CUtensorMap& tw, const CUtensorMap& to,
                const Args& a, cudaStream_t stream);
int launch_rows(bool dx, const Plan& plan, const CUtensorMap& ta, const CUtensorMap& tw, const Args& a,
                cudaStream_t stream);

__device__ __forceinline__ void umma_f8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_f8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Instruction descriptor: f32 accumulators, e4m3 operands (format code 0 of kind::f8f6f4).
__host__ __device__ constexpr uint32_t idesc_e4m3(bool a_mn_major, bool b_mn_major, int m, int n) {
  return umma_idesc_f16_ab(0u, a_mn_major, b_mn_major, m, n);
}
// Descriptor of the kk-th 32-wide step of a 128-byte-swizzled tile of 128-byte rows. K-major: a row
// holds 128 reduction indices, a step is 32 bytes along it. MN-major: a row is one reduction
// index of 128 columns, a step is 32 rows.
__device__ __forceinline__ uint64_t step_desc(uint32_t tile, int kk, bool mn_major) {
  return mn_major ? umma_desc_sw128(tile + kk * 4096, 16384, 1024) : umma_desc_sw128(tile + kk * 32, 16, 1024);
}

}  // namespace fp8
}  // namespace moss
