// Shared declarations of the coded activations (activation_codes.cu, codes_gemm.cu, codes_rows.cu).
//
// A row of values is held as int8 codes with one power of two for each block of 32 columns:
//   x ~ code * 2^p,  p the least with max|x| <= 127 * 2^p, within [-126, cap] (cap: 9 for f16, else 121)
// The exponent byte is p + 127. A block with an infinity or NaN has the byte 255 and zero codes: its scale
// reads as an infinity, and 0 * inf as NaN. A code has 7 bits and a sign and the scale is a power of two, so a
// decoded value is exact in the type that was encoded, and in bf16 and f32 in any case: what a product reads is what the codes
// stand for. f16 has no room for codes of the other types with large p (they read as infinities there) or small p (rounded).
#pragma once

#include "common.cuh"
#include "dequant.cuh"
#include "errors.cuh"
#include "gemm_args.cuh"

namespace moss {
namespace codes {

constexpr int kBlock = 32;
constexpr int kCodeMax = 127;

// The weight gradient dW[n, k] = sum over rows m of dY[m, n] * X[m, k].
struct Args {
  int M, N, K;              // rows, features of dY, columns of X
  const void* dy;           // few features: [M, N] dense
  const int8_t* codes;      // few features: [M, K] with pitch ld
  int64_t ld;
  const uint8_t* exponents; // [M][ceil(K / 32)]
  void* out;                // [N, K] dense
  int out_kind;
  float* partial;           // splits > 1: f32 [split][part_rows][part_cols]
  int64_t part_rows, part_cols;
  int splits, per_split;    // per_split: reduction steps (GEMM) or rows (few features) of a split
  int tiles_m, tiles_n, group_m;
  StatusSink status;
};

// Features that codes_rows.cu takes: two operand tiles of 16, what its sums have registers for. 9216 x 3072, this kernel against the
// GEMM behind a decode, us: 18 and 33 for 8 features, 18 and 29 for 16, 20 and 29 for 32; from there the GEMM alone, 33 for 40,
// 30 for 48, 27 for 64.
constexpr int kFewFeatures = 32;
constexpr int kRowsColumns = 128;  // columns of X that one of its CTAs takes
constexpr int kRowsMost = 2048;    // rows of one split (its dY rows stay in shared memory)
constexpr int kStep = 128;         // reduction rows per stage of the GEMM

int launch_decode(const int8_t* codes, int64_t ld, const uint8_t* exponents, int64_t rows, int64_t cols, void* out,
                  int64_t out_ld, int kind, cudaStream_t stream);
int launch_gemm(bool pair, int kind, const CUtensorMap& ty, const CUtensorMap& tx, const Args& a, cudaStream_t stream);
int launch_rows(int kind, const Args& a, cudaStream_t stream);

}  // namespace codes
}  // namespace moss
