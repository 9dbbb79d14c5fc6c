// Shared declarations of the orthogonalised update (orthogonalize.cu, ns_gemm.cu, ns_small.cu).
#pragma once

#include "common.cuh"
#include "errors.cuh"
#include "gemm_args.cuh"

namespace moss {
namespace ns {

// One product of a Newton-Schulz step over a batch of matrices. r <= c are the sides; X is [batch][r][cp] f16
// (hi + lo), A and B [batch][r][sp] f16, with columns padded by zeros to cp, a multiple of 128, and sp, of 64.
enum Mode {
  kGram,    // A = alpha X X^T                 (upper tiles, mirrored)
  kSquare,  // B = beta A + alpha A A          (upper tiles, mirrored)
  kUpdate,  // X' = beta X + alpha B X
};
struct Args {
  int r, c, sp, cp, batch;
  int tiles_m, tiles_n, tiles;  // per matrix (tiles: those computed)
  float alpha, beta;
  const float* shifts;   // [batch]: X is held times 1 / shift. kGram: alpha times its square; last kUpdate: both times it
  const __half* add_hi;  // kSquare: A; kUpdate: X
  const __half* add_lo;  // kUpdate: X's low parts, or null
  __half* out_hi;        // A, B or X'
  __half* out_lo;        // kUpdate: X' low parts, or null
  __nv_bfloat16* result; // last kUpdate: the caller's [batch][rows][cols], else null
  int tall;              // result is the transpose [c][r]
  StatusSink status;
};
int launch_gemm(Mode mode, const __half* left, const __half* right, const Args& a, cudaStream_t stream);

// Matrices with a short side of at most kSmallSide iterate on its square in f32.
constexpr int kSmallSide = 64;
constexpr int kMaxSteps = 16;
struct Small {
  const void* g;
  int dtype;
  int64_t batch;
  int r, c, tall, steps;
  int wide, out_wide;  // 4-value reads of G's rows, 8-value writes of the result's are aligned and whole
  float coefficients[3 * kMaxSteps];
  float eps_fraction;  // eps = fraction 2^exponent
  int eps_exponent;
  __nv_bfloat16* out;
  int chunks;      // column ranges per matrix of the Gram kernel
  float* partial;  // [batch][chunks][side * side], each times 4^-exponent
  int* exponents;  // [batch][chunks]
  __half* q;       // [batch][hi, lo][side * side], scaled by a power of two
  float* factors;  // [batch][2]: X's scale in the product with Q, and the product's own
};
int small_side(int r);
int small_chunks(int64_t batch, int r, int c, int sms);
int launch_small(const Small& s, cudaStream_t stream);

int sm_count();

}  // namespace ns
}  // namespace moss
