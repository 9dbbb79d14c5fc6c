// Shared declarations of the attention to another sequence (cross_forward.cu, cross_backward.cu, cross_attention.cu).
//
// For each sequence s and query head h, with key head h / group and the keys that are allowed:
//   S = Q K^T,  P = softmax(scale S),  O = P V            (a query without keys: zeros)
//   delta = rowsum(O dO),  dS = P (dO V^T - delta),  dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO
// Exponentials are taken in base 2: P = 2^(S scale log2(e) - L), with L the row's log2 of its sum (kept for the backward
// pass; an infinity for a row without keys, which makes its P zero).
//
// Sequences are batch entries of one length, or runs of packed rows between device-side boundaries; rows behind the
// last boundary belong to one more sequence that has nothing to look at (and nobody who looks at it). What the boundaries
// hold is clamped to the tensors.
#pragma once

#include "common.cuh"
#include "dequant.cuh"
#include "errors.cuh"
#include "gemm_args.cuh"

namespace moss {
namespace cross {

constexpr int kTile = 128;  // queries, and keys, of one tile

struct Args {
  int batch, q_heads, k_heads, group, head_dim;
  int tq, tk;                // rows of each batch entry, or of the whole packed stream
  const int64_t* q_offsets;  // [batch + 1], packed; null for batch entries
  const int64_t* k_offsets;
  const uint8_t* mask;       // [batch][mask_ld] or null: non-zero where a key may be looked at
  int64_t mask_ld;
  float scale, scale_log2;
  // results, dense [rows][heads][head_dim]; rows of a batch entry b start at b * tq (b * tk)
  void* out;
  float* lse;                // [q_heads][batch * tq or packed rows]
  int64_t q_rows, k_rows;    // all rows
  // splits > 1: f32 partials of each split, joined by a second kernel
  float* partial;            // [split][q_rows][q_heads][head_dim] (forward, dq); [2][split][tail unit][128][head_dim] (dk, dv)
  float* partial_lse;        // [split][q_heads][q_rows]
  int splits;
  int tiles;                 // tiles (or pairs of tiles) of all sequences, at most
  int whole, tail;           // dk, dv: units that are not split, and those that are (the last ones)
  // backward
  const void* o;             // dense
  const void* grad;          // dense
  float* delta;              // [q_heads][q_rows]
  int* sizes;                // f16: [2][sequences][k_heads], exponents of the greatest |V|^2 and |dO|^2 (of a row's halves); else null
  void* dk;
  void* dv;
  StatusSink status;
};

struct Sequence {
  int q0, qn, k0, kn;  // rows in the tensor map's token dimension
  int entry;           // and the map's batch coordinate
  int index;
  int64_t q_row, k_row;  // the first rows among all
};

__device__ __forceinline__ int clamped(const int64_t* offsets, int i, int total) {
  return i == 0 ? 0 : static_cast<int>(max(int64_t{0}, min(static_cast<int64_t>(total), __ldg(offsets + i))));
}

__device__ __forceinline__ Sequence sequence_of(const Args& a, int s) {
  Sequence r;
  r.index = s;
  if (a.q_offsets == nullptr) {
    r.q0 = r.k0 = 0;
    r.qn = a.tq;
    r.kn = a.tk;
    r.entry = s;
    r.q_row = static_cast<int64_t>(s) * a.tq;
    r.k_row = static_cast<int64_t>(s) * a.tk;
  } else {
    r.entry = 0;
    r.q0 = clamped(a.q_offsets, s, a.tq);
    r.k0 = clamped(a.k_offsets, s, a.tk);
    // rows behind the last sequence: queries without keys, and keys without queries
    r.qn = (s < a.batch ? clamped(a.q_offsets, s + 1, a.tq) : a.tq) - r.q0;
    r.kn = (s < a.batch ? clamped(a.k_offsets, s + 1, a.tk) : a.tk) - r.k0;
    r.qn = max(r.qn, 0);
    r.kn = max(r.kn, 0);
    r.q_row = r.q0;
    r.k_row = r.k0;
  }
  return r;
}

// Tile t (of `rows` rows) of all sequences: whose it is, and which. By a whole warp. False past the last one.
template <bool kOfKeys>
__device__ __forceinline__ bool find_tile(const Args& a, int rows, int t, int& seq, int& tile) {
  if (a.q_offsets == nullptr) {
    const int each = ((kOfKeys ? a.tk : a.tq) + rows - 1) / rows;
    seq = t / each;
    tile = t - seq * each;
    return seq < a.batch;
  }
  const int lane = threadIdx.x & 31;
  const int64_t* offsets = kOfKeys ? a.k_offsets : a.q_offsets;
  const int total = kOfKeys ? a.tk : a.tq;
  int before = 0;
  for (int s0 = 0; s0 <= a.batch; s0 += 32) {
    const int s = s0 + lane;
    int n = 0;
    if (s <= a.batch) {
      const int end = s < a.batch ? clamped(offsets, s + 1, total) : total;
      n = (max(end - clamped(offsets, s, total), 0) + rows - 1) / rows;
    }
    int upto = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += v;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, before + upto > t);
    if (past != 0) {
      const int first = __ffs(past) - 1;
      seq = s0 + first;
      tile = t - before - __shfl_sync(0xffffffffu, upto - n, first);
      return true;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  return false;
}

// Which of the 128 keys from `key` on exist and are allowed, as four words. By a whole warp.
struct KeyBits {
  uint32_t w[4];
  __device__ __forceinline__ bool all() const { return (w[0] & w[1] & w[2] & w[3]) == 0xffffffffu; }
};
__device__ __forceinline__ KeyBits key_bits(const Args& a, const Sequence& s, int key, bool whole = false) {
  KeyBits b;
  if (whole || (a.mask == nullptr && s.kn - key >= kTile)) {
    b.w[0] = b.w[1] = b.w[2] = b.w[3] = 0xffffffffu;
    return b;
  }
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int k = key + i * 32 + lane;
    bool ok = k < s.kn;
    if (ok && a.mask != nullptr) ok = __ldg(a.mask + s.entry * a.mask_ld + k) != 0;
    b.w[i] = __ballot_sync(0xffffffffu, ok);
  }
  return b;
}

// Bounded wait that polls: a thread that try_wait suspends is woken some 500 cycles after the phase completes, several times
// a tile on the way from the products to the softmax and back (4096 x 512 tokens, 2 x 24 x 128: 85 us with it).
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}
__device__ __forceinline__ bool mbar_poll(uint32_t bar, uint32_t parity, volatile int* abort_flag, StatusSink status, int code) {
  if (mbar_test(bar, parity)) return true;
  const long long start = clock64();
  while (true) {
#pragma unroll 1
    for (int i = 0; i < 64; ++i)
      if (mbar_test(bar, parity)) return true;
    if (*abort_flag) return false;
    if (clock64() - start > kWaitBudgetCycles) {
      *abort_flag = 1;
      report_status(status, code);
      return false;
    }
  }
}

// Bounded wait of a whole warp, which leaves it together with one answer.
__device__ __forceinline__ bool wait_together(uint32_t bar, uint32_t parity, volatile int* abort_flag, StatusSink status,
                                              int code) {
  return __all_sync(0xffffffffu, mbar_poll(bar, parity, abort_flag, status, code)) != 0;
}
// The same for waits that are long and not on the way of a tile (loads far ahead): the warp is suspended meanwhile.
__device__ __forceinline__ bool wait_suspended(uint32_t bar, uint32_t parity, volatile int* abort_flag, StatusSink status,
                                               int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, status, code)) != 0;
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2,
                                            int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
__device__ __forceinline__ void tma_store_4d(const CUtensorMap* map, uint32_t src, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(src), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
               : "memory");
}
// The same rows into the L2 cache only.
template <int kD>
__device__ __forceinline__ void prefetch_tile(const CUtensorMap* map, int row, int head, int entry) {
#pragma unroll
  for (int c = 0; c < kD / 64; ++c)
    asm volatile("cp.async.bulk.prefetch.tensor.4d.L2.global [%0, {%1, %2, %3, %4}];" ::"l"(reinterpret_cast<uint64_t>(map)),
                 "r"(c * 64), "r"(row), "r"(head), "r"(entry)
                 : "memory");
}
// 128 rows of a head as boxes of 64 values (what lies past the head's values reads as zero).
template <int kD>
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, uint32_t bar, int row, int head, int entry) {
#pragma unroll
  for (int c = 0; c < kD / 64; ++c) tma_load_4d(dst + c * 16384, map, bar, c * 64, row, head, entry);
}

// D[tmem] (+)= A[tmem, 16-bit pairs along the columns] * B[smem desc].
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 128 x 128 products over a tile's values: A and B by rows (both reduced along the head).
template <int kD>
__device__ __forceinline__ void mma_over_head(uint32_t d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc) {
#pragma unroll
  for (int kk = 0; kk < kD / 16; ++kk) {
    const uint64_t at = ((kk >> 2) * 16384 + (kk & 3) * 32) >> 4;
    umma_f16(d, a_desc + at, b_desc + at, idesc, kk > 0 ? 1u : 0u);
  }
}
// 128 x kD products over 64 of a tile's rows: A in TMEM, B by columns.
__device__ __forceinline__ void mma_over_keys(uint32_t d, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, bool accumulate) {
#pragma unroll
  for (int kk = 0; kk < kTile / 2 / 16; ++kk)
    umma_f16_ts(d, a_tmem + kk * 8, b_desc + kk * (2048 >> 4), idesc, accumulate || kk > 0 ? 1u : 0u);
}
__device__ __forceinline__ uint64_t by_rows_desc(uint32_t tile) { return umma_desc_sw128(tile, 16, 1024); }
__device__ __forceinline__ uint64_t by_columns_desc(uint32_t tile) { return umma_desc_sw128(tile, 16384, 1024); }

// tcgen05.wait::ld that also orders the use of the loaded registers behind it.
__device__ __forceinline__ void wait_ld_of(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Pairs of f32 in one register pair: the CUDA cores take two of them an instruction.
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) {
  uint64_t p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(lo), "f"(hi));
  return p;
}
__device__ __forceinline__ void split_pair(uint64_t p, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(p)); }
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t mul_pair(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// 2^x of a pair on the CUDA cores, x up to 127 (below -126.5 zero, -inf too; NaN and +inf give NaN): 2^n p(f) with n the
// nearest whole number and p the polynomial of degree 4 that is nearest to 2^f on [-1/2, 1/2] in relative error (Remez'
// exchange), 2^-18.5 off at most. A multiprocessor's special-function units give 16 exponentials a cycle, which is what bounds
// the softmax; a part of them is computed here meanwhile. 2^n is a factor, not an addition to p's exponent bits: a sum of
// bits would turn a NaN into a number. n = -127 has the bits of zero.
__device__ __forceinline__ uint64_t exp2_pair(uint64_t x) {
  float x0, x1;
  split_pair(x, x0, x1);
  x = pair_of(max_nan(x0, -127.0f), max_nan(x1, -127.0f));
  const uint64_t t = add_pair(x, pair_of(12582912.0f, 12582912.0f));  // 1.5 * 2^23: the low bits are n
  const uint64_t n = add_pair(t, pair_of(-12582912.0f, -12582912.0f));
  const uint64_t f = fma_pair(n, pair_of(-1.0f, -1.0f), x);
  uint64_t p = fma_pair(f, pair_of(0.009570102207362652f, 0.009570102207362652f), pair_of(0.05591785907745361f, 0.05591785907745361f));
  p = fma_pair(f, p, pair_of(0.240247443318367f, 0.240247443318367f));
  p = fma_pair(f, p, pair_of(0.6931217908859253f, 0.6931217908859253f));
  p = fma_pair(f, p, pair_of(0.9999992847442627f, 0.9999992847442627f));
  float t0, t1;
  split_pair(t, t0, t1);
  return mul_pair(p, pair_of(__uint_as_float((__float_as_uint(t0) << 23) + 0x3f800000u),
                             __uint_as_float((__float_as_uint(t1) << 23) + 0x3f800000u)));
}
// Of `i`-th pairs, those that are computed that way.
__device__ __forceinline__ constexpr bool by_polynomial(int i) { return i % 3 == 2; }

// 2^(s scale - shift) of the i-th pair s of a row.
__device__ __forceinline__ uint64_t exponentials(int i, uint64_t s, uint64_t scale, uint64_t minus_shift) {
  const uint64_t x = fma_pair(s, scale, minus_shift);
  if (by_polynomial(i)) return exp2_pair(x);
  float x0, x1;
  split_pair(x, x0, x1);
  return pair_of(exp2_approx(x0), exp2_approx(x1));
}

// A warp zeroes the rows of a 128-row tile whose bit is not set (what lies there may be anything, and 0 * NaN is NaN), a row
// a lane, then makes that visible to the tensor cores.
template <int kD>
__device__ __forceinline__ void scrub_rows(uint32_t tile, const KeyBits& keep) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if ((keep.w[i] >> lane) & 1u) continue;
    const uint32_t row = tile + (i * 32 + lane) * 128;
#pragma unroll
    for (int c = 0; c < kD / 8; ++c)  // (in an order of its own in each lane: neighbouring rows meet the same banks)
      gemm::sts128(row + (c >> 3) * 16384 + (((c + lane) & 7) << 4), make_uint4(0, 0, 0, 0));
  }
  fence_proxy_async_smem();
  __syncwarp();
}

// Which key tiles have a key that may be looked at, a bit for each tile of each entry, so that the others are passed over; and
// in a second row of bits which have no other (their masks are not read again). Masks of more tiles go without.
constexpr int kMaxTileBits = 256;
__device__ __forceinline__ bool has_tile_bits(const Args& a, int key_tiles) {
  return a.mask != nullptr && static_cast<int64_t>(a.batch) * key_tiles <= kMaxTileBits;
}
// By the whole CTA, with a barrier behind it; `bits` is zero before.
__device__ __forceinline__ void find_tile_bits(const Args& a, int key_tiles, uint32_t* bits) {
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int total = a.batch * key_tiles;
  for (int i = threadIdx.x >> 5; i < total; i += warps) {
    const int entry = i / key_tiles, key = (i - entry * key_tiles) * kTile;
    bool any = false, all = true;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = key + j * 32 + lane;
      const bool seen = k < a.tk && __ldg(a.mask + entry * a.mask_ld + k) != 0;
      any = any || seen;
      all = all && seen;
    }
    any = __any_sync(0xffffffffu, any);
    all = __all_sync(0xffffffffu, all);
    if (any && lane == 0) atomicOr(bits + (i >> 5), 1u << (i & 31));
    if (all && lane == 0) atomicOr(bits + kMaxTileBits / 32 + (i >> 5), 1u << (i & 31));
  }
}
struct TileBits {
  const uint32_t* bits;  // null: every tile
  int key_tiles;
  // whether all keys of a tile may be looked at (known only with bits)
  __device__ __forceinline__ bool whole(int entry, int tile) const {
    const int i = entry * key_tiles + tile;
    return bits != nullptr && ((bits[kMaxTileBits / 32 + (i >> 5)] >> (i & 31)) & 1u) != 0;
  }
  __device__ __forceinline__ bool has(int entry, int tile) const {
    const int i = entry * key_tiles + tile;
    return bits == nullptr || ((bits[i >> 5] >> (i & 31)) & 1u) != 0;
  }
  // the first tile from t on that is taken, or end
  __device__ __forceinline__ int next(int entry, int t, int end) const {
    while (t < end && !has(entry, t)) ++t;
    return t;
  }
};

// Whether all keys that the sequence's queries look at are in one tile.
__device__ __forceinline__ bool one_tile(const TileBits& taken, const Sequence& s) {
  const int tiles = (s.kn + kTile - 1) / kTile, first = taken.next(s.entry, 0, tiles);
  return first < tiles && taken.next(s.entry, first + 1, tiles) == tiles;
}

// Whether the sequence's queries look at one key alone. P is then 1 whatever the logit is, and the gradient of the logit nothing
// times dP - delta, whose rounding would be left otherwise. By a whole warp; the mask is read again only where its tiles do not
// tell, up to the second key.
__device__ __forceinline__ bool only_key(const Args& a, const TileBits& taken, const Sequence& s, bool in_one_tile) {
  if (s.kn == 1 || a.mask == nullptr) return s.kn == 1;
  if (taken.bits != nullptr && !in_one_tile) return false;
  const int tiles = (s.kn + kTile - 1) / kTile;
  int seen = 0;
  for (int t = taken.next(s.entry, 0, tiles); t < tiles && seen < 2; t = taken.next(s.entry, t + 1, tiles)) {
    const KeyBits b = key_bits(a, s, t * kTile, taken.whole(s.entry, t));
    seen += __popc(b.w[0]) + __popc(b.w[1]) + __popc(b.w[2]) + __popc(b.w[3]);
  }
  return seen == 1;
}

// 32 consecutive values of a row, the first `count` of them (a multiple of 8).
template <int kKind>
__device__ __forceinline__ void store_row32(uint16_t* to, bool wide, int count, const float (&v)[32]) {
  uint32_t w[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) w[j] = gemm::pack2_kind<kKind>(v[2 * j], v[2 * j + 1]);
  if (wide && count >= 32) {  // 32-byte aligned
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t o[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = w[8 * h + j];
      gemm::stg256(to + 16 * h, o);
    }
    return;
  }
#pragma unroll
  for (int h = 0; h < 4; ++h)
    if (8 * h < count) *reinterpret_cast<uint4*>(to + 8 * h) = make_uint4(w[4 * h], w[4 * h + 1], w[4 * h + 2], w[4 * h + 3]);
}
__device__ __forceinline__ void store_row32_f32(float* to, int count, const float (&v)[32]) {
#pragma unroll
  for (int h = 0; h < 8; ++h)
    if (4 * h < count) *reinterpret_cast<float4*>(to + 4 * h) = make_float4(v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]);
}

// f16 has no normal values below 2^-14, and dS = P (dP - delta) is often smaller: it is held times 2^e, e as large as its bound
// allows. |dP| and |delta| are at most |dO| |V| (O is a mean of rows of V), so |dS| <= 2 |dO| |V|, with the greatest |V| of the
// keys that the sequence looks at, and for dQ a row's |dO|, for dK the greatest of the sequence's rows. The biased exponents of
// |V|^2 and of the greater half of |dO|^2 give log2 of 2 |dO| |V| within 2; the bound is placed at 2^14, so that a term keeps
// its 11 bits down to 2^-26 of it. (Where V or dO is infinite, what e is does not matter.)
__device__ __forceinline__ int lift_of(int v_exponent, int grad_exponent) {
  const int log2_product = (v_exponent + grad_exponent - 251 + 1) >> 1;  // of |dO| |V|, rounded up
  return max(-30, min(62, 13 - log2_product));
}
__device__ __forceinline__ int exponent_of(float square) { return static_cast<int>(__float_as_uint(square) >> 23); }  // not negative
// Whether other CTAs came first or not, the greatest stays.
__device__ __forceinline__ void raise_to(int* at, int value) {
  if (value > *static_cast<volatile int*>(at)) atomicMax(at, value);
}

struct Maps {
  CUtensorMap q, k, v;
  CUtensorMap grad, o;  // dense (the forward pass has no grad)
};

int launch_forward(int kind, const Maps& maps, const Args& a, cudaStream_t stream);
int launch_dq(int kind, const Maps& maps, const Args& a, cudaStream_t stream);
int launch_dkv(int kind, const Maps& maps, const Args& a, cudaStream_t stream);

}  // namespace cross
}  // namespace moss
