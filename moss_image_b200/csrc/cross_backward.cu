// Backward pass of the attention to another sequence, on the tensor cores (tcgen05.mma.kind::f16).
//
// Two kernels, each of which owns the rows it sums over, so that no gradient needs atomics or a pass in f32 over HBM:
//   dq:  a tile of 128 queries of one head against its key tiles:  S, dP = dO V^T, then dQ += dS K
//   dkv: a tile of 128 keys of one key head against the query tiles of its heads, everything turned:
//        S^T = K Q^T, dP^T = V dO^T, then dV += P^T dO and dK += dS^T Q
// Seven products for a tile pair where five would do with dQ added up across CTAs: a dQ value would be written and read in
// f32 for every key tile, 900 MB for 2 x 24 heads of 128, 4096 x 512 tokens, 140 us against 40 for the two products more.
// The dq kernel also takes delta = rowsum(O dO) on the way, which the other reads. Where all of a sequence's keys are in one tile, it
// is rowsum(P dP) instead, in f32: O's rounding is half of what dP - delta is off by there (8 keys: dQ 0.0031 off in the 2-norm,
// bf16, and 0.0024 so), and less with more keys.
//
// In both, P and dS are written over S and dP in TMEM as 16-bit pairs and feed the next product from there; a thread has a
// row and half of the columns (two warpgroups). P and dS are rounded to the inputs' type, half a step of each term (f16: times
// a power of two, see lift_of); sums are f32. The next tile's S and dP run while a tile's elements are worked on.
#include <algorithm>
#include <cmath>
#include <cstring>

#include "cross_args.cuh"

// Bound by latency: 2 x 24 heads of 128, 4096 x (308 and 512) tokens, bf16: dq 155 us, of which the start and end of its units take
// 40% (3.5 key tiles a unit), dkv 119 us (5,000 cycles a tile pair for 2,048 of products); all products of both 61 us
// at the GPU's rate.
namespace moss {
namespace cross {
namespace {

constexpr int kThreads = 384;
constexpr int kMathWarps = 8;
constexpr int kMiscRegs = 72, kMathRegs = 216;
static_assert(kMiscRegs + 2 * kMathRegs <= 3 * 168, "a larger split would wait forever");
constexpr int kHalf = kTile / 2;  // columns of one warpgroup
// f16 has no normal values below 2^-14: there dV is summed from 2^14 P (at most 2^14) and scaled back at the end.
template <int kKind>
constexpr float kLift = kKind == kF16 ? 14.0f : 0.0f;

template <int kD>
struct Shape {
  static constexpr uint32_t kTileBytes = kTile * kD * 2;
  static constexpr int kStages = kD == 128 ? 5 : 8;
  static constexpr uint32_t kDataBytes = (2 + kStages) * kTileBytes;
  static constexpr int kStats = kD == 128 ? 2 : 4;  // row sums and deltas of so many tiles
  // (shared memory starts on 1024 bytes, which is checked: there is no room for padding)
  static constexpr uint32_t kSmemBytes = kDataBytes + kStats * 2 * kTile * 4 + 512 + 2 * 2 * kTile;
  static_assert(kSmemBytes <= 227 * 1024, "tiles exceed the shared memory a CTA may use");
};
constexpr int kMaxStages = 8;

struct Barriers {
  uint64_t held_full, held_empty;                    // the tiles that stay: Q and dO, or K and V
  uint64_t empty[kMaxStages];                        // the tiles that pass, by stage
  // dkv: by stage; dq: K (and V) by number, modulo the stages (its masking warp waits for K alone, and a barrier by stage would go
  // on to a V tile unseen)
  uint64_t full[kMaxStages], v_full[kMaxStages];
  uint64_t clean[kMaxStages];                        // masked or foreign rows of the n-th tile that needs it are zero
  uint64_t stat_full[4], stat_free[4];
  uint64_t s_full, dp_full, p_ready, ds_ready;
  uint64_t acc_full, acc_free;
  uint64_t drain;
  uint32_t tile_bits[2 * kMaxTileBits / 32];
  uint32_t tmem_base;
  int abort_flag;
};
static_assert(sizeof(Barriers) <= 512, "barrier block too large");

__device__ __forceinline__ void init_barriers(Barriers* bars, int stages, int stats, int stat_writers) {
  auto init = [](uint64_t& b, uint32_t n) { mbar_init(smem_u32(&b), n); };
  init(bars->held_full, 1);
  init(bars->held_empty, 1);
  for (int s = 0; s < stages; ++s) {
    init(bars->full[s], 1);
    init(bars->v_full[s], 1);
    init(bars->empty[s], 1);
    init(bars->clean[s], 1);
  }
  for (int s = 0; s < stats; ++s) {
    init(bars->stat_full[s], stat_writers);
    init(bars->stat_free[s], kMathWarps);
  }
  init(bars->s_full, 1);
  init(bars->dp_full, 1);
  init(bars->p_ready, kMathWarps);
  init(bars->ds_ready, kMathWarps);
  init(bars->acc_full, 1);
  init(bars->acc_free, kMathWarps);
  init(bars->drain, 1);
  for (int i = 0; i < 2 * kMaxTileBits / 32; ++i) bars->tile_bits[i] = 0;
  bars->abort_flag = 0;
  fence_mbar_init();
}

// What every role of a kernel knows.
template <int kD>
struct Cta {
  using S = Shape<kD>;
  uint32_t base;  // two tiles that stay, then the ring
  Barriers* bars;
  float* stats;   // [kStats][2][128]
  uint8_t* sizes; // dq: [2][2][128], exponents of halves of |dO|^2
  volatile int* abort_flag;
  StatusSink status;
  __device__ __forceinline__ explicit Cta(uint8_t* raw, StatusSink sink) : status(sink) {
    base = smem_u32(raw);
    stats = reinterpret_cast<float*>(raw + S::kDataBytes);
    bars = reinterpret_cast<Barriers*>(raw + S::kDataBytes + S::kStats * 2 * kTile * 4);
    sizes = reinterpret_cast<uint8_t*>(bars) + 512;
    abort_flag = &bars->abort_flag;
  }
  // The tiles' swizzle wants 1024-byte addresses.
  __device__ __forceinline__ bool misplaced() const {
    if ((base & 1023u) == 0) return false;
    if (threadIdx.x == 0) report_status(status, MOSS_STATUS_TIMEOUT_LOAD);
    return true;
  }
  __device__ __forceinline__ uint32_t held(int i) const { return base + i * S::kTileBytes; }
  __device__ __forceinline__ uint32_t ring(uint32_t pos) const { return base + (2 + pos % S::kStages) * S::kTileBytes; }
  __device__ __forceinline__ bool wait(uint64_t& b, uint32_t parity, int code) const {
    return wait_together(smem_u32(&b), parity & 1u, abort_flag, status, code);
  }
  // a wait of loads that run ahead
  __device__ __forceinline__ bool wait_long(uint64_t& b, uint32_t parity) const {
    return wait_suspended(smem_u32(&b), parity & 1u, abort_flag, status, MOSS_STATUS_TIMEOUT_LOAD);
  }
  // one thread's wait
  __device__ __forceinline__ bool wait_alone(uint64_t& b, uint32_t parity) const {
    return mbar_poll(smem_u32(&b), parity & 1u, abort_flag, status, MOSS_STATUS_TIMEOUT_MMA);
  }
  __device__ __forceinline__ uint64_t& full(uint32_t pos) const { return bars->full[pos % S::kStages]; }
  __device__ __forceinline__ uint64_t& v_full(uint32_t nth) const { return bars->v_full[nth % S::kStages]; }
  __device__ __forceinline__ uint64_t& empty(uint32_t pos) const { return bars->empty[pos % S::kStages]; }
  __device__ __forceinline__ uint64_t& clean(uint32_t nth) const { return bars->clean[nth % S::kStages]; }
  __device__ __forceinline__ static uint32_t round_of(uint32_t pos) { return pos / S::kStages; }
  __device__ __forceinline__ float* stat(uint32_t nth) const { return stats + (nth % S::kStats) * 2 * kTile; }
  // One lane waits for copies that are under way when the loads end.
  __device__ __forceinline__ void landed(uint64_t& b, uint32_t parity) const {
    const long long start = clock64();
    while (!mbar_try_wait(smem_u32(&b), parity & 1u)) {
      if (clock64() - start > kWaitBudgetCycles) {
        report_status(status, MOSS_STATUS_TIMEOUT_DRAIN);
        break;
      }
    }
  }
  // The loads of a role: tiles that stay (two at once) and tiles that pass.
  struct Loads {
    uint32_t pos = 0, held = 0;
  };
  __device__ __forceinline__ bool load_held(Loads& l, const CUtensorMap* first, const CUtensorMap* second, int row, int head, int entry) const {
    if (!wait_long(bars->held_empty, l.held ^ 1u)) return false;
    if ((threadIdx.x & 31) == 0) {
      const uint32_t b = smem_u32(&bars->held_full);
      mbar_arrive_expect_tx(b, 2 * S::kTileBytes);
      load_tile<kD>(held(0), first, b, row, head, entry);
      load_tile<kD>(held(1), second, b, row, head, entry);
    }
    ++l.held;
    __syncwarp();
    return true;
  }
  __device__ __forceinline__ bool load_next(Loads& l, uint64_t& full, const CUtensorMap* map, int row, int head, int entry) const {
    if (!wait_long(empty(l.pos), round_of(l.pos) ^ 1u)) return false;
    if ((threadIdx.x & 31) == 0) {
      const uint32_t b = smem_u32(&full);
      mbar_arrive_expect_tx(b, S::kTileBytes);
      load_tile<kD>(ring(l.pos), map, b, row, head, entry);
    }
    ++l.pos;
    __syncwarp();
    return true;
  }
  __device__ __forceinline__ void finish(const Loads& l, bool by_number) const {
    if ((threadIdx.x & 31) != 0) return;
    const uint32_t count = by_number ? l.pos / 2 : l.pos;
    for (uint32_t p = count > S::kStages ? count - S::kStages : 0; p < count; ++p) {
      landed(full(p), round_of(p));
      if (by_number) landed(v_full(p), round_of(p));
    }
    if (l.held > 0) landed(bars->held_full, l.held - 1);
  }
  __device__ __forceinline__ void drain(bool issued) const {
    if ((threadIdx.x & 31) == 0 && issued) {
      umma_commit(smem_u32(&bars->drain));
      landed(bars->drain, 0);
    }
    __syncwarp();
  }
};

// Shared prologue: barriers, the mask's tiles, TMEM.
template <int kD>
__device__ __forceinline__ TileBits begin(const Cta<kD>& cta, const Args& args, bool masked, int stat_writers) {
  if (threadIdx.x == 0) init_barriers(cta.bars, Shape<kD>::kStages, Shape<kD>::kStats, stat_writers);
  const int key_tiles = (args.tk + kTile - 1) / kTile;
  const bool use_bits = masked && has_tile_bits(args, key_tiles);
  if (use_bits) {
    __syncthreads();
    find_tile_bits(args, key_tiles, cta.bars->tile_bits);
  }
  if ((threadIdx.x >> 5) == 1) {
    tmem_alloc(smem_u32(&cta.bars->tmem_base), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  return TileBits{use_bits ? cta.bars->tile_bits : nullptr, key_tiles};
}
template <int kD>
__device__ __forceinline__ void end(uint32_t tmem) {
  tc_fence_before();
  __syncthreads();
  if ((threadIdx.x >> 5) == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// 64 consecutive columns of a thread's row.
__device__ __forceinline__ void load64(uint32_t tmem, uint32_t (&r)[2][32]) {
  tmem_ld_32x32b_x32(tmem, r[0]);
  tmem_ld_32x32b_x32(tmem + 32, r[1]);
  wait_ld_of(r[0]);
  wait_ld_of(r[1]);
}
// 64 values of a thread's row as 16-bit pairs.
template <int kKind>
__device__ __forceinline__ void store64(uint32_t tmem, const float (&v)[64]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t w[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) w[j] = gemm::pack2_kind<kKind>(v[32 * h + 2 * j], v[32 * h + 2 * j + 1]);
    tmem_st_32x32b_x16(tmem + 16 * h, w);
  }
}
// A in TMEM as the two warpgroups leave it: rows 0-63 of the reduction's 128 as pairs from `a`, 64-127 from `a` + 64.
__device__ __forceinline__ void mma_over_halves(uint32_t d, uint32_t a, uint64_t b_desc, uint32_t idesc, bool accumulate) {
#pragma unroll
  for (int kk = 0; kk < kTile / 16; ++kk)
    umma_f16_ts(d, a + (kk >> 2) * kHalf + (kk & 3) * 8, b_desc + kk * (2048 >> 4), idesc, accumulate || kk > 0 ? 1u : 0u);
}

// ---------------------------------------------------------------- dq
struct QueryUnit {
  Sequence s;
  int head, split, row, first, end;
};
__device__ __forceinline__ bool locate(const Args& a, const TileBits& taken, int u, QueryUnit& unit) {
  const int t = u % a.tiles, rest = u / a.tiles;
  unit.split = rest % a.splits;
  unit.head = rest / a.splits;
  int seq, tile;
  if (!find_tile<false>(a, kTile, t, seq, tile)) return false;
  unit.s = sequence_of(a, seq);
  if (seq >= a.batch) unit.s.kn = 0;
  unit.row = tile * kTile;
  const int keys = (unit.s.kn + kTile - 1) / kTile, each = (keys + a.splits - 1) / a.splits;
  unit.end = min(keys, (unit.split + 1) * each);
  unit.first = taken.next(unit.s.entry, min(keys, unit.split * each), unit.end);
  return true;
}

// 16 values of a row of O or dO, the first `count` of them (a multiple of 8).
template <int kKind>
__device__ __forceinline__ void load_row16(const uint16_t* p, int count, float (&v)[16]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float f[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (8 * h < count) load8<kKind>(p, 8 * h, 8, true, f);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[8 * h + j] = f[j];
  }
}

template <int kKind, int kD, bool kMask>
__global__ void __launch_bounds__(kThreads, 1)
    cross_dq_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                    const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_grad,
                    const __grid_constant__ CUtensorMap tm_o, const Args args) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const Cta<kD> cta(smem_raw, args.status);
  if (cta.misplaced()) return;
  Barriers* const bars = cta.bars;
  const TileBits taken = begin<kD>(cta, args, kMask, kMathWarps);
  const uint32_t tmem = bars->tmem_base;  // S (and dS) of two key tiles, dP, dQ
  const uint32_t dp_tmem = tmem + 2 * kTile, dq_tmem = tmem + 3 * kTile;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int num_units = args.tiles * args.splits * args.q_heads;
  bool ok = true;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kMiscRegs));
    if (warp == 0) {
      // ---------------------------------------------------------------- loads: K and V of a tile one after the other
      typename Cta<kD>::Loads l;
      if (lane == 0) {
        tma_prefetch_desc(&tm_q);
        tma_prefetch_desc(&tm_k);
        tma_prefetch_desc(&tm_v);
        tma_prefetch_desc(&tm_grad);
      }
      for (int u = blockIdx.x; u < num_units && ok; u += gridDim.x) {
        QueryUnit w;
        if (!locate(args, taken, u, w) || w.first >= w.end) continue;
        const int k_head = w.head / args.group;
        ok = cta.load_held(l, &tm_q, &tm_grad, w.s.q0 + w.row, w.head, w.s.entry);
        // all CTAs ask for their next tiles at about the same time: those are on their way to L2 a unit ahead
        QueryUnit ahead;
        if (ok && u + static_cast<int>(gridDim.x) < num_units && locate(args, taken, u + gridDim.x, ahead) && lane == 0) {
          prefetch_tile<kD>(&tm_q, ahead.s.q0 + ahead.row, ahead.head, ahead.s.entry);
          prefetch_tile<kD>(&tm_grad, ahead.s.q0 + ahead.row, ahead.head, ahead.s.entry);
          prefetch_tile<kD>(&tm_o, ahead.s.q0 + ahead.row, ahead.head, ahead.s.entry);
        }
        __syncwarp();
        for (int t = w.first; t < w.end && ok; t = taken.next(w.s.entry, t + 1, w.end)) {
          const int row = w.s.k0 + t * kTile;
          ok = cta.load_next(l, cta.full(l.pos / 2), &tm_k, row, k_head, w.s.entry) &&
               cta.load_next(l, cta.v_full(l.pos / 2), &tm_v, row, k_head, w.s.entry);
        }
      }
      cta.finish(l, true);
    } else if (warp == 1) {
      // ---------------------------------------------------------------- MMAs
      constexpr uint32_t kFormat = kKind == kBF16 ? 1u : 0u;
      constexpr uint32_t s_idesc = umma_idesc_f16(kFormat, false, kTile, kTile);
      constexpr uint32_t d_idesc = umma_idesc_f16(kFormat, true, kTile, kD);
      uint32_t pos = 0, held = 0, steps = 0, accs = 0;
      bool issued = false;
      for (int u = blockIdx.x; u < num_units && ok; u += gridDim.x) {
        QueryUnit w;
        if (!locate(args, taken, u, w) || w.first >= w.end) continue;
        int n = 0;
        for (int t = w.first; t < w.end; t = taken.next(w.s.entry, t + 1, w.end)) ++n;
        if (elect_one()) {  // one thread waits and issues for the whole unit
          // key tile i of the unit: K at ring position pos + 2 i, V behind it
          auto scores = [&](int i) {
            const uint32_t p = pos + 2 * i;
            ok = ok && cta.wait_alone(kMask ? cta.clean(p / 2) : cta.full(p / 2), cta.round_of(p / 2));
            if (!ok) return;
            tc_fence_after();
            mma_over_head<kD>(tmem + (i & 1) * kTile, by_rows_desc(cta.held(0)), by_rows_desc(cta.ring(p)), s_idesc);
          };
          auto grads = [&](int i) {
            const uint32_t p = pos + 2 * i + 1;
            ok = ok && cta.wait_alone(cta.v_full(p / 2), cta.round_of(p / 2));
            if (!ok) return;
            tc_fence_after();
            mma_over_head<kD>(dp_tmem, by_rows_desc(cta.held(1)), by_rows_desc(cta.ring(p)), s_idesc);
            umma_commit(smem_u32(&bars->dp_full));  // (S of this tile is done then too)
            umma_commit(smem_u32(&cta.empty(p)));
            if (i + 1 == n) umma_commit(smem_u32(&bars->held_empty));
          };
          ok = cta.wait_alone(bars->held_full, held);
          scores(0);
          grads(0);
          if (n > 1) scores(1);
          for (int i = 0; i < n && ok; ++i) {
            if (!(ok = cta.wait_alone(bars->ds_ready, steps + i))) break;
            if (i + 1 < n) grads(i + 1);
            if (i == 0) ok = ok && cta.wait_alone(bars->acc_free, accs ^ 1u);
            if (!ok) break;
            tc_fence_after();
            const uint32_t p = pos + 2 * i;
            mma_over_halves(dq_tmem, tmem + (i & 1) * kTile, by_columns_desc(cta.ring(p)), d_idesc, i > 0);
            umma_commit(smem_u32(&cta.empty(p)));
            if (i + 1 == n) umma_commit(smem_u32(&bars->acc_full));
            if (i + 2 < n) scores(i + 2);
          }
        }
        ok = __all_sync(0xffffffffu, ok) != 0;
        issued = true;
        ++held;
        ++accs;
        steps += n;
        pos += 2 * n;
      }
      cta.drain(issued);
    } else if (warp == 2) {
      // ---------------------------------------------------------------- masked rows of K
      if (kMask) {
        uint32_t pos = 0;
        for (int u = blockIdx.x; u < num_units && ok; u += gridDim.x) {
          QueryUnit w;
          if (!locate(args, taken, u, w) || w.first >= w.end) continue;
          for (int t = w.first; t < w.end; t = taken.next(w.s.entry, t + 1, w.end), pos += 2) {
            const KeyBits keep = key_bits(args, w.s, t * kTile, taken.whole(w.s.entry, t));
            ok = cta.wait(cta.full(pos / 2), cta.round_of(pos / 2), MOSS_STATUS_TIMEOUT_LOAD);
            if (!ok) break;
            if (!keep.all()) scrub_rows<kD>(cta.ring(pos), keep);
            if (lane == 0) mbar_arrive(smem_u32(&cta.clean(pos / 2)));
          }
        }
      }
    }
  } else {
    // ---------------------------------------------------------------- P and dS, and the output
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kMathRegs));
    const int half = (warp - 4) >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const bool wide = args.head_dim % 16 == 0 && (reinterpret_cast<uintptr_t>(args.out) & 31) == 0;
    uint32_t steps = 0, accs = 0, nth = 0;
    for (int u = blockIdx.x; u < num_units && ok; u += gridDim.x) {
      QueryUnit w;
      if (!locate(args, taken, u, w)) continue;
      // delta = rowsum(O dO): each warpgroup takes half of the head, and they meet in shared memory (in a slot that was last
      // read two units ago, before the meeting of the unit between)
      const int at = w.row + row;
      const bool live = at < w.s.qn;
      const int64_t q_row = w.s.q_row + at;
      float lse = INFINITY, delta = 0.0f, square = 0.0f;
      if (live) {
        lse = __ldg(args.lse + w.head * args.q_rows + q_row);
        const int64_t from = (q_row * args.q_heads + w.head) * args.head_dim + half * (kD / 2);
        const uint16_t* o = static_cast<const uint16_t*>(args.o) + from;
        const uint16_t* g = static_cast<const uint16_t*>(args.grad) + from;
        const int count = args.head_dim - half * (kD / 2);
#pragma unroll
        for (int c = 0; c < kD / 32; ++c) {
          float x[16], y[16];
          load_row16<kKind>(o + c * 16, count - c * 16, x);
          load_row16<kKind>(g + c * 16, count - c * 16, y);
#pragma unroll
          for (int j = 0; j < 16; ++j) delta = fmaf(x[j], y[j], delta);
          if constexpr (kKind == kF16) {
#pragma unroll
            for (int j = 0; j < 16; ++j) square = fmaf(y[j], y[j], square);
          }
        }
      }
      // the sum of both warpgroups' halves of a row's value
      auto meet = [&](float value) {
        float* const slot = cta.stats + (nth & 1u) * 2 * kTile;
        slot[half * kTile + row] = value;
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bars->stat_full[nth & 1u]));
        ok = cta.wait(bars->stat_full[nth & 1u], nth >> 1, MOSS_STATUS_TIMEOUT_EPILOGUE);
        ++nth;
        return slot[row] + slot[kTile + row];
      };
      const uint8_t* const sizes = cta.sizes + (nth & 1u) * 2 * kTile;
      if constexpr (kKind == kF16) cta.sizes[(nth & 1u) * 2 * kTile + half * kTile + row] = static_cast<uint8_t>(exponent_of(fabsf(square)));
      delta = meet(delta);
      if (!ok) break;
      const bool single = one_tile(taken, w.s);
      if (live && half == 0 && w.split == 0 && !single) args.delta[w.head * args.q_rows + q_row] = delta;
      int lift = 0;
      if constexpr (kKind == kF16) {
        const int size = max(sizes[row], sizes[kTile + row]), at_sizes = w.s.index * args.k_heads + w.head / args.group;
        lift = lift_of(args.sizes[at_sizes], size);
        const int most = __reduce_max_sync(0xffffffffu, size);
        if (half == 0 && w.split == 0 && lane == 0) raise_to(args.sizes + (args.batch + 1) * args.k_heads + at_sizes, most);
      }
      const bool alone = w.first < w.end && only_key(args, taken, w.s, single);
      const float raised = kKind == kF16 ? pow2(lift) : 1.0f;
      int i = 0;
      for (int t = w.first; t < w.end; t = taken.next(w.s.entry, t + 1, w.end), ++i) {
        KeyBits keep;
        if constexpr (kMask) keep = key_bits(args, w.s, t * kTile, taken.whole(w.s.entry, t));
        const int keys = w.s.kn - t * kTile - half * kHalf;
        ok = cta.wait(bars->dp_full, steps++, MOSS_STATUS_TIMEOUT_EPILOGUE);
        if (!ok) break;
        tc_fence_after();
        const uint32_t s_tmem = tmem + (i & 1) * kTile + half * kHalf + lanes;
        const uint64_t scale2 = pair_of(args.scale_log2, args.scale_log2), minus_lse = pair_of(-lse, -lse), raise2 = pair_of(raised, raised);
        if (single) {  // all of the row's keys are here: delta = sum P dP in f32
          uint64_t sum2 = 0;
#pragma unroll 1
          for (int c = 0; c < 2; ++c) {
            const int count = keys - 32 * c;
            const uint32_t k = kMask ? (half == 0 ? (c == 0 ? keep.w[0] : keep.w[1]) : c == 0 ? keep.w[2] : keep.w[3])
                                     : count >= 32 ? 0xffffffffu : count <= 0 ? 0u : (1u << count) - 1u;
            uint32_t x[32], y[32];
            tmem_ld_32x32b_x32(s_tmem + 32 * c, x);
            tmem_ld_32x32b_x32(dp_tmem + half * kHalf + lanes + 32 * c, y);
            wait_ld_of(x);
            wait_ld_of(y);
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              float p0, p1;
              split_pair(exponentials(j / 2, pair_of(__uint_as_float(x[j]), __uint_as_float(x[j + 1])), scale2, minus_lse), p0, p1);
              const bool in0 = ((k >> j) & 1u) != 0, in1 = ((k >> j) & 2u) != 0;
              sum2 = fma_pair(pair_of(in0 ? p0 : 0.0f, in1 ? p1 : 0.0f),
                              pair_of(in0 ? __uint_as_float(y[j]) : 0.0f, in1 ? __uint_as_float(y[j + 1]) : 0.0f), sum2);
            }
          }
          float sum0, sum1;
          split_pair(sum2, sum0, sum1);
          delta = meet(sum0 + sum1);
          if (!ok) break;
          if (live && half == 0) args.delta[w.head * args.q_rows + q_row] = delta;
        }
        uint32_t s[2][32], g[2][32];
        load64(s_tmem, s);
        load64(dp_tmem + half * kHalf + lanes, g);
        float v[64];
        // (a row without keys has lse = inf, which makes its exponentials zero)
        const uint64_t minus_delta = pair_of(-delta * raised, -delta * raised);
#pragma unroll
        for (int j = 0; j < 64; j += 2) {
          const uint64_t p = exponentials(j / 2, pair_of(__uint_as_float(s[j >> 5][j & 31]), __uint_as_float(s[j >> 5][(j & 31) + 1])),
                                                 scale2, minus_lse);
          const uint64_t dp = pair_of(__uint_as_float(g[j >> 5][j & 31]), __uint_as_float(g[j >> 5][(j & 31) + 1]));
          const uint64_t d = kKind == kF16 ? fma_pair(dp, raise2, minus_delta) : add_pair(dp, minus_delta);
          split_pair(mul_pair(p, d), v[j], v[j + 1]);
        }
        if constexpr (kMask) {
          if (!keep.all()) {
            const uint32_t k0 = half == 0 ? keep.w[0] : keep.w[2], k1 = half == 0 ? keep.w[1] : keep.w[3];
#pragma unroll
            for (int j = 0; j < 64; ++j)
              if ((((j < 32 ? k0 : k1) >> (j & 31)) & 1u) == 0) v[j] = 0.0f;
          }
        } else if (keys < kHalf) {
#pragma unroll
          for (int j = 0; j < 64; ++j)
            if (j >= keys) v[j] = 0.0f;
        }
        if (alone) {  // (NaN stays)
#pragma unroll
          for (int j = 0; j < 64; ++j) v[j] *= 0.0f;
        }
        store64<kKind>(s_tmem, v);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bars->ds_ready));
      }
      if (!ok) break;
      const bool any_keys = w.first < w.end;
      if (any_keys) {
        ok = cta.wait(bars->acc_full, accs++, MOSS_STATUS_TIMEOUT_EPILOGUE);
        if (!ok) break;
        tc_fence_after();
      }
      const int64_t to = (q_row * args.q_heads + w.head) * args.head_dim;
      const float factor = kKind == kF16 ? args.scale * pow2(-lift) : args.scale;
#pragma unroll
      for (int c = 0; c < kD / 64; ++c) {  // this warpgroup's half of the head
        const int col = half * (kD / 2) + c * 32;
        uint32_t o[32];
        float v[32];
        __syncwarp();
        if (any_keys) {
          tmem_ld_32x32b_x32(dq_tmem + col + lanes, o);
          wait_ld_of(o);
          if (c == kD / 64 - 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&bars->acc_free));
          }
        }
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = any_keys ? __uint_as_float(o[j]) * factor : 0.0f;
        const int count = args.head_dim - col;
        if (live && count > 0) {
          if (args.splits > 1)
            store_row32_f32(args.partial + w.split * args.q_rows * args.q_heads * args.head_dim + to + col, count, v);
          else
            store_row32<kKind>(static_cast<uint16_t*>(args.out) + to + col, wide, count, v);
        }
      }
    }
  }
  end<kD>(tmem);
}

// ---------------------------------------------------------------- dk and dv
struct KeyUnit {
  Sequence s;
  int head, split, tail, row, first, end, q_tiles;  // head: of the keys; first to end: tiles of the group's heads, one head after another
};
// The units of the last round, which would leave multiprocessors idle, are split over their queries: tail says which one it is
// (-1: a whole unit).
__device__ __forceinline__ bool locate(const Args& a, const TileBits& taken, int u, KeyUnit& unit) {
  int splits = 1, of = u;
  unit.split = 0;
  unit.tail = -1;
  if (u >= a.whole) {
    splits = a.splits;
    unit.tail = (u - a.whole) / splits;
    unit.split = u - a.whole - unit.tail * splits;
    of = a.whole + unit.tail;
  }
  const int t = of % a.tiles;
  unit.head = of / a.tiles;
  int seq, tile;
  if (!find_tile<true>(a, kTile, t, seq, tile)) return false;
  unit.s = sequence_of(a, seq);
  if (seq >= a.batch) unit.s.qn = 0;
  unit.row = tile * kTile;
  unit.q_tiles = (unit.s.qn + kTile - 1) / kTile;
  const int all = taken.has(unit.s.entry, tile) ? unit.q_tiles * a.group : 0, each = (all + splits - 1) / splits;
  unit.first = min(all, unit.split * each);
  unit.end = min(all, unit.first + each);
  return true;
}

template <int kKind, int kD, bool kPacked>
__global__ void __launch_bounds__(kThreads, 1)
    cross_dkv_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                     const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_grad,
                     const __grid_constant__ CUtensorMap tm_o, const Args args) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const Cta<kD> cta(smem_raw, args.status);
  if (cta.misplaced()) return;
  Barriers* const bars = cta.bars;
  const TileBits taken = begin<kD>(cta, args, !kPacked, 1);
  const uint32_t tmem = bars->tmem_base;  // S^T (and P^T), dP^T (and dS^T), dV, dK
  const uint32_t dp_tmem = tmem + kTile, dv_tmem = tmem + 2 * kTile, dk_tmem = tmem + 3 * kTile;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int num_units = args.whole + args.tail * args.splits;
  bool ok = true;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kMiscRegs));
    if (warp == 0) {
      // ---------------------------------------------------------------- loads: Q and dO of a tile one after the other
      typename Cta<kD>::Loads l;
      if (lane == 0) {
        tma_prefetch_desc(&tm_q);
        tma_prefetch_desc(&tm_k);
        tma_prefetch_desc(&tm_v);
        tma_prefetch_desc(&tm_grad);
      }
      for (int u = blockIdx.x; u < num_units && ok; u += gridDim.x) {
        KeyUnit w;
        if (!locate(args, taken, u, w) || w.first == w.end) continue;
        ok = cta.load_held(l, &tm_k, &tm_v, w.s.k0 + w.row, w.head, w.s.entry);
        for (int i = w.first; i < w.end && ok; ++i) {
          const int g = i / w.q_tiles, row = w.s.q0 + (i - g * w.q_tiles) * kTile, head = w.head * args.group + g;
          ok = cta.load_next(l, cta.full(l.pos), &tm_q, row, head, w.s.entry) &&
               cta.load_next(l, cta.full(l.pos), &tm_grad, row, head, w.s.entry);
        }
      }
      cta.finish(l, false);
    } else if (warp == 1) {
      // ---------------------------------------------------------------- MMAs
      constexpr uint32_t kFormat = kKind == kBF16 ? 1u : 0u;
      constexpr uint32_t s_idesc = umma_idesc_f16(kFormat, false, kTile, kTile);
      constexpr uint32_t d_idesc = umma_idesc_f16(kFormat, true, kTile, kD);
      uint32_t pos = 0, held = 0, steps = 0, accs = 0;
      bool issued = false;
      for (int u = blockIdx.x; u < num_units && ok; u += gridDim.x) {
        KeyUnit w;
        if (!locate(args, taken, u, w) || w.first == w.end) continue;
        const int n = w.end - w.first;
        if (elect_one()) {  // one thread waits and issues for the whole unit
          // query tile i of the unit: Q at ring position pos + 2 i, dO behind it
          auto product = [&](int i, int which) {  // 0: S^T = K Q^T, 1: dP^T = V dO^T
            const uint32_t p = pos + 2 * i + which;
            ok = ok && (kPacked ? cta.wait_alone(cta.clean(p), cta.round_of(p)) : cta.wait_alone(cta.full(p), cta.round_of(p)));
            if (!ok) return;
            tc_fence_after();
            mma_over_head<kD>(tmem + which * kTile, by_rows_desc(cta.held(which)), by_rows_desc(cta.ring(p)), s_idesc);
            umma_commit(which == 0 ? smem_u32(&bars->s_full) : smem_u32(&bars->dp_full));
            if (which == 1 && i + 1 == n) umma_commit(smem_u32(&bars->held_empty));
          };
          ok = cta.wait_alone(bars->held_full, held);
          product(0, 0);
          product(0, 1);
          for (int i = 0; i < n && ok; ++i) {
            const uint32_t p = pos + 2 * i;
            ok = cta.wait_alone(bars->p_ready, steps + i) && (i > 0 || cta.wait_alone(bars->acc_free, accs ^ 1u));
            if (!ok) break;
            tc_fence_after();
            mma_over_halves(dv_tmem, tmem, by_columns_desc(cta.ring(p + 1)), d_idesc, i > 0);
            umma_commit(smem_u32(&cta.empty(p + 1)));
            if (i + 1 < n) product(i + 1, 0);
            ok = ok && cta.wait_alone(bars->ds_ready, steps + i);
            if (!ok) break;
            tc_fence_after();
            mma_over_halves(dk_tmem, dp_tmem, by_columns_desc(cta.ring(p)), d_idesc, i > 0);
            umma_commit(smem_u32(&cta.empty(p)));
            if (i + 1 == n) umma_commit(smem_u32(&bars->acc_full));
            if (i + 1 < n) product(i + 1, 1);
          }
        }
        ok = __all_sync(0xffffffffu, ok) != 0;
        issued = true;
        ++held;
        ++accs;
        steps += n;
        pos += 2 * n;
      }
      cta.drain(issued);
    } else if (warp == 2) {
      // ---------------------------------------------------------------- rows of the next sequence in a last tile of Q and dO
      if (kPacked) {
        uint32_t pos = 0;
        for (int u = blockIdx.x; u < num_units && ok; u += gridDim.x) {
          KeyUnit w;
          if (!locate(args, taken, u, w) || w.first == w.end) continue;
          for (int i = w.first; i < w.end && ok; ++i) {
            const int rows = w.s.qn - i % w.q_tiles * kTile;
            KeyBits keep;
#pragma unroll
            for (int j = 0; j < 4; ++j) keep.w[j] = rows >= 32 * j + 32 ? 0xffffffffu : rows <= 32 * j ? 0u : (1u << (rows - 32 * j)) - 1u;
            for (int which = 0; which < 2 && ok; ++which, ++pos) {
              ok = cta.wait(cta.full(pos), cta.round_of(pos), MOSS_STATUS_TIMEOUT_LOAD);
              if (!ok) break;
              if (rows < kTile) scrub_rows<kD>(cta.ring(pos), keep);
              if (lane == 0) mbar_arrive(smem_u32(&cta.clean(pos)));
            }
          }
        }
      }
    } else {
      // ---------------------------------------------------------------- row sums and deltas of the query tiles
      uint32_t nth = 0;
      for (int u = blockIdx.x; u < num_units && ok; u += gridDim.x) {
        KeyUnit w;
        if (!locate(args, taken, u, w) || w.first == w.end) continue;
        for (int i = w.first; i < w.end; ++i, ++nth) {
          const int g = i / w.q_tiles, row = (i - g * w.q_tiles) * kTile;
          const int64_t at = (w.head * args.group + g) * args.q_rows + w.s.q_row + row;
          float l[4], d[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int r = j * 32 + lane;
            const bool live = row + r < w.s.qn;
            l[j] = live ? kLift<kKind> - __ldg(args.lse + at + r) : -INFINITY;
            d[j] = live ? -__ldg(args.delta + at + r) : 0.0f;
          }
          ok = cta.wait(bars->stat_free[nth % Shape<kD>::kStats], (nth / Shape<kD>::kStats) ^ 1u, MOSS_STATUS_TIMEOUT_LOAD);
          if (!ok) break;
          float* to = cta.stat(nth);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            to[j * 32 + lane] = l[j];
            to[kTile + j * 32 + lane] = d[j];
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&bars->stat_full[nth % Shape<kD>::kStats]));
        }
      }
    }
  } else {
    // ---------------------------------------------------------------- P^T and dS^T, and the output
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kMathRegs));
    const int half = (warp - 4) >> 2;
    const int row = (warp & 3) * 32 + lane;  // of the keys
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    void* const result = half == 0 ? args.dv : args.dk;
    const bool wide = args.head_dim % 16 == 0 && (reinterpret_cast<uintptr_t>(result) & 31) == 0;
    uint32_t steps = 0, accs = 0;
    const uint64_t scale2 = pair_of(args.scale_log2, args.scale_log2);
    for (int u = blockIdx.x; u < num_units && ok; u += gridDim.x) {
      KeyUnit w;
      if (!locate(args, taken, u, w)) continue;
      const int key = w.row + row;
      bool seen = key < w.s.kn;
      if (seen && args.mask != nullptr) seen = __ldg(args.mask + w.s.entry * args.mask_ld + key) != 0;
      const bool alone = w.first < w.end && only_key(args, taken, w.s, one_tile(taken, w.s));
      int lift = 0;
      if constexpr (kKind == kF16) {
        const int* const sizes = args.sizes + w.s.index * args.k_heads + w.head;
        lift = lift_of(__ldg(sizes), __ldg(sizes + (args.batch + 1) * args.k_heads));
      }
      const float of_p = pow2(lift - static_cast<int>(kLift<kKind>));  // what P, which is lifted for dV, takes to be lifted for dS
      for (int i = w.first; i < w.end; ++i, ++steps) {
        const int rows = w.s.qn - i % w.q_tiles * kTile - half * kHalf;  // query columns of this thread that exist
        const uint32_t slot = steps % Shape<kD>::kStats;
        ok = cta.wait(bars->stat_full[slot], steps / Shape<kD>::kStats, MOSS_STATUS_TIMEOUT_EPILOGUE) &&
             cta.wait(bars->s_full, steps, MOSS_STATUS_TIMEOUT_EPILOGUE);
        if (!ok) break;
        tc_fence_after();
        const float* lse = cta.stat(steps) + half * kHalf;
        uint32_t r[2][32];
        float v[64];
        load64(tmem + half * kHalf + lanes, r);
#pragma unroll
        for (int j = 0; j < 64; j += 4) {  // (the sums are kept negated, and lifted)
          const float4 l = *reinterpret_cast<const float4*>(lse + j);
          const uint64_t lo = exponentials(j / 2, pair_of(__uint_as_float(r[j >> 5][j & 31]), __uint_as_float(r[j >> 5][(j & 31) + 1])),
                                                  scale2, pair_of(l.x, l.y));
          const uint64_t hi = exponentials(j / 2 + 1, pair_of(__uint_as_float(r[j >> 5][(j & 31) + 2]), __uint_as_float(r[j >> 5][(j & 31) + 3])),
                                                  scale2, pair_of(l.z, l.w));
          split_pair(lo, v[j], v[j + 1]);
          split_pair(hi, v[j + 2], v[j + 3]);
        }
        if (!seen || rows < kHalf) {
#pragma unroll
          for (int j = 0; j < 64; ++j)
            if (!seen || j >= rows) v[j] = 0.0f;
        }
        __syncwarp();
        store64<kKind>(tmem + half * kHalf + lanes, v);
        if constexpr (kKind == kF16) {
#pragma unroll
          for (int j = 0; j < 64; ++j) v[j] *= of_p;
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bars->p_ready));
        ok = cta.wait(bars->dp_full, steps, MOSS_STATUS_TIMEOUT_EPILOGUE);
        if (!ok) break;
        tc_fence_after();
        load64(dp_tmem + half * kHalf + lanes, r);
#pragma unroll
        for (int j = 0; j < 64; j += 4) {
          const float4 d = *reinterpret_cast<const float4*>(lse + kTile + j);  // negated
          const uint64_t lo = add_pair(pair_of(__uint_as_float(r[j >> 5][j & 31]), __uint_as_float(r[j >> 5][(j & 31) + 1])), pair_of(d.x, d.y));
          const uint64_t hi = add_pair(pair_of(__uint_as_float(r[j >> 5][(j & 31) + 2]), __uint_as_float(r[j >> 5][(j & 31) + 3])), pair_of(d.z, d.w));
          split_pair(mul_pair(pair_of(v[j], v[j + 1]), lo), v[j], v[j + 1]);
          split_pair(mul_pair(pair_of(v[j + 2], v[j + 3]), hi), v[j + 2], v[j + 3]);
        }
        if (!seen || rows < kHalf) {
#pragma unroll
          for (int j = 0; j < 64; ++j)
            if (!seen || j >= rows) v[j] = 0.0f;
        }
        if (alone) {  // (NaN stays)
#pragma unroll
          for (int j = 0; j < 64; ++j) v[j] *= 0.0f;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bars->stat_free[slot]));
        store64<kKind>(dp_tmem + half * kHalf + lanes, v);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bars->ds_ready));
      }
      if (!ok) break;
      const bool any = w.first < w.end;
      if (any) {
        ok = cta.wait(bars->acc_full, accs++, MOSS_STATUS_TIMEOUT_EPILOGUE);
        if (!ok) break;
        tc_fence_after();
      }
      float* const part = args.partial + ((static_cast<int64_t>(half) * args.splits + w.split) * args.tail + w.tail) * kTile * args.head_dim;
      const int64_t to = ((w.s.k_row + key) * args.k_heads + w.head) * args.head_dim;
      const uint32_t from = (half == 0 ? dv_tmem : dk_tmem) + lanes;
      const float factor = half == 1 ? args.scale * pow2(-lift) : pow2(-static_cast<int>(kLift<kKind>));
#pragma unroll
      for (int c = 0; c < kD / 32; ++c) {
        uint32_t o[32];
        float out[32];
        __syncwarp();
        if (any) {
          tmem_ld_32x32b_x32(from + c * 32, o);
          wait_ld_of(o);
          if (c == kD / 32 - 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&bars->acc_free));
          }
        }
#pragma unroll
        for (int j = 0; j < 32; ++j) out[j] = any ? __uint_as_float(o[j]) * factor : 0.0f;
        const int count = args.head_dim - c * 32;
        if (key < w.s.kn && count > 0) {
          if (w.tail >= 0)
            store_row32_f32(part + row * args.head_dim + c * 32, count, out);
          else
            store_row32<kKind>(static_cast<uint16_t*>(result) + to + c * 32, wide, count, out);
        }
      }
    }
  }
  end<kD>(tmem);
}

template <int kD, typename F>
int launch(const char* what, F* kern, DeviceSetup& setup, int64_t units, const Maps& maps, const Args& a, cudaStream_t stream) {
  const int rc = setup(what, nullptr, [&](int*) {
    return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<kD>::kSmemBytes);
  });
  if (rc != MOSS_OK) return rc;
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(units, device_sm_count()));
  kern<<<grid, kThreads, Shape<kD>::kSmemBytes, stream>>>(maps.q, maps.k, maps.v, maps.grad, maps.o, a);
  return check_cuda(cudaGetLastError(), what);
}

template <int kKind, int kD, bool kMask>
int launch_dq_typed(const Maps& maps, const Args& a, cudaStream_t stream) {
  static DeviceSetup setup;
  return launch<kD>("cross_dq_kernel", cross_dq_kernel<kKind, kD, kMask>, setup, static_cast<int64_t>(a.tiles) * a.splits * a.q_heads,
                    maps, a, stream);
}
template <int kKind, int kD, bool kPacked>
int launch_dkv_typed(const Maps& maps, const Args& a, cudaStream_t stream) {
  static DeviceSetup setup;
  return launch<kD>("cross_dkv_kernel", cross_dkv_kernel<kKind, kD, kPacked>, setup,
                    a.whole + static_cast<int64_t>(a.tail) * a.splits, maps, a, stream);
}
template <int kKind, int kD>
int launch_shape(bool keys, const Maps& maps, const Args& a, cudaStream_t stream) {
  const bool packed = a.q_offsets != nullptr;
  if (keys) return packed ? launch_dkv_typed<kKind, kD, true>(maps, a, stream) : launch_dkv_typed<kKind, kD, false>(maps, a, stream);
  return packed || a.mask != nullptr ? launch_dq_typed<kKind, kD, true>(maps, a, stream)
                                     : launch_dq_typed<kKind, kD, false>(maps, a, stream);
}
int launch_kind(bool keys, int kind, const Maps& maps, const Args& a, cudaStream_t stream) {
  if (kind == kBF16)
    return a.head_dim <= 64 ? launch_shape<kBF16, 64>(keys, maps, a, stream) : launch_shape<kBF16, 128>(keys, maps, a, stream);
  return a.head_dim <= 64 ? launch_shape<kF16, 64>(keys, maps, a, stream) : launch_shape<kF16, 128>(keys, maps, a, stream);
}

}  // namespace

int launch_dq(int kind, const Maps& maps, const Args& a, cudaStream_t stream) { return launch_kind(false, kind, maps, a, stream); }
int launch_dkv(int kind, const Maps& maps, const Args& a, cudaStream_t stream) { return launch_kind(true, kind, maps, a, stream); }

}  // namespace cross
}  // namespace moss
