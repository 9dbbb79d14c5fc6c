// Forward pass of the attention to another sequence, on the tensor cores (tcgen05.mma.kind::f16).
//
// A CTA takes two tiles of 128 queries of one head. For each tile of 128 keys: S = Q K^T into TMEM, a warpgroup for
// each query tile reads its rows (a thread a row, so a row's maximum and sum need no shuffles), writes P back to TMEM as
// 16-bit pairs over S, and O += P V takes P from there. While one tile's rows are exponentiated, the tensor cores
// work for the other. O stays in TMEM; it is rescaled only where a row's maximum grows by more than 2^8 over the one
// its exponentials are taken against (P up to 256 loses nothing: its sum is f32, and 16-bit rounding is relative).
// The CTAs are persistent: the next pair's loads and first S run during the last tile's softmax.
//
// Warps: 0 loads by TMA, 1 and 3 issue the MMAs of a query tile each, 2 zeroes masked rows of V (0 * NaN is NaN) and stores,
// 4-7 and 8-11 do the softmax.
//
// Bound by the latency between its roles: 2 x 24 heads of 128, 4096 x 512 tokens, bf16 77 us (670 TFLOP/s; the products
// alone 31 us at the GPU's rate, the exponentials 22). The warpgroups run in step, so they meet at the special-function
// units (1250 of a half tile's 1600 cycles) and leave them idle together. Halves of key tiles, because S and P of a whole
// one leave no room in TMEM for the next; smaller ones would make every product wait for its operands.
//
// P is rounded to the inputs' 16-bit type (half a step of each term; the sum it is divided by is of the unrounded values).
#include <algorithm>
#include <cmath>
#include <cstring>

#include "cross_args.cuh"

namespace moss {
namespace cross {
namespace {

constexpr int kThreads = 384;
constexpr int kMiscRegs = 88, kSoftmaxRegs = 208;
static_assert(kMiscRegs + 2 * kSoftmaxRegs <= 3 * 168, "a larger split would wait forever");
constexpr int kHalf = kTile / 2;  // keys of one step
constexpr float kGrowth = 8.0f;
// f16 has no normal values below 2^-14: there the exponentials are 2^7 larger (up to 2^15 with kGrowth), which their sum is too.
template <int kKind>
constexpr float kLift = kKind == kF16 ? 7.0f : 0.0f;

template <int kD>
struct Shape {
  static constexpr uint32_t kTileBytes = kTile * kD * 2;
  static constexpr int kStages = kD == 128 ? 3 : 8;  // tiles of K and V on their way
  static constexpr uint32_t kDataBytes = (4 + kStages) * kTileBytes;
  static constexpr uint32_t kSmemBytes = kDataBytes + 1024 + 768;
  static_assert(kSmemBytes <= 227 * 1024, "tiles exceed the shared memory a CTA may use");
};
constexpr int kMaxStages = 8;

struct Barriers {
  uint64_t q_full[4], q_empty[4];  // by pair (they take turns) and tile
  uint64_t empty[kMaxStages];   // by stage
  // by number, modulo the stages (who waits for one of them waits for each: a barrier by stage would go on to the other
  // tensor's tile unseen)
  uint64_t k_full[kMaxStages], v_full[kMaxStages];
  uint64_t clean[kMaxStages];   // masked rows of a V tile are zero
  uint64_t s_full[2][2];       // by query tile and buffer: S is there
  uint64_t p_ready[2][2];      // P is there, O may be added to
  uint64_t pv_done[2];         // a product with P is done
  uint64_t o_full[2], o_free[2];
  // the results are in shared memory, by pair and tile as q_full: a pair's next results come after its next queries, and those after
  // its stores. (By tile alone, one softmax warpgroup finished two units while the stores waited for the other, and the
  // barrier went on unseen.)
  uint64_t out_full[4];
  uint64_t drain[2];
  uint32_t tile_bits[2 * kMaxTileBits / 32];
  uint32_t tmem_base;
  int abort_flag;
};
static_assert(sizeof(Barriers) <= 768, "barrier block too large");

// Work unit: a pair of query tiles of one head, and a run of its key tiles.
struct Unit {
  Sequence s;
  int head, split, row, first, end;  // row: the pair's first within the sequence
  __device__ __forceinline__ int tiles() const { return s.qn - row > kTile ? 2 : 1; }
  __device__ __forceinline__ int next(const TileBits& taken, int t) const { return taken.next(s.entry, t + 1, end); }
  // the halves of key tile t that hold keys
  __device__ __forceinline__ int halves(int t) const { return s.kn - t * kTile > kHalf ? 2 : 1; }
};
__device__ __forceinline__ bool locate(const Args& a, const TileBits& taken, int u, Unit& unit) {
  const int t = u % a.tiles, rest = u / a.tiles;
  unit.split = rest % a.splits;
  unit.head = rest / a.splits;
  int seq, tile;
  if (!find_tile<false>(a, 2 * kTile, t, seq, tile)) return false;
  unit.s = sequence_of(a, seq);
  if (seq >= a.batch) unit.s.kn = 0;
  unit.row = tile * 2 * kTile;
  const int keys = (unit.s.kn + kTile - 1) / kTile, each = (keys + a.splits - 1) / a.splits;
  unit.end = min(keys, (unit.split + 1) * each);
  unit.first = taken.next(unit.s.entry, min(keys, unit.split * each), unit.end);
  return true;
}

// A tile of a batch entry leaves through the shared memory of its queries, which nothing reads any more, by TMA (rows past
// the entry are not written). Rows of a packed sequence's last tile, splits and queries without keys go by their threads.
template <bool kMask>
__device__ __forceinline__ bool leaves_by_tma(const Args& a, const Unit& w, int x) {
  return a.splits == 1 && (!kMask || a.q_offsets == nullptr || w.s.qn - (w.row + x * kTile) >= kTile);
}

// kMask: keys may be masked, or a tile may hold rows of the next sequence.
template <int kKind, int kD, bool kMask>
__global__ void __launch_bounds__(kThreads, 1)
    cross_forward_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                         const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_out,
                         const Args args) {
  using S = Shape<kD>;
  constexpr uint32_t kTileBytes = S::kTileBytes;
  constexpr int kStages = S::kStages;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_base = smem_u32(smem_raw);
  const uint32_t base = (raw_base + 1023u) & ~1023u;
  const uint32_t ring = base + 4 * kTileBytes;
  Barriers* bars = reinterpret_cast<Barriers*>(smem_raw + (base - raw_base) + S::kDataBytes);
  auto bar = [&](uint64_t& b) { return smem_u32(&b); };
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int num_units = args.tiles * args.splits * args.q_heads;

  if (threadIdx.x == 0) {
    for (int x = 0; x < 4; ++x) {
      mbar_init(bar(bars->q_full[x]), 1);
      mbar_init(bar(bars->q_empty[x]), 1);
      mbar_init(bar(bars->out_full[x]), 4);
    }
    for (int x = 0; x < 2; ++x) {
      for (int b = 0; b < 2; ++b) {
        mbar_init(bar(bars->s_full[x][b]), 1);
        mbar_init(bar(bars->p_ready[x][b]), 4);
      }
      mbar_init(bar(bars->pv_done[x]), 1);
      mbar_init(bar(bars->o_full[x]), 1);
      mbar_init(bar(bars->o_free[x]), 4);
    }
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar(bars->k_full[s]), 1);
      mbar_init(bar(bars->v_full[s]), 1);
      mbar_init(bar(bars->empty[s]), 2);
      mbar_init(bar(bars->clean[s]), 1);
    }
    for (int x = 0; x < 2; ++x) mbar_init(bar(bars->drain[x]), 1);
    bars->abort_flag = 0;
    for (int i = 0; i < 2 * kMaxTileBits / 32; ++i) bars->tile_bits[i] = 0;
    fence_mbar_init();
  }
  const int key_tiles = (args.tk + kTile - 1) / kTile;
  const bool use_bits = kMask && has_tile_bits(args, key_tiles);
  if (use_bits) {
    __syncthreads();
    find_tile_bits(args, key_tiles, bars->tile_bits);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&bars->tmem_base), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const TileBits taken{use_bits ? bars->tile_bits : nullptr, key_tiles};
  // for each of the two query tiles: S (and P) of two halves of key tiles, then O
  const uint32_t tmem = bars->tmem_base;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kMiscRegs));
    if (warp == 0) {
      // ---------------------------------------------------------------- loads
      // Queries are loaded a whole unit ahead (all CTAs ask for theirs at about the same time, and half a unit's work
      // does not cover that), keys and values as the ring allows.
      uint32_t pos = 0, q_uses[4] = {0, 0, 0, 0};
      int u = blockIdx.x, ahead = u;
      uint32_t asked = 0;  // units whose queries were asked for
      bool ok = true;
      if (lane == 0) {
        tma_prefetch_desc(&tm_q);
        tma_prefetch_desc(&tm_k);
        tma_prefetch_desc(&tm_v);
      }
      auto load_q = [&](const Unit& w, int x) {
        const int slot = (asked & 1u) * 2 + x;
        if (!wait_suspended(bar(bars->q_empty[slot]), (q_uses[slot] & 1u) ^ 1u, abort_flag, args.status, MOSS_STATUS_TIMEOUT_LOAD))
          return false;
        if (lane == 0) {
          mbar_arrive_expect_tx(bar(bars->q_full[slot]), kTileBytes);
          load_tile<kD>(base + slot * kTileBytes, &tm_q, bar(bars->q_full[slot]), w.s.q0 + w.row + x * kTile, w.head, w.s.entry);
        }
        ++q_uses[slot];
        __syncwarp();
        return true;
      };
      auto load_kv = [&](const CUtensorMap* map, const Unit& w, int tile) {
        const uint32_t stage = pos % kStages, phase = (pos / kStages) & 1u;
        if (!wait_suspended(bar(bars->empty[stage]), phase ^ 1u, abort_flag, args.status, MOSS_STATUS_TIMEOUT_LOAD)) return false;
        if (lane == 0) {
          uint64_t& full = (pos & 1u) == 0 ? bars->k_full[pos / 2 % kStages] : bars->v_full[pos / 2 % kStages];
          mbar_arrive_expect_tx(bar(full), kTileBytes);
          load_tile<kD>(ring + stage * kTileBytes, map, bar(full), w.s.k0 + tile * kTile, w.head / args.group, w.s.entry);
        }
        ++pos;
        __syncwarp();
        return true;
      };
      // the queries of the next unit that has keys
      auto ask = [&]() {
        for (; ahead < num_units; ahead += gridDim.x) {
          Unit w;
          if (!locate(args, taken, ahead, w) || w.first == w.end) continue;
          if (!load_q(w, 0) || (w.tiles() > 1 && !load_q(w, 1))) return false;
          ++asked;
          ahead += gridDim.x;
          break;
        }
        return true;
      };
      ok = ask();
      for (; u < num_units && ok; u += gridDim.x) {
        Unit w;
        if (!locate(args, taken, u, w) || w.first == w.end) continue;
        ok = load_kv(&tm_k, w, w.first) && load_kv(&tm_v, w, w.first) && ask();
        for (int t = w.next(taken, w.first); t < w.end && ok; t = w.next(taken, t)) ok = load_kv(&tm_k, w, t) && load_kv(&tm_v, w, t);
      }
      if (lane == 0) {  // the copies land before the CTA may leave
        auto landed = [&](uint64_t& b, uint32_t parity) {
          const long long start = clock64();
          while (!mbar_try_wait(bar(b), parity)) {
            if (clock64() - start > kWaitBudgetCycles) {
              report_status(args.status, MOSS_STATUS_TIMEOUT_DRAIN);
              break;
            }
          }
        };
        for (uint32_t n = pos / 2 > kStages ? pos / 2 - kStages : 0; n < pos / 2; ++n) {
          landed(bars->k_full[n % kStages], (n / kStages) & 1u);
          landed(bars->v_full[n % kStages], (n / kStages) & 1u);
        }
        for (int x = 0; x < 4; ++x)
          if (q_uses[x] > 0) landed(bars->q_full[x], (q_uses[x] - 1) & 1u);
      }
    } else if (warp == 1 || warp == 3) {
      // ---------------------------------------------------------------- MMAs, a warp for each query tile
      // (One for both issued too slowly: each wait costs it 200 cycles, of the 1000 that the products of half a tile take.)
      const int x = warp >> 1;
      constexpr uint32_t kFormat = kKind == kBF16 ? 1u : 0u;
      constexpr uint32_t s_idesc = umma_idesc_f16(kFormat, false, kTile, kHalf);
      constexpr uint32_t o_idesc = umma_idesc_f16(kFormat, true, kTile, kD);
      const uint64_t q_desc = by_rows_desc(base), k_desc = by_rows_desc(ring), v_desc = by_columns_desc(ring);
      const uint32_t s_tmem = tmem + x * 2 * kTile, o_tmem = s_tmem + kTile;
      uint32_t pos = 0, units = 0, q_uses[2] = {0, 0}, steps = 0, o_uses = 0;
      bool ok = true, issued = false;
      for (int u = blockIdx.x; u < num_units && ok; u += gridDim.x) {
        Unit w;
        if (!locate(args, taken, u, w) || w.first == w.end) continue;
        int n = 0, m = 0;  // key tiles, and halves of them: only the last tile may have one
        for (int t = w.first; t < w.end; t = w.next(taken, t)) {
          ++n;
          m += w.halves(t);
        }
        const uint32_t q_slot = (units & 1u) * 2 + x;
        // one thread waits and issues for the whole unit
        if (elect_one()) {
          auto wait = [&](uint64_t& b, uint32_t parity) {
            ok = ok && mbar_poll(bar(b), parity & 1u, abort_flag, args.status, MOSS_STATUS_TIMEOUT_MMA);
            return ok;
          };
          auto k_there = [&](uint32_t p) { return wait(bars->k_full[p / 2 % kStages], p / 2 / kStages); };
          auto v_there = [&](uint32_t p) { return wait(bars->v_full[p / 2 % kStages], p / 2 / kStages); };
          auto release = [&](uint32_t p) { umma_commit(bar(bars->empty[p % kStages])); };
          if (x >= w.tiles()) {  // the other warp's keys and values pass by
            for (int i = 0; i < 2 * n && ((i & 1) == 0 ? k_there(pos + i) : v_there(pos + i)); ++i)
              mbar_arrive(bar(bars->empty[(pos + i) % kStages]));
          } else {
            // S against half j of the unit's key tiles
            auto scores = [&](int j) {
              const uint32_t g = steps + j, p = pos + (j & ~1);
              tc_fence_after();
              mma_over_head<kD>(s_tmem + (g & 1u) * kHalf, q_desc + ((q_slot * kTileBytes) >> 4),
                                k_desc + (((p % kStages) * kTileBytes + (j & 1) * kHalf * 128) >> 4), s_idesc);
              umma_commit(bar(bars->s_full[x][g & 1u]));
            };
            if (k_there(pos) && wait(bars->q_full[q_slot], q_uses[units & 1u])) {
              scores(0);
              if (m > 1) scores(1);
              release(pos);
              wait(bars->o_free[x], o_uses ^ 1u);
            }
            for (int j = 0; j < m && ok; ++j) {
              const uint32_t pv = pos + (j & ~1) + 1;  // of V; the next tile's K is behind it
              const uint32_t g = steps + j;
              if ((j & 1) == 0) {
                const uint32_t nth = pv / 2;  // of the V tiles: what `clean` counts
                if (!(kMask ? wait(bars->clean[nth % kStages], nth / kStages) : v_there(pv))) break;
              }
              if (!wait(bars->p_ready[x][g & 1u], g >> 1)) break;
              tc_fence_after();
              mma_over_keys(o_tmem, s_tmem + (g & 1u) * kHalf, v_desc + (((pv % kStages) * kTileBytes + (j & 1) * kHalf * 128) >> 4),
                            o_idesc, j > 0);
              umma_commit(bar(j + 1 < m ? bars->pv_done[x] : bars->o_full[x]));
              const bool last_half = (j & 1) == 1;
              if (last_half || j + 1 == m) release(pv);
              if (j + 2 < m) {
                if (!last_half && !k_there(pv + 1)) break;
                scores(j + 2);
                if (last_half || j + 3 == m) release(pv + 1);
              }
            }
          }
        }
        ok = __all_sync(0xffffffffu, ok) != 0;
        if (x < w.tiles()) {
          issued = true;
          ++q_uses[units & 1u];
          ++o_uses;
          steps += m;
        }
        ++units;
        pos += 2 * n;
      }
      if (lane == 0 && issued) {
        umma_commit(bar(bars->drain[x]));
        const long long start = clock64();
        while (!mbar_try_wait(bar(bars->drain[x]), 0)) {
          if (clock64() - start > kWaitBudgetCycles) {
            report_status(args.status, MOSS_STATUS_TIMEOUT_DRAIN);
            break;
          }
        }
      }
      __syncwarp();
    } else {
      // ---------------------------------------------------------------- masked rows of V, and the stores (which a softmax warp
      // would wait 1500 cycles a tile for)
      uint32_t pos = 0, units = 0, uses[4] = {0, 0, 0, 0};
      bool ok = true;
      for (int u = blockIdx.x; u < num_units && ok; u += gridDim.x) {
        Unit w;
        if (!locate(args, taken, u, w) || w.first == w.end) continue;
        if constexpr (kMask) {
          for (int t = w.first; t < w.end; t = w.next(taken, t), pos += 2) {
            const KeyBits keep = key_bits(args, w.s, t * kTile, taken.whole(w.s.entry, t));
            const uint32_t stage = (pos + 1) % kStages;
            ok = wait_together(bar(bars->v_full[(pos / 2) % kStages]), (pos / 2 / kStages) & 1u, abort_flag, args.status, MOSS_STATUS_TIMEOUT_LOAD);
            if (!ok) break;
            if (!keep.all()) scrub_rows<kD>(ring + stage * kTileBytes, keep);
            if (lane == 0) mbar_arrive(bar(bars->clean[(pos / 2) % kStages]));
          }
        }
        for (int x = 0; x < w.tiles() && ok; ++x) {
          const uint32_t slot = (units & 1u) * 2 + x;
          ok = wait_suspended(bar(bars->out_full[slot]), uses[slot]++ & 1u, abort_flag, args.status, MOSS_STATUS_TIMEOUT_EPILOGUE);
          if (!ok) break;
          if (lane == 0) {
            if (leaves_by_tma<kMask>(args, w, x)) {
#pragma unroll
              for (int c = 0; c < kD / 64; ++c)
                tma_store_4d(&tm_out, base + slot * kTileBytes + c * 16384, c * 64, w.s.q0 + w.row + x * kTile, w.head, w.s.entry);
              bulk_commit();
              bulk_wait_read();
            }
            mbar_arrive(bar(bars->q_empty[slot]));
          }
          __syncwarp();
        }
        ++units;
      }
      if (lane == 0) bulk_wait();
    }
  } else {
    // ---------------------------------------------------------------- softmax and output
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int x = (warp - 4) >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tile_tmem = tmem + x * 2 * kTile + lanes, o_tmem = tile_tmem + kTile;
    const bool wide = args.head_dim % 16 == 0 && (reinterpret_cast<uintptr_t>(args.out) & 31) == 0;
    uint32_t step = 0, products = 0, o_uses = 0, units = 0;
    bool ok = true;
    for (int u = blockIdx.x; u < num_units && ok; u += gridDim.x) {
      Unit w;
      if (!locate(args, taken, u, w)) continue;
      const bool any_keys = w.first < w.end;
      const uint32_t slot = (units & 1u) * 2 + x;
      if (any_keys) ++units;
      if (x >= w.tiles()) continue;
      const int at = w.row + x * kTile + row;  // within the sequence
      const int64_t q_row = w.s.q_row + at;
      const bool live = at < w.s.qn;
      float top = -INFINITY, sum = 0.0f;  // the exponentials' reference, times scale_log2
      bool begun = false;
      for (int t = w.first; t < w.end && ok; t = w.next(taken, t)) {
        KeyBits keep;
        if constexpr (kMask) keep = key_bits(args, w.s, t * kTile, taken.whole(w.s.entry, t));
        const int halves = w.halves(t);
#pragma unroll 1
        for (int half = 0; half < halves; ++half, ++step) {
          const int keys = w.s.kn - t * kTile - half * kHalf;
          const uint32_t s_tmem = tile_tmem + (step & 1u) * kHalf;
          ok = wait_together(bar(bars->s_full[x][step & 1u]), (step >> 1) & 1u, abort_flag, args.status, MOSS_STATUS_TIMEOUT_EPILOGUE);
          if (!ok) break;
          tc_fence_after();
          uint32_t r[2][32];
          tmem_ld_32x32b_x32(s_tmem, r[0]);
          tmem_ld_32x32b_x32(s_tmem + 32, r[1]);
          wait_ld_of(r[0]);
          wait_ld_of(r[1]);
          if constexpr (kMask) {
            const uint32_t k0 = half == 0 ? keep.w[0] : keep.w[2], k1 = half == 0 ? keep.w[1] : keep.w[3];
            if ((k0 & k1) != 0xffffffffu) {
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                if (((k0 >> j) & 1u) == 0) r[0][j] = 0xff800000u;
                if (((k1 >> j) & 1u) == 0) r[1][j] = 0xff800000u;
              }
            }
          } else {
            if (keys < kHalf) {
#pragma unroll
              for (int j = 0; j < 64; ++j)
                if (j >= keys) r[j >> 5][j & 31] = 0xff800000u;
            }
          }
          float most[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int j = 0; j < 64; ++j) most[j & 3] = fmaxf(most[j & 3], __uint_as_float(r[j >> 5][j & 31]));
          // (the scale is positive, so the greatest product gives the greatest logit; fmaxf drops NaN, whose exponential is NaN against
          // any reference)
          const float here = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])) * args.scale_log2;
          const bool grows = here > top + kGrowth;  // (from -inf always, unless all keys are masked)
          if (__any_sync(0xffffffffu, grows)) {
            const float factor = grows ? exp2_approx(top - here) : 1.0f;
            if (grows) top = here;
            sum *= factor;
            if (begun) {  // the last product has to be done before its sums are touched
              ok = wait_together(bar(bars->pv_done[x]), (products - 1) & 1u, abort_flag, args.status, MOSS_STATUS_TIMEOUT_EPILOGUE);
              if (!ok) break;
              tc_fence_after();
#pragma unroll
              for (int c = 0; c < kD / 32; ++c) {
                uint32_t o[32];
                tmem_ld_32x32b_x32(o_tmem + c * 32, o);
                wait_ld_of(o);
                uint32_t lo[16], hi[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                  lo[j] = __float_as_uint(__uint_as_float(o[j]) * factor);
                  hi[j] = __float_as_uint(__uint_as_float(o[16 + j]) * factor);
                }
                tmem_st_32x32b_x16(o_tmem + c * 32, lo);
                tmem_st_32x32b_x16(o_tmem + c * 32 + 16, hi);
              }
            }
          }
          const float shift = top == -INFINITY ? 0.0f : top - kLift<kKind>;
          const uint64_t scale2 = pair_of(args.scale_log2, args.scale_log2), minus_shift = pair_of(-shift, -shift);
          uint64_t add[2] = {0, 0};
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t p[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const uint64_t e = exponentials(c * 16 + j, pair_of(__uint_as_float(r[c][2 * j]), __uint_as_float(r[c][2 * j + 1])),
                                              scale2, minus_shift);
              add[j & 1] = add_pair(add[j & 1], e);
              float e0, e1;
              split_pair(e, e0, e1);
              p[j] = gemm::pack2_kind<kKind>(e0, e1);
            }
            tmem_st_32x32b_x16(s_tmem + c * 16, p);
          }
          float add0, add1;
          split_pair(add_pair(add[0], add[1]), add0, add1);
          sum += add0 + add1;
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(bars->p_ready[x][step & 1u]));
          begun = true;
          ++products;
        }
      }
      if (!ok) break;
      if (begun) --products;  // the unit's last product is told by o_full
      if (any_keys) {
        ok = wait_together(bar(bars->o_full[x]), o_uses++ & 1u, abort_flag, args.status, MOSS_STATUS_TIMEOUT_EPILOGUE);
        if (!ok) break;
        tc_fence_after();
      }
      const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
      const int64_t at_out = (q_row * args.q_heads + w.head) * args.head_dim;
      const bool by_tma = any_keys && leaves_by_tma<kMask>(args, w, x);
      const uint32_t staged = base + slot * kTileBytes + row * 128;
#pragma unroll
      for (int c = 0; c < kD / 32; ++c) {
        uint32_t o[32];
        float v[32];
        __syncwarp();  // (lanes past the last row have nothing to store)
        if (any_keys) {
          tmem_ld_32x32b_x32(o_tmem + c * 32, o);
          wait_ld_of(o);
          if (c == kD / 32 - 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(bars->o_free[x]));
          }
        }
        // (a row whose keys are all masked has zeros in O, and an empty one nothing)
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = any_keys ? __uint_as_float(o[j]) * inverse : 0.0f;
        const int count = args.head_dim - c * 32;
        if (by_tma) {
#pragma unroll
          for (int h = 0; h < 4; ++h)
            gemm::sts128(staged + (c >> 1) * 16384 + ((((c & 1) * 4 + h) ^ (row & 7)) << 4),
                         make_uint4(gemm::pack2_kind<kKind>(v[8 * h], v[8 * h + 1]), gemm::pack2_kind<kKind>(v[8 * h + 2], v[8 * h + 3]),
                                    gemm::pack2_kind<kKind>(v[8 * h + 4], v[8 * h + 5]), gemm::pack2_kind<kKind>(v[8 * h + 6], v[8 * h + 7])));
        } else if (live && count > 0) {
          if (args.splits > 1)
            store_row32_f32(args.partial + w.split * args.q_rows * args.q_heads * args.head_dim + at_out + c * 32, count, v);
          else
            store_row32<kKind>(static_cast<uint16_t*>(args.out) + at_out + c * 32, wide, count, v);
        }
      }
      if (any_keys) {
        if (by_tma) fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(bars->out_full[slot]));
      }
      if (live) {
        const float l = sum == 0.0f ? -INFINITY : top - kLift<kKind> + log2f(sum);
        if (args.splits > 1)
          args.partial_lse[(static_cast<int64_t>(w.split) * args.q_heads + w.head) * args.q_rows + q_row] = l;
        else if (args.lse != nullptr)
          args.lse[w.head * args.q_rows + q_row] = sum == 0.0f ? INFINITY : l;
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int kKind, int kD, bool kMask>
int launch_typed(const Maps& maps, const Args& a, cudaStream_t stream) {
  auto kern = cross_forward_kernel<kKind, kD, kMask>;
  static DeviceSetup setup;
  const int rc = setup("cross_forward_kernel", nullptr, [&](int*) {
    return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<kD>::kSmemBytes);
  });
  if (rc != MOSS_OK) return rc;
  const int64_t units = static_cast<int64_t>(a.tiles) * a.splits * a.q_heads;
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(units, device_sm_count()));
  kern<<<grid, kThreads, Shape<kD>::kSmemBytes, stream>>>(maps.q, maps.k, maps.v, maps.o, a);
  return check_cuda(cudaGetLastError(), "cross_forward_kernel");
}

template <int kKind, int kD>
int launch_mask(const Maps& maps, const Args& a, cudaStream_t stream) {
  return a.mask != nullptr || a.q_offsets != nullptr ? launch_typed<kKind, kD, true>(maps, a, stream)
                                                     : launch_typed<kKind, kD, false>(maps, a, stream);
}

}  // namespace

int launch_forward(int kind, const Maps& maps, const Args& a, cudaStream_t stream) {
  if (kind == kBF16)
    return a.head_dim <= 64 ? launch_mask<kBF16, 64>(maps, a, stream) : launch_mask<kBF16, 128>(maps, a, stream);
  return a.head_dim <= 64 ? launch_mask<kF16, 64>(maps, a, stream) : launch_mask<kF16, 128>(maps, a, stream);
}

}  // namespace cross
}  // namespace moss
