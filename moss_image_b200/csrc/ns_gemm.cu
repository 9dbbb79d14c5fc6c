// The products of a Newton-Schulz step on the tensor cores (tcgen05.mma.kind::f16, f32 sums).
//
// Three shapes of one kernel: a CTA pair on 256 x 256 tiles where those fill the GPU, one CTA on
// 128 x 128 or 128 x 64 tiles where they do not. Warp 0 streams 128-wide reduction steps by TMA (one
// box per operand), warp 1 issues the MMAs into one of two TMEM accumulators, warps 2-9 drain the
// other. A and B are symmetric: only tiles on and above the diagonal are computed, and written
// twice; both orders of a diagonal tile's products sum alike, so A and B stay symmetric bit for
// bit, and the update may read B by rows. X is read by columns there (MN-major), from the same
// storage.
//
// Bound by the tensor cores at the sides the update is worth its time for: 2 r^2 c products for
// X', half of that for A, and r^3 for B, against 4 r c + 2 r^2 values moved. 4 x 3072 x 3072: X' 162 us
// (1.43 PFLOP/s), A and B 100 us each (4.2 rounds of pair tiles take the time of 5). Few tiles are bound by
// latency, 5 us a product: 1.3 us from the launch to the first tile, the steps, the epilogue.
#include <algorithm>
#include <cstring>

#include "dequant.cuh"
#include "ns_args.cuh"

namespace moss {
namespace ns {
namespace {

constexpr int kHalf = 128;
constexpr int kStep = 128;  // reduction indices per stage: two 64-wide boxes
constexpr int kEpiWarp0 = 2;
constexpr int kEpiWarps = 8;  // two per quarter of the lanes, each with half of the columns
constexpr int kThreads = (kEpiWarp0 + kEpiWarps) * 32;
constexpr int kMaxStages = 4;
constexpr uint32_t kLeftBytes = kHalf * kStep * 2;  // 32 KB

// kN: columns of a tile (of the pair's, where there is one).
template <int kCtas, int kN>
struct Shape {
  static constexpr int kTileM = kHalf * kCtas;
  static constexpr int kRight = kN / kCtas;  // columns this CTA holds of the right operand
  static constexpr uint32_t kRightBytes = kRight * kStep * 2;
  static constexpr uint32_t kStageBytes = kLeftBytes + kRightBytes;
  static constexpr int kStages = kRight == 64 ? 4 : 3;
  static constexpr uint32_t kDataBytes = kStages * kStageBytes;
  static constexpr uint32_t kSmemBytes = kDataBytes + 1024 + 512;
  static_assert(kSmemBytes <= 227 * 1024, "rings exceed the shared memory a CTA may use");
};
constexpr long long kExitBudgetCycles = (kMaxStages + 4) * kWaitBudgetCycles;

struct Barriers {
  uint64_t full[kMaxStages];   // leader: both CTAs' operands landed
  uint64_t empty[kMaxStages];  // local
  uint64_t acc_full[2];     // local
  uint64_t acc_empty[2];    // leader
  uint64_t drain;
  uint64_t exit_bar;
  uint32_t tmem_base;
  int abort_flag;
};
static_assert(sizeof(Barriers) <= 512, "barrier block too large");

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2,
                                            int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
__device__ __forceinline__ void tma_load_4d_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1,
                                                 int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

// Tile t of a symmetric product: column n holds the n + 1 tiles (0..n, n).
__device__ __forceinline__ void upper_tile(int t, int& m, int& n) {
  n = static_cast<int>((sqrtf(8.0f * static_cast<float>(t) + 1.0f) - 1.0f) * 0.5f);
  while (n * (n + 1) / 2 > t) --n;
  while ((n + 1) * (n + 2) / 2 <= t) ++n;
  m = t - n * (n + 1) / 2;
}

// Unit u: matrix b, row tile m, column tile n (of kN columns; a 128-row tile's diagonal block is two of 64).
template <Mode kMode, int kN>
__device__ __forceinline__ void locate(const Args& a, int u, int& b, int& m, int& n) {
  b = u / a.tiles;
  const int t = u - b * a.tiles;
  if constexpr (kMode == kUpdate) {
    gemm::tile_coords(t, a.tiles_m, a.tiles_n, m, n);
  } else if constexpr (kN == 64) {
    upper_tile(t >> 1, m, n);
    n = 2 * n + (t & 1);
  } else {
    upper_tile(t, m, n);
  }
}

// 32 consecutive values of the operand that is added to a tile's row, as they are stored. They do not depend
// on the products, so they are on their way before the accumulator is done (one at a time after it, they
// took half of a small tile's life).
struct Added {
  uint32_t hi[16], lo[16];  // unset in lanes past the last row, which store nothing
};
// 64 bytes in two whole sectors a lane: what lies in between belongs to other lanes' rows, and 16-byte loads would
// ask L1 for every sector twice.
__device__ __forceinline__ void load64(const __half* p, uint32_t (&w)[16]) {
#pragma unroll
  for (int h = 0; h < 16; h += 8)
    asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[h]), "=r"(w[h + 1]), "=r"(w[h + 2]), "=r"(w[h + 3]), "=r"(w[h + 4]), "=r"(w[h + 5]),
                   "=r"(w[h + 6]), "=r"(w[h + 7])
                 : "l"(p + 2 * h));
}
template <Mode kMode>
__device__ __forceinline__ void fetch32(const Args& a, int b, int i, int j, Added& x) {
  const int cols = kMode == kUpdate ? a.cp : a.sp;
  if (kMode == kGram || i >= a.r || j >= cols) return;
  const int64_t at = (static_cast<int64_t>(b) * a.r + i) * cols + j;
  load64(a.add_hi + at, x.hi);
  if (kMode == kUpdate && a.add_lo != nullptr) load64(a.add_lo + at, x.lo);
}
__device__ __forceinline__ void widen32(const uint32_t (&w)[16], float (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void store32(__half* p, const float (&v)[32]) {
  uint32_t w0[8], w1[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    w0[j] = gemm::pack2_kind<kF16>(v[2 * j], v[2 * j + 1]);
    w1[j] = gemm::pack2_kind<kF16>(v[16 + 2 * j], v[16 + 2 * j + 1]);
  }
  gemm::stg256(p, w0);
  gemm::stg256(p + 16, w1);
}

// A warp's 32 x 32 block of the result, lane by lane a row, written by columns: rows of any alignment, 64 bytes of
// one at a time (stores of each lane along its own row meet 32 sectors each: with them 149 x 176 x 2546 took
// 1.4 times as long). Turned by shuffles: shared memory for it would be taken from the L1
// cache, and the products that read and write much were 10% slower.
__device__ __forceinline__ void store_turned(const Args& a, __nv_bfloat16* out, int i0, int j, const float (&v)[32]) {
  const int lane = threadIdx.x & 31;
  uint32_t w[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) w[e] = gemm::pack2_kind<kBF16>(v[2 * e], v[2 * e + 1]);
  // within each half of the warp: word k of lane l becomes word l of lane k
#pragma unroll
  for (int d = 8; d > 0; d >>= 1) {
    const bool upper = (lane & d) != 0;
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      if (k & d) continue;
      const uint32_t got = __shfl_xor_sync(0xffffffffu, upper ? w[k] : w[k + d], d);
      if (upper)
        w[k] = got;
      else
        w[k + d] = got;
    }
  }
  const int first = i0 + (lane & 16), rows = min(16, a.r - first);
  const int col = j + 2 * (lane & 15);
  __nv_bfloat16* to = out + static_cast<int64_t>(first) * a.c + col;
  const bool words = a.c % 2 == 0 && (reinterpret_cast<uintptr_t>(out) & 3) == 0;
#pragma unroll
  for (int k = 0; k < 16; ++k, to += a.c) {
    if (k >= rows || col >= a.c) continue;
    if (words) {
      *reinterpret_cast<uint32_t*>(to) = w[k];
    } else {
      const __nv_bfloat162 pair = *reinterpret_cast<const __nv_bfloat162*>(&w[k]);
      to[0] = __low2bfloat16(pair);
      if (col + 1 < a.c) to[1] = __high2bfloat16(pair);
    }
  }
}

// 32 consecutive accumulators of one row through the mode's epilogue. i, j: row and first column.
template <Mode kMode>
__device__ __forceinline__ void finish32(const Args& a, float alpha, float beta, int b, int i, int j, bool mirror,
                                         const Added& added, float (&v)[32]) {
  if constexpr (kMode == kUpdate) {
    const int64_t at = (static_cast<int64_t>(b) * a.r + i) * a.cp + j;
    float x[32];
    widen32(added.hi, x);
    if (a.add_lo != nullptr) {
      float lo[32];
      widen32(added.lo, lo);
#pragma unroll
      for (int e = 0; e < 32; ++e) x[e] += lo[e];
    }
#pragma unroll
    for (int e = 0; e < 32; ++e) v[e] = fmaf(beta, x[e], alpha * v[e]);
    if (a.result != nullptr) {
      __nv_bfloat16* out = a.result + static_cast<int64_t>(b) * a.r * a.c;
      if (a.tall) {  // lanes hold consecutive rows: 64 contiguous bytes per column
        if (i >= a.r) return;
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (j + e < a.c) out[static_cast<int64_t>(j + e) * a.r + i] = __float2bfloat16_rn(v[e]);
      } else {
        // one choice for the whole warp: a row's alignment is the matrix's where c is a multiple of 16
        if (j + 32 <= a.c && a.c % 16 == 0 && (reinterpret_cast<uintptr_t>(out) & 31) == 0) {
          if (i >= a.r) return;
          __nv_bfloat16* row = out + static_cast<int64_t>(i) * a.c + j;
          uint32_t w0[8], w1[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            w0[e] = gemm::pack2_kind<kBF16>(v[2 * e], v[2 * e + 1]);
            w1[e] = gemm::pack2_kind<kBF16>(v[16 + 2 * e], v[16 + 2 * e + 1]);
          }
          gemm::stg256(row, w0);
          gemm::stg256(row + 16, w1);
        } else {
          store_turned(a, out, i - static_cast<int>(threadIdx.x & 31), j, v);
        }
      }
      return;
    }
    if (i >= a.r) return;
    store32(a.out_hi + at, v);
    if (a.out_lo != nullptr) {
#pragma unroll
      for (int e = 0; e < 32; ++e) v[e] -= __half2float(__float2half_rn(v[e]));
      store32(a.out_lo + at, v);
    }
  } else {
    const int64_t base = static_cast<int64_t>(b) * a.r * a.sp;
    const int64_t at = base + static_cast<int64_t>(i) * a.sp + j;
    if constexpr (kMode == kSquare) {
      float x[32];
      widen32(added.hi, x);
#pragma unroll
      for (int e = 0; e < 32; ++e) v[e] = fmaf(beta, x[e], alpha * v[e]);
    } else {
#pragma unroll
      for (int e = 0; e < 32; ++e) v[e] *= alpha;
    }
    store32(a.out_hi + at, v);
    if (mirror) {
      const int64_t down = base + static_cast<int64_t>(j) * a.sp + i;
      if (j + 32 <= a.r) {  // 32 conditions would cost small products 6%
#pragma unroll
        for (int e = 0; e < 32; ++e) a.out_hi[down + static_cast<int64_t>(e) * a.sp] = __float2half_rn(v[e]);
      } else {
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (j + e < a.r) a.out_hi[down + static_cast<int64_t>(e) * a.sp] = __float2half_rn(v[e]);
      }
    }
  }
}

template <Mode kMode, int kCtas, int kN>
__global__ void __launch_bounds__(kThreads, 1)
    ns_gemm_kernel(const __grid_constant__ CUtensorMap tm_left, const __grid_constant__ CUtensorMap tm_right,
                   const Args args) {
  constexpr bool kColumns = kMode == kUpdate;  // the right operand is read by columns (MN-major)
  using S = Shape<kCtas, kN>;
  constexpr int kTileM = S::kTileM, kStages = S::kStages;
  constexpr uint32_t kStageBytes = S::kStageBytes;
  constexpr uint32_t kTmemCols = 2 * kN;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_base = smem_u32(smem_raw);
  const uint32_t base = (raw_base + 1023u) & ~1023u;
  Barriers* bars = reinterpret_cast<Barriers*>(smem_raw + (base - raw_base) + S::kDataBytes);
  auto bar = [&](uint64_t& b) { return smem_u32(&b); };
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = kCtas == 2 ? cluster_ctarank() : 0;
  const bool leader = rank == 0;
  const int first_unit = blockIdx.x / kCtas;
  const int unit_step = gridDim.x / kCtas;
  const int num_units = args.tiles * args.batch;
  const int steps = ((kMode == kGram ? args.cp : args.sp) + kStep - 1) / kStep;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar(bars->full[s]), 1);
      mbar_init(bar(bars->empty[s]), 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(bar(bars->acc_full[s]), 1);
      mbar_init(bar(bars->acc_empty[s]), kCtas * kEpiWarps);
    }
    mbar_init(bar(bars->drain), 1);
    mbar_init(bar(bars->exit_bar), 1);
    bars->abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    if constexpr (kCtas == 2) {
      tmem_alloc_pair(smem_u32(&bars->tmem_base), kTmemCols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_u32(&bars->tmem_base), kTmemCols);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  if constexpr (kCtas == 2)
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  else
    __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = bars->tmem_base;
  pdl_trigger();
  pdl_wait();

  if (warp == 0) {
    // ---------------------------------------------------------------- producer (every CTA)
    if (lane == 0) {
      tma_prefetch_desc(&tm_left);
      tma_prefetch_desc(&tm_right);
    }
    int stage = 0;
    uint32_t phase = 0, used = 0, last_phase = 0;
    bool ok = true;
    for (int u = first_unit; u < num_units && ok; u += unit_step) {
      int b, m, n;
      locate<kMode, kN>(args, u, b, m, n);
      const int m0 = m * kTileM + static_cast<int>(rank) * kHalf;  // row of the left operand
      const int n0 = n * kN + static_cast<int>(rank) * S::kRight;  // this CTA's columns
      for (int s = 0; s < steps; ++s) {
        if (!mbar_wait_cluster(bar(bars->empty[stage]), phase ^ 1u, abort_flag, args.status,
                               MOSS_STATUS_TIMEOUT_LOAD)) {
          ok = false;
          break;
        }
        if (lane == 0) {
          const uint32_t dst = base + stage * kStageBytes;
          const int ry = kColumns ? s * kStep : n0;
          const int rz = kColumns ? n0 / 64 : s * 2;
          if constexpr (kCtas == 2) {
            if (leader) mbar_arrive_expect_tx(bar(bars->full[stage]), kCtas * kStageBytes);
            const uint32_t fb = mapa_shared(bar(bars->full[stage]), 0);
            tma_load_4d_pair(dst, &tm_left, fb, 0, m0, s * 2, b);
            tma_load_4d_pair(dst + kLeftBytes, &tm_right, fb, 0, ry, rz, b);
          } else {
            mbar_arrive_expect_tx(bar(bars->full[stage]), kStageBytes);
            tma_load_4d(dst, &tm_left, bar(bars->full[stage]), 0, m0, s * 2, b);
            tma_load_4d(dst + kLeftBytes, &tm_right, bar(bars->full[stage]), 0, ry, rz, b);
          }
          used |= 1u << stage;
          last_phase = (last_phase & ~(1u << stage)) | (phase << stage);
        }
        __syncwarp();
        if (++stage == kStages) { stage = 0; phase ^= 1u; }
      }
    }
    if (lane == 0 && leader) {  // the copies land before the CTA may leave (the peer waits for the leader)
      for (int s = 0; s < kStages; ++s) {
        if (!((used >> s) & 1u)) continue;
        const long long start = clock64();
        while (!mbar_try_wait(bar(bars->full[s]), (last_phase >> s) & 1u)) {
          if (clock64() - start > kWaitBudgetCycles) {
            report_status(args.status, MOSS_STATUS_TIMEOUT_DRAIN);
            break;
          }
        }
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer (leader)
    if (leader) {
      constexpr uint32_t idesc = umma_idesc_f16(0u, kColumns, kTileM, kN);
      // descriptors of the first stage; every other differs by multiples of 16 bytes in the address field.
      // K-major: [2 boxes][rows][64 values]; by columns: [boxes of 64 columns][128 rows]
      const uint64_t left0 = umma_desc_sw128(base, 16, 1024);
      const uint64_t right0 = umma_desc_sw128(base + kLeftBytes, kColumns ? 16384 : 16, 1024);
      int stage = 0, it = 0;
      uint32_t phase = 0;
      bool ok = true, issued = false;
      for (int u = first_unit; u < num_units && ok; u += unit_step, ++it) {
        const int acc = it & 1;
        if (!mbar_wait_cluster(bar(bars->acc_empty[acc]), ((it >> 1) & 1) ^ 1u, abort_flag, args.status,
                               MOSS_STATUS_TIMEOUT_MMA))
          break;
        tc_fence_after();
        const uint32_t d = tmem_base + static_cast<uint32_t>(acc * kN);
        for (int s = 0; s < steps; ++s) {
          if (!mbar_wait_cluster(bar(bars->full[stage]), phase, abort_flag, args.status, MOSS_STATUS_TIMEOUT_MMA)) {
            ok = false;
            break;
          }
          tc_fence_after();
          if (elect_one()) {
            const uint64_t at_stage = static_cast<uint64_t>(stage) * (kStageBytes >> 4);
#pragma unroll
            for (int kk = 0; kk < kStep / 16; ++kk) {
              const uint64_t ld = left0 + at_stage + (((kk >> 2) * (kLeftBytes / 2) + (kk & 3) * 32) >> 4);
              const uint64_t rd = right0 + at_stage +
                                  ((kColumns ? kk * 2048 : (kk >> 2) * (S::kRightBytes / 2) + (kk & 3) * 32) >> 4);
              if constexpr (kCtas == 2)
                umma_f16_pair(d, ld, rd, idesc, (s > 0 || kk > 0) ? 1u : 0u);
              else
                umma_f16(d, ld, rd, idesc, (s > 0 || kk > 0) ? 1u : 0u);
            }
            if constexpr (kCtas == 2)
              umma_commit_pair_mc(bar(bars->empty[stage]), 0x3);
            else
              umma_commit(bar(bars->empty[stage]));
          }
          issued = true;
          __syncwarp();
          if (++stage == kStages) { stage = 0; phase ^= 1u; }
        }
        if (!ok) break;
        if (elect_one()) {
          if constexpr (kCtas == 2)
            umma_commit_pair_mc(bar(bars->acc_full[acc]), 0x3);
          else
            umma_commit(bar(bars->acc_full[acc]));
        }
        __syncwarp();
      }
      if (lane == 0 && issued) {
        if constexpr (kCtas == 2)
          umma_commit_pair(bar(bars->drain));
        else
          umma_commit(bar(bars->drain));
        const long long start = clock64();
        while (!mbar_try_wait(bar(bars->drain), 0)) {
          if (clock64() - start > kWaitBudgetCycles) {
            report_status(args.status, MOSS_STATUS_TIMEOUT_DRAIN);
            break;
          }
        }
      }
      __syncwarp();
    }
  } else {
    // ---------------------------------------------------------------- epilogue (every CTA)
    constexpr int kGroups = kN / 2 / 32;  // groups of 32 columns of one warp
    const int q = warp & 3;
    const int half = (warp - kEpiWarp0) >> 2;
    const uint32_t lane_addr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(half * (kN / 2));
    const int cols = kMode == kUpdate ? args.cp : args.sp;
    int it = 0;
    for (int u = first_unit; u < num_units; u += unit_step, ++it) {
      int b, m, n;
      locate<kMode, kN>(args, u, b, m, n);
      const int i = m * kTileM + static_cast<int>(rank) * kHalf + q * 32 + lane;
      const int j0 = n * kN + half * (kN / 2);
      float alpha = args.alpha, beta = args.beta;
      if (kMode == kGram || (kMode == kUpdate && args.result != nullptr)) {
        const float shift = __ldg(args.shifts + b);
        alpha *= shift;
        if (kMode == kGram) alpha *= shift;
        beta *= shift;
      }
      Added added[2];
      fetch32<kMode>(args, b, i, j0, added[0]);
      if constexpr (kGroups > 1) fetch32<kMode>(args, b, i, j0 + 32, added[1]);
      const int acc = it & 1;
      if (!mbar_wait_cluster(bar(bars->acc_full[acc]), (it >> 1) & 1, abort_flag, args.status,
                             MOSS_STATUS_TIMEOUT_EPILOGUE))
        break;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < kGroups; ++c) {
        uint32_t r[32];
        tmem_ld_32x32b_x32(lane_addr + static_cast<uint32_t>(acc * kN + c * 32), r);
        tmem_wait_ld();
        if (c == kGroups - 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            const uint32_t eb = bar(bars->acc_empty[acc]);
            if (kCtas == 1 || leader)
              mbar_arrive(eb);
            else
              mbar_arrive_cluster(mapa_shared(eb, 0));
          }
        }
        const int j = j0 + c * 32;
        // the update's last rows leave by the whole warp
        if ((kMode == kUpdate ? i - lane : i) < args.r && j < cols) {
          float v[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = __uint_as_float(r[e]);
          finish32<kMode>(args, alpha, beta, b, i, j, kN == 64 ? m != n >> 1 : m != n, added[c & 1], v);
        }
        if constexpr (kMode == kUpdate) __syncwarp();  // lanes past the last row left early
        if (c + 2 < kGroups) fetch32<kMode>(args, b, i, j + 64, added[c & 1]);
      }
    }
  }

  // Leave together (the pair reads and signals each other's shared memory and TMEM).
  tc_fence_before();
  __syncthreads();
  if constexpr (kCtas == 2) {
    if (threadIdx.x == 0) {
      if (*abort_flag) st_shared_cluster_u32(mapa_shared(smem_u32(&bars->abort_flag), rank ^ 1u), 1u);
      mbar_arrive_cluster(mapa_shared(bar(bars->exit_bar), rank ^ 1u));
      const long long start = clock64();
      while (!mbar_try_wait_cluster(bar(bars->exit_bar), 0)) {
        if (clock64() - start > kExitBudgetCycles) {
          report_status(args.status, MOSS_STATUS_TIMEOUT_DRAIN);
          break;
        }
      }
    }
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    if constexpr (kCtas == 2)
      tmem_dealloc_pair(tmem_base, kTmemCols);
    else
      tmem_dealloc(tmem_base, kTmemCols);
  }
}

template <Mode kMode, int kCtas, int kN>
int launch_typed(const CUtensorMap& tl, const CUtensorMap& tr, Args a, cudaStream_t stream) {
  constexpr uint32_t kSmemBytes = Shape<kCtas, kN>::kSmemBytes;
  auto kern = ns_gemm_kernel<kMode, kCtas, kN>;
  static DeviceSetup setup;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kCtas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmemBytes;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int max_groups = 0;
  const int rc = setup("ns_gemm_kernel", &max_groups, [&](int* groups) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
    *groups = sm_count() / kCtas;
    if (e == cudaSuccess && kCtas > 1) {
      cfg.gridDim = dim3(kCtas * *groups);
      int clusters = 0;
      if (cudaOccupancyMaxActiveClusters(&clusters, kern, &cfg) == cudaSuccess && clusters > 0)
        *groups = clusters;
      else
        cudaGetLastError();
    }
    return e;
  });
  if (rc != MOSS_OK) return rc;
  a.tiles_m = (a.r + kHalf * kCtas - 1) / (kHalf * kCtas);
  a.tiles_n = ((kMode == kUpdate ? a.cp : a.sp) + kN - 1) / kN;
  a.tiles = kMode == kUpdate ? a.tiles_m * a.tiles_n : a.tiles_m * (a.tiles_m + 1) / 2 * (kN == 64 ? 2 : 1);
  const int64_t units = static_cast<int64_t>(a.tiles) * a.batch;
  if (units > INT32_MAX) return fail(MOSS_ERR_INVALID_ARGUMENT, "too many matrices to orthogonalize in one call");
  cfg.gridDim = dim3(static_cast<unsigned>(kCtas * std::min<int64_t>(units, max_groups)));
  cfg.stream = stream;
  cfg.numAttrs = 2;  // the kernel before it in the stream is one of this call
  return check_cuda(cudaLaunchKernelEx(&cfg, kern, tl, tr, a), "ns_gemm_kernel");
}

// The tile columns (256: a pair) whose rounds over the GPU take least. Relative cost of a round: a pair tile
// has four times the products of a 128 x 128 one in twice its MMA time; single tiles are bound by what a
// multiprocessor can read, 64 KB a step for 128 columns and 48 KB for 64 (700 and 530 cycles measured).
int tile_columns(Mode mode, const Args& a) {
  const int64_t sms = sm_count();
  auto rounds = [&](int64_t tm, int64_t tn, int64_t slots) {
    const int64_t tiles = mode == kUpdate ? tm * tn : tm * (tm + 1) / 2 * (tn / tm);
    return (tiles * a.batch + slots - 1) / slots;
  };
  const int64_t tm = (a.r + 127) / 128, tn = mode == kUpdate ? a.cp / 128 : tm;
  const int64_t pair = rounds((tm + 1) / 2, (tn + 1) / 2, std::max<int64_t>(1, sms / 2)) * 20;
  const int64_t wide = rounds(tm, tn, sms) * 13;
  const int64_t narrow = rounds(tm, 2 * tn, sms) * 9;
  if (pair <= wide && pair <= narrow) return 256;
  return wide <= narrow ? 128 : 64;
}

template <Mode kMode>
int launch_mode(int columns, const CUtensorMap& tl, const CUtensorMap& tr, const Args& a, cudaStream_t stream) {
  if (columns == 256) return launch_typed<kMode, 2, 256>(tl, tr, a, stream);
  if (columns == 128) return launch_typed<kMode, 1, 128>(tl, tr, a, stream);
  return launch_typed<kMode, 1, 64>(tl, tr, a, stream);
}

}  // namespace

int launch_gemm(Mode mode, const __half* left, const __half* right, const Args& a, cudaStream_t stream) {
  const int columns = tile_columns(mode, a);
  const uint32_t held = columns == 64 ? 64 : 128;  // columns of the right operand in one CTA
  // [batch][r][cols] viewed as {64, r, cols / 64, batch}: a box is rows of 64-wide columns, and what it holds past
  // the matrix's last row or column is zero, whatever the next matrix holds
  auto map = [&](CUtensorMap* m, const __half* p, int cols, uint32_t rows, uint32_t wide) {
    memset(m, 0, sizeof(*m));
    const uint64_t dims[4] = {64, static_cast<uint64_t>(a.r), static_cast<uint64_t>(cols / 64), static_cast<uint64_t>(a.batch)};
    const uint64_t strides[3] = {static_cast<uint64_t>(cols) * 2, 128, static_cast<uint64_t>(a.r) * cols * 2};
    const uint32_t box[4] = {64, rows, wide, 1};
    return gemm::make_map_nd(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, p, 4, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  };
  CUtensorMap tl, tr;
  const bool by_columns = mode == kUpdate;
  if (!map(&tl, left, mode == kGram ? a.cp : a.sp, 128, 2) ||
      !map(&tr, right, mode == kSquare ? a.sp : a.cp, by_columns ? 128 : held, by_columns ? held / 64 : 2))
    return fail(MOSS_ERR_CUDA, "the driver refused a tensor map of the orthogonalised update");
  switch (mode) {
    case kGram:
      return launch_mode<kGram>(columns, tl, tr, a, stream);
    case kSquare:
      return launch_mode<kSquare>(columns, tl, tr, a, stream);
    default:
      return launch_mode<kUpdate>(columns, tl, tr, a, stream);
  }
}

}  // namespace ns
}  // namespace moss
