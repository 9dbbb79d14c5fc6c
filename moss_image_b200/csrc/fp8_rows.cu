// Block-scaled fp8 GEMM for few rows: the weight's output columns in the accumulator's lanes.
//
// With at most 64 rows the product is a walk over the weight, bound by its bytes. Each CTA takes
// 128 output columns (one scale block) of one reduction split, streams their weight tiles by
// TMA through a ring of several blocks, and multiplies them with operands swapped: the 128
// weight columns are the M of tcgen05.mma and the rows its N (16, 32 or 64), so that no tensor
// or shared-memory work is spent on rows that are not there. Splitting the reduction gives
// every SM a share of the weight; the f32 partials are summed in split order.
// Two CTAs fit one SM, so that one streams while the other starts or stores.
//
// Up to 32 rows are quantised here: four warps turn each 128 columns of the rows into codes in the stage
// that holds the weight tiles of the same columns. Every column tile does that again, but for so few
// rows it is less than a launch (2 rows x 3072 -> 18432: 16.4 us a call instead of 18.5).
#include <algorithm>

#include "fp8_args.cuh"
#include "fp8_codes.cuh"

namespace moss {
namespace fp8 {
namespace {

constexpr int kFeatures = 128;
constexpr int kQuantWarp0 = 6;
constexpr int kQuantWarps = 4;
constexpr uint32_t kWBytes = kFeatures * kBlock;
constexpr int kBufs = 4;  // block products in TMEM: the drain's latency hides behind three more

template <int kTN>
struct Ring {
  static constexpr bool kQuantises = kTN <= 32;
  static constexpr int kThreads = (kQuantises ? kQuantWarp0 + kQuantWarps : kQuantWarp0) * 32;
  static constexpr uint32_t kTBytes = kTN * kBlock;
  static constexpr uint32_t kStageBytes = kWBytes + kTBytes;
  static constexpr int kStages = kTN <= 16 ? 6 : kTN <= 32 ? 5 : 4;
  static constexpr uint32_t kDataBytes = kStages * kStageBytes;
  // row scales of the blocks between the quantiser and the epilogue: the ring's and those in TMEM
  static constexpr int kScales = kStages + kBufs;
  static constexpr uint32_t kScaleBytes = kQuantises ? kScales * kTN * 4 : 0;
  static constexpr uint32_t kSmemBytes = kDataBytes + kScaleBytes + 1024 + 256;
  static_assert(2 * (kSmemBytes + 1024) <= 228 * 1024, "two CTAs fit one SM");
};

template <int kStages>
struct Barriers {
  uint64_t full[kStages], empty[kStages], acc_full[kBufs], acc_empty[kBufs], drain;
  uint32_t tmem_base;
  int abort_flag;
};

// Rows r, r + 8, .. of the tile's TN, one half-warp each: their 128 columns of block kb on their way.
template <int kKind, int kTN>
struct RowBlocks {
  static constexpr int kRows = kTN / (2 * kQuantWarps);
  Raw<kKind> raw[kRows];
  __device__ __forceinline__ void fetch(const Args& a, int m0, int kb, int half_warp, int sub) {
    const int64_t c0 = static_cast<int64_t>(kb) * kBlock + sub * 8;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int64_t row = m0 + half_warp + i * 2 * kQuantWarps;
      raw[i] = Raw<kKind>{};
      if (row >= a.M || c0 >= a.x_cols) continue;
      const int64_t at = row * a.x_cols + c0;
      if (a.x_wide) {
        raw[i] = load_raw<kKind>(a.x, at);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (c0 + j >= a.x_cols) break;
          if constexpr (kKind == kF32)
            raw[i].w[j] = __ldg(static_cast<const uint32_t*>(a.x) + at + j);
          else
            raw[i].w[j / 2] |= static_cast<uint32_t>(__ldg(static_cast<const uint16_t*>(a.x) + at + j)) << (16 * (j & 1));
        }
      }
    }
  }
  // Codes into a K-major tile of 128-byte rows (128-byte swizzle), scales beside it.
  __device__ __forceinline__ void put(uint32_t tile, float* scales, int half_warp, int sub) const {
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int r = half_warp + i * 2 * kQuantWarps;
      const float amax = half_warp_max(max_nan(kAmaxFloor, amax_of<kKind>(raw[i])));
      float v[8], scale;
      values_of<kKind>(raw[i], v);
      const uint2 q = block_codes(v, amax, scale);
      asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(tile + r * 128 + (((sub >> 1) ^ (r & 7)) << 4) + (sub & 1) * 8),
                   "r"(q.x), "r"(q.y)
                   : "memory");
      if (sub == 0) scales[r] = scale;
    }
  }
};

template <int kKind, int kTN, typename Bars>
__device__ __forceinline__ void quantise_rows(const Args& args, uint32_t base, float* scales, Bars* bars, int m0, int kb0,
                                              int kb1, int warp, int lane) {
  using R = Ring<kTN>;
  const int half_warp = (warp - kQuantWarp0) * 2 + (lane >> 4), sub = lane & 15;
  // All of this split's columns of the rows are asked for at once: block by block, each would wait for DRAM.
  constexpr int kElem = kKind == kF32 ? 4 : 2, kLines = kBlock * kElem / 128;  // 128-byte lines per row and block
  const int rows = min(kTN, args.M - m0);
  for (int e = (warp - kQuantWarp0) * 32 + lane; e < (kb1 - kb0) * kLines * rows; e += kQuantWarps * 32) {
    const int64_t col = (static_cast<int64_t>(kb0) * kLines + e / rows) * (128 / kElem);
    if (col < args.x_cols)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const uint8_t*>(args.x) +
                                                    ((m0 + e % rows) * args.x_cols + col) * kElem));
  }
  RowBlocks<kKind, kTN> next;
  next.fetch(args, m0, kb0, half_warp, sub);
  int stage = 0;
  uint32_t phase = 0;
  for (int kb = kb0; kb < kb1; ++kb) {
    const RowBlocks<kKind, kTN> now = next;
    if (kb + 1 < kb1) next.fetch(args, m0, kb + 1, half_warp, sub);
    if (!mbar_wait(smem_u32(&bars->empty[stage]), phase ^ 1u, &bars->abort_flag, args.status,
                   MOSS_STATUS_TIMEOUT_CONVERT))
      return;
    now.put(base + stage * R::kStageBytes + kWBytes, scales + (kb - kb0) % R::kScales * kTN, half_warp, sub);
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&bars->full[stage]));
    if (++stage == R::kStages) {
      stage = 0;
      phase ^= 1u;
    }
  }
}

template <bool kDX, int kTN>
__global__ void __launch_bounds__(Ring<kTN>::kThreads, 2)
    fp8_rows_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_w, const Args args) {
  using R = Ring<kTN>;
  constexpr int kStages = R::kStages;
  constexpr uint32_t kTmemCols = kBufs * kTN;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_base = smem_u32(smem_raw);
  const uint32_t base = (raw_base + 1023u) & ~1023u;
  using Bars = Barriers<kStages>;
  static_assert(sizeof(Bars) <= 256, "barrier block too large");
  float* scales = reinterpret_cast<float*>(smem_raw + (base - raw_base) + R::kDataBytes);
  Bars* bars = reinterpret_cast<Bars*>(smem_raw + (base - raw_base) + R::kDataBytes + R::kScaleBytes);
  auto bar = [&](uint64_t& b) { return smem_u32(&b); };
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  const int split = blockIdx.x % args.splits;
  const int tile = blockIdx.x / args.splits;
  const int f0 = (tile / args.tiles_m) * kFeatures;  // the row tiles of one weight tile run side by side
  const int m0 = (tile % args.tiles_m) * kTN;
  const int kb0 = split * args.kb_per_split, kb1 = min(args.kb, kb0 + args.kb_per_split);

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar(bars->full[s]), R::kQuantises ? 1 + kQuantWarps : 1);
      mbar_init(bar(bars->empty[s]), 1);
    }
    for (int s = 0; s < kBufs; ++s) {
      mbar_init(bar(bars->acc_full[s]), 1);
      mbar_init(bar(bars->acc_empty[s]), 4);
    }
    mbar_init(bar(bars->drain), 1);
    bars->abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&bars->tmem_base), kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = bars->tmem_base;
  pdl_trigger();

  if (warp == 0) {
    // ---------------------------------------------------------------- producer
    if (lane == 0) {
      if constexpr (!R::kQuantises) tma_prefetch_desc(&tm_a);
      tma_prefetch_desc(&tm_w);
    }
    // The weight does not depend on the quantiser that runs before: a ring of it is on its way meanwhile.
    const int early = min(kStages, kb1 - kb0);
    auto load_weight = [&](int stage, int kb) {
      mbar_arrive_expect_tx(bar(bars->full[stage]), R::kQuantises ? kWBytes : R::kStageBytes);
      tma_load_2d(base + stage * R::kStageBytes, &tm_w, bar(bars->full[stage]), kDX ? f0 : kb * kBlock,
                  kDX ? kb * kBlock : f0);
    };
    int stage = 0;
    uint32_t phase = 0, used = 0, last_phase = 0;
    if (lane == 0) {
      for (int i = 0; i < early; ++i) load_weight(i, kb0 + i);
      used = (1u << early) - 1u;  // waited for below, even if the loop is left at once
    }
    pdl_wait();
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!mbar_wait(bar(bars->empty[stage]), phase ^ 1u, abort_flag, args.status, MOSS_STATUS_TIMEOUT_LOAD)) break;
      if (lane == 0) {
        if (kb - kb0 >= early) load_weight(stage, kb);
        if constexpr (!R::kQuantises)
          tma_load_2d(base + stage * R::kStageBytes + kWBytes, &tm_a, bar(bars->full[stage]), kb * kBlock, m0);
        last_phase = (last_phase & ~(1u << stage)) | (phase << stage);
      }
      __syncwarp();
      if (++stage == kStages) { stage = 0; phase ^= 1u; }
    }
    if (lane == 0) {  // the copies land before the CTA may leave
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
    // ---------------------------------------------------------------- MMA issuer
    pdl_wait();
    constexpr uint32_t idesc = idesc_e4m3(kDX, false, kFeatures, kTN);
    const uint64_t w_desc0 = step_desc(base, 0, kDX), a_desc0 = step_desc(base + kWBytes, 0, false);
    int stage = 0;
    uint32_t phase = 0;
    bool issued = false;
    for (int kb = kb0; kb < kb1; ++kb) {
      const int it = kb - kb0, acc = it % kBufs;
      if (!mbar_wait(bar(bars->acc_empty[acc]), ((it / kBufs) & 1) ^ 1u, abort_flag, args.status,
                     MOSS_STATUS_TIMEOUT_MMA) ||
          !mbar_wait(bar(bars->full[stage]), phase, abort_flag, args.status, MOSS_STATUS_TIMEOUT_MMA))
        break;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t at_stage = static_cast<uint64_t>(stage) * (R::kStageBytes >> 4);
        const uint32_t d = tmem_base + static_cast<uint32_t>(acc * kTN);
#pragma unroll
        for (int kk = 0; kk < kBlock / 32; ++kk)
          umma_f8(d, w_desc0 + at_stage + kk * ((kDX ? 4096 : 32) >> 4), a_desc0 + at_stage + kk * (32 >> 4), idesc, kk > 0);
        umma_commit(bar(bars->acc_full[acc]));
        umma_commit(bar(bars->empty[stage]));
      }
      issued = true;
      __syncwarp();
      if (++stage == kStages) { stage = 0; phase ^= 1u; }
    }
    if (lane == 0 && issued) {
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
  } else if (R::kQuantises && warp >= kQuantWarp0) {
    // ---------------------------------------------------------------- quantisers
    if constexpr (R::kQuantises) {
      if (args.x_kind == kBF16)
        quantise_rows<kBF16, kTN>(args, base, scales, bars, m0, kb0, kb1, warp, lane);
      else if (args.x_kind == kF16)
        quantise_rows<kF16, kTN>(args, base, scales, bars, m0, kb0, kb1, warp, lane);
      else
        quantise_rows<kF32, kTN>(args, base, scales, bars, m0, kb0, kb1, warp, lane);
    }
  } else {
    // ---------------------------------------------------------------- epilogue
    pdl_wait();
    const int q = warp & 3;
    const int feature = f0 + q * 32 + lane;
    const uint32_t lane_addr = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
    const float* w_scale = args.w_scale + static_cast<int64_t>(f0 / kBlock) * args.ws_col;
    const float bias = args.splits == 1 && args.bias != nullptr && feature < args.Nc
                           ? load_as_float(args.bias, args.bias_kind, feature)
                           : 0.0f;
    float sum[kTN];
#pragma unroll
    for (int j = 0; j < kTN; ++j) sum[j] = 0.0f;
    bool ok = true;
    for (int kb = kb0; kb < kb1; ++kb) {
      const int it = kb - kb0, acc = it % kBufs;
      const float sw = __ldg(w_scale + static_cast<int64_t>(kb) * args.ws_red);
      // the pitch covers whole row tiles: scales past M are read and never used
      const float4* sa = R::kQuantises ? reinterpret_cast<const float4*>(scales + it % R::kScales * kTN)
                                       : reinterpret_cast<const float4*>(args.row_scale + kb * args.row_pitch + m0);
      if (!mbar_wait(bar(bars->acc_full[acc]), (it / kBufs) & 1, abort_flag, args.status,
                     MOSS_STATUS_TIMEOUT_EPILOGUE)) {
        ok = false;
        break;
      }
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < kTN / 16; ++c) {
        uint32_t r[16];
        tmem_ld_32x32b_x16(lane_addr + static_cast<uint32_t>(acc * kTN + c * 16), r);
        float4 s[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] = R::kQuantises ? sa[c * 4 + j] : __ldg(sa + c * 4 + j);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float* t = sum + c * 16 + j * 4;
          t[0] = fmaf(__uint_as_float(r[4 * j]), s[j].x * sw, t[0]);
          t[1] = fmaf(__uint_as_float(r[4 * j + 1]), s[j].y * sw, t[1]);
          t[2] = fmaf(__uint_as_float(r[4 * j + 2]), s[j].z * sw, t[2]);
          t[3] = fmaf(__uint_as_float(r[4 * j + 3]), s[j].w * sw, t[3]);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(bars->acc_empty[acc]));
    }
    if (ok && feature < args.Nc) {
#pragma unroll
      for (int j = 0; j < kTN; ++j) {
        if (m0 + j >= args.M) break;
        const int64_t row = m0 + j;
        if (args.splits > 1)
          args.partial[(split * static_cast<int64_t>(args.M) + row) * args.Nc + feature] = sum[j];
        else
          store_from_float(args.out, args.out_kind, row * args.Nc + feature, sum[j] + bias);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

template <bool kDX, int kTN>
int launch_typed(const CUtensorMap& ta, const CUtensorMap& tw, const Args& a, cudaStream_t stream) {
  auto kern = fp8_rows_kernel<kDX, kTN>;
  static DeviceSetup setup;
  const int rc = setup("fp8_rows_kernel", nullptr, [&](int*) {
    return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Ring<kTN>::kSmemBytes);
  });
  if (rc != MOSS_OK) return rc;
  if (Ring<kTN>::kQuantises) {  // the call's first kernel
    kern<<<static_cast<unsigned>(a.tiles_m * a.tiles_n * a.splits), Ring<kTN>::kThreads, Ring<kTN>::kSmemBytes, stream>>>(
        ta, tw, a);
    return check_cuda(cudaGetLastError(), "fp8_rows_kernel");
  }
  return launch_dependent("fp8_rows_kernel", kern, dim3(static_cast<unsigned>(a.tiles_m * a.tiles_n * a.splits)),
                          dim3(Ring<kTN>::kThreads), Ring<kTN>::kSmemBytes, stream, ta, tw, a);
}

}  // namespace

int launch_rows(bool dx, const Plan& plan, const CUtensorMap& ta, const CUtensorMap& tw, const Args& a,
                cudaStream_t stream) {
  if (plan.tn == 16) return dx ? launch_typed<true, 16>(ta, tw, a, stream) : launch_typed<false, 16>(ta, tw, a, stream);
  if (plan.tn == 32) return dx ? launch_typed<true, 32>(ta, tw, a, stream) : launch_typed<false, 32>(ta, tw, a, stream);
  return dx ? launch_typed<true, 64>(ta, tw, a, stream) : launch_typed<false, 64>(ta, tw, a, stream);
}

}  // namespace fp8
}  // namespace moss
