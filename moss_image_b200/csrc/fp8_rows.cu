// Block-scaled fp8 GEMM for few rows: the weight's output columns in the accumulator's lanes.
//
// With at most 64 rows the product is a walk over the weight, bound by its bytes. Each CTA takes
// 128 output columns (one scale block) of one reduction split, streams their weight tiles by
// TMA through a ring of several blocks, and multiplies them with operands swapped: the 128
// weight columns are the M of tcgen05.mma and the rows its N (16, 32 or 64), so that no tensor
// or shared-memory work is spent on rows that are not there. Splitting the reduction gives
// every SM a share of the weight; the f32 partials are summed in split order.
// Two CTAs fit one SM, so that one streams while the other starts or stores.
#include <algorithm>
#include <mutex>

#include "fp8_args.cuh"

namespace moss {
namespace fp8 {
namespace {

constexpr int kFeatures = 128;
constexpr int kThreads = 6 * 32;
constexpr uint32_t kWBytes = kFeatures * kBlock;
constexpr int kBufs = 4;  // block products in TMEM: the drain's latency hides behind three more

template <int kTN>
struct Ring {
  static constexpr uint32_t kTBytes = kTN * kBlock;
  static constexpr uint32_t kStageBytes = kWBytes + kTBytes;
  static constexpr int kStages = kTN <= 16 ? 6 : kTN <= 32 ? 5 : 4;
  static constexpr uint32_t kDataBytes = kStages * kStageBytes;
  static constexpr uint32_t kSmemBytes = kDataBytes + 1024 + 256;
  static_assert(2 * (kSmemBytes + 1024) <= 228 * 1024, "two CTAs fit one SM");
};

template <int kStages>
struct Barriers {
  uint64_t full[kStages], empty[kStages], acc_full[kBufs], acc_empty[kBufs], drain;
  uint32_t tmem_base;
  int abort_flag;
};

template <bool kDX, int kTN>
__global__ void __launch_bounds__(kThreads, 2)
    fp8_rows_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_w, const Args args) {
  using R = Ring<kTN>;
  constexpr int kStages = R::kStages;
  constexpr uint32_t kTmemCols = kBufs * kTN;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_base = smem_u32(smem_raw);
  const uint32_t base = (raw_base + 1023u) & ~1023u;
  using Bars = Barriers<kStages>;
  static_assert(sizeof(Bars) <= 256, "barrier block too large");
  Bars* bars = reinterpret_cast<Bars*>(smem_raw + (base - raw_base) + R::kDataBytes);
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
      mbar_init(bar(bars->full[s]), 1);
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
      tma_prefetch_desc(&tm_a);
      tma_prefetch_desc(&tm_w);
    }
    // The weight does not depend on the quantiser that runs before: a ring of it is on its way meanwhile.
    const int early = min(kStages, kb1 - kb0);
    auto load_weight = [&](int stage, int kb) {
      mbar_arrive_expect_tx(bar(bars->full[stage]), R::kStageBytes);
      tma_load_2d(base + stage * R::kStageBytes, &tm_w, bar(bars->full[stage]), kDX ? f0 : kb * kBlock,
                  kDX ? kb * kBlock : f0);
    };
    if (lane == 0)
      for (int i = 0; i < early; ++i) load_weight(i, kb0 + i);
    pdl_wait();
    int stage = 0;
    uint32_t phase = 0, used = 0, last_phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!mbar_wait(bar(bars->empty[stage]), phase ^ 1u, abort_flag, args.status, MOSS_STATUS_TIMEOUT_LOAD)) break;
      if (lane == 0) {
        if (kb - kb0 >= early) load_weight(stage, kb);
        tma_load_2d(base + stage * R::kStageBytes + kWBytes, &tm_a, bar(bars->full[stage]), kb * kBlock, m0);
        used |= 1u << stage;
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
  } else {
    // ---------------------------------------------------------------- epilogue
    pdl_wait();
    const int q = warp & 3;
    const int feature = f0 + q * 32 + lane;
    const uint32_t lane_addr = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
    const float* w_scale = args.w_scale + static_cast<int64_t>(f0 / kBlock) * args.ws_col;
    float sum[kTN];
#pragma unroll
    for (int j = 0; j < kTN; ++j) sum[j] = 0.0f;
    bool ok = true;
    for (int kb = kb0; kb < kb1; ++kb) {
      const int it = kb - kb0, acc = it % kBufs;
      const float sw = __ldg(w_scale + static_cast<int64_t>(kb) * args.ws_red);
      // the pitch covers whole row tiles: scales past M are read and never used
      const float4* sa = reinterpret_cast<const float4*>(args.row_scale + kb * args.row_pitch + m0);
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
        for (int j = 0; j < 4; ++j) s[j] = __ldg(sa + c * 4 + j);
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
      const float bias =
          args.splits == 1 && args.bias != nullptr ? load_as_float(args.bias, args.bias_kind, feature) : 0.0f;
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
  static std::once_flag once;
  static cudaError_t attr_err = cudaSuccess;
  std::call_once(once, [&] {
    attr_err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Ring<kTN>::kSmemBytes);
  });
  MOSS_CUDA_TRY(attr_err);
  return launch_dependent("fp8_rows_kernel", kern, dim3(static_cast<unsigned>(a.tiles_m * a.tiles_n * a.splits)),
                          dim3(kThreads), Ring<kTN>::kSmemBytes, stream, ta, tw, a);
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
