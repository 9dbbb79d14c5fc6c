// Weight gradients of many features: dW[n, k] = sum over rows m of dY[m, n] * X[m, k], f32 sums on the
// tensor cores (tcgen05.mma.kind::f16).
//
// Both operands are reduced along their rows, so both are read by columns (MN-major) from the layout they have:
// boxes of 64 columns x 128 rows, 128-byte swizzle. Two shapes of one kernel: a CTA pair on 256 x 256 tiles where
// those fill the GPU, one CTA on 128 x 128 tiles with the reduction split where they do not. Warp 0 streams the
// boxes by TMA, warp 1 issues the MMAs into one of two TMEM accumulators, warps 2-9 drain the other. Split sums
// leave as f32 and are added in split order by a second kernel. Bound by the tensor cores: 9216 rows, 3072 x 3072: 107 us,
// 1.63 PFLOP/s in short runs.
#include <algorithm>
#include <cstring>

#include "codes_args.cuh"

namespace moss {
namespace codes {
namespace {

constexpr int kHalf = 128;  // rows of dW and columns of it that one CTA reads operands for
constexpr int kEpiWarp0 = 2;
constexpr int kEpiWarps = 8;  // two per quarter of the lanes, each with half of the columns
constexpr int kThreads = (kEpiWarp0 + kEpiWarps) * 32;
constexpr int kStages = 3;
constexpr uint32_t kBoxBytes = 64 * kStep * 2;         // 16 KB: 64 columns of 128 rows
constexpr uint32_t kOperandBytes = 2 * kBoxBytes;      // 128 columns
constexpr uint32_t kStageBytes = 2 * kOperandBytes;
constexpr uint32_t kDataBytes = kStages * kStageBytes;
constexpr uint32_t kSmemBytes = kDataBytes + 1024 + 512;
static_assert(kSmemBytes <= 227 * 1024, "rings exceed the shared memory a CTA may use");
// The final wait for the peer outlasts every other bounded wait of the pair.
constexpr long long kExitBudgetCycles = (kStages + 4) * kWaitBudgetCycles;

struct Barriers {
  uint64_t full[kStages];   // leader: both CTAs' operands landed
  uint64_t empty[kStages];  // local
  uint64_t acc_full[2];     // local
  uint64_t acc_empty[2];    // leader
  uint64_t drain;
  uint64_t exit_bar;
  uint32_t tmem_base;
  int abort_flag;
};
static_assert(sizeof(Barriers) <= 512, "barrier block too large");

// A warp's 32 x 32 block of 16-bit results, lane by lane a row, written by columns: rows of any alignment. Turned by
// shuffles within each half of the warp: word k of lane l becomes word l of lane k.
template <int K>
__device__ __forceinline__ void store_turned(const Args& a, int i0, int j, const float (&v)[32]) {
  const int lane = threadIdx.x & 31;
  uint32_t w[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) w[e] = gemm::pack2_kind<K>(v[2 * e], v[2 * e + 1]);
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
  const int first = i0 + (lane & 16), rows = min(16, a.N - first);
  const int col = j + 2 * (lane & 15);
  uint16_t* to = static_cast<uint16_t*>(a.out) + static_cast<int64_t>(first) * a.K + col;
  const bool words = a.K % 2 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 3) == 0;
#pragma unroll
  for (int k = 0; k < 16; ++k, to += a.K) {
    if (k >= rows || col >= a.K) continue;
    if (words) {
      *reinterpret_cast<uint32_t*>(to) = w[k];
    } else {
      to[0] = static_cast<uint16_t>(w[k] & 0xffffu);
      if (col + 1 < a.K) to[1] = static_cast<uint16_t>(w[k] >> 16);
    }
  }
}

// 32 consecutive sums of row i; the whole warp takes part.
__device__ __forceinline__ void finish32(const Args& a, int split, int i, int j, const float (&v)[32]) {
  const int lane = threadIdx.x & 31;
  if (a.splits > 1) {
    float* to = a.partial + (split * a.part_rows + i) * a.part_cols + j;
#pragma unroll
    for (int h = 0; h < 32; h += 8) {
      uint32_t w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = __float_as_uint(v[h + e]);
      gemm::stg256(to + h, w);
    }
    return;
  }
  if (j >= a.K || i - lane >= a.N) return;  // the same for the whole warp
  if (a.out_kind == kF32) {
    if (i >= a.N) return;
    float* to = static_cast<float*>(a.out) + static_cast<int64_t>(i) * a.K + j;
    if (j + 32 <= a.K && a.K % 8 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 31) == 0) {
#pragma unroll
      for (int h = 0; h < 32; h += 8) {
        uint32_t w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = __float_as_uint(v[h + e]);
        gemm::stg256(to + h, w);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 32; ++e)
        if (j + e < a.K) to[e] = v[e];
    }
    return;
  }
  if (j + 32 <= a.K && a.K % 16 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 31) == 0) {
    if (i >= a.N) return;
    uint16_t* to = static_cast<uint16_t*>(a.out) + static_cast<int64_t>(i) * a.K + j;
#pragma unroll
    for (int h = 0; h < 32; h += 16) {
      uint32_t w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        w[e] = a.out_kind == kBF16 ? gemm::pack2_kind<kBF16>(v[h + 2 * e], v[h + 2 * e + 1])
                                   : gemm::pack2_kind<kF16>(v[h + 2 * e], v[h + 2 * e + 1]);
      gemm::stg256(to + h, w);
    }
  } else if (a.out_kind == kBF16) {
    store_turned<kBF16>(a, i - lane, j, v);
  } else {
    store_turned<kF16>(a, i - lane, j, v);
  }
}

template <int K, int kCtas>
__global__ void __launch_bounds__(kThreads, 1)
    codes_gemm_kernel(const __grid_constant__ CUtensorMap tm_y, const __grid_constant__ CUtensorMap tm_x, const Args args) {
  constexpr int kTile = kHalf * kCtas;
  constexpr uint32_t kTmemCols = 2 * kTile;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_base = smem_u32(smem_raw);
  const uint32_t base = (raw_base + 1023u) & ~1023u;
  Barriers* bars = reinterpret_cast<Barriers*>(smem_raw + (base - raw_base) + kDataBytes);
  auto bar = [&](uint64_t& b) { return smem_u32(&b); };
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = kCtas == 2 ? cluster_ctarank() : 0;
  const bool leader = rank == 0;
  const int first_unit = blockIdx.x / kCtas;
  const int unit_step = gridDim.x / kCtas;
  const int num_units = args.tiles_m * args.tiles_n * args.splits;
  const int steps = (args.M + kStep - 1) / kStep;

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

  // unit u: split u % splits of tile u / splits
  auto locate = [&](int u, int& m_blk, int& n_blk, int& first, int& end) {
    const int tile = args.splits == 1 ? u : u / args.splits, split = u - tile * args.splits;
    gemm::tile_coords(tile, args.tiles_m, args.tiles_n, m_blk, n_blk, args.group_m);
    first = split * args.per_split;
    end = min(steps, first + args.per_split);
    return split;
  };

  if (warp == 0) {
    // ---------------------------------------------------------------- producer (every CTA)
    if (lane == 0) {
      tma_prefetch_desc(&tm_y);
      tma_prefetch_desc(&tm_x);
    }
    int stage = 0;
    uint32_t phase = 0, used = 0, last_phase = 0;
    bool ok = true;
    for (int u = first_unit; u < num_units && ok; u += unit_step) {
      int m_blk, n_blk, first, end;
      locate(u, m_blk, n_blk, first, end);
      const int y0 = m_blk * kTile + static_cast<int>(rank) * kHalf;
      const int x0 = n_blk * kTile + static_cast<int>(rank) * kHalf;
      for (int s = first; s < end; ++s) {
        if (!mbar_wait_cluster(bar(bars->empty[stage]), phase ^ 1u, abort_flag, args.status, MOSS_STATUS_TIMEOUT_LOAD)) {
          ok = false;
          break;
        }
        if (lane == 0) {
          const uint32_t dst = base + stage * kStageBytes;
          if constexpr (kCtas == 2) {
            // the leader's barrier counts both CTAs' bytes; the peer's copies signal it too
            if (leader) mbar_arrive_expect_tx(bar(bars->full[stage]), kCtas * kStageBytes);
            const uint32_t fb = mapa_shared(bar(bars->full[stage]), 0);
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              tma_load_2d_pair(dst + b * kBoxBytes, &tm_y, fb, y0 + b * 64, s * kStep);
              tma_load_2d_pair(dst + kOperandBytes + b * kBoxBytes, &tm_x, fb, x0 + b * 64, s * kStep);
            }
          } else {
            mbar_arrive_expect_tx(bar(bars->full[stage]), kStageBytes);
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              tma_load_2d(dst + b * kBoxBytes, &tm_y, bar(bars->full[stage]), y0 + b * 64, s * kStep);
              tma_load_2d(dst + kOperandBytes + b * kBoxBytes, &tm_x, bar(bars->full[stage]), x0 + b * 64, s * kStep);
            }
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
      constexpr uint32_t idesc = umma_idesc_f16_ab(K == kBF16 ? 1u : 0u, true, true, kTile, kTile);
      // [boxes of 64 columns][128 rows]: 16 rows of the reduction are 2048 bytes further
      const uint64_t y_desc0 = umma_desc_sw128(base, kBoxBytes, 1024);
      const uint64_t x_desc0 = umma_desc_sw128(base + kOperandBytes, kBoxBytes, 1024);
      int stage = 0, it = 0;
      uint32_t phase = 0;
      bool ok = true, issued = false;
      for (int u = first_unit; u < num_units && ok; u += unit_step, ++it) {
        int m_blk, n_blk, first, end;
        locate(u, m_blk, n_blk, first, end);
        const int acc = it & 1;
        if (!mbar_wait_cluster(bar(bars->acc_empty[acc]), ((it >> 1) & 1) ^ 1u, abort_flag, args.status,
                               MOSS_STATUS_TIMEOUT_MMA))
          break;
        tc_fence_after();
        const uint32_t d = tmem_base + static_cast<uint32_t>(acc * kTile);
        for (int s = first; s < end; ++s) {
          if (!mbar_wait_cluster(bar(bars->full[stage]), phase, abort_flag, args.status, MOSS_STATUS_TIMEOUT_MMA)) {
            ok = false;
            break;
          }
          tc_fence_after();
          if (elect_one()) {
            const uint64_t at_stage = static_cast<uint64_t>(stage) * (kStageBytes >> 4);
#pragma unroll
            for (int kk = 0; kk < kStep / 16; ++kk) {
              const uint64_t yd = y_desc0 + at_stage + kk * (2048 >> 4);
              const uint64_t xd = x_desc0 + at_stage + kk * (2048 >> 4);
              if constexpr (kCtas == 2)
                umma_f16_pair(d, yd, xd, idesc, (s > first || kk > 0) ? 1u : 0u);
              else
                umma_f16(d, yd, xd, idesc, (s > first || kk > 0) ? 1u : 0u);
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
    constexpr int kGroups = kTile / 2 / 32;  // groups of 32 columns of one warp
    const int q = warp & 3;
    const int half = (warp - kEpiWarp0) >> 2;
    const uint32_t lane_addr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(half * (kTile / 2));
    int it = 0;
    for (int u = first_unit; u < num_units; u += unit_step, ++it) {
      int m_blk, n_blk, first, end;
      const int split = locate(u, m_blk, n_blk, first, end);
      const int i = m_blk * kTile + static_cast<int>(rank) * kHalf + q * 32 + lane;
      const int j0 = n_blk * kTile + half * (kTile / 2);
      const int acc = it & 1;
      if (!mbar_wait_cluster(bar(bars->acc_full[acc]), (it >> 1) & 1, abort_flag, args.status,
                             MOSS_STATUS_TIMEOUT_EPILOGUE))
        break;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < kGroups; ++c) {
        uint32_t r[32];
        tmem_ld_32x32b_x32(lane_addr + static_cast<uint32_t>(acc * kTile + c * 32), r);
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
        float v[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = __uint_as_float(r[e]);
        finish32(args, split, i, j0 + c * 32, v);
        __syncwarp();  // lanes past the last row left early
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

template <int K, int kCtas>
int launch_typed(const CUtensorMap& ty, const CUtensorMap& tx, const Args& a, cudaStream_t stream) {
  auto kern = codes_gemm_kernel<K, kCtas>;
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
  const int rc = setup("codes_gemm_kernel", &max_groups, [&](int* groups) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
    *groups = device_sm_count() / kCtas;
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
  const int64_t units = static_cast<int64_t>(a.tiles_m) * a.tiles_n * a.splits;
  cfg.gridDim = dim3(static_cast<unsigned>(kCtas * std::max<int64_t>(1, std::min<int64_t>(units, max_groups))));
  cfg.stream = stream;
  cfg.numAttrs = 2;  // the kernel before it in the stream is one of this call
  return check_cuda(cudaLaunchKernelEx(&cfg, kern, ty, tx, a), "codes_gemm_kernel");
}

}  // namespace

int launch_gemm(bool pair, int kind, const CUtensorMap& ty, const CUtensorMap& tx, const Args& a, cudaStream_t stream) {
  if (kind == kBF16) return pair ? launch_typed<kBF16, 2>(ty, tx, a, stream) : launch_typed<kBF16, 1>(ty, tx, a, stream);
  return pair ? launch_typed<kF16, 2>(ty, tx, a, stream) : launch_typed<kF16, 1>(ty, tx, a, stream);
}

}  // namespace codes
}  // namespace moss
