// Block-scaled fp8 GEMM with the rows (tokens) in the accumulator's lanes, for sm_100a.
//
// Two shapes of one kernel:
//   * a CTA pair (cta_group::2) on 256 x 256 output tiles, for problems that fill the GPU with
//     them: every operand byte in shared memory feeds twice the products of a 128 x 128 tile;
//   * one CTA on 128 x 128 tiles, for those that do not.
// Warp 0 streams 128-wide reduction blocks by TMA (both operands straight from their 8-bit
// storage: no decode), warp 1 issues four 32-wide tcgen05.mma per block into one of two
// TMEM buffers, and eight warps take each finished block out of TMEM, multiply it by its two
// scales and add it into f32 registers while the tensor cores run the next block. The
// grad-input reads the same [out, in] weight codes: there the tile is MN-major.
//
// What bounds it: the MMAs of a 256 x 256 x 128 block take 715 cycles here (512 by the pipe's rate), and the
// epilogue keeps pace with them; the staging of a finished tile is the rest. 9216 x 3072 -> 12288: 310 us
// or 2.25 PFLOP/s in short runs (the MMAs alone 233 us; cuBLAS with one scale per tensor 245; a call in a long loop, the
// rows quantised first and the clock under the power cap, 385). What each part of the
// epilogue is there for: with 16 warps of 64 sums it lost 7%, with direct row stores 20%, with packed
// f32x2 multiply-adds 25% (register moves), with a scale load waited for in the loop 15%.
#include <algorithm>
#include <cstring>

#include "dequant.cuh"
#include "fp8_args.cuh"

namespace moss {
namespace fp8 {
namespace {

constexpr int kHalf = 128;  // rows of A and columns (or half of the pair's columns) of W per CTA
constexpr int kEpiWarp0 = 4;
constexpr int kEpiWarps = 8;
constexpr int kThreads = (kEpiWarp0 + kEpiWarps) * 32;
// Registers of the pair kernel's warpgroups: 384 threads start with 168 each; the first warpgroup
// (producer and issuer) gives its share to the two that hold 128 sums and two loads in flight a thread.
constexpr int kIssueRegs = 40, kEpiRegs = 232;
static_assert(kIssueRegs + 2 * kEpiRegs <= 3 * 168, "a larger split would wait forever");
constexpr int kStages = 4;
constexpr uint32_t kTileBytes = kHalf * kBlock;      // 16 KB: 128 rows of 128 bytes
constexpr uint32_t kStageBytes = 2 * kTileBytes;     // A rows and W columns
constexpr uint32_t kBoxBytes = kHalf * 64 * 2;       // one store box: 128 rows of 64 16-bit outputs
constexpr uint32_t kRingBytes = kStages * kStageBytes;
constexpr uint32_t kDataBytes = kRingBytes + 4 * kBoxBytes;
constexpr uint32_t kBiasBytes = 2 * kHalf * 4;       // f32 bias of each epilogue warpgroup's columns
constexpr uint32_t kSmemBytes = kDataBytes + kBiasBytes + 1024 + 512;
// The final wait for the peer outlasts every other bounded wait of the pair (each gives up within
// kWaitBudgetCycles, the drain of the ring within kStages more).
constexpr long long kExitBudgetCycles = (kStages + 4) * kWaitBudgetCycles;
static_assert(kSmemBytes <= 227 * 1024, "rings exceed the shared memory a CTA may use");

struct Barriers {
  uint64_t full[kStages];   // leader: both CTAs' operands of a stage landed
  uint64_t empty[kStages];  // local: stage free (MMA commit)
  uint64_t acc_full[2];     // local: block product ready (MMA commit)
  uint64_t acc_empty[2];    // leader: block product taken by every epilogue warp
  uint64_t out_free[2];     // local, by warpgroup: its store boxes are free and its bias is there
  uint64_t out_full[2];     // local: its outputs are staged
  uint64_t drain;           // leader: all MMAs retired
  uint64_t exit_bar;        // local: peer finished
  uint32_t tmem_base;
  int abort_flag;
};
static_assert(sizeof(Barriers) <= 512, "barrier block too large");

// tcgen05.wait::ld that also orders the use of the loaded registers behind it.
__device__ __forceinline__ void tmem_wait_ld_of(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}

// 32 outputs of one row, rounded, as chunks 4 h .. 4 h + 3 of a store box (128-byte swizzle).
template <int kKind>
__device__ __forceinline__ void stage32(uint32_t box, int row, int h, const float (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint4 w;
    w.x = gemm::pack2_kind<kKind>(v[8 * i], v[8 * i + 1]);
    w.y = gemm::pack2_kind<kKind>(v[8 * i + 2], v[8 * i + 3]);
    w.z = gemm::pack2_kind<kKind>(v[8 * i + 4], v[8 * i + 5]);
    w.w = gemm::pack2_kind<kKind>(v[8 * i + 6], v[8 * i + 7]);
    // no memory clobber: the next group's bias may be read meanwhile (a proxy fence or a warp barrier follows)
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(box + row * 128 + (((4 * h + i) ^ (row & 7)) << 4)),
                 "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w));
  }
}

// A warp's 32 x 32 block of f32 outputs, lane by lane a row, plus the bias: turned in the warp's `slice` of the store
// boxes, so that a row leaves as its 128 consecutive bytes. (Each lane along its own row: 9216 x 3072 -> 12288
// took 1340 us, 430 now.)
constexpr int kSlicePitch = 36;  // floats: 16-byte rows, whose quarters meet in different banks
constexpr uint32_t kSliceBytes = 2 * kBoxBytes / 4;
static_assert(32 * kSlicePitch * 4 <= kSliceBytes, "a turned block fits a warp's slice");
__device__ __forceinline__ void store_f32_block(const Args& args, float* slice, int row0, int col, const float (&v)[32]) {
  const int lane = threadIdx.x & 31;
  __syncwarp();  // the block before has been read
#pragma unroll
  for (int j = 0; j < 32; j += 4)
    *reinterpret_cast<float4*>(slice + lane * kSlicePitch + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
  __syncwarp();
  float* out = static_cast<float*>(args.out) + static_cast<int64_t>(row0) * args.Nc + col;
  const int rows = min(32, args.M - row0);
  auto bias = [&](int j) {
    return args.bias != nullptr && col + j < args.Nc ? load_as_float(args.bias, args.bias_kind, col + j) : 0.0f;
  };
  if (args.Nc % 4 == 0 && (reinterpret_cast<uintptr_t>(args.out) & 15) == 0) {
    const int j = (lane & 7) * 4;
    if (col + j >= args.Nc) return;
    const float b[4] = {bias(j), bias(j + 1), bias(j + 2), bias(j + 3)};
#pragma unroll 4
    for (int i = lane >> 3; i < rows; i += 4) {
      const float4 w = *reinterpret_cast<const float4*>(slice + i * kSlicePitch + j);
      *reinterpret_cast<float4*>(out + static_cast<int64_t>(i) * args.Nc + j) =
          make_float4(w.x + b[0], w.y + b[1], w.z + b[2], w.w + b[3]);
    }
  } else {
    if (col + lane >= args.Nc) return;
    const float b = bias(lane);
#pragma unroll 4
    for (int i = 0; i < rows; ++i) out[static_cast<int64_t>(i) * args.Nc + lane] = slice[i * kSlicePitch + lane] + b;
  }
}

// kF32Out: f32 outputs that are not split (a variant of its own, since its code costs the others registers: 1%).
template <bool kDX, int kCtas, bool kF32Out>
__global__ void __launch_bounds__(kThreads, 1)
    fp8_gemm_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_w,
                    const __grid_constant__ CUtensorMap tm_out, const Args args) {
  constexpr int kTileM = kHalf * kCtas;
  constexpr int kTileN = kHalf * kCtas;
  constexpr int kCols = kTileN / 2;  // accumulator columns of one epilogue thread
  constexpr uint32_t kTmemCols = 2 * kTileN;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_base = smem_u32(smem_raw);
  const uint32_t base = (raw_base + 1023u) & ~1023u;
  float* const bias_smem = reinterpret_cast<float*>(smem_raw + (base - raw_base) + kDataBytes);
  Barriers* bars = reinterpret_cast<Barriers*>(smem_raw + (base - raw_base) + kDataBytes + kBiasBytes);
  auto bar = [&](uint64_t& b) { return smem_u32(&b); };
  volatile int* abort_flag = &bars->abort_flag;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = kCtas == 2 ? cluster_ctarank() : 0;
  const bool leader = rank == 0;
  const int first_unit = blockIdx.x / kCtas;
  const int unit_step = gridDim.x / kCtas;
  const int num_units = args.tiles_m * args.tiles_n * args.splits;
  // outputs that are rounded here: staged in shared memory, whichever way they leave it
  const bool staged = !kF32Out && args.splits == 1;
  const gemm::TileWalk walk(args.tiles_m, args.tiles_n, args.group_m);

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar(bars->full[s]), 1);
      mbar_init(bar(bars->empty[s]), 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(bar(bars->acc_full[s]), 1);
      mbar_init(bar(bars->acc_empty[s]), kCtas * kEpiWarps);
    }
    for (int h = 0; h < 2; ++h) {
      mbar_init(bar(bars->out_free[h]), 1);
      mbar_init(bar(bars->out_full[h]), 4);
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
  if constexpr (kCtas == 2)  // both CTAs' barriers exist before any arrival from the peer
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  else
    __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = bars->tmem_base;
  pdl_trigger();
  pdl_wait();

  if (warp < kEpiWarp0) {
    if constexpr (kCtas == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
    if (warp == 0) {
      // ---------------------------------------------------------------- producer (every CTA)
      if (lane == 0) {
        tma_prefetch_desc(&tm_a);
        tma_prefetch_desc(&tm_w);
      }
      int stage = 0;
      uint32_t phase = 0, used = 0, last_phase = 0;
      bool ok = true;
      for (int u = first_unit; u < num_units && ok; u += unit_step) {
        const int tile = args.splits == 1 ? u : u / args.splits, split = u - tile * args.splits;
        int m_blk, n_blk;
        walk.at(tile, m_blk, n_blk);
        const int m0 = m_blk * kTileM + static_cast<int>(rank) * kHalf;
        const int n0 = n_blk * kTileN + static_cast<int>(rank) * kHalf;
        const int kb1 = min(args.kb, (split + 1) * args.kb_per_split);
        for (int kb = split * args.kb_per_split; kb < kb1; ++kb) {
          if (!mbar_wait_cluster(bar(bars->empty[stage]), phase ^ 1u, abort_flag, args.status,
                                 MOSS_STATUS_TIMEOUT_LOAD)) {
            ok = false;
            break;
          }
          if (lane == 0) {
            const uint32_t a_dst = base + stage * kStageBytes;
            const int wx = kDX ? n0 : kb * kBlock, wy = kDX ? kb * kBlock : n0;
            if constexpr (kCtas == 2) {
              // the leader's barrier counts both CTAs' bytes; the peer's copies signal it too
              if (leader) mbar_arrive_expect_tx(bar(bars->full[stage]), kCtas * kStageBytes);
              const uint32_t fb = mapa_shared(bar(bars->full[stage]), 0);
              tma_load_2d_pair(a_dst, &tm_a, fb, kb * kBlock, m0);
              tma_load_2d_pair(a_dst + kTileBytes, &tm_w, fb, wx, wy);
            } else {
              mbar_arrive_expect_tx(bar(bars->full[stage]), kStageBytes);
              tma_load_2d(a_dst, &tm_a, bar(bars->full[stage]), kb * kBlock, m0);
              tma_load_2d(a_dst + kTileBytes, &tm_w, bar(bars->full[stage]), wx, wy);
            }
            used |= 1u << stage;
            last_phase = (last_phase & ~(1u << stage)) | (phase << stage);
          }
          __syncwarp();
          if (++stage == kStages) { stage = 0; phase ^= 1u; }
        }
      }
      // The copies land before the CTA may leave. The leader sees the peer's too, and the peer
      // leaves only after the leader's exit arrival.
      if (lane == 0 && leader) {
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
        constexpr uint32_t idesc = idesc_e4m3(false, kDX, kTileM, kTileN);
        // descriptors of the first stage; every other differs by multiples of 16 bytes in the address field
        const uint64_t a_desc0 = step_desc(base, 0, false), w_desc0 = step_desc(base + kTileBytes, 0, kDX);
        int stage = 0, it = 0;
        uint32_t phase = 0;
        bool ok = true, issued = false;
        for (int u = first_unit; u < num_units && ok; u += unit_step) {
          const int split = args.splits == 1 ? 0 : u % args.splits;
          const int kb1 = min(args.kb, (split + 1) * args.kb_per_split);
          for (int kb = split * args.kb_per_split; kb < kb1 && ok; ++kb, ++it) {
            const int buf = it & 1;
            // operands first: they are there long before the accumulator, whose wait is the critical one
            if (!mbar_wait_cluster(bar(bars->full[stage]), phase, abort_flag, args.status, MOSS_STATUS_TIMEOUT_MMA) ||
                !mbar_wait_cluster(bar(bars->acc_empty[buf]), ((it >> 1) & 1) ^ 1u, abort_flag, args.status,
                                   MOSS_STATUS_TIMEOUT_MMA)) {
              ok = false;
              break;
            }
            tc_fence_after();
            if (elect_one()) {
              const uint64_t at_stage = static_cast<uint64_t>(stage) * (kStageBytes >> 4);
              const uint32_t d = tmem_base + static_cast<uint32_t>(buf * kTileN);
#pragma unroll
              for (int kk = 0; kk < kBlock / 32; ++kk) {
                const uint64_t ad = a_desc0 + at_stage + kk * (32 >> 4);
                const uint64_t wd = w_desc0 + at_stage + kk * ((kDX ? 4096 : 32) >> 4);
                if constexpr (kCtas == 2)
                  umma_f8_pair(d, ad, wd, idesc, kk > 0);
                else
                  umma_f8(d, ad, wd, idesc, kk > 0);
              }
              if constexpr (kCtas == 2) {
                umma_commit_pair_mc(bar(bars->acc_full[buf]), 0x3);
                umma_commit_pair_mc(bar(bars->empty[stage]), 0x3);
              } else {
                umma_commit(bar(bars->acc_full[buf]));
                umma_commit(bar(bars->empty[stage]));
              }
            }
            issued = true;
            __syncwarp();
            if (++stage == kStages) { stage = 0; phase ^= 1u; }
          }
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
    } else if (staged) {
      // ---------------------------------------------------------------- store warps (every CTA)
      // Warp 2 + h serves epilogue warpgroup h: it brings the bias, and issues the stores, whose queue
      // would hold an epilogue warp up for a thousand cycles a tile.
      const int h = warp - 2;
      int it = 0;
      for (int u = first_unit; u < num_units; u += unit_step, ++it) {
        int m_blk, n_blk;
        walk.at(u, m_blk, n_blk);
        const int row0 = m_blk * kTileM + static_cast<int>(rank) * kHalf;
        const int col0 = n_blk * kTileN + h * kCols;
        for (int j = lane; j < kCols; j += 32)
          bias_smem[h * kHalf + j] =
              args.bias != nullptr && col0 + j < args.Nc ? load_as_float(args.bias, args.bias_kind, col0 + j) : 0.0f;
        if (lane == 0) bulk_wait_read();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(bars->out_free[h]));
        if (!mbar_wait(bar(bars->out_full[h]), it & 1, abort_flag, args.status, MOSS_STATUS_TIMEOUT_EPILOGUE)) break;
        if (args.tma_out != 0 && lane == 0) {
          const uint32_t boxes = base + kRingBytes + h * 2 * kBoxBytes;
#pragma unroll
          for (int p = 0; p < kCols / 64; ++p)
            if (row0 < args.M && col0 + p * 64 < args.Nc) tma_store_2d(&tm_out, boxes + p * kBoxBytes, col0 + p * 64, row0);
          bulk_commit();
        }
      }
      if (lane == 0) bulk_wait();
    }
  } else {
    // ---------------------------------------------------------------- epilogue (every CTA)
    if constexpr (kCtas == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kEpiRegs));
    const int q = warp & 3;
    const int half = (warp - kEpiWarp0) >> 2;
    const uint32_t lane_addr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(half * kCols);
    // acc_empty[0] of the leader, as this CTA sees it; acc_empty[1] is 8 bytes further
    const uint32_t release = kCtas == 2 ? mapa_shared(bar(bars->acc_empty[0]), 0) : bar(bars->acc_empty[0]);
    const uint32_t boxes = base + kRingBytes + half * 2 * kBoxBytes;
    int it = 0, tiles_done = 0;
    bool ok = true;
    for (int u = first_unit; u < num_units && ok; u += unit_step) {
      const int tile = args.splits == 1 ? u : u / args.splits, split = u - tile * args.splits;
      int m_blk, n_blk;
      walk.at(tile, m_blk, n_blk);
      const int row = m_blk * kTileM + static_cast<int>(rank) * kHalf + q * 32 + lane;
      const int col0 = n_blk * kTileN + half * kCols;  // this thread's columns: all in one weight block
      const int kb0 = split * args.kb_per_split, kb1 = min(args.kb, kb0 + args.kb_per_split);
      float sum[kCols];
#pragma unroll
      for (int j = 0; j < kCols; ++j) sum[j] = 0.0f;
      // The scales come from L2, two blocks ahead, in two slots that take turns (the loop body exists once
      // for each): a copy from slot to slot would wait for the load.
      const float* row_scale = args.row_scale + kb0 * args.row_pitch + min(row, args.M - 1);
      const float* w_scale = args.w_scale + static_cast<int64_t>(kb0) * args.ws_red +
                             static_cast<int64_t>(min(col0 / kBlock, args.col_blocks - 1)) * args.ws_col;
      int left = kb1 - kb0;  // blocks whose scales are still to be fetched
      float sr[2], sw[2];
      auto fetch = [&](int slot) {
        if (left > 0) {
          sr[slot] = __ldg(row_scale);
          sw[slot] = __ldg(w_scale);
          row_scale += args.row_pitch;
          w_scale += args.ws_red;
          --left;
        }
      };
      auto add_block = [&](int slot) {
        const int buf = it & 1;
        if (!mbar_wait_cluster(bar(bars->acc_full[buf]), (it >> 1) & 1, abort_flag, args.status,
                               MOSS_STATUS_TIMEOUT_EPILOGUE))
          return false;
        ++it;
        tc_fence_after();
        // the next 32 columns are on their way out of TMEM while these are added
        uint32_t r[2][32];
        const uint32_t buf_addr = lane_addr + static_cast<uint32_t>(buf * kTileN);
        tmem_ld_32x32b_x32(buf_addr, r[0]);
        const float s = sr[slot] * sw[slot];
        fetch(slot);
#pragma unroll
        for (int c = 0; c < kCols / 32; ++c) {
          tmem_wait_ld_of(r[c & 1]);
          if (c + 1 < kCols / 32) {
            tmem_ld_32x32b_x32(buf_addr + (c + 1) * 32, r[(c + 1) & 1]);
          } else {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              if constexpr (kCtas == 2)
                mbar_arrive_cluster(release + buf * 8);
              else
                mbar_arrive(release + buf * 8);
            }
          }
#pragma unroll
          for (int j = 0; j < 32; ++j) sum[c * 32 + j] = fmaf(__uint_as_float(r[c & 1][j]), s, sum[c * 32 + j]);
        }
        return true;
      };
      fetch(0);
      fetch(1);
      for (int kb = kb0; kb < kb1 && ok; kb += 2) {
        ok = add_block(0);
        if (ok && kb + 1 < kb1) ok = add_block(1);
      }
      if (!ok) break;
      if (staged && !mbar_wait(bar(bars->out_free[half]), tiles_done & 1, abort_flag, args.status,
                               MOSS_STATUS_TIMEOUT_EPILOGUE))
        break;
      ++tiles_done;
#pragma unroll
      for (int c = 0; c < kCols / 32; ++c) {
        const int col = col0 + c * 32;
        float v[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = sum[c * 32 + j];
        if constexpr (kF32Out) {
          if (col < args.Nc)
            store_f32_block(args, reinterpret_cast<float*>(smem_raw + (boxes - raw_base) + q * kSliceBytes), row - lane,
                            col, v);
        } else if (staged) {
          if (args.bias != nullptr)
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const float4 b = *reinterpret_cast<const float4*>(bias_smem + half * kHalf + c * 32 + j);
            v[j] += b.x;
            v[j + 1] += b.y;
            v[j + 2] += b.z;
            v[j + 3] += b.w;
          }
          const uint32_t box = boxes + (c >> 1) * kBoxBytes;
          if (args.out_kind == kBF16)
            stage32<kBF16>(box, q * 32 + lane, c & 1, v);
          else
            stage32<kF16>(box, q * 32 + lane, c & 1, v);
        } else {
          // by columns: a warp's 32 rows are contiguous
          float* dst = args.partial + ((static_cast<int64_t>(split) * args.tiles_m * args.tiles_n + tile) * kTileN +
                                       half * kCols + c * 32) * kTileM + q * 32 + lane;
#pragma unroll
          for (int j = 0; j < 32; ++j) dst[j * kTileM] = v[j];
        }
      }
      if (staged && args.tma_out != 0) fence_proxy_async_smem();
      __syncwarp();
      if (staged && args.tma_out == 0) {
        // rows that TMA cannot address (an odd width): the warp writes its own, 64 columns at a time
        const uint16_t* rows16 = reinterpret_cast<const uint16_t*>(smem_raw + (boxes - raw_base)) + q * 32 * 64;
        const int row0 = row - lane;
        for (int i = 0; i < 32 && row0 + i < args.M; ++i) {
          uint16_t* dst = static_cast<uint16_t*>(args.out) + static_cast<int64_t>(row0 + i) * args.Nc + col0;
#pragma unroll
          for (int e = 0; e < kCols / 32; ++e) {
            const int j = e * 32 + lane, k = j & 63;
            const uint16_t v16 = rows16[(j >> 6) * (kBoxBytes / 2) + i * 64 + (((k >> 3) ^ (i & 7)) << 3) + (k & 7)];
            if (col0 + j < args.Nc) dst[j] = v16;
          }
        }
        __syncwarp();
      }
      if (staged && lane == 0) mbar_arrive(bar(bars->out_full[half]));
    }
  }

  // Leave together: the leader's MMAs read the peer's shared memory and write its TMEM, and the
  // peer arrives on the leader's barriers, so neither CTA exits or frees TMEM first.
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

template <bool kDX, int kCtas, bool kF32Out>
int launch_typed(const CUtensorMap& ta, const CUtensorMap& tw, const CUtensorMap& to, const Args& a, cudaStream_t stream) {
  auto kern = fp8_gemm_kernel<kDX, kCtas, kF32Out>;
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
  const int rc = setup("fp8_gemm_kernel", &max_groups, [&](int* groups) {
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
  const int64_t units = static_cast<int64_t>(a.tiles_m) * a.tiles_n * a.splits;
  cfg.gridDim = dim3(static_cast<unsigned>(kCtas * std::max<int64_t>(1, std::min<int64_t>(units, max_groups))));
  cfg.stream = stream;
  cfg.numAttrs = 2;  // after this call's quantiser
  return check_cuda(cudaLaunchKernelEx(&cfg, kern, ta, tw, to, a), "fp8_gemm_kernel");
}

template <bool kDX, int kCtas>
int launch_out(const CUtensorMap& ta, const CUtensorMap& tw, const CUtensorMap& to, const Args& a, cudaStream_t stream) {
  return a.out_kind == kF32 && a.splits == 1 ? launch_typed<kDX, kCtas, true>(ta, tw, to, a, stream)
                                             : launch_typed<kDX, kCtas, false>(ta, tw, to, a, stream);
}

}  // namespace

int launch_gemm(bool dx, const Plan& plan, const CUtensorMap& ta, const CUtensorMap& tw, const CUtensorMap& to,
                const Args& a, cudaStream_t stream) {
  if (plan.kind == Plan::kPair)
    return dx ? launch_out<true, 2>(ta, tw, to, a, stream) : launch_out<false, 2>(ta, tw, to, a, stream);
  return dx ? launch_out<true, 1>(ta, tw, to, a, stream) : launch_out<false, 1>(ta, tw, to, a, stream);
}

}  // namespace fp8
}  // namespace moss
