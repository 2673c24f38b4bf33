// e4m3 GEMM whose operands carry one scale per 128 columns of K:
//   out[m, n] = sum_kb a_scale[m, kb] * b_scale[n / 128, kb] * sum_{k in block kb} A[m, k] B[n, k]
//               (+ bias[n]); with a residual: residual[m, n] + gate[n] * (.)
// The scales differ from block to block of K, so the tensor cores' running sum cannot hold the
// result: each block's 128-deep partial product is finished in TMEM on its own, read back, and
// added with its scale to an fp32 accumulator in registers.
#include <algorithm>
#include <atomic>

#include <cuda_fp16.h>

#include "common.cuh"
#include "sm100_ptx.cuh"

namespace sb {
namespace {

using namespace sm100;

constexpr int kBlockK = 128;  // columns per scale = one 128-byte swizzle span of e4m3
constexpr int kGroupM = 16;   // tiles are visited in groups of 16 row-tiles, rows fastest

// Instruction descriptor for kind::f8f6f4 with e4m3 A and B, fp32 accumulation, K-major.
__host__ __device__ constexpr uint32_t idesc_e4m3_f32(int M, int N) {
  return (1u << 4)                     // D format: f32
         | (0u << 7) | (0u << 10)      // A, B format: e4m3
         | ((uint32_t)(N >> 3) << 17)  // K-major A and B
         | ((uint32_t)(M >> 4) << 24);
}

struct BlockGemmParams {
  const float* a_scale;  // a_scale[m * a_row_stride + kb * a_block_stride]
  const float* b_scale;  // [ceil(N / 128), k_blocks]
  int64_t a_row_stride, a_block_stride;
  const float* bias;      // optional [N]
  const void* residual;   // optional [M, N], the output's type
  const float* gate;      // optional [N] (1), with a residual
  void* out;              // [M, N] bf16 or fp32
  int a_vec;              // 1: a row's scales are consecutive and its first is 16-byte aligned
  int tma_out;            // 1: rows of whole 16-byte vectors, written by TMA stores
  int* status;
  int64_t M;
  int N, K, k_blocks;
  int m_tiles, n_tiles;
};

// ------------------------------------------------------------------ CTA-pair kernel
// A cluster of two CTAs computes a 256 x 256 tile with tcgen05.mma.cta_group::2, one k-block per
// stage.  A k-block's partial product goes to TMEM as two halves of 128 columns, each with its own
// barriers, in two buffers: the issue of a half waits for the read-back of the half four issues
// before it, and TMEM holds no more, so what counts is the time from a half's last MMA to its
// next first one (the commit, the read-back, the arrival at rank 0) against the time of the
// three halves between.  Halves shorten both the MMAs and the read-back in that loop.
//   full[s]      rank 0 only: armed for both CTAs' bytes of a stage
//   empty[s]     both CTAs: the commits of both halves' MMAs release the stage
//   acc_full[a]  both CTAs, a = 2 * buffer + half: the commit after a half's four MMAs
//   acc_empty[a] rank 0 only: one arrival per epilogue warp of that half in both CTAs (8)
//   scale_full[c], scale_empty[c]  per CTA: a chunk of 8 k-blocks' scales, from the scale warp to
//                the epilogue warps
//   mma_done     both CTAs: the final commits of both issuers, waited before TMEM is freed
// Each half has its own issuing warp: one waiting for its half's read-back does not hold up the other.
// Eight epilogue warps per CTA: warp w reads TMEM lanes 32 (w % 4) .. (its 32 rows) of half w / 4
// (one weight block), so a k-block has ONE scale per thread, a_scale * b_scale.  The 128
// accumulators of a thread stay in registers for the whole tile (setmaxnreg moves registers of
// the other four warps to these eight).
constexpr int kEpiWarps = 8;
constexpr int kEpiThreads = 32 * kEpiWarps;
constexpr int kProducerWarp = kEpiWarps, kScaleWarp = kEpiWarps + 1, kIssuerWarp = kEpiWarps + 2;  // and + 3
constexpr int kPairThreads = kEpiThreads + 128;
constexpr int kLaunchRegs = 168, kEpiRegs = 208, kOtherRegs = 88;  // per thread
static_assert(kEpiRegs * kEpiThreads + kOtherRegs * 128 == kLaunchRegs * kPairThreads,
              "setmaxnreg redistributes exactly what the CTA was launched with");
constexpr int kPairStages = 5;
constexpr int kChunk = 8;  // k-blocks of scales per chunk; two chunks in shared memory
constexpr int kPairOpBytes = 128 * kBlockK;       // one operand's 128 rows of a stage
constexpr int kPairStageBytes = 2 * kPairOpBytes;  // A half + B half per CTA
constexpr int kPairHalfBytes = 64 * kBlockK;      // a CTA's B rows of one half of the tile
constexpr uint32_t kPairAccCols = 128;            // columns of a half; two halves x two buffers
constexpr int kPairOutBox = 32 * 64;           // one epilogue warp's 32 rows x 64 bytes
constexpr int kPairOutBytes = kEpiWarps * 2 * kPairOutBox;  // two boxes per warp
constexpr int kChunkFloats = kChunk * 2 * 128;  // [k-block][weight block of the tile][row]
constexpr int kScaleBytes = 2 * kChunkFloats * 4;

struct __align__(8) PairControl {
  uint64_t full[kPairStages], empty[kPairStages];
  uint64_t acc_full[4], acc_empty[4];
  uint64_t scale_full[2], scale_empty[2];
  uint64_t mma_done;
  uint32_t tmem_base;
  int abort_flag;
};

// Relaxed: what the arrival hands over are TMEM columns whose loads have completed (wait::ld); a
// release would also wait for the thread's unrelated memory accesses.
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar_cluster, int x,
                                                 int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar_cluster)
      : "memory");
}
__device__ __forceinline__ void mma_f8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrives on the barrier at the same offset of both CTAs.
__device__ __forceinline__ void tc_commit_both(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
      "h"((uint16_t)3)
      : "memory");
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t holder_smem, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(holder_smem), "r"(ncols)
               : "memory");
}
__device__ __forceinline__ void tmem_relinquish_pair() {
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}

// Grouped raster: groups of kGroupM row-tiles; inside a group rows move fastest, so the
// pairs running at one time share a few B panels and a few A panels (both stay in L2).
__device__ __forceinline__ void tile_coords(int64_t t, int m_tiles, int n_tiles, int& mt, int& nt) {
  const int64_t per_group = (int64_t)kGroupM * n_tiles;
  const int group = (int)(t / per_group);
  const int first_m = group * kGroupM;
  const int gm = min(kGroupM, m_tiles - first_m);
  const int within = (int)(t - (int64_t)group * per_group);
  mt = first_m + within % gm;
  nt = within / gm;
}

// 16 bytes of a row of T as fp32.
template <typename T>
__device__ __forceinline__ void unpack16(const uint4& raw, float* v) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (sizeof(T) == 2) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      v[i] = __uint_as_float(w[i]);
    }
  }
}

// A warp's 32 rows x 64 bytes between shared memory (16-byte chunk q of row r at q ^ ((r >> 1) & 3))
// and rows m0 .. of a matrix with N columns, from column nc on; rows from M and columns from N on
// are left out.  For matrices whose rows are no whole 16-byte vectors: four bytes per lane, two
// rows at a time, where rows start on four bytes, else two.
template <typename T, bool STORE>
__device__ __forceinline__ void copy_rows(uint32_t stage, T* matrix, int64_t m0, int64_t M, int nc, int N, int lane) {
  const int rows = (int)min((int64_t)32, M - m0);
  if (sizeof(T) == 4 || N % 2 == 0) {
    const int u = lane & 15, col = nc + u * (4 / (int)sizeof(T));
    if (col >= N) return;
    T* at = matrix + (m0 + (lane >> 4)) * N + col;
#pragma unroll 8
    for (int r = lane >> 4; r < rows; r += 2, at += 2 * (int64_t)N) {
      const uint32_t s = stage + (uint32_t)(r * 64 + (((u >> 2) ^ ((r >> 1) & 3)) * 16) + (u & 3) * 4);
      uint32_t v;
      if (STORE) {
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(s) : "memory");
        *reinterpret_cast<uint32_t*>(at) = v;
      } else {
        v = *reinterpret_cast<const uint32_t*>(at);
        asm volatile("st.shared.b32 [%0], %1;" ::"r"(s), "r"(v) : "memory");
      }
    }
  } else {
    if (nc + lane >= N) return;
    T* at = matrix + m0 * N + nc + lane;
#pragma unroll 8
    for (int r = 0; r < rows; ++r, at += N) {
      const uint32_t s = stage + (uint32_t)(r * 64 + (((lane >> 3) ^ ((r >> 1) & 3)) * 16) + (lane & 7) * 2);
      uint16_t v;
      if (STORE) {
        asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"(s) : "memory");
        *reinterpret_cast<uint16_t*>(at) = v;
      } else {
        v = *reinterpret_cast<const uint16_t*>(at);
        asm volatile("st.shared.b16 [%0], %1;" ::"r"(s), "h"(v) : "memory");
      }
    }
  }
}

// The bounded wait of a converged warp: true once the phase is complete.
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status,
                                          int site) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, status, site));
}

template <typename T>
__global__ void __launch_bounds__(kPairThreads, 1)
fp8_gemm_blocks_pair_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                            const __grid_constant__ CUtensorMap tm_out, BlockGemmParams p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  // Same layout in both CTAs, so both take the same branch here.
  const bool aligned = (smem_u32(smem) & 1023u) == 0u;
  uint8_t* sOut = smem + kPairStages * kPairStageBytes;  // output staging of the TMA stores
  float* sScale = reinterpret_cast<float*>(sOut + kPairOutBytes);  // [2][kChunkFloats]
  PairControl& C = *reinterpret_cast<PairControl*>(sOut + kPairOutBytes + kScaleBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  if (aligned && threadIdx.x == 0) {
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(smem_u32(&C.full[s]), 1);
      mbar_init(smem_u32(&C.empty[s]), 2);
    }
    for (int b = 0; b < 4; ++b) {
      mbar_init(smem_u32(&C.acc_full[b]), 1);
      mbar_init(smem_u32(&C.acc_empty[b]), kEpiWarps);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&C.scale_full[b]), 1);
      mbar_init(smem_u32(&C.scale_empty[b]), kEpiWarps);
    }
    mbar_init(smem_u32(&C.mma_done), 2);
    C.abort_flag = 0;
    fence_barrier_init();
  }
  cluster_sync_all();  // every barrier of the pair exists before either CTA signals one
  if (!aligned) {
    if (threadIdx.x == 0 && p.status) atomicExch(p.status, 912);
    return;
  }
  if (warp == kIssuerWarp) {
    tmem_alloc_pair(smem_u32(&C.tmem_base), 4 * kPairAccCols);
    tmem_relinquish_pair();
  }
  if (warp == kProducerWarp && lane == 0) {
    prefetch_tensormap(&tm_a);
    prefetch_tensormap(&tm_b);
    if (p.tma_out) prefetch_tensormap(&tm_out);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = C.tmem_base;
  volatile int* abort_flag = &C.abort_flag;
  const uint32_t base = smem_u32(smem);
  const int64_t pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int64_t total_tiles = (int64_t)p.m_tiles * p.n_tiles;  // 256 x 256 tiles

  if (warp >= kEpiWarps) {
    setmaxnreg_dec<kOtherRegs>();
    if (warp == kProducerWarp) {
      // ------------------------------------------------------------ producer (both CTAs)
      if (elect_one()) {
        int s = 0, use = 0;
        int64_t issued = 0;  // stages
        bool ok = true;
        for (int64_t t = pair; ok && t < total_tiles; t += pairs) {
          int mt, nt;
          tile_coords(t, p.m_tiles, p.n_tiles, mt, nt);
          for (int kb = 0; kb < p.k_blocks; ++kb) {
            if (!mbar_wait(smem_u32(&C.empty[s]), (uint32_t)((use & 1) ^ 1), abort_flag, p.status, 431)) {
              ok = false;
              break;
            }
            const uint32_t full_leader = mapa_shared(smem_u32(&C.full[s]), 0);
            if (leader) mbar_arrive_expect_tx(smem_u32(&C.full[s]), 2 * kPairStageBytes);
            ++issued;
            const uint32_t st = base + s * kPairStageBytes;
            tma_load_2d_pair(st, &tm_a, full_leader, kb * kBlockK, mt * 256 + (int)rank * 128);
            // of each half's 128 weight rows this CTA holds 64
            tma_load_2d_pair(st + kPairOpBytes, &tm_b, full_leader, kb * kBlockK, nt * 256 + (int)rank * 64);
            tma_load_2d_pair(st + kPairOpBytes + kPairHalfBytes, &tm_b, full_leader, kb * kBlockK,
                             nt * 256 + 128 + (int)rank * 64);
            if (++s == kPairStages) {
              s = 0;
              ++use;
            }
          }
        }
        // rank 0's full barriers complete only once both CTAs' bytes have landed
        if (leader)
          for (int st = 0; st < kPairStages; ++st)
            if (issued > st) mbar_drain(smem_u32(&C.full[st]), (uint32_t)(((issued - 1 - st) / kPairStages) & 1));
      }
    } else if (warp >= kIssuerWarp) {
      // ------------------------------------------------------------ MMA issuers (rank 0), one per half
      const int h = warp - kIssuerWarp;
      if (leader && elect_one()) {
        constexpr uint32_t idesc = idesc_e4m3_f32(256, 128);
        const uint64_t adesc0 = smem_desc_sw128(base, 16, 1024);
        const uint64_t bdesc0 = adesc0 + (uint64_t)((kPairOpBytes + h * kPairHalfBytes) >> 4);
        int s = 0, buf = 0;
        uint32_t use = 0, round = 0;  // how often all stages / both accumulators have been filled
        bool ok = true;
        for (int64_t t = pair; ok && t < total_tiles; t += pairs) {
          for (int kb = 0; kb < p.k_blocks; ++kb) {
            if (!mbar_wait(smem_u32(&C.full[s]), use & 1u, abort_flag, p.status, 433) ||
                !mbar_wait(smem_u32(&C.acc_empty[2 * buf + h]), (round & 1u) ^ 1u, abort_flag, p.status, 432)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint64_t off = (uint64_t)((s * kPairStageBytes) >> 4);
  #pragma unroll
            for (int kk = 0; kk < kBlockK / 32; ++kk)
              mma_f8_pair(tmem + (2 * buf + h) * kPairAccCols, adesc0 + off + (uint64_t)(kk * 2),
                          bdesc0 + off + (uint64_t)(kk * 2), idesc, kk > 0 ? 1u : 0u);
            tc_commit_both(smem_u32(&C.acc_full[2 * buf + h]));
            tc_commit_both(smem_u32(&C.empty[s]));
            if (++s == kPairStages) {
              s = 0;
              ++use;
            }
            if (++buf == 2) {
              buf = 0;
              ++round;
            }
          }
        }
        tc_commit_both(smem_u32(&C.mma_done));  // covers this warp's MMAs
      }
    } else if (warp == kScaleWarp) {
      // ------------------------------------------------------------ scales (both CTAs)
      // a_scale[m, kb] * b_scale[n / 128, kb] for the CTA's 128 rows and the tile's two weight
      // blocks, kChunk k-blocks at a time: lane l serves rows l, l + 32, l + 64 and l + 96.
      int buf = 0;
      uint32_t round = 0;
      bool ok = true;
      for (int64_t t = pair; ok && t < total_tiles; t += pairs) {
        int mt, nt;
        tile_coords(t, p.m_tiles, p.n_tiles, mt, nt);
        const int64_t m0 = (int64_t)mt * 256 + rank * 128 + lane;
        const float* sb0 = p.b_scale + (int64_t)(nt * 2) * p.k_blocks;
        const bool two = nt * 256 + 128 < p.N;
        for (int k0 = 0; ok && k0 < p.k_blocks; k0 += kChunk) {
          float a[4][kChunk];
  #pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int64_t m = m0 + 32 * i;
            const float* sa = p.a_scale + m * p.a_row_stride;
            if (m < p.M && p.a_vec && k0 + kChunk <= p.k_blocks) {
              load8(sa + k0, a[i]);
            } else {
  #pragma unroll
              for (int e = 0; e < kChunk; ++e)
                a[i][e] = m < p.M && k0 + e < p.k_blocks ? __ldg(sa + (k0 + e) * p.a_block_stride) : 0.f;
            }
          }
          const bool got = mbar_wait(smem_u32(&C.scale_empty[buf]), (round & 1u) ^ 1u, abort_flag, p.status, 435);
          ok = __all_sync(0xffffffffu, got);
          if (!ok) break;
          float* dst = sScale + buf * kChunkFloats + lane;
  #pragma unroll
          for (int e = 0; e < kChunk; ++e) {
            const bool in = k0 + e < p.k_blocks;
            const float b0 = in ? __ldg(sb0 + k0 + e) : 0.f;
            const float b1 = in && two ? __ldg(sb0 + p.k_blocks + k0 + e) : 0.f;
  #pragma unroll
            for (int i = 0; i < 4; ++i) {
              dst[(2 * e) * 128 + 32 * i] = a[i][e] * b0;
              dst[(2 * e + 1) * 128 + 32 * i] = a[i][e] * b1;
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&C.scale_full[buf]));
          if (++buf == 2) {
            buf = 0;
            ++round;
          }
        }
      }
    }
  } else {
    setmaxnreg_inc<kEpiRegs>();
    // ------------------------------------------------------------ epilogue (both CTAs)
    const int quad = warp & 3, half = warp >> 2;
    const uint32_t lane_base = (uint32_t)(quad * 32) << 16;
    const uint32_t stages = smem_u32(sOut) + (uint32_t)(warp * 2 * kPairOutBox);
    const uint32_t acc_empty = mapa_shared(smem_u32(&C.acc_empty[half]), 0);  // + 16 bytes for buffer 1
    constexpr int kOutCols = 64 / (int)sizeof(T);  // columns of a staged 64-byte row
    constexpr int kVec = 16 / (int)sizeof(T);
    const float* my_scale = sScale + half * 128 + quad * 32 + lane;
    const uint32_t cols0 = tmem + lane_base + half * kPairAccCols;  // + 2 * kPairAccCols for buffer 1
    const uint32_t acc_full = smem_u32(&C.acc_full[half]);          // + 16 bytes for buffer 1
    const uint32_t scale_full = smem_u32(&C.scale_full[0]);
    int chunk = 0;  // scale chunk in use
    uint32_t it = 0, chunk_round = 0;
    bool ok = true;
    for (int64_t t = pair; ok && t < total_tiles; t += pairs) {
      uint64_t acc[64];
#pragma unroll
      for (int i = 0; i < 64; ++i) acc[i] = 0;
      for (int left = p.k_blocks; left > 0; left -= kChunk) {
        if (!wait_warp(scale_full + chunk * 8, chunk_round & 1u, abort_flag, p.status, 436)) {
          ok = false;
          break;
        }
        const float* chunk_scale = my_scale + chunk * kChunkFloats;
        const int in_chunk = min(left, kChunk);
#pragma unroll 2
        for (int e = 0; e < in_chunk; ++e, ++it) {
          const uint32_t buf = it & 1u;  // accumulator
          const float scale = chunk_scale[e * 256];
          if (!wait_warp(acc_full + buf * 16, (it >> 1) & 1u, abort_flag, p.status, 434)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t col0 = cols0 + buf * 2 * kPairAccCols;
          const uint64_t s2 = f2_pack(scale, scale);
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            uint32_t r[16];
            tmem_ld16(col0 + 16 * c, r);
            tmem_wait_ld();
            if (c == 7) {  // all of this half is in registers
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive_cluster(acc_empty + buf * 16);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
              acc[8 * c + i] = f2_fma(f2_pack(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), s2, acc[8 * c + i]);
          }
        }
        if (!ok) break;
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&C.scale_empty[chunk]));
        if (++chunk == 2) {
          chunk = 0;
          ++chunk_round;
        }
      }
      if (!ok) break;
      int mt, nt;
      tile_coords(t, p.m_tiles, p.n_tiles, mt, nt);
      const int64_t m = (int64_t)mt * 256 + rank * 128 + quad * 32 + lane;
      const int n0 = nt * 256 + half * 128;
      if (n0 >= p.N) continue;
      // ---------------------------------------------------------- output
      const bool row_ok = m < p.M;
      const int64_t row0 = m - lane;
      // A lane's 16-byte chunk q of its staged row sits at q ^ ((row >> 1) & 3) (64-byte swizzle).
      const uint32_t swizzle = (uint32_t)((lane >> 1) & 3);
#pragma unroll
      for (int g = 0; g < 128 / kOutCols; ++g) {
        const int nc = n0 + g * kOutCols;
        const uint32_t stage = stages + (uint32_t)((g & 1) * kPairOutBox), my_stage = stage + (uint32_t)(lane * 64);
        if (p.tma_out && lane == 0) bulk_wait_group_read<1>();  // the store before the last one
        __syncwarp();  // the stage is free
        if (!p.tma_out && p.residual != nullptr) {
          copy_rows<T, false>(stage, static_cast<T*>(const_cast<void*>(p.residual)), row0, p.M, nc, p.N, lane);
          __syncwarp();
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {  // 16 bytes of the row at a time
          const int n = nc + q * kVec;
          const uint32_t chunk = my_stage + (((uint32_t)q ^ swizzle) * 16u);
          float f[kVec];
#pragma unroll
          for (int i = 0; i < kVec / 2; ++i)
            f2_unpack(acc[(g * kOutCols + q * kVec) / 2 + i], f[2 * i], f[2 * i + 1]);
          if (p.bias != nullptr) {
#pragma unroll
            for (int i = 0; i < kVec; ++i)
              if (n + i < p.N) f[i] += __ldg(p.bias + n + i);
          }
          if (p.residual != nullptr) {
            // The residual may be the output: its loads are plain and precede the row's store.
            uint4 raw = make_uint4(0u, 0u, 0u, 0u);
            if (p.tma_out) {
              if (row_ok && n < p.N)
                raw = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.residual) + m * p.N + n);
            } else {
              asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                           : "=r"(raw.x), "=r"(raw.y), "=r"(raw.z), "=r"(raw.w)
                           : "r"(chunk)
                           : "memory");
            }
            float res[kVec];
            unpack16<T>(raw, res);
#pragma unroll
            for (int i = 0; i < kVec; ++i)
              if (n + i < p.N) f[i] = fmaf(p.gate != nullptr ? __ldg(p.gate + n + i) : 1.f, f[i], res[i]);
          }
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            w[e] = sizeof(T) == 2 ? cvt_bf16x2(f[(2 * e) % kVec], f[(2 * e + 1) % kVec]) : __float_as_uint(f[e]);
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(chunk), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                       : "memory");
        }
        if (p.tma_out) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {  // rows past M and columns past N are clipped by the store
            if (nc < p.N && row0 < p.M) tma_store_2d(&tm_out, stage, nc, (int)row0);
            bulk_commit_group();
          }
        } else {
          __syncwarp();
          copy_rows<T, true>(stage, static_cast<T*>(p.out), row0, p.M, nc, p.N, lane);
        }
      }
    }
    if (p.tma_out) {
      if (lane == 0) bulk_wait_group<0>();  // every output store has landed before the CTA exits
      __syncwarp();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kIssuerWarp) {
    tc_fence_after();
    mbar_drain(smem_u32(&C.mma_done), 0);  // rank 0's MMAs write both CTAs' TMEM
  }
  cluster_sync_all();  // no signal to the peer's shared memory is still in flight
  if (warp == kIssuerWarp) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 4 * kPairAccCols);
  }
}

// ------------------------------------------------------------------ few rows: plain streaming
// For one or two rows of A the product is the reading of B once: each thread multiplies its 16
// bytes of a weight row with its 16 columns of the M rows, which it keeps as fp32, so weights go
// from global memory to registers with no staging, and no TMEM, barrier or tensor map has to be
// set up.  A CTA of 8 warps takes kRows weight rows per row group; `k_warps` warps split K (512
// columns each at a time) and the sums meet in shared memory.  1 x 4096 x 4096: 6.7 us (swap 8.5).
constexpr int kStreamThreads = 256;
constexpr int kRows = 8;

__device__ __forceinline__ void e4m3x16_to_float(const uint4& raw, float* f) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)(w[i >> 1] >> (16 * (i & 1)))));
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h));
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
}

template <typename T, int M>
__global__ void __launch_bounds__(kStreamThreads) fp8_gemm_blocks_stream_kernel(const uint8_t* __restrict__ a,
                                                                                const uint8_t* __restrict__ b,
                                                                                int k_warps, BlockGemmParams p) {
  __shared__ float part[kStreamThreads / 32][kRows * M];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = warp / k_warps, kw = warp - group * k_warps;
  const int n0 = (blockIdx.x * (kStreamThreads / 32 / k_warps) + group) * kRows;
  float acc[kRows * M];  // [row][m]
#pragma unroll
  for (int i = 0; i < kRows * M; ++i) acc[i] = 0.f;
  if (n0 < p.N) {
    const float* sb = p.b_scale + (int64_t)(n0 >> 7) * p.k_blocks;  // kRows divides 128: one weight block
    for (int64_t k = (kw * 32 + lane) * 16; k < p.K; k += (int64_t)k_warps * 512) {
      uint4 w[kRows];
#pragma unroll
      for (int r = 0; r < kRows; ++r)
        w[r] = __ldg(reinterpret_cast<const uint4*>(b + (int64_t)min(n0 + r, p.N - 1) * p.K + k));
      const int kb = (int)(k >> 7);
      const float s = __ldg(sb + kb);
      float sm[M];
#pragma unroll
      for (int m = 0; m < M; ++m) sm[m] = s * __ldg(p.a_scale + m * p.a_row_stride + kb * p.a_block_stride);
      float x[M][16];
#pragma unroll
      for (int m = 0; m < M; ++m)
        e4m3x16_to_float(__ldg(reinterpret_cast<const uint4*>(a + (int64_t)m * p.K + k)), x[m]);
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        float y[16];
        e4m3x16_to_float(w[r], y);
#pragma unroll
        for (int m = 0; m < M; ++m) {
          float d = x[m][0] * y[0];
#pragma unroll
          for (int i = 1; i < 16; ++i) d = fmaf(x[m][i], y[i], d);
          acc[r * M + m] = fmaf(d, sm[m], acc[r * M + m]);
        }
      }
    }
  }
  // Sums over the lanes: each step halves the values a lane holds until each holds one or few.
  int held = kRows * M;
  int index = 0;  // the first of the values this lane holds
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if (held > 1) {
      held >>= 1;
      const bool upper = (lane & o) != 0;
#pragma unroll
      for (int i = 0; i < kRows * M / 2; ++i) {
        if (i < held) {
          const float keep = upper ? acc[i + held] : acc[i];
          const float give = upper ? acc[i] : acc[i + held];
          acc[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
      }
      if (upper) index += held;
    } else {
      acc[0] += __shfl_xor_sync(0xffffffffu, acc[0], o);
    }
  }
  // kRows * M is 8 or 16: one value per lane, held by 4 or 2 lanes
  if (lane % (32 / (kRows * M)) == 0) part[warp][index] = acc[0];
  __syncthreads();
  const int groups = kStreamThreads / 32 / k_warps;
  for (int i = threadIdx.x; i < groups * kRows * M; i += kStreamThreads) {
    const int g = i / (kRows * M), e = i - g * (kRows * M);
    const int n = (blockIdx.x * groups + g) * kRows + e / M, m = e % M;
    if (n >= p.N) continue;
    float f = 0.f;
    for (int w = 0; w < k_warps; ++w) f += part[g * k_warps + w][e];
    if (p.bias != nullptr) f += __ldg(p.bias + n);
    const int64_t at = (int64_t)m * p.N + n;
    if (p.residual != nullptr)
      f = fmaf(p.gate != nullptr ? __ldg(p.gate + n) : 1.f, f, Elem<T>::to_f(static_cast<const T*>(p.residual)[at]));
    static_cast<T*>(p.out)[at] = Elem<T>::from_f(f);
  }
}

int sm_count() {
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

// The split of the stream kernel's warps along K with the fewest passes over K times waves of CTAs, and its
// time in us, launch included: a fit of the times below, 0 where one pass of one wave does it all.  An
// SM holds four CTAs for one row (62 registers a thread), two for two (99).
double stream_shape(int64_t M, int N, int K, int sms, int* k_warps) {
  const int64_t resident = (int64_t)sms * (M == 1 ? 4 : 2);
  int64_t best = 0;
  double estimate = 0;
  for (int w = 1; w <= 8; w *= 2) {
    const int64_t passes = ((int64_t)K + 512 * w - 1) / (512 * w);
    const int64_t ctas = ((int64_t)N + kRows * (8 / w) - 1) / (kRows * (8 / w));
    const int64_t waves = (ctas + resident - 1) / resident;
    if (w == 1 || passes * waves < best) {
      best = passes * waves;
      estimate = best == 1 ? 0 : 2.5 + (waves == 1 ? 3.2 : 4.0) * (double)best;
      *k_warps = w;
    }
  }
  return estimate;
}

template <typename T>
int launch_stream(const uint8_t* a, const uint8_t* b, int k_warps, const BlockGemmParams& p, cudaStream_t s) {
  const int rows = kRows * (kStreamThreads / 32 / k_warps);
  const unsigned grid = (unsigned)((p.N + rows - 1) / rows);
  if (p.M == 1)
    fp8_gemm_blocks_stream_kernel<T, 1><<<grid, kStreamThreads, 0, s>>>(a, b, k_warps, p);
  else
    fp8_gemm_blocks_stream_kernel<T, 2><<<grid, kStreamThreads, 0, s>>>(a, b, k_warps, p);
  SB_CHECK_LAUNCH("sb_fp8_gemm_blocks launch");
  return SB_OK;
}

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      ptr = nullptr;
    return reinterpret_cast<EncodeTiledFn>(ptr);
  }();
  return fn;
}

// Row-major [rows, cols] as boxes of 128 bytes x box_rows (loads, 128-byte swizzle) or 64 bytes x
// box_rows (stores, 64-byte swizzle).
int make_map(CUtensorMap* map, CUtensorMapDataType type, int elem, const void* base, uint64_t cols, uint64_t rows,
             uint32_t box_rows, bool load) {
  EncodeTiledFn encode = encode_fn();
  if (encode == nullptr) {
    set_error("sb_fp8_gemm_blocks: cuTensorMapEncodeTiled is unavailable");
    return SB_ERR_CUDA;
  }
  const cuuint64_t dims[2] = {cols, rows};
  const cuuint64_t strides[1] = {cols * (uint64_t)elem};
  const cuuint32_t box[2] = {(cuuint32_t)((load ? 128 : 64) / elem), box_rows};
  const cuuint32_t estr[2] = {1, 1};
  CUresult r = encode(map, type, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                      load ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                      load ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B : CU_TENSOR_MAP_L2_PROMOTION_NONE,
                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("sb_fp8_gemm_blocks: cuTensorMapEncodeTiled failed (CUresult %d)", (int)r);
    return SB_ERR_CUDA;
  }
  return SB_OK;
}

// ------------------------------------------------------------------ some rows: weights as MMA rows
// A tile is 128 weight rows (the MMA's M) x T rows of A (its N, a multiple of 16 up to 64), so a
// few rows of A do not fill a 256-row tile with padding.  CTAs are small and several share an SM,
// which hides each one's set-up and hand-overs behind the others' loads; where the tiles alone do
// not fill the GPU, the CTAs of a cluster split K and add their sums, in rank order, through
// distributed shared memory.  Thread = weight row: the scale of accumulator column j is
// a_scale[row j] * b_scale, read from shared memory by all lanes at once.
constexpr int kSwapProducer = 4, kSwapIssuer = 5, kSwapScales = 6;  // warps 0-3: epilogue
constexpr int kSwapThreads = 224;
constexpr int kSwapTokens = 64;
constexpr int kSwapMaxStages = 4;

struct __align__(8) SwapControl {
  uint64_t full[kSwapMaxStages], empty[kSwapMaxStages];
  uint64_t acc_full[2], acc_empty[2];
  uint64_t scale_full[2], scale_empty[2];
  uint64_t mma_done;
  uint32_t tmem_base;
  int abort_flag;
};

struct SwapShape {
  int tokens;      // T: rows of A per tile
  int m_tiles;
  int splits;      // CTAs of a cluster
  int group;       // k-blocks per stage and per TMEM buffer
  int stages;
  uint32_t acc_stride;  // TMEM columns per k-block; 2 * group * acc_stride are allocated
};

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void mma_f8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// One output value from its sum.
template <typename T>
__device__ __forceinline__ void finish_value(const BlockGemmParams& p, int64_t m, int n, float f) {
  if (p.bias != nullptr) f += __ldg(p.bias + n);
  const int64_t at = m * p.N + n;
  if (p.residual != nullptr)
    f = fmaf(p.gate != nullptr ? __ldg(p.gate + n) : 1.f, f, Elem<T>::to_f(static_cast<const T*>(p.residual)[at]));
  static_cast<T*>(p.out)[at] = Elem<T>::from_f(f);
}

template <typename T, int CW>
__global__ void __launch_bounds__(kSwapThreads, 2)
fp8_gemm_blocks_swap_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                            BlockGemmParams p, SwapShape q) {
  extern __shared__ __align__(1024) uint8_t smem[];
  const bool aligned = (smem_u32(smem) & 1023u) == 0u;  // alike in every CTA
  const int tokens = q.tokens;
  const int span_bytes = kPairOpBytes + tokens * kBlockK;  // a k-block's weights and rows of A
  const int stage_bytes = q.group * span_bytes;
  float* sScale = reinterpret_cast<float*>(smem + q.stages * stage_bytes);  // [2][kChunk][tokens]
  SwapControl& C = *reinterpret_cast<SwapControl*>(sScale + 2 * kChunk * tokens);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x % q.splits;
  const int tile = blockIdx.x / q.splits;
  const int mt = tile % q.m_tiles, nt = tile / q.m_tiles;  // tiles of one weight panel run together
  const int kb0 = (int)((int64_t)p.k_blocks * rank / q.splits);
  const int kb1 = (int)((int64_t)p.k_blocks * (rank + 1) / q.splits);
  if (!aligned) {
    if (threadIdx.x == 0 && p.status) atomicExch(p.status, 913);
    return;
  }
  if (warp == kSwapProducer && lane == 0) {
    prefetch_tensormap(&tm_a);
    prefetch_tensormap(&tm_b);
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < kSwapMaxStages; ++s) {
      mbar_init(smem_u32(&C.full[s]), 1);
      mbar_init(smem_u32(&C.empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&C.acc_full[b]), 1);
      mbar_init(smem_u32(&C.acc_empty[b]), 4);
      mbar_init(smem_u32(&C.scale_full[b]), 1);
      mbar_init(smem_u32(&C.scale_empty[b]), 4);
    }
    mbar_init(smem_u32(&C.mma_done), 1);
    C.abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == kSwapIssuer) {
    tmem_alloc(smem_u32(&C.tmem_base), 2 * q.group * q.acc_stride);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = C.tmem_base;
  volatile int* abort_flag = &C.abort_flag;
  const uint32_t base = smem_u32(smem);

  float acc[CW];
#pragma unroll
  for (int i = 0; i < CW; ++i) acc[i] = 0.f;
  const int quad = warp & 3;

  if (warp == kSwapProducer) {
    // ------------------------------------------------------------ producer
    if (elect_one()) {
      int s = 0;
      uint32_t use = 0;
      int issued = 0;
      for (int kb = kb0; kb < kb1; kb += q.group) {
        if (!mbar_wait(smem_u32(&C.empty[s]), (use & 1u) ^ 1u, abort_flag, p.status, 441)) break;
        const uint32_t full = smem_u32(&C.full[s]);
        const int g = min(q.group, kb1 - kb);
        mbar_arrive_expect_tx(full, g * span_bytes);
        for (int i = 0; i < g; ++i) {  // g * 128 consecutive bytes of each weight row
          const uint32_t st = base + s * stage_bytes + i * span_bytes;
          tma_load_2d(st, &tm_b, full, (kb + i) * kBlockK, nt * 128);
          tma_load_2d(st + kPairOpBytes, &tm_a, full, (kb + i) * kBlockK, mt * tokens);
        }
        ++issued;
        if (++s == q.stages) {
          s = 0;
          ++use;
        }
      }
      for (int st = 0; st < q.stages; ++st)
        if (issued > st) mbar_drain(smem_u32(&C.full[st]), (uint32_t)(((issued - 1 - st) / q.stages) & 1));
    }
  } else if (warp == kSwapIssuer) {
    // ------------------------------------------------------------ MMA issuer
    if (elect_one()) {
      const uint32_t idesc = idesc_e4m3_f32(128, tokens);
      const uint64_t desc0 = smem_desc_sw128(base, 16, 1024);
      int s = 0, buf = 0;
      uint32_t use = 0, round = 0;
      for (int kb = kb0; kb < kb1; kb += q.group) {
        if (!mbar_wait(smem_u32(&C.full[s]), use & 1u, abort_flag, p.status, 442) ||
            !mbar_wait(smem_u32(&C.acc_empty[buf]), (round & 1u) ^ 1u, abort_flag, p.status, 443))
          break;
        tc_fence_after();
        const int g = min(q.group, kb1 - kb);
        for (int i = 0; i < g; ++i) {
          const uint64_t dw = desc0 + (uint64_t)((s * stage_bytes + i * span_bytes) >> 4);
          const uint64_t dx = dw + (uint64_t)(kPairOpBytes >> 4);
#pragma unroll
          for (int kk = 0; kk < kBlockK / 32; ++kk)
            mma_f8(tmem + (buf * q.group + i) * q.acc_stride, dw + (uint64_t)(kk * 2), dx + (uint64_t)(kk * 2), idesc,
                   kk > 0 ? 1u : 0u);
        }
        tc_commit(smem_u32(&C.acc_full[buf]));
        tc_commit(smem_u32(&C.empty[s]));
        if (++s == q.stages) {
          s = 0;
          ++use;
        }
        if (++buf == 2) {
          buf = 0;
          ++round;
        }
      }
      tc_commit(smem_u32(&C.mma_done));
    }
  } else if (warp == kSwapScales) {
    // ------------------------------------------------------------ scales
    const float* sb = p.b_scale + (int64_t)nt * p.k_blocks;
    int buf = 0;
    uint32_t round = 0;
    for (int k0 = kb0; k0 < kb1; k0 += kChunk) {
      const bool got = mbar_wait(smem_u32(&C.scale_empty[buf]), (round & 1u) ^ 1u, abort_flag, p.status, 444);
      if (!__all_sync(0xffffffffu, got)) break;
      for (int j = lane; j < tokens; j += 32) {
        const int64_t m = (int64_t)mt * tokens + j;
        const float* sa = p.a_scale + m * p.a_row_stride;
        float v[kChunk];
#pragma unroll
        for (int e = 0; e < kChunk; ++e)
          v[e] = m < p.M && k0 + e < kb1 ? __ldg(sa + (k0 + e) * p.a_block_stride) * __ldg(sb + k0 + e) : 0.f;
#pragma unroll
        for (int e = 0; e < kChunk; ++e) sScale[(buf * kChunk + e) * tokens + j] = v[e];
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&C.scale_full[buf]));
      if (++buf == 2) {
        buf = 0;
        ++round;
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const uint32_t lane_base = (uint32_t)(quad * 32) << 16;
    const uint32_t acc_full = smem_u32(&C.acc_full[0]), scale_full = smem_u32(&C.scale_full[0]);
    uint32_t it = 0;  // groups done: buffer it & 1
    for (int k0 = kb0; k0 < kb1; k0 += kChunk) {
      const uint32_t chunks = (uint32_t)(k0 - kb0) / kChunk, chunk = chunks & 1u;
      if (!wait_warp(scale_full + chunk * 8, (chunks >> 1) & 1u, abort_flag, p.status, 445)) break;
      const int in_chunk = min(kb1 - k0, kChunk);
      bool ok = true;
      for (int e0 = 0; e0 < in_chunk; e0 += q.group, ++it) {  // groups divide chunks
        const uint32_t buf = it & 1u;
        ok = wait_warp(acc_full + buf * 8, (it >> 1) & 1u, abort_flag, p.status, 446);
        if (!ok) break;
        tc_fence_after();
        const int g = min(q.group, in_chunk - e0);
        const float4* scale = reinterpret_cast<const float4*>(sScale + (chunk * kChunk + e0) * tokens);
        uint32_t src = tmem + lane_base + buf * q.group * q.acc_stride;
        for (int k = 0; k < g; ++k, scale += tokens / 4, src += q.acc_stride) {
#pragma unroll
          for (int c = 0; c < CW; c += 16) {
            if (c < tokens) {
              uint32_t r[16];
              tmem_ld16(src + c, r);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float4 s = scale[c / 4 + i];
                acc[c + 4 * i + 0] = fmaf(__uint_as_float(r[4 * i + 0]), s.x, acc[c + 4 * i + 0]);
                acc[c + 4 * i + 1] = fmaf(__uint_as_float(r[4 * i + 1]), s.y, acc[c + 4 * i + 1]);
                acc[c + 4 * i + 2] = fmaf(__uint_as_float(r[4 * i + 2]), s.z, acc[c + 4 * i + 2]);
                acc[c + 4 * i + 3] = fmaf(__uint_as_float(r[4 * i + 3]), s.w, acc[c + 4 * i + 3]);
              }
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&C.acc_empty[buf]));
      }
      if (!ok) break;
      if (lane == 0) mbar_arrive(smem_u32(&C.scale_empty[chunk]));
    }
    const int n = nt * 128 + quad * 32 + lane;
    if (q.splits == 1) {
      if (n < p.N) {
#pragma unroll
        for (int j = 0; j < CW; ++j) {
          const int64_t m = (int64_t)mt * tokens + j;
          if (j < tokens && m < p.M) finish_value<T>(p, m, n, acc[j]);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kSwapIssuer) {
    tc_fence_after();
    mbar_drain(smem_u32(&C.mma_done), 0);
    tmem_dealloc(tmem, 2 * q.group * q.acc_stride);
  }
  if (q.splits > 1) {
    // Every stage has been read: the stages hold this CTA's sums as [column][weight row].
    __syncthreads();
    float* part = reinterpret_cast<float*>(smem);
    if (warp < 4) {
#pragma unroll
      for (int j = 0; j < CW; ++j)
        if (j < tokens) part[j * 128 + quad * 32 + lane] = acc[j];
    }
    cluster_sync_all();
    const int per = tokens / q.splits;  // columns this CTA finishes; splits divides 16
    for (int i = threadIdx.x; i < per * 128; i += kSwapThreads) {
      const int j = rank * per + i / 128, row = i % 128;
      float f = 0.f;
      for (int r = 0; r < q.splits; ++r)
        f += __uint_as_float(ld_shared_cluster_u32(mapa_shared(smem_u32(part + j * 128 + row), r)));
      const int64_t m = (int64_t)mt * tokens + j;
      const int n = nt * 128 + row;
      if (m < p.M && n < p.N) finish_value<T>(p, m, n, f);
    }
    cluster_sync_all();  // no CTA leaves while another reads its sums
  }
}


template <typename T>
int launch_pair(const uint8_t* a, const uint8_t* b, BlockGemmParams p, cudaStream_t s) {
  CUtensorMap ma, mb, mo;
  int rc;
  if ((rc = make_map(&ma, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a, p.K, p.M, 128, true)) != SB_OK) return rc;
  if ((rc = make_map(&mb, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, b, p.K, p.N, 64, true)) != SB_OK) return rc;
  mo = ma;
  if (p.tma_out &&
      (rc = make_map(&mo, sizeof(T) == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, sizeof(T),
                     p.out, p.N, p.M, 32, false)) != SB_OK)
    return rc;
  p.m_tiles = (int)((p.M + 255) / 256);
  p.n_tiles = (p.N + 255) / 256;
  // setmaxnreg waits for registers that the launch did not bring: refuse a build with other counts.
  static std::atomic<bool> fits{false};
  if (!fits.load(std::memory_order_relaxed)) {
    cudaFuncAttributes fa{};
    cudaError_t e = cudaFuncGetAttributes(&fa, fp8_gemm_blocks_pair_kernel<T>);
    if (e != cudaSuccess) return cuda_error(e, "sb_fp8_gemm_blocks: kernel attributes");
    if (fa.numRegs != kLaunchRegs) {
      set_error("sb_fp8_gemm_blocks: the kernel was built with %d registers per thread, not %d", fa.numRegs, kLaunchRegs);
      return SB_ERR_UNSUPPORTED;
    }
    fits.store(true, std::memory_order_relaxed);
  }
  const size_t smem = (size_t)kPairStages * kPairStageBytes + kPairOutBytes + kScaleBytes + sizeof(PairControl);
  cudaError_t err =
      cudaFuncSetAttribute(fp8_gemm_blocks_pair_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (err != cudaSuccess) return cuda_error(err, "sb_fp8_gemm_blocks: set smem");
  const int pairs = (int)std::max<int64_t>(1, std::min<int64_t>((int64_t)p.m_tiles * p.n_tiles, sm_count() / 2));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * pairs, 1, 1);
  cfg.blockDim = dim3(kPairThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  err = cudaLaunchKernelEx(&cfg, fp8_gemm_blocks_pair_kernel<T>, ma, mb, mo, p);
  if (err != cudaSuccess) return cuda_error(err, "sb_fp8_gemm_blocks: cluster launch");
  SB_CHECK_LAUNCH("sb_fp8_gemm_blocks launch");
  return SB_OK;
}

template <typename T, int CW>
int launch_swap(const uint8_t* a, const uint8_t* b, const BlockGemmParams& p, SwapShape q, cudaStream_t s) {
  CUtensorMap ma, mb;
  int rc;
  if ((rc = make_map(&ma, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a, p.K, p.M, q.tokens, true)) != SB_OK) return rc;
  if ((rc = make_map(&mb, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, b, p.K, p.N, 128, true)) != SB_OK) return rc;
  const size_t smem = (size_t)q.stages * q.group * (kPairOpBytes + q.tokens * kBlockK) + (size_t)2 * kChunk * q.tokens * 4 +
                      sizeof(SwapControl);
  auto kernel = fp8_gemm_blocks_swap_kernel<T, CW>;
  cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (err != cudaSuccess) return cuda_error(err, "sb_fp8_gemm_blocks: set smem");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((int64_t)q.m_tiles * ((p.N + 127) / 128) * q.splits), 1, 1);
  cfg.blockDim = dim3(kSwapThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = q.splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  err = cudaLaunchKernelEx(&cfg, kernel, ma, mb, p, q);
  if (err != cudaSuccess) return cuda_error(err, "sb_fp8_gemm_blocks: cluster launch");
  SB_CHECK_LAUNCH("sb_fp8_gemm_blocks launch");
  return SB_OK;
}

// Which kernel, and its shape.  The estimates are fits (in us, most within 20 %) of times measured on
// one B200, launch included, over 3 to 5208 rows, 76 to 28672 columns and K of 192 to 16384:
//   pair: 7.5 + 0.43 per k-block and wave of tiles (one 256 x 256 tile per CTA pair);
//   swap: 4.5, + 2 where a cluster adds up its splits of K, + 2.5 with more than one CTA per SM, + the
//         larger of the weights' bytes at 5.5 TB/s and 0.55 (up to 32 rows of A: 0.20) per k-block
//         of a CTA, 0.78 (0.35) with two CTAs per SM.
// Both sides, swap and pair, at M x N x K: 64 x 4096 x 4096 11.5, 20.1; 85 x 143 x 1952 7.1, 13.4;
// 1000 x 392 x 4112 15.0, 22.5; 64 x 28672 x 5376 36.0, 47; 2659 x 167 x 1536 12.1, 13.3;
// 256 x 4096 x 4096 22.5, 20.1; 128 x 14336 x 5376 34.9, 29.6; 5000 x 256 x 2048 18.4, 13.9.
double pair_estimate(int64_t M, int N, int k_blocks, int sms) {
  const int64_t tiles = (M + 255) / 256 * (((int64_t)N + 255) / 256), pairs = sms / 2;
  return 7.5 + 0.43 * (double)((tiles + pairs - 1) / pairs) * k_blocks;
}

double swap_shape(int64_t M, int N, int k_blocks, int sms, SwapShape* shape) {
  SwapShape q{};
  const int64_t m_tiles = (M + kSwapTokens - 1) / kSwapTokens;
  const int64_t tiles = m_tiles * (((int64_t)N + 127) / 128);
  if (tiles > 8 * (int64_t)sms && m_tiles > 1) return 1e30;  // never the better one, and a grid of any size
  q.m_tiles = (int)m_tiles;
  q.tokens = (int)(((M + m_tiles - 1) / m_tiles + 15) / 16 * 16);
  const bool narrow = q.tokens <= 32;
  const double weights = (double)N * k_blocks * kBlockK / 5.5e6;
  double best = 0;
  // Splits of K by 1, 2, 4 or 8, each of at least two k-blocks, as long as all CTAs are resident (two
  // per SM): 64 x 28672 x 5376 split by 8 takes 76 us.
  for (int splits = 1; splits <= 8; splits *= 2) {
    const int64_t ctas = tiles * splits;
    if (splits > 1 && (k_blocks < 2 * splits || ctas > 2 * sms)) break;
    const int64_t waves = (ctas + 2 * sms - 1) / (2 * sms);
    const bool one = ctas <= sms;
    const double loop = (one ? (narrow ? 0.20 : 0.55) : (narrow ? 0.35 : 0.78)) * (double)waves * k_blocks / splits;
    const double t = 4.5 + (splits > 1 ? 2.0 : 0.0) + (one ? 0.0 : 2.5) + std::max(loop, weights);
    if (splits == 1 || t < best) {
      best = t;
      q.splits = splits;
      // Two k-blocks per stage read 256 consecutive bytes of each weight row and halve the
      // hand-overs; with two CTAs per SM the stages of a CTA have to fit 113 KB.
      q.group = one || narrow ? 2 : 1;
      q.stages = one ? (narrow ? 4 : 3) : (narrow ? 2 : 4);
    }
  }
  q.acc_stride = narrow ? 32 : 64;
  *shape = q;
  return best;
}

template <typename T>
int dispatch(const uint8_t* a, const uint8_t* b, const BlockGemmParams& p, cudaStream_t s) {
  const int sms = sm_count();
  SwapShape q{};
  const double pair = pair_estimate(p.M, p.N, p.k_blocks, sms), swap = swap_shape(p.M, p.N, p.k_blocks, sms, &q);
  // One or two rows: streaming starts sooner, swap reads faster (256-byte bursts by TMA).  Measured (stream,
  // swap; us, in a graph, weights from HBM): one row in one pass 4096 x 1024 5.6, 6.0; 4096 x 4096 6.7, 8.5;
  // in more 5376 x 4096 9.9, 10.5; 512 x 16384 14.9, 8.7; two rows in one pass 2048 x 4096 6.1, 11.9; in
  // more 2000 x 8192 9.7, 14.0; 8192 x 2048 10.3, 8.4; 4096 x 5376 17.2, 9.7.  Larger weights, one row:
  // 4096 x 16384 18.3, 16.6; 28672 x 5376 42.4, 28.5.
  int k_warps = 1;
  if (p.M <= 2 && (int64_t)p.N * p.K <= (24 << 20) &&
      stream_shape(p.M, p.N, p.K, sms, &k_warps) < std::min(swap, pair))
    return launch_stream<T>(a, b, k_warps, p, s);
  if (swap < pair) {
    if (q.tokens <= 16) return launch_swap<T, 16>(a, b, p, q, s);
    if (q.tokens <= 32) return launch_swap<T, 32>(a, b, p, q, s);
    return launch_swap<T, 64>(a, b, p, q, s);
  }
  // A few rows past whole 256-row tiles can cost a wave of nearly empty tiles: they get a launch
  // of their own where that is cheaper (259 x 28672 x 5376: 99 us as one launch).
  const int64_t rest = p.M % 256, whole = p.M - rest;
  if (whole > 0 && rest > 0 && rest <= kSwapTokens &&
      pair_estimate(whole, p.N, p.k_blocks, sms) + swap_shape(rest, p.N, p.k_blocks, sms, &q) < pair) {
    BlockGemmParams head = p, tail = p;
    head.M = whole;
    tail.M = rest;
    tail.a_scale += whole * p.a_row_stride;
    tail.out = static_cast<T*>(p.out) + whole * p.N;
    if (p.residual != nullptr) tail.residual = static_cast<const T*>(p.residual) + whole * p.N;
    const int rc = launch_pair<T>(a, b, head, s);
    return rc != SB_OK ? rc : dispatch<T>(a + whole * p.K, b, tail, s);
  }
  return launch_pair<T>(a, b, p, s);
}

}  // namespace
}  // namespace sb

using namespace sb;

extern "C" int sb_fp8_gemm_blocks(const uint8_t* a, const float* a_scale, int64_t a_row_stride, int64_t a_block_stride,
                                  const uint8_t* b, const float* b_scale, int64_t M, int N, int K, const float* bias,
                                  const void* residual, const float* gate, void* out, int out_dtype, void* stream) {
  SB_CHECK_ARG(a && a_scale && b && b_scale && out, "sb_fp8_gemm_blocks: null pointer");
  SB_CHECK_ARG(out_dtype == SB_F32 || out_dtype == SB_BF16, "sb_fp8_gemm_blocks: bad output dtype");
  SB_CHECK_ARG(M > 0 && N > 0 && K > 0, "sb_fp8_gemm_blocks: M, N, K must be positive");
  SB_CHECK_ARG(M <= 0x7fffff00ll && N <= 0x7fffff00 && K <= 0x7fffff00,
               "sb_fp8_gemm_blocks: M, N and K must be at most 2^31 - 256");
  SB_CHECK_ARG(K % 16 == 0, "sb_fp8_gemm_blocks: K must be a multiple of 16 (TMA row pitch), got %d", K);
  SB_CHECK_ARG(((uintptr_t)a % 16) == 0 && ((uintptr_t)b % 16) == 0 && ((uintptr_t)out % 16) == 0 &&
                   ((uintptr_t)residual % 16) == 0,
               "sb_fp8_gemm_blocks: A, B, the residual and the output must be 16-byte aligned");
  SB_CHECK_ARG(((uintptr_t)a_scale | (uintptr_t)b_scale | (uintptr_t)bias | (uintptr_t)gate) % 4 == 0,
               "sb_fp8_gemm_blocks: scales, bias and gate must be 4-byte aligned");
  SB_CHECK_ARG(gate == nullptr || residual != nullptr, "sb_fp8_gemm_blocks: a gate needs a residual");
  SB_CHECK_ARG(a_row_stride >= 0 && a_block_stride >= 0, "sb_fp8_gemm_blocks: scale strides must not be negative");
  BlockGemmParams p{};
  p.status = device_status_ptr();
  if (p.status == nullptr) return cuda_error(cudaGetLastError(), "sb_fp8_gemm_blocks: status word");
  p.a_scale = a_scale;
  p.b_scale = b_scale;
  p.a_row_stride = a_row_stride;
  p.a_block_stride = a_block_stride;
  p.bias = bias;
  p.residual = residual;
  p.gate = gate;
  p.out = out;
  p.M = M;
  p.N = N;
  p.K = K;
  p.k_blocks = (K + kBlockK - 1) / kBlockK;
  p.a_vec = a_block_stride == 1 && a_row_stride % 4 == 0 && (uintptr_t)a_scale % 16 == 0;
  p.tma_out = (int64_t)N * (out_dtype == SB_BF16 ? 2 : 4) % 16 == 0;
  cudaStream_t s = (cudaStream_t)stream;
  return out_dtype == SB_BF16 ? dispatch<__nv_bfloat16>(a, b, p, s) : dispatch<float>(a, b, p, s);
}
