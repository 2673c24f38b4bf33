// e4m3 GEMM whose operands carry one scale per 128 columns of K:
//   out[m, n] = sum_kb a_scale[m, kb] * b_scale[n / 128, kb] * sum_{k in block kb} A[m, k] B[n, k]
//               (+ bias[n]); with a residual: residual[m, n] + gate[n] * (.)
// The scales differ from block to block of K, so the tensor cores' running sum cannot hold the
// result: each block's 128-deep partial product is finished in TMEM on its own, read back, and
// added with its scale to an fp32 accumulator in registers.
#include <algorithm>

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
  int tma_out;            // 1: rows of whole 16-byte vectors, written by TMA stores
  int* status;
  int64_t M;
  int N, K, k_blocks;
  int m_tiles, n_tiles;
};

// ------------------------------------------------------------------ CTA-pair kernel
// A cluster of two CTAs computes a 256 x 256 tile with tcgen05.mma.cta_group::2 (the pair's
// operand and barrier protocol of fp8_gemm.cu), one k-block per stage and per TMEM buffer:
//   full[s]      rank 0 only: armed for both CTAs' bytes of a stage
//   empty[s]     both CTAs: the MMA's commit releases the stage
//   acc_full[b]  both CTAs: the commit after a k-block's four MMAs
//   acc_empty[b] rank 0 only: one arrival per epilogue warp of both CTAs (16)
//   mma_done     both CTAs: final commit, waited before TMEM is freed
// Eight epilogue warps per CTA: warp w reads TMEM lanes 32 (w % 4) .. (its 32 rows) and columns
// 128 (w / 4) .. (one weight block), so a k-block has ONE scale per thread, a_scale * b_scale.
// The 128 accumulators of a thread stay in registers for the whole tile.
constexpr int kPairThreads = 320;  // warps 0-7 epilogue, 8 TMA producer, 9 MMA issuer
constexpr int kPairStages = 6;
constexpr int kPairOpBytes = 128 * kBlockK;       // one operand's 128 rows of a stage
constexpr int kPairStageBytes = 2 * kPairOpBytes;  // A half + B half per CTA
constexpr uint32_t kPairAccCols = 256;
constexpr int kPairOutBox = 32 * 128;          // one epilogue warp's 32 rows x 128 bytes
constexpr int kPairOutBytes = 8 * kPairOutBox;

struct __align__(8) PairControl {
  uint64_t full[kPairStages], empty[kPairStages];
  uint64_t acc_full[2], acc_empty[2];
  uint64_t mma_done;
  uint32_t tmem_base;
  int abort_flag;
};

__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
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
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, {%5, %5, %5, %5, %5, %5, %5, %5}, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(0u)
      : "memory");
}
__device__ __forceinline__ void tc_commit_pair(uint32_t bar_cluster) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar_cluster)
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

// Bias, gate and residual of `n` columns from column n0 of row m applied to f.
template <typename T, int NCOLS>
__device__ __forceinline__ void finish_columns(const BlockGemmParams& p, int64_t m, bool row_ok, int n0, float* f) {
  if (p.bias != nullptr) {
#pragma unroll
    for (int i = 0; i < NCOLS; ++i)
      if (n0 + i < p.N) f[i] += __ldg(p.bias + n0 + i);
  }
  if (p.residual != nullptr && row_ok) {
    const T* res = static_cast<const T*>(p.residual) + m * p.N + n0;
    if (p.tma_out && n0 + NCOLS <= p.N) {
#pragma unroll
      for (int i = 0; i < NCOLS; i += 8) {
        float r[8];
        load8_plain(res + i, r);  // the output may be the residual
#pragma unroll
        for (int e = 0; e < 8; ++e) f[i + e] = fmaf(p.gate ? __ldg(p.gate + n0 + i + e) : 1.f, f[i + e], r[e]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NCOLS; ++i)
        if (n0 + i < p.N) f[i] = fmaf(p.gate ? __ldg(p.gate + n0 + i) : 1.f, f[i], Elem<T>::to_f(res[i]));
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kPairThreads, 1)
fp8_gemm_blocks_pair_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                            const __grid_constant__ CUtensorMap tm_out, BlockGemmParams p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  // Same layout in both CTAs, so both take the same branch here.
  const bool aligned = (smem_u32(smem) & 1023u) == 0u;
  uint8_t* sOut = smem + kPairStages * kPairStageBytes;  // output staging of the TMA stores
  PairControl& C = *reinterpret_cast<PairControl*>(sOut + kPairOutBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  if (aligned && threadIdx.x == 0) {
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(smem_u32(&C.full[s]), 1);
      mbar_init(smem_u32(&C.empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&C.acc_full[b]), 1);
      mbar_init(smem_u32(&C.acc_empty[b]), 16);
    }
    mbar_init(smem_u32(&C.mma_done), 1);
    C.abort_flag = 0;
    fence_barrier_init();
  }
  cluster_sync_all();  // every barrier of the pair exists before either CTA signals one
  if (!aligned) {
    if (threadIdx.x == 0 && p.status) atomicExch(p.status, 912);
    return;
  }
  if (warp == 9) {
    tmem_alloc_pair(smem_u32(&C.tmem_base), 2 * kPairAccCols);
    tmem_relinquish_pair();
  }
  if (warp == 8 && lane == 0) {
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

  if (warp == 8) {
    // ------------------------------------------------------------ producer (both CTAs)
    if (lane == 0) {
      int s = 0, use = 0;
      int armed[kPairStages] = {};
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
          ++armed[s];
          const uint32_t st = base + s * kPairStageBytes;
          tma_load_2d_pair(st, &tm_a, full_leader, kb * kBlockK, mt * 256 + (int)rank * 128);
          tma_load_2d_pair(st + kPairOpBytes, &tm_b, full_leader, kb * kBlockK, nt * 256 + (int)rank * 128);
          if (++s == kPairStages) {
            s = 0;
            ++use;
          }
        }
      }
      // rank 0's full barriers complete only once both CTAs' bytes have landed
      if (leader)
        for (int st = 0; st < kPairStages; ++st)
          if (armed[st] > 0) mbar_drain(smem_u32(&C.full[st]), (uint32_t)((armed[st] - 1) & 1));
    }
  } else if (warp == 9) {
    // ------------------------------------------------------------ MMA issuer (rank 0)
    if (lane == 0 && leader) {
      constexpr uint32_t idesc = idesc_e4m3_f32(256, 256);
      const uint64_t adesc0 = smem_desc_sw128(base, 16, 1024);
      int s = 0, use = 0, buf = 0;
      uint32_t round = 0;  // how often both accumulators have been filled
      bool ok = true;
      for (int64_t t = pair; ok && t < total_tiles; t += pairs) {
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          if (!mbar_wait(smem_u32(&C.acc_empty[buf]), (round & 1u) ^ 1u, abort_flag, p.status, 432) ||
              !mbar_wait(smem_u32(&C.full[s]), (uint32_t)(use & 1), abort_flag, p.status, 433)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t acc = tmem + buf * kPairAccCols;
          const uint64_t sa = adesc0 + (uint64_t)((s * kPairStageBytes) >> 4);
          const uint64_t sb = sa + (uint64_t)(kPairOpBytes >> 4);
#pragma unroll
          for (int kk = 0; kk < kBlockK / 32; ++kk)
            mma_f8_pair(acc, sa + (uint64_t)(kk * 2), sb + (uint64_t)(kk * 2), idesc, kk > 0 ? 1u : 0u);
          const uint32_t f = smem_u32(&C.acc_full[buf]), e = smem_u32(&C.empty[s]);
          tc_commit_pair(mapa_shared(f, 0));
          tc_commit_pair(mapa_shared(f, 1));
          tc_commit_pair(mapa_shared(e, 0));
          tc_commit_pair(mapa_shared(e, 1));
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
      const uint32_t d = smem_u32(&C.mma_done);  // covers every MMA of the pair
      tc_commit_pair(mapa_shared(d, 0));
      tc_commit_pair(mapa_shared(d, 1));
    }
  } else {
    // ------------------------------------------------------------ epilogue (both CTAs)
    const int quad = warp & 3, half = warp >> 2;
    const uint32_t lane_base = (uint32_t)(quad * 32) << 16;
    const uint32_t stage = smem_u32(sOut) + (uint32_t)(warp * kPairOutBox);
    const uint32_t acc_empty0 = mapa_shared(smem_u32(&C.acc_empty[0]), 0);
    const uint32_t acc_empty1 = mapa_shared(smem_u32(&C.acc_empty[1]), 0);
    constexpr int kOutCols = 128 / (int)sizeof(T);  // columns of a staged 128-byte row
    int buf = 0;
    uint32_t round = 0;
    bool ok = true;
    for (int64_t t = pair; ok && t < total_tiles; t += pairs) {
      int mt, nt;
      tile_coords(t, p.m_tiles, p.n_tiles, mt, nt);
      const int64_t m = (int64_t)mt * 256 + rank * 128 + quad * 32 + lane;
      const int n0 = nt * 256 + half * 128;
      const bool row_ok = m < p.M && n0 < p.N;
      // Rows and column blocks outside the matrix hold zeros in TMEM; their scale is 0.
      const float* sa = p.a_scale + (row_ok ? m * p.a_row_stride : 0);
      const float* sb = p.b_scale + (row_ok ? (int64_t)(n0 >> 7) * p.k_blocks : 0);
      uint64_t acc[64];
#pragma unroll
      for (int i = 0; i < 64; ++i) acc[i] = 0;
      float scale = row_ok ? __ldg(sa) * __ldg(sb) : 0.f;
      for (int kb = 0; kb < p.k_blocks; ++kb) {
        float next = 0.f;
        if (row_ok && kb + 1 < p.k_blocks) next = __ldg(sa + (kb + 1) * p.a_block_stride) * __ldg(sb + kb + 1);
        const bool got = mbar_wait(smem_u32(&C.acc_full[buf]), round & 1u, abort_flag, p.status, 434);
        if (!__all_sync(0xffffffffu, got)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint64_t s2 = f2_pack(scale, scale);
        const uint32_t col0 = tmem + lane_base + buf * kPairAccCols + half * 128;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t r[32];
          tmem_ld32(col0 + 32 * c, r);
          tmem_wait_ld();
          if (c == 3) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(buf == 0 ? acc_empty0 : acc_empty1);
          }
#pragma unroll
          for (int i = 0; i < 16; ++i)
            acc[16 * c + i] = f2_fma(f2_pack(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), s2,
                                     acc[16 * c + i]);
        }
        scale = next;
        if (++buf == 2) {
          buf = 0;
          ++round;
        }
      }
      if (!ok) break;
      if (n0 >= p.N) continue;
      // ---------------------------------------------------------- output
#pragma unroll
      for (int g = 0; g < 128 / kOutCols; ++g) {
        float f[kOutCols];
#pragma unroll
        for (int i = 0; i < kOutCols / 2; ++i) f2_unpack(acc[g * (kOutCols / 2) + i], f[2 * i], f[2 * i + 1]);
        const int nc = n0 + g * kOutCols;
        finish_columns<T, kOutCols>(p, m, row_ok, nc, f);
        if (p.tma_out) {
          // 16-byte chunk q of staged row r sits at q ^ (r & 7) (128-byte swizzle)
          if (lane == 0) bulk_wait_group_read<0>();
          __syncwarp();
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              w[e] = sizeof(T) == 2 ? cvt_bf16x2(f[(8 * q + 2 * e) % kOutCols], f[(8 * q + 2 * e + 1) % kOutCols])
                                    : __float_as_uint(f[(4 * q + e) % kOutCols]);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + (uint32_t)(lane * 128 +
                                                                                            ((q ^ (lane & 7)) * 16))),
                         "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                         : "memory");
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {  // rows past M and columns past N are clipped by the store
            const int64_t row0 = (int64_t)mt * 256 + rank * 128 + quad * 32;
            if (nc < p.N && row0 < p.M) tma_store_2d(&tm_out, stage, nc, (int)row0);
            bulk_commit_group();
          }
        } else if (row_ok) {
          T* out = static_cast<T*>(p.out) + m * p.N;
#pragma unroll
          for (int i = 0; i < kOutCols; ++i)
            if (nc + i < p.N) out[nc + i] = Elem<T>::from_f(f[i]);
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
  if (warp == 9) {
    tc_fence_after();
    mbar_drain(smem_u32(&C.mma_done), 0);  // rank 0's MMAs write both CTAs' TMEM
  }
  cluster_sync_all();  // no signal to the peer's shared memory is still in flight
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 2 * kPairAccCols);
  }
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

// Row-major [rows, cols] as boxes of 128 bytes x box_rows, 128-byte swizzle.
int make_map(CUtensorMap* map, CUtensorMapDataType type, int elem, const void* base, uint64_t cols, uint64_t rows,
             uint32_t box_rows, bool load) {
  EncodeTiledFn encode = encode_fn();
  if (encode == nullptr) {
    set_error("sb_fp8_gemm_blocks: cuTensorMapEncodeTiled is unavailable");
    return SB_ERR_CUDA;
  }
  const cuuint64_t dims[2] = {cols, rows};
  const cuuint64_t strides[1] = {cols * (uint64_t)elem};
  const cuuint32_t box[2] = {(cuuint32_t)(128 / elem), box_rows};
  const cuuint32_t estr[2] = {1, 1};
  CUresult r = encode(map, type, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                      CU_TENSOR_MAP_SWIZZLE_128B,
                      load ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B : CU_TENSOR_MAP_L2_PROMOTION_NONE,
                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("sb_fp8_gemm_blocks: cuTensorMapEncodeTiled failed (CUresult %d)", (int)r);
    return SB_ERR_CUDA;
  }
  return SB_OK;
}

int sm_count() {
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

template <typename T>
int launch_pair(const uint8_t* a, const uint8_t* b, BlockGemmParams p, cudaStream_t s) {
  CUtensorMap ma, mb, mo;
  int rc;
  if ((rc = make_map(&ma, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a, p.K, p.M, 128, true)) != SB_OK) return rc;
  if ((rc = make_map(&mb, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, b, p.K, p.N, 128, true)) != SB_OK) return rc;
  mo = ma;
  if (p.tma_out &&
      (rc = make_map(&mo, sizeof(T) == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, sizeof(T),
                     p.out, p.N, p.M, 32, false)) != SB_OK)
    return rc;
  p.m_tiles = (int)((p.M + 255) / 256);
  p.n_tiles = (p.N + 255) / 256;
  const size_t smem = (size_t)kPairStages * kPairStageBytes + kPairOutBytes + sizeof(PairControl);
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
  p.tma_out = (int64_t)N * (out_dtype == SB_BF16 ? 2 : 4) % 16 == 0;
  cudaStream_t s = (cudaStream_t)stream;
  return out_dtype == SB_BF16 ? launch_pair<__nv_bfloat16>(a, b, p, s) : launch_pair<float>(a, b, p, s);
}
