// e4m3 quantisers with one scale per row and 128 columns, and the fused residual + RMSNorm +
// quantiser.  Each value is read once and kept in registers between the reduction that fixes
// its scale and the store of its code; all of them are bound by HBM.
//
// Scales and special values follow torch's spelling of the same arithmetic: scale =
// max(absmax * fp32(1/448), 1e-12) and the maximum propagates NaN, so a NaN in a group makes
// the whole group NaN, and an infinity makes its group's finite values 0 and itself NaN.
//
// A code is e4m3(y * (1 / scale)): one division per group instead of one per value.  The
// quotient is off by at most 2^-23 of itself, so a code differs from e4m3(y / scale) only where
// y / scale lies that close to the middle of two codes.
#include "common.cuh"

namespace sb {
namespace {

constexpr int kGroup = 128;        // columns per scale
constexpr float kInv448 = 1.0f / 448.0f;

__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// Maximum over the 16 lanes of a half warp.
__device__ __forceinline__ float half_warp_max(float x) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) x = max_nan(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}
__device__ __forceinline__ float absmax8(const float* v) {
  float m = fabsf(v[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) m = max_nan(m, fabsf(v[i]));
  return m;
}

// 8 values from column c of a row with `cols` columns; columns past the end read as 0.  `vec`:
// the row's vectors are 16-byte aligned (its columns are then a multiple of 8).
template <typename T>
__device__ __forceinline__ void load_cols(const T* row, int c, int cols, bool vec, float* v) {
  if (vec) {
    if (c < cols) {
      load8_plain(row + c, v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < cols ? Elem<T>::to_f(row[c + i]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store_cols(T* row, int c, int cols, bool vec, const float* v) {
  if (vec) {
    if (c < cols) store8(row + c, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < cols) row[c + i] = Elem<T>::from_f(v[i]);
  }
}
// Codes of 8 values; cvt.satfinite clamps to +-448 and keeps NaN.
__device__ __forceinline__ void store_codes(uint8_t* row, int c, int cols, bool vec, const float* v, float inv) {
  uint16_t packed[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(packed[i]) : "f"(v[2 * i + 1] * inv), "f"(v[2 * i] * inv));
  if (vec) {
    if (c < cols) *reinterpret_cast<uint2*>(row + c) = *reinterpret_cast<uint2*>(packed);
  } else {
    const uint8_t* bytes = reinterpret_cast<const uint8_t*>(packed);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < cols) row[c + i] = bytes[i];
  }
}

enum Activation { kNone = 0, kSwiglu = 1, kGelu = 2 };

// One half warp per group of 128 columns: lane l holds columns 8l .. 8l + 7.
constexpr int kQuantThreads = 256;

template <typename T, int ACT>
__global__ void __launch_bounds__(kQuantThreads) quantize_blocks_kernel(const T* __restrict__ x, int64_t x_stride,
                                                                        int64_t groups_total, int groups, int K,
                                                                        int vec, uint8_t* __restrict__ out,
                                                                        float* __restrict__ scales) {
  const int64_t g = (int64_t)blockIdx.x * (kQuantThreads / 16) + (threadIdx.x >> 4);
  if ((g & ~1ll) >= groups_total) return;  // whole warps leave together
  const bool live = g < groups_total;
  const int64_t row = live ? g / groups : 0;
  const int kb = live ? (int)(g - row * groups) : 0;
  const int c = kb * kGroup + (threadIdx.x & 15) * 8;
  const T* xr = x + row * x_stride;
  float v[8];
  load_cols(xr, c, K, vec, v);
  if (ACT == kSwiglu) {
    float gate[8];
    load_cols(xr + K, c, K, vec, gate);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = v[i] * gate[i] * (1.f / (1.f + __expf(-gate[i])));
  } else if (ACT == kGelu) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.5f * v[i] * (1.f + erff(v[i] * 0.70710678118654752f));
  }
  const float amax = half_warp_max(absmax8(v));
  if (!live) return;
  const float scale = max_nan(amax * kInv448, 1e-12f);
  if ((threadIdx.x & 15) == 0) scales[g] = scale;
  store_codes(out + row * K, c, K, vec, v, 1.f / scale);
}

struct NormParams {
  const void* x;
  const void* residual;  // optional
  const float* gate;     // optional (1), with a residual
  const float* weight;   // optional (1)
  const float* shift;    // optional (0)
  void* summed;          // residual + gate * x, with a residual
  uint8_t* out;
  float* scales;
  int64_t x_stride, residual_stride;               // elements between rows
  int64_t gate_stride, weight_stride, shift_stride;  // floats between samples
  int64_t M, rows_per_sample;
  int C, groups;
  int vec, vec_params;  // 16-byte accesses to the rows / to the parameter vectors
  float eps;
};

__device__ __forceinline__ void load_params(const float* p, int c, int C, bool vec, float fill, float* v) {
  if (p == nullptr) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = fill;
  } else {
    load_cols(p, c, C, vec, v);
  }
}

template <int THREADS, bool MAX>
__device__ __forceinline__ float block_reduce(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float w = __shfl_xor_sync(0xffffffffu, v, o);
    v = MAX ? max_nan(v, w) : v + w;
  }
  if (THREADS == 32) return v;
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int i = 1; i < THREADS / 32; ++i) v = MAX ? max_nan(v, red[i]) : v + red[i];
  return v;
}

// One CTA of THREADS per row, VPT vectors of 8 columns per thread, the row in registers.  The
// sum is rounded once, where it is stored; the norm works on the unrounded fp32 sum.
template <typename T, int THREADS, int VPT, bool BLOCKS>
__global__ void __launch_bounds__(THREADS) add_rms_norm_quantize_kernel(NormParams p) {
  __shared__ float red[2][THREADS / 32];
  const int64_t row = blockIdx.x;
  const int64_t sample = row / p.rows_per_sample;
  const T* xr = static_cast<const T*>(p.x) + row * p.x_stride;
  const T* rr = static_cast<const T*>(p.residual) + row * p.residual_stride;
  float v[VPT][8];
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int c = (j * THREADS + threadIdx.x) * 8;
    load_cols(xr, c, p.C, p.vec, v[j]);
    if (p.residual != nullptr) {
      float r[8], g[8];
      load_cols(rr, c, p.C, p.vec, r);
      load_params(p.gate == nullptr ? nullptr : p.gate + sample * p.gate_stride, c, p.C, p.vec_params, 1.f, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[j][i] = fmaf(g[i], v[j][i], r[i]);
      store_cols(static_cast<T*>(p.summed) + row * p.C, c, p.C, p.vec, v[j]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(v[j][i], v[j][i], ss);
  }
  const float rstd = rsqrtf(block_reduce<THREADS, false>(ss, red[0]) / (float)p.C + p.eps);
  float amax = 0.f;
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int c = (j * THREADS + threadIdx.x) * 8;
    float w[8], b[8];
    load_params(p.weight == nullptr ? nullptr : p.weight + sample * p.weight_stride, c, p.C, p.vec_params, 1.f, w);
    load_params(p.shift == nullptr ? nullptr : p.shift + sample * p.shift_stride, c, p.C, p.vec_params, 0.f, b);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[j][i] = c + i < p.C ? fmaf(v[j][i] * rstd, w[i], b[i]) : 0.f;
    const float m = absmax8(v[j]);
    if (BLOCKS) {
      const float scale = max_nan(half_warp_max(m) * kInv448, 1e-12f);
      const int kb = c / kGroup;
      if ((threadIdx.x & 15) == 0 && kb < p.groups) p.scales[row * p.groups + kb] = scale;
      store_codes(p.out + row * p.C, c, p.C, p.vec, v[j], 1.f / scale);
    } else {
      amax = max_nan(amax, m);
    }
  }
  if (!BLOCKS) {
    const float scale = max_nan(block_reduce<THREADS, true>(amax, red[1]) * kInv448, 1e-12f);
    if (threadIdx.x == 0) p.scales[row] = scale;
    const float inv = 1.f / scale;
#pragma unroll
    for (int j = 0; j < VPT; ++j)
      store_codes(p.out + row * p.C, (j * THREADS + threadIdx.x) * 8, p.C, p.vec, v[j], inv);
  }
}

template <typename T, int THREADS, int VPT>
void launch_norm(const NormParams& p, bool blocks, cudaStream_t s) {
  if (blocks)
    add_rms_norm_quantize_kernel<T, THREADS, VPT, true><<<(unsigned)p.M, THREADS, 0, s>>>(p);
  else
    add_rms_norm_quantize_kernel<T, THREADS, VPT, false><<<(unsigned)p.M, THREADS, 0, s>>>(p);
}

template <typename T>
void dispatch_norm(const NormParams& p, bool blocks, cudaStream_t s) {
  if (p.C <= 256) return launch_norm<T, 32, 1>(p, blocks, s);
  if (p.C <= 1024) return launch_norm<T, 128, 1>(p, blocks, s);
  if (p.C <= 4096) return launch_norm<T, 128, 4>(p, blocks, s);
  if (p.C <= 8192) return launch_norm<T, 256, 4>(p, blocks, s);
  return launch_norm<T, 512, 4>(p, blocks, s);
}

bool aligned16(const void* p) { return ((uintptr_t)p % 16) == 0; }

template <int ACT>
int quantize_blocks(const char* what, const void* x, int64_t x_stride, int dtype, int64_t M, int K, uint8_t* out,
                    float* scales, void* stream) {
  SB_CHECK_ARG(x && out && scales, "%s: null pointer", what);
  SB_CHECK_ARG(dtype == SB_F32 || dtype == SB_BF16, "%s: bad dtype", what);
  SB_CHECK_ARG(M > 0 && K > 0 && M < (1ll << 31) && K <= (1 << 30), "%s: M in [1, 2^31) and K in [1, 2^30]", what);
  const int cols = ACT == kSwiglu ? 2 * K : K;
  SB_CHECK_ARG(x_stride >= cols, "%s: rows overlap (stride %lld, %d columns)", what, (long long)x_stride, cols);
  const int size = dtype == SB_BF16 ? 2 : 4;
  SB_CHECK_ARG((uintptr_t)x % size == 0 && (uintptr_t)scales % 4 == 0, "%s: x and scales must be aligned to their elements",
               what);
  const int groups = ceil_div(K, kGroup);
  const int64_t total = M * groups;
  const int64_t grid = (total + kQuantThreads / 16 - 1) / (kQuantThreads / 16);
  SB_CHECK_ARG(grid < (1ll << 31), "%s: too many rows", what);
  // 16-byte loads need every row (and the gate half) on a 16-byte boundary.
  const int vec = K % 8 == 0 && x_stride * size % 16 == 0 && aligned16(x) && (uintptr_t)out % 8 == 0;
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == SB_BF16)
    quantize_blocks_kernel<__nv_bfloat16, ACT><<<(unsigned)grid, kQuantThreads, 0, s>>>(
        (const __nv_bfloat16*)x, x_stride, total, groups, K, vec, out, scales);
  else
    quantize_blocks_kernel<float, ACT><<<(unsigned)grid, kQuantThreads, 0, s>>>((const float*)x, x_stride, total, groups,
                                                                              K, vec, out, scales);
  SB_CHECK_LAUNCH(what);
  return SB_OK;
}

}  // namespace
}  // namespace sb

using namespace sb;

extern "C" int sb_fp8_quantize_blocks(const void* x, int64_t x_stride, int dtype, int64_t M, int K, uint8_t* out,
                                      float* scales, void* stream) {
  return quantize_blocks<kNone>("sb_fp8_quantize_blocks", x, x_stride, dtype, M, K, out, scales, stream);
}

extern "C" int sb_fp8_swiglu_quantize_blocks(const void* h, int64_t h_stride, int dtype, int64_t M, int K, uint8_t* out,
                                             float* scales, void* stream) {
  return quantize_blocks<kSwiglu>("sb_fp8_swiglu_quantize_blocks", h, h_stride, dtype, M, K, out, scales, stream);
}

extern "C" int sb_fp8_gelu_quantize_blocks(const void* x, int64_t x_stride, int dtype, int64_t M, int K, uint8_t* out,
                                           float* scales, void* stream) {
  return quantize_blocks<kGelu>("sb_fp8_gelu_quantize_blocks", x, x_stride, dtype, M, K, out, scales, stream);
}

extern "C" int sb_fp8_add_rms_norm_quantize(const void* x, int64_t x_stride, const void* residual,
                                            int64_t residual_stride, const float* gate, int64_t gate_stride,
                                            const float* weight, int64_t weight_stride, const float* shift,
                                            int64_t shift_stride, int dtype, int64_t M, int C, int64_t rows_per_sample,
                                            float eps, int blocks, void* summed, uint8_t* out, float* scales,
                                            void* stream) {
  SB_CHECK_ARG(x && out && scales, "sb_fp8_add_rms_norm_quantize: null pointer");
  SB_CHECK_ARG(dtype == SB_F32 || dtype == SB_BF16, "sb_fp8_add_rms_norm_quantize: bad dtype");
  SB_CHECK_ARG(M > 0 && C > 0 && M < (1ll << 31), "sb_fp8_add_rms_norm_quantize: M in [1, 2^31) and C positive");
  SB_CHECK_ARG((residual != nullptr) == (summed != nullptr),
               "sb_fp8_add_rms_norm_quantize: a residual and its sum come together");
  SB_CHECK_ARG(gate == nullptr || residual != nullptr, "sb_fp8_add_rms_norm_quantize: a gate needs a residual");
  SB_CHECK_ARG(x_stride >= C && (residual == nullptr || residual_stride >= C),
               "sb_fp8_add_rms_norm_quantize: rows overlap");
  SB_CHECK_ARG(rows_per_sample > 0 && M % rows_per_sample == 0,
               "sb_fp8_add_rms_norm_quantize: M must be a whole number of samples");
  SB_CHECK_ARG(blocks == 0 || blocks == 1, "sb_fp8_add_rms_norm_quantize: blocks must be 0 or 1");
  const int size = dtype == SB_BF16 ? 2 : 4;
  SB_CHECK_ARG(((uintptr_t)x | (uintptr_t)residual | (uintptr_t)summed) % size == 0 &&
                   ((uintptr_t)gate | (uintptr_t)weight | (uintptr_t)shift | (uintptr_t)scales) % 4 == 0,
               "sb_fp8_add_rms_norm_quantize: tensors must be aligned to their elements");
  if (C > 16384) {
    set_error("sb_fp8_add_rms_norm_quantize: rows of at most 16384 columns are supported, got %d", C);
    return SB_ERR_UNSUPPORTED;
  }
  NormParams p{};
  p.x = x;
  p.residual = residual;
  p.gate = gate;
  p.weight = weight;
  p.shift = shift;
  p.summed = summed;
  p.out = out;
  p.scales = scales;
  p.x_stride = x_stride;
  p.residual_stride = residual_stride;
  p.gate_stride = gate_stride;
  p.weight_stride = weight_stride;
  p.shift_stride = shift_stride;
  p.M = M;
  p.rows_per_sample = rows_per_sample;
  p.C = C;
  p.groups = ceil_div(C, kGroup);
  p.eps = eps;
  p.vec = C % 8 == 0 && x_stride * size % 16 == 0 && aligned16(x) && (uintptr_t)out % 8 == 0 &&
          (residual == nullptr || (residual_stride * size % 16 == 0 && aligned16(residual) && aligned16(summed)));
  p.vec_params = C % 8 == 0 && (gate == nullptr || (aligned16(gate) && gate_stride % 4 == 0)) &&
                 (weight == nullptr || (aligned16(weight) && weight_stride % 4 == 0)) &&
                 (shift == nullptr || (aligned16(shift) && shift_stride % 4 == 0));
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == SB_BF16)
    dispatch_norm<__nv_bfloat16>(p, blocks != 0, s);
  else
    dispatch_norm<float>(p, blocks != 0, s);
  SB_CHECK_LAUNCH("sb_fp8_add_rms_norm_quantize launch");
  return SB_OK;
}
