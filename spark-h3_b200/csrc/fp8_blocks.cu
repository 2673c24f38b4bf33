// e4m3 quantisers with one scale per row and 128 columns, and the fused residual + RMSNorm +
// quantiser.  Each value is read once and kept in registers between the reduction that fixes
// its scale and the store of its code.
//
// A warp holds a group of 128 columns, four consecutive ones per lane, so the group's maximum is
// one warp-wide reduction instruction.  What bounds these kernels is HBM once the instructions per
// value are few: at 6.5 TB/s an SM issues about 17 per bf16 value in the time that its three bytes
// take (the first form, half a warp per group with eight shuffle steps, 64-bit index divisions and
// exact divisions, took 24 and ran at 4.5 TB/s; GELU with erff took 50).
//
// Scales and special values follow torch's spelling of the same arithmetic: scale =
// max(absmax * fp32(1/448), 1e-12) and the maximum propagates NaN, so a NaN in a group makes
// the whole group NaN, and an infinity makes its group's finite values 0 and itself NaN.
//
// A code is e4m3(y * r), r the hardware reciprocal of the scale (off by at most 2^-23 of itself):
// the quotient is off by less than 2^-22 of itself, so a code differs from e4m3(y / scale) only
// where y / scale lies that close to the middle of two codes.
#include "common.cuh"
#include "sm100_ptx.cuh"

namespace sb {
namespace {

constexpr int kGroup = 128;        // columns per scale
constexpr float kInv448 = 1.0f / 448.0f;

__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float absmax4(const float* v) {
  float m, d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(v[0]), "f"(v[1]), "f"(v[2]));
  asm("max.NaN.abs.f32 %0, %1, %2, %2;" : "=f"(d) : "f"(m), "f"(v[3]));
  return d;
}
// Maximum magnitude over the warp.
__device__ __forceinline__ float warp_absmax(float x) {
  float d;
  asm volatile("redux.sync.max.abs.NaN.f32 %0, %1, 0xffffffff;" : "=f"(d) : "f"(x));
  return d;
}
__device__ __forceinline__ float reciprocal(float x) {
  float d;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(x));
  return d;
}
__device__ __forceinline__ float group_scale(float absmax) { return max_nan(absmax * kInv448, 1e-12f); }

__device__ __forceinline__ void load4(const __nv_bfloat16* p, float* v) {
  const uint2 raw = *reinterpret_cast<const uint2*>(p);
  v[0] = __uint_as_float(raw.x << 16);
  v[1] = __uint_as_float(raw.x & 0xffff0000u);
  v[2] = __uint_as_float(raw.y << 16);
  v[3] = __uint_as_float(raw.y & 0xffff0000u);
}
__device__ __forceinline__ void load4(const float* p, float* v) {
  const float4 a = *reinterpret_cast<const float4*>(p);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, const float* v) {
  *reinterpret_cast<uint2*>(p) = make_uint2(sm100::cvt_bf16x2(v[0], v[1]), sm100::cvt_bf16x2(v[2], v[3]));
}
__device__ __forceinline__ void store4(float* p, const float* v) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}

// 4 values from column c of a row with `cols` columns; columns past the end read as `fill`.  `vec`:
// the row's groups of four are aligned to their size (its columns are then a multiple of 4).
template <typename T>
__device__ __forceinline__ void load_cols(const T* row, int c, int cols, bool vec, float* v, float fill = 0.f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = fill;
  if (vec) {
    if (c < cols) load4(row + c, v);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c + i < cols) v[i] = Elem<T>::to_f(row[c + i]);
  }
}
template <typename T>
__device__ __forceinline__ void store_cols(T* row, int c, int cols, bool vec, const float* v) {
  if (vec) {
    if (c < cols) store4(row + c, v);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c + i < cols) row[c + i] = Elem<T>::from_f(v[i]);
  }
}
// Codes of 4 values; cvt.satfinite clamps to +-448 and keeps NaN.
__device__ __forceinline__ void store_codes(uint8_t* row, int c, int cols, bool vec, const float* v, float inv) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(v[1] * inv), "f"(v[0] * inv));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(v[3] * inv), "f"(v[2] * inv));
  const uint32_t codes = (uint32_t)lo | (uint32_t)hi << 16;
  if (vec) {
    if (c < cols) *reinterpret_cast<uint32_t*>(row + c) = codes;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c + i < cols) row[c + i] = (uint8_t)(codes >> (8 * i));
  }
}

enum Activation { kNone = 0, kSwiglu = 1, kGelu = 2 };

// a * g * sigmoid(g).  1 + 2^(-g log2 e) may be infinite: its reciprocal is then 0, as in the limit.
__device__ __forceinline__ float swiglu(float a, float g) {
  return a * g * reciprocal(1.f + sm100::ex2_approx(g * -kLog2e));
}

// x * Phi(x).  For x <= 0, Phi(x) = e^(-x^2 / 2) R(|x|) with R(t) = erfcx(t / sqrt 2) / 2 (half the
// scaled complementary error function), smooth and without a reciprocal: a degree-11 polynomial on
// [0, 5.25], fitted here by iteratively reweighted least squares at Chebyshev nodes with weight
// e^(-t^2 / 2) (1 + t).  Phi is off by at most 1.2e-7 (two steps of fp32 below 1), erff's own
// spelling 0.5 (1 + erf) by 0.9e-7; R keeps its last value past 5.25, where Phi < 1e-7.
__device__ __forceinline__ void gelu4(float* x) {
  constexpr float kR[12] = {0.49999991059303284f,     -0.3989359736442566f,   0.24991749227046967f,
                            -0.13254864513874054f,    0.061310868710279465f,  -0.024627279490232468f,
                            0.008287804201245308f,    -0.00220593623816967f,  0.0004333607212174684f,
                            -5.778570630354807e-05f,  4.603743946063332e-06f, -1.6388463563998812e-07f};
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    const uint64_t t = sm100::f2_pack(fminf(fabsf(x[i]), 5.25f), fminf(fabsf(x[i + 1]), 5.25f));
    uint64_t r = sm100::f2_pack(kR[11], kR[11]);
#pragma unroll
    for (int k = 10; k >= 0; --k) r = sm100::f2_fma(r, t, sm100::f2_pack(kR[k], kR[k]));
    const uint64_t xx = sm100::f2_pack(x[i], x[i + 1]);
    const uint64_t e = sm100::f2_mul(sm100::f2_mul(xx, xx), sm100::f2_pack(-0.5f * kLog2e, -0.5f * kLog2e));
    float e0, e1, q0, q1;
    sm100::f2_unpack(e, e0, e1);
    sm100::f2_unpack(sm100::f2_mul(r, sm100::f2_pack(sm100::ex2_approx(e0), sm100::ex2_approx(e1))), q0, q1);
    x[i] *= x[i] < 0.f ? q0 : 1.f - q0;
    x[i + 1] *= x[i + 1] < 0.f ? q1 : 1.f - q1;
  }
}

// A warp takes U consecutive groups of a row; `row_warps` (1, 2, 4 or 8) warps of a CTA share a
// row, blockIdx.y counts further 8 * U groups.
constexpr int kQuantThreads = 256;

template <typename T, int ACT, int U>
__global__ void __launch_bounds__(kQuantThreads) quantize_blocks_kernel(const T* __restrict__ x, int64_t x_stride,
                                                                        int64_t M, int groups, int K, int row_shift,
                                                                        int vec, uint8_t* __restrict__ out,
                                                                        float* __restrict__ scales) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = ((int64_t)blockIdx.x << (3 - row_shift)) + (warp >> row_shift);
  const int g0 = (blockIdx.y * 8 + (warp & ((1 << row_shift) - 1))) * U;
  if (row >= M || g0 >= groups) return;  // whole warps leave
  const T* xr = x + row * x_stride;
  uint8_t* yr = out + row * K;
  const int c0 = g0 * kGroup + lane * 4;
  float v[U][4], w[ACT == kSwiglu ? U : 1][4];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    load_cols(xr, c0 + u * kGroup, K, vec, v[u]);
    if (ACT == kSwiglu) load_cols(xr + K, c0 + u * kGroup, K, vec, w[u]);
  }
  float mine = 0.f;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (ACT == kSwiglu) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[u][i] = swiglu(v[u][i], w[u][i]);
    } else if (ACT == kGelu) {
      gelu4(v[u]);
    }
    const float scale = group_scale(warp_absmax(absmax4(v[u])));
    if (lane == u) mine = scale;
    store_codes(yr, c0 + u * kGroup, K, vec, v[u], reciprocal(scale));
  }
  if (lane < U && g0 + lane < groups) scales[row * groups + g0 + lane] = mine;
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
  int vec, vec_params;  // vector accesses to the rows / to the parameter vectors
  float eps;
};

// R consecutive rows of one sample per CTA of W warps (W = 1: one row per warp, eight to a CTA), V
// groups of 128 columns per warp and row, all in registers.  Two rows share the loads of gate,
// weight and shift, which outweigh a row's own bytes.  The sum is rounded once, where it is
// stored; the norm works on the unrounded fp32 sum.
template <typename T, int W, int V, int R, bool BLOCKS>
__global__ void __launch_bounds__(32 * (W == 1 ? 8 : W)) add_rms_norm_quantize_kernel(NormParams p) {
  __shared__ float red[2][R][W];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int part = W == 1 ? 0 : warp;
  const int64_t row0 = W == 1 ? (int64_t)blockIdx.x * 8 + warp : (int64_t)blockIdx.x * R;
  if (W == 1 && row0 >= p.M) return;  // whole warps leave
  const int rows = R == 1 ? 1 : (int)min((int64_t)R, p.M - row0);
  const int64_t sample = p.rows_per_sample == p.M ? 0 : (uint32_t)row0 / (uint32_t)p.rows_per_sample;
  const T* x = static_cast<const T*>(p.x) + row0 * p.x_stride;
  float v[R][V][4];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c = (j * W + part) * kGroup + lane * 4;
#pragma unroll
    for (int r = 0; r < R; ++r) load_cols(x + (r < rows ? r : 0) * p.x_stride, c, p.C, p.vec, v[r][j]);
  }
  float ss[R];
#pragma unroll
  for (int r = 0; r < R; ++r) ss[r] = 0.f;
  if (p.residual != nullptr) {
    const T* res = static_cast<const T*>(p.residual) + row0 * p.residual_stride;
    const float* gate = p.gate != nullptr ? p.gate + sample * p.gate_stride : nullptr;
    T* sum = static_cast<T*>(p.summed) + row0 * p.C;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (j * W + part) * kGroup + lane * 4;
      float g[4] = {1.f, 1.f, 1.f, 1.f};
      if (gate != nullptr) load_cols(gate, c, p.C, p.vec_params, g);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float s[4];
        load_cols(res + (r < rows ? r : 0) * p.residual_stride, c, p.C, p.vec, s);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[r][j][i] = fmaf(g[i], v[r][j][i], s[i]);
      }
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (r < rows) store_cols(sum + (int64_t)r * p.C, c, p.C, p.vec, v[r][j]);
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) ss[r] = fmaf(v[r][j][i], v[r][j][i], ss[r]);
    ss[r] = warp_sum(ss[r]);
    if (W > 1 && lane == 0) red[0][r][part] = ss[r];
  }
  if (W > 1) {
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      ss[r] = red[0][r][0];
#pragma unroll
      for (int i = 1; i < W; ++i) ss[r] += red[0][r][i];
    }
  }
  float rstd[R], amax[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    rstd[r] = rsqrtf(ss[r] / (float)p.C + p.eps);
    amax[r] = 0.f;
  }
  const float* weight = p.weight != nullptr ? p.weight + sample * p.weight_stride : nullptr;
  const float* shift = p.shift != nullptr ? p.shift + sample * p.shift_stride : nullptr;
  uint8_t* out = p.out + row0 * p.C;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int kb = j * W + part, c = kb * kGroup + lane * 4;
    float w[4] = {1.f, 1.f, 1.f, 1.f}, b[4] = {0.f, 0.f, 0.f, 0.f};
    if (weight != nullptr) load_cols(weight, c, p.C, p.vec_params, w);
    if (shift != nullptr) load_cols(shift, c, p.C, p.vec_params, b);
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[r][j][i] = fmaf(v[r][j][i] * rstd[r], w[i], b[i]);
      // Columns past the end stay out of the maximum: their value is 0 unless rstd is not finite
      // (w and b read as 0 there), and then the whole row is NaN or 0 already.
      const float m = absmax4(v[r][j]);
      if (BLOCKS) {
        const float scale = group_scale(warp_absmax(m));
        if (r < rows) {
          if (lane == 0 && kb < p.groups) p.scales[(row0 + r) * p.groups + kb] = scale;
          store_codes(out + (int64_t)r * p.C, c, p.C, p.vec, v[r][j], reciprocal(scale));
        }
      } else {
        amax[r] = max_nan(amax[r], m);
      }
    }
  }
  if (!BLOCKS) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      amax[r] = warp_absmax(amax[r]);
      if (W > 1 && lane == 0) red[1][r][part] = amax[r];
    }
    if (W > 1) __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (W > 1) {
        amax[r] = red[1][r][0];
#pragma unroll
        for (int i = 1; i < W; ++i) amax[r] = max_nan(amax[r], red[1][r][i]);
      }
      if (r >= rows) continue;
      const float scale = group_scale(amax[r]);
      if (part == 0 && lane == 0) p.scales[row0 + r] = scale;
      const float inv = reciprocal(scale);
#pragma unroll
      for (int j = 0; j < V; ++j)
        store_codes(out + (int64_t)r * p.C, (j * W + part) * kGroup + lane * 4, p.C, p.vec, v[r][j], inv);
    }
  }
}

template <typename T, int W, int V, int R>
void launch_norm(const NormParams& p, bool blocks, cudaStream_t s) {
  const unsigned grid = (unsigned)(W == 1 ? (p.M + 7) / 8 : (p.M + R - 1) / R);
  if (blocks)
    add_rms_norm_quantize_kernel<T, W, V, R, true><<<grid, 32 * (W == 1 ? 8 : W), 0, s>>>(p);
  else
    add_rms_norm_quantize_kernel<T, W, V, R, false><<<grid, 32 * (W == 1 ? 8 : W), 0, s>>>(p);
}

template <typename T>
void dispatch_norm(const NormParams& p, bool blocks, cudaStream_t s) {
  // Two rows per CTA where they belong to one sample and leave enough CTAs to fill the GPU.
  const bool two = p.rows_per_sample % 2 == 0 && p.M >= 4096;
  if (p.C <= 128) return launch_norm<T, 1, 1, 1>(p, blocks, s);
  if (p.C <= 256) return launch_norm<T, 1, 2, 1>(p, blocks, s);
  if (p.C <= 512) return launch_norm<T, 1, 4, 1>(p, blocks, s);
  if (p.C <= 1024 && p.M >= 4096) return launch_norm<T, 1, 8, 1>(p, blocks, s);
  if (p.C <= 2048) return two ? launch_norm<T, 4, 4, 2>(p, blocks, s) : launch_norm<T, 8, 2, 1>(p, blocks, s);
  if (p.C <= 4096) return two ? launch_norm<T, 8, 4, 2>(p, blocks, s) : launch_norm<T, 8, 4, 1>(p, blocks, s);
  if (p.C <= 8192) return two ? launch_norm<T, 16, 4, 2>(p, blocks, s) : launch_norm<T, 16, 4, 1>(p, blocks, s);
  return launch_norm<T, 16, 8, 1>(p, blocks, s);
}

bool aligned16(const void* p) { return ((uintptr_t)p % 16) == 0; }

template <int ACT>
int quantize_blocks(const char* what, const void* x, int64_t x_stride, int dtype, int64_t M, int K, uint8_t* out,
                    float* scales, void* stream) {
  SB_CHECK_ARG(x && out && scales, "%s: null pointer", what);
  SB_CHECK_ARG(dtype == SB_F32 || dtype == SB_BF16, "%s: bad dtype", what);
  SB_CHECK_ARG(M > 0 && K > 0 && M < (1ll << 31) && K <= (1 << 24), "%s: M in [1, 2^31) and K in [1, 2^24]", what);
  const int cols = ACT == kSwiglu ? 2 * K : K;
  SB_CHECK_ARG(x_stride >= cols, "%s: rows overlap (stride %lld, %d columns)", what, (long long)x_stride, cols);
  const int size = dtype == SB_BF16 ? 2 : 4;
  SB_CHECK_ARG((uintptr_t)x % size == 0 && (uintptr_t)scales % 4 == 0, "%s: x and scales must be aligned to their elements",
               what);
  const int groups = ceil_div(K, kGroup);
  // Vector accesses need every row (and the gate half) on a boundary of four elements.
  const int vec = K % 4 == 0 && x_stride % 4 == 0 && (uintptr_t)x % (4 * size) == 0 && (uintptr_t)out % 4 == 0;
  cudaStream_t s = (cudaStream_t)stream;
  // Few rows: one group per warp, for the most warps; otherwise four loads in flight per lane.
  const bool four = groups >= 4 && M * groups >= 4096;
  const int parts = four ? ceil_div(groups, 4) : groups;
  int row_shift = 0;
  while (row_shift < 3 && (1 << row_shift) < parts) ++row_shift;
  const int rows = 8 >> row_shift;
  const dim3 grid((unsigned)((M + rows - 1) / rows), (unsigned)ceil_div(parts, 8));
  if (dtype == SB_BF16) {
    const __nv_bfloat16* h = (const __nv_bfloat16*)x;
    if (four)
      quantize_blocks_kernel<__nv_bfloat16, ACT, 4>
          <<<grid, kQuantThreads, 0, s>>>(h, x_stride, M, groups, K, row_shift, vec, out, scales);
    else
      quantize_blocks_kernel<__nv_bfloat16, ACT, 1>
          <<<grid, kQuantThreads, 0, s>>>(h, x_stride, M, groups, K, row_shift, vec, out, scales);
  } else {
    const float* f = (const float*)x;
    if (four)
      quantize_blocks_kernel<float, ACT, 4>
          <<<grid, kQuantThreads, 0, s>>>(f, x_stride, M, groups, K, row_shift, vec, out, scales);
    else
      quantize_blocks_kernel<float, ACT, 1>
          <<<grid, kQuantThreads, 0, s>>>(f, x_stride, M, groups, K, row_shift, vec, out, scales);
  }
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
  const uintptr_t row_bytes = 4 * size;
  p.vec = C % 4 == 0 && x_stride % 4 == 0 && (uintptr_t)x % row_bytes == 0 && (uintptr_t)out % 4 == 0 &&
          (residual == nullptr || (residual_stride % 4 == 0 && (uintptr_t)residual % row_bytes == 0 &&
                                   (uintptr_t)summed % row_bytes == 0));
  p.vec_params = C % 4 == 0 && (gate == nullptr || (aligned16(gate) && gate_stride % 4 == 0)) &&
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
