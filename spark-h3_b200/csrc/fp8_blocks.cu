// e4m3 quantisers with one scale per row and 128 columns, and the fused residual + RMSNorm +
// quantiser.  Each value is read once and kept in registers between the reduction that fixes
// its scale and the store of its code (norm rows of more than 8192 fp32 columns spill up to 280 bytes
// per thread).
//
// A warp holds a group of 128 columns, four consecutive ones per lane, so the group's maximum is
// one warp-wide reduction instruction.  What bounds these kernels is HBM once the instructions per
// value are few: at 6.5 TB/s an SM issues about 17 per bf16 value in the time that its three bytes
// take.  124992 x 4096 bf16: 232 us, 6.6 TB/s (half a warp per group with shuffles, 64-bit index
// divisions and exact divisions: 341); SwiGLU of 124992 x 2 x 2048: 226 us, 5.7 TB/s; GELU: 472 us,
// bound by its instructions.
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

// N (1, 2 or 4) consecutive elements in one access.
template <int N>
__device__ __forceinline__ void load_n(const __nv_bfloat16* p, float* v) {
  if (N == 1) {
    v[0] = __bfloat162float(*p);
  } else {
    uint32_t w[N / 2 > 0 ? N / 2 : 1];
    if (N == 4) {
      const uint2 raw = *reinterpret_cast<const uint2*>(p);
      w[0] = raw.x;
      w[N / 2 - 1] = raw.y;
    } else {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}
template <int N>
__device__ __forceinline__ void load_n(const float* p, float* v) {
  if (N == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    v[0] = a.x; v[1] = a.y; v[N - 2] = a.z; v[N - 1] = a.w;
  } else if (N == 2) {
    const float2 a = *reinterpret_cast<const float2*>(p);
    v[0] = a.x; v[N - 1] = a.y;
  } else {
    v[0] = *p;
  }
}
template <int N>
__device__ __forceinline__ void store_n(__nv_bfloat16* p, const float* v) {
  if (N == 4)
    *reinterpret_cast<uint2*>(p) = make_uint2(sm100::cvt_bf16x2(v[0], v[N > 1 ? 1 : 0]),
                                              sm100::cvt_bf16x2(v[N - 2 > 0 ? N - 2 : 0], v[N - 1]));
  else if (N == 2)
    *reinterpret_cast<uint32_t*>(p) = sm100::cvt_bf16x2(v[0], v[N - 1]);
  else
    *p = __float2bfloat16_rn(v[0]);
}
template <int N>
__device__ __forceinline__ void store_n(float* p, const float* v) {
  if (N == 4)
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[N > 1 ? 1 : 0], v[N - 2 > 0 ? N - 2 : 0], v[N - 1]);
  else if (N == 2)
    *reinterpret_cast<float2*>(p) = make_float2(v[0], v[N - 1]);
  else
    *p = v[0];
}

// A lane's four values from column c of a row with `cols` columns, N at a time (cols is then a
// multiple of N and the row's elements are aligned to N); columns past the end read as 0.
template <int N, typename T>
__device__ __forceinline__ void load_cols(const T* row, int c, int cols, float* v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = 0.f;
#pragma unroll
  for (int i = 0; i < 4; i += N)
    if (c + i < cols) load_n<N>(row + c + i, v + i);
}
template <int N, typename T>
__device__ __forceinline__ void store_cols(T* row, int c, int cols, const float* v) {
#pragma unroll
  for (int i = 0; i < 4; i += N)
    if (c + i < cols) store_n<N>(row + c + i, v + i);
}
// Codes of 4 values; cvt.satfinite clamps to +-448 and keeps NaN.
template <int N>
__device__ __forceinline__ void store_codes(uint8_t* row, int c, int cols, const float* v, float inv) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(v[1] * inv), "f"(v[0] * inv));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(v[3] * inv), "f"(v[2] * inv));
  if (N == 4) {
    if (c < cols) *reinterpret_cast<uint32_t*>(row + c) = (uint32_t)lo | (uint32_t)hi << 16;
  } else if (N == 2) {
    if (c < cols) *reinterpret_cast<uint16_t*>(row + c) = lo;
    if (c + 2 < cols) *reinterpret_cast<uint16_t*>(row + c + 2) = hi;
  } else {
    const uint32_t codes = (uint32_t)lo | (uint32_t)hi << 16;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c + i < cols) row[c + i] = (uint8_t)(codes >> (8 * i));
  }
}

enum Activation { kNone = 0, kSwiglu = 1, kGelu = 2 };

// a * sigmoid(g) * g, in this order: a * g alone may overflow where the value does not, and what
// underflows in a * sigmoid(g) stays far below the smallest scale.  1 + 2^(-g log2 e) may be infinite:
// its reciprocal is then 0, as in the limit.  (124992 x 2 x 2048 in 226 us; g * sigmoid(g) first takes two
// registers more, 34, so that six CTAs share an SM instead of eight: 263.)
__device__ __forceinline__ float swiglu(float a, float g) {
  return a * reciprocal(1.f + sm100::ex2_approx(g * -kLog2e)) * g;
}

// x * Phi(x).  A group may hold nothing but the negative tail, and its scale and codes need that tail
// relative to its size: Phi(-|x|) e^(x^2 / 2) is a polynomial of degree 7 in t = 1 / (1 + 0.26 |x|)
// without a constant term, fitted here for the least relative error (3e-7 up to |x| = 9.5; the value
// is below 1e-19 from there on, and the smallest scale 1e-12).  With its roundings y is off by less
// than (2^-18 + 1.25 x^2 2^-24) of itself.  Two special function units' results and 13 products per
// value (124992 x 4096: 472 us); erff's spelling, which cancels in the tail, takes 725 us.
__device__ __forceinline__ float gelu(float x) {
  constexpr float c1 = 0.103412218f, c2 = 0.108374767f, c3 = 0.0678653568f, c4 = 0.179113671f, c5 = -0.122419536f,
                  c6 = 0.239316165f, c7 = -0.0756627843f;
  const float t = reciprocal(fmaf(0.26f, fabsf(x), 1.f));
  const float poly = fmaf(fmaf(fmaf(fmaf(fmaf(fmaf(c7, t, c6), t, c5), t, c4), t, c3), t, c2), t, c1) * t;
  const float q = sm100::ex2_approx(x * x * (-0.5f * kLog2e)) * poly;
  return x * (x < 0.f ? q : 1.f - q);
}

// A warp takes U consecutive groups of a row; 2^row_shift (1, 2, 4 or 8) warps of a CTA share a row,
// blockIdx.y counts further 8 * U groups.
constexpr int kQuantThreads = 256;

template <typename T, int ACT, int U, int N>
__global__ void __launch_bounds__(kQuantThreads) quantize_blocks_kernel(const T* __restrict__ x, int64_t x_stride,
                                                                        int64_t M, int groups, int K, int row_shift,
                                                                        uint8_t* __restrict__ out,
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
    load_cols<N>(xr, c0 + u * kGroup, K, v[u]);
    if (ACT == kSwiglu) load_cols<N>(xr + K, c0 + u * kGroup, K, w[u]);
  }
  float mine = 0.f;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (ACT == kSwiglu) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[u][i] = swiglu(v[u][i], w[u][i]);
    } else if (ACT == kGelu) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[u][i] = gelu(v[u][i]);
    }
    const float scale = group_scale(warp_absmax(absmax4(v[u])));
    if (lane == u) mine = scale;
    store_codes<N>(yr, c0 + u * kGroup, K, v[u], reciprocal(scale));
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
  float eps;
};

// Four elements as loaded, unconverted.
template <typename T> struct Raw4;
template <> struct Raw4<__nv_bfloat16> {
  uint2 r;
  template <int N>
  __device__ __forceinline__ void load(const __nv_bfloat16* row, int c, int cols) {
    r = make_uint2(0u, 0u);
    if (N == 4) {
      if (c < cols) r = *reinterpret_cast<const uint2*>(row + c);
    } else if (N == 2) {
      if (c < cols) r.x = *reinterpret_cast<const uint32_t*>(row + c);
      if (c + 2 < cols) r.y = *reinterpret_cast<const uint32_t*>(row + c + 2);
    } else {
      const uint16_t* h = reinterpret_cast<const uint16_t*>(row);
      if (c + 0 < cols) r.x = h[c];
      if (c + 1 < cols) r.x |= (uint32_t)h[c + 1] << 16;
      if (c + 2 < cols) r.y = h[c + 2];
      if (c + 3 < cols) r.y |= (uint32_t)h[c + 3] << 16;
    }
  }
  __device__ __forceinline__ void get(float* v) const {
    v[0] = __uint_as_float(r.x << 16);
    v[1] = __uint_as_float(r.x & 0xffff0000u);
    v[2] = __uint_as_float(r.y << 16);
    v[3] = __uint_as_float(r.y & 0xffff0000u);
  }
};
template <> struct Raw4<float> {
  float r[4];
  template <int N>
  __device__ __forceinline__ void load(const float* row, int c, int cols) { load_cols<N>(row, c, cols, r); }
  __device__ __forceinline__ void get(float* v) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = r[i];
  }
};

constexpr int norm_threads(int W) { return 32 * (W == 1 ? 8 : W); }
// Rows up to 8192 columns (V <= 4) keep their columns of weight and shift in registers.
constexpr bool norm_keeps(int V) { return V <= 4; }
constexpr int norm_ctas(int W, int V) { return (V == 4 ? 512 : 768) / norm_threads(W); }  // per SM

// W warps per row (W = 1: eight rows per CTA), V groups of 128 columns per warp, in registers.  CTAs
// stay and walk the rows, R at a time: a row's work is a chain (sum over the CTA, then scale, then
// codes) of about 2000 cycles, so R rows go through it together, the next R rows in flight
// (unconverted) meanwhile.  The sum is rounded once, where it is stored; the norm works on the
// unrounded fp32 sum.  Measured at 124992 x 4096 bf16 with residual, gate and shift (3.6 GB): 600 us,
// 6.0 TB/s; 64-bit row arithmetic 615, one row at a time 659, one row per CTA without rows in flight
// 832, access-by-access alignment checks instead of the template's 746.
template <typename T, int W, int V, int R, bool BLOCKS, int N>
__global__ void __launch_bounds__(norm_threads(W), norm_ctas(W, V)) add_rms_norm_quantize_kernel(NormParams p) {
  constexpr bool KEEP = norm_keeps(V);
  __shared__ float red[2][2][R][W];  // [parity][sum, maximum][row][warp]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int part = W == 1 ? 0 : warp;
  const int c0 = part * kGroup + lane * 4;  // + j * W * kGroup
  // Row numbers and the few steps past the last one fit 32 bits (M < 2^31).
  const uint32_t M = (uint32_t)p.M, step = W == 1 ? gridDim.x * 8 : gridDim.x;
  uint32_t row = W == 1 ? blockIdx.x * 8 + warp : blockIdx.x;
  const T* x = static_cast<const T*>(p.x);
  const T* res = static_cast<const T*>(p.residual);
  Raw4<T> xr[R][V], rr[R][V];
  auto fetch = [&](uint32_t at) {
#pragma unroll
    for (int r = 0; r < R; ++r, at += step) {
      if (at >= M) break;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        xr[r][j].template load<N>(x + at * p.x_stride, c0 + j * W * kGroup, p.C);
        if (res != nullptr) rr[r][j].template load<N>(res + at * p.residual_stride, c0 + j * W * kGroup, p.C);
      }
    }
  };
  auto params = [&](const float* base, int64_t at, int j, float fill, float* v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = fill;
    if (base != nullptr) load_cols<N>(base + at, c0 + j * W * kGroup, p.C, v);
  };
  // The rows only go forward, so a sample is looked up (a division) only past the last one's end.
  const uint32_t per_sample = (uint32_t)p.rows_per_sample;
  uint32_t current = 0, current_end = per_sample;
  auto sample_of = [&](uint32_t at) {
    if (at >= current_end) {
      current = at / per_sample;
      current_end = (current + 1) * per_sample;
    }
    return current;
  };
  float weight[KEEP ? V : 1][4], shift[KEEP ? V : 1][4];
  uint32_t kept = ~0u;  // the sample of weight and shift

#pragma unroll
  for (int r = 0; r < R; ++r)  // rows past the end are computed on zeros and not stored
#pragma unroll
    for (int j = 0; j < V; ++j) {
      xr[r][j] = Raw4<T>{};
      rr[r][j] = Raw4<T>{};
    }
  if (row < M) fetch(row);
  for (int parity = 0; row < M; row += R * step, parity ^= 1) {
    float v[R][V][4], ss[R], rstd[R], amax[R];
    uint32_t sample[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint32_t at = row + r * step;
      sample[r] = at < M ? sample_of(at) : 0;
      const float* gate = p.gate == nullptr ? nullptr : p.gate + sample[r] * p.gate_stride;
      ss[r] = 0.f;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        xr[r][j].get(v[r][j]);
        if (res != nullptr) {
          float s[4], g[4];
          params(gate, 0, j, 1.f, g);
          rr[r][j].get(s);
#pragma unroll
          for (int i = 0; i < 4; ++i) v[r][j][i] = fmaf(g[i], v[r][j][i], s[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) ss[r] = fmaf(v[r][j][i], v[r][j][i], ss[r]);
      }
    }
    fetch(row + R * step);
    if (res != nullptr) {
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (row + r * step < M) {
#pragma unroll
          for (int j = 0; j < V; ++j)
            store_cols<N>(static_cast<T*>(p.summed) + (int64_t)(row + r * step) * p.C, c0 + j * W * kGroup, p.C, v[r][j]);
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      ss[r] = warp_sum(ss[r]);
      if (W > 1 && lane == 0) red[parity][0][r][part] = ss[r];
    }
    if (W > 1) {
      __syncthreads();  // also separates this use of red from the one two turns ago
#pragma unroll
      for (int r = 0; r < R; ++r) {
        ss[r] = red[parity][0][r][0];
#pragma unroll
        for (int i = 1; i < W; ++i) ss[r] += red[parity][0][r][i];
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      rstd[r] = rsqrtf(ss[r] / (float)p.C + p.eps);
      amax[r] = 0.f;
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t at = row + r * step;
      if (at >= M) break;
      if (KEEP && sample[r] != kept) {
#pragma unroll
        for (int j = 0; j < (KEEP ? V : 1); ++j) {
          params(p.weight, sample[r] * p.weight_stride, j, 1.f, weight[j]);
          params(p.shift, sample[r] * p.shift_stride, j, 0.f, shift[j]);
        }
      }
      kept = sample[r];
      uint8_t* out = p.out + at * p.C;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int kb = j * W + part;
        float w[4], b[4];
        if (!KEEP) {
          params(p.weight, sample[r] * p.weight_stride, j, 1.f, w);
          params(p.shift, sample[r] * p.shift_stride, j, 0.f, b);
        }
        // Columns past the end hold 0 * rstd (and a shift of 0), which adds nothing to the
        // maximum: rstd is NaN only where the row's values are too.
#pragma unroll
        for (int i = 0; i < 4; ++i)
          v[r][j][i] = fmaf(v[r][j][i] * rstd[r], KEEP ? weight[KEEP ? j : 0][i] : w[i], KEEP ? shift[KEEP ? j : 0][i] : b[i]);
        const float m = absmax4(v[r][j]);
        if (BLOCKS) {
          const float scale = group_scale(warp_absmax(m));
          if (lane == 0 && kb < p.groups) p.scales[at * p.groups + kb] = scale;
          store_codes<N>(out, c0 + j * W * kGroup, p.C, v[r][j], reciprocal(scale));
        } else {
          amax[r] = max_nan(amax[r], m);
        }
      }
    }
    if (!BLOCKS) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        amax[r] = warp_absmax(amax[r]);
        if (W > 1 && lane == 0) red[parity][1][r][part] = amax[r];
      }
      if (W > 1) __syncthreads();
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int64_t at = row + r * step;
        if (at >= M) break;
        if (W > 1) {
          amax[r] = red[parity][1][r][0];
#pragma unroll
          for (int i = 1; i < W; ++i) amax[r] = max_nan(amax[r], red[parity][1][r][i]);
        }
        const float scale = group_scale(amax[r]);
        if (part == 0 && lane == 0) p.scales[at] = scale;
        const float inv = reciprocal(scale);
#pragma unroll
        for (int j = 0; j < V; ++j) store_codes<N>(p.out + at * p.C, c0 + j * W * kGroup, p.C, v[r][j], inv);
      }
    }
  }
}

int sm_count() {
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

template <typename T, int W, int V, int N>
void launch_norm_n(const NormParams& p, bool blocks, cudaStream_t s) {
  // Two rows at a time where their unconverted columns take few registers.
  constexpr int kTogether = sizeof(T) == 2 && norm_keeps(V) && W > 1 ? 2 : 1;
  const int64_t ctas = W == 1 ? (p.M + 7) / 8 : p.M, resident = (int64_t)sm_count() * norm_ctas(W, V);
  const unsigned grid = (unsigned)(ctas < resident ? ctas : resident);
  if (blocks)
    add_rms_norm_quantize_kernel<T, W, V, kTogether, true, N><<<grid, norm_threads(W), 0, s>>>(p);
  else
    add_rms_norm_quantize_kernel<T, W, V, kTogether, false, N><<<grid, norm_threads(W), 0, s>>>(p);
}

template <typename T, int N>
void dispatch_norm(const NormParams& p, bool blocks, cudaStream_t s) {
  if (p.C <= 128) return launch_norm_n<T, 1, 1, N>(p, blocks, s);
  if (p.C <= 256) return launch_norm_n<T, 1, 2, N>(p, blocks, s);
  if (p.C <= 512) return launch_norm_n<T, 1, 4, N>(p, blocks, s);
  if (p.C <= 1024) return launch_norm_n<T, 4, 2, N>(p, blocks, s);
  if (p.C <= 2048) return launch_norm_n<T, 8, 2, N>(p, blocks, s);
  if (p.C <= 4096) return launch_norm_n<T, 8, 4, N>(p, blocks, s);
  if (p.C <= 6144) return launch_norm_n<T, 12, 4, N>(p, blocks, s);
  if (p.C <= 8192) return launch_norm_n<T, 16, 4, N>(p, blocks, s);
  return launch_norm_n<T, 24, 6, N>(p, blocks, s);
}

// Whether everything allows accesses of n elements: element counts and strides that are multiples of
// n, pointers aligned to n elements (size bytes each).
bool fits(int n, const void* p, int size, int64_t stride = 0) {
  return p == nullptr || ((uintptr_t)p % (uintptr_t)(n * size) == 0 && stride % n == 0);
}

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
  // Elements per access: every row (and the gate half) starts on that boundary.
  auto wide = [&](int n) { return K % n == 0 && fits(n, x, size, x_stride) && fits(n, out, 1); };
  const int n = wide(4) ? 4 : wide(2) ? 2 : 1;
  cudaStream_t s = (cudaStream_t)stream;
  // Few rows: one group per warp, for the most warps; otherwise four loads in flight per lane.
  const bool four = groups >= 4 && M * groups >= 4096;
  const int parts = four ? ceil_div(groups, 4) : groups;
  int row_shift = 0;
  while (row_shift < 3 && (1 << row_shift) < parts) ++row_shift;
  const int rows = 8 >> row_shift;
  const dim3 grid((unsigned)((M + rows - 1) / rows), (unsigned)ceil_div(parts, 8));
  auto launch = [&](auto element) {
    using T = decltype(element);
    auto kernel = four ? (n == 4   ? quantize_blocks_kernel<T, ACT, 4, 4>
                          : n == 2 ? quantize_blocks_kernel<T, ACT, 4, 2>
                                   : quantize_blocks_kernel<T, ACT, 4, 1>)
                       : (n == 4   ? quantize_blocks_kernel<T, ACT, 1, 4>
                          : n == 2 ? quantize_blocks_kernel<T, ACT, 1, 2>
                                   : quantize_blocks_kernel<T, ACT, 1, 1>);
    kernel<<<grid, kQuantThreads, 0, s>>>((const T*)x, x_stride, M, groups, K, row_shift, out, scales);
  };
  if (dtype == SB_BF16)
    launch(__nv_bfloat16{});
  else
    launch(float{});
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
  SB_CHECK_ARG(gate_stride >= 0 && weight_stride >= 0 && shift_stride >= 0,
               "sb_fp8_add_rms_norm_quantize: sample strides must not be negative");
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
  auto wide = [&](int n) {
    return C % n == 0 && fits(n, x, size, x_stride) && fits(n, residual, size, residual_stride) && fits(n, summed, size) &&
           fits(n, out, 1) && fits(n, gate, 4, gate_stride) && fits(n, weight, 4, weight_stride) &&
           fits(n, shift, 4, shift_stride);
  };
  const int n = wide(4) ? 4 : wide(2) ? 2 : 1;  // elements per access
  auto dispatch = [&](auto element) {
    using T = decltype(element);
    auto run = n == 4 ? dispatch_norm<T, 4> : n == 2 ? dispatch_norm<T, 2> : dispatch_norm<T, 1>;
    run(p, blocks != 0, (cudaStream_t)stream);
  };
  if (dtype == SB_BF16)
    dispatch(__nv_bfloat16{});
  else
    dispatch(float{});
  SB_CHECK_LAUNCH("sb_fp8_add_rms_norm_quantize launch");
  return SB_OK;
}
