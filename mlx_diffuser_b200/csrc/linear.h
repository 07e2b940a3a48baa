// The projection's shared pieces: operands, the fused epilogue, and what the two matrix-product
// kernels (linear_tc.cu on the tensor cores, linear.cu on the CUDA cores) take.
#pragma once

#include "common.cuh"

namespace sv {

inline int elem_size(int dtype) {
  return dtype == SV_FLOAT32 ? 4 : (dtype == SV_FLOAT8_E4M3 ? 1 : 2);
}

// One operand of C[i][j] = sum_l A(i, l) B(j, l): element (i, l) is at p[i * ld + l], or at
// p[l * ld + i] when `mn` is set (the rows of the product run along memory).
struct Operand {
  const void* p;
  int64_t ld;
  bool mn;
};

// y = act(acc * row_scale[i] * col_scale[j] + bias[j]) + residual[i][j], every pointer optional;
// `preact` receives the activation's argument in fp32: rounded to 16 bits it would put a third of a
// step into every gradient, next to the step that rounding dz costs. With `partial` set the kernel
// stores its raw fp32 sums there ([splits][M][N]) and a second pass applies the rest.
struct Epilogue {
  const void* bias;      // [N], out_dtype
  const void* residual;  // out_dtype, rows ld_res apart
  int64_t ld_res;
  const float* row_scale;
  const float* col_scale;
  void* out;     // [M][N] contiguous, out_dtype
  float* preact;  // [M][N] contiguous
  float* partial;
  int out_dtype;
  int act;
};

struct Gemm {
  Operand a, b;
  int64_t m, n, k;
  int dtype;
  int splits;  // parts of the k axis
  Epilogue ep;
};

// Tensor-core tiles: 256 rows by a pair of CTAs, or 128 by one, and their columns.
enum class TcTile { kPair256, kPair128, kOne128, kOne64 };

// linear_tc.cu. Operands 16-byte aligned with row strides of a multiple of 16 bytes; no split of the
// k axis may be empty.
int gemm_tc(const Gemm& g, TcTile tile, int32_t* status, cudaStream_t s);

#ifdef __CUDACC__
constexpr float SQRT_HALF = 0.70710678118654752f;
constexpr float LOG2_E = 1.4426950408889634f;
constexpr float GELU_TANH_2C = 1.5957691216057308f;  // 2 sqrt(2 / pi)
constexpr float GELU_CUBE = 0.044715f;

__device__ __forceinline__ float exp2_half(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_half(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// exp and the quotient are the fast forms: within a few fp32 ulp of the value over the whole
// range (x / (1 + inf) is 0), which is the error the fp32 path's tolerance counts.
__device__ __forceinline__ float sigmoid_f(float x) {
  return __fdividef(1.0f, 1.0f + __expf(-x));
}

__device__ __forceinline__ float activate(float z, int act) {
  if (act == SV_ACT_SILU) return z * sigmoid_f(z);
  if (act == SV_ACT_GELU) return 0.5f * z * (1.0f + erff(z * SQRT_HALF));
  // 0.5 (1 + tanh(u)) = sigmoid(2u): no cancellation for negative z
  if (act == SV_ACT_GELU_TANH) return z * sigmoid_f(GELU_TANH_2C * (z + GELU_CUBE * z * z * z));
  return z;
}

// Phi(z), the normal distribution's integral, by Abramowitz and Stegun's 7.1.26, off by at most
// 7.5e-8: for the 16-bit types, whose rounding is far above that. `gauss`: exp(-z^2 / 2).
__device__ __forceinline__ float normal_half(float z, float gauss) {
  const float t = rcp_half(fmaf(0.3275911f * SQRT_HALF, fabsf(z), 1.0f));
  const float p = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f),
                                   -0.284496736f), 0.254829592f);
  const float tail = 0.5f * p * gauss;
  return z < 0.0f ? tail : 1.0f - tail;
}

// The activation for results of 16 bits: the approximate reciprocal and exponential are off by an
// fp32 ulp or two, and the factors of the exponent are folded.
__device__ __forceinline__ float activate_half(float z, int act) {
  if (act == SV_ACT_SILU) return z * rcp_half(1.0f + exp2_half(-LOG2_E * z));
  if (act == SV_ACT_GELU) return z * normal_half(z, exp2_half(-0.5f * LOG2_E * z * z));
  if (act == SV_ACT_GELU_TANH) {
    constexpr float A = -GELU_TANH_2C * LOG2_E;
    return z * rcp_half(1.0f + exp2_half(z * fmaf(A * GELU_CUBE, z * z, A)));
  }
  return z;
}

// The activation's derivative.
__device__ __forceinline__ float activate_slope(float z, int act) {
  if (act == SV_ACT_SILU) {
    const float g = sigmoid_f(z);
    return g * (1.0f + z * (1.0f - g));
  }
  if (act == SV_ACT_GELU)
    return 0.5f * (1.0f + erff(z * SQRT_HALF)) +
           z * 0.39894228040143268f * __expf(-0.5f * z * z);
  if (act == SV_ACT_GELU_TANH) {
    const float g = sigmoid_f(GELU_TANH_2C * (z + GELU_CUBE * z * z * z));
    // 1 - g is zero long before z^2 overflows
    return g + z * g * (1.0f - g) * GELU_TANH_2C * (1.0f + 3.0f * GELU_CUBE * fminf(z * z, 1e30f));
  }
  return 1.0f;
}

__device__ __forceinline__ float activate_slope_half(float z, int act) {
  if (act == SV_ACT_GELU) {
    const float gauss = exp2_half(-0.5f * LOG2_E * z * z);
    return normal_half(z, gauss) + z * 0.39894228040143268f * gauss;
  }
  return activate_slope(z, act);
}

template <typename O>
__device__ __forceinline__ void epilogue_store(const Epilogue& ep, int64_t i, int64_t j, int64_t n,
                                               float acc) {
  if (ep.row_scale) acc *= __ldg(ep.row_scale + i);
  if (ep.col_scale) acc *= __ldg(ep.col_scale + j);
  if (ep.bias) acc += to_f32(static_cast<const O*>(ep.bias)[j]);
  if (ep.preact) ep.preact[i * n + j] = acc;
  acc = activate(acc, ep.act);
  if (ep.residual) acc += to_f32(static_cast<const O*>(ep.residual)[i * ep.ld_res + j]);
  static_cast<O*>(ep.out)[i * n + j] = from_f32<O>(acc);
}
#endif

}  // namespace sv
