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

// The logistic function and its slope, from exp(-|x|): neither overflows, and neither is a difference
// of nearly equal numbers, so both are within a few fp32 ulp down to the subnormal numbers.
struct Sigmoid {
  float value, slope;
};
__device__ __forceinline__ Sigmoid sigmoid_f(float x) {
  const float e = expf(-fabsf(x));
  const float inv = 1.0f / (1.0f + e);
  return {x < 0.0f ? e * inv : inv, e * inv * inv};
}

// For fp32 results. The fast exponential is off by 2 + 1.16 |x| ulp, which the tails would show. Phi(z)
// is half of erfc(-z / sqrt 2): 1 + erf cancels for negative z. What is left in the tails is the rounding of
// the argument, which the function multiplies: by |u| for the tanh form's u, by z^2 for Phi.
__device__ __forceinline__ float tanh_argument(float z) {
  return GELU_TANH_2C * (z + GELU_CUBE * z * z * z);
}
__device__ __forceinline__ float activate(float z, int act) {
  if (act == SV_ACT_SILU) return z * sigmoid_f(z).value;
  if (act == SV_ACT_GELU) return 0.5f * z * erfcf(-z * SQRT_HALF);
  // 0.5 (1 + tanh(u)) = sigmoid(2u): no cancellation for negative z
  if (act == SV_ACT_GELU_TANH) return z * sigmoid_f(tanh_argument(z)).value;
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
    const Sigmoid g = sigmoid_f(z);
    return g.value + z * g.slope;
  }
  if (act == SV_ACT_GELU)
    return 0.5f * erfcf(-z * SQRT_HALF) + z * 0.39894228040143268f * expf(-0.5f * z * z);
  if (act == SV_ACT_GELU_TANH) {
    const Sigmoid g = sigmoid_f(tanh_argument(z));
    // g.slope is zero long before z^2 overflows
    return g.value + z * g.slope * GELU_TANH_2C * (1.0f + 3.0f * GELU_CUBE * fminf(z * z, 1e30f));
  }
  return 1.0f;
}

// And for 16 bits, by the approximate exponential and reciprocal.
__device__ __forceinline__ Sigmoid sigmoid_half(float x) {
  const float e = exp2_half(-LOG2_E * fabsf(x));
  const float inv = rcp_half(1.0f + e);
  return {x < 0.0f ? e * inv : inv, e * inv * inv};
}
__device__ __forceinline__ float activate_slope_half(float z, int act) {
  if (act == SV_ACT_SILU) {
    const Sigmoid g = sigmoid_half(z);
    return g.value + z * g.slope;
  }
  if (act == SV_ACT_GELU) {
    const float gauss = exp2_half(-0.5f * LOG2_E * z * z);
    return normal_half(z, gauss) + z * 0.39894228040143268f * gauss;
  }
  if (act == SV_ACT_GELU_TANH) {
    const Sigmoid g = sigmoid_half(tanh_argument(z));
    return g.value + z * g.slope * GELU_TANH_2C * (1.0f + 3.0f * GELU_CUBE * fminf(z * z, 1e30f));
  }
  return 1.0f;
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
