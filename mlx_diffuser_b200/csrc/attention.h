// Windowed attention with a learned relative position bias: what its kernels share.
#pragma once

#include "common.cuh"

namespace sv {

constexpr int ATTN_MAX_DIM = 128;
constexpr int ATTN_MAX_BUCKETS = 25;   // per axis
constexpr int ATTN_MAX_REACH = 1023;   // offsets beyond it share the outermost entries
constexpr int ATTN_MAX_HEADS = 65535;

// One row of the attention plan, in window order: the coordinates, the window's range of
// positions, and the feature row.
struct alignas(16) PlanRow {
  int32_t x, y, z;
  int32_t row;    // -1: not a row of the tensor (reported when the plan was built)
  int32_t start, end;
  int32_t pad[2];
};
static_assert(sizeof(PlanRow) == 32, "sv_window_plan writes 32 bytes a row");

struct AttnArgs {
  const void *q, *k, *v, *o, *dout;  // [n, heads, dim], the last axis contiguous
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;  // strides in elements
  void *out, *dq, *dk, *dv;          // contiguous [n, heads, dim]
  const PlanRow* plan;               // [n]
  const void* table;                 // [heads, nb, nb, nb]
  const int32_t* lut;                // [2 * reach + 1]
  float* lse;                        // [heads, n] by position: log of the softmax's denominator
  float* delta;                      // [heads, n] by position: sum_d dout * o
  unsigned long long* dtable;        // [heads, nb^3] fixed point, or null
  unsigned* norms;                   // [heads, 2]: bits of max |dout_i|^2 and max |v_j|^2
  int64_t n;
  int heads, dim, nb, reach;
  float scale;
};

#ifdef __CUDACC__
// Difference of two coordinates without wrap-around.
__device__ __forceinline__ int sub_sat(int a, int b) {
  int d;
  asm("sub.sat.s32 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

__device__ __forceinline__ int lut_at(const AttnArgs& a, int d) {
  const int v = __ldg(a.lut + max(-a.reach, min(a.reach, d)) + a.reach);
  return max(0, min(a.nb - 1, v));
}

// The bias table's fixed-point unit for a head: sums of |dS| over a row are at most
// 2 max|dout_i| max|v_j| (a softmax row sums to one and delta is a mean of the products it is
// subtracted from), so n rows of them stay below 2^62 in units of 2^-exponent. Integer sums do not
// depend on the order of the additions. INT_MAX when the bound is not finite.
__device__ __forceinline__ int dtable_exponent(const AttnArgs& a, int head) {
  const float g2 = __uint_as_float(a.norms[2 * head]), v2 = __uint_as_float(a.norms[2 * head + 1]);
  const double bound = 2.0 * sqrt((double)g2) * sqrt((double)v2) * (double)a.n;
  if (!(bound < 1e300)) return INT_MAX;
  if (bound == 0.0) return 0;
  int e;
  frexp(bound, &e);  // bound < 2^e
  return 61 - e;
}
#endif

}  // namespace sv
