// fp16 gradients as operands of a product, shared by linear.cu and expert.cu.
#pragma once

#include <algorithm>

#include "common.cuh"

namespace sv {

// dz is rounded to the feature type, since the tensor cores take it as an operand of both products: half
// a step more beside the result's own (0.0023 against 0.0017 over the gradients of 12,001 x 1024 x 1024
// bf16). fp16's is raised by a power of two first, and the products' column scales take that back: below
// 2^-14 a half has no 11 bits, and the gradients of a mean loss lie there. The power puts the largest |dy|
// times the largest |weight| that it is multiplied by below 2^15 (the activations' slopes are below 1.13),
// so values down to 2^-28 of it keep all their bits. It costs a pass over dy: 12,001 x 1024 in 7 us.
struct Raise {
  unsigned* top;  // [2]: bits of the largest |dy|, as a half, and of the largest finite |weight|; null: dz
                  // is not raised
  float* down;    // [k]: what the products are multiplied by
  int64_t k;
};
__device__ __forceinline__ float raise_of(unsigned top) {
  if (top == 0u || top >= 0x7c00u) return 1.0f;  // nothing, or not a number
  const float x = __half2float(__ushort_as_half((unsigned short)top));
  return __uint_as_float((268u - (__float_as_uint(x) >> 23)) << 23);  // 2^14 <= x * this < 2^15
}
// The power of two that puts the weight with these bits into [1/2, 1), between 2^-100 and 2^64: with
// raise_of's (2^-1 to 2^38) it and its reciprocal stay normal numbers.
__device__ __forceinline__ float room_of(unsigned weight) {
  return __uint_as_float(min(max(253 - (int)(weight >> 23), 27), 191) << 23);
}

namespace {
// The larger magnitudes of two pairs of halves; FINITE: infinities and NaN count as nothing.
template <bool FINITE>
__device__ __forceinline__ unsigned larger(unsigned most, unsigned x) {
  x &= 0x7fff7fffu;
  if constexpr (FINITE) x &= ~__vcmpgeu2(x, 0x7c007c00u);
  return __vmaxu2(most, x);
}

template <int V, bool FINITE>
__global__ void __launch_bounds__(256)
    top_kernel(const unsigned short* __restrict__ x, int64_t cells, const float* __restrict__ weights,
               int64_t count, unsigned* __restrict__ top) {
  unsigned most = 0u;  // of both halves of a word
  const int64_t step = (int64_t)gridDim.x * 256 * V;
#pragma unroll 4
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V; i < cells; i += step) {
    if constexpr (V == 8) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(x + i));
      most = larger<FINITE>(larger<FINITE>(most, v.x), v.y);
      most = larger<FINITE>(larger<FINITE>(most, v.z), v.w);
    } else {
      most = larger<FINITE>(most, x[i]);
    }
  }
  __shared__ unsigned s_top[2][8];
  unsigned heavy = 0u;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) {
    const unsigned w = __float_as_uint(__ldg(weights + i)) & 0x7fffffffu;
    if (w < 0x7f800000u) heavy = max(heavy, w);
  }
  const unsigned one = __reduce_max_sync(0xffffffffu, max(most & 0xffffu, most >> 16));
  heavy = __reduce_max_sync(0xffffffffu, heavy);
  if ((threadIdx.x & 31) == 0) {
    s_top[0][threadIdx.x >> 5] = one;
    s_top[1][threadIdx.x >> 5] = heavy;
  }
  __syncthreads();
  if (threadIdx.x < 32) {  // one atomic a block: one a warp took 11 us
    const unsigned all = __reduce_max_sync(0xffffffffu, threadIdx.x < 8 ? s_top[0][threadIdx.x] : 0u);
    heavy = __reduce_max_sync(0xffffffffu, threadIdx.x < 8 ? s_top[1][threadIdx.x] : 0u);
    if (threadIdx.x == 0 && all) atomicMax(top, all);
    if (threadIdx.x == 0 && heavy) atomicMax(top + 1, heavy);
  }
}

// top[0] = the largest magnitude of `cells` halves, as the bits of a half, top[1] = that of `count` weights.
template <bool FINITE>
inline int find_top(const void* dy, int64_t cells, const float* weights, int64_t count, unsigned* top,
                    cudaStream_t s) {
  SV_CUDA_TRY(cudaMemsetAsync(top, 0, 2 * sizeof(unsigned), s));
  const unsigned short* x = static_cast<const unsigned short*>(dy);
  const bool wide = cells % 8 == 0 && aligned16(dy);
  const unsigned blocks = (unsigned)std::min<int64_t>((cells / (wide ? 8 : 1) + 255) / 256,
                                                      (int64_t)num_sms() * 8);
  if (wide) top_kernel<8, FINITE><<<blocks, 256, 0, s>>>(x, cells, weights, count, top);
  else top_kernel<1, FINITE><<<blocks, 256, 0, s>>>(x, cells, weights, count, top);
  SV_LAUNCH_CHECK();
  return SV_OK;
}
}  // namespace

}  // namespace sv
