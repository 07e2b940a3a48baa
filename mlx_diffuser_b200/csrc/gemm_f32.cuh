// Register tiles of exact fp32 products, shared by linear.cu and expert.cu.
#pragma once

#include "linear.h"

namespace sv {

constexpr int FK = 16;  // k per shared-memory stage

// Two fp32 multiply-adds in one instruction, each rounded like fmaf's.
__device__ __forceinline__ void fma_pair(uint64_t& c, uint64_t a, uint64_t b) {
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(c) : "l"(a), "l"(b));
}
__device__ __forceinline__ uint64_t twice(float x) {
  const uint32_t u = __float_as_uint(x);
  return (uint64_t)u << 32 | u;
}

// One operand's T rows x FK steps of a stage, by 256 threads in accesses of V elements: from global
// memory into registers, and from there into shared memory, steps outermost.
template <int T, int V>
struct Stage {
  static constexpr int PER = T * FK / 256;  // elements a thread
  // The e-th access's row r and step l, along one of which its elements lie.
  static __device__ __forceinline__ void place(bool mn, int e, int* r, int* l) {
    const int at = threadIdx.x + 256 * e;
    *r = mn ? at % (T / V) * V : at / (FK / V);
    *l = mn ? at / (T / V) : at % (FK / V) * V;
  }
  static __device__ __forceinline__ void fetch(const Operand& o, int64_t r0, int64_t rows,
                                               int64_t l0, int64_t l1, float (&v)[PER]) {
    const float* p = static_cast<const float*>(o.p);
#pragma unroll
    for (int e = 0; e < PER / V; ++e) {
      int r, l;
      place(o.mn, e, &r, &l);
      const int64_t i = r0 + r, ll = l0 + l;
      const float* from = p + (o.mn ? ll * o.ld + i : i * o.ld + ll);
      const int64_t left = i < rows && ll < l1 ? (o.mn ? rows - i : l1 - ll) : 0;
      if (V == 4 && left >= 4) {
        const float4 x = __ldg(reinterpret_cast<const float4*>(from));
        v[V * e] = x.x;
        v[V * e + 1 % V] = x.y;
        v[V * e + 2 % V] = x.z;
        v[V * e + 3 % V] = x.w;
      } else {
#pragma unroll
        for (int x = 0; x < V; ++x) v[V * e + x] = x < left ? __ldg(from + x) : 0.f;
      }
    }
  }
  static __device__ __forceinline__ void put(bool mn, float (*s)[T + 4], const float (&v)[PER]) {
#pragma unroll
    for (int e = 0; e < PER / V; ++e) {
      int r, l;
      place(mn, e, &r, &l);
      if (V == 4 && mn) {
        *reinterpret_cast<float4*>(&s[l][r]) =
            make_float4(v[V * e], v[V * e + 1 % V], v[V * e + 2 % V], v[V * e + 3 % V]);
      } else {
#pragma unroll
        for (int x = 0; x < V; ++x) {
          if (mn) s[l][r + x] = v[V * e + x];
          else s[l + x][r] = v[V * e + x];
        }
      }
    }
  }
};

// The sums of a tile of 16 R x 16 R by 256 threads: thread (tx, ty) = (tid % 16, tid / 16) has rows
// 64 (i / 4) + 4 ty + i % 4 and columns 64 (j / 4) + 4 tx + j % 4, two neighbouring columns a word.
// Rows from i0 below m, columns from j0 below n, k from k0 to k1.
template <int R, int VA, int VB>
__device__ __forceinline__ void tile_f32(const Operand& a, int64_t i0, int64_t m, const Operand& b,
                                         int64_t j0, int64_t n, int64_t k0, int64_t k1,
                                         float (*sa)[FK][16 * R + 4], float (*sb)[FK][16 * R + 4],
                                         uint64_t (&acc)[R][R / 2]) {
  using SA = Stage<16 * R, VA>;
  using SB = Stage<16 * R, VB>;
  const int tid = threadIdx.x;
  const int tx = tid % 16, ty = tid / 16;
  float ra[SA::PER], rb[SB::PER];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < R / 2; ++j) acc[i][j] = 0;
  SA::fetch(a, i0, m, k0, k1, ra);
  SB::fetch(b, j0, n, k0, k1, rb);
  SA::put(a.mn, sa[0], ra);
  SB::put(b.mn, sb[0], rb);
  __syncthreads();
  int buf = 0;
  for (int64_t l0 = k0; l0 < k1; l0 += FK, buf ^= 1) {
    const bool more = l0 + FK < k1;
    if (more) {
      SA::fetch(a, i0, m, l0 + FK, k1, ra);
      SB::fetch(b, j0, n, l0 + FK, k1, rb);
    }
#pragma unroll
    for (int l = 0; l < FK; ++l) {
      uint64_t av[R], bv[R / 2];
#pragma unroll
      for (int q = 0; q < R / 4; ++q) {
        const float4 x = *reinterpret_cast<const float4*>(&sa[buf][l][64 * q + 4 * ty]);
        av[4 * q] = twice(x.x);
        av[4 * q + 1] = twice(x.y);
        av[4 * q + 2] = twice(x.z);
        av[4 * q + 3] = twice(x.w);
        const ulonglong2 y =
            *reinterpret_cast<const ulonglong2*>(&sb[buf][l][64 * q + 4 * tx]);
        bv[2 * q] = y.x;
        bv[2 * q + 1] = y.y;
      }
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int j = 0; j < R / 2; ++j) fma_pair(acc[i][j], av[i], bv[j]);
    }
    if (more) {
      SA::put(a.mn, sa[buf ^ 1], ra);
      SB::put(b.mn, sb[buf ^ 1], rb);
      __syncthreads();
    }
  }
}

}  // namespace sv
