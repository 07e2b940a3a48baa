// Pieces that the tensor-core products share (linear_tc.cu, expert_tc.cu): the tile's constants, what a
// pair of CTAs needs, and the fused epilogue.
#pragma once

#include "linear.h"

namespace sv {

constexpr int TM = 128;  // rows of a CTA's tile
constexpr int TC_THREADS = 320;
constexpr int EPI_THREADS = 256;
constexpr int EPI_WARPS = EPI_THREADS / 32;
constexpr uint32_t ATOM = 1024;           // 8 rows of 128 bytes
constexpr uint32_t MN_STRIDE = 8 * ATOM;  // next 64 rows of an MN-major operand
constexpr int CHUNK_LD = 36;  // floats between staged rows: 16-byte rows in different banks

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The address of the first CTA's copy of a shared-memory object.
__device__ __forceinline__ uint32_t in_first(uint32_t addr) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}

__device__ __forceinline__ void arrive_at(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr)
               : "memory");
}

__device__ __forceinline__ void tma_load_pair(uint32_t dst, const void* tmap, uint32_t bar,
                                              int32_t x, int32_t y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(tmap), "r"(bar), "r"(x), "r"(y)
      : "memory");
}

template <bool PAIR, bool F8>
__device__ __forceinline__ void issue_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                          uint32_t more) {
#define SV_MMA(group, kind)                                                    \
  asm volatile(                                                                \
      "{\n\t.reg .pred p;\n\t"                                                 \
      "setp.ne.b32 p, %4, 0;\n\t"                                              \
      "tcgen05.mma.cta_group::" group ".kind::" kind " [%0], %1, %2, %3, p;\n\t}" ::"r"(d), \
      "l"(a), "l"(b), "r"(idesc), "r"(more)                                    \
      : "memory")
  if constexpr (PAIR && F8) SV_MMA("2", "f8f6f4");
  else if constexpr (PAIR) SV_MMA("2", "f16");
  else if constexpr (F8) SV_MMA("1", "f8f6f4");
  else SV_MMA("1", "f16");
#undef SV_MMA
}

// Arrive, in both CTAs of a pair, when every product issued so far has completed.
template <bool PAIR>
__device__ __forceinline__ void commit(uint64_t* bar) {
  if constexpr (PAIR)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
        "[%0], %1;" ::"r"(smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
  else
    tc_commit(bar);
}

template <bool PAIR>
__device__ __forceinline__ void alloc_tmem(uint32_t* dst, uint32_t cols) {
  if constexpr (PAIR) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(dst)),
                 "r"(cols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  } else {
    tmem_alloc(dst, cols);
    tmem_relinquish();
  }
}

template <bool PAIR>
__device__ __forceinline__ void free_tmem(uint32_t addr, uint32_t cols) {
  if constexpr (PAIR)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols));
  else
    tmem_dealloc(addr, cols);
}

__device__ __forceinline__ void epi_sync() {
  asm volatile("bar.sync 1, %0;" ::"n"(EPI_THREADS) : "memory");
}

template <int ACT, int R, int W>
__device__ __forceinline__ void activate_all(float (&v)[R][W]) {
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < W; ++j) v[i][j] = activate_half(v[i][j], ACT);
}

// R rows of W consecutive columns: scale, bias, activation, residual, stores. Step by step over all
// of them, so that the rows' loads are in flight together. `at`, `at_res`: the first row's offsets.
template <typename O, int R, int W>
__device__ __forceinline__ void finish(const Epilogue& ep, float (&v)[R][W], const float* bias,
                                       const float* scale, bool scaled, int64_t row, int step,
                                       int rows, int64_t n, int64_t col) {
  O res[R][W];
  if (ep.residual) {
    const O* src = static_cast<const O*>(ep.residual) + row * ep.ld_res + col;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if constexpr (W == 8) {
        if (i * step < rows)
          *reinterpret_cast<uint4*>(res[i]) =
              __ldg(reinterpret_cast<const uint4*>(src + i * step * ep.ld_res));
      } else {
        // no branch (the last row again): behind one, each load was waited for in turn, and an odd
        // 5,041 x 331 -> 517 took 25 us
        res[i][0] = __ldg(src);
        src += (i + 1) * step < rows ? step * ep.ld_res : 0;
      }
    }
  }
  if (scaled) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const float by = ep.row_scale && i * step < rows ? __ldg(ep.row_scale + row + i * step) : 1.f;
#pragma unroll
      for (int j = 0; j < W; ++j) v[i][j] *= by * scale[j];
    }
  }
  if (ep.bias) {
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < W; ++j) v[i][j] += bias[j];
  }
  if (ep.preact) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (i * step < rows) {
        float* dst = ep.preact + (row + i * step) * n + col;
        if constexpr (W == 8) {
          *reinterpret_cast<float4*>(dst) = *reinterpret_cast<const float4*>(v[i]);
          *reinterpret_cast<float4*>(dst + 4) = *reinterpret_cast<const float4*>(v[i] + 4);
        } else {
          *dst = v[i][0];
        }
      }
    }
  }
  if (ep.act == SV_ACT_SILU) activate_all<SV_ACT_SILU>(v);
  else if (ep.act == SV_ACT_GELU) activate_all<SV_ACT_GELU>(v);
  else if (ep.act == SV_ACT_GELU_TANH) activate_all<SV_ACT_GELU_TANH>(v);
  if (ep.residual) {
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < W; ++j) v[i][j] += to_f32(res[i][j]);
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (i * step < rows) {
      O* dst = static_cast<O*>(ep.out) + (row + i * step) * n + col;
      if constexpr (W == 8) {
        uint4 raw;
        O* e = reinterpret_cast<O*>(&raw);
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = from_f32<O>(v[i][j]);
        *reinterpret_cast<uint4*>(dst) = raw;
      } else {
        *dst = from_f32<O>(v[i][0]);
      }
    }
  }
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                              const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault,
                                         &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeFn>(p);
  }();
  return fn;
}

}  // namespace sv
