// The projection's matrix product on the 5th-generation tensor cores (fp16, bf16, e4m3).
//
//     C[i][j] = sum_l A(i, l) B(j, l), fp32 accumulation in TMEM, then the fused epilogue
//
// A tile is 128 rows by BN columns; a persistent CTA per SM takes tiles blockIdx.x, + gridDim.x,
// ... in an order whose columns vary fastest, so the tiles that run together share rows of A and
// the whole of B out of L2. Operands come by TMA in stages of 128 bytes of k (64 16-bit or 128
// 8-bit elements), 128-byte swizzled:
//   K-major (rows of the operand run along k): a box is 128 bytes of k by 128 / BN rows;
//   MN-major (the gradients' operands, transposed in place): a box is 64 rows by 64 k, laid out as
//   8-k-row atoms; boxes follow each other 8 KB apart along the rows.
// Warp roles (320 threads):
//   warp 0      TMA producer;
//   warp 1      TMEM allocator (two BN-column accumulators) and the tcgen05.mma issuer;
//   warps 2-9   epilogue: two warps per 32-lane quadrant, half of the columns each, overlapped
//               with the next tile's products through the second accumulator.
// Every wait is bounded (2 s, CTA abort flag); on expiry SV_DEVICE_WAIT_TIMEOUT is reported and the
// copies and products in flight are waited for before the CTA ends.
#include <algorithm>

#include "linear.h"

namespace sv {
namespace {

constexpr int TM = 128;
constexpr int TC_THREADS = 320;
constexpr int EPI_THREADS = 256;
constexpr uint32_t ATOM = 1024;           // 8 rows of 128 bytes
constexpr uint32_t MN_STRIDE = 8 * ATOM;  // next 64 rows of an MN-major operand

template <int BN>
struct TcLayout {
  static constexpr int A_STAGE = TM * 128;
  static constexpr int B_STAGE = BN * 128;
  static constexpr int FIT = (192 * 1024) / (A_STAGE + B_STAGE);
  static constexpr int STAGES = FIT > 8 ? 8 : FIT;
  static constexpr int A_OFF = 0;
  static constexpr int B_OFF = STAGES * A_STAGE;
  static constexpr int COL_OFF = B_OFF + STAGES * B_STAGE;  // float [2 buffers][2][BN]
  static constexpr int MISC_OFF = COL_OFF + 2 * 2 * BN * 4;
  static constexpr int BAR_OFF = MISC_OFF + 16;
  static constexpr int NUM_BARS = 2 * STAGES + 5;
  static constexpr int SMEM = BAR_OFF + NUM_BARS * 8 + 1024;
  static_assert(SMEM <= 227 * 1024, "shared memory budget");
};

struct TcArgs {
  int64_t m, n;
  int32_t tiles_n, tiles;    // tiles of one split
  int32_t total;             // tiles * splits
  int32_t steps, part;       // 128-byte k steps in all, and of one split
  uint32_t idesc;
  bool e4m3, a_mn, b_mn, wide_io;
};

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ void tc_mma_f8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                          uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void epi_sync() {
  asm volatile("bar.sync 1, %0;" ::"n"(EPI_THREADS) : "memory");
}

struct Tile {
  int32_t split, m0, n0, k0, k1;  // k in 128-byte steps
};

template <int BN>
__device__ __forceinline__ Tile tile_at(const TcArgs& a, int32_t t) {
  Tile o;
  o.split = t / a.tiles;
  const int32_t r = t - o.split * a.tiles;
  const int32_t row = r / a.tiles_n;
  o.m0 = row * TM;
  o.n0 = (r - row * a.tiles_n) * BN;
  o.k0 = o.split * a.part;
  o.k1 = min(o.k0 + a.part, a.steps);
  return o;
}

// 32 consecutive columns of one row from fp32 sums to the output. `vec`: 16-byte accesses.
template <typename O>
__device__ __forceinline__ void finish_chunk(const Epilogue& ep, const float* s_bias,
                                             const float* s_scale, int64_t row, int64_t col,
                                             int64_t n, float row_scale, bool vec, bool scaled,
                                             float (&v)[32]) {
  if (scaled) {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] *= row_scale * s_scale[j];
  }
  if (ep.bias) {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] += s_bias[j];
  }
  constexpr int E = 16 / sizeof(O);
  const bool full = vec && col + 32 <= n;
  auto store = [&](void* base) {
    O* dst = static_cast<O*>(base) + row * n + col;
    if (full) {
#pragma unroll
      for (int q = 0; q < 32 / E; ++q) {
        uint4 raw;
        O* e = reinterpret_cast<O*>(&raw);
#pragma unroll
        for (int j = 0; j < E; ++j) e[j] = from_f32<O>(v[q * E + j]);
        reinterpret_cast<uint4*>(dst)[q] = raw;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (col + j < n) dst[j] = from_f32<O>(v[j]);
    }
  };
  if (ep.preact) store(ep.preact);
  if (ep.act == SV_ACT_SILU) {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = activate(v[j], SV_ACT_SILU);
  } else if (ep.act == SV_ACT_GELU) {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = activate(v[j], SV_ACT_GELU);
  } else if (ep.act == SV_ACT_GELU_TANH) {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = activate(v[j], SV_ACT_GELU_TANH);
  }
  if (ep.residual) {
    const O* src = static_cast<const O*>(ep.residual) + row * ep.ld_res + col;
    if (full) {
#pragma unroll
      for (int q = 0; q < 32 / E; ++q) {
        const uint4 raw = __ldg(reinterpret_cast<const uint4*>(src) + q);
        const O* e = reinterpret_cast<const O*>(&raw);
#pragma unroll
        for (int j = 0; j < E; ++j) v[q * E + j] += to_f32(e[j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (col + j < n) v[j] += to_f32(src[j]);
    }
  }
  store(ep.out);
}

template <int BN, typename O>
__global__ void __launch_bounds__(TC_THREADS, 1)
    gemm_tc_kernel(const __grid_constant__ CUtensorMap map_a,
                   const __grid_constant__ CUtensorMap map_b, TcArgs a, Epilogue ep,
                   int32_t* status) {
  using L = TcLayout<BN>;
  constexpr int S = L::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  float* s_cols = reinterpret_cast<float*>(smem + L::COL_OFF);
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(smem + L::MISC_OFF);
  volatile int* s_abort = reinterpret_cast<volatile int*>(smem + L::MISC_OFF + 4);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BAR_OFF);
  uint64_t* full = bars;
  uint64_t* empty = bars + S;
  uint64_t* acc_full = bars + 2 * S;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* drained = acc_empty + 2;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], EPI_THREADS);
    }
    mbar_init(drained, 1);
    *s_abort = 0;
    fence_mbar_init();
    prefetch_tmap(&map_a);
    prefetch_tmap(&map_b);
  }
  if (warp == 1) {
    tmem_alloc(s_tmem, 2 * BN);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  bool ok = true;

  if (warp == 0) {
    if (lane == 0) {
      int it = 0;
      const int per = a.e4m3 ? 128 : 64;  // elements of a k step
      for (int32_t t = blockIdx.x; t < a.total && ok; t += gridDim.x) {
        const Tile w = tile_at<BN>(a, t);
        for (int k = w.k0; k < w.k1; ++k, ++it) {
          const int slot = it % S;
          if (!mbar_wait_bounded(&empty[slot], ((it / S) & 1) ^ 1, s_abort)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&full[slot], L::A_STAGE + L::B_STAGE);
          const uint32_t sa = smem_u32(smem + L::A_OFF + slot * L::A_STAGE);
          const uint32_t sb = smem_u32(smem + L::B_OFF + slot * L::B_STAGE);
          const int kk = k * per;
          if (a.a_mn) {
#pragma unroll
            for (int r = 0; r < TM / 64; ++r)
              tma_load_2d(sa + r * MN_STRIDE, &map_a, &full[slot], w.m0 + 64 * r, kk);
          } else {
            tma_load_2d(sa, &map_a, &full[slot], kk, w.m0);
          }
          if (a.b_mn) {
#pragma unroll
            for (int r = 0; r < BN / 64; ++r)
              tma_load_2d(sb + r * MN_STRIDE, &map_b, &full[slot], w.n0 + 64 * r, kk);
          } else {
            tma_load_2d(sb, &map_b, &full[slot], kk, w.n0);
          }
        }
      }
      if (!ok) {
        report(status, SV_DEVICE_WAIT_TIMEOUT);
        // the copies in flight write this CTA's shared memory: let them land
        const uint64_t t0 = global_timer_ns();
        for (int j = max(0, it - S); j < it; ++j)
          while (!mbar_try_wait(&full[j % S], (j / S) & 1) && global_timer_ns() - t0 < 1000000000ull) {
          }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      int it = 0, local = 0;
      for (int32_t t = blockIdx.x; t < a.total && ok; t += gridDim.x, ++local) {
        const Tile w = tile_at<BN>(a, t);
        const int ab = local & 1;
        if (!mbar_wait_bounded(&acc_empty[ab], ((local >> 1) & 1) ^ 1, s_abort)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem + (uint32_t)(ab * BN);
        for (int k = w.k0; k < w.k1; ++k, ++it) {
          const int slot = it % S;
          if (!mbar_wait_bounded(&full[slot], (it / S) & 1, s_abort)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + L::A_OFF + slot * L::A_STAGE);
          const uint32_t sb = smem_u32(smem + L::B_OFF + slot * L::B_STAGE);
#pragma unroll
          for (int j = 0; j < 4; ++j) {  // 32 bytes of k: one instruction
            const uint64_t da = a.a_mn ? smem_desc_mn_sw128(sa + j * 2 * ATOM, MN_STRIDE, ATOM)
                                       : smem_desc_sw128(sa + j * 32);
            const uint64_t db = a.b_mn ? smem_desc_mn_sw128(sb + j * 2 * ATOM, MN_STRIDE, ATOM)
                                       : smem_desc_sw128(sb + j * 32);
            const uint32_t more = (k > w.k0 || j > 0) ? 1u : 0u;
            if (a.e4m3)
              tc_mma_f8(d, da, db, a.idesc, more);
            else
              tc_mma_f16(d, da, db, a.idesc, more);
          }
          tc_commit(&empty[slot]);
        }
        if (ok) tc_commit(&acc_full[ab]);
      }
      if (!ok) report(status, SV_DEVICE_WAIT_TIMEOUT);
      // the products in flight read this CTA's shared memory: let them finish
      tc_commit(drained);
      const uint64_t t0 = global_timer_ns();
      while (!mbar_try_wait(drained, 0) && global_timer_ns() - t0 < 1000000000ull) {
      }
    }
  } else {
    const int q = warp & 3;            // TMEM lanes 32 q .. 32 q + 31
    const int half = (warp - 2) >> 2;  // columns half * BN / 2 ..
    const int e = threadIdx.x - 64;
    const bool scaled = ep.row_scale != nullptr || ep.col_scale != nullptr;
    int local = 0;
    for (int32_t t = blockIdx.x; t < a.total; t += gridDim.x, ++local) {
      const Tile w = tile_at<BN>(a, t);
      const int ab = local & 1;
      float* s_bias = s_cols + ab * 2 * BN;
      float* s_scale = s_bias + BN;
      if (ep.partial == nullptr) {
        // this buffer's last readers were two tiles ago, before the previous epi_sync
        for (int c = e; c < BN; c += EPI_THREADS) {
          const bool in = w.n0 + c < a.n;
          if (ep.bias) s_bias[c] = in ? to_f32(static_cast<const O*>(ep.bias)[w.n0 + c]) : 0.f;
          if (scaled) s_scale[c] = in && ep.col_scale ? __ldg(ep.col_scale + w.n0 + c) : 1.f;
        }
        epi_sync();
      }
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(&acc_full[ab], (local >> 1) & 1, s_abort))) {
        ok = false;
        break;
      }
      tc_fence_after();
      const int64_t row = w.m0 + q * 32 + lane;
      const bool live = row < a.m;
      const float row_scale = live && ep.row_scale ? __ldg(ep.row_scale + row) : 1.f;
      const uint32_t t_row = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(ab * BN);
#pragma unroll 1
      for (int c = half * (BN / 2); c < (half + 1) * (BN / 2); c += 32) {
        uint32_t raw[32];
        __syncwarp();  // lanes past the last row skip the rest of a round
        tmem_ld_32x32b_x32(t_row + c, raw);
        tc_wait_ld();
        const int64_t col = w.n0 + c;
        if (!live || col >= a.n) continue;
        float v[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(raw[j]);
        if (ep.partial) {
          float* dst = ep.partial + ((int64_t)w.split * a.m + row) * a.n + col;
          if (a.n % 4 == 0 && col + 32 <= a.n) {
#pragma unroll
            for (int j = 0; j < 32; j += 4)
              *reinterpret_cast<float4*>(dst + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (col + j < a.n) dst[j] = v[j];
          }
        } else {
          finish_chunk<O>(ep, s_bias + c, s_scale + c, row, col, a.n, row_scale, a.wide_io, scaled,
                          v);
        }
      }
      tc_fence_before();
      mbar_arrive(&acc_empty[ab]);
    }
    if (!ok) report(status, SV_DEVICE_WAIT_TIMEOUT);
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 2 * BN);
  }
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                              const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
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

// Rows past the operand's end and k past its length are filled with zeros.
int operand_map(const Operand& o, int64_t outer, int64_t k, int dtype, int box_rows,
                CUtensorMap* map) {
  EncodeFn encode = encode_fn();
  if (encode == nullptr) SV_FAIL(SV_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
  const int es = elem_size(dtype);
  const cuuint64_t dims[2] = {(cuuint64_t)(o.mn ? outer : k), (cuuint64_t)(o.mn ? k : outer)};
  const cuuint64_t stride[1] = {(cuuint64_t)o.ld * es};
  const cuuint32_t box[2] = {(cuuint32_t)(128 / es), (cuuint32_t)(o.mn ? 64 : box_rows)};
  const cuuint32_t steps[2] = {1, 1};
  const CUtensorMapDataType type = dtype == SV_FLOAT8_E4M3 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                   : dtype == SV_BFLOAT16  ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                           : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  if (encode(map, type, 2, const_cast<void*>(o.p), dims, stride, box, steps,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    SV_FAIL(SV_ERR_CUDA, "cuTensorMapEncodeTiled failed for an operand of the projection");
  return SV_OK;
}

template <int BN, typename O>
int launch_tc(const Gemm& g, int32_t* status, cudaStream_t s) {
  using L = TcLayout<BN>;
  int dev = 0;
  SV_CUDA_TRY(cudaGetDevice(&dev));
  static bool attr_done[256] = {};
  if (dev >= 256 || !attr_done[dev]) {
    SV_CUDA_TRY(cudaFuncSetAttribute(gemm_tc_kernel<BN, O>,
                                     cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM));
    if (dev < 256) attr_done[dev] = true;
  }
  CUtensorMap map_a, map_b;
  int rc = operand_map(g.a, g.m, g.k, g.dtype, TM, &map_a);
  if (rc == SV_OK) rc = operand_map(g.b, g.n, g.k, g.dtype, BN, &map_b);
  if (rc != SV_OK) return rc;
  TcArgs a{};
  a.m = g.m;
  a.n = g.n;
  a.tiles_n = (int32_t)((g.n + BN - 1) / BN);
  const int64_t tiles = (g.m + TM - 1) / TM * a.tiles_n;
  if (tiles * g.splits > INT32_MAX / 2) SV_FAIL(SV_ERR_UNSUPPORTED, "linear: too many tiles");
  a.tiles = (int32_t)tiles;
  a.total = (int32_t)(tiles * g.splits);
  const int per = 128 / elem_size(g.dtype);
  a.steps = (int32_t)((g.k + per - 1) / per);
  a.part = (a.steps + g.splits - 1) / g.splits;
  a.e4m3 = g.dtype == SV_FLOAT8_E4M3;
  a.a_mn = g.a.mn;
  a.b_mn = g.b.mn;
  a.idesc = a.e4m3 ? idesc_f16(false, TM, BN)  // the same fields; format 0 is e4m3
                   : idesc_f16_major(g.dtype == SV_BFLOAT16, TM, BN, g.a.mn, g.b.mn);
  const Epilogue& ep = g.ep;
  const int e = 16 / elem_size(ep.out_dtype);
  a.wide_io = g.n % e == 0 && aligned16(ep.out) && (!ep.preact || aligned16(ep.preact)) &&
              (!ep.residual || (aligned16(ep.residual) && ep.ld_res % e == 0));
  const int grid = (int)std::min<int64_t>(a.total, num_sms());
  gemm_tc_kernel<BN, O><<<grid, TC_THREADS, L::SMEM, s>>>(map_a, map_b, a, ep, status);
  SV_LAUNCH_CHECK();
  return SV_OK;
}

template <typename O>
int launch_typed(const Gemm& g, int bn, int32_t* status, cudaStream_t s) {
  if (bn == 256) return launch_tc<256, O>(g, status, s);
  if (bn == 128) return launch_tc<128, O>(g, status, s);
  return launch_tc<64, O>(g, status, s);
}

}  // namespace

int gemm_tc(const Gemm& g, int bn, int32_t* status, cudaStream_t s) {
  return g.ep.out_dtype == SV_FLOAT16 ? launch_typed<__half>(g, bn, status, s)
                                      : launch_typed<__nv_bfloat16>(g, bn, status, s);
}

}  // namespace sv
