// The projection's matrix product on the 5th-generation tensor cores (fp16, bf16, e4m3).
//
//     C[i][j] = sum_l A(i, l) B(j, l), fp32 accumulation in TMEM, then the fused epilogue
//
// PAIR: two CTAs of a cluster form one 256-row tile (cta_group::2): each holds 128 rows of A, half of
// the tile's rows of B and its own 128 rows of the sums, so a row of B crosses L2 once per 256 rows
// of the result. Otherwise a CTA forms a 128-row tile by itself, for products too small to give every
// pair a tile. What bounds single tiles is that traffic: 128 x 256 ones ran at 10.6 TB/s out of L2 with
// the tensor pipe 56% busy. 40,662 x 1024 -> 4096 bf16 with bias and GELU: 367 us so, 288 us in pairs
// (1,184 TFLOP/s); 40,662 x 4096 -> 1024 e4m3 with scales and residual: 140 us (2,440 TFLOP/s);
// 12,001 x 1024 x 1024 bf16: 32.5 us (775 TFLOP/s: three rounds of tiles, the last one half full).
// Columns that are not a multiple of 8 are written in 2-byte pieces: 20,000 x 1024 -> 1001 takes 70 us,
// -> 1024 takes 44.
//
// A persistent unit (CTA or pair) takes tiles unit, + units, ... in an order whose columns vary
// fastest, so the tiles that run together share rows of A and the whole of B out of L2. Operands
// come by TMA in stages of 128 bytes of k (64 16-bit or 128 8-bit elements), 128-byte swizzled:
//   K-major (rows of the operand run along k): a box is 128 bytes of k by the CTA's rows;
//   MN-major (the gradients' operands, transposed in place): a box is 64 rows by 64 k, laid out as
//   8-k-row atoms; boxes follow each other 8 KB apart along the rows.
// Warp roles (320 threads):
//   warp 0      TMA producer, each CTA for its own rows; the bytes of both count on the first
//               CTA's barrier;
//   warp 1      TMEM allocator (two BN-column accumulators) and, in the first CTA, the tcgen05.mma
//               issuer, whose commits free the stages of both CTAs;
//   warps 2-9   epilogue: two warps per 32-lane quadrant, half of the columns each, overlapped
//               with the next tile's products through the second accumulator. Sums go through
//               shared memory, 32 x 32 at a time, so that bias, residual and results are read and
//               written in whole row segments.
// Every wait on an mbarrier is bounded (2 s, CTA abort flag); on expiry SV_DEVICE_WAIT_TIMEOUT is
// reported and the copies and products in flight are waited for before the CTA ends. An epilogue warp
// that has given up still walks its remaining tiles, without waiting, reading sums or storing: the warps
// decide one by one, and the others' named barrier counts it.
#include <algorithm>

#include "linear.h"

namespace sv {
namespace {

constexpr int TM = 128;  // rows of a CTA's tile
constexpr int TC_THREADS = 320;
constexpr int EPI_THREADS = 256;
constexpr int EPI_WARPS = EPI_THREADS / 32;
constexpr uint32_t ATOM = 1024;           // 8 rows of 128 bytes
constexpr uint32_t MN_STRIDE = 8 * ATOM;  // next 64 rows of an MN-major operand
constexpr int CHUNK_LD = 36;  // floats between staged rows: 16-byte rows in different banks

template <int BN, bool PAIR>
struct TcLayout {
  static constexpr int B_ROWS = PAIR ? BN / 2 : BN;  // of one CTA
  static constexpr int A_STAGE = TM * 128;
  static constexpr int B_STAGE = B_ROWS * 128;
  static constexpr int FIT = (176 * 1024) / (A_STAGE + B_STAGE);
  static constexpr int STAGES = FIT > 7 ? 7 : FIT;
  static constexpr int A_OFF = 0;
  static constexpr int B_OFF = STAGES * A_STAGE;
  static constexpr int CHUNK_OFF = B_OFF + STAGES * B_STAGE;  // float [8 warps][32][CHUNK_LD]
  static constexpr int COL_OFF = CHUNK_OFF + EPI_WARPS * 32 * CHUNK_LD * 4;  // [2][bias, scale][BN]
  static constexpr int MISC_OFF = COL_OFF + 2 * 2 * BN * 4;
  static constexpr int BAR_OFF = MISC_OFF + 16;
  static constexpr int NUM_BARS = 2 * STAGES + 5;
  static constexpr int SMEM = BAR_OFF + NUM_BARS * 8 + 1024;
  static_assert(SMEM <= 227 * 1024, "shared memory budget");
  static_assert(STAGES >= 4, "pipeline depth");
};

struct TcArgs {
  int64_t m, n;
  int32_t tiles_n, tiles;    // tiles of one split
  int32_t total;             // tiles * splits
  int32_t units;             // CTAs, or pairs
  int32_t steps, part;       // 128-byte k steps in all, and of one split
  uint32_t idesc;
  bool e4m3, a_mn, b_mn, wide_io;
};

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

struct Tile {
  int32_t split, m0, n0, k0, k1;  // k in 128-byte steps; m0 of the whole tile
};

template <int BN, bool PAIR>
__device__ __forceinline__ Tile tile_at(const TcArgs& a, int32_t t) {
  Tile o;
  o.split = t / a.tiles;
  const int32_t r = t - o.split * a.tiles;
  const int32_t row = r / a.tiles_n;
  o.m0 = row * (PAIR ? 2 * TM : TM);
  o.n0 = (r - row * a.tiles_n) * BN;
  o.k0 = o.split * a.part;
  o.k1 = min(o.k0 + a.part, a.steps);
  return o;
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

template <int BN, bool PAIR, typename O, bool F8>
__global__ void __launch_bounds__(TC_THREADS, 1)
    gemm_tc_kernel(const __grid_constant__ CUtensorMap map_a,
                   const __grid_constant__ CUtensorMap map_b, TcArgs a, Epilogue ep,
                   int32_t* status) {
  using L = TcLayout<BN, PAIR>;
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
  const uint32_t rank = PAIR ? cluster_rank() : 0u;
  const int32_t unit = PAIR ? blockIdx.x >> 1 : blockIdx.x;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], (PAIR ? 2 : 1) * EPI_WARPS);
    }
    mbar_init(drained, 1);
    *s_abort = 0;
    fence_mbar_init();
    prefetch_tmap(&map_a);
    prefetch_tmap(&map_b);
  }
  if (warp == 1) alloc_tmem<PAIR>(s_tmem, 2 * BN);
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync();  // the other CTA's barriers are ready too
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  bool ok = true;

  if (warp == 0) {
    if (lane == 0) {
      int it = 0;
      constexpr int per = F8 ? 128 : 64;  // elements of a k step
      for (int32_t t = unit; t < a.total && ok; t += a.units) {
        const Tile w = tile_at<BN, PAIR>(a, t);
        const int32_t m0 = w.m0 + (int32_t)rank * TM, n0 = w.n0 + (int32_t)rank * L::B_ROWS;
        for (int k = w.k0; k < w.k1; ++k, ++it) {
          const int slot = it % S;
          if (!mbar_wait_bounded(&empty[slot], ((it / S) & 1) ^ 1, s_abort)) {
            ok = false;
            break;
          }
          if (rank == 0)
            mbar_arrive_expect_tx(&full[slot], (PAIR ? 2 : 1) * (L::A_STAGE + L::B_STAGE));
          const uint32_t sa = smem_u32(smem + L::A_OFF + slot * L::A_STAGE);
          const uint32_t sb = smem_u32(smem + L::B_OFF + slot * L::B_STAGE);
          const int kk = k * per;
          const uint32_t bar = PAIR ? in_first(smem_u32(&full[slot])) : 0u;
          auto load = [&](uint32_t dst, const CUtensorMap* map, int x, int y) {
            if constexpr (PAIR) tma_load_pair(dst, map, bar, x, y);
            else tma_load_2d(dst, map, &full[slot], x, y);
          };
          if (!F8 && a.a_mn) {
#pragma unroll
            for (int r = 0; r < TM / 64; ++r) load(sa + r * MN_STRIDE, &map_a, m0 + 64 * r, kk);
          } else {
            load(sa, &map_a, kk, m0);
          }
          if (!F8 && a.b_mn) {
#pragma unroll
            for (int r = 0; r < L::B_ROWS / 64; ++r)
              load(sb + r * MN_STRIDE, &map_b, n0 + 64 * r, kk);
          } else {
            load(sb, &map_b, kk, n0);
          }
        }
      }
      if (!ok) {
        report(status, SV_DEVICE_WAIT_TIMEOUT);
        // the copies in flight write this CTA's shared memory: let them land
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 10000000ull) {
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      int it = 0, local = 0;
      for (int32_t t = unit; t < a.total && ok; t += a.units, ++local) {
        const Tile w = tile_at<BN, PAIR>(a, t);
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
            const uint64_t da = !F8 && a.a_mn
                                    ? smem_desc_mn_sw128(sa + j * 2 * ATOM, MN_STRIDE, ATOM)
                                    : smem_desc_sw128(sa + j * 32);
            const uint64_t db = !F8 && a.b_mn
                                    ? smem_desc_mn_sw128(sb + j * 2 * ATOM, MN_STRIDE, ATOM)
                                    : smem_desc_sw128(sb + j * 32);
            issue_mma<PAIR, F8>(d, da, db, a.idesc, (k > w.k0 || j > 0) ? 1u : 0u);
          }
          commit<PAIR>(&empty[slot]);
        }
        if (ok) commit<PAIR>(&acc_full[ab]);
      }
      if (!ok) report(status, SV_DEVICE_WAIT_TIMEOUT);
      // the products in flight read both CTAs' shared memory: let them finish
      commit<PAIR>(drained);
      const uint64_t t0 = global_timer_ns();
      while (!mbar_try_wait(drained, 0) && global_timer_ns() - t0 < 1000000000ull) {
      }
    }
  } else {
    const int q = warp & 3;            // TMEM lanes 32 q .. 32 q + 31
    const int half = (warp - 2) >> 2;  // columns half * BN / 2 ..
    const int e = threadIdx.x - 64;
    float* chunk = reinterpret_cast<float*>(smem + L::CHUNK_OFF) + (warp - 2) * 32 * CHUNK_LD;
    const bool scaled = ep.row_scale != nullptr || ep.col_scale != nullptr;
    int local = 0;
    for (int32_t t = unit; t < a.total; t += a.units, ++local) {  // left by all warps alike
      const Tile w = tile_at<BN, PAIR>(a, t);
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
      if (!ok) continue;
      const int64_t row0 = (int64_t)w.m0 + rank * TM + q * 32;  // the warp's first row
      const int rows = (int)max((int64_t)0, min((int64_t)32, a.m - row0));
      if (ep.residual && lane < rows) {
        // into L2 while the products run
        const O* src = static_cast<const O*>(ep.residual) + (row0 + lane) * ep.ld_res;
        for (int64_t c = (int64_t)w.n0 + half * (BN / 2), end = min(c + BN / 2, a.n); c < end; c += 64)
          asm volatile("prefetch.global.L2 [%0];" ::"l"(src + c));
      }
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(&acc_full[ab], (local >> 1) & 1, s_abort))) {
        ok = false;
        continue;
      }
      tc_fence_after();
      const uint32_t t_row = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(ab * BN);
#pragma unroll 1
      for (int c = half * (BN / 2); c < (half + 1) * (BN / 2); c += 32) {
        uint32_t raw[32];
        tmem_ld_32x32b_x32(t_row + c, raw);
        tc_wait_ld();
        const int64_t col = (int64_t)w.n0 + c;
        if (rows == 0 || col >= a.n) continue;  // the same in all lanes
        __syncwarp();                           // the previous chunk has been read
#pragma unroll
        for (int j = 0; j < 32; j += 4)
          *reinterpret_cast<uint4*>(chunk + lane * CHUNK_LD + j) =
              make_uint4(raw[j], raw[j + 1], raw[j + 2], raw[j + 3]);
        __syncwarp();
        const int cols = (int)min((int64_t)32, a.n - col);
        if (ep.partial) {
          float* dst = ep.partial + ((int64_t)w.split * a.m + row0) * a.n + col;
          if (a.n % 4 == 0 && cols == 32) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int r = i * 4 + (lane >> 3), j = (lane & 7) * 4;
              if (r < rows)
                *reinterpret_cast<float4*>(dst + r * a.n + j) =
                    *reinterpret_cast<const float4*>(chunk + r * CHUNK_LD + j);
            }
          } else if (lane < cols) {
            for (int r = 0; r < rows; ++r) dst[r * a.n + lane] = chunk[r * CHUNK_LD + lane];
          }
        } else if (a.wide_io && cols == 32) {
          const int j = (lane & 3) * 8;  // four lanes a row, eight rows at a time
          float bias[8], scale[8];
#pragma unroll
          for (int x = 0; x < 8; x += 4) {
            if (ep.bias)
              *reinterpret_cast<float4*>(bias + x) =
                  *reinterpret_cast<const float4*>(s_bias + c + j + x);
            if (scaled)
              *reinterpret_cast<float4*>(scale + x) =
                  *reinterpret_cast<const float4*>(s_scale + c + j + x);
          }
          float v[4][8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float* src = chunk + (i * 8 + (lane >> 2)) * CHUNK_LD + j;
            *reinterpret_cast<float4*>(v[i]) = *reinterpret_cast<const float4*>(src);
            *reinterpret_cast<float4*>(v[i] + 4) = *reinterpret_cast<const float4*>(src + 4);
          }
          finish<O, 4, 8>(ep, v, bias, scale, scaled, row0 + (lane >> 2), 8, rows - (lane >> 2),
                          a.n, col + j);
        } else if (lane < cols) {
          const float bias[1] = {ep.bias ? s_bias[c + lane] : 0.f};
          const float scale[1] = {scaled ? s_scale[c + lane] : 1.f};
#pragma unroll 1
          for (int r = 0; r < rows; r += 16) {
            float v[16][1];
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i][0] = chunk[(r + i) * CHUNK_LD + lane];
            finish<O, 16, 1>(ep, v, bias, scale, scaled, row0 + r, 1, rows - r, a.n, col + lane);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (PAIR) arrive_at(in_first(smem_u32(&acc_empty[ab])));
        else arrive_at(smem_u32(&acc_empty[ab]));
      }
    }
    if (!ok) report(status, SV_DEVICE_WAIT_TIMEOUT);
  }

  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync();  // nothing of the pair still reads or signals this CTA
  if (warp == 1) {
    tc_fence_after();
    free_tmem<PAIR>(tmem, 2 * BN);
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

template <int BN, bool PAIR, typename O, bool F8>
int launch_tc(const Gemm& g, int32_t* status, cudaStream_t s) {
  using L = TcLayout<BN, PAIR>;
  auto kernel = gemm_tc_kernel<BN, PAIR, O, F8>;
  int dev = 0;
  SV_CUDA_TRY(cudaGetDevice(&dev));
  cudaLaunchConfig_t config{};
  config.blockDim = dim3(TC_THREADS);
  config.dynamicSmemBytes = L::SMEM;
  config.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = PAIR ? 2 : 1;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  config.attrs = &attr;
  config.numAttrs = 1;
  // Units that run at the same time: one more would run after all the others.
  static int units_of[256] = {};
  int units = dev < 256 ? units_of[dev] : 0;
  if (units == 0) {
    SV_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     L::SMEM));
    units = num_sms();
    if constexpr (PAIR) {
      config.gridDim = dim3(num_sms() / 2 * 2);
      SV_CUDA_TRY(cudaOccupancyMaxActiveClusters(&units, kernel, &config));
      if (units < 1) SV_FAIL(SV_ERR_CUDA, "linear: no CTA pair fits this device");
      units = std::min(units, num_sms() / 2);
    }
    if (dev < 256) units_of[dev] = units;
  }
  CUtensorMap map_a, map_b;
  int rc = operand_map(g.a, g.m, g.k, g.dtype, TM, &map_a);
  if (rc == SV_OK) rc = operand_map(g.b, g.n, g.k, g.dtype, L::B_ROWS, &map_b);
  if (rc != SV_OK) return rc;
  constexpr int ROWS = PAIR ? 2 * TM : TM;
  TcArgs a{};
  a.m = g.m;
  a.n = g.n;
  a.tiles_n = (int32_t)((g.n + BN - 1) / BN);
  const int64_t tiles = (g.m + ROWS - 1) / ROWS * a.tiles_n;
  if (tiles * g.splits > INT32_MAX / 2) SV_FAIL(SV_ERR_UNSUPPORTED, "linear: too many tiles");
  a.tiles = (int32_t)tiles;
  a.total = (int32_t)(tiles * g.splits);
  a.units = std::min(a.total, units);
  const int per = 128 / elem_size(g.dtype);
  a.steps = (int32_t)((g.k + per - 1) / per);
  a.part = (a.steps + g.splits - 1) / g.splits;
  a.a_mn = g.a.mn;
  a.b_mn = g.b.mn;
  a.idesc = F8 ? idesc_f16(false, ROWS, BN)  // the same fields; format 0 is e4m3
               : idesc_f16_major(g.dtype == SV_BFLOAT16, ROWS, BN, g.a.mn, g.b.mn);
  const Epilogue& ep = g.ep;
  a.wide_io = g.n % 8 == 0 && aligned16(ep.out) && (!ep.preact || aligned16(ep.preact)) &&
              (!ep.residual || (aligned16(ep.residual) && ep.ld_res % 8 == 0));
  config.gridDim = dim3((unsigned)(a.units * (PAIR ? 2 : 1)));
  SV_CUDA_TRY(cudaLaunchKernelEx(&config, kernel, map_a, map_b, a, ep, status));
  return SV_OK;
}

template <typename O, bool F8>
int launch_typed(const Gemm& g, TcTile tile, int32_t* status, cudaStream_t s) {
  switch (tile) {
    case TcTile::kPair256: return launch_tc<256, true, O, F8>(g, status, s);
    case TcTile::kPair128: return launch_tc<128, true, O, F8>(g, status, s);
    case TcTile::kOne128: return launch_tc<128, false, O, F8>(g, status, s);
    default: return launch_tc<64, false, O, F8>(g, status, s);
  }
}

}  // namespace

int gemm_tc(const Gemm& g, TcTile tile, int32_t* status, cudaStream_t s) {
  const bool half = g.ep.out_dtype == SV_FLOAT16;
  if (g.dtype == SV_FLOAT8_E4M3)
    return half ? launch_typed<__half, true>(g, tile, status, s)
                : launch_typed<__nv_bfloat16, true>(g, tile, status, s);
  return half ? launch_typed<__half, false>(g, tile, status, s)
              : launch_typed<__nv_bfloat16, false>(g, tile, status, s);
}

}  // namespace sv
