// The products grouped by expert on the 5th-generation tensor cores (fp16, bf16).
//
// The tiles, stages and warp roles are those of linear_tc.cu: persistent CTAs, or pairs of them
// (cta_group::2) on tiles of 256 rows, operands by TMA into 128-byte swizzled stages, one issuing
// thread, two accumulators in TMEM, and epilogue warps that work on one tile while the next is
// formed. What differs is where the tiles are:
//
//   kRows      Every expert's positions are cut into tiles of their own, so that a tile has one weight.
//              The CTAs count the tiles of all experts on the device (a scan over the offsets in
//              shared memory) and look a tile's expert up by bisection. A tile's last rows may be the
//              next expert's: they are formed and not stored. Weights are read through a
//              three-dimensional map, so that what lies past an expert's matrix is zeros and not
//              its neighbour.
//   kWeights   The sum runs over an expert's positions, from any first row to any last. The steps of 64
//              positions start at the first; the rows past the last one have to be zeros in both
//              operands (0 times a neighbour's infinity is not 0), which a TMA load gives past the end of
//              its map: every expert has a copy of the two maps whose extent ends with its last
//              position, written by expert_maps_kernel.
//
// 81,324 positions of 8 experts, 1024 -> 4096 bf16 with bias and GELU: 525 us (1,300 TFLOP/s), 482 without
// an activation (the library's product of that size without groups: 478). What bounds it is the epilogue:
// a tile's products are 8,200 cycles of a pair, GELU's special functions alone 4,100 of a CTA. 24,002
// positions of 16 experts, 2048 -> 1024: 93 us forward (113 where the sum over k is made of runs, see
// run_steps), 86 dx, 98 dW (1,080, 890, 1,170 and 1,030 TFLOP/s; 5.5 rounds of tiles, of which an expert's last
// is half empty).
//
// Every wait on an mbarrier is bounded, and unwinds as in linear_tc.cu.
#include <algorithm>
#include <type_traits>

#include "expert.h"
#include "gemm_tc.cuh"
#include "group.h"

namespace sv {
namespace {

constexpr int EX_MAX = 1024;  // experts
// Eight epilogue warps: sixteen have 96 registers each, and took 868,000 cycles where eight take 714,000
// (81,324 x 1024 x 4096 without an activation).
constexpr int EX_EPI_WARPS = 8;
constexpr int EX_EPI_THREADS = 32 * EX_EPI_WARPS;
constexpr int EX_THREADS = 64 + EX_EPI_THREADS;

__device__ __forceinline__ void ex_epi_sync() {
  asm volatile("bar.sync 1, %0;" ::"n"(EX_EPI_THREADS) : "memory");
}

template <int BN, bool PAIR>
struct ExLayout {
  static constexpr int B_ROWS = PAIR ? BN / 2 : BN;  // of one CTA
  static constexpr int A_STAGE = TM * 128;
  static constexpr int B_STAGE = B_ROWS * 128;
  static constexpr int FIT = (160 * 1024) / (A_STAGE + B_STAGE);
  static constexpr int STAGES = FIT > 7 ? 7 : FIT;
  static constexpr int A_OFF = 0;
  static constexpr int B_OFF = STAGES * A_STAGE;
  static constexpr int CHUNK_OFF = B_OFF + STAGES * B_STAGE;  // float [warps][32][CHUNK_LD]
  static constexpr int COL_OFF = CHUNK_OFF + EX_EPI_WARPS * 32 * CHUNK_LD * 4;  // [2][bias, scale][BN]
  static constexpr int FIRST_OFF = COL_OFF + 2 * 2 * BN * 4;  // int [experts + 1]
  static constexpr int SEG_OFF = FIRST_OFF + (EX_MAX + 4) * 4;  // int2 [experts]
  static constexpr int MISC_OFF = SEG_OFF + EX_MAX * 8;
  static constexpr int BAR_OFF = MISC_OFF + 16;
  static constexpr int NUM_BARS = 2 * STAGES + 5;
  static constexpr int SMEM = BAR_OFF + NUM_BARS * 8 + 1024;
  static_assert(SMEM <= 227 * 1024, "shared memory budget");
  static_assert(STAGES >= 4, "pipeline depth");
};

// True in one lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one != 0;
}

// The tensor cores cut off what lies below a sum's last place at every addition, so that a sum's error grows with
// k and has one sign: 2.1e-6 of the result at k 2048, where an fp32 sum is 3.9e-7 off. 16 bits do not
// show it, but what is formed from results held in fp32 does (the gradients of the routing's weights: 1.9e-6
// off, and 4.4e-7 so). For them the tensor cores add up runs of a few steps of 64, and the epilogue warps add
// the runs up in fp32: of 4 steps up to k 512 (2.3e-7, where an fp32 sum is 1.6e-7 off), else of up to 8
// (4.7e-7; the fp32 sum 2.5e-7 at k 1024). An epilogue warp takes 1,200 cycles for a run beside its stores:
// 24,002 x 2048 -> 1024 takes 95 us in one sum, 113 in runs of 8 and took 16 more in runs of 4.
inline int run_steps(int64_t steps) { return steps <= 8 ? 4 : 8; }

struct ExArgs {
  const int32_t* offsets;
  int32_t experts, slots;
  int64_t m, n;            // m: kWeights
  int32_t tiles_m, tiles_n;  // tiles_m: kWeights
  int32_t steps;           // kRows
  int32_t run, runs;       // not kOne: steps of a run, and runs of a tile
  uint32_t idesc;
  bool b_mn, wide_io, zero_rest;
  bool direct;             // the result's rows are multiples of 16 columns on 32-byte boundaries
  const CUtensorMap* maps;  // kWeights: [experts][2]
};

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const void* tmap, uint64_t* bar, int32_t x,
                                            int32_t y, int32_t z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(tmap), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const void* tmap, uint32_t bar,
                                                 int32_t x, int32_t y, int32_t z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(tmap), "r"(bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}

struct ExTile {
  int32_t e, row, last, n0, k1;  // row: first position (kRows), or row of the expert's result
  int32_t base;                  // kWeights: the expert's first position
};

template <int BN, bool PAIR, bool WEIGHTS>
__device__ __forceinline__ ExTile ex_tile(const ExArgs& a, const int32_t* first, const int2* seg,
                                          int32_t t) {
  constexpr int ROWS = PAIR ? 2 * TM : TM;
  ExTile o;
  const int32_t piece = t / a.tiles_n;
  o.n0 = (t - piece * a.tiles_n) * BN;
  if constexpr (WEIGHTS) {
    o.e = piece / a.tiles_m;
    o.row = (piece - o.e * a.tiles_m) * ROWS;
    o.last = (int32_t)a.m;
    const int2 s = seg[o.e];
    o.base = s.x;
    o.k1 = (s.y - s.x + 63) / 64;
  } else {
    int lo = 0, hi = a.experts;  // first[lo] <= piece < first[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (first[mid] <= piece) lo = mid;
      else hi = mid;
    }
    const int2 s = seg[lo];
    o.e = lo;
    o.row = s.x + (piece - first[lo]) * ROWS;
    o.last = s.y;
    o.base = 0;
    o.k1 = a.steps;
  }
  return o;
}

// The epilogue of R rows of W consecutive columns that came through shared memory: scale, bias, argument
// kept, activation, and results in O or, WIDE, in fp32.
template <typename O, bool WIDE, int R, int W>
__device__ __forceinline__ void ex_finish(const Epilogue& ep, float (&v)[R][W], const float* bias,
                                          const float* scale, int64_t row, int step, int rows,
                                          int64_t n, int64_t col) {
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < W; ++j) {
      if (ep.col_scale) v[i][j] *= scale[j];
      if (ep.bias) v[i][j] += bias[j];
    }
  auto store = [&](auto* to) {
    using S = std::remove_pointer_t<decltype(to)>;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (i * step >= rows) continue;
      S* dst = to + (row + i * step) * n + col;
      alignas(16) S e[W];
#pragma unroll
      for (int j = 0; j < W; ++j) e[j] = from_f32<S>(v[i][j]);
      if constexpr (W == 8) {
#pragma unroll
        for (int j = 0; j < (int)sizeof(e) / 16; ++j)
          reinterpret_cast<uint4*>(dst)[j] = reinterpret_cast<const uint4*>(e)[j];
      } else {
        *dst = e[0];
      }
    }
  };
  if (ep.preact) store(ep.preact);
  if (ep.act == SV_ACT_SILU) activate_all<SV_ACT_SILU>(v);
  else if (ep.act == SV_ACT_GELU) activate_all<SV_ACT_GELU>(v);
  else if (ep.act == SV_ACT_GELU_TANH) activate_all<SV_ACT_GELU_TANH>(v);
  if constexpr (WIDE) store(static_cast<float*>(ep.out));
  else store(static_cast<O*>(ep.out));
}

// 32 bytes to global memory in one access: a whole sector by one lane.
__device__ __forceinline__ void store_sector(void* p, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]),
               "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// Adds COLS columns from TMEM to a lane's sums.
template <int COLS>
__device__ __forceinline__ void ex_add(float (&sum)[COLS], uint32_t t_row) {
#pragma unroll
  for (int i = 0; i < COLS; i += 16) {
    uint32_t raw[16];
    tmem_ld_32x32b_x16(t_row + i, raw);
    tc_wait_ld();
#pragma unroll
    for (int j = 0; j < 16; ++j) sum[i + j] += __uint_as_float(raw[j]);
  }
}

// Sums that were added up in registers, without an activation: scaled, and to whole sectors of the lane's
// row `to`, the columns from c0 on that are below c1. Arguments as ex_direct's.
template <int COLS>
__device__ __forceinline__ void ex_sums(const float (&sum)[COLS], int c0, int c1, const float* bias,
                                        const float* scale, bool in, float* to) {
#pragma unroll
  for (int i = 0; i < COLS; i += 8) {
    const int c = c0 + i;
    if (c >= c1) continue;
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; j += 4) {
      const float4 m = *reinterpret_cast<const float4*>(scale + c + j);
      const float4 s = *reinterpret_cast<const float4*>(bias + c + j);
      w[j] = __float_as_uint(fmaf(sum[i + j], m.x, s.x));
      w[j + 1] = __float_as_uint(fmaf(sum[i + j + 1], m.y, s.y));
      w[j + 2] = __float_as_uint(fmaf(sum[i + j + 2], m.z, s.z));
      w[j + 3] = __float_as_uint(fmaf(sum[i + j + 3], m.w, s.w));
    }
    if (in) store_sector(to + c, w);
  }
}

// Columns [at, at + 32) of a lane's sums into its row of the warp's staging.
template <int COLS>
__device__ __forceinline__ void ex_stage(const float (&sum)[COLS], int at, float* row) {
#pragma unroll
  for (int i = 0; i < COLS; i += 32) {
    if (i != at) continue;  // registers have no index
#pragma unroll
    for (int j = 0; j < 32; j += 4)
      *reinterpret_cast<float4*>(row + j) =
          make_float4(sum[i + j], sum[i + j + 1], sum[i + j + 2], sum[i + j + 3]);
  }
}

// A warp's columns [c0, c1) of a tile, a row a lane, straight from TMEM to whole sectors of global memory: no
// turn through shared memory, half of the instructions an element. `bias`, `scale`: in shared memory, the
// same address in all lanes, 0 and 1 where there are none: a multiply-add an element and no branch, which
// between 4 elements each cost more than the elements (12 cycles an element of the tile's 256 a scheduler).
// `to`, `kept`: the lane's row at column 0 of the tile; formed: the sums are there, else they are zeros.
template <typename O, bool WIDE, int ACT>
__device__ __forceinline__ void ex_direct(uint32_t t_row, int c0, int c1, const float* bias,
                                          const float* scale, bool formed, bool in, void* to,
                                          float* kept) {
#pragma unroll 1
  for (int c = c0; c < c1; c += 16) {
    uint32_t raw[16];
    tmem_ld_32x32b_x16(t_row + c, raw);
    float v[1][16];
    float4 m[4], s[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      m[j] = *reinterpret_cast<const float4*>(scale + c + 4 * j);
      s[j] = *reinterpret_cast<const float4*>(bias + c + 4 * j);
    }
    tc_wait_ld();
#pragma unroll
    for (int j = 0; j < 16; ++j) v[0][j] = formed ? __uint_as_float(raw[j]) : 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[0][4 * j] = fmaf(v[0][4 * j], m[j].x, s[j].x);
      v[0][4 * j + 1] = fmaf(v[0][4 * j + 1], m[j].y, s[j].y);
      v[0][4 * j + 2] = fmaf(v[0][4 * j + 2], m[j].z, s[j].z);
      v[0][4 * j + 3] = fmaf(v[0][4 * j + 3], m[j].w, s[j].w);
    }
    auto store32 = [&](float* at) {
#pragma unroll
      for (int j = 0; j < 16; j += 8) {
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(v[0][j + i]);
        if (in) store_sector(at + j, w);
      }
    };
    if (kept) store32(kept + c);
    activate_all<ACT>(v);
    if constexpr (WIDE) {
      store32(static_cast<float*>(to) + c);
    } else {
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = pack_two<O>(v[0][2 * i], v[0][2 * i + 1]);
      if (in) store_sector(static_cast<O*>(to) + c, w);
    }
  }
}

// Adds the sums of a tile's runs but the last one up, a row a lane and COLS columns from t_row on, and gives
// their accumulators back. False: a wait has run out.
template <int COLS, int BN, typename Give>
__device__ __forceinline__ bool ex_collect(float (&sum)[COLS], uint32_t t_row, int runs, int& local,
                                           uint64_t* acc_full, volatile int* abort_flag, Give&& give) {
#pragma unroll
  for (int i = 0; i < COLS; ++i) sum[i] = 0.f;
  for (int r = 1; r < runs; ++r, ++local) {
    const int ab = local & 1;
    if (!__all_sync(0xffffffffu, mbar_wait_bounded(&acc_full[ab], (local >> 1) & 1, abort_flag)))
      return false;
    tc_fence_after();
    ex_add<COLS>(sum, t_row + (uint32_t)(ab * BN));
    give(ab);
  }
  return true;
}

// What a sum over k is made of, and where its result goes from.
enum class Sums {
  kOne,     // one sum in TMEM
  kRuns,    // kRows in fp32: runs, added up in registers and stored from there in whole sectors, without an
            // activation
  kStaged,  // kRows in fp32: runs, with an activation or other columns: through shared memory (its registers
            // spill: 580 bytes a thread, where kRuns spills 78)
};

template <int BN, bool PAIR, typename O, bool WEIGHTS, bool WIDE, Sums SUMS>
__global__ void __launch_bounds__(EX_THREADS, 1)
    expert_tc_kernel(const __grid_constant__ CUtensorMap map_a,
                     const __grid_constant__ CUtensorMap map_b, ExArgs a, Epilogue ep,
                     int32_t* status) {
  using L = ExLayout<BN, PAIR>;
  constexpr int S = L::STAGES;
  constexpr int ROWS = PAIR ? 2 * TM : TM;
  constexpr bool RUNS = SUMS != Sums::kOne;
  static_assert(!RUNS || (WIDE && !WEIGHTS), "results in fp32");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  float* s_cols = reinterpret_cast<float*>(smem + L::COL_OFF);
  int32_t* s_first = reinterpret_cast<int32_t*>(smem + L::FIRST_OFF);
  int2* s_seg = reinterpret_cast<int2*>(smem + L::SEG_OFF);
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
  const int32_t units = PAIR ? gridDim.x >> 1 : gridDim.x;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], (PAIR ? 2 : 1) * EX_EPI_WARPS);
    }
    mbar_init(drained, 1);
    *s_abort = 0;
    fence_mbar_init();
    if constexpr (!WEIGHTS) {
      prefetch_tmap(&map_a);
      prefetch_tmap(&map_b);
    }
  }
  if (warp == 1) alloc_tmem<PAIR>(s_tmem, 2 * BN);
  for (int e = threadIdx.x; e < a.experts; e += EX_THREADS) {
    s_seg[e] = make_int2(inside(a.offsets, e, a.slots), inside(a.offsets, e + 1, a.slots));
  }
  __syncthreads();
  if (warp == 2) {  // segments that do not overlap (group.h), and the tiles of the experts before each
    int before = 0, top = 0;
    for (int e0 = 0; e0 < a.experts; e0 += 32) {
      const bool in = e0 + lane < a.experts;
      int2 seg = in ? s_seg[e0 + lane] : make_int2(0, 0);
      seg.x = rising(seg.x, top);
      seg.y = in ? max(seg.x, seg.y) : seg.x;
      top = __shfl_sync(0xffffffffu, seg.x, 31);
      int v = (seg.y - seg.x + ROWS - 1) / ROWS;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      v += before;
      if (in) {
        s_seg[e0 + lane] = seg;
        s_first[e0 + lane + 1] = v;
      }
      before = __shfl_sync(0xffffffffu, v, 31);
    }
    if (lane == 0) s_first[0] = 0;
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync();  // the other CTA's barriers are ready too
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  const int32_t total = (WEIGHTS ? a.experts * a.tiles_m : s_first[a.experts]) * a.tiles_n;
  bool ok = true;

  if (warp == 0) {
    if (lane == 0) {
      int slot = 0, phase = 1, seen = -1;
      for (int32_t t = unit; t < total && ok; t += units) {
        const ExTile w = ex_tile<BN, PAIR, WEIGHTS>(a, s_first, s_seg, t);
        const CUtensorMap* ma = &map_a;
        const CUtensorMap* mb = &map_b;
        if constexpr (WEIGHTS) {
          ma = a.maps + 2 * w.e;
          mb = ma + 1;
          if (w.e != seen) {  // written by another kernel through the generic proxy
            asm volatile("fence.proxy.tensormap::generic.acquire.gpu [%0], 128;" ::"l"(ma) : "memory");
            asm volatile("fence.proxy.tensormap::generic.acquire.gpu [%0], 128;" ::"l"(mb) : "memory");
            seen = w.e;
          }
        }
        const int32_t m0 = w.row + (int32_t)rank * TM, n0 = w.n0 + (int32_t)rank * L::B_ROWS;
        for (int k = 0; k < w.k1; ++k) {
          if (!mbar_wait_bounded(&empty[slot], phase, s_abort)) {
            ok = false;
            break;
          }
          if (rank == 0)
            mbar_arrive_expect_tx(&full[slot], (PAIR ? 2 : 1) * (L::A_STAGE + L::B_STAGE));
          const uint32_t sa = smem_u32(smem + L::A_OFF + slot * L::A_STAGE);
          const uint32_t sb = smem_u32(smem + L::B_OFF + slot * L::B_STAGE);
          const int kk = k * 64;
          const uint32_t bar = PAIR ? in_first(smem_u32(&full[slot])) : 0u;
          auto load = [&](uint32_t dst, const CUtensorMap* map, int x, int y) {
            if constexpr (PAIR) tma_load_pair(dst, map, bar, x, y);
            else tma_load_2d(dst, map, &full[slot], x, y);
          };
          auto load3 = [&](uint32_t dst, const CUtensorMap* map, int x, int y) {
            if constexpr (PAIR) tma_load_3d_pair(dst, map, bar, x, y, w.e);
            else tma_load_3d(dst, map, &full[slot], x, y, w.e);
          };
          if constexpr (WEIGHTS) {
#pragma unroll
            for (int r = 0; r < TM / 64; ++r) load(sa + r * MN_STRIDE, ma, m0 + 64 * r, w.base + kk);
#pragma unroll
            for (int r = 0; r < L::B_ROWS / 64; ++r)
              load(sb + r * MN_STRIDE, mb, n0 + 64 * r, w.base + kk);
          } else {
            load(sa, ma, kk, m0);
            if (a.b_mn) {
#pragma unroll
              for (int r = 0; r < L::B_ROWS / 64; ++r)
                load3(sb + r * MN_STRIDE, mb, n0 + 64 * r, kk);
            } else {
              load3(sb, mb, kk, n0);
            }
          }
          if (++slot == S) {
            slot = 0;
            phase ^= 1;
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
    if (rank == 0) {
      // What this warp does a k step has to fit into the step's 512 cycles beside the epilogue warps on its
      // scheduler. All of it walks the loop, so that descriptors and addresses are uniform registers, one
      // lane issues; the next step's barrier is tried before this step's products are issued.
      const bool lead = elect_one();
      const uint64_t a0 = WEIGHTS ? smem_desc_mn_sw128(smem_u32(smem + L::A_OFF), MN_STRIDE, ATOM)
                                  : smem_desc_sw128(smem_u32(smem + L::A_OFF));
      const bool b_mn = WEIGHTS || a.b_mn;
      const uint64_t b0 = b_mn ? smem_desc_mn_sw128(smem_u32(smem + L::B_OFF), MN_STRIDE, ATOM)
                               : smem_desc_sw128(smem_u32(smem + L::B_OFF));
      constexpr uint32_t A_STEP = WEIGHTS ? 2 * ATOM / 16 : 2;  // 16 of k, in the descriptor's units
      const uint32_t b_step = b_mn ? 2 * ATOM / 16 : 2;
      const uint32_t a_high = (uint32_t)(a0 >> 32), b_high = (uint32_t)(b0 >> 32);
      int slot = 0, phase = 0, local = 0;
      bool there = false;
      for (int32_t t = unit; t < total && ok; t += units, ++local) {
        const int32_t k1 = (int32_t)__reduce_max_sync(
            0xffffffffu, (uint32_t)ex_tile<BN, PAIR, WEIGHTS>(a, s_first, s_seg, t).k1);
        const int ab = local & 1;
        ok = __all_sync(0xffffffffu,
                        mbar_wait_bounded(&acc_empty[ab], ((local >> 1) & 1) ^ 1, s_abort));
        if (!ok) break;
        tc_fence_after();
        uint32_t d = tmem + (uint32_t)(ab * BN);
        int first = 0;  // the sum's first step
        for (int k = 0; k < k1; ++k) {
          if constexpr (RUNS) {
            if (k - first == a.run) {  // the next sum, in the other accumulator
              if (lead) commit<PAIR>(&acc_full[local & 1]);
              __syncwarp();
              ++local;
              ok = __all_sync(0xffffffffu, mbar_wait_bounded(&acc_empty[local & 1],
                                                             ((local >> 1) & 1) ^ 1, s_abort));
              if (!ok) break;
              tc_fence_after();
              d = tmem + (uint32_t)((local & 1) * BN);
              first = k;
            }
          }
          if (!there) {
            ok = __all_sync(0xffffffffu, mbar_wait_bounded(&full[slot], phase, s_abort));
            if (!ok) break;
          }
          tc_fence_after();
          const uint32_t a_low = (uint32_t)a0 + slot * (L::A_STAGE / 16);
          const uint32_t b_low = (uint32_t)b0 + slot * (L::B_STAGE / 16);
          uint64_t* const free_slot = &empty[slot];
          if (++slot == S) {
            slot = 0;
            phase ^= 1;
          }
          there = __all_sync(0xffffffffu, mbar_try_wait(&full[slot], phase));
          if (lead) {
#pragma unroll
            for (int j = 0; j < 4; ++j)  // 16 of k: one instruction
              issue_mma<PAIR, false>(d, (uint64_t)a_high << 32 | (a_low + j * A_STEP),
                                     (uint64_t)b_high << 32 | (b_low + j * b_step), a.idesc,
                                     (k > first || j > 0) ? 1u : 0u);
            commit<PAIR>(free_slot);
          }
          __syncwarp();
        }
        if (ok && lead) commit<PAIR>(&acc_full[local & 1]);
        __syncwarp();
      }
      if (lead) {
        if (!ok) report(status, SV_DEVICE_WAIT_TIMEOUT);
        // the products in flight read both CTAs' shared memory: let them finish
        commit<PAIR>(drained);
        const uint64_t t0 = global_timer_ns();
        while (!mbar_try_wait(drained, 0) && global_timer_ns() - t0 < 1000000000ull) {
        }
      }
      __syncwarp();
    }
  } else {
    const int q = warp & 3;            // TMEM lanes 32 q .. 32 q + 31
    constexpr int PARTS = BN >= 128 ? EX_EPI_WARPS / 4 : 2, COLS = BN / PARTS;  // a warp's columns
    const int part = (warp - 2) >> 2;
    const int e = threadIdx.x - 64;
    float* chunk = reinterpret_cast<float*>(smem + L::CHUNK_OFF) + (warp - 2) * 32 * CHUNK_LD;
    const bool scaled = ep.col_scale != nullptr;
    static_assert(BN <= EX_EPI_THREADS, "a thread holds a column's bias");
    ExTile w{};
    float bias_held = 0.f, scale_held = 1.f;
    // the tile and its columns' bias, found while the tile before is worked on: 1,500 cycles a tile
    auto look_up = [&](int32_t t) {
      if (t >= total) return;
      w = ex_tile<BN, PAIR, WEIGHTS>(a, s_first, s_seg, t);
      const bool in = e < BN && w.n0 + e < a.n;
      if (ep.bias) bias_held = in ? to_f32(static_cast<const O*>(ep.bias)[w.e * a.n + w.n0 + e]) : 0.f;
      if (scaled) scale_held = in ? __ldg(ep.col_scale + w.n0 + e) : 1.f;
    };
    auto give = [&](int ab) {  // the accumulator has been read
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (PAIR) arrive_at(in_first(smem_u32(&acc_empty[ab])));
        else arrive_at(smem_u32(&acc_empty[ab]));
      }
    };
    const uint32_t t_warp = tmem + ((uint32_t)(q * 32) << 16);
    look_up(unit);
    int local = 0, turn = 0;
    for (int32_t t = unit; t < total; t += units, ++local, turn ^= 1) {  // left by all warps alike
      if constexpr (RUNS) look_up(t);  // registers are short there, and time is not
      float* s_bias = s_cols + turn * 2 * BN;
      float* s_scale = s_bias + BN;
      Epilogue out = ep;
      if constexpr (WEIGHTS) out.out = static_cast<O*>(ep.out) + (int64_t)w.e * a.m * a.n;
      // this buffer's last readers were two tiles ago, before the previous barrier
      if (e < BN) {
        s_bias[e] = bias_held;
        s_scale[e] = scale_held;
      }
      ex_epi_sync();
      const int64_t row0 = (int64_t)w.row + rank * TM + q * 32;  // the warp's first row
      const int rows = (int)max((int64_t)0, min((int64_t)32, w.last - row0));
      const int n0 = w.n0;
      const bool formed = w.k1 > 0;  // an expert without positions: nothing was
      if constexpr (!RUNS) look_up(t + units);
      if (!ok) continue;
      float sum[RUNS ? COLS : 1];
      if constexpr (RUNS) {
        ok = ex_collect<COLS, BN>(sum, t_warp + part * COLS, a.runs, local, acc_full, s_abort, give);
        if (!ok) continue;
      }
      const int ab = local & 1;
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(&acc_full[ab], (local >> 1) & 1, s_abort))) {
        ok = false;
        continue;
      }
      tc_fence_after();
      const uint32_t t_row = t_warp + (uint32_t)(ab * BN);
      if constexpr (RUNS) {
        ex_add<COLS>(sum, t_row + part * COLS);
        give(ab);  // the next tile's sums need not wait for the stores
        if constexpr (SUMS == Sums::kRuns) {
          ex_sums<COLS>(sum, part * COLS, (int)min(a.n - n0, (int64_t)BN), s_bias, s_scale, lane < rows,
                        static_cast<float*>(out.out) + (row0 + lane) * a.n + n0);
          continue;
        }
      }
      if (!RUNS && a.direct && rows > 0) {
        using R = std::conditional_t<WIDE, float, O>;
        const int c1 = (int)min(a.n - n0, (int64_t)min((part + 1) * COLS, BN));
        const int64_t at = (row0 + min(lane, rows - 1)) * a.n + n0;
        R* to = static_cast<R*>(out.out) + at;
        float* kept = out.preact ? out.preact + at : nullptr;
        auto columns = [&](auto act) {
          ex_direct<O, WIDE, decltype(act)::value>(t_row, part * COLS, c1, s_bias, s_scale, formed,
                                                   lane < rows, to, kept);
        };
        if (WEIGHTS || ep.act == SV_ACT_NONE) columns(std::integral_constant<int, SV_ACT_NONE>());
        else if (ep.act == SV_ACT_SILU) columns(std::integral_constant<int, SV_ACT_SILU>());
        else if (ep.act == SV_ACT_GELU) columns(std::integral_constant<int, SV_ACT_GELU>());
        else columns(std::integral_constant<int, SV_ACT_GELU_TANH>());
        __syncwarp();
      }
#pragma unroll 1
      for (int c = part * COLS; c < min((part + 1) * COLS, BN); c += 32) {
        const int64_t col = (int64_t)n0 + c;
        if ((!RUNS && a.direct) || rows == 0 || col >= a.n) continue;  // the same in all lanes
        __syncwarp();  // the previous chunk has been read
        if constexpr (RUNS) {
          ex_stage<COLS>(sum, c - part * COLS, chunk + lane * CHUNK_LD);
        } else {
#pragma unroll
          for (int h = 0; h < 32; h += 16) {
            uint32_t raw[16];
            tmem_ld_32x32b_x16(t_row + c + h, raw);
            tc_wait_ld();
#pragma unroll
            for (int j = 0; j < 16; j += 4)
              *reinterpret_cast<uint4*>(chunk + lane * CHUNK_LD + h + j) =
                  formed ? make_uint4(raw[j], raw[j + 1], raw[j + 2], raw[j + 3])
                         : make_uint4(0u, 0u, 0u, 0u);
          }
        }
        __syncwarp();
        const int cols = (int)min((int64_t)32, a.n - col);
        if (a.wide_io && cols == 32) {
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
#pragma unroll 1
          for (int i = 0; i < 32; i += 16) {  // two groups of eight rows
            float v[2][8];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const float* src = chunk + (i + x * 8 + (lane >> 2)) * CHUNK_LD + j;
              *reinterpret_cast<float4*>(v[x]) = *reinterpret_cast<const float4*>(src);
              *reinterpret_cast<float4*>(v[x] + 4) = *reinterpret_cast<const float4*>(src + 4);
            }
            ex_finish<O, WIDE, 2, 8>(out, v, bias, scale, row0 + i + (lane >> 2), 8,
                                     rows - i - (lane >> 2), a.n, col + j);
          }
        } else if (lane < cols) {
          const float bias[1] = {ep.bias ? s_bias[c + lane] : 0.f};
          const float scale[1] = {scaled ? s_scale[c + lane] : 1.f};
#pragma unroll 1
          for (int r = 0; r < rows; r += 8) {
            float v[8][1];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i][0] = chunk[(r + i) * CHUNK_LD + lane];
            ex_finish<O, WIDE, 8, 1>(out, v, bias, scale, row0 + r, 1, rows - r, a.n, col + lane);
          }
        }
      }
      if constexpr (!RUNS) give(ab);
    }
    if (!ok) report(status, SV_DEVICE_WAIT_TIMEOUT);
    if (!WEIGHTS && a.zero_rest) {
      const int64_t head = s_seg[0].x * a.n, skip = s_seg[a.experts - 1].y * a.n - head;
      for (int64_t i = (int64_t)blockIdx.x * EX_EPI_THREADS + e; i < a.slots * a.n - skip;
           i += (int64_t)gridDim.x * EX_EPI_THREADS)
        static_cast<O*>(ep.out)[i < head ? i : i + skip] = from_f32<O>(0.f);
    }
  }

  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync();  // nothing of the pair still reads or signals this CTA
  if (warp == 1) {
    tc_fence_after();
    free_tmem<PAIR>(tmem, 2 * BN);
  }
}

// Copies of the operands' maps whose rows end with each expert's last position.
__global__ void __launch_bounds__(32)
    expert_maps_kernel(const __grid_constant__ CUtensorMap map_a,
                       const __grid_constant__ CUtensorMap map_b, const int32_t* offsets, int slots,
                       CUtensorMap* maps) {
  __shared__ alignas(128) uint32_t held[2][32];
  const int e = blockIdx.x, lane = threadIdx.x;
  held[0][lane] = reinterpret_cast<const uint32_t*>(&map_a)[lane];
  held[1][lane] = reinterpret_cast<const uint32_t*>(&map_b)[lane];
  // an expert without positions is not loaded; an extent is at least one
  const uint32_t rows = (uint32_t)max(1, segment_at(offsets, e, slots).last);
  __syncwarp();
  if (lane < 2) {
    asm volatile("tensormap.replace.tile.global_dim.shared::cta.b1024.b32 [%0], 1, %1;" ::"r"(
                     smem_u32(held[lane])),
                 "r"(rows)
                 : "memory");
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 2; ++i)
    asm volatile(
        "tensormap.cp_fenceproxy.global.shared::cta.tensormap::generic.release.gpu.sync.aligned"
        " [%0], [%1], 128;" ::"l"(maps + 2 * e + i),
        "r"(smem_u32(held[i]))
        : "memory");
}

// A map over `dims` elements (innermost first), with boxes of 128 bytes by `box_rows`. What is past
// the end of a dimension is filled with zeros.
int expert_map(const void* p, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
               int dtype, int box_rows, CUtensorMap* map) {
  EncodeFn encode = encode_fn();
  if (encode == nullptr) SV_FAIL(SV_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
  const cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1};
  const cuuint32_t steps[3] = {1, 1, 1};
  const CUtensorMapDataType type = dtype == SV_BFLOAT16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                        : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  if (encode(map, type, rank, const_cast<void*>(p), dims, strides, box, steps,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    SV_FAIL(SV_ERR_CUDA, "cuTensorMapEncodeTiled failed for an operand of the experts");
  return SV_OK;
}

bool direct_of(const ExpertGemm& g) {
  auto sectors = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 31u) == 0; };
  return g.n % 16 == 0 && sectors(g.ep.out) && sectors(g.ep.preact);
}

template <int BN, bool PAIR, typename O, bool WEIGHTS, bool WIDE, Sums SUMS>
int launch_expert(const ExpertGemm& g, CUtensorMap* maps, int32_t* status, cudaStream_t s) {
  using L = ExLayout<BN, PAIR>;
  auto kernel = expert_tc_kernel<BN, PAIR, O, WEIGHTS, WIDE, SUMS>;
  constexpr int ROWS = PAIR ? 2 * TM : TM;
  int dev = 0;
  SV_CUDA_TRY(cudaGetDevice(&dev));
  cudaLaunchConfig_t config{};
  config.blockDim = dim3(EX_THREADS);
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
    SV_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM));
    units = num_sms();
    if constexpr (PAIR) {
      config.gridDim = dim3(num_sms() / 2 * 2);
      SV_CUDA_TRY(cudaOccupancyMaxActiveClusters(&units, kernel, &config));
      if (units < 1) SV_FAIL(SV_ERR_CUDA, "expert_linear: no CTA pair fits this device");
      units = std::min(units, num_sms() / 2);
    }
    if (dev < 256) units_of[dev] = units;
  }
  constexpr int ES = 2;
  CUtensorMap map_a, map_b;
  const cuuint64_t slots = (cuuint64_t)g.slots;
  int rc;
  if constexpr (WEIGHTS) {
    const cuuint64_t da[2] = {(cuuint64_t)g.m, slots}, db[2] = {(cuuint64_t)g.n, slots};
    const cuuint64_t sa = (cuuint64_t)g.a.ld * ES, sb = (cuuint64_t)g.b.ld * ES;
    rc = expert_map(g.a.p, 2, da, &sa, g.dtype, 64, &map_a);
    if (rc == SV_OK) rc = expert_map(g.b.p, 2, db, &sb, g.dtype, 64, &map_b);
    if (rc != SV_OK) return rc;
    expert_maps_kernel<<<g.experts, 32, 0, s>>>(map_a, map_b, g.offsets, (int)g.slots, maps);
    SV_LAUNCH_CHECK();
  } else {
    const cuuint64_t da[2] = {(cuuint64_t)g.k, slots};
    const cuuint64_t sa = (cuuint64_t)g.a.ld * ES;
    rc = expert_map(g.a.p, 2, da, &sa, g.dtype, TM, &map_a);
    const cuuint64_t db[3] = {(cuuint64_t)(g.b.mn ? g.n : g.k), (cuuint64_t)(g.b.mn ? g.k : g.n),
                              (cuuint64_t)g.experts};
    const cuuint64_t sb[2] = {(cuuint64_t)g.b.ld * ES, (cuuint64_t)g.b_expert * ES};
    if (rc == SV_OK) rc = expert_map(g.b.p, 3, db, sb, g.dtype, g.b.mn ? 64 : L::B_ROWS, &map_b);
    if (rc != SV_OK) return rc;
  }
  ExArgs a{};
  a.offsets = g.offsets;
  a.experts = g.experts;
  a.slots = (int32_t)g.slots;
  a.m = g.m;
  a.n = g.n;
  a.tiles_n = (int32_t)((g.n + BN - 1) / BN);
  a.tiles_m = (int32_t)((g.m + ROWS - 1) / ROWS);
  a.steps = (int32_t)((g.k + 63) / 64);
  if constexpr (SUMS != Sums::kOne) {  // of one length, but for the last
    const int32_t most = run_steps(a.steps), sums = (a.steps + most - 1) / most;
    a.run = (a.steps + sums - 1) / sums;
    a.runs = (a.steps + a.run - 1) / a.run;
  }
  a.b_mn = g.b.mn;
  a.zero_rest = g.zero_rest;
  a.maps = maps;
  a.idesc = idesc_f16_major(g.dtype == SV_BFLOAT16, ROWS, BN, WEIGHTS, WEIGHTS || g.b.mn);
  const int64_t pieces = WEIGHTS ? (int64_t)g.experts * a.tiles_m : g.slots / ROWS + g.experts;
  if (pieces * a.tiles_n > INT32_MAX / 2) SV_FAIL(SV_ERR_UNSUPPORTED, "expert_linear: too many tiles");
  const Epilogue& ep = g.ep;
  a.wide_io = g.n % 8 == 0 && aligned16(ep.out) && (!ep.preact || aligned16(ep.preact));
  a.direct = direct_of(g);
  units = (int)std::min<int64_t>(pieces * a.tiles_n, units);
  config.gridDim = dim3((unsigned)(units * (PAIR ? 2 : 1)));
  SV_CUDA_TRY(cudaLaunchKernelEx(&config, kernel, map_a, map_b, a, ep, status));
  return SV_OK;
}

template <typename O, bool WEIGHTS, bool WIDE, Sums SUMS>
int launch_form(const ExpertGemm& g, ExpertTile tile, CUtensorMap* maps, int32_t* status,
                cudaStream_t s) {
  switch (tile) {
    case ExpertTile::kPair256: return launch_expert<256, true, O, WEIGHTS, WIDE, SUMS>(g, maps, status, s);
    case ExpertTile::kPair128: return launch_expert<128, true, O, WEIGHTS, WIDE, SUMS>(g, maps, status, s);
    case ExpertTile::kOne128: return launch_expert<128, false, O, WEIGHTS, WIDE, SUMS>(g, maps, status, s);
    default: return launch_expert<64, false, O, WEIGHTS, WIDE, SUMS>(g, maps, status, s);
  }
}

template <typename O>
int launch_typed(const ExpertGemm& g, ExpertTile tile, CUtensorMap* maps, int32_t* status,
                 cudaStream_t s) {
  if (g.form == ExpertForm::kWeights)
    return launch_form<O, true, false, Sums::kOne>(g, tile, maps, status, s);
  if (g.ep.out_dtype != SV_FLOAT32)
    return launch_form<O, false, false, Sums::kOne>(g, tile, maps, status, s);
  if (!g.runs || g.k <= 64 * run_steps((g.k + 63) / 64))
    return launch_form<O, false, true, Sums::kOne>(g, tile, maps, status, s);
  return direct_of(g) && g.ep.act == SV_ACT_NONE
             ? launch_form<O, false, true, Sums::kRuns>(g, tile, maps, status, s)
             : launch_form<O, false, true, Sums::kStaged>(g, tile, maps, status, s);
}

}  // namespace

size_t expert_maps_bytes(int experts) { return (size_t)experts * 2 * sizeof(CUtensorMap); }

int expert_gemm_tc(const ExpertGemm& g, ExpertTile tile, void* maps, int32_t* status,
                   cudaStream_t s) {
  CUtensorMap* at = static_cast<CUtensorMap*>(maps);
  return g.dtype == SV_FLOAT16 ? launch_typed<__half>(g, tile, at, status, s)
                               : launch_typed<__nv_bfloat16>(g, tile, at, status, s);
}

}  // namespace sv
