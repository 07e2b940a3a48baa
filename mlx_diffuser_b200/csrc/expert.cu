// Linear projections grouped by expert, with the gather of the rows that the router sent to each expert
// before them and the weighted sum of the experts' results behind them, and their gradients.
//
//     x_p = x[order[p] / k] (gathered) or x[p],   z_p = x_p W_e^T + b_e,   r_p = act(z_p)
//     y   = r, in the order of the experts, or y_n = sum_j w_nj r[place_nj] (combined)
//     dr_p = w dy[order[p] / k] or dy[p],  dz = dr act'(z)
//     dW_e = sum over e's p of dz_p^T x_p,  db_e = sum dz_p,  dw_nj = dy_n . r[place_nj]
//     dx_p = dz_p W_e, and dx_n = sum_j dx[place_nj] where x was gathered
//
// The products' sizes differ by expert and are known on the device only. Three kernels form them:
//   expert_few_kernel   up to FEW_SLOTS positions: the chosen experts' weights read once, on the CUDA cores;
//   expert_f32_kernel   fp32: the register tiles of gemm_f32.cuh;
//   expert_tc.cu        fp16 / bf16: tcgen05 tiles fed by TMA.
// What is summed over a row's choices is held in fp32: rounded to 16 bits before, it costs the sum a second
// rounding (dx 0.0029 of its size off, against 0.0023), and the products with dy, which the weights'
// gradients are, all bits past the type's.
#include <algorithm>
#include <type_traits>

#include "expert.h"
#include "gemm_f32.cuh"
#include "group.h"
#include "raise.cuh"

namespace sv {
namespace {

constexpr int EXPERT_MAX = 1024;
constexpr int FEW_ROWS = 8;     // positions of a piece
// Positions that the kernel for few takes. bf16, against the tensor cores' tiles: 16 experts of 1024 -> 4096
// 8 positions 27 us (44), 16 55 (44); 8 of 1024 -> 1024 8 8.4 (17), 16 13.7 (17); 2 of 1024 -> 4096 8
// 18.5 (17), 16 32 (17). What decides is the positions an expert, which the host does not know: where few
// experts share eight, the tiles would be as quick. fp32 takes up to 32, whose tiles took 285, 56 and 56 us for 32
// positions where bf16 took 95, 22 and 59 by this kernel.
constexpr int FEW_SLOTS = 8, FEW_SLOTS_F32 = 32;
constexpr int DZ_ROWS = 64;     // positions of a piece of the backward pass's element-wise step
constexpr int ALIGN = 256;

struct Routing {
  const int32_t* order;
  const int32_t* offsets;
  const int32_t* place;
  const float* weights;
  int64_t n;      // rows
  int k;          // choices
  int experts;
  int64_t slots;  // n * k
};

// The row of a position, or -1 where the entry is not one.
__device__ __forceinline__ int64_t row_of(const Routing& r, int64_t p) {
  const int32_t slot = __ldg(r.order + p);
  return slot >= 0 && slot < r.slots ? slot / r.k : -1;
}

// Zeros in the rows that no expert has, by 256 threads of each of `blocks` blocks.
template <typename T>
__device__ __forceinline__ void clear_rest(const Routing& r, int64_t n, T* out, int block, int blocks) {
  const Segment has = covered(r.offsets, r.experts, (int)r.slots);
  const int64_t head = has.first * n, skip = (has.last - has.first) * n;
  for (int64_t i = (int64_t)block * 256 + threadIdx.x; i < r.slots * n - skip; i += (int64_t)blocks * 256)
    out[i < head ? i : i + skip] = from_f32<T>(0.f);
}

// ---- few positions -------------------------------------------------------------------------------

// The epilogue of one sum, into T or fp32.
template <typename T>
__device__ __forceinline__ void store_result(const Epilogue& ep, int64_t i, int64_t j, int64_t n,
                                             float acc) {
  if (ep.out_dtype != SV_FLOAT32) return epilogue_store<T>(ep, i, j, n, acc);
  if (ep.bias) acc += to_f32(static_cast<const T*>(ep.bias)[j]);
  if (ep.preact) ep.preact[i * n + j] = acc;
  static_cast<float*>(ep.out)[i * n + j] = activate(acc, ep.act);
}

// One column's sums for up to ROWS rows of a piece: W warps a column (8: the block's), lanes along k in
// accesses of V elements, the rows' accesses in flight together (rows past the last read it again).
template <typename T, int ROWS, int V, int W>
__device__ __forceinline__ void few_rows(const T* x, int64_t ldx, const T* w, const Routing& r,
                                         bool gather, const Piece& p, int64_t j, int64_t n, int64_t k,
                                         const Epilogue& ep, float (&part)[8][FEW_ROWS],
                                         int32_t* status) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slot = W > 1 ? (int)threadIdx.x : lane;
  const T* from[ROWS];
  bool bad[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int at = min(p.first + i, p.last - 1);
    const int64_t row = gather ? row_of(r, at) : at;
    bad[i] = row < 0;
    from[i] = x + (bad[i] ? 0 : row) * ldx;
    if (bad[i] && threadIdx.x == 0) report(status, SV_DEVICE_BAD_INDEX);
  }
  float acc[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) acc[i] = 0.f;
  if (j < n) {
#pragma unroll(ROWS <= 2 ? 4 : 2)
    for (int64_t c = (int64_t)slot * V; c < k; c += 32 * W * V) {
      alignas(16) T we[V];
      if constexpr (V * sizeof(T) == 16)
        *reinterpret_cast<uint4*>(we) = __ldg(reinterpret_cast<const uint4*>(w + c));
      else
        we[0] = w[c];
      alignas(16) T xe[ROWS][V];
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        if constexpr (V * sizeof(T) == 16)
          *reinterpret_cast<uint4*>(xe[i]) = __ldg(reinterpret_cast<const uint4*>(from[i] + c));
        else
          xe[i][0] = from[i][c];
      }
#pragma unroll
      for (int i = 0; i < ROWS; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) acc[i] = fmaf(to_f32(xe[i][e]), to_f32(we[e]), acc[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
    if (bad[i]) acc[i] = 0.f;
  }
  const int rows = p.last - p.first;
  if constexpr (W > 1) {
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < ROWS; ++i) part[warp][i] = acc[i];
    }
    __syncthreads();
    if ((int)threadIdx.x < min(ROWS, rows)) {
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) v += part[i][threadIdx.x];
      store_result<T>(ep, p.first + threadIdx.x, j, n, v);
    }
  } else if (j < n) {
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
      if (lane == i && i < rows) store_result<T>(ep, p.first + i, j, n, acc[i]);
  }
}

// A block takes a piece of an expert's positions (blockIdx.y) and eight columns, a warp each, or one
// column with all its warps, by the code for as many rows as the piece has: experts mostly have one
// or two, and the code for eight reads x eight times (8 positions of 16 experts, 1024 x 4096: 40 us by the
// code for four, 27 so). LONE: pieces of one position, whose code alone has more warps an SM (7.1 against
// 9.2 us).
template <typename T, bool LONE, int V, int W>
__global__ void __launch_bounds__(256)
    expert_few_kernel(const T* __restrict__ x, int64_t ldx, const T* __restrict__ w, int64_t ldw,
                      int64_t w_expert, Routing r, bool gather, bool zero_rest, int64_t n,
                      int64_t k, Epilogue ep, int32_t* status) {
  __shared__ float part[8][FEW_ROWS];
  if (zero_rest && blockIdx.y == 0) clear_rest(r, n, static_cast<T*>(ep.out), blockIdx.x, gridDim.x);
  const Piece p = find_piece<false>(r.offsets, r.experts, (int)r.slots, LONE ? 1 : FEW_ROWS, blockIdx.y);
  if (p.group < 0) return;
  const int64_t j = W > 1 ? blockIdx.x : (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const T* we = w + p.group * w_expert + min(j, n - 1) * ldw;
  if (ep.bias) ep.bias = static_cast<const T*>(ep.bias) + p.group * n;
  const int rows = p.last - p.first;
  if constexpr (LONE) few_rows<T, 1, V, W>(x, ldx, we, r, gather, p, j, n, k, ep, part, status);
  else if (rows == 1) few_rows<T, 1, V, W>(x, ldx, we, r, gather, p, j, n, k, ep, part, status);
  else if (rows == 2) few_rows<T, 2, V, W>(x, ldx, we, r, gather, p, j, n, k, ep, part, status);
  else if (rows <= 4) few_rows<T, 4, V, W>(x, ldx, we, r, gather, p, j, n, k, ep, part, status);
  else few_rows<T, FEW_ROWS, V, W>(x, ldx, we, r, gather, p, j, n, k, ep, part, status);
}

template <typename T>
__global__ void __launch_bounds__(256) expert_rest_kernel(Routing r, int64_t n, T* out) {
  clear_rest(r, n, out, blockIdx.x, gridDim.x);
}

// ---- fp32 ----------------------------------------------------------------------------------------

// C tile of 16 R x 16 R, columns fastest: of an expert (blockIdx.y) with WEIGHTS, otherwise of a piece of
// 16 R positions.
template <int R, int VA, int VB, bool WEIGHTS>
__global__ void __launch_bounds__(256, 2) expert_f32_kernel(ExpertGemm g) {
  constexpr int T = 16 * R;
  __shared__ __align__(16) float sa[2][FK][T + 4];
  __shared__ __align__(16) float sb[2][FK][T + 4];
  const unsigned across = (unsigned)((g.n + T - 1) / T);
  Operand b = g.b;
  Epilogue ep = g.ep;
  int64_t i0, j0, m, k0 = 0, k1 = g.k;
  if constexpr (WEIGHTS) {
    const int e = blockIdx.y;
    i0 = (int64_t)(blockIdx.x / across) * T;
    j0 = (int64_t)(blockIdx.x % across) * T;
    m = g.m;
    const Segment seg = segment_at(g.offsets, e, (int)g.slots);
    k0 = seg.first;
    k1 = seg.last;
    ep.out = static_cast<float*>(ep.out) + e * g.m * g.n;
  } else {
    const Piece p = find_piece<false>(g.offsets, g.experts, (int)g.slots, T, blockIdx.x / across);
    if (p.group < 0) return;
    i0 = p.first;
    m = p.last;
    j0 = (int64_t)(blockIdx.x % across) * T;
    b.p = static_cast<const float*>(b.p) + p.group * g.b_expert;
    if (ep.bias) ep.bias = static_cast<const float*>(ep.bias) + p.group * g.n;
  }
  uint64_t acc[R][R / 2];
  tile_f32<R, VA, VB>(g.a, i0, m, b, j0, g.n, k0, k1, sa, sb, acc);
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int64_t row = i0 + 64 * (i / 4) + 4 * ty + i % 4;
    if (row >= m) continue;
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const int64_t col = j0 + 64 * (j / 4) + 4 * tx + j % 4;
      if (col >= g.n) continue;
      epilogue_store<float>(ep, row, col, g.n,
                            __uint_as_float((uint32_t)(acc[i][j / 2] >> (j % 2 * 32))));
    }
  }
}

template <int R, bool WEIGHTS>
void launch_f32(const ExpertGemm& g, dim3 grid, cudaStream_t s) {
  const bool va = aligned16(g.a.p) && g.a.ld % 4 == 0;
  const bool vb = aligned16(g.b.p) && g.b.ld % 4 == 0 && g.b_expert % 4 == 0;
  auto kernel = va ? (vb ? expert_f32_kernel<R, 4, 4, WEIGHTS> : expert_f32_kernel<R, 4, 1, WEIGHTS>)
                   : (vb ? expert_f32_kernel<R, 1, 4, WEIGHTS> : expert_f32_kernel<R, 1, 1, WEIGHTS>);
  kernel<<<grid, 256, 0, s>>>(g);
}

// Tiles of 128 x 128 where they give every SM one, else of 64 x 64.
int expert_gemm_f32(const ExpertGemm& g, cudaStream_t s) {
  const bool weights = g.form == ExpertForm::kWeights;
  auto tiles_of = [&](int64_t t) {  // of an expert, or in all
    return ((g.n + t - 1) / t) * (weights ? (g.m + t - 1) / t : g.slots / t + g.experts);
  };
  const int64_t large = weights ? g.experts * tiles_of(128) : tiles_of(128) - g.experts * ((g.n + 127) / 128);
  const bool small = large < num_sms();
  const int64_t tiles = tiles_of(small ? 64 : 128);
  if (tiles > INT32_MAX) SV_FAIL(SV_ERR_UNSUPPORTED, "expert_linear: too many tiles");
  const dim3 grid((unsigned)tiles, weights ? (unsigned)g.experts : 1u);
  if (weights) {
    if (small) launch_f32<4, true>(g, grid, s);
    else launch_f32<8, true>(g, grid, s);
  } else {
    if (small) launch_f32<4, false>(g, grid, s);
    else launch_f32<8, false>(g, grid, s);
  }
  SV_LAUNCH_CHECK();
  return SV_OK;
}

// ---- rows in the order of the experts ------------------------------------------------------------

// out[p] = x[order[p] / k], rows `ld_out` apart, zeros behind column `cols`. A warp takes a position, four
// 16-byte accesses of a lane in flight. WIDE: rows are read as they are stored, element by element
// otherwise. 81,324 x 1024 bf16 is 250 MB: 38 us of HBM.
template <typename E, bool WIDE>
__global__ void __launch_bounds__(256)
    expert_gather_kernel(const E* __restrict__ x, int64_t ldx, Routing r, bool gather, int64_t cols,
                         E* __restrict__ out, int64_t ld_out, int32_t* status) {
  constexpr int W = 16 / sizeof(E), AHEAD = WIDE ? 4 : 1;
  const int lane = threadIdx.x & 31, across = (int)(ld_out / W);
  const int64_t step = (int64_t)gridDim.x * 8;
  for (int64_t p = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); p < r.slots; p += step) {
    const int64_t row = gather ? row_of(r, p) : p;
    if (row < 0 && lane == 0) report(status, SV_DEVICE_BAD_INDEX);
    const E* from = x + (row < 0 ? 0 : row) * ldx;
    for (int c0 = lane; c0 < across; c0 += 32 * AHEAD) {
      alignas(16) E e[AHEAD][W];
#pragma unroll
      for (int s = 0; s < AHEAD; ++s) {
        const int c = c0 + 32 * s;
        if constexpr (WIDE) {
          if (c < across) *reinterpret_cast<uint4*>(e[s]) = __ldg(reinterpret_cast<const uint4*>(from) + c);
        } else {
#pragma unroll
          for (int i = 0; i < W; ++i)
            e[s][i] = (int64_t)c * W + i < cols ? __ldg(from + (int64_t)c * W + i) : E(0);
        }
      }
#pragma unroll
      for (int s = 0; s < AHEAD; ++s) {
        const int c = c0 + 32 * s;
        if (c < across)
          reinterpret_cast<uint4*>(out + p * ld_out)[c] =
              row < 0 ? make_uint4(0u, 0u, 0u, 0u) : *reinterpret_cast<const uint4*>(e[s]);
      }
    }
  }
}

// The experts' weights in rows of a multiple of 16 bytes.
template <typename E>
__global__ void __launch_bounds__(256)
    expert_pad_kernel(const E* __restrict__ w, int64_t ld, int64_t expert, int64_t rows,
                      int64_t cols, int64_t total, E* __restrict__ out, int64_t ld_out) {
  constexpr int W = 16 / sizeof(E);
  const int64_t across = ld_out / W;
  for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < total;
       at += (int64_t)gridDim.x * 256) {
    const int64_t row = at / across, c = (at - row * across) * W, e = row / rows;
    const E* from = w + e * expert + (row - e * rows) * ld + c;
    alignas(16) E v[W];
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = c + i < cols ? __ldg(from + i) : E(0);
    *reinterpret_cast<uint4*>(out + row * ld_out + c) = *reinterpret_cast<const uint4*>(v);
  }
}

// V elements, in 16-byte accesses where that many bytes are whole ones.
template <typename T, int V>
__device__ __forceinline__ void load_v(const T* p, float (&v)[V]) {
  if constexpr (V * sizeof(T) % 16 == 0) {
    alignas(16) T e[V];
#pragma unroll
    for (int i = 0; i < (int)sizeof(e) / 16; ++i)
      reinterpret_cast<uint4*>(e)[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = to_f32(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = to_f32(p[i]);
  }
}

template <typename T, int V>
__device__ __forceinline__ void store_v(T* p, const float (&v)[V]) {
  if constexpr (V == 8) {
    uint4 w[sizeof(T) / 2];
    pack_eight<T>(v, w);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(p)[i] = w[i];
  } else if constexpr (V * sizeof(T) == 16) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) p[i] = from_f32<T>(v[i]);
  }
}

// out[n] = sum_j w_nj rows[place_nj], in the order of the choices (not weighted: ones), over the places that
// an expert has: the others' rows were not formed. V elements a thread.
template <typename T, int V>
__global__ void __launch_bounds__(256)
    expert_combine_kernel(const float* __restrict__ rows, Routing r, bool weighted, int64_t cols,
                          T* __restrict__ out) {
  const int64_t across = cols / V, total = r.n * across;
  const Segment has = covered(r.offsets, r.experts, (int)r.slots);
  for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < total;
       at += (int64_t)gridDim.x * 256) {
    const int64_t n = total <= UINT32_MAX ? (uint32_t)at / (uint32_t)across : at / across;
    const int64_t c = (at - n * across) * V;
    float sum[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = 0.f;
#pragma unroll 2
    for (int j = 0; j < r.k; ++j) {
      const int32_t p = __ldg(r.place + n * r.k + j);
      if (p < has.first || p >= has.last) continue;
      const float w = weighted ? __ldg(r.weights + n * r.k + j) : 1.f;
      float v[V];
      load_v<float, V>(rows + (int64_t)p * cols + c, v);
#pragma unroll
      for (int i = 0; i < V; ++i) sum[i] = fmaf(w, v[i], sum[i]);
    }
    store_v<T, V>(out + n * cols + c, sum);
  }
}

// ---- the backward pass's element-wise step -------------------------------------------------------

struct DzArgs {
  Routing r;
  const void* dy;        // [n] or [slots] rows of `cols`
  const float* preact;   // [slots][cols], or null
  bool combine;
  int64_t cols;
  void* dz;              // rows ld_dz apart, or null
  int64_t ld_dz;
  float* partial;        // [pieces][cols], or null
  Raise raise;           // fp16
};

// dz_p = w dy act'(z), rounded to the feature type as the products' operand (raise.cuh), and the column
// sums of the unrounded values over a piece of DZ_ROWS positions of one expert: 32 V columns a block,
// eight rows at a time.
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(256, 4) expert_dz_kernel(const __grid_constant__ DzArgs a) {
  __shared__ float s_sum[8][32 * V + 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float up = 1.0f;
  if constexpr (std::is_same<T, __half>::value) {
    if (a.raise.top != nullptr) {
      // the largest finite |dy|: one expert's infinity leaves the others' gradients their range
      up = raise_of(__ldg(a.raise.top));
      if (a.combine) up *= room_of(__ldg(a.raise.top + 1));
      if (blockIdx.x == 0 && blockIdx.y == 0)
        for (int64_t i = threadIdx.x; i < a.raise.k; i += 256) a.raise.down[i] = 1.0f / up;
    }
  }
  const Piece p = find_piece<false>(a.r.offsets, a.r.experts, (int)a.r.slots, DZ_ROWS, blockIdx.x);
  if (p.group < 0) return;
  // the piece's rows and weights once: found row by row, two dependent loads stood before each row's own
  __shared__ int s_row[DZ_ROWS];
  __shared__ float s_weight[DZ_ROWS];
  if (a.combine) {
    if ((int)threadIdx.x < p.last - p.first) {
      const int32_t slot = __ldg(a.r.order + p.first + threadIdx.x);
      const bool in = slot >= 0 && slot < a.r.slots;
      s_row[threadIdx.x] = in ? slot / a.r.k : -1;
      s_weight[threadIdx.x] = in ? __ldg(a.r.weights + slot) : 0.0f;
    }
    __syncthreads();
  }
  const int64_t c = ((int64_t)blockIdx.y * 32 + lane) * V;
  float sum[V];
#pragma unroll
  for (int i = 0; i < V; ++i) sum[i] = 0.f;
  if (c < a.cols) {
#pragma unroll(ACT == SV_ACT_NONE ? 4 : 2)
    for (int at = p.first + warp; at < p.last; at += 8) {
      const int64_t row = a.combine ? s_row[at - p.first] : at;
      float d[V];
      load_v<T, V>(static_cast<const T*>(a.dy) + max(row, (int64_t)0) * a.cols + c, d);
      if (a.combine) {
        const float w = s_weight[at - p.first];
#pragma unroll
        for (int i = 0; i < V; ++i) d[i] = row < 0 ? 0.f : d[i] * w;
      }
      if constexpr (ACT != SV_ACT_NONE) {
        float z[V];
        const float* from = a.preact + (int64_t)at * a.cols + c;
#pragma unroll
        for (int i = 0; i < V; i += V >= 4 ? 4 : 1) {
          if constexpr (V >= 4) {
            const float4 q = __ldg(reinterpret_cast<const float4*>(from + i));
            z[i] = q.x; z[i + 1] = q.y; z[i + 2] = q.z; z[i + 3] = q.w;
          } else {
            z[i] = __ldg(from + i);
          }
        }
#pragma unroll
        for (int i = 0; i < V; ++i)
          d[i] *= sizeof(T) == 2 ? activate_slope_half(z[i], ACT) : activate_slope(z[i], ACT);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        sum[i] += d[i];
        d[i] *= up;
      }
      if (a.dz) store_v<T, V>(static_cast<T*>(a.dz) + (int64_t)at * a.ld_dz + c, d);
    }
  }
  if (a.partial == nullptr) return;
#pragma unroll
  for (int i = 0; i < V; ++i) s_sum[warp][lane * V + i] = sum[i];
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * V; i += 256) {
    const int64_t col = (int64_t)blockIdx.y * 32 * V + i;
    if (col < a.cols) {
      float v = s_sum[0][i];
#pragma unroll
      for (int w = 1; w < 8; ++w) v += s_sum[w][i];
      a.partial[(int64_t)blockIdx.x * a.cols + col] = v;
    }
  }
}

// db_e = the sums of e's pieces in order. blockIdx.y: the expert; 32 columns a block.
template <typename T>
__global__ void __launch_bounds__(256)
    expert_dbias_kernel(const float* __restrict__ partial, Routing r, int64_t cols, T* out) {
  __shared__ float s[8][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = blockIdx.y;
  const int2 pieces = pieces_at(r.offsets, e, (int)r.slots, DZ_ROWS);
  const int first = pieces.x, mine = pieces.y;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  float v = 0.f;
  if (c < cols)
    for (int p = warp; p < mine; p += 8) v += __ldg(partial + (int64_t)(first + p) * cols + c);
  s[warp][lane] = v;
  __syncthreads();
  if (warp == 0 && c < cols) {
#pragma unroll
    for (int i = 1; i < 8; ++i) v += s[i][lane];
    out[e * cols + c] = from_f32<T>(v);
  }
}

// dw_nj = dy_n . r[place_nj], a warp a row and choice; 0 where the choice has no expert.
template <typename T, int V>
__global__ void __launch_bounds__(256)
    expert_dweights_kernel(const T* __restrict__ dy, const float* __restrict__ rows, Routing r,
                           int64_t cols, float* __restrict__ out) {
  const int lane = threadIdx.x & 31;
  const int64_t step = (int64_t)gridDim.x * 8;
  const Segment has = covered(r.offsets, r.experts, (int)r.slots);
  for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < r.slots; i += step) {
    const int32_t p = __ldg(r.place + i);
    float sum = 0.f;
    if (p >= has.first && p < has.last) {
      const T* g = dy + i / r.k * cols;
      const float* v = rows + (int64_t)p * cols;
#pragma unroll 2
      for (int64_t c = lane * V; c < cols; c += 32 * V) {
        float x[V], y[V];
        load_v<T, V>(g + c, x);
        load_v<float, V>(v + c, y);
#pragma unroll
        for (int q = 0; q < V; ++q) sum = fmaf(x[q], y[q], sum);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) out[i] = sum;
  }
}

// ---- host ----------------------------------------------------------------------------------------

bool float_type(int d) { return d == SV_FLOAT32 || d == SV_FLOAT16 || d == SV_BFLOAT16; }

unsigned grid_for(int64_t items, int per_sm) {
  return (unsigned)std::max<int64_t>(1, std::min<int64_t>((items + 255) / 256, (int64_t)num_sms() * per_sm));
}

// 16-byte rows: what TMA can read.
int64_t padded(int64_t cols, int dtype) {
  const int es = elem_size(dtype);
  return (int64_t)align_up((size_t)cols * es, 16) / es;
}
bool ready(const void* p, int64_t ld, int dtype) {
  return aligned16(p) && ld * elem_size(dtype) % 16 == 0;
}

Routing routing_of(const sv_expert_args& g) {
  return {g.order, g.offsets, g.place, g.weights, g.n, g.k, g.experts, g.n * g.k};
}

// Rows in the order of the experts, or as they are where those of a product need padding.
int gather_rows(const void* x, int64_t ldx, const Routing& r, bool gather, int64_t cols, int dtype,
                void* out, int64_t ld_out, int32_t* status, cudaStream_t s) {
  const int es = elem_size(dtype);
  if (r.slots == 0 || ld_out == 0) return SV_OK;
  const unsigned blocks = grid_for(r.slots * 32, 8);
  const bool wide = ready(x, ldx, dtype) && cols == ld_out;
#define SV_GATHER(E, WIDE)                                                               \
  expert_gather_kernel<E, WIDE><<<blocks, 256, 0, s>>>(static_cast<const E*>(x), ldx, r, \
                                                       gather, cols, static_cast<E*>(out), \
                                                       ld_out, status)
  if (es == 4) {
    if (wide) SV_GATHER(uint32_t, true);
    else SV_GATHER(uint32_t, false);
  } else {
    if (wide) SV_GATHER(uint16_t, true);
    else SV_GATHER(uint16_t, false);
  }
#undef SV_GATHER
  SV_LAUNCH_CHECK();
  return SV_OK;
}

template <typename T>
int combine_typed(const float* rows, const Routing& r, bool weighted, int64_t cols, void* out,
                  cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  T* to = static_cast<T*>(out);
  const bool wide = cols % V == 0 && aligned16(rows) && aligned16(out);
  const int64_t items = r.n * cols / (wide ? V : 1);
  if (items == 0) return SV_OK;
  if (wide)
    expert_combine_kernel<T, V><<<grid_for(items, 16), 256, 0, s>>>(rows, r, weighted, cols, to);
  else
    expert_combine_kernel<T, 1><<<grid_for(items, 16), 256, 0, s>>>(rows, r, weighted, cols, to);
  SV_LAUNCH_CHECK();
  return SV_OK;
}

int combine(const float* rows, const Routing& r, bool weighted, int64_t cols, int dtype, void* out,
            cudaStream_t s) {
  switch (dtype) {
    case SV_FLOAT32: return combine_typed<float>(rows, r, weighted, cols, out, s);
    case SV_FLOAT16: return combine_typed<__half>(rows, r, weighted, cols, out, s);
    default: return combine_typed<__nv_bfloat16>(rows, r, weighted, cols, out, s);
  }
}

template <typename T>
int few_typed(const sv_expert_args& g, const Routing& r, const Epilogue& ep, int32_t* status,
              cudaStream_t s) {
  constexpr int VE = 16 / sizeof(T);
  const T* x = static_cast<const T*>(g.x);
  const T* w = static_cast<const T*>(g.weight);
  const bool vec = aligned16(x) && aligned16(w) && g.inputs % VE == 0 && g.ldx % VE == 0 &&
                   g.ldw % VE == 0 && g.w_expert % VE == 0;
  // One row's choices are mostly different experts: a piece each, and one that is named twice has two.
  const bool lone = g.n == 1 && r.slots <= FEW_SLOTS_F32;
  // pieces: every slot its own expert at most, or whole pieces and a ragged one an expert
  const int64_t pieces =
      lone ? r.slots
           : std::min<int64_t>(r.slots, r.slots / FEW_ROWS + std::min<int64_t>(g.experts, r.slots));
  if (pieces > 65535) SV_FAIL(SV_ERR_UNSUPPORTED, "expert_linear: too many rows without inputs");
  const bool wide = g.outputs * pieces >= 8 * num_sms();
  const dim3 grid((unsigned)(wide ? (g.outputs + 7) / 8 : g.outputs), (unsigned)pieces);
  auto pick = [&](auto lone) {
    constexpr bool L = decltype(lone)::value;
    return vec ? (wide ? expert_few_kernel<T, L, VE, 1> : expert_few_kernel<T, L, VE, 8>)
               : (wide ? expert_few_kernel<T, L, 1, 1> : expert_few_kernel<T, L, 1, 8>);
  };
  auto kernel = lone ? pick(std::true_type()) : pick(std::false_type());
  kernel<<<grid, 256, 0, s>>>(x, g.ldx, w, g.ldw, g.w_expert, r, g.gather != 0, !g.combine, g.outputs,
                              g.inputs, ep, status);
  SV_LAUNCH_CHECK();
  return SV_OK;
}

// The tile with the least estimated time: linear.cu's estimate for an expert's mean share of positions.
ExpertTile pick_tile(int64_t experts, int64_t m, int64_t n, int64_t k) {
  const int64_t sms = num_sms(), steps = (k + 63) / 64;
  struct { ExpertTile tile; int rows, cols, step_cycles; int64_t units; } const choices[] = {
      {ExpertTile::kPair256, 256, 256, 512, sms / 2},
      {ExpertTile::kPair128, 256, 128, 384, sms / 2},
      {ExpertTile::kOne128, 128, 128, 512, sms},
      {ExpertTile::kOne64, 128, 64, 384, sms},
  };
  ExpertTile best = ExpertTile::kOne64;
  int64_t least = INT64_MAX;
  for (const auto& c : choices) {
    const int64_t tiles = experts * ((m + c.rows - 1) / c.rows) * ((n + c.cols - 1) / c.cols);
    const int64_t cost = (tiles + c.units - 1) / c.units * (steps * c.step_cycles + 1500);
    if (cost < least) {
      least = cost;
      best = c.tile;
    }
  }
  return best;
}

int product(const ExpertGemm& g, void* maps, int32_t* status, cudaStream_t s) {
  if (g.dtype == SV_FLOAT32) {
    const int rc = expert_gemm_f32(g, s);
    if (rc != SV_OK || !g.zero_rest) return rc;
    const Routing r{nullptr, g.offsets, nullptr, nullptr, 0, 1, g.experts, g.slots};
    expert_rest_kernel<float><<<num_sms(), 256, 0, s>>>(r, g.n, static_cast<float*>(g.ep.out));
    SV_LAUNCH_CHECK();
    return SV_OK;
  }
  const int64_t share = std::max<int64_t>(1, g.slots / g.experts);
  const int64_t busy = std::min<int64_t>(g.experts, g.slots);
  const ExpertTile tile = g.form == ExpertForm::kWeights ? pick_tile(g.experts, g.m, g.n, share)
                                                         : pick_tile(busy, share, g.n, g.k);
  return expert_gemm_tc(g, tile, maps, status, s);
}

struct Layout {
  size_t x, w, rows, dz, partial, raise, maps, total;
  int64_t ldx, ldw, ld_dz;
  int64_t pieces;
};

bool few(const sv_expert_args& g) {
  return g.n * g.k <= (g.dtype == SV_FLOAT32 ? FEW_SLOTS_F32 : FEW_SLOTS) || g.inputs == 0;
}
bool pad_x(const sv_expert_args& g) {
  return g.gather || (g.dtype != SV_FLOAT32 && !ready(g.x, g.ldx, g.dtype));
}
bool pad_w(const sv_expert_args& g) {
  return g.dtype != SV_FLOAT32 &&
         (!ready(g.weight, g.ldw, g.dtype) || g.w_expert * elem_size(g.dtype) % 16 != 0);
}

Layout forward_layout(const sv_expert_args& g) {
  Layout l{};
  const size_t es = elem_size(g.dtype);
  const int64_t slots = g.n * g.k;
  l.ldx = padded(g.inputs, g.dtype);
  l.ldw = padded(g.inputs, g.dtype);
  size_t at = 0;
  l.x = at;
  if (!few(g) && pad_x(g)) at += align_up(slots * l.ldx * es, ALIGN);
  l.w = at;
  if (!few(g) && pad_w(g)) at += align_up((size_t)g.experts * g.outputs * l.ldw * es, ALIGN);
  l.total = at;
  return l;
}

Layout backward_layout(const sv_expert_args& g, bool want_dx, bool want_dw, bool hold) {
  Layout l{};
  const size_t es = elem_size(g.dtype);
  const int64_t slots = g.n * g.k;
  l.ldx = l.ldw = padded(g.inputs, g.dtype);
  l.ld_dz = hold ? padded(g.outputs, g.dtype) : g.outputs;
  l.pieces = slots / DZ_ROWS + g.experts;
  size_t at = 0;
  l.dz = at;
  if (hold) at += align_up(slots * l.ld_dz * es, ALIGN);
  l.partial = at;
  at += align_up((size_t)l.pieces * g.outputs * sizeof(float), ALIGN);
  l.raise = at;
  if (hold && g.dtype == SV_FLOAT16) at += ALIGN + align_up(g.inputs * sizeof(float), ALIGN);
  l.maps = at;
  if (want_dw && g.dtype != SV_FLOAT32) at += align_up(expert_maps_bytes(g.experts), ALIGN);
  l.w = at;
  if (want_dx && pad_w(g)) at += align_up((size_t)g.experts * g.outputs * l.ldw * es, ALIGN);
  // the gathered x is read by dW only and dx in the order of the experts is written after it
  l.x = l.rows = at;
  size_t shared = 0;
  if (want_dw && pad_x(g)) shared = slots * l.ldx * es;
  if (want_dx && g.gather) shared = std::max(shared, (size_t)(slots * g.inputs) * sizeof(float));
  l.total = at + align_up(shared, ALIGN);
  return l;
}

int pad_weights(const sv_expert_args& g, void* out, int64_t ld_out, cudaStream_t s) {
  const int64_t items = (int64_t)g.experts * g.outputs * (ld_out / 8);
  if (items == 0) return SV_OK;
  expert_pad_kernel<uint16_t><<<grid_for(items, 16), 256, 0, s>>>(
      static_cast<const uint16_t*>(g.weight), g.ldw, g.w_expert, g.outputs, g.inputs, items,
      static_cast<uint16_t*>(out), ld_out);
  SV_LAUNCH_CHECK();
  return SV_OK;
}

int check_args(const sv_expert_args* g, const char* what) {
  const std::string at = what;
  if (!g) SV_FAIL(SV_ERR_INVALID_ARGUMENT, at + ": null arguments");
  if (g->n < 0 || g->k < 1 || g->experts < 1 || g->inputs < 0 || g->outputs < 0)
    SV_FAIL(SV_ERR_INVALID_ARGUMENT, at + ": bad size");
  if (!float_type(g->dtype)) SV_FAIL(SV_ERR_BAD_DTYPE, at + ": unknown dtype");
  if (g->activation < SV_ACT_NONE || g->activation > SV_ACT_GELU_TANH)
    SV_FAIL(SV_ERR_INVALID_ARGUMENT, at + ": unknown activation");
  if (g->experts > EXPERT_MAX)
    SV_FAIL(SV_ERR_UNSUPPORTED, at + ": more than " + std::to_string(EXPERT_MAX) + " experts");
  if (g->n > INT32_MAX / g->k - 1024 || g->inputs > INT32_MAX - 256 || g->outputs > INT32_MAX - 256)
    SV_FAIL(SV_ERR_UNSUPPORTED, at + ": sizes must be below 2^31 - 256");
  if (g->ldx < g->inputs || g->ldw < g->inputs || g->w_expert < 0)
    SV_FAIL(SV_ERR_INVALID_ARGUMENT, at + ": row stride below the row length");
  return SV_OK;
}

template <typename T, int V>
int launch_dz(const DzArgs& a, int act, dim3 grid, cudaStream_t s) {
  auto kernel = act == SV_ACT_SILU        ? expert_dz_kernel<T, V, SV_ACT_SILU>
                : act == SV_ACT_GELU      ? expert_dz_kernel<T, V, SV_ACT_GELU>
                : act == SV_ACT_GELU_TANH ? expert_dz_kernel<T, V, SV_ACT_GELU_TANH>
                                          : expert_dz_kernel<T, V, SV_ACT_NONE>;
  kernel<<<grid, 256, 0, s>>>(a);
  SV_LAUNCH_CHECK();
  return SV_OK;
}

template <typename T>
int elementwise_back(const sv_expert_args& g, const DzArgs& a, int64_t pieces, const void* dy,
                     float* dweights, void* dbias, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  if (dweights) {
    const bool wide = g.outputs % V == 0 && aligned16(dy) && aligned16(g.rows);
    const unsigned blocks = grid_for(a.r.slots * 32, 16);
    if (wide)
      expert_dweights_kernel<T, V><<<blocks, 256, 0, s>>>(
          static_cast<const T*>(dy), g.rows, a.r, g.outputs, dweights);
    else
      expert_dweights_kernel<T, 1><<<blocks, 256, 0, s>>>(
          static_cast<const T*>(dy), g.rows, a.r, g.outputs, dweights);
    SV_LAUNCH_CHECK();
  }
  if (!a.dz && !a.partial) return SV_OK;
  const bool wide = g.outputs % V == 0 && aligned16(dy) && (!a.preact || aligned16(a.preact));
  const int64_t across = (g.outputs + 32 * (wide ? V : 1) - 1) / (32 * (wide ? V : 1));
  if (across > 65535) SV_FAIL(SV_ERR_UNSUPPORTED, "expert_linear: too many outputs");
  const dim3 grid((unsigned)pieces, (unsigned)across);
  const int act = a.preact ? g.activation : (int)SV_ACT_NONE;
  const int rc = wide ? launch_dz<T, V>(a, act, grid, s) : launch_dz<T, 1>(a, act, grid, s);
  if (rc != SV_OK || !dbias) return rc;
  const dim3 columns((unsigned)((g.outputs + 31) / 32), (unsigned)g.experts);
  expert_dbias_kernel<T><<<columns, 256, 0, s>>>(a.partial, a.r, g.outputs, static_cast<T*>(dbias));
  SV_LAUNCH_CHECK();
  return SV_OK;
}

}  // namespace
}  // namespace sv

using namespace sv;

extern "C" size_t sv_expert_linear_workspace_bytes(const sv_expert_args* args, int pass, int want_dx,
                                                   int want_dw, const void* dout) {
  if (check_args(args, "sv_expert_linear_workspace_bytes") != SV_OK) return 0;
  if (pass == SV_LINEAR_FORWARD) return forward_layout(*args).total;
  const bool hold = args->combine || args->activation != SV_ACT_NONE ||
                    (args->dtype != SV_FLOAT32 && !ready(dout, args->outputs, args->dtype));
  return backward_layout(*args, want_dx != 0, want_dw != 0, hold).total;
}

extern "C" int sv_expert_linear(const sv_expert_args* args, void* out, void* workspace,
                                size_t workspace_bytes, int32_t* status, sv_stream_t stream) {
  const int rc = check_args(args, "sv_expert_linear");
  if (rc != SV_OK) return rc;
  const sv_expert_args& g = *args;
  const Routing r = routing_of(g);
  if (g.n == 0 || g.outputs == 0) return SV_OK;
  void* rows = g.combine ? g.rows : out;
  if (!out || !rows || !r.offsets || (g.gather && !r.order) ||
      (g.combine && (!r.place || !r.weights)) || (g.inputs > 0 && (!g.x || !g.weight)))
    SV_FAIL(SV_ERR_INVALID_ARGUMENT, "sv_expert_linear: null pointer");
  const Layout l = forward_layout(g);
  if (l.total && (!workspace || workspace_bytes < l.total || !aligned16(workspace)))
    SV_FAIL(SV_ERR_WORKSPACE, "sv_expert_linear: workspace too small or unaligned");
  cudaStream_t s = to_stream(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const Epilogue ep{g.bias, nullptr, 0, nullptr, nullptr, rows, g.preact, nullptr,
                    g.combine ? (int)SV_FLOAT32 : g.dtype, g.activation};
  int bad;
  if (few(g)) {
    bad = g.dtype == SV_FLOAT32   ? few_typed<float>(g, r, ep, status, s)
          : g.dtype == SV_FLOAT16 ? few_typed<__half>(g, r, ep, status, s)
                                  : few_typed<__nv_bfloat16>(g, r, ep, status, s);
  } else {
    ExpertGemm e{};
    e.form = ExpertForm::kRows;
    e.a = {g.x, g.ldx, false};
    e.b = {g.weight, g.ldw, false};
    e.b_expert = g.w_expert;
    e.offsets = r.offsets;
    e.experts = g.experts;
    e.slots = r.slots;
    e.n = g.outputs;
    e.k = g.inputs;
    e.dtype = g.dtype;
    e.zero_rest = !g.combine;
    e.runs = g.combine > 1;
    e.ep = ep;
    if (g.inputs > 0 && pad_x(g)) {
      bad = gather_rows(g.x, g.ldx, r, g.gather != 0, g.inputs, g.dtype, ws + l.x, l.ldx, status, s);
      if (bad != SV_OK) return bad;
      e.a = {ws + l.x, l.ldx, false};
    }
    if (g.inputs > 0 && pad_w(g)) {
      bad = pad_weights(g, ws + l.w, l.ldw, s);
      if (bad != SV_OK) return bad;
      e.b = {ws + l.w, l.ldw, false};
      e.b_expert = (int64_t)g.outputs * l.ldw;
    }
    bad = product(e, nullptr, status, s);
  }
  if (bad != SV_OK || !g.combine) return bad;
  return combine(g.rows, r, true, g.outputs, g.dtype, out, s);
}

extern "C" int sv_expert_linear_backward(const sv_expert_args* args, const void* dout, void* dx,
                                         void* dweight, void* dbias, float* dweights,
                                         void* workspace, size_t workspace_bytes, int32_t* status,
                                         sv_stream_t stream) {
  const int rc = check_args(args, "sv_expert_linear_backward");
  if (rc != SV_OK) return rc;
  const sv_expert_args& g = *args;
  const Routing r = routing_of(g);
  cudaStream_t s = to_stream(stream);
  const size_t es = elem_size(g.dtype);
  const bool terms = r.slots > 0 && g.outputs > 0;
  if (r.slots == 0 || g.inputs == 0) dx = nullptr;
  if (g.outputs == 0 || g.inputs == 0) dweight = nullptr;
  if (g.outputs == 0) dbias = nullptr;
  if (r.slots == 0 || !g.combine) dweights = nullptr;
  if (!dx && !dweight && !dbias && !dweights) return SV_OK;
  if (!terms) {
    const int64_t rows = g.gather ? g.n : r.slots;
    if (dx) SV_CUDA_TRY(cudaMemsetAsync(dx, 0, rows * g.inputs * es, s));
    if (dweight) SV_CUDA_TRY(cudaMemsetAsync(dweight, 0, (size_t)g.experts * g.outputs * g.inputs * es, s));
    if (dbias) SV_CUDA_TRY(cudaMemsetAsync(dbias, 0, (size_t)g.experts * g.outputs * es, s));
    if (dweights) SV_CUDA_TRY(cudaMemsetAsync(dweights, 0, r.slots * sizeof(float), s));
    return SV_OK;
  }
  const bool act = g.activation != SV_ACT_NONE;
  if (!dout || !r.offsets || !r.order || !r.place || (g.combine && !r.weights) ||
      (act && !g.preact) || (dweights && !g.rows) || (dx && !g.weight) || (dweight && !g.x))
    SV_FAIL(SV_ERR_INVALID_ARGUMENT, "sv_expert_linear_backward: null pointer");
  const bool hold = g.combine || act || (g.dtype != SV_FLOAT32 && !ready(dout, g.outputs, g.dtype));
  const Layout l = backward_layout(g, dx != nullptr, dweight != nullptr, hold);
  if (!workspace || workspace_bytes < l.total || !aligned16(workspace) ||
      (reinterpret_cast<uintptr_t>(workspace) & 127u) != 0)
    SV_FAIL(SV_ERR_WORKSPACE, "sv_expert_linear_backward: workspace too small or unaligned");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  DzArgs a{};
  a.r = r;
  a.dy = dout;
  a.preact = act ? g.preact : nullptr;
  a.combine = g.combine != 0;
  a.cols = g.outputs;
  a.dz = hold && (dx || dweight) ? ws + l.dz : nullptr;
  a.ld_dz = l.ld_dz;
  a.partial = dbias ? reinterpret_cast<float*>(ws + l.partial) : nullptr;
  if (a.dz && (act || g.combine) && g.dtype == SV_FLOAT16) {
    a.raise = {reinterpret_cast<unsigned*>(ws + l.raise),
               reinterpret_cast<float*>(ws + l.raise + ALIGN), g.inputs};
    const int bad = g.combine ? find_top<true>(dout, g.n * g.outputs, g.weights, r.slots, a.raise.top, s)
                              : find_top<true>(dout, r.slots * g.outputs, nullptr, 0, a.raise.top, s);
    if (bad != SV_OK) return bad;
  }
  int bad = g.dtype == SV_FLOAT32
                ? elementwise_back<float>(g, a, l.pieces, dout, dweights, dbias, s)
            : g.dtype == SV_FLOAT16
                ? elementwise_back<__half>(g, a, l.pieces, dout, dweights, dbias, s)
                : elementwise_back<__nv_bfloat16>(g, a, l.pieces, dout, dweights, dbias, s);
  if (bad != SV_OK) return bad;
  const void* dz = hold ? ws + l.dz : dout;
  ExpertGemm e{};
  e.offsets = r.offsets;
  e.experts = g.experts;
  e.slots = r.slots;
  e.dtype = g.dtype;
  if (dweight) {
    e.form = ExpertForm::kWeights;
    e.a = {dz, l.ld_dz, true};
    e.b = {g.x, g.ldx, true};
    if (pad_x(g)) {
      bad = gather_rows(g.x, g.ldx, r, g.gather != 0, g.inputs, g.dtype, ws + l.x, l.ldx, status, s);
      if (bad != SV_OK) return bad;
      e.b = {ws + l.x, l.ldx, true};
    }
    e.m = g.outputs;
    e.n = g.inputs;
    e.ep = {nullptr, nullptr, 0, nullptr, a.raise.down, dweight, nullptr, nullptr, g.dtype, SV_ACT_NONE};
    bad = product(e, ws + l.maps, status, s);
    if (bad != SV_OK) return bad;
  }
  if (!dx) return SV_OK;
  void* rows = g.gather ? ws + l.rows : dx;
  e.form = ExpertForm::kRows;
  e.a = {dz, l.ld_dz, false};
  e.b = {g.weight, g.ldw, true};
  e.b_expert = g.w_expert;
  if (pad_w(g)) {
    bad = pad_weights(g, ws + l.w, l.ldw, s);
    if (bad != SV_OK) return bad;
    e.b = {ws + l.w, l.ldw, true};
    e.b_expert = (int64_t)g.outputs * l.ldw;
  }
  e.n = g.inputs;
  e.k = g.outputs;
  e.zero_rest = !g.gather;
  e.ep = {nullptr, nullptr, 0, nullptr, a.raise.down, rows, nullptr, nullptr,
          g.gather ? (int)SV_FLOAT32 : g.dtype, SV_ACT_NONE};
  bad = product(e, nullptr, status, s);
  if (bad != SV_OK || !g.gather) return bad;
  return combine(static_cast<const float*>(rows), r, false, g.inputs, g.dtype, dx, s);
}
