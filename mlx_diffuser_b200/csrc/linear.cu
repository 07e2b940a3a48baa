// Linear projection of feature rows with bias, activation and residual in its epilogue, and its
// gradients.
//
//     z = x W^T [* x_scale[i] * w_scale[j]] + b        x [m, k], W [n, k]
//     y = act(z) + residual
//     dz = dy * act'(z),  db = column sums of dz,  dx = dz W,  dW = dz^T x
//
// Three kernels form the products:
//   few_rows_kernel   up to FEW_ROWS rows (any type): one pass over W, which is all the bytes
//                     there are; a warp or a block per output column;
//   gemm_f32_kernel   fp32: register tiles of FFMAs, exact fp32 products and sums;
//   linear_tc.cu      fp16 / bf16 / e4m3: tcgen05 tiles fed by TMA.
// A product with too few tiles to fill the machine splits its k axis; the parts' fp32 sums are
// joined in a fixed order by finish_kernel, which then applies the epilogue. TMA wants 16-byte
// aligned rows: an operand that has none (an odd channel count, a sliced view) is first copied
// into padded rows in the workspace, one pass over it.
#include <cuda_fp8.h>

#include <algorithm>
#include <type_traits>

#include "linear.h"

namespace sv {
namespace {

constexpr int FEW_ROWS = 8;
constexpr int COPY_ALIGN = 256;

__device__ __forceinline__ float to_float(__nv_fp8_e4m3 v) { return static_cast<float>(v); }
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// ---- few rows ----------------------------------------------------------------------------------

// W warps per output column (1: eight columns a block, 8: one), lanes along k in accesses of V
// elements. Every lane holds the partial sums of all rows; x comes out of L1, all rows' accesses in
// flight together (rows past the last read it again: behind a branch each waited for the one
// before, 8 x 2048 -> 2048 bf16 19 us).
template <typename T, typename O, int ROWS, int V, int W>
__global__ void __launch_bounds__(256)
    few_rows_kernel(const T* __restrict__ x, int64_t ldx, const T* __restrict__ w, int64_t ldw,
                    int m, int64_t n, int64_t k, Epilogue ep) {
  __shared__ float part[W > 1 ? 8 : 1][ROWS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t j = W > 1 ? blockIdx.x : (int64_t)blockIdx.x * 8 + warp;
  const int slot = W > 1 ? (int)threadIdx.x : lane;
  float acc[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) acc[r] = 0.f;
  if (j < n) {
    const T* wr = w + j * ldw;
#pragma unroll 2
    for (int64_t c = (int64_t)slot * V; c < k; c += 32 * W * V) {
      T we[V];
      if constexpr (V * sizeof(T) == 16)
        *reinterpret_cast<uint4*>(we) = __ldg(reinterpret_cast<const uint4*>(wr + c));
      else
        we[0] = wr[c];
      alignas(16) T xe[ROWS][V];
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        const T* from = x + min(r, m - 1) * ldx + c;
        if constexpr (V * sizeof(T) == 16)
          *reinterpret_cast<uint4*>(xe[r]) = __ldg(reinterpret_cast<const uint4*>(from));
        else
          xe[r][0] = *from;
      }
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int e = 0; e < V; ++e) acc[r] = fmaf(to_float(xe[r][e]), to_float(we[e]), acc[r]);
    }
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc[r] += __shfl_xor_sync(0xffffffffu, acc[r], o);
  }
  if constexpr (W > 1) {
    if (lane == 0) {
#pragma unroll
      for (int r = 0; r < ROWS; ++r) part[warp][r] = acc[r];
    }
    __syncthreads();
    if (threadIdx.x < ROWS && (int)threadIdx.x < m) {
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) v += part[i][threadIdx.x];
      epilogue_store<O>(ep, threadIdx.x, j, n, v);
    }
  } else if (j < n) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
      if (lane == r && r < m) epilogue_store<O>(ep, r, j, n, acc[r]);
  }
}

template <typename T, typename O, int ROWS>
int launch_few(const Gemm& g, cudaStream_t s) {
  constexpr int VE = 16 / sizeof(T);
  const T* x = static_cast<const T*>(g.a.p);
  const T* w = static_cast<const T*>(g.b.p);
  const bool vec = aligned16(x) && aligned16(w) && g.k % VE == 0 && g.a.ld % VE == 0 &&
                   g.b.ld % VE == 0;
  // A warp per column needs n / 8 blocks to cover the machine; below that a block per column
  // brings eight times the loads in flight.
  const bool wide = g.n >= 8 * num_sms();
  const unsigned blocks = (unsigned)(wide ? (g.n + 7) / 8 : g.n);
  auto kernel = vec ? (wide ? few_rows_kernel<T, O, ROWS, VE, 1> : few_rows_kernel<T, O, ROWS, VE, 8>)
                    : (wide ? few_rows_kernel<T, O, ROWS, 1, 1> : few_rows_kernel<T, O, ROWS, 1, 8>);
  kernel<<<blocks, 256, 0, s>>>(x, g.a.ld, w, g.b.ld, (int)g.m, g.n, g.k, g.ep);
  SV_LAUNCH_CHECK();
  return SV_OK;
}

template <typename T, typename O>
int few_typed(const Gemm& g, cudaStream_t s) {
  if (g.m <= 1) return launch_few<T, O, 1>(g, s);
  if (g.m <= 2) return launch_few<T, O, 2>(g, s);
  if (g.m <= 4) return launch_few<T, O, 4>(g, s);
  return launch_few<T, O, FEW_ROWS>(g, s);
}

int gemm_few(const Gemm& g, cudaStream_t s) {
  switch (g.dtype) {
    case SV_FLOAT32: return few_typed<float, float>(g, s);
    case SV_FLOAT16: return few_typed<__half, __half>(g, s);
    case SV_BFLOAT16: return few_typed<__nv_bfloat16, __nv_bfloat16>(g, s);
    default:
      return g.ep.out_dtype == SV_FLOAT16 ? few_typed<__nv_fp8_e4m3, __half>(g, s)
                                          : few_typed<__nv_fp8_e4m3, __nv_bfloat16>(g, s);
  }
}

// ---- fp32 tiles --------------------------------------------------------------------------------

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

// C tile of 16 R x 16 R, 256 threads with R x R sums each (R / 4 groups of four rows and columns,
// 64 apart, so that the shared-memory reads are 16-byte and conflict-free). VA, VB: elements of an
// access to each operand. 12,001 x 1024 x 1024, the three products of a training step: 668 us on
// average (37.7 TFLOP/s; two blocks an SM, 2.5 rounds of tiles), 755 us with one multiply-add an
// instruction, and 1,127 us element by element with one block an SM. The library's fp32 product: 455.
template <int R, int VA, int VB>
__global__ void __launch_bounds__(256, 2)
    gemm_f32_kernel(Operand a, Operand b, int64_t m, int64_t n, int64_t k, int64_t k_part,
                    Epilogue ep) {
  constexpr int T = 16 * R;
  using SA = Stage<T, VA>;
  using SB = Stage<T, VB>;
  __shared__ __align__(16) float sa[2][FK][T + 4];
  __shared__ __align__(16) float sb[2][FK][T + 4];
  const int tid = threadIdx.x;
  const int tx = tid % 16, ty = tid / 16;
  // columns vary fastest: blocks that run together share the rows of A
  const unsigned across = (unsigned)((n + T - 1) / T);
  const int64_t i0 = (int64_t)(blockIdx.x / across) * T, j0 = (int64_t)(blockIdx.x % across) * T;
  const int64_t k0 = (int64_t)blockIdx.y * k_part;
  const int64_t k1 = k0 + k_part < k ? k0 + k_part : k;
  float ra[SA::PER], rb[SB::PER];
  uint64_t acc[R][R / 2];  // two neighbouring columns each
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
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int64_t row = i0 + 64 * (i / 4) + 4 * ty + i % 4;
    if (row >= m) continue;
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const int64_t col = j0 + 64 * (j / 4) + 4 * tx + j % 4;
      if (col >= n) continue;
      const float v = __uint_as_float((uint32_t)(acc[i][j / 2] >> (j % 2 * 32)));
      if (ep.partial)
        ep.partial[((int64_t)blockIdx.y * m + row) * n + col] = v;
      else
        epilogue_store<float>(ep, row, col, n, v);
    }
  }
}

template <int R>
void launch_f32(const Gemm& g, dim3 grid, int64_t k_part, cudaStream_t s) {
  const bool va = aligned16(g.a.p) && g.a.ld % 4 == 0, vb = aligned16(g.b.p) && g.b.ld % 4 == 0;
  auto kernel = va ? (vb ? gemm_f32_kernel<R, 4, 4> : gemm_f32_kernel<R, 4, 1>)
                   : (vb ? gemm_f32_kernel<R, 1, 4> : gemm_f32_kernel<R, 1, 1>);
  kernel<<<grid, 256, 0, s>>>(g.a, g.b, g.m, g.n, g.k, k_part, g.ep);
}

int gemm_f32(const Gemm& g, bool small, cudaStream_t s) {
  const int tile = small ? 64 : 128;
  const int64_t k_part = (((g.k + g.splits - 1) / g.splits + FK - 1) / FK) * FK;
  const int64_t tiles = ((g.m + tile - 1) / tile) * ((g.n + tile - 1) / tile);
  if (tiles > INT32_MAX) SV_FAIL(SV_ERR_UNSUPPORTED, "linear: too many tiles");
  const dim3 grid((unsigned)tiles, (unsigned)g.splits);
  if (small)
    launch_f32<4>(g, grid, k_part, s);
  else
    launch_f32<8>(g, grid, k_part, s);
  SV_LAUNCH_CHECK();
  return SV_OK;
}

// ---- second passes -----------------------------------------------------------------------------

// Adds the parts of a split product in order and applies the epilogue (no parts: sums of zero), V
// consecutive columns a thread. V 4: n a multiple of 4 and every pointer on its boundary. One MB of
// bf16 sums out of 16 parts took 9.3 us an element a thread and 5.6 us four.
template <typename O, int V>
__global__ void __launch_bounds__(256)
    finish_kernel(const float* __restrict__ partial, int splits, int64_t m, int64_t n,
                  Epilogue ep) {
  const int64_t cells = m * n;
  for (int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V; at < cells;
       at += (int64_t)gridDim.x * 256 * V) {
    float v[V];
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = 0.f;
#pragma unroll 8
    for (int p = 0; p < splits; ++p) {
      const float* from = partial + p * cells + at;
      if constexpr (V == 4) {
        const float4 x = __ldg(reinterpret_cast<const float4*>(from));
        v[0] += x.x;
        v[1] += x.y;
        v[2] += x.z;
        v[3] += x.w;
      } else {
        v[0] += __ldg(from);
      }
    }
    const int64_t i = at / n, j = at - i * n;
    if constexpr (V == 4) {
      if (!ep.bias && !ep.residual && !ep.preact && !ep.row_scale && !ep.col_scale &&
          ep.act == SV_ACT_NONE) {
        alignas(16) O out[V];
#pragma unroll
        for (int e = 0; e < V; ++e) out[e] = from_f32<O>(v[e]);
        O* dst = static_cast<O*>(ep.out) + at;
        if constexpr (sizeof(O) == 4)
          *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(out);
        else
          *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(out);
        continue;
      }
    }
#pragma unroll
    for (int e = 0; e < V; ++e) epilogue_store<O>(ep, i, j + e, n, v[e]);
  }
}

template <typename O>
int finish_typed(const Gemm& g, const Epilogue& ep, const float* partial, int splits,
                 cudaStream_t s) {
  // `partial` is the start of a workspace, its parts m * n floats apart
  const bool wide = g.n % 4 == 0 && aligned16(partial) && aligned16(ep.out);
  const int64_t items = g.m * g.n / (wide ? 4 : 1);
  const unsigned blocks =
      (unsigned)std::min<int64_t>((items + 255) / 256, (int64_t)num_sms() * 8);
  if (wide)
    finish_kernel<O, 4><<<blocks, 256, 0, s>>>(partial, splits, g.m, g.n, ep);
  else
    finish_kernel<O, 1><<<blocks, 256, 0, s>>>(partial, splits, g.m, g.n, ep);
  SV_LAUNCH_CHECK();
  return SV_OK;
}

int finish(const Gemm& g, const float* partial, int splits, cudaStream_t s) {
  Epilogue ep = g.ep;
  ep.partial = nullptr;
  switch (ep.out_dtype) {
    case SV_FLOAT32: return finish_typed<float>(g, ep, partial, splits, s);
    case SV_FLOAT16: return finish_typed<__half>(g, ep, partial, splits, s);
    default: return finish_typed<__nv_bfloat16>(g, ep, partial, splits, s);
  }
}

// Operands whose rows TMA cannot read, into rows of a multiple of 16 bytes: up to two in one launch,
// in elements of E. A thread gathers 16 bytes of a row, element by element, and stores them at once
// (5,041 x 331 fp16: 9.0 us an element a thread).
struct Pad {
  const void* in;
  int64_t rows, words, ld_in;
  void* out;
  int64_t ld_out;
};

template <typename E>
__global__ void __launch_bounds__(256) pad_rows_kernel(Pad first, Pad second) {
  constexpr int W = 16 / sizeof(E);
  const Pad& p = blockIdx.y ? second : first;
  const E* in = static_cast<const E*>(p.in);
  const int64_t across = p.ld_out / W, total = p.rows * across;
  for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < total;
       at += (int64_t)gridDim.x * 256) {
    const int64_t r = total <= UINT32_MAX ? (uint32_t)at / (uint32_t)across : at / across;
    const int64_t c = (at - r * across) * W;
    const E* from = in + r * p.ld_in + c;
    alignas(16) E e[W];
#pragma unroll
    for (int i = 0; i < W; ++i) e[i] = c + i < p.words ? __ldg(from + i) : E(0);
    *reinterpret_cast<uint4*>(static_cast<E*>(p.out) + r * p.ld_out + c) =
        *reinterpret_cast<const uint4*>(e);
  }
}

int pad_rows(const Pad* pads, int count, int es, cudaStream_t s) {
  int64_t most = 0;
  for (int i = 0; i < count; ++i)
    most = std::max(most, pads[i].rows * (pads[i].ld_out * es / 16));
  const dim3 grid((unsigned)std::min<int64_t>((most + 255) / 256, (int64_t)num_sms() * 16),
                  (unsigned)count);
  const Pad& second = pads[count - 1];
  if (es == 2)
    pad_rows_kernel<uint16_t><<<grid, 256, 0, s>>>(pads[0], second);
  else
    pad_rows_kernel<uint8_t><<<grid, 256, 0, s>>>(pads[0], second);
  SV_LAUNCH_CHECK();
  return SV_OK;
}

// dz is rounded to the feature type, since the tensor cores take it as an operand of both products: half
// a step more beside the result's own (0.0023 against 0.0017 over the gradients of 12,001 x 1024 x 1024
// bf16). fp16's is raised by a power of two first, and the products' column scales take that back: below 2^-14 a half has no 11 bits, and the gradients of a mean loss lie there. The power puts the
// largest |dy| below 2^15 (the activations' slopes are below 1.13), so values down to 2^-28 of it keep
// all their bits. It costs a pass over dy: 12,001 x 1024 in 7 us.
struct Raise {
  unsigned* top;  // bits of the largest |dy|, as a half; null: dz is not raised
  float* down;    // [k]: what the products are multiplied by
  int64_t k;
};
__device__ __forceinline__ float raise_of(unsigned top) {
  if (top == 0u || top >= 0x7c00u) return 1.0f;  // nothing, or not a number
  const float x = __half2float(__ushort_as_half((unsigned short)top));
  return __uint_as_float((268u - (__float_as_uint(x) >> 23)) << 23);  // 2^14 <= x * this < 2^15
}

template <int V>
__global__ void __launch_bounds__(256)
    top_kernel(const unsigned short* __restrict__ x, int64_t cells, unsigned* __restrict__ top) {
  unsigned most = 0u;  // of both halves of a word
  const int64_t step = (int64_t)gridDim.x * 256 * V;
#pragma unroll 4
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V; i < cells; i += step) {
    if constexpr (V == 8) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(x + i));
      most = __vmaxu2(most, __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu),
                                     __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu)));
    } else {
      most = __vmaxu2(most, x[i] & 0x7fffu);
    }
  }
  __shared__ unsigned s_top[8];
  const unsigned one = __reduce_max_sync(0xffffffffu, max(most & 0xffffu, most >> 16));
  if ((threadIdx.x & 31) == 0) s_top[threadIdx.x >> 5] = one;
  __syncthreads();
  if (threadIdx.x < 32) {  // one atomic a block: one a warp took 11 us
    const unsigned all = __reduce_max_sync(0xffffffffu, threadIdx.x < 8 ? s_top[threadIdx.x] : 0u);
    if (threadIdx.x == 0 && all) atomicMax(top, all);
  }
}

// dz = dy * act'(z), rows `ld` apart, and the column sums of dz: a block takes 32 V columns (V to a
// thread) of a strip of rows, eight rows at a time, and writes one row of `partial` for its strip.
// dz and partial may be null. A pass over 8 bytes of bf16 and fp32 an element (12,001 x 1024: 18 us,
// 5.5 TB/s): six blocks an SM with two rows each in flight; three with four rows took 28 us.
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(256, 6)
    dz_kernel(const T* __restrict__ dy, const float* __restrict__ z, int64_t m, int64_t n,
              int64_t rows_per_strip, T* __restrict__ dz, int64_t ld, float* __restrict__ partial,
              Raise raise) {
  __shared__ float s_sum[8][32 * V + 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = ((int64_t)blockIdx.x * 32 + lane) * V;
  const int64_t r0 = (int64_t)blockIdx.y * rows_per_strip;
  const int64_t r1 = r0 + rows_per_strip < m ? r0 + rows_per_strip : m;
  float sum[V];
#pragma unroll
  for (int e = 0; e < V; ++e) sum[e] = 0.f;
  float up = 1.0f;
  if constexpr (std::is_same<T, __half>::value) {
    if (raise.top != nullptr) {
      up = raise_of(__ldg(raise.top));
      if (blockIdx.x == 0 && blockIdx.y == 0)
        for (int64_t i = threadIdx.x; i < raise.k; i += 256) raise.down[i] = 1.0f / up;
    }
  }
  if (c < n) {
#pragma unroll 2
    for (int64_t r = r0 + warp; r < r1; r += 8) {
      alignas(16) T d[V];
      alignas(16) float zz[V];
      auto fetch = [](auto* to, const auto* from) {
        if constexpr (V * sizeof(T) == 8)
          *reinterpret_cast<uint2*>(to) = __ldg(reinterpret_cast<const uint2*>(from));
        else if constexpr (V * sizeof(T) == 16)
          *reinterpret_cast<uint4*>(to) = __ldg(reinterpret_cast<const uint4*>(from));
        else
          to[0] = from[0];
      };
      fetch(d, dy + r * n + c);
      if constexpr (ACT == SV_ACT_NONE) {
#pragma unroll
        for (int e = 0; e < V; ++e) sum[e] += to_float(d[e]);
      } else {
        if constexpr (V == 4)
          *reinterpret_cast<float4*>(zz) = __ldg(reinterpret_cast<const float4*>(z + r * n + c));
        else
          zz[0] = z[r * n + c];
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float v = to_float(d[e]) * (sizeof(T) == 2 ? activate_slope_half(zz[e], ACT)
                                                           : activate_slope(zz[e], ACT));
          sum[e] += v;
          d[e] = from_f32<T>(v * up);
        }
      }
      if (dz) {
        T* to = dz + r * ld + c;
        if constexpr (V * sizeof(T) == 8)
          *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(d);
        else if constexpr (V * sizeof(T) == 16)
          *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(d);
        else
          to[0] = d[0];
      }
    }
  }
  if (partial == nullptr) return;
#pragma unroll
  for (int e = 0; e < V; ++e) s_sum[warp][lane * V + e] = sum[e];
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * V; i += 256) {
    const int64_t col = (int64_t)blockIdx.x * 32 * V + i;
    if (col < n) {
      float v = s_sum[0][i];
#pragma unroll
      for (int w = 1; w < 8; ++w) v += s_sum[w][i];
      partial[(int64_t)blockIdx.y * n + col] = v;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256)
    dbias_kernel(const float* __restrict__ partial, int strips, int64_t n, T* __restrict__ out) {
  __shared__ float s[8][33];
  const int lane = threadIdx.x & 31, r0 = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  float v = 0.f;
  if (c < n)
    for (int r = r0; r < strips; r += 8) v += partial[(int64_t)r * n + c];
  s[r0][lane] = v;
  __syncthreads();
  if (r0 == 0 && c < n) {
#pragma unroll
    for (int i = 1; i < 8; ++i) v += s[i][lane];
    out[c] = from_f32<T>(v);
  }
}

constexpr int MAX_STRIPS = 888;

int strips_for(int64_t m, int64_t n, int v) {
  const int64_t across = (n + 32 * v - 1) / (32 * v);
  const int64_t want = std::max<int64_t>(1, MAX_STRIPS / across);
  return (int)std::min<int64_t>(want, (m + 7) / 8);
}

template <typename T, int V>
int launch_dz(const T* dy, const float* z, int64_t m, int64_t n, int act, T* dz, int64_t ld, T* db,
              float* partial, const Raise& raise, cudaStream_t s) {
  const int strips = strips_for(m, n, V);
  const int64_t per = (m + strips - 1) / strips;
  const dim3 grid((unsigned)((n + 32 * V - 1) / (32 * V)), (unsigned)strips);
  auto kernel = act == SV_ACT_SILU        ? dz_kernel<T, V, SV_ACT_SILU>
                : act == SV_ACT_GELU      ? dz_kernel<T, V, SV_ACT_GELU>
                : act == SV_ACT_GELU_TANH ? dz_kernel<T, V, SV_ACT_GELU_TANH>
                                          : dz_kernel<T, V, SV_ACT_NONE>;
  kernel<<<grid, 256, 0, s>>>(dy, z, m, n, per, dz, ld, db ? partial : nullptr, raise);
  SV_LAUNCH_CHECK();
  if (db) {
    dbias_kernel<T><<<(unsigned)((n + 31) / 32), 256, 0, s>>>(partial, strips, n, db);
    SV_LAUNCH_CHECK();
  }
  return SV_OK;
}

template <typename T>
int dz_typed(const void* dy, const float* z, int64_t m, int64_t n, int act, void* dz, int64_t ld,
             void* db, float* partial, const Raise& raise, cudaStream_t s) {
  if (raise.top) {
    SV_CUDA_TRY(cudaMemsetAsync(raise.top, 0, sizeof(unsigned), s));
    const unsigned short* x = static_cast<const unsigned short*>(dy);
    const int64_t cells = m * n;
    const bool wide = cells % 8 == 0 && aligned16(dy);
    const unsigned blocks = (unsigned)std::min<int64_t>(
        (cells / (wide ? 8 : 1) + 255) / 256, (int64_t)num_sms() * 8);
    if (wide) top_kernel<8><<<blocks, 256, 0, s>>>(x, cells, raise.top);
    else top_kernel<1><<<blocks, 256, 0, s>>>(x, cells, raise.top);
    SV_LAUNCH_CHECK();
  }
  const bool vec = n % 4 == 0 && aligned16(dy) && aligned16(z) && aligned16(dz);
  const T* g = static_cast<const T*>(dy);
  T *d = static_cast<T*>(dz), *b = static_cast<T*>(db);
  return vec ? launch_dz<T, 4>(g, z, m, n, act, d, ld, b, partial, raise, s)
             : launch_dz<T, 1>(g, z, m, n, act, d, ld, b, partial, raise, s);
}

// ---- the plan of one product -------------------------------------------------------------------

enum class Path { kEmpty, kFew, kF32, kTensor };

struct Plan {
  Path path;
  TcTile tile;  // tensor cores
  bool small;   // fp32: 64 x 64 tiles
  int splits;
  size_t partial_bytes;
};

// The operand's extent in memory: `rows` rows of `cols` consecutive elements.
struct Extent {
  int64_t rows, cols;
};
Extent extent(bool mn, int64_t outer, int64_t k) {
  return mn ? Extent{k, outer} : Extent{outer, k};
}

bool tma_ready(const Operand& o, int dtype) {
  return aligned16(o.p) && o.ld * elem_size(dtype) % 16 == 0;
}

size_t copy_bytes(const Extent& e, int dtype) {
  return align_up((size_t)e.rows * align_up((size_t)e.cols * elem_size(dtype), 16), COPY_ALIGN);
}

void set_splits(Plan* p, int64_t want, int64_t steps, int64_t m, int64_t n) {
  if (want <= 1) return;
  want = std::min<int64_t>(want, 64);
  const int64_t part = (steps + want - 1) / want;
  p->splits = (int)((steps + part - 1) / part);  // no part is empty
  if (p->splits > 1) p->partial_bytes = align_up((size_t)p->splits * m * n * 4, COPY_ALIGN);
}

Plan plan_gemm(int64_t m, int64_t n, int64_t k, int dtype, bool a_mn, bool b_mn) {
  Plan p{};
  p.splits = 1;
  if (m == 0 || n == 0 || k == 0) {
    p.path = Path::kEmpty;
    return p;
  }
  if (m <= FEW_ROWS && !a_mn && !b_mn) {
    p.path = Path::kFew;
    return p;
  }
  const int64_t sms = num_sms();
  if (dtype == SV_FLOAT32) {
    p.path = Path::kF32;
    // Tiles of 128 x 128 where they and the parts of a split k axis, each at least 4 steps of 64 long,
    // give every SM one; of 64 x 64 otherwise. 12,001 x 1024 x 1024, before the paired
    // multiply-adds: dW in parts took 812 us, in small tiles 855 us.
    const int64_t steps = (k + 4 * FK - 1) / (4 * FK), most = std::max<int64_t>(1, steps / 4);
    int64_t tiles = ((m + 127) / 128) * ((n + 127) / 128);
    p.small = tiles * most < sms;
    if (p.small) tiles = ((m + 63) / 64) * ((n + 63) / 64);
    if (tiles < sms) set_splits(&p, std::min((2 * sms + tiles - 1) / tiles, most), steps, m, n);
    return p;
  }
  p.path = Path::kTensor;
  // The tile and the split of the k axis with the least estimated time, in cycles: a 128-byte k step
  // costs the stage's bytes at the 64 bytes a cycle that an SM draws from L2, a round of tiles
  // its steps and about 1500 cycles to fill the pipeline and drain the accumulator, and a split
  // its fp32 sums written and read at about 3 KB a cycle, plus a launch.
  const int64_t steps = (k * elem_size(dtype) + 127) / 128;
  struct { TcTile tile; int rows, cols, step_cycles; int64_t units; } const choices[] = {
      {TcTile::kPair256, 256, 256, 512, sms / 2},
      {TcTile::kPair128, 256, 128, 384, sms / 2},
      {TcTile::kOne128, 128, 128, 512, sms},
      {TcTile::kOne64, 128, 64, 384, sms},
  };
  int64_t best = INT64_MAX, splits = 1;
  for (const auto& c : choices) {
    const int64_t tiles = ((m + c.rows - 1) / c.rows) * ((n + c.cols - 1) / c.cols);
    const int64_t most = tiles < c.units ? std::max<int64_t>(1, std::min(c.units / tiles, steps / 4)) : 1;
    for (int64_t parts = 1; parts <= most; parts = parts < most && parts * 2 > most ? most : parts * 2) {
      const int64_t rounds = (tiles * parts + c.units - 1) / c.units;
      int64_t cost = rounds * ((steps + parts - 1) / parts * c.step_cycles + 1500);
      if (parts > 1) cost += parts * m * n * 8 / 3000 + 4000;
      if (cost < best) {
        best = cost;
        p.tile = c.tile;
        splits = parts;
      }
    }
  }
  set_splits(&p, splits, steps, m, n);
  return p;
}

size_t plan_bytes(const Plan& p, int64_t m, int64_t n, int64_t k, int dtype, bool a_mn, bool b_mn,
                  bool copy_a, bool copy_b) {
  size_t bytes = p.partial_bytes;
  if (p.path == Path::kTensor) {
    if (copy_a) bytes += copy_bytes(extent(a_mn, m, k), dtype);
    if (copy_b) bytes += copy_bytes(extent(b_mn, n, k), dtype);
  }
  return bytes;
}

// The operand as it will be in its copy at `*at`.
Pad copy_operand(Operand* o, const Extent& e, int dtype, uint8_t** at) {
  const int es = elem_size(dtype);
  const int64_t to = (int64_t)align_up((size_t)e.cols * es, 16) / es;
  const Pad p{o->p, e.rows, e.cols, o->ld, *at, to};
  o->p = *at;
  o->ld = to;
  *at += copy_bytes(e, dtype);
  return p;
}

int run_gemm(Gemm g, void* workspace, size_t workspace_bytes, int32_t* status, cudaStream_t s,
             const char* what) {
  const Plan p = plan_gemm(g.m, g.n, g.k, g.dtype, g.a.mn, g.b.mn);
  if (g.m == 0 || g.n == 0) return SV_OK;
  if (p.path == Path::kEmpty) return finish(g, nullptr, 0, s);
  if (p.path == Path::kFew) return gemm_few(g, s);
  const bool copy_a = !tma_ready(g.a, g.dtype), copy_b = !tma_ready(g.b, g.dtype);
  const size_t need = plan_bytes(p, g.m, g.n, g.k, g.dtype, g.a.mn, g.b.mn, copy_a, copy_b);
  if (need && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    SV_FAIL(SV_ERR_WORKSPACE, std::string(what) + ": workspace too small or unaligned");
  uint8_t* at = static_cast<uint8_t*>(workspace);
  float* partial = nullptr;
  g.splits = p.splits;
  if (p.splits > 1) {
    partial = reinterpret_cast<float*>(at);
    at += p.partial_bytes;
    g.ep.partial = partial;
  }
  int rc;
  if (p.path == Path::kF32) {
    rc = gemm_f32(g, p.small, s);
  } else {
    Pad pads[2];
    int count = 0;
    if (copy_a) pads[count++] = copy_operand(&g.a, extent(g.a.mn, g.m, g.k), g.dtype, &at);
    if (copy_b) pads[count++] = copy_operand(&g.b, extent(g.b.mn, g.n, g.k), g.dtype, &at);
    if (count && (rc = pad_rows(pads, count, elem_size(g.dtype), s)) != SV_OK) return rc;
    rc = gemm_tc(g, p.tile, status, s);
  }
  if (rc != SV_OK || p.splits == 1) return rc;
  return finish(g, partial, p.splits, s);
}

// The backward pass's workspace: dz in rows of a multiple of 16 bytes, where it is not dout itself; the
// bias's partial sums; what raises fp16's dz; and what the larger of the two products needs.
struct BackLayout {
  size_t bias, raise, scratch, total;  // dz is at the start
  int64_t ld;
};
BackLayout back_layout(int64_t m, int64_t k, int64_t n, int dtype, bool copy_x, bool copy_w,
                       bool hold) {
  BackLayout l;
  const size_t row = align_up((size_t)n * elem_size(dtype), 16);
  l.ld = hold ? (int64_t)(row / elem_size(dtype)) : n;
  l.bias = hold ? align_up(m * row, COPY_ALIGN) : 0;
  l.raise = l.bias + align_up((size_t)MAX_STRIPS * n * sizeof(float), COPY_ALIGN);
  l.scratch = l.raise;
  if (hold && dtype == SV_FLOAT16) l.scratch += COPY_ALIGN + align_up(k * sizeof(float), COPY_ALIGN);
  l.total = l.scratch +
            std::max(plan_bytes(plan_gemm(m, k, n, dtype, false, true), m, k, n, dtype, false, true,
                                false, copy_w),
                     plan_bytes(plan_gemm(n, k, m, dtype, true, true), n, k, m, dtype, true, true,
                                false, copy_x));
  return l;
}

bool float_dtype(int d) { return d == SV_FLOAT32 || d == SV_FLOAT16 || d == SV_BFLOAT16; }

int check_sizes(int64_t m, int64_t k, int64_t n, const char* what) {
  if (m < 0 || k < 0 || n < 0)
    SV_FAIL(SV_ERR_INVALID_ARGUMENT, std::string(what) + ": negative size");
  if (m > INT32_MAX - 256 || k > INT32_MAX - 256 || n > INT32_MAX - 256)
    SV_FAIL(SV_ERR_UNSUPPORTED, std::string(what) + ": sizes must be below 2^31 - 256");
  return SV_OK;
}

}  // namespace
}  // namespace sv

using namespace sv;

extern "C" size_t sv_linear_workspace_bytes(int pass, int64_t m, int64_t k, int64_t n, int dtype,
                                            int copies) {
  if (m < 0 || k < 0 || n < 0 || (!float_dtype(dtype) && dtype != SV_FLOAT8_E4M3)) return 0;
  const bool a = copies & 1, b = copies & 2;
  if (pass == SV_LINEAR_FORWARD)
    return plan_bytes(plan_gemm(m, n, k, dtype, false, false), m, n, k, dtype, false, false, a, b);
  if (pass != SV_LINEAR_BACKWARD || !float_dtype(dtype)) return 0;
  return back_layout(m, k, n, dtype, a, b, copies & 4).total;
}

extern "C" int sv_linear_forward(const void* x, int64_t ldx, const void* weight, int64_t ldw,
                                 const void* bias, const void* residual, int64_t ld_res,
                                 const float* x_scale, const float* w_scale, int64_t m, int64_t k,
                                 int64_t n, int dtype, int out_dtype, int activation, void* out,
                                 float* preact, void* workspace, size_t workspace_bytes,
                                 int32_t* status, sv_stream_t stream) {
  const int rc = check_sizes(m, k, n, "sv_linear_forward");
  if (rc != SV_OK) return rc;
  const bool e4m3 = dtype == SV_FLOAT8_E4M3;
  if (!float_dtype(dtype) && !e4m3)
    SV_FAIL(SV_ERR_BAD_DTYPE, "sv_linear_forward: unknown dtype");
  if (e4m3 ? (out_dtype != SV_FLOAT16 && out_dtype != SV_BFLOAT16) : out_dtype != dtype)
    SV_FAIL(SV_ERR_BAD_DTYPE,
            "sv_linear_forward: the output has the operands' type, or is fp16 / bf16 for e4m3");
  if (activation < SV_ACT_NONE || activation > SV_ACT_GELU_TANH)
    SV_FAIL(SV_ERR_INVALID_ARGUMENT, "sv_linear_forward: unknown activation");
  if (m == 0 || n == 0) return SV_OK;
  if (!out || (k > 0 && (!x || !weight)))
    SV_FAIL(SV_ERR_INVALID_ARGUMENT, "sv_linear_forward: null pointer");
  if (ldx < k || ldw < k || (residual && ld_res < n))
    SV_FAIL(SV_ERR_INVALID_ARGUMENT, "sv_linear_forward: row stride below the row length");
  Gemm g{{x, ldx, false}, {weight, ldw, false}, m, n, k, dtype, 1,
         {bias, residual, ld_res, x_scale, w_scale, out, preact, nullptr, out_dtype, activation}};
  return run_gemm(g, workspace, workspace_bytes, status, to_stream(stream), "sv_linear_forward");
}

extern "C" int sv_linear_backward(const void* dout, const float* preact, const void* x, int64_t ldx,
                                  const void* weight, int64_t ldw, int64_t m, int64_t k, int64_t n,
                                  int dtype, int activation, void* dx, void* dw, void* dbias,
                                  void* workspace, size_t workspace_bytes, int32_t* status,
                                  sv_stream_t stream) {
  const int rc = check_sizes(m, k, n, "sv_linear_backward");
  if (rc != SV_OK) return rc;
  if (!float_dtype(dtype)) SV_FAIL(SV_ERR_BAD_DTYPE, "sv_linear_backward: unknown dtype");
  if (activation < SV_ACT_NONE || activation > SV_ACT_GELU_TANH)
    SV_FAIL(SV_ERR_INVALID_ARGUMENT, "sv_linear_backward: unknown activation");
  if (m == 0 || k == 0) dx = nullptr;
  if (n == 0 || k == 0) dw = nullptr;
  if (n == 0) dbias = nullptr;
  if (!dx && !dw && !dbias) return SV_OK;
  const bool act = activation != SV_ACT_NONE, terms = m > 0 && n > 0;
  if (terms && (!dout || (act && !preact) || (dx && !weight) || (dw && !x)))
    SV_FAIL(SV_ERR_INVALID_ARGUMENT, "sv_linear_backward: null pointer");
  if ((dx && ldw < k) || (dw && ldx < k))
    SV_FAIL(SV_ERR_INVALID_ARGUMENT, "sv_linear_backward: row stride below the row length");
  cudaStream_t s = to_stream(stream);
  const Operand xo{x, ldx, true}, wo{weight, ldw, true};
  // dz is dout without an activation, unless TMA cannot read its rows
  const bool hold = act || (dtype != SV_FLOAT32 && !tma_ready({dout, n, false}, dtype));
  const BackLayout l = back_layout(m, k, n, dtype, dw && !tma_ready(xo, dtype),
                                   dx && !tma_ready(wo, dtype), hold);
  if (!workspace || workspace_bytes < l.total || !aligned16(workspace))
    SV_FAIL(SV_ERR_WORKSPACE, "sv_linear_backward: workspace too small or unaligned");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const void* dz = hold ? ws : dout;
  Raise raise{};
  if (!terms) {
    if (dbias) SV_CUDA_TRY(cudaMemsetAsync(dbias, 0, n * elem_size(dtype), s));
  } else if (dbias || (hold && (dx || dw))) {
    void* to = hold && (dx || dw) ? ws : nullptr;
    float* partial = reinterpret_cast<float*>(ws + l.bias);
    if (to && act && dtype == SV_FLOAT16)
      raise = {reinterpret_cast<unsigned*>(ws + l.raise),
               reinterpret_cast<float*>(ws + l.raise + COPY_ALIGN), k};
    const int bad =
        dtype == SV_FLOAT32
            ? dz_typed<float>(dout, preact, m, n, activation, to, l.ld, dbias, partial, raise, s)
        : dtype == SV_FLOAT16
            ? dz_typed<__half>(dout, preact, m, n, activation, to, l.ld, dbias, partial, raise, s)
            : dz_typed<__nv_bfloat16>(dout, preact, m, n, activation, to, l.ld, dbias, partial, raise,
                                      s);
    if (bad != SV_OK) return bad;
  }
  const size_t left = workspace_bytes - l.scratch;
  if (dx) {
    const Gemm g{{dz, l.ld, false}, wo, m, k, n, dtype, 1,
                 {nullptr, nullptr, 0, nullptr, raise.down, dx, nullptr, nullptr, dtype, SV_ACT_NONE}};
    const int bad = run_gemm(g, ws + l.scratch, left, status, s, "sv_linear_backward (dx)");
    if (bad != SV_OK) return bad;
  }
  if (!dw) return SV_OK;
  const Gemm g{{dz, l.ld, true}, xo, n, k, m, dtype, 1,
               {nullptr, nullptr, 0, nullptr, raise.down, dw, nullptr, nullptr, dtype, SV_ACT_NONE}};
  return run_gemm(g, ws + l.scratch, left, status, s, "sv_linear_backward (dw)");
}
