// Root-mean-square norm of feature rows with the residual's addition, an optional 8-bit output
// with one scale per row, and its gradients.
//
//     h    = round(x + residual)                     (x itself without a residual)
//     rstd = 1 / sqrt(mean(h^2) + eps)
//     y    = h * rstd * w
//     8 bits: s = max|y| / 448 (1 for a row of zeros), q = round_e4m3(y / s)
//     dx   = rstd * (g - h * rstd^2 * mean(g h)) + dh,  g = dy * w   (the residual's gradient too)
//     dw_c = sum over the rows of dy_c * h_c * rstd
//
// h is rounded to the feature type before it is normed: it is the residual stream that the next
// block reads, and the backward pass then differentiates at the point the forward pass used.
// Everything else stays in fp32 with one rounding at the end.
//
// Both passes move each row once and do about ten operations per element, so HBM bounds them. A
// row lives in the registers of TPR threads (J accesses of V elements each; 16-byte accesses when
// the rows allow them, single elements otherwise).
#include <cuda_fp8.h>

#include <algorithm>
#include <type_traits>

#include "rows.cuh"

namespace sv {
namespace {

constexpr int RMS_THREADS = 256;
constexpr float E4M3_MAX = 448.0f;
constexpr int RMS_MAX_CHANNELS = 8192;

struct RmsArgs {
  int64_t n;
  int channels;
  int64_t x_stride, res_stride;  // elements between rows
  float eps;
  const float* weight;  // [C] or null
  float* rstd;          // [n] or null
  float* scale;         // [n], 8-bit output only
};

// 16-byte vectors go through uint4, so that they are one access.
template <typename T, int V>
__device__ __forceinline__ void load_row(const T* p, float (&v)[V]) {
  if constexpr (V * sizeof(T) == 16) {
    const uint4 raw = *reinterpret_cast<const uint4*>(p);
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = to_f32(e[k]);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = to_f32(p[k]);
  }
}

template <typename T, int V>
__device__ __forceinline__ void store_row(T* p, const float (&v)[V]) {
  if constexpr (V * sizeof(T) == 16) {
    uint4 raw;
    T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int k = 0; k < V; ++k) e[k] = from_f32<T>(v[k]);
    *reinterpret_cast<uint4*>(p) = raw;
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) p[k] = from_f32<T>(v[k]);
  }
}

template <int V>
__device__ __forceinline__ void load_weight(const float* w, int c, float (&v)[V]) {
  if (w == nullptr) {
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = 1.f;
  } else if constexpr (V % 4 == 0) {
#pragma unroll
    for (int k = 0; k < V; k += 4) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(w + c + k));
      v[k] = f.x; v[k + 1] = f.y; v[k + 2] = f.z; v[k + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = __ldg(w + c + k);
  }
}

struct Sum {
  static __device__ __forceinline__ float of(float a, float b) { return a + b; }
};
// Keeps a NaN (fmaxf drops it), so that a row with one gets a NaN scale.
struct Max {
  static __device__ __forceinline__ float of(float a, float b) {
    return a > b || a != a ? a : b;
  }
};

// Reduction over the TPR threads of a row; every thread gets the result. With TPR > 32 the block
// is one row and `part` holds a word per warp.
template <typename Op, int TPR>
__device__ __forceinline__ float row_reduce(float v, float* part) {
#pragma unroll
  for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1)
    v = Op::of(v, __shfl_xor_sync(0xffffffffu, v, o));
  if constexpr (TPR > 32) {
    constexpr int W = TPR / 32;
    __syncthreads();  // the previous use of `part` is over
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int i = 1; i < W; ++i) v = Op::of(v, part[i]);
  }
  return v;
}

template <int TPR>
constexpr int kBlock = TPR > 32 ? TPR : RMS_THREADS;

template <int V>
__device__ __forceinline__ void store_e4m3(uint8_t* q, const float (&v)[V], float inv) {
  if constexpr (V % 4 == 0) {
    uint32_t packed[V / 4];
#pragma unroll
    for (int k = 0; k < V; k += 4) {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[k] * inv, v[k + 1] * inv),
                                                   __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[k + 2] * inv, v[k + 3] * inv),
                                                   __NV_SATFINITE, __NV_E4M3);
      packed[k / 4] = lo | hi << 16;
    }
    if constexpr (V == 8)
      *reinterpret_cast<uint2*>(q) = make_uint2(packed[0], packed[1]);
    else
      *reinterpret_cast<uint32_t*>(q) = packed[0];
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k)
      q[k] = __nv_cvt_float_to_fp8(v[k] * inv, __NV_SATFINITE, __NV_E4M3);
  }
}

// A row's scale from its largest magnitude, and the factor its values are stored with: their product
// with the reciprocal is within 2^-23 of the quotient, and a division an element cost 22 us of 88 at
// 40,662 x 1024. Next to the smallest numbers the reciprocal would overflow, so the values are raised
// first.
template <int J, int V>
__device__ __forceinline__ float e4m3_scale(float top, float (&v)[J][V], float* inv) {
  float scale = 1.f;
  if (top != 0.f) {
    scale = top / E4M3_MAX;
    if (scale < 0x1p-149f) scale = 0x1p-149f;
  }
  if (scale < 0x1p-120f) {
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int k = 0; k < V; ++k) v[j][k] *= 0x1p40f;
    *inv = 1.0f / (scale * 0x1p40f);
  } else {
    *inv = 1.0f / scale;
  }
  return scale;
}

template <typename T, int V, int TPR, int J, bool Q8>
__global__ void __launch_bounds__(kBlock<TPR>)
    rms_kernel(const T* __restrict__ x, const T* __restrict__ res, RmsArgs a, T* __restrict__ h_out,
               void* __restrict__ out) {
  constexpr int ROWS = kBlock<TPR> / TPR;
  __shared__ float part[TPR > 32 ? TPR / 32 : 1];
  const int sub = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / TPR;
  const bool live = row < a.n;
  const int C = a.channels;
  float v[J][V];
  float sq = 0.f;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int c = (sub + TPR * j) * V;
    if (live && c < C) {
      load_row<T, V>(x + row * a.x_stride + c, v[j]);
      if (res != nullptr) {
        float r[V];
        load_row<T, V>(res + row * a.res_stride + c, r);
#pragma unroll
        for (int k = 0; k < V; ++k) v[j][k] = to_f32(from_f32<T>(v[j][k] + r[k]));
        if (h_out != nullptr) store_row<T, V>(h_out + row * C + c, v[j]);
      }
#pragma unroll
      for (int k = 0; k < V; ++k) sq = fmaf(v[j][k], v[j][k], sq);
    }
  }
  sq = row_reduce<Sum, TPR>(sq, part);
  const float rstd = 1.0f / sqrtf(sq / (float)C + a.eps);
  if (live && sub == 0 && a.rstd != nullptr) a.rstd[row] = rstd;
  float top = 0.f;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int c = (sub + TPR * j) * V;
    if (live && c < C) {
      float w[V];
      load_weight<V>(a.weight, c, w);
#pragma unroll
      for (int k = 0; k < V; ++k) v[j][k] = v[j][k] * rstd * w[k];
      if constexpr (Q8) {
#pragma unroll
        for (int k = 0; k < V; ++k) top = Max::of(top, fabsf(v[j][k]));
      } else {
        store_row<T, V>(static_cast<T*>(out) + row * C + c, v[j]);
      }
    }
  }
  if constexpr (Q8) {
    top = row_reduce<Max, TPR>(top, part);
    if (!live) return;
    float inv;
    const float scale = e4m3_scale(top, v, &inv);
    if (sub == 0) a.scale[row] = scale;
    uint8_t* q = static_cast<uint8_t*>(out) + row * C;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int c = (sub + TPR * j) * V;
      if (c < C) store_e4m3<V>(q + c, v[j], inv);
    }
  }
}

// Gradients: each group of TPR threads takes R rows at a time (so that R rows' loads are in flight)
// and keeps its channels' share of dw in registers; a block adds its groups in order through shared
// memory and writes one row of `partial` ([gridDim.x, C]), which column_sum_kernel adds in a fixed
// order.
template <typename T, int V, int TPR, int J, int R>
__global__ void __launch_bounds__(kBlock<TPR>)
    rms_backward_kernel(const T* __restrict__ h, const T* __restrict__ dy,
                        const T* __restrict__ dh, RmsArgs a, T* __restrict__ dx,
                        float* __restrict__ partial) {
  constexpr int GROUPS = kBlock<TPR> / TPR;
  constexpr int W = TPR > 32 ? TPR / 32 : 1;
  extern __shared__ float s_dw[];  // [C] when dw is wanted
  __shared__ float part[2][R][W];
  const int sub = threadIdx.x % TPR;
  const int group = threadIdx.x / TPR;
  const int C = a.channels;
  float w[J][V], dw[J][V];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int c = (sub + TPR * j) * V;
#pragma unroll
    for (int k = 0; k < V; ++k) dw[j][k] = 0.f;
    if (c < C) load_weight<V>(a.weight, c, w[j]);
  }
  const float inv_c = 1.0f / (float)C;
  int flip = 0;
  // the block's groups take consecutive rows, so every group makes the same number of rounds
  for (int64_t base = (int64_t)blockIdx.x * GROUPS * R; base < a.n;
       base += (int64_t)gridDim.x * GROUPS * R, flip ^= 1) {
    const int64_t row0 = base + group * R;
    float hv[R][J][V], g[R][J][V];
    float dot[R], rstd[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool live = row0 + r < a.n;
      rstd[r] = live ? __ldg(a.rstd + row0 + r) : 0.f;
      dot[r] = 0.f;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int c = (sub + TPR * j) * V;
        if (live && c < C) {
          load_row<T, V>(h + (row0 + r) * a.x_stride + c, hv[r][j]);
          load_row<T, V>(dy + (row0 + r) * C + c, g[r][j]);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int j = 0; j < J; ++j) {
        if (row0 + r < a.n && (sub + TPR * j) * V < C) {
#pragma unroll
          for (int k = 0; k < V; ++k) {
            dw[j][k] = fmaf(g[r][j][k], hv[r][j][k] * rstd[r], dw[j][k]);
            g[r][j][k] *= w[j][k];
            dot[r] = fmaf(g[r][j][k], hv[r][j][k], dot[r]);
          }
        }
      }
#pragma unroll
      for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1)
        dot[r] += __shfl_xor_sync(0xffffffffu, dot[r], o);
      if (TPR > 32 && (threadIdx.x & 31) == 0) part[flip][r][threadIdx.x >> 5] = dot[r];
    }
    if constexpr (TPR > 32) {
      __syncthreads();  // two copies: the next round's writes do not meet this round's reads
#pragma unroll
      for (int r = 0; r < R; ++r) {
        dot[r] = part[flip][r][0];
#pragma unroll
        for (int i = 1; i < W; ++i) dot[r] += part[flip][r][i];
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float pull = dot[r] * rstd[r] * rstd[r] * inv_c;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int c = (sub + TPR * j) * V;
        if (row0 + r < a.n && c < C) {
          float d[V];
#pragma unroll
          for (int k = 0; k < V; ++k) d[k] = rstd[r] * (g[r][j][k] - hv[r][j][k] * pull);
          if (dh != nullptr) {
            float e[V];
            load_row<T, V>(dh + (row0 + r) * C + c, e);
#pragma unroll
            for (int k = 0; k < V; ++k) d[k] += e[k];
          }
          store_row<T, V>(dx + (row0 + r) * C + c, d);
        }
      }
    }
  }
  if (partial == nullptr) return;
  for (int q = 0; q < GROUPS; ++q) {
    if (group == q) {
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int c = (sub + TPR * j) * V;
        if (c < C) {
#pragma unroll
          for (int k = 0; k < V; ++k)
            s_dw[c + k] = q == 0 ? dw[j][k] : s_dw[c + k] + dw[j][k];
        }
      }
    }
    __syncthreads();
  }
  for (int c = threadIdx.x; c < C; c += blockDim.x)
    partial[(int64_t)blockIdx.x * C + c] = s_dw[c];
}

// ---- long runs of rows: a pipeline per warp ------------------------------------------------------
//
// A warp takes rows warp, + warps, ... and keeps STAGES of them in flight by bulk copies into shared
// memory of its own (no barrier with other warps), its lanes holding the same channels of every
// row, so the weight and dw stay in registers. Loads in registers alone left HBM idle between a
// row's load and its store. 40,662 x 1024 bf16 + residual to e4m3: 75 -> 50 us (5.9 TB/s); the backward
// pass of 20,331 rows: 72 -> 35 us (4.8 TB/s).

template <typename T, int J, bool Q8>
__global__ void __launch_bounds__(32 * ROW_WARPS, 2)
    rms_rows_kernel(const T* __restrict__ x, const T* __restrict__ res, RmsArgs a,
                    T* __restrict__ h_out, void* __restrict__ out, int32_t* status) {
  using Ring = RowRing<T, J>;
  constexpr int V = Ring::V, STAGES = 3;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int s_abort;
  const int lane = threadIdx.x & 31;
  const int C = a.channels;
  if (threadIdx.x == 0) s_abort = 0;
  __syncthreads();
  float w[J][V];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int c = (lane + 32 * j) * V;
    if (c < C) load_weight<V>(a.weight, c, w[j]);
  }
  const bool ok = run_rows<T, J, 2, STAGES>(
      smem, (int64_t)blockIdx.x * ROW_WARPS + (threadIdx.x >> 5), (int64_t)gridDim.x * ROW_WARPS,
      a.n,
      C * (int)sizeof(T), res != nullptr ? 2 : 1, &s_abort,
      [](int64_t r, int64_t) { return r; }, [&](int t, int64_t r) -> const void* {
        return t == 0 ? x + r * a.x_stride : res + r * a.res_stride;
      },
      [&](int64_t row, int64_t, const uint8_t* stage, auto&& release) {
        float v[J][V];
        float sq = 0.f;
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const int q = lane + 32 * j;
          if (q * V < C) {
            unpack<T>(reinterpret_cast<const uint4*>(stage)[q], v[j]);
            if (res != nullptr) {
              float r[V];
              unpack<T>(reinterpret_cast<const uint4*>(stage + Ring::ROW)[q], r);
#pragma unroll
              for (int k = 0; k < V; ++k) v[j][k] = to_f32(from_f32<T>(v[j][k] + r[k]));
            }
#pragma unroll
            for (int k = 0; k < V; ++k) sq = fmaf(v[j][k], v[j][k], sq);
          }
        }
        release();
        if (res != nullptr && h_out != nullptr) {
#pragma unroll
          for (int j = 0; j < J; ++j) {
            const int c = (lane + 32 * j) * V;
            if (c < C) store_row<T, V>(h_out + row * C + c, v[j]);
          }
        }
        sq = row_reduce<Sum, 32>(sq, nullptr);
        const float rstd = 1.0f / sqrtf(sq / (float)C + a.eps);
        if (lane == 0 && a.rstd != nullptr) a.rstd[row] = rstd;
        [[maybe_unused]] float top = 0.f;
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const int c = (lane + 32 * j) * V;
          if (c < C) {
#pragma unroll
            for (int k = 0; k < V; ++k) {
              v[j][k] = v[j][k] * rstd * w[j][k];
              if constexpr (Q8) top = Max::of(top, fabsf(v[j][k]));
            }
            if constexpr (!Q8) store_row<T, V>(static_cast<T*>(out) + row * C + c, v[j]);
          }
        }
        if constexpr (Q8) {
          top = row_reduce<Max, 32>(top, nullptr);
          float inv;
          const float scale = e4m3_scale(top, v, &inv);
          if (lane == 0) a.scale[row] = scale;
#pragma unroll
          for (int j = 0; j < J; ++j) {
            const int c = (lane + 32 * j) * V;
            if (c < C) store_e4m3<V>(static_cast<uint8_t*>(out) + row * C + c, v[j], inv);
          }
        }
      });
  if (!ok && lane == 0) report(status, SV_DEVICE_WAIT_TIMEOUT);
}

template <typename T, int J>
__global__ void __launch_bounds__(32 * ROW_WARPS, 2)
    rms_rows_backward_kernel(const T* __restrict__ h, const T* __restrict__ dy,
                             const T* __restrict__ dh, RmsArgs a, T* __restrict__ dx,
                             float* __restrict__ partial, int32_t* status) {
  using Ring = RowRing<T, J>;
  constexpr int V = Ring::V, STAGES = 2;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int s_abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int C = a.channels;
  if (threadIdx.x == 0) s_abort = 0;
  __syncthreads();
  float w[J][V], dw[J][V];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int c = (lane + 32 * j) * V;
#pragma unroll
    for (int k = 0; k < V; ++k) dw[j][k] = 0.f;
    if (c < C) load_weight<V>(a.weight, c, w[j]);
  }
  const float inv_c = 1.0f / (float)C;
  const bool ok = run_rows<T, J, 3, STAGES>(
      smem, (int64_t)blockIdx.x * ROW_WARPS + (threadIdx.x >> 5), (int64_t)gridDim.x * ROW_WARPS,
      a.n,
      C * (int)sizeof(T), dh != nullptr ? 3 : 2, &s_abort,
      [](int64_t r, int64_t) { return r; }, [&](int t, int64_t r) -> const void* {
        return t == 0 ? h + r * a.x_stride : (t == 1 ? dy : dh) + r * C;
      },
      [&](int64_t row, int64_t, const uint8_t* stage, auto&& release) {
        const float rstd = __ldg(a.rstd + row);
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const int q = lane + 32 * j;
          if (q * V < C) {
            float hv[V], g[V];
            unpack<T>(reinterpret_cast<const uint4*>(stage)[q], hv);
            unpack<T>(reinterpret_cast<const uint4*>(stage + Ring::ROW)[q], g);
#pragma unroll
            for (int k = 0; k < V; ++k) {
              dw[j][k] = fmaf(g[k], hv[k] * rstd, dw[j][k]);
              dot = fmaf(g[k] * w[j][k], hv[k], dot);
            }
          }
        }
        dot = row_reduce<Sum, 32>(dot, nullptr);
        const float pull = dot * rstd * rstd * inv_c;
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const int q = lane + 32 * j;
          if (q * V < C) {  // the row is read again: cheaper than 2 J V registers
            float hv[V], g[V];
            unpack<T>(reinterpret_cast<const uint4*>(stage)[q], hv);
            unpack<T>(reinterpret_cast<const uint4*>(stage + Ring::ROW)[q], g);
#pragma unroll
            for (int k = 0; k < V; ++k) g[k] = rstd * (g[k] * w[j][k] - hv[k] * pull);
            if (dh != nullptr) {
              unpack<T>(reinterpret_cast<const uint4*>(stage + 2 * Ring::ROW)[q], hv);
#pragma unroll
              for (int k = 0; k < V; ++k) g[k] += hv[k];
            }
            store_row<T, V>(dx + row * C + q * V, g);
          }
        }
        release();
      });
  if (!ok && lane == 0) report(status, SV_DEVICE_WAIT_TIMEOUT);
  if (partial == nullptr) return;
  __syncthreads();
  float* s_dw = reinterpret_cast<float*>(smem);  // the rings are done with
  for (int q = 0; q < ROW_WARPS; ++q) {
    if (warp == q) {
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int c = (lane + 32 * j) * V;
        if (c < C) {
#pragma unroll
          for (int k = 0; k < V; ++k)
            s_dw[c + k] = q == 0 ? dw[j][k] : s_dw[c + k] + dw[j][k];
        }
      }
    }
    __syncthreads();
  }
  for (int c = threadIdx.x; c < C; c += blockDim.x)
    partial[(int64_t)blockIdx.x * C + c] = s_dw[c];
}

// out[c] = sum of partial[0..rows)[c] in a fixed order: 32 channels a block, 8 strided row sums
// a channel, joined in order.
__global__ void __launch_bounds__(256) column_sum_kernel(const float* __restrict__ partial,
                                                         int rows, int channels,
                                                         float* __restrict__ out) {
  __shared__ float s[8][33];
  const int lane = threadIdx.x & 31, r0 = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float v = 0.f;
  if (c < channels)
    for (int r = r0; r < rows; r += 8) v += partial[(int64_t)r * channels + c];
  s[r0][lane] = v;
  __syncthreads();
  if (r0 == 0 && c < channels) {
#pragma unroll
    for (int i = 1; i < 8; ++i) v += s[i][lane];
    out[c] = v;
  }
}

template <int N>
using Int = std::integral_constant<int, N>;

// Threads of a row and accesses of a thread for rows of nv accesses of V elements; widths that V
// elements an access never reach are not compiled.
template <int V, typename F>
int by_width(int nv, F&& f) {
  if (nv <= 8) return f(Int<8>{}, Int<1>{});
  if (nv <= 32) return f(Int<32>{}, Int<1>{});
  if (nv <= 64) return f(Int<32>{}, Int<2>{});
  if (nv <= 128) return f(Int<32>{}, Int<4>{});
  if (nv <= 512) return f(Int<128>{}, Int<4>{});
  if constexpr (RMS_MAX_CHANNELS / V > 2048) {
    if (nv > 2048) return f(Int<512>{}, Int<16>{});
  }
  return f(Int<512>{}, Int<4>{});
}

// The backward pass holds more of a row (h, dy, w, dw), so it spreads one over more threads.
template <int V, typename F>
int by_width_backward(int nv, F&& f) {
  if (nv <= 8) return f(Int<8>{}, Int<1>{}, Int<2>{});
  if (nv <= 32) return f(Int<32>{}, Int<1>{}, Int<4>{});
  if (nv <= 64) return f(Int<32>{}, Int<2>{}, Int<2>{});
  if (nv <= 128) return f(Int<128>{}, Int<1>{}, Int<4>{});
  if (nv <= 256) return f(Int<128>{}, Int<2>{}, Int<2>{});
  if constexpr (RMS_MAX_CHANNELS / V > 1024) {
    if constexpr (RMS_MAX_CHANNELS / V > 2048) {
      if (nv > 2048) return f(Int<512>{}, Int<16>{}, Int<1>{});
    }
    if (nv > 1024) return f(Int<512>{}, Int<4>{}, Int<1>{});
  }
  return f(Int<512>{}, Int<2>{}, Int<1>{});
}

constexpr int BACKWARD_BLOCKS = 888;  // at most six per SM; also the rows of the dw partials

// Whether rows go through the warps' pipelines: rows of 33 to 128 16-byte accesses, and enough of them
// that every warp gets four (below that the direct kernels start sooner: 8 x 1024 bf16 2.1 against 3 us).
// Wider rows do not fit a warp's registers beside the weight and dw, and keep the direct kernels. 20,331
// rows, launch included, with residual / backward: 1024 channels of bf16 33 / 33 us (the direct kernel's
// backward pass took 72 at that width), 1280 57 / 88, 2048 72 / 102, 4096 127 / 211, 8192 322 / 272 us;
// 512 of fp32 33 / 29, 1024 57 / 51, 2048 107 / 121, 4096 201 / 172 us.
constexpr int ROW_BLOCKS_PER_SM = 2;
bool pipelined(int64_t n, int nv) {
  return nv > 32 && nv <= 128 && n >= (int64_t)4 * ROW_WARPS * ROW_BLOCKS_PER_SM * num_sms();
}

template <typename K>
int allow_smem(K kernel, int bytes) {
  SV_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  return SV_OK;
}

template <typename T, int J>
int launch_rows(const void* x, const void* res, const RmsArgs& a, void* h_out, void* out, bool q8,
                int32_t* status, cudaStream_t s) {
  auto kernel = q8 ? rms_rows_kernel<T, J, true> : rms_rows_kernel<T, J, false>;
  constexpr int bytes = RowRing<T, J>::SMEM(2, 3);
  const int rc = allow_smem(kernel, bytes);
  if (rc != SV_OK) return rc;
  kernel<<<ROW_BLOCKS_PER_SM * num_sms(), 32 * ROW_WARPS, bytes, s>>>(
      static_cast<const T*>(x), static_cast<const T*>(res), a, static_cast<T*>(h_out), out, status);
  SV_LAUNCH_CHECK();
  return SV_OK;
}

template <typename T, int J>
int launch_rows_backward(const void* h, const void* dy, const void* dh, const RmsArgs& a, void* dx,
                         float* partial, float* dw, int32_t* status, cudaStream_t s) {
  constexpr int bytes = RowRing<T, J>::SMEM(3, 2);
  const int rc = allow_smem(rms_rows_backward_kernel<T, J>, bytes);
  if (rc != SV_OK) return rc;
  const int blocks = std::min(ROW_BLOCKS_PER_SM * num_sms(), BACKWARD_BLOCKS);
  rms_rows_backward_kernel<T, J><<<blocks, 32 * ROW_WARPS, bytes, s>>>(
      static_cast<const T*>(h), static_cast<const T*>(dy), static_cast<const T*>(dh), a,
      static_cast<T*>(dx), dw ? partial : nullptr, status);
  SV_LAUNCH_CHECK();
  if (dw != nullptr) {
    column_sum_kernel<<<(a.channels + 31) / 32, 256, 0, s>>>(partial, blocks, a.channels, dw);
    SV_LAUNCH_CHECK();
  }
  return SV_OK;
}

template <typename T, int V>
int launch_rms(const void* x, const void* res, const RmsArgs& a, void* h_out, void* out, bool q8,
               int32_t* status, cudaStream_t s) {
  if constexpr (V > 1) {
    const int nv = a.channels / V;
    if (pipelined(a.n, nv))
      return nv <= 64 ? launch_rows<T, 2>(x, res, a, h_out, out, q8, status, s)
                      : launch_rows<T, 4>(x, res, a, h_out, out, q8, status, s);
  }
  return by_width<V>((a.channels + V - 1) / V, [&](auto tpr, auto j) -> int {
    constexpr int TPR = decltype(tpr)::value, J = decltype(j)::value;
    constexpr int ROWS = kBlock<TPR> / TPR;
    const int64_t blocks = (a.n + ROWS - 1) / ROWS;
    auto kernel = q8 ? rms_kernel<T, V, TPR, J, true> : rms_kernel<T, V, TPR, J, false>;
    kernel<<<(unsigned)blocks, kBlock<TPR>, 0, s>>>(
        static_cast<const T*>(x), static_cast<const T*>(res), a, static_cast<T*>(h_out), out);
    SV_LAUNCH_CHECK();
    return SV_OK;
  });
}

template <typename T, int V>
int launch_rms_backward(const void* h, const void* dy, const void* dh, const RmsArgs& a, void* dx,
                        float* partial, float* dw, int32_t* status, cudaStream_t s) {
  if constexpr (V > 1) {
    const int nv = a.channels / V;
    if (pipelined(a.n, nv))
      return nv <= 64 ? launch_rows_backward<T, 2>(h, dy, dh, a, dx, partial, dw, status, s)
                      : launch_rows_backward<T, 4>(h, dy, dh, a, dx, partial, dw, status, s);
  }
  return by_width_backward<V>((a.channels + V - 1) / V, [&](auto tpr, auto j, auto r) -> int {
    constexpr int TPR = decltype(tpr)::value, J = decltype(j)::value, R = decltype(r)::value;
    constexpr int ROWS = kBlock<TPR> / TPR * R;
    const int64_t want = (a.n + ROWS - 1) / ROWS;
    const int blocks = (int)(want < BACKWARD_BLOCKS ? want : BACKWARD_BLOCKS);
    rms_backward_kernel<T, V, TPR, J, R>
        <<<blocks, kBlock<TPR>, dw ? a.channels * sizeof(float) : 0, s>>>(
            static_cast<const T*>(h), static_cast<const T*>(dy), static_cast<const T*>(dh), a,
            static_cast<T*>(dx), dw ? partial : nullptr);
    SV_LAUNCH_CHECK();
    if (dw != nullptr) {
      column_sum_kernel<<<(a.channels + 31) / 32, 256, 0, s>>>(partial, blocks, a.channels, dw);
      SV_LAUNCH_CHECK();
    }
    return SV_OK;
  });
}

bool vec_ok(const void* p, int64_t stride, int esize) {
  return p == nullptr || (aligned16(p) && stride * esize % 16 == 0);
}

int check_common(int64_t n, int channels, int dtype, float eps, const char* what) {
  if (dtype != SV_FLOAT32 && dtype != SV_FLOAT16 && dtype != SV_BFLOAT16)
    SV_FAIL(SV_ERR_BAD_DTYPE, std::string(what) + ": unknown dtype");
  if (n < 0 || channels < 0) SV_FAIL(SV_ERR_INVALID_ARGUMENT, std::string(what) + ": negative size");
  if (channels > RMS_MAX_CHANNELS)
    SV_FAIL(SV_ERR_UNSUPPORTED, std::string(what) + ": at most 8192 channels");
  if (n > (int64_t)INT32_MAX)
    SV_FAIL(SV_ERR_UNSUPPORTED, std::string(what) + ": at most 2^31 - 1 rows");
  if (!(eps >= 0.f)) SV_FAIL(SV_ERR_INVALID_ARGUMENT, std::string(what) + ": negative eps");
  return SV_OK;
}

}  // namespace
}  // namespace sv

using namespace sv;

extern "C" int sv_rms_norm(const void* x, int64_t x_stride, const void* residual,
                           int64_t residual_stride, int64_t n, int channels, int dtype, float eps,
                           const float* weight, void* h, float* rstd, void* out, int out_dtype,
                           float* scale, int32_t* status, sv_stream_t stream) {
  const int rc = check_common(n, channels, dtype, eps, "sv_rms_norm");
  if (rc != SV_OK) return rc;
  const bool q8 = out_dtype == SV_FLOAT8_E4M3;
  if (!q8 && out_dtype != dtype)
    SV_FAIL(SV_ERR_BAD_DTYPE, "sv_rms_norm: the output has the input's type or is e4m3");
  if (n == 0 || (channels == 0 && !q8)) return SV_OK;  // rows of nothing still have scales
  if ((channels > 0 && (!x || !out)) || (q8 && !scale))
    SV_FAIL(SV_ERR_INVALID_ARGUMENT, "sv_rms_norm: null pointer");
  if (x_stride < channels || (residual && residual_stride < channels))
    SV_FAIL(SV_ERR_INVALID_ARGUMENT, "sv_rms_norm: row stride below the channel count");
  RmsArgs a{n, channels, x_stride, residual_stride, eps, weight, rstd, scale};
  const int es = dtype_size(dtype);
  const bool vec = channels * es % 16 == 0 && vec_ok(x, x_stride, es) &&
                   vec_ok(residual, residual_stride, es) && vec_ok(h, channels, es) &&
                   aligned16(out) && (!weight || aligned16(weight));
  cudaStream_t s = to_stream(stream);
  if (dtype == SV_FLOAT32)
    return vec ? launch_rms<float, 4>(x, residual, a, h, out, q8, status, s)
               : launch_rms<float, 1>(x, residual, a, h, out, q8, status, s);
  if (dtype == SV_FLOAT16)
    return vec ? launch_rms<__half, 8>(x, residual, a, h, out, q8, status, s)
               : launch_rms<__half, 1>(x, residual, a, h, out, q8, status, s);
  return vec ? launch_rms<__nv_bfloat16, 8>(x, residual, a, h, out, q8, status, s)
             : launch_rms<__nv_bfloat16, 1>(x, residual, a, h, out, q8, status, s);
}

extern "C" size_t sv_rms_norm_backward_workspace_bytes(int channels) {
  if (channels <= 0 || channels > RMS_MAX_CHANNELS) return 0;
  return (size_t)BACKWARD_BLOCKS * channels * sizeof(float);
}

extern "C" int sv_rms_norm_backward(const void* h, int64_t h_stride, const void* dy,
                                    const void* dh, int64_t n, int channels, int dtype,
                                    const float* weight, const float* rstd, void* dx, float* dw,
                                    void* workspace, size_t workspace_bytes, int32_t* status,
                                    sv_stream_t stream) {
  const int rc = check_common(n, channels, dtype, 0.f, "sv_rms_norm_backward");
  if (rc != SV_OK) return rc;
  cudaStream_t s = to_stream(stream);
  if (channels == 0) return SV_OK;
  if (n == 0) {
    if (dw) SV_CUDA_TRY(cudaMemsetAsync(dw, 0, channels * sizeof(float), s));
    return SV_OK;
  }
  if (!h || !dy || !rstd || !dx)
    SV_FAIL(SV_ERR_INVALID_ARGUMENT, "sv_rms_norm_backward: null pointer");
  if (h_stride < channels)
    SV_FAIL(SV_ERR_INVALID_ARGUMENT, "sv_rms_norm_backward: row stride below the channel count");
  if (dw && (!workspace || workspace_bytes < sv_rms_norm_backward_workspace_bytes(channels)))
    SV_FAIL(SV_ERR_WORKSPACE, "sv_rms_norm_backward: workspace too small");
  RmsArgs a{n, channels, h_stride, 0, 0.f, weight, const_cast<float*>(rstd), nullptr};
  float* partial = static_cast<float*>(workspace);
  const int es = dtype_size(dtype);
  const bool vec = channels * es % 16 == 0 && vec_ok(h, h_stride, es) &&
                   vec_ok(dy, channels, es) && vec_ok(dh, channels, es) &&
                   vec_ok(dx, channels, es) && (!weight || aligned16(weight));
  if (dtype == SV_FLOAT32)
    return vec ? launch_rms_backward<float, 4>(h, dy, dh, a, dx, partial, dw, status, s)
               : launch_rms_backward<float, 1>(h, dy, dh, a, dx, partial, dw, status, s);
  if (dtype == SV_FLOAT16)
    return vec ? launch_rms_backward<__half, 8>(h, dy, dh, a, dx, partial, dw, status, s)
               : launch_rms_backward<__half, 1>(h, dy, dh, a, dx, partial, dw, status, s);
  return vec ? launch_rms_backward<__nv_bfloat16, 8>(h, dy, dh, a, dx, partial, dw, status, s)
             : launch_rms_backward<__nv_bfloat16, 1>(h, dy, dh, a, dx, partial, dw, status, s);
}
