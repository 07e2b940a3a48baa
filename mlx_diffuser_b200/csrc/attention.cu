// Self-attention inside coordinate windows with a learned relative position bias, and its
// gradients.
//
//     s_ij = scale * q_i . k_j + T[h][L[x_j - x_i]][L[y_j - y_i]][L[z_j - z_i]]   (i, j in a window)
//     p_ij = softmax_j(s_ij),  o_i = sum_j p_ij v_j
//     dv_j = sum_i p_ij do_i,  ds_ij = p_ij (do_i . v_j - delta_i),  delta_i = do_i . o_i
//     dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dT[h][b] = sum of ds over b's pairs
//
// L maps an offset along an axis, clamped to the table's reach, to a bucket. The windows come as a
// plan: rows in window order with each window's range of positions (sv_window_plan).
//
// The kernels here take any type and head size: a warp per row and head, lanes along the other
// side's rows for the scores and along the head's channels for the sums. They keep fp32 exactly
// (products and sums), so they are the fp32 path.
//
// The table's gradient sums in 64-bit fixed point, so that neither the order of the atomics nor
// the number of blocks changes it.
#include <limits.h>

#include "attention.h"

namespace sv {
namespace {

constexpr int ROW_WARPS = 8;

__global__ void __launch_bounds__(256)
    window_plan_kernel(const int32_t* __restrict__ coords, const int32_t* __restrict__ perm,
                       const int32_t* __restrict__ offsets, int64_t groups, int64_t n,
                       PlanRow* __restrict__ plan, int32_t* status) {
  const int64_t p = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (p >= n) return;
  int64_t lo = 0, hi = groups;  // offsets[lo] <= p < offsets[hi]
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) / 2;
    if (__ldg(offsets + mid) <= p) lo = mid; else hi = mid;
  }
  PlanRow r{};
  const int32_t start = __ldg(offsets + lo), end = __ldg(offsets + lo + 1);
  r.row = __ldg(perm + p);
  if (r.row < 0 || r.row >= n || start > p || end <= p || start < 0 || end > n) {
    report(status, SV_DEVICE_BAD_INDEX);
    r.row = -1;
    r.start = r.end = (int32_t)p;
  } else {
    const int4 c = __ldg(reinterpret_cast<const int4*>(coords) + r.row);
    r.x = c.y;
    r.y = c.z;
    r.z = c.w;
    r.start = start;
    r.end = end;
  }
  plan[p] = r;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float w = __shfl_xor_sync(0xffffffffu, v, o);
    v = v > w || v != v ? v : w;  // keeps a NaN
  }
  return v;
}

template <typename T>
__device__ __forceinline__ float dot_row(const float* s, const T* p, int dim) {
  float acc = 0.f;
  constexpr int E = 16 / sizeof(T);
  if (dim % E == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
    for (int d = 0; d < dim; d += E) {
      const uint4 raw = __ldg(reinterpret_cast<const uint4*>(p + d));
      const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int k = 0; k < E; ++k) acc = fmaf(s[d + k], to_f32(e[k]), acc);
    }
  } else {
    for (int d = 0; d < dim; ++d) acc = fmaf(s[d], to_f32(p[d]), acc);
  }
  return acc;
}

__device__ __forceinline__ int bucket_of(const AttnArgs& a, const PlanRow& query, const PlanRow& key) {
  const int x = lut_at(a, sub_sat(key.x, query.x));
  const int y = lut_at(a, sub_sat(key.y, query.y));
  const int z = lut_at(a, sub_sat(key.z, query.z));
  return (x * a.nb + y) * a.nb + z;
}

__device__ __forceinline__ PlanRow plan_at(const PlanRow* plan, int64_t p) {
  PlanRow r;
  const int4* s = reinterpret_cast<const int4*>(plan + p);
  *reinterpret_cast<int4*>(&r) = __ldg(s);
  *(reinterpret_cast<int4*>(&r) + 1) = __ldg(s + 1);
  return r;
}

constexpr int CH = ATTN_MAX_DIM / 32;  // channels a lane sums

template <typename T>
__global__ void __launch_bounds__(32 * ROW_WARPS) attn_rows_kernel(AttnArgs a) {
  __shared__ float s_q[ROW_WARPS][ATTN_MAX_DIM];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t p = (int64_t)blockIdx.x * ROW_WARPS + warp;
  const int h = blockIdx.y;
  if (p >= a.n) return;
  const PlanRow me = plan_at(a.plan, p);
  if (me.row < 0) return;
  const T* q = static_cast<const T*>(a.q) + me.row * a.q_row + h * a.q_head;
  const T* k = static_cast<const T*>(a.k) + h * a.k_head;
  const T* v = static_cast<const T*>(a.v) + h * a.v_head;
  const T* table = static_cast<const T*>(a.table) + (int64_t)h * a.nb * a.nb * a.nb;
  for (int d = lane; d < a.dim; d += 32) s_q[warp][d] = to_f32(q[d]) * a.scale;
  __syncwarp();
  float o[CH] = {}, top = -INFINITY, sum = 0.f;
  for (int j0 = me.start; j0 < me.end; j0 += 32) {
    const int j = j0 + lane;
    float s = -INFINITY;
    int row = -1;
    if (j < me.end) {
      const PlanRow key = plan_at(a.plan, j);
      row = key.row;
      if (row >= 0)
        s = dot_row(s_q[warp], k + row * a.k_row, a.dim) + to_f32(table[bucket_of(a, me, key)]);
    }
    const float m = fmaxf(top, warp_max(s));
    const float base = m == -INFINITY ? 0.f : m;
    const float keep = expf(top - base);
    const float e = expf(s - base);
    sum = sum * keep + warp_sum(e);
#pragma unroll
    for (int c = 0; c < CH; ++c) o[c] *= keep;
    const int count = min(32, me.end - j0);
    for (int i = 0; i < count; ++i) {
      const float w = __shfl_sync(0xffffffffu, e, i);
      const int r = __shfl_sync(0xffffffffu, row, i);
      if (r < 0) continue;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int d = lane + 32 * c;
        if (d < a.dim) o[c] = fmaf(w, to_f32(v[r * a.v_row + d]), o[c]);
      }
    }
    top = m;
  }
  T* out = static_cast<T*>(a.out) + (me.row * (int64_t)a.heads + h) * a.dim;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int d = lane + 32 * c;
    if (d < a.dim) out[d] = from_f32<T>(sum == 0.f ? 0.f : o[c] / sum);
  }
  // a row whose every score is -inf has weights of zero: exp(s - inf) in the backward pass too
  if (lane == 0 && a.lse) a.lse[h * a.n + p] = sum == 0.f ? INFINITY : top + logf(sum);
}

// dq, delta and the table's gradient: a warp per query.
template <typename T>
__global__ void __launch_bounds__(32 * ROW_WARPS) attn_dq_rows_kernel(AttnArgs a) {
  __shared__ float s_q[ROW_WARPS][ATTN_MAX_DIM];
  __shared__ float s_g[ROW_WARPS][ATTN_MAX_DIM];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t p = (int64_t)blockIdx.x * ROW_WARPS + warp;
  const int h = blockIdx.y;
  if (p >= a.n) return;
  const PlanRow me = plan_at(a.plan, p);
  if (me.row < 0) return;
  const int64_t own = (me.row * (int64_t)a.heads + h) * a.dim;
  const T* q = static_cast<const T*>(a.q) + me.row * a.q_row + h * a.q_head;
  const T* k = static_cast<const T*>(a.k) + h * a.k_head;
  const T* v = static_cast<const T*>(a.v) + h * a.v_head;
  const T* g = static_cast<const T*>(a.dout) + own;
  const T* o = static_cast<const T*>(a.o) + own;
  const int64_t cells = (int64_t)a.nb * a.nb * a.nb;
  const T* table = static_cast<const T*>(a.table) + h * cells;
  float delta = 0.f;
  for (int d = lane; d < a.dim; d += 32) {
    s_q[warp][d] = to_f32(q[d]) * a.scale;
    s_g[warp][d] = to_f32(g[d]);
    delta = fmaf(s_g[warp][d], to_f32(o[d]), delta);
  }
  delta = warp_sum(delta);
  if (lane == 0) a.delta[h * a.n + p] = delta;
  __syncwarp();
  const float lse = a.lse[h * a.n + p];
  const int exponent = a.dtable ? dtable_exponent(a, h) : INT_MAX;
  const double unit = exponent == INT_MAX ? 0.0 : ldexp(1.0, exponent);
  float acc[CH] = {};
  for (int j0 = me.start; j0 < me.end; j0 += 32) {
    const int j = j0 + lane;
    float ds = 0.f;
    int row = -1;
    if (j < me.end) {
      const PlanRow key = plan_at(a.plan, j);
      row = key.row;
      if (row >= 0) {
        const int b = bucket_of(a, me, key);
        const float s = dot_row(s_q[warp], k + row * a.k_row, a.dim) + to_f32(table[b]);
        const float dp = dot_row(s_g[warp], v + row * a.v_row, a.dim);
        ds = expf(s - lse) * (dp - delta);
        if (!(fabsf(ds) < INFINITY))
          atomicMax(a.norms + 2 * h, 0x7fffffffu);  // the head's table gradient is NaN
        else if (exponent != INT_MAX)
          atomicAdd(a.dtable + h * cells + b,
                    (unsigned long long)__double2ll_rn((double)ds * unit));
      }
    }
    const int count = min(32, me.end - j0);
    for (int i = 0; i < count; ++i) {
      const float w = __shfl_sync(0xffffffffu, ds, i);
      const int r = __shfl_sync(0xffffffffu, row, i);
      if (r < 0) continue;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int d = lane + 32 * c;
        if (d < a.dim) acc[c] = fmaf(w, to_f32(k[r * a.k_row + d]), acc[c]);
      }
    }
  }
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int d = lane + 32 * c;
    if (d < a.dim) static_cast<T*>(a.dq)[own + d] = from_f32<T>(acc[c] * a.scale);
  }
}

// dk and dv: a warp per key.
template <typename T>
__global__ void __launch_bounds__(32 * ROW_WARPS) attn_dkv_rows_kernel(AttnArgs a) {
  __shared__ float s_k[ROW_WARPS][ATTN_MAX_DIM];
  __shared__ float s_v[ROW_WARPS][ATTN_MAX_DIM];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t p = (int64_t)blockIdx.x * ROW_WARPS + warp;
  const int h = blockIdx.y;
  if (p >= a.n) return;
  const PlanRow me = plan_at(a.plan, p);
  if (me.row < 0) return;
  const T* q = static_cast<const T*>(a.q) + h * a.q_head;
  const T* k = static_cast<const T*>(a.k) + me.row * a.k_row + h * a.k_head;
  const T* v = static_cast<const T*>(a.v) + me.row * a.v_row + h * a.v_head;
  const T* g = static_cast<const T*>(a.dout) + (int64_t)h * a.dim;
  const int64_t g_row = (int64_t)a.heads * a.dim;
  const T* table = static_cast<const T*>(a.table) + (int64_t)h * a.nb * a.nb * a.nb;
  for (int d = lane; d < a.dim; d += 32) {
    s_k[warp][d] = to_f32(k[d]) * a.scale;
    s_v[warp][d] = to_f32(v[d]);
  }
  __syncwarp();
  float dk[CH] = {}, dv[CH] = {};
  for (int i0 = me.start; i0 < me.end; i0 += 32) {
    const int i = i0 + lane;
    float w = 0.f, ds = 0.f;
    int row = -1;
    if (i < me.end) {
      const PlanRow query = plan_at(a.plan, i);
      row = query.row;
      if (row >= 0) {
        const float s = dot_row(s_k[warp], q + row * a.q_row, a.dim) +
                        to_f32(table[bucket_of(a, query, me)]);
        w = expf(s - a.lse[h * a.n + i]);
        ds = w * (dot_row(s_v[warp], g + row * g_row, a.dim) - a.delta[h * a.n + i]);
      }
    }
    const int count = min(32, me.end - i0);
    for (int t = 0; t < count; ++t) {
      const float pw = __shfl_sync(0xffffffffu, w, t);
      const float dw = __shfl_sync(0xffffffffu, ds, t);
      const int r = __shfl_sync(0xffffffffu, row, t);
      if (r < 0) continue;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int d = lane + 32 * c;
        if (d < a.dim) {
          dv[c] = fmaf(pw, to_f32(g[r * g_row + d]), dv[c]);
          dk[c] = fmaf(dw, to_f32(q[r * a.q_row + d]), dk[c]);
        }
      }
    }
  }
  const int64_t own = (me.row * (int64_t)a.heads + h) * a.dim;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int d = lane + 32 * c;
    if (d < a.dim) {
      static_cast<T*>(a.dk)[own + d] = from_f32<T>(dk[c] * a.scale);
      static_cast<T*>(a.dv)[own + d] = from_f32<T>(dv[c]);
    }
  }
}

// norms[h] = bits of the largest |dout_i|^2 and |v_j|^2 of a head. Squares are not negative, so
// their bits order like the values, and a NaN stays above everything.
template <typename T>
__global__ void __launch_bounds__(256) attn_norms_kernel(AttnArgs a, unsigned* norms) {
  __shared__ unsigned s_top[2];
  const int h = blockIdx.y;
  if (threadIdx.x < 2) s_top[threadIdx.x] = 0u;
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int64_t r = (int64_t)blockIdx.x * 8 + warp; r < a.n; r += (int64_t)gridDim.x * 8) {
    const T* g = static_cast<const T*>(a.dout) + (r * a.heads + h) * a.dim;
    const T* v = static_cast<const T*>(a.v) + r * a.v_row + h * a.v_head;
    float g2 = 0.f, v2 = 0.f;
    for (int d = lane; d < a.dim; d += 32) {
      const float x = to_f32(g[d]), y = to_f32(v[d]);
      g2 = fmaf(x, x, g2);
      v2 = fmaf(y, y, v2);
    }
    g2 = warp_sum(g2);
    v2 = warp_sum(v2);
    if (lane == 0) {
      atomicMax(&s_top[0], __float_as_uint(g2) & 0x7fffffffu);
      atomicMax(&s_top[1], __float_as_uint(v2) & 0x7fffffffu);
    }
  }
  __syncthreads();
  if (threadIdx.x < 2) atomicMax(norms + 2 * h + threadIdx.x, s_top[threadIdx.x]);
}

template <typename T>
__global__ void __launch_bounds__(256)
    dtable_finish_kernel(AttnArgs a, T* __restrict__ out) {
  const int64_t cells = (int64_t)a.nb * a.nb * a.nb;
  const int h = blockIdx.y;
  const int exponent = dtable_exponent(a, h);
  for (int64_t b = (int64_t)blockIdx.x * 256 + threadIdx.x; b < cells;
       b += (int64_t)gridDim.x * 256) {
    const double v = exponent == INT_MAX
                         ? __longlong_as_double(0x7ff8000000000000ll)  // the inputs were not finite
                         : ldexp((double)(long long)a.dtable[h * cells + b], -exponent);
    out[h * cells + b] = from_f32<T>((float)v);
  }
}

dim3 row_grid(const AttnArgs& a) {
  return dim3((unsigned)((a.n + ROW_WARPS - 1) / ROW_WARPS), (unsigned)a.heads);
}

template <typename T>
int forward_typed(const AttnArgs& a, cudaStream_t s) {
  attn_rows_kernel<T><<<row_grid(a), 32 * ROW_WARPS, 0, s>>>(a);
  SV_LAUNCH_CHECK();
  return SV_OK;
}

template <typename T>
int backward_typed(const AttnArgs& a, unsigned* norms, void* dtable, cudaStream_t s) {
  if (dtable) {
    const unsigned blocks = (unsigned)((a.n + 63) / 64 < 512 ? (a.n + 63) / 64 : 512);
    attn_norms_kernel<T><<<dim3(blocks, a.heads), 256, 0, s>>>(a, norms);
    SV_LAUNCH_CHECK();
  }
  attn_dq_rows_kernel<T><<<row_grid(a), 32 * ROW_WARPS, 0, s>>>(a);
  SV_LAUNCH_CHECK();
  attn_dkv_rows_kernel<T><<<row_grid(a), 32 * ROW_WARPS, 0, s>>>(a);
  SV_LAUNCH_CHECK();
  if (dtable) {
    const unsigned blocks = (unsigned)((a.nb * a.nb * a.nb + 255) / 256);
    dtable_finish_kernel<T><<<dim3(blocks, a.heads), 256, 0, s>>>(a, static_cast<T*>(dtable));
    SV_LAUNCH_CHECK();
  }
  return SV_OK;
}

int check(int64_t n, int heads, int dim, int dtype, int nb, int reach, const char* what) {
  if (dtype != SV_FLOAT32 && dtype != SV_FLOAT16 && dtype != SV_BFLOAT16)
    SV_FAIL(SV_ERR_BAD_DTYPE, std::string(what) + ": unknown dtype");
  if (n < 0 || heads < 0 || dim < 0 || nb < 1 || reach < 0)
    SV_FAIL(SV_ERR_INVALID_ARGUMENT, std::string(what) + ": negative size");
  if (n > (1 << 25) || heads > ATTN_MAX_HEADS || dim > ATTN_MAX_DIM || nb > ATTN_MAX_BUCKETS ||
      reach > ATTN_MAX_REACH)
    SV_FAIL(SV_ERR_UNSUPPORTED,
            std::string(what) +
                ": at most 2^25 rows, 65535 heads, 128 channels a head, 25 buckets an axis and a "
                "reach of 1023");
  return SV_OK;
}

// Workspace of the backward pass: fixed-point table, norms, delta.
struct Layout {
  size_t table, norms, delta, total;
};
Layout layout(int64_t n, int heads, int nb) {
  Layout l;
  l.table = 0;
  l.norms = l.table + align_up((size_t)heads * nb * nb * nb * 8, 256);
  l.delta = l.norms + align_up((size_t)heads * 8, 256);
  l.total = l.delta + align_up((size_t)heads * n * 4, 256);
  return l;
}

}  // namespace
}  // namespace sv

using namespace sv;

extern "C" size_t sv_window_plan_bytes(int64_t n) { return n > 0 ? (size_t)n * sizeof(PlanRow) : 0; }

extern "C" int sv_window_plan(const int32_t* coords, const int32_t* perm, const int32_t* offsets,
                              int64_t groups, int64_t n, void* plan, int32_t* status,
                              sv_stream_t stream) {
  if (n < 0 || groups < 0) SV_FAIL(SV_ERR_INVALID_ARGUMENT, "sv_window_plan: negative size");
  if (n > (1 << 25)) SV_FAIL(SV_ERR_UNSUPPORTED, "sv_window_plan: at most 2^25 rows");
  if (n == 0) return SV_OK;
  if (!coords || !perm || !offsets || !plan || groups < 1 || !aligned16(coords) || !aligned16(plan))
    SV_FAIL(SV_ERR_INVALID_ARGUMENT, "sv_window_plan: null or misaligned pointer, or no group");
  window_plan_kernel<<<(unsigned)((n + 255) / 256), 256, 0, to_stream(stream)>>>(
      coords, perm, offsets, groups, n, static_cast<PlanRow*>(plan), status);
  SV_LAUNCH_CHECK();
  return SV_OK;
}

extern "C" int sv_window_attention(const void* q, const void* k, const void* v,
                                   const int64_t* strides, int64_t n, int heads, int dim,
                                   int dtype, const void* plan, const void* table, int buckets,
                                   const int32_t* lut, int reach, float scale, void* out,
                                   float* lse, sv_stream_t stream) {
  const int rc = check(n, heads, dim, dtype, buckets, reach, "sv_window_attention");
  if (rc != SV_OK) return rc;
  if (n == 0 || heads == 0 || dim == 0) return SV_OK;
  if (!q || !k || !v || !strides || !plan || !table || !lut || !out || !aligned16(plan))
    SV_FAIL(SV_ERR_INVALID_ARGUMENT, "sv_window_attention: null pointer");
  AttnArgs a{};
  a.q = q; a.k = k; a.v = v; a.out = out;
  a.q_row = strides[0]; a.q_head = strides[1];
  a.k_row = strides[2]; a.k_head = strides[3];
  a.v_row = strides[4]; a.v_head = strides[5];
  a.plan = static_cast<const PlanRow*>(plan);
  a.table = table; a.lut = lut; a.lse = lse;
  a.n = n; a.heads = heads; a.dim = dim; a.nb = buckets; a.reach = reach; a.scale = scale;
  cudaStream_t s = to_stream(stream);
  if (dtype == SV_FLOAT32) return forward_typed<float>(a, s);
  if (dtype == SV_FLOAT16) return forward_typed<__half>(a, s);
  return forward_typed<__nv_bfloat16>(a, s);
}

extern "C" size_t sv_window_attention_backward_workspace_bytes(int64_t n, int heads, int buckets) {
  if (n < 0 || heads < 0 || buckets < 1 || buckets > ATTN_MAX_BUCKETS) return 0;
  return layout(n, heads, buckets).total;
}

extern "C" int sv_window_attention_backward(
    const void* q, const void* k, const void* v, const int64_t* strides, const void* o,
    const void* dout, const float* lse, int64_t n, int heads, int dim, int dtype, const void* plan,
    const void* table, int buckets, const int32_t* lut, int reach, float scale, void* dq, void* dk,
    void* dv, void* dtable, void* workspace, size_t workspace_bytes, sv_stream_t stream) {
  const int rc = check(n, heads, dim, dtype, buckets, reach, "sv_window_attention_backward");
  if (rc != SV_OK) return rc;
  cudaStream_t s = to_stream(stream);
  const size_t cells = (size_t)heads * buckets * buckets * buckets;
  if (n == 0 || heads == 0 || dim == 0) {
    if (dtable && cells) SV_CUDA_TRY(cudaMemsetAsync(dtable, 0, cells * dtype_size(dtype), s));
    return SV_OK;
  }
  if (!q || !k || !v || !strides || !o || !dout || !lse || !plan || !table || !lut || !dq || !dk ||
      !dv || !aligned16(plan))
    SV_FAIL(SV_ERR_INVALID_ARGUMENT, "sv_window_attention_backward: null pointer");
  const Layout l = layout(n, heads, buckets);
  if (!workspace || workspace_bytes < l.total || !aligned16(workspace))
    SV_FAIL(SV_ERR_WORKSPACE, "sv_window_attention_backward: workspace too small or unaligned");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  AttnArgs a{};
  a.q = q; a.k = k; a.v = v; a.o = o; a.dout = dout;
  a.q_row = strides[0]; a.q_head = strides[1];
  a.k_row = strides[2]; a.k_head = strides[3];
  a.v_row = strides[4]; a.v_head = strides[5];
  a.dq = dq; a.dk = dk; a.dv = dv;
  a.plan = static_cast<const PlanRow*>(plan);
  a.table = table; a.lut = lut; a.lse = const_cast<float*>(lse);
  a.delta = reinterpret_cast<float*>(ws + l.delta);
  a.n = n; a.heads = heads; a.dim = dim; a.nb = buckets; a.reach = reach; a.scale = scale;
  unsigned* norms = reinterpret_cast<unsigned*>(ws + l.norms);
  a.norms = norms;
  if (dtable) {
    a.dtable = reinterpret_cast<unsigned long long*>(ws + l.table);
    SV_CUDA_TRY(cudaMemsetAsync(ws, 0, l.delta, s));  // the table and the norms
  }
  if (dtype == SV_FLOAT32) return backward_typed<float>(a, norms, dtable, s);
  if (dtype == SV_FLOAT16) return backward_typed<__half>(a, norms, dtable, s);
  return backward_typed<__nv_bfloat16>(a, norms, dtable, s);
}
