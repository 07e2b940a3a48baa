// Windowed attention with a learned relative position bias: what its kernels share.
#pragma once

#include <limits.h>

#include <type_traits>

#include "common.cuh"

namespace sv {

constexpr int ATTN_MAX_DIM = 128;
constexpr int ATTN_MAX_BUCKETS = 25;   // per axis
constexpr int ATTN_MAX_REACH = 1023;   // offsets beyond it share the outermost entries
constexpr int ATTN_MAX_HEADS = 65535;

// attention_tc.cu: the fp16 / bf16 kernels.
struct AttnArgs;
int attention_tc_forward(const AttnArgs& a, bool bf16, cudaStream_t s);
int attention_tc_parts(int64_t n, int heads, int dim, int64_t windows);
// attention_f32.cu: the fp32 ones.
int attention_f32_forward(const AttnArgs& a, cudaStream_t s);
int attention_f32_backward(const AttnArgs& a, void* dtable, cudaStream_t s);
int attention_tc_backward(const AttnArgs& a, bool bf16, void* dtable, cudaStream_t s);

// One row of the attention plan, in window order: the coordinates, the window's range of
// positions, and the feature row.
struct alignas(16) PlanRow {
  int32_t x, y, z;
  int32_t row;    // -1: not a row of the tensor (reported when the plan was built)
  int32_t start, end;
  int32_t span;   // the window's largest extent along an axis
  int32_t pad;
};
static_assert(sizeof(PlanRow) == 32, "sv_window_plan writes 32 bytes a row");

// Behind the rows: the blocks of at most 64 and at most 128 positions that the fp16 / bf16 kernels
// take, each {first position, positions} and in no particular order. A window of more than half a
// block has blocks of its own; smaller ones that start in the same stretch of half a block share one.
// So all rows of a block of a large window see the same positions: against blocks of 64 or 128
// consecutive positions, whichever windows those cut, 84% instead of 60% of the tiles need no mask,
// and no warp waits for another window's tiles.
struct PlanBlocks {
  int64_t count, block[2], cap[2], total;  // byte offsets of int32 [2] and int2 [cap]; 64, 128
};
__host__ __device__ inline PlanBlocks plan_blocks(int64_t n) {
  PlanBlocks b;
  b.count = n * (int64_t)sizeof(PlanRow);
  // at most 2 n / B blocks of large windows, and one of small ones per stretch of B / 2
  b.cap[0] = n / 16 + 2;
  b.cap[1] = n / 32 + 2;
  b.block[0] = b.count + 16;
  b.block[1] = b.block[0] + (b.cap[0] + 1) / 2 * 16;
  b.total = b.block[1] + (b.cap[1] + 1) / 2 * 16;
  return b;
}

struct AttnArgs {
  const void *q, *k, *v, *o, *o_rest, *dout;  // [n, heads, dim], the last axis contiguous
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;  // strides in elements
  void *out, *out_rest, *dq, *dk, *dv;        // contiguous [n, heads, dim]
  const PlanRow* plan;               // [n]
  const void* table;                 // [heads, nb, nb, nb]
  const int32_t* lut;                // [2 * reach + 1]
  float2* stats;                     // [heads, n] by position: the softmax's maximum and 1 / sum
  float* delta;                      // [heads, n] by position: sum_d dout * o
  unsigned long long* dtable;        // [heads, nb^3] fixed point, or null
  unsigned* norms;                   // [heads, 2]: bits of max |dout_i|^2 and max |v_j|^2 (fp32)
  unsigned* tops;                    // [heads, nb^3]: bits of each bucket's max |dS| (fp16 / bf16)
  float2* part_stats;                // parts > 1: [parts, heads, n] by position, base and sum
  float* part_out;                   // and [parts, heads, n, dim], not yet divided by the sum
  int64_t n;
  int heads, dim, nb, reach;
  int parts;                         // of every block's positions (fp16 / bf16 forward pass)
  float scale;
};

#ifdef __CUDACC__
// Difference of two coordinates without wrap-around.
__device__ __forceinline__ int sub_sat(int a, int b) {
  int d;
  asm("sub.sat.s32 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

__device__ __forceinline__ int lut_at(const AttnArgs& a, int d) {
  const int v = __ldg(a.lut + max(-a.reach, min(a.reach, d)) + a.reach);
  return max(0, min(a.nb - 1, v));
}

// The bias table's fixed-point unit for a head: sums of |dS| over a row are at most
// 2 max|dout_i| max|v_j| (a softmax row sums to one and delta is a mean of the products it is
// subtracted from), so n rows of them stay below 2^62 in units of 2^-exponent. Integer sums do not
// depend on the order of the additions. INT_MAX when the bound is not finite.
__device__ __forceinline__ int dtable_exponent(const AttnArgs& a, int head) {
  const float g2 = __uint_as_float(a.norms[2 * head]), v2 = __uint_as_float(a.norms[2 * head + 1]);
  const double bound = 2.0 * sqrt((double)g2) * sqrt((double)v2) * (double)a.n;
  if (!(bound < 1e300)) return INT_MAX;
  if (bound == 0.0) return 0;
  int e;
  frexp(bound, &e);  // bound < 2^e
  return 61 - e;
}
// A row's softmax: maximum and 1 / sum, kept apart because their joint logarithm would lose the sum
// next to scores of the type's lowest value. A row whose every score is -inf has weights of zero.
__device__ __forceinline__ float2 row_stats(float top, float sum) {
  return sum == 0.f ? make_float2(0.f, 0.f) : make_float2(top, 1.0f / sum);
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

// A row that sees one position has a weight of one whatever its score, so its score gradient is zero;
// dP - delta, which the passes round differently, would leave a trace of rounding errors.
__device__ __forceinline__ bool lone(const PlanRow& r) { return r.end - r.start == 1; }

constexpr int ATTN_CH = ATTN_MAX_DIM / 32;  // channels a lane sums

// What rounding `x` to T left out, to be rounded itself: nothing for fp32, nor next to an overflow. For
// fp16 it is 2^11 times that, no larger than x: as it is, it would be lost below the type's smallest
// numbers wherever |x| is below 2^-14.
template <typename T>
constexpr float REST_RAISE = std::is_same<T, __half>::value ? 2048.f : 1.f;
template <typename T>
__device__ __forceinline__ float rest_of(float x) {
  const float r = x - to_f32(from_f32<T>(x));
  return fabsf(r) < INFINITY ? r * REST_RAISE<T> : 0.f;
}
// x again, from its rounded value and a stored rest.
template <typename T>
__device__ __forceinline__ float whole_of(T x, T rest) {
  return fmaf(to_f32(rest), 1.f / REST_RAISE<T>, to_f32(x));
}

// ---- one row of one head computed again, by a warp: lanes along the other side's rows for the
// ---- scores, along the head's channels for the sums, fp32 throughout

// Scores as the kernel keeps them: natural (fp32 path), or times log2(e) for the fp16 / bf16 kernels,
// whose statistics the rows computed again share.
constexpr float ATTN_LOG2E = 1.4426950408889634f;
// x log2(e), finite for every finite x: the type's lowest value stays a score like any other.
__device__ __forceinline__ float times_log2e(float x) {
  const float y = x * ATTN_LOG2E;
  return fabsf(x) < INFINITY ? fminf(fmaxf(y, -3.402823466e38f), 3.402823466e38f) : y;
}
template <bool LOG2>
__device__ __forceinline__ float score_of(float s) { return LOG2 ? times_log2e(s) : s; }
template <bool LOG2>
__device__ __forceinline__ float weight_of(float d) { return LOG2 ? exp2f(d) : expf(d); }

// `s_q`: ATTN_MAX_DIM floats of the warp's own.
template <typename T, bool LOG2>
__device__ void row_forward(const AttnArgs& a, int64_t p, int h, float* s_q) {
  const int lane = threadIdx.x & 31;
  const PlanRow me = plan_at(a.plan, p);
  if (me.row < 0) return;
  const T* q = static_cast<const T*>(a.q) + me.row * a.q_row + h * a.q_head;
  const T* k = static_cast<const T*>(a.k) + h * a.k_head;
  const T* v = static_cast<const T*>(a.v) + h * a.v_head;
  const T* table = static_cast<const T*>(a.table) + (int64_t)h * a.nb * a.nb * a.nb;
  for (int d = lane; d < a.dim; d += 32) s_q[d] = to_f32(q[d]) * a.scale;
  __syncwarp();
  float o[ATTN_CH] = {}, top = -INFINITY, sum = 0.f;
  for (int j0 = me.start; j0 < me.end; j0 += 32) {
    const int j = j0 + lane;
    float s = -INFINITY;
    int row = -1;
    if (j < me.end) {
      const PlanRow key = plan_at(a.plan, j);
      row = key.row;
      if (row >= 0)
        s = score_of<LOG2>(dot_row(s_q, k + row * a.k_row, a.dim) +
                           to_f32(table[bucket_of(a, me, key)]));
    }
    const float m = fmaxf(top, warp_max(s));
    const float base = m == -INFINITY ? 0.f : m;
    const float keep = weight_of<LOG2>(top - base);
    const float e = weight_of<LOG2>(s - base);
    sum = sum * keep + warp_sum(e);
#pragma unroll
    for (int c = 0; c < ATTN_CH; ++c) o[c] *= keep;
    const int count = min(32, me.end - j0);
    for (int i = 0; i < count; ++i) {
      const float w = __shfl_sync(0xffffffffu, e, i);
      const int r = __shfl_sync(0xffffffffu, row, i);
      if (r < 0) continue;
#pragma unroll
      for (int c = 0; c < ATTN_CH; ++c) {
        const int d = lane + 32 * c;
        if (d < a.dim) o[c] = fmaf(w, to_f32(v[r * a.v_row + d]), o[c]);
      }
    }
    top = m;
  }
  const int64_t own = (me.row * (int64_t)a.heads + h) * a.dim;
  T* out = static_cast<T*>(a.out) + own;
#pragma unroll
  for (int c = 0; c < ATTN_CH; ++c) {
    const int d = lane + 32 * c;
    const float x = sum == 0.f ? 0.f : o[c] / sum;
    if (d < a.dim) out[d] = from_f32<T>(x);
    if (d < a.dim && a.out_rest)
      static_cast<T*>(a.out_rest)[own + d] = from_f32<T>(rest_of<T>(x));
  }
  if (lane == 0 && a.stats) a.stats[h * a.n + p] = row_stats(top, sum);
  __syncwarp();
}

// dq of a query. `scratch`: 2 * ATTN_MAX_DIM.
template <typename T, bool LOG2>
__device__ void row_dq(const AttnArgs& a, int64_t p, int h, float* scratch) {
  const int lane = threadIdx.x & 31;
  const PlanRow me = plan_at(a.plan, p);
  if (me.row < 0) return;
  float *s_q = scratch, *s_g = scratch + ATTN_MAX_DIM;
  const int64_t own = (me.row * (int64_t)a.heads + h) * a.dim;
  const T* q = static_cast<const T*>(a.q) + me.row * a.q_row + h * a.q_head;
  const T* k = static_cast<const T*>(a.k) + h * a.k_head;
  const T* v = static_cast<const T*>(a.v) + h * a.v_head;
  const T* g = static_cast<const T*>(a.dout) + own;
  const T* o = static_cast<const T*>(a.o) + own;
  const T* o_rest = a.o_rest ? static_cast<const T*>(a.o_rest) + own : nullptr;
  const T* table = static_cast<const T*>(a.table) + (int64_t)h * a.nb * a.nb * a.nb;
  float delta = 0.f;
  for (int d = lane; d < a.dim; d += 32) {
    s_q[d] = to_f32(q[d]) * a.scale;
    s_g[d] = to_f32(g[d]);
    delta = fmaf(s_g[d], o_rest ? whole_of(o[d], o_rest[d]) : to_f32(o[d]), delta);
  }
  delta = warp_sum(delta);
  __syncwarp();
  const float2 stats = a.stats[h * a.n + p];
  float acc[ATTN_CH] = {};
  const int end = lone(me) ? me.start : me.end;
  for (int j0 = me.start; j0 < end; j0 += 32) {
    const int j = j0 + lane;
    float ds = 0.f;
    int row = -1;
    if (j < end) {
      const PlanRow key = plan_at(a.plan, j);
      row = key.row;
      if (row >= 0) {
        const float s = score_of<LOG2>(dot_row(s_q, k + row * a.k_row, a.dim) +
                                       to_f32(table[bucket_of(a, me, key)]));
        const float dp = dot_row(s_g, v + row * a.v_row, a.dim);
        ds = weight_of<LOG2>(s - stats.x) * stats.y * (dp - delta);
      }
    }
    const int count = min(32, end - j0);
    for (int i = 0; i < count; ++i) {
      const float w = __shfl_sync(0xffffffffu, ds, i);
      const int r = __shfl_sync(0xffffffffu, row, i);
      if (r < 0) continue;
#pragma unroll
      for (int c = 0; c < ATTN_CH; ++c) {
        const int d = lane + 32 * c;
        if (d < a.dim) acc[c] = fmaf(w, to_f32(k[r * a.k_row + d]), acc[c]);
      }
    }
  }
#pragma unroll
  for (int c = 0; c < ATTN_CH; ++c) {
    const int d = lane + 32 * c;
    if (d < a.dim) static_cast<T*>(a.dq)[own + d] = from_f32<T>(acc[c] * a.scale);
  }
  __syncwarp();
}

// dk and dv of a key. `scratch`: 2 * ATTN_MAX_DIM.
template <typename T, bool LOG2>
__device__ void row_dkv(const AttnArgs& a, int64_t p, int h, float* scratch) {
  const int lane = threadIdx.x & 31;
  const PlanRow me = plan_at(a.plan, p);
  if (me.row < 0) return;
  float *s_k = scratch, *s_v = scratch + ATTN_MAX_DIM;
  const T* q = static_cast<const T*>(a.q) + h * a.q_head;
  const T* k = static_cast<const T*>(a.k) + me.row * a.k_row + h * a.k_head;
  const T* v = static_cast<const T*>(a.v) + me.row * a.v_row + h * a.v_head;
  const T* g = static_cast<const T*>(a.dout) + (int64_t)h * a.dim;
  const int64_t g_row = (int64_t)a.heads * a.dim;
  const T* table = static_cast<const T*>(a.table) + (int64_t)h * a.nb * a.nb * a.nb;
  for (int d = lane; d < a.dim; d += 32) {
    s_k[d] = to_f32(k[d]) * a.scale;
    s_v[d] = to_f32(v[d]);
  }
  __syncwarp();
  float dk[ATTN_CH] = {}, dv[ATTN_CH] = {};
  for (int i0 = me.start; i0 < me.end; i0 += 32) {
    const int i = i0 + lane;
    float w = 0.f, ds = 0.f;
    int row = -1;
    if (i < me.end) {
      const PlanRow query = plan_at(a.plan, i);
      row = query.row;
      if (row >= 0) {
        const float2 stats = a.stats[h * a.n + i];
        const float s = score_of<LOG2>(dot_row(s_k, q + row * a.q_row, a.dim) +
                                       to_f32(table[bucket_of(a, query, me)]));
        w = weight_of<LOG2>(s - stats.x) * stats.y;
        if (!lone(me)) ds = w * (dot_row(s_v, g + row * g_row, a.dim) - a.delta[h * a.n + i]);
      }
    }
    const int count = min(32, me.end - i0);
    for (int t = 0; t < count; ++t) {
      const float pw = __shfl_sync(0xffffffffu, w, t);
      const float dw = __shfl_sync(0xffffffffu, ds, t);
      const int r = __shfl_sync(0xffffffffu, row, t);
      if (r < 0) continue;
#pragma unroll
      for (int c = 0; c < ATTN_CH; ++c) {
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
  for (int c = 0; c < ATTN_CH; ++c) {
    const int d = lane + 32 * c;
    if (d < a.dim) {
      static_cast<T*>(a.dk)[own + d] = from_f32<T>(dk[c] * a.scale);
      static_cast<T*>(a.dv)[own + d] = from_f32<T>(dv[c]);
    }
  }
  __syncwarp();
}
#endif

}  // namespace sv
