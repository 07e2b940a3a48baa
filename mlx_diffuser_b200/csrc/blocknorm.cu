// The border between two blocks of a transformer, one pass over the rows in each direction.
//
//     d = drop(branch),  u = N(d) * wb  (d itself without a norm behind the branch)
//     h = round(x + alpha * gate[b] * u)
//     y = (N(h) * w + beta) * (1 + scale[b]) + shift[b]
//     N(v) = (v - mean) * rstd (layer) or v * rstd (rms), rstd = 1 / sqrt(mean square + eps)
//
// h is the residual stream that goes on, rounded to the feature type before it is normed. With n = N(h),
// a = w (1 + scale) and gg = alpha gate wb, the gradients are
//     D  = dh + rstd (dy a - mean(dy a) - n mean(dy a n))      the gradient of h, and of x
//     dd = rstd_d (gg D - mean(gg D) - N(d) mean(gg D N(d))),  dbranch = drop(dd)
// (without the means of the first order for rms), and three sums over the rows of each batch element,
//     A = sum dy n,  B = sum dy,  E = sum D N(d),
// give all the others: dshift = B, dscale = w A + beta B, dgate = alpha wb E, and over the batch elements
// dw = sum (1 + scale) A, dbeta = sum (1 + scale) B, dwb = sum alpha gate E.
//
// The passes move 4 and 6 values an element and do 14 and 30 operations: HBM's bytes and the instructions
// around them bound the passes alike. 40,662 x 1024 bf16, both norms, forward: 60 us (5.5 TB/s); 20,331
// rows, layer norm, gate and modulation, forward / backward: 32 / 51 us, with dropout 43 / 68. A row
// lives in the registers of TPR threads, J accesses of V elements each, or of a warp. The sums have a fixed order:
// the backward pass walks the rows by batch element (a stable counting sort of their indices), cut into
// pieces; a block holds the three sums of its piece in registers and writes them out once.
#include <algorithm>

#include "dropout.cuh"
#include "group.h"
#include "rows.cuh"

namespace sv {
namespace {

constexpr int BN_MAX_CHANNELS = 8192;
constexpr int BN_CHUNKS = BN_MAX_CHANNELS / 32;

// A row or rows of coefficients in any float type; null: the neutral value.
struct Coef {
  const void* p;
  int64_t stride;  // elements between batch elements; 0: one row for all
  int dtype;
};

struct BlockArgs {
  int64_t n;
  int channels;
  const void* x;
  int64_t x_stride;
  const void* branch;
  int64_t branch_stride;
  bool layer, branch_norm;
  float alpha, eps;
  Coef weight, bias, branch_weight, gate, scale, shift;
  bool per_batch;         // otherwise every row is batch element 0
  const int32_t* coords;  // [n][4]
  int64_t batch;
  Dropout drop;
  void* h;
  void* y;
  float4* stats;  // of h and of d: mean, rstd; or null
  int32_t* status;
};

struct BackArgs {
  BlockArgs f;  // h is read; x and y are not used
  const void* dy;
  const void* dh;
  void* dx;
  void* dbranch;
  const int32_t* perm;     // rows by batch element, or null: as they are
  const int32_t* offsets;  // [batch + 1], or null: one group
  int piece;               // rows of a piece
  float* partial;          // [pieces][3][C], or null: no sums are wanted
  int* done;               // BN_CHUNKS counters, set to zero
  int* starts;             // [batch + 1], or null: the first piece of each batch element that has rows
  bool want_e;
};

template <int V>
__device__ __forceinline__ void load_coef(const Coef& c, int64_t b, int col, float neutral,
                                          float (&v)[V]) {
  if (c.p == nullptr) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = neutral;
    return;
  }
  const int64_t at = b * c.stride + col;
  if (c.dtype == SV_FLOAT32) {
    const float* p = static_cast<const float*>(c.p) + at;
    if constexpr (V == 8) {
      const float4 lo = __ldg(reinterpret_cast<const float4*>(p));
      const float4 hi = __ldg(reinterpret_cast<const float4*>(p) + 1);
      v[0] = lo.x; v[1] = lo.y; v[2] = lo.z; v[3] = lo.w;
      v[4] = hi.x; v[5] = hi.y; v[6] = hi.z; v[7] = hi.w;
    } else {
      v[0] = __ldg(p);
    }
    return;
  }
  const uint16_t* p = static_cast<const uint16_t*>(c.p) + at;
  alignas(16) uint16_t e[V];
  if constexpr (V == 8)
    *reinterpret_cast<uint4*>(e) = __ldg(reinterpret_cast<const uint4*>(p));
  else
    e[0] = __ldg(p);
#pragma unroll
  for (int i = 0; i < V; ++i)
    v[i] = c.dtype == SV_FLOAT16 ? __half2float(__ushort_as_half(e[i]))
                                 : __uint_as_float((uint32_t)e[i] << 16);
}

__device__ __forceinline__ float coef_at(const Coef& c, int64_t b, int col, float neutral) {
  float v[1];
  load_coef<1>(c, b, col, neutral, v);
  return v[0];
}

// V elements of a row as they are in memory, so that the next row's can be on their way while this one's
// are worked on.
template <typename T, int V>
struct Raw {
  alignas(V == 8 ? 16 : sizeof(T)) T e[V];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (V == 8) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(e) / 16; ++i)
        reinterpret_cast<uint4*>(e)[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    } else {
      e[0] = __ldg(p);
    }
  }
  __device__ __forceinline__ void clear() {
    if constexpr (V == 8) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(e) / 16; ++i)
        reinterpret_cast<uint4*>(e)[i] = make_uint4(0u, 0u, 0u, 0u);
    } else {
      e[0] = from_f32<T>(0.0f);
    }
  }
  __device__ __forceinline__ void unpack(float (&v)[V]) const {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = to_f32(e[i]);
  }
};

template <typename T, int V, int J, int TPR>
__device__ __forceinline__ void load_row(Raw<T, V> (&raw)[J], const void* p, int64_t at, bool in,
                                         int channels, int t) {
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int c = (j * TPR + t) * V;
    if (in && c < channels) raw[j].load(static_cast<const T*>(p) + at + c);
    else raw[j].clear();
  }
}
template <typename T, int V, int J>
__device__ __forceinline__ void unpack_row(const Raw<T, V> (&raw)[J], float (&v)[J][V]) {
#pragma unroll
  for (int j = 0; j < J; ++j) raw[j].unpack(v[j]);
}

template <typename T, int V>
__device__ __forceinline__ void store_row(T* p, const float (&v)[V]) {
  if constexpr (V == 8) {
    uint4 w[sizeof(T) / 2];
    pack_eight<T>(v, w);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(p)[i] = w[i];
  } else {
    *p = from_f32<T>(v[0]);
  }
}

template <int TPR>
constexpr int kThreads = TPR > 128 ? TPR : 128;

// Sums of W values over the TPR threads of a row, the same in all of them. Rows of more than a warp meet
// in `part`, two buffers in turn: the next sum but one writes a buffer again only after every thread has
// passed the barrier in between, so one barrier a sum is enough.
template <int TPR>
struct RowSum {
  float2* part;  // [2][warps of the block]
  int turn;
  template <int W>
  __device__ __forceinline__ void add(float (&v)[W]) {
#pragma unroll
    for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1)
#pragma unroll
      for (int w = 0; w < W; ++w) v[w] += __shfl_xor_sync(0xffffffffu, v[w], o);
    if constexpr (TPR > 32) {
      constexpr int ALL = kThreads<TPR> / 32, WARPS = TPR / 32;
      float2* to = part + turn * ALL;
      turn ^= 1;
      const int warp = threadIdx.x >> 5;
      if ((threadIdx.x & 31) == 0) to[warp] = make_float2(v[0], v[W - 1]);
      __syncthreads();
      const int first = warp / WARPS * WARPS;
      float2 all = to[first];
#pragma unroll
      for (int i = 1; i < WARPS; ++i) {
        all.x += to[first + i].x;
        all.y += to[first + i].y;
      }
      v[W - 1] = all.y;
      v[0] = all.x;
    }
  }
  __device__ __forceinline__ float one(float a) {
    float v[1] = {a};
    add(v);
    return v[0];
  }
  __device__ __forceinline__ float2 two(float a, float b) {
    float v[2] = {a, b};
    add(v);
    return make_float2(v[0], v[1]);
  }
};

// The row's channel of a thread's access j.
template <int V, int TPR>
__device__ __forceinline__ int column(int j, int t) {
  return (j * TPR + t) * V;
}

// Which of a thread's elements are kept, bit i of word j: the V elements of access j.
template <int V, int J, int TPR>
__device__ __forceinline__ void kept_row(uint32_t (&kept)[J], int64_t row, int channels, int t,
                                         const PhiloxKeys& keys, const Dropout& d) {
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int c = (j * TPR + t) * V;
    kept[j] = 0u;
    if (c >= channels) continue;
    const uint64_t at = (uint64_t)row * channels + c;
    kept[j] = V == 8 ? kept_eight(philox(at >> 3, d.subsequence, keys), d) : kept_one(at, keys, d);
  }
}
template <int V, int J>
__device__ __forceinline__ void drop_row(float (&v)[J][V], const uint32_t (&kept)[J], float scale) {
#pragma unroll
  for (int j = 0; j < J; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) v[j][i] = kept[j] >> i & 1u ? v[j][i] * scale : 0.0f;
}

// mean and rstd of a row in registers (zeros behind the last channel).
template <int V, int J, int TPR>
__device__ __forceinline__ float2 row_stats(const float (&v)[J][V], int t, int channels, bool layer,
                                            float eps, RowSum<TPR>& sum) {
  const float inv = 1.0f / (float)channels;
  float mean = 0.0f;
  if (layer) {
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) s += v[j][i];
    mean = sum.one(s) * inv;
  }
  float q = 0.0f;
#pragma unroll
  for (int j = 0; j < J; ++j)
    if (column<V, TPR>(j, t) < channels) {
#pragma unroll
      for (int i = 0; i < V; ++i) q = fmaf(v[j][i] - mean, v[j][i] - mean, q);
    }
  return make_float2(mean, rsqrtf(fmaf(sum.one(q), inv, eps)));
}

__device__ __forceinline__ int64_t batch_of(const BlockArgs& a, int64_t row) {
  if (!a.per_batch) return 0;
  const int64_t b = __ldg(a.coords + row * 4);
  return b >= 0 && b < a.batch ? b : -1;
}

template <typename T, int V, int J, int TPR>
__global__ void __launch_bounds__(kThreads<TPR>)
    block_norm_kernel(const __grid_constant__ BlockArgs a) {
  constexpr int ROWS = kThreads<TPR> / TPR;
  // up to two accesses a thread: the coefficients of a batch element stay in registers, and the next row
  // is loaded while this one is worked on
  constexpr bool KEEP = J <= 2;
  __shared__ float2 part[2 * kThreads<TPR> / 32];
  RowSum<TPR> sum{part, 0};
  const int t = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const int C = a.channels;
  PhiloxKeys keys(a.drop.cut ? seed_of(a.drop) : 0);
  keys.held();
  float gg[J][V], mul[J][V], add[J][V];
  int64_t held = -2, b_next = -2;
  Raw<T, V> raw_x[J], raw_d[J];
  auto fetch = [&](int64_t row) {
    const bool in = row < a.n;
    load_row<T, V, J, TPR>(raw_x, a.x, row * a.x_stride, in, C, t);
    load_row<T, V, J, TPR>(raw_d, a.branch, row * a.branch_stride, in, C, t);
    if (in) b_next = batch_of(a, row);
  };
  const int64_t step = (int64_t)gridDim.x * ROWS;
  if constexpr (KEEP) fetch((int64_t)blockIdx.x * ROWS + group);
  for (int64_t r0 = (int64_t)blockIdx.x * ROWS; r0 < a.n; r0 += step) {
    const int64_t row = r0 + group;
    const bool in = row < a.n;
    float x[J][V], d[J][V];
    if constexpr (!KEEP) fetch(row);
    unpack_row(raw_x, x);
    unpack_row(raw_d, d);
    const int64_t b = in ? b_next : held;
    if constexpr (KEEP) fetch(row + step);
    if (b == -1 && in && t == 0) report(a.status, SV_DEVICE_BAD_INDEX);
    // a row without a batch element is not modulated
    auto coefs = [&](int j, float (&g)[V], float (&m)[V], float (&s)[V]) {
      const int c = column<V, TPR>(j, t);
      if (c >= C) return;
      float w[V], beta[V], wb[V];
      load_coef(a.weight, 0, c, 1.0f, w);
      load_coef(a.bias, 0, c, 0.0f, beta);
      load_coef(a.branch_weight, 0, c, 1.0f, wb);
      if (b >= 0) {
        load_coef(a.gate, b, c, 1.0f, g);
        load_coef(a.scale, b, c, 0.0f, m);
        load_coef(a.shift, b, c, 0.0f, s);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (b < 0) g[i] = 1.0f, m[i] = s[i] = 0.0f;
        g[i] *= a.alpha * wb[i];
        s[i] = fmaf(beta[i], 1.0f + m[i], s[i]);
        m[i] = w[i] * (1.0f + m[i]);
      }
    };
    if (KEEP && b != held) {
      held = b;
#pragma unroll
      for (int j = 0; j < J; ++j) coefs(j, gg[j], mul[j], add[j]);
    }
    if (a.drop.cut) {
      uint32_t kept[J];
      kept_row<V, J, TPR>(kept, row, C, t, keys, a.drop);
      drop_row<V, J>(d, kept, a.drop.scale);
    }
    float2 sd = make_float2(0.0f, 1.0f);
    if (a.branch_norm) sd = row_stats<V, J, TPR>(d, t, C, a.layer, a.eps, sum);
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int c = column<V, TPR>(j, t);
      if constexpr (!KEEP) coefs(j, gg[0], mul[0], add[0]);
      if (c < C) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float u = (d[j][i] - sd.x) * sd.y;
          x[j][i] = to_f32(from_f32<T>(fmaf(gg[KEEP ? j : 0][i], u, x[j][i])));
        }
        if (in) store_row<T, V>(static_cast<T*>(a.h) + row * C + c, x[j]);
      }
    }
    const float2 sh = row_stats<V, J, TPR>(x, t, C, a.layer, a.eps, sum);
    if (a.stats && in && t == 0) a.stats[row] = make_float4(sh.x, sh.y, sd.x, sd.y);
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int c = column<V, TPR>(j, t);
      if constexpr (!KEEP) coefs(j, gg[0], mul[0], add[0]);
      if (in && c < C) {
#pragma unroll
        for (int i = 0; i < V; ++i)
          x[j][i] = fmaf((x[j][i] - sh.x) * sh.y, mul[KEEP ? j : 0][i], add[KEEP ? j : 0][i]);
        store_row<T, V>(static_cast<T*>(a.y) + row * C + c, x[j]);
      }
    }
  }
}

template <typename T, int V, int J, int TPR>
__global__ void __launch_bounds__(kThreads<TPR>)
    block_norm_backward_kernel(const __grid_constant__ BackArgs a) {
  constexpr int THREADS = kThreads<TPR>, ROWS = THREADS / TPR;
  constexpr bool KEEP = J <= 2;
  __shared__ float2 part[2 * THREADS / 32];
  __shared__ float joined[ROWS > 1 ? THREADS * V * J : 1];
  RowSum<TPR> sum{part, 0};
  const BlockArgs& f = a.f;
  if (a.done && blockIdx.x == 0)
    for (int i = threadIdx.x; i < BN_CHUNKS; i += THREADS) a.done[i] = 0;
  const int t = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const int C = f.channels;
  Piece p{0, 0, 0};
  if (a.offsets) {
    p = find_piece<true>(a.offsets, (int)f.batch, (int)f.n, a.piece, blockIdx.x);
  } else {
    p.first = (int)min((int64_t)blockIdx.x * a.piece, f.n);
    p.last = (int)min((int64_t)p.first + a.piece, f.n);
    if (p.first >= p.last) p.group = -1;
  }
  if (p.group < 0) return;  // the whole block
  if (a.starts && threadIdx.x == 0 && p.first == __ldg(a.offsets + p.group)) a.starts[p.group] = blockIdx.x;
  const int64_t b = p.group < f.batch ? p.group : -1;
  PhiloxKeys keys(f.drop.cut ? seed_of(f.drop) : 0);
  keys.held();
  float gg[J][V], mul[J][V];
  auto coefs = [&](int j, float (&g)[V], float (&m)[V]) {
    const int c = column<V, TPR>(j, t);
    if (c >= C) return;
    float w[V], wb[V];
    load_coef(f.weight, 0, c, 1.0f, w);
    load_coef(f.branch_weight, 0, c, 1.0f, wb);
    if (b >= 0) {
      load_coef(f.gate, b, c, 1.0f, g);
      load_coef(f.scale, b, c, 0.0f, m);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (b < 0) g[i] = 1.0f, m[i] = 0.0f;
      g[i] *= f.alpha * wb[i];
      m[i] = w[i] * (1.0f + m[i]);
    }
  };
  if constexpr (KEEP) {
#pragma unroll
    for (int j = 0; j < J; ++j) coefs(j, gg[j], mul[j]);
  }
  float sum_a[J][V], sum_b[J][V], sum_e[J][V];
#pragma unroll
  for (int j = 0; j < J; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) sum_a[j][i] = sum_b[j][i] = sum_e[j][i] = 0.0f;
  const float inv = 1.0f / (float)C;
  const bool with_d = f.branch_norm || a.want_e;
  Raw<T, V> raw_y[J], raw_h[J], raw_d[J], raw_D[J];
  float4 st_next = make_float4(0.0f, 0.0f, 0.0f, 1.0f);
  auto row_at = [&](int at) {
    const int64_t i = min(at, p.last - 1);
    return a.perm ? (int64_t)__ldg(a.perm + i) : i;
  };
  auto fetch = [&](int64_t row, bool in) {
    load_row<T, V, J, TPR>(raw_y, a.dy, row * C, in && a.dy, C, t);
    load_row<T, V, J, TPR>(raw_h, f.h, row * C, in, C, t);
    load_row<T, V, J, TPR>(raw_d, f.branch, row * f.branch_stride, in && with_d, C, t);
    load_row<T, V, J, TPR>(raw_D, a.dh, row * C, in && a.dh, C, t);
    st_next = in ? __ldg(f.stats + row) : make_float4(0.0f, 0.0f, 0.0f, 1.0f);
  };
  int64_t row_next = row_at(p.first + group), row_after = 0;
  if constexpr (KEEP) {
    row_after = row_at(p.first + ROWS + group);
    fetch(row_next, p.first + group < p.last);
  }
  for (int r0 = p.first; r0 < p.last; r0 += ROWS) {
    const bool in = r0 + group < p.last;
    if constexpr (!KEEP) {
      row_next = row_at(r0 + group);
      fetch(row_next, in);
    }
    const int64_t row = row_next;
    const float4 st = st_next;
    float dy[J][V], n[J][V], d[J][V], D[J][V];
    unpack_row(raw_y, dy);
    unpack_row(raw_h, n);
    unpack_row(raw_d, d);
    unpack_row(raw_D, D);
    if constexpr (KEEP) {
      row_next = row_after;
      fetch(row_next, r0 + ROWS + group < p.last);
      row_after = row_at(r0 + 2 * ROWS + group);
    }
    uint32_t kept[J];  // for the branch and for its gradient
    if (f.drop.cut) {
      kept_row<V, J, TPR>(kept, row, C, t, keys, f.drop);
      drop_row<V, J>(d, kept, f.drop.scale);
    }
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if (column<V, TPR>(j, t) >= C) continue;
      if constexpr (!KEEP) coefs(j, gg[0], mul[0]);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        n[j][i] = (n[j][i] - st.x) * st.y;
        sum_a[j][i] = fmaf(dy[j][i], in ? n[j][i] : 0.0f, sum_a[j][i]);
        sum_b[j][i] += dy[j][i];
        dy[j][i] *= mul[KEEP ? j : 0][i];
        s1 += dy[j][i];
        s2 = fmaf(dy[j][i], n[j][i], s2);
      }
    }
    const float2 m = f.layer ? sum.two(s1, s2) : make_float2(0.0f, sum.one(s2));
    const float m1 = m.x * inv, m2 = m.y * inv;
    s1 = s2 = 0.0f;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int c = column<V, TPR>(j, t);
      if (c >= C) continue;
      if constexpr (!KEEP) coefs(j, gg[0], mul[0]);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        D[j][i] = fmaf(st.y, dy[j][i] - m1 - n[j][i] * m2, D[j][i]);
        d[j][i] = (d[j][i] - st.z) * st.w;
        if (in) sum_e[j][i] = fmaf(D[j][i], d[j][i], sum_e[j][i]);
      }
      if (in && a.dx) store_row<T, V>(static_cast<T*>(a.dx) + row * C + c, D[j]);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        D[j][i] *= gg[KEEP ? j : 0][i];
        if (f.branch_norm) {
          s1 += D[j][i];
          s2 = fmaf(D[j][i], d[j][i], s2);
        }
      }
    }
    if (f.branch_norm) {
      const float2 e = f.layer ? sum.two(s1, s2) : make_float2(0.0f, sum.one(s2));
      const float e1 = e.x * inv, e2 = e.y * inv;
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) D[j][i] = st.w * (D[j][i] - e1 - d[j][i] * e2);
    }
    if (in && a.dbranch) {
      if (f.drop.cut) drop_row<V, J>(D, kept, f.drop.scale);
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int c = column<V, TPR>(j, t);
        if (c < C) store_row<T, V>(static_cast<T*>(a.dbranch) + row * C + c, D[j]);
      }
    }
  }
  if (a.partial == nullptr) return;
  float* to = a.partial + (int64_t)blockIdx.x * 3 * C;
  auto join = [&](const float (&v)[J][V], float* out) {
    if constexpr (ROWS == 1) {
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (column<V, TPR>(j, t) < C) out[column<V, TPR>(j, t) + i] = v[j][i];
    } else {
      __syncthreads();  // the previous sums have been read
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) joined[group * TPR * V * J + column<V, TPR>(j, t) + i] = v[j][i];
      __syncthreads();
      for (int c = threadIdx.x; c < C; c += THREADS) {
        float all = joined[c];
#pragma unroll
        for (int g = 1; g < ROWS; ++g) all += joined[g * TPR * V * J + c];
        out[c] = all;
      }
    }
  };
  join(sum_a, to);
  join(sum_b, to + C);
  join(sum_e, to + 2 * C);
}

// ---- long runs of rows: a pipeline per warp ------------------------------------------------------
//
// A warp has a row to itself (the sums need no barrier), 2 to 4 times 8 elements a lane, and keeps the next
// rows in flight by bulk copies (rows.cuh). The coefficients of one batch element stand in shared
// memory, folded: what differs from row to row is added up in registers, and HBM is not waited for.

// Folded coefficients, planes of four: element c of plane k is at [(k * 2 + c / 4 % 2) * 4 * Q + c / 8 * 4
// + c % 4], so that the lanes' 16-byte accesses of neighbouring eights do not meet in a bank.
template <int J>
struct Folded {
  static constexpr int Q = 32 * J;  // eights of a row
  static constexpr int PLANE = 8 * Q;
  float* at;
  __device__ __forceinline__ void load(int k, int q, float (&v)[8]) const {
    *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(at + (k * 2) * 4 * Q + q * 4);
    *reinterpret_cast<float4*>(v + 4) = *reinterpret_cast<const float4*>(at + (k * 2 + 1) * 4 * Q + q * 4);
  }
  __device__ __forceinline__ void store(int k, int q, const float (&v)[8]) const {
    *reinterpret_cast<float4*>(at + (k * 2) * 4 * Q + q * 4) = *reinterpret_cast<const float4*>(v);
    *reinterpret_cast<float4*>(at + (k * 2 + 1) * 4 * Q + q * 4) = *reinterpret_cast<const float4*>(v + 4);
  }
};

// gate alpha wb; w (1 + scale); beta (1 + scale) + shift: for eight channels of batch element b, b < 0: a
// row without one.
__device__ __forceinline__ void fold(const BlockArgs& a, int64_t b, int c, float (&g)[8], float (&m)[8],
                                     float (&s)[8]) {
  float w[8], beta[8], wb[8];
  load_coef(a.weight, 0, c, 1.0f, w);
  load_coef(a.bias, 0, c, 0.0f, beta);
  load_coef(a.branch_weight, 0, c, 1.0f, wb);
  if (b >= 0) {
    load_coef(a.gate, b, c, 1.0f, g);
    load_coef(a.scale, b, c, 0.0f, m);
    load_coef(a.shift, b, c, 0.0f, s);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (b < 0) g[i] = 1.0f, m[i] = s[i] = 0.0f;
    g[i] *= a.alpha * wb[i];
    s[i] = fmaf(beta[i], 1.0f + m[i], s[i]);
    m[i] = w[i] * (1.0f + m[i]);
  }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename T>
__device__ __forceinline__ void load_eight(const uint8_t* stage, int q, float (&v)[8]) {
  alignas(16) T e[8];
#pragma unroll
  for (int i = 0; i < (int)sizeof(e) / 16; ++i)
    reinterpret_cast<uint4*>(e)[i] = reinterpret_cast<const uint4*>(stage)[q * (sizeof(e) / 16) + i];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = to_f32(e[i]);
}

// x and branch, two rows ahead, and the tables of two batch elements: two blocks an SM of 16-bit rows, or
// one of fp32 rows.
template <typename T, int J>
struct RowsLayout {
  using Ring = RowRing<T, J * (int)sizeof(T) / 2>;  // 32 J eights: as many 16-byte accesses, twice for fp32
  static constexpr int STAGES = 2;
  static constexpr int TABLE = Ring::SMEM(2, STAGES);
  static constexpr int SMEM = TABLE + 6 * Folded<J>::PLANE * 4;
  static_assert(SMEM <= 227 * 1024, "shared memory budget");
};

template <typename T, int J, bool LAYER, bool BRANCH>
__global__ void __launch_bounds__(32 * ROW_WARPS, sizeof(T) == 2 ? 2 : 1)
    block_norm_rows_kernel(const __grid_constant__ BlockArgs a) {
  using L = RowsLayout<T, J>;
  using Ring = typename L::Ring;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int s_abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int C = a.channels;
  const Folded<J> tables{reinterpret_cast<float*>(smem + L::TABLE)};
  if (threadIdx.x == 0) s_abort = 0;
  // The block's rows are neighbours, of one batch element or of two: those of its first and last row have
  // tables. Rows of others fold their coefficients again, waiting for L2: one block that did so for half
  // of its rows took as long as the others' whole pass.
  const int64_t per = (a.n + gridDim.x - 1) / gridDim.x;
  const int64_t first = min(blockIdx.x * per, a.n), last = min(first + per, a.n);
  const int64_t held0 = first < last ? batch_of(a, first) : 0;
  const int64_t held1 = first < last ? batch_of(a, last - 1) : 0;
  for (int q = threadIdx.x; q * 8 < C; q += 32 * ROW_WARPS) {
    float g[8], m[8], s[8];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (i == 1 && held1 == held0) break;
      fold(a, i ? held1 : held0, q * 8, g, m, s);
      tables.store(3 * i, q, g);
      tables.store(3 * i + 1, q, m);
      tables.store(3 * i + 2, q, s);
    }
  }
  __syncthreads();
  int b_lane = 0;  // the batch elements of the warp's next 32 rows, a lane each
  PhiloxKeys keys(a.drop.cut ? seed_of(a.drop) : 0);
  keys.held();
  const float inv = 1.0f / (float)C;
  const bool ok = run_rows<T, J * (int)sizeof(T) / 2, 2, L::STAGES>(
      smem, first + warp, ROW_WARPS, last, C * (int)sizeof(T), 2, &s_abort,
      [](int64_t r, int64_t) { return r; },
      [&](int t, int64_t r) -> const void* {
        return t == 0 ? static_cast<const T*>(a.x) + r * a.x_stride
                      : static_cast<const T*>(a.branch) + r * a.branch_stride;
      },
      [&](int64_t row, int64_t k, const uint8_t* stage, auto&& release) {
        if (a.per_batch && (k & 31) == 0) {
          const int64_t mine = row + lane * ROW_WARPS;
          b_lane = mine < last ? (int)batch_of(a, mine) : 0;
        }
        const int64_t b = __shfl_sync(0xffffffffu, b_lane, (int)(k & 31));
        if (b < 0 && lane == 0) report(a.status, SV_DEVICE_BAD_INDEX);
        const int table = b == held0 ? 0 : b == held1 ? 3 : -1;
        float x[J][8], d[J][8];
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const int q = lane + 32 * j;
          if (q * 8 < C) {
            load_eight<T>(stage, q, x[j]);
            load_eight<T>(stage + Ring::ROW, q, d[j]);
            if (a.drop.cut)
              drop_eight(d[j], philox(((uint64_t)row * C >> 3) + q, a.drop.subsequence, keys), a.drop);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[j][i] = d[j][i] = 0.0f;
          }
        }
        release();
        float dm = 0.0f, dr = 1.0f;
        if constexpr (BRANCH) {
          if constexpr (LAYER) {
            float s = 0.0f;
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
              for (int i = 0; i < 8; ++i) s += d[j][i];
            dm = warp_sum(s) * inv;
          }
          float s = 0.0f;
#pragma unroll
          for (int j = 0; j < J; ++j)
            if ((lane + 32 * j) * 8 < C) {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                if constexpr (LAYER) d[j][i] -= dm;
                s = fmaf(d[j][i], d[j][i], s);
              }
            }
          dr = rsqrtf(fmaf(warp_sum(s), inv, a.eps));
        }
        float hm = 0.0f, s = 0.0f;
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const int q = lane + 32 * j;
          if (q * 8 >= C) continue;
          float g[8], unused[8], other[8];
          if (table >= 0) tables.load(table, q, g);
          else fold(a, b, q * 8, g, unused, other);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            x[j][i] = fmaf(g[i], BRANCH ? d[j][i] * dr : d[j][i], x[j][i]);
          alignas(16) uint4 e[sizeof(T) / 2];
          pack_eight<T>(x[j], e);
          uint4* to = reinterpret_cast<uint4*>(static_cast<T*>(a.h) + row * C + q * 8);
#pragma unroll
          for (int i = 0; i < (int)sizeof(T) / 2; ++i) to[i] = e[i];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            x[j][i] = to_f32(reinterpret_cast<const T*>(e)[i]);
            if constexpr (LAYER) s += x[j][i];
            else s = fmaf(x[j][i], x[j][i], s);
          }
        }
        if constexpr (LAYER) {
          hm = warp_sum(s) * inv;
          s = 0.0f;
#pragma unroll
          for (int j = 0; j < J; ++j)
            if ((lane + 32 * j) * 8 < C) {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                x[j][i] -= hm;
                s = fmaf(x[j][i], x[j][i], s);
              }
            }
        }
        const float hr = rsqrtf(fmaf(warp_sum(s), inv, a.eps));
        if (a.stats && lane == 0) a.stats[row] = make_float4(hm, hr, dm, dr);
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const int q = lane + 32 * j;
          if (q * 8 >= C) continue;
          float unused[8], m[8], add[8];
          if (table >= 0) {
            tables.load(table + 1, q, m);
            tables.load(table + 2, q, add);
          } else {
            fold(a, b, q * 8, unused, m, add);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) m[i] = fmaf(x[j][i] * hr, m[i], add[i]);
          store_row<T, 8>(static_cast<T*>(a.y) + row * C + q * 8, m);
        }
      });
  if (!ok && lane == 0) report(a.status, SV_DEVICE_WAIT_TIMEOUT);
}

// ---- the coefficients' gradients from the pieces' sums -------------------------------------------

struct Grad {
  void* p;
  int64_t stride;  // between batch elements; 0: summed over them
  int dtype;
};
struct SumArgs {
  BlockArgs f;
  const int32_t* offsets;
  int piece;
  const float* partial;
  int groups;   // batch elements, and one for the rows without
  const int* starts;  // block_norm_join_many_kernel: a group's first piece
  float* sums;  // [groups][3][C]
  int* done;    // zeroed by the kernel before
  Grad weight, bias, branch_weight, gate, scale, shift;
};

__device__ __forceinline__ void store_grad(const Grad& g, int64_t b, int c, float v) {
  const int64_t at = b * g.stride + c;
  if (g.dtype == SV_FLOAT32) static_cast<float*>(g.p)[at] = v;
  else if (g.dtype == SV_FLOAT16) static_cast<__half*>(g.p)[at] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(g.p)[at] = __float2bfloat16_rn(v);
}

// What the sums of a group (a batch element, or the rows without one) give one channel, added to `all` and,
// where a gradient has a row per batch element, stored.
struct ChannelSums {
  float dw, dbeta, dwb, dgate, dscale, dshift;
};
__device__ __forceinline__ void add_group(const SumArgs& a, int g, int c, float A, float B, float E,
                                          float w, float beta, float wb, ChannelSums& all) {
  const BlockArgs& f = a.f;
  const bool mod = !f.per_batch || g < f.batch;  // rows without a batch element are not modulated
  const float one = 1.0f + (mod ? coef_at(f.scale, g, c, 0.0f) : 0.0f);
  const float gate = mod ? coef_at(f.gate, g, c, 1.0f) : 1.0f;
  all.dw = fmaf(one, A, all.dw);
  all.dbeta = fmaf(one, B, all.dbeta);
  all.dwb = fmaf(f.alpha * gate, E, all.dwb);
  if (!mod) return;
  const float eg = f.alpha * wb * E, es = fmaf(w, A, beta * B);
  if (a.gate.p && a.gate.stride) store_grad(a.gate, g, c, eg);
  if (a.scale.p && a.scale.stride) store_grad(a.scale, g, c, es);
  if (a.shift.p && a.shift.stride) store_grad(a.shift, g, c, B);
  all.dgate += eg;
  all.dscale += es;
  all.dshift += B;
}
__device__ __forceinline__ void store_channel(const SumArgs& a, int c, const ChannelSums& all) {
  if (a.weight.p) store_grad(a.weight, 0, c, all.dw);
  if (a.bias.p) store_grad(a.bias, 0, c, all.dbeta);
  if (a.branch_weight.p) store_grad(a.branch_weight, 0, c, all.dwb);
  if (a.gate.p && !a.gate.stride) store_grad(a.gate, 0, c, all.dgate);
  if (a.scale.p && !a.scale.stride) store_grad(a.scale, 0, c, all.dscale);
  if (a.shift.p && !a.shift.stride) store_grad(a.shift, 0, c, all.dshift);
}

// What the sums of every batch element give one channel.
__device__ __forceinline__ void finish_channel(const SumArgs& a, int c) {
  const BlockArgs& f = a.f;
  const int C = f.channels;
  ChannelSums all{};
  const float w = coef_at(f.weight, 0, c, 1.0f), beta = coef_at(f.bias, 0, c, 0.0f);
  const float wb = coef_at(f.branch_weight, 0, c, 1.0f);
  for (int g = 0; g < a.groups; ++g) {
    const float* from = a.sums + (int64_t)g * 3 * C + c;  // written by this launch: not through L1
    add_group(a, g, c, __ldcg(from), __ldcg(from + C), __ldcg(from + 2 * C), w, beta, wb, all);
  }
  store_channel(a, c, all);
}

// The sums of a batch element's pieces (blockIdx.y), 32 of the 3 C columns a block: its 32 warps share the
// pieces and are joined in order. The block that ends last then forms the gradients: which one that is
// changes no sum.
__global__ void __launch_bounds__(1024) block_norm_join_kernel(const __grid_constant__ SumArgs a) {
  __shared__ float s[32][33];
  __shared__ bool is_last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t cols = 3 * (int64_t)a.f.channels, c = (int64_t)blockIdx.x * 32 + lane;
  int64_t first = 0, pieces = (a.f.n + a.piece - 1) / a.piece;
  if (a.offsets) {
    for (int g0 = 0; g0 <= (int)blockIdx.y; g0 += 32) {
      const int g = g0 + lane;
      int mine = 0;
      if (g <= (int)blockIdx.y) {
        const int rows = (g < a.f.batch ? __ldg(a.offsets + g + 1) : (int)a.f.n) - __ldg(a.offsets + g);
        mine = (rows + a.piece - 1) / a.piece;
      }
      first += __reduce_add_sync(0xffffffffu, g < (int)blockIdx.y ? mine : 0);
      pieces = __reduce_add_sync(0xffffffffu, g == (int)blockIdx.y ? mine : 0);
    }
  }
  float v = 0.0f;
  if (c < cols) {
    const float* from = a.partial + (first + warp) * cols + c;
#pragma unroll 8
    for (int64_t p = warp; p < pieces; p += 32, from += 32 * cols) v += __ldg(from);
  }
  s[warp][lane] = v;
  __syncthreads();
  if (warp == 0 && c < cols) {
#pragma unroll
    for (int i = 1; i < 32; ++i) v += s[i][lane];
    a.sums[blockIdx.y * cols + c] = v;
    __threadfence();
  }
  __syncthreads();
  if (threadIdx.x == 0) is_last = atomicAdd(a.done, 1) == (int)(gridDim.x * gridDim.y) - 1;
  __syncthreads();
  if (!is_last) return;
  __threadfence();
  for (int i = threadIdx.x; i < a.f.channels; i += 1024) finish_channel(a, i);
}

// The same for many batch elements: 32 channels a block (blockIdx.x), a warp for each of 32 groups
// (blockIdx.y), which adds up the group's pieces in order and stores what has a row per batch element. What is
// summed over the groups is left to the block of these channels that ends last: its warps share the groups and
// are joined in order. With a block for every group and 32 columns, each looking its pieces up, and one
// block for all that follows, 1,000 batch elements of 1024 channels took 5.8 ms (17 us so) and 4,095 of 8192
// took 522 (0.5).
__global__ void __launch_bounds__(1024) block_norm_join_many_kernel(const __grid_constant__ SumArgs a) {
  __shared__ float s[6][32][33];
  __shared__ bool is_last;
  const BlockArgs& f = a.f;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int C = f.channels, c = blockIdx.x * 32 + lane, g = blockIdx.y * 32 + warp;
  const bool in = c < C;
  float w = 0.0f, beta = 0.0f, wb = 0.0f;
  if (in) {
    w = coef_at(f.weight, 0, c, 1.0f);
    beta = coef_at(f.bias, 0, c, 0.0f);
    wb = coef_at(f.branch_weight, 0, c, 1.0f);
  }
  // gradients that are summed over the groups; the others are stored here
  const bool summed = a.weight.p || a.bias.p || a.branch_weight.p || (a.gate.p && !a.gate.stride) ||
                      (a.scale.p && !a.scale.stride) || (a.shift.p && !a.shift.stride);
  if (g < a.groups && in) {
    const int rows = (g < f.batch ? __ldg(a.offsets + g + 1) : (int)f.n) - __ldg(a.offsets + g);
    const int pieces = (rows + a.piece - 1) / a.piece;
    float A = 0.0f, B = 0.0f, E = 0.0f;
    if (pieces > 0) {
      const float* from = a.partial + (int64_t)__ldg(a.starts + g) * 3 * C + c;
#pragma unroll 4
      for (int p = 0; p < pieces; ++p, from += 3 * (int64_t)C) {
        A += __ldg(from);
        B += __ldg(from + C);
        E += __ldg(from + 2 * C);
      }
    }
    if (summed) {
      float* to = a.sums + (int64_t)g * 3 * C + c;
      to[0] = A;
      to[C] = B;
      to[2 * C] = E;
      __threadfence();
    }
    ChannelSums unused{};
    add_group(a, g, c, A, B, E, w, beta, wb, unused);
  }
  if (!summed) return;
  __syncthreads();
  if (threadIdx.x == 0) is_last = atomicAdd(a.done + blockIdx.x, 1) == (int)gridDim.y - 1;
  __syncthreads();
  if (!is_last) return;
  __threadfence();
  ChannelSums all{};
  if (in) {
    SumArgs none = a;  // the rows per batch element are stored already
    none.gate.p = none.scale.p = none.shift.p = nullptr;
    for (int i = warp; i < a.groups; i += 32) {
      const float* from = a.sums + (int64_t)i * 3 * C + c;
      add_group(none, i, c, __ldcg(from), __ldcg(from + C), __ldcg(from + 2 * C), w, beta, wb, all);
    }
  }
  s[0][warp][lane] = all.dw;
  s[1][warp][lane] = all.dbeta;
  s[2][warp][lane] = all.dwb;
  s[3][warp][lane] = all.dgate;
  s[4][warp][lane] = all.dscale;
  s[5][warp][lane] = all.dshift;
  __syncthreads();
  if (warp != 0 || !in) return;
  for (int i = 1; i < 32; ++i) {
    all.dw += s[0][i][lane];
    all.dbeta += s[1][i][lane];
    all.dwb += s[2][i][lane];
    all.dgate += s[3][i][lane];
    all.dscale += s[4][i][lane];
    all.dshift += s[5][i][lane];
  }
  store_channel(a, c, all);
}

// ---- host ----------------------------------------------------------------------------------------

bool float_type(int d) { return d == SV_FLOAT32 || d == SV_FLOAT16 || d == SV_BFLOAT16; }

bool wide_coef(const Coef& c) { return !c.p || (aligned16(c.p) && c.stride % 8 == 0); }

// 16-byte accesses: rows of a multiple of eight elements on 16-byte boundaries. Everything else goes element by
// element, with the coefficients loaded for every row and a generator call an element: 40,662 x 331 bf16
// takes 122 us forward (328 channels: 33), 200 with dropout (43), 246 backward (65).
bool wide_rows(const BlockArgs& a) {
  return a.channels % 8 == 0 && a.x_stride % 8 == 0 && a.branch_stride % 8 == 0 && aligned16(a.x) &&
         aligned16(a.branch) && aligned16(a.h) && aligned16(a.y) && wide_coef(a.weight) &&
         wide_coef(a.bias) && wide_coef(a.branch_weight) && wide_coef(a.gate) &&
         wide_coef(a.scale) && wide_coef(a.shift);
}

template <typename T, int V, int J, int TPR>
int launch_forward(const BlockArgs& a, cudaStream_t s) {
  constexpr int ROWS = kThreads<TPR> / TPR;
  const unsigned blocks = (unsigned)std::min<int64_t>((a.n + ROWS - 1) / ROWS,
                                                      (int64_t)num_sms() * 16);
  block_norm_kernel<T, V, J, TPR><<<blocks, kThreads<TPR>, 0, s>>>(a);
  SV_LAUNCH_CHECK();
  return SV_OK;
}

template <typename T, int V, int J, int TPR>
int launch_backward(const BackArgs& a, unsigned blocks, cudaStream_t s) {
  block_norm_backward_kernel<T, V, J, TPR><<<blocks, kThreads<TPR>, 0, s>>>(a);
  SV_LAUNCH_CHECK();
  return SV_OK;
}

// A row's threads: as few as hold it with 16 elements each. What a thread does once a row (addresses, the
// steps of the sums, the loop) is as much as the work on 8 elements.
#define SV_BLOCK_NORM_PICK(call, C, wide)                                          \
  if (wide) {                                                                      \
    if ((C) <= 64) return call(8, 1, 8);                                           \
    if ((C) <= 128) return call(8, 2, 8);                                          \
    if ((C) <= 256) return call(8, 2, 16);                                         \
    if ((C) <= 512) return call(8, 2, 32);                                         \
    if ((C) <= 1024) return call(8, 2, 64);                                        \
    if ((C) <= 2048) return call(8, 2, 128);                                       \
    if ((C) <= 4096) return call(8, 2, 256);                                       \
    return call(8, 4, 256);                                                        \
  }                                                                                \
  if ((C) <= 256) return call(1, 8, 32);                                           \
  if ((C) <= 1024) return call(1, 8, 128);                                         \
  if ((C) <= 2048) return call(1, 8, 256);                                         \
  return call(1, 32, 256)

template <typename T, int J>
int rows_forward(const BlockArgs& a, cudaStream_t s) {
  auto kernel = a.layer ? (a.branch_norm ? block_norm_rows_kernel<T, J, true, true>
                                         : block_norm_rows_kernel<T, J, true, false>)
                        : (a.branch_norm ? block_norm_rows_kernel<T, J, false, true>
                                         : block_norm_rows_kernel<T, J, false, false>);
  constexpr int bytes = RowsLayout<T, J>::SMEM;
  SV_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  kernel<<<num_sms() * (sizeof(T) == 2 ? 2 : 1), 32 * ROW_WARPS, bytes, s>>>(a);
  SV_LAUNCH_CHECK();
  return SV_OK;
}

// Whether rows go through the warps' pipelines: rows that two to four eights a lane hold, and enough of
// them that every warp gets four. 9,472 rows, launch included, pipelined against the direct kernel: 1024
// channels of bf16 14.3 / 22.1 us, 512 9.1 / 15.0, 320 9.0 / 15.3; 1024 of fp32 28.5 / 33.5. The backward pass has no such form: its three sums leave
// one block an SM (1024 channels of bf16, 40,000 rows: 101 us so, 95 us by the direct kernel; 320: 66 / 48).
bool pipelined(int64_t n, int channels, bool wide) {
  return wide && channels > 256 && channels <= 1024 && n >= (int64_t)4 * ROW_WARPS * 2 * num_sms();
}
template <typename T>
int forward_typed(const BlockArgs& a, cudaStream_t s) {
  if (pipelined(a.n, a.channels, wide_rows(a)))
    return a.channels <= 512 ? rows_forward<T, 2>(a, s) : rows_forward<T, 4>(a, s);
#define SV_CALL(V, J, TPR) launch_forward<T, V, J, TPR>(a, s)
  SV_BLOCK_NORM_PICK(SV_CALL, a.channels, wide_rows(a));
#undef SV_CALL
}

template <typename T>
int backward_typed(const BackArgs& a, bool wide, unsigned blocks, cudaStream_t s) {
#define SV_CALL(V, J, TPR) launch_backward<T, V, J, TPR>(a, blocks, s)
  SV_BLOCK_NORM_PICK(SV_CALL, a.f.channels, wide);
#undef SV_CALL
}

// Rows of a piece, and how many pieces there can be (each batch element's last one is ragged): four blocks
// an SM run at the same time.
struct Pieces {
  int rows;
  int64_t most;
};
Pieces pieces_of(int64_t n, int64_t groups) {
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>((n + 15) / 16, (int64_t)num_sms() * 4));
  Pieces p;
  p.rows = (int)std::max<int64_t>(1, (n + want - 1) / want);
  p.most = (n + p.rows - 1) / p.rows + groups;
  return p;
}

struct BackPlan {
  Pieces pieces;
  size_t joined, done, starts, perm, offsets, scratch, total;  // `partial` is at the start
};
// Batch elements from which on the join takes a warp for each, instead of 32 warps for each and 32 columns.
// 20,331 rows, 256 / 1024 channels: with 8 of them 17.5 / 28.6 us (13.8 / 33.4), 12 13.8 / 21.8 (18.2 / 45.7),
// 100 9.8 / 13.2 (122 / 304); with 2 48 / 91 (7.6 / 13.4).
constexpr int64_t BN_MANY = 12;
BackPlan back_plan(int64_t n, int channels, int64_t groups) {  // groups 0: rows are not sorted
  BackPlan p;
  p.pieces = pieces_of(n, groups ? groups + 1 : 0);
  p.joined = align_up((size_t)p.pieces.most * 3 * channels * sizeof(float), 256);
  p.done = p.joined + align_up((size_t)(groups + 1) * 3 * channels * sizeof(float), 256);
  p.starts = p.done + BN_CHUNKS * sizeof(int);
  p.perm = p.starts + (groups ? align_up((size_t)(groups + 1) * sizeof(int), 256) : 0);
  p.offsets = p.perm + (groups ? align_up((size_t)n * sizeof(int32_t), 256) : 0);
  p.scratch = p.offsets + (groups ? align_up((size_t)(groups + 1) * sizeof(int32_t), 256) : 0);
  p.total = p.scratch + (groups ? group_rows_bytes(n, (int)groups) : 0);
  return p;
}

Coef to_coef(const sv_rows& r) { return {r.data, r.stride, r.dtype}; }
Grad to_grad(const sv_rows& r) { return {const_cast<void*>(r.data), r.stride, r.dtype}; }

int check_rows(const sv_rows& r, const char* name, const char* what) {
  if (!r.data) return SV_OK;
  if (!float_type(r.dtype)) SV_FAIL(SV_ERR_BAD_DTYPE, std::string(what) + ": unknown dtype of " + name);
  if (r.stride < 0) SV_FAIL(SV_ERR_INVALID_ARGUMENT, std::string(what) + ": negative stride of " + name);
  return SV_OK;
}

int fill(const sv_block_norm_args* g, const char* what, BlockArgs* a) {
  const std::string at = what;
  if (!g) SV_FAIL(SV_ERR_INVALID_ARGUMENT, at + ": null arguments");
  if (g->n < 0 || g->channels < 0 || g->batch < 0)
    SV_FAIL(SV_ERR_INVALID_ARGUMENT, at + ": negative size");
  if (!float_type(g->dtype)) SV_FAIL(SV_ERR_BAD_DTYPE, at + ": unknown dtype");
  if (g->channels > BN_MAX_CHANNELS)
    SV_FAIL(SV_ERR_UNSUPPORTED, at + ": more than " + std::to_string(BN_MAX_CHANNELS) + " channels");
  if (g->n > INT32_MAX - 1024) SV_FAIL(SV_ERR_UNSUPPORTED, at + ": too many rows");
  if (!(g->dropout >= 0.0 && g->dropout <= 1.0))
    SV_FAIL(SV_ERR_INVALID_ARGUMENT, at + ": dropout outside [0, 1]");
  if (!(g->eps >= 0.0f)) SV_FAIL(SV_ERR_INVALID_ARGUMENT, at + ": eps must not be negative");
  const struct { const sv_rows* r; const char* name; } rows[] = {
      {&g->weight, "weight"}, {&g->bias, "bias"}, {&g->branch_weight, "branch_weight"},
      {&g->gate, "gate"}, {&g->scale, "scale"}, {&g->shift, "shift"}};
  for (const auto& r : rows) {
    const int rc = check_rows(*r.r, r.name, what);
    if (rc != SV_OK) return rc;
  }
  if (g->branch_weight.data && !g->branch_norm)
    SV_FAIL(SV_ERR_INVALID_ARGUMENT, at + ": a branch weight goes with the branch's norm");
  const bool per_batch = (g->gate.data && g->gate.stride) || (g->scale.data && g->scale.stride) ||
                         (g->shift.data && g->shift.stride);
  if (per_batch && g->n > 0 && !g->coords)
    SV_FAIL(SV_ERR_INVALID_ARGUMENT, at + ": rows of coefficients per batch element need coords");
  if (per_batch && g->batch > GROUP_MAX_BINS - 1)
    SV_FAIL(SV_ERR_UNSUPPORTED, at + ": more than " + std::to_string(GROUP_MAX_BINS - 1) + " batch elements");
  *a = BlockArgs{};
  a->n = g->n;
  a->channels = g->channels;
  a->x = g->x;
  a->x_stride = g->x_stride;
  a->branch = g->branch;
  a->branch_stride = g->branch_stride;
  a->layer = g->layer != 0;
  a->branch_norm = g->branch_norm != 0;
  a->alpha = g->residual_scale;
  a->eps = g->eps;
  a->weight = to_coef(g->weight);
  a->bias = to_coef(g->bias);
  a->branch_weight = to_coef(g->branch_weight);
  a->gate = to_coef(g->gate);
  a->scale = to_coef(g->scale);
  a->shift = to_coef(g->shift);
  a->weight.stride = a->bias.stride = a->branch_weight.stride = 0;
  a->per_batch = per_batch;
  a->coords = g->coords;
  a->batch = per_batch ? g->batch : 1;
  a->drop = make_dropout(g->dropout, g->seed, g->seed_at, g->subsequence);
  a->h = g->h;
  a->stats = reinterpret_cast<float4*>(g->stats);
  return SV_OK;
}

}  // namespace
}  // namespace sv

using namespace sv;

extern "C" int sv_block_norm(const sv_block_norm_args* args, void* y, int32_t* status,
                             sv_stream_t stream) {
  BlockArgs a;
  const int rc = fill(args, "sv_block_norm", &a);
  if (rc != SV_OK) return rc;
  if (a.n == 0 || a.channels == 0) return SV_OK;
  if (!a.x || !a.branch || !a.h || !y)
    SV_FAIL(SV_ERR_INVALID_ARGUMENT, "sv_block_norm: null pointer");
  if (a.x_stride < a.channels || a.branch_stride < a.channels)
    SV_FAIL(SV_ERR_INVALID_ARGUMENT, "sv_block_norm: row stride below the row length");
  if (a.stats && !aligned16(a.stats))
    SV_FAIL(SV_ERR_INVALID_ARGUMENT, "sv_block_norm: stats must be 16-byte aligned");
  a.y = y;
  a.status = status;
  switch (args->dtype) {
    case SV_FLOAT32: return forward_typed<float>(a, to_stream(stream));
    case SV_FLOAT16: return forward_typed<__half>(a, to_stream(stream));
    default: return forward_typed<__nv_bfloat16>(a, to_stream(stream));
  }
}

extern "C" size_t sv_block_norm_backward_workspace_bytes(int64_t n, int channels, int64_t batch) {
  if (n < 0 || channels < 0 || batch < 0 || batch > GROUP_MAX_BINS - 1) return 0;
  return back_plan(n, channels, batch).total;
}

extern "C" int sv_block_norm_backward(const sv_block_norm_args* args, const void* dy, const void* dh,
                                      void* dx, void* dbranch, const sv_block_norm_grads* grads,
                                      void* workspace, size_t workspace_bytes, int32_t* status,
                                      sv_stream_t stream) {
  BlockArgs f;
  const int rc = fill(args, "sv_block_norm_backward", &f);
  if (rc != SV_OK) return rc;
  if (!grads) SV_FAIL(SV_ERR_INVALID_ARGUMENT, "sv_block_norm_backward: null arguments");
  const struct { const sv_rows* r; const Coef* c; const char* name; } rows[] = {
      {&grads->weight, &f.weight, "dweight"}, {&grads->bias, &f.bias, "dbias"},
      {&grads->branch_weight, &f.branch_weight, "dbranch_weight"}, {&grads->gate, &f.gate, "dgate"},
      {&grads->scale, &f.scale, "dscale"}, {&grads->shift, &f.shift, "dshift"}};
  bool sums = false;
  for (const auto& r : rows) {
    const int bad = check_rows(*r.r, r.name, "sv_block_norm_backward");
    if (bad != SV_OK) return bad;
    if (r.r->data && (!r.c->p || (r.r->stride != 0) != (r.c->stride != 0)))
      SV_FAIL(SV_ERR_INVALID_ARGUMENT,
              std::string("sv_block_norm_backward: ") + r.name + " has no coefficients of its shape");
    sums |= r.r->data != nullptr;
  }
  if (f.channels == 0 || !(sums || dx || dbranch)) return SV_OK;
  if (f.n > 0 && (!f.h || !f.stats || !f.branch || !(dy || dh)))
    SV_FAIL(SV_ERR_INVALID_ARGUMENT, "sv_block_norm_backward: null pointer");
  if (f.branch_stride < f.channels)
    SV_FAIL(SV_ERR_INVALID_ARGUMENT, "sv_block_norm_backward: row stride below the row length");
  if (!aligned16(f.stats))
    SV_FAIL(SV_ERR_INVALID_ARGUMENT, "sv_block_norm_backward: stats must be 16-byte aligned");
  // Rows are sorted where coefficients differ by batch element: the pieces then have one element each.
  const int64_t groups = f.per_batch ? f.batch : 0;
  const BackPlan plan = back_plan(f.n, f.channels, groups);
  if ((sums || groups) && (!workspace || workspace_bytes < plan.total || !aligned16(workspace)))
    SV_FAIL(SV_ERR_WORKSPACE, "sv_block_norm_backward: workspace too small or unaligned");
  cudaStream_t s = to_stream(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  f.status = status;
  BackArgs a{};
  a.f = f;
  a.dy = dy;
  a.dh = dh;
  a.dx = dx;
  a.dbranch = dbranch;
  a.piece = plan.pieces.rows;
  a.partial = sums ? reinterpret_cast<float*>(ws) : nullptr;
  a.done = sums ? reinterpret_cast<int*>(ws + plan.done) : nullptr;
  a.want_e = grads->gate.data || grads->branch_weight.data;
  if (groups) {
    int32_t* perm = reinterpret_cast<int32_t*>(ws + plan.perm);
    int32_t* offsets = reinterpret_cast<int32_t*>(ws + plan.offsets);
    const int bad = group_rows(f.coords, 4, f.n, (int)groups, perm, offsets, nullptr,
                               ws + plan.scratch, s);
    if (bad != SV_OK) return bad;
    a.perm = perm;
    a.offsets = offsets;
    a.starts = sums && groups >= BN_MANY ? reinterpret_cast<int*>(ws + plan.starts) : nullptr;
  }
  if (f.n > 0) {
    BlockArgs ready = f;  // what the backward pass reads has to be aligned; x and y are not there
    ready.x = nullptr;
    ready.x_stride = 0;
    const bool wide = wide_rows(ready) && aligned16(dy) && aligned16(dh) && aligned16(dx) &&
                      aligned16(dbranch);
    const unsigned blocks = (unsigned)plan.pieces.most;
    const int bad = args->dtype == SV_FLOAT32   ? backward_typed<float>(a, wide, blocks, s)
                    : args->dtype == SV_FLOAT16 ? backward_typed<__half>(a, wide, blocks, s)
                                                : backward_typed<__nv_bfloat16>(a, wide, blocks, s);
    if (bad != SV_OK) return bad;
  }
  if (!sums) return SV_OK;
  if (f.n == 0) SV_CUDA_TRY(cudaMemsetAsync(a.done, 0, BN_CHUNKS * sizeof(int), s));
  SumArgs g{};
  g.f = f;
  g.offsets = a.offsets;
  g.piece = a.piece;
  g.partial = a.partial;
  g.groups = f.per_batch ? (int)f.batch + 1 : 1;
  g.sums = reinterpret_cast<float*>(ws + plan.joined);
  g.done = a.done;
  g.weight = to_grad(grads->weight);
  g.bias = to_grad(grads->bias);
  g.branch_weight = to_grad(grads->branch_weight);
  g.gate = to_grad(grads->gate);
  g.scale = to_grad(grads->scale);
  g.shift = to_grad(grads->shift);
  g.weight.stride = g.bias.stride = g.branch_weight.stride = 0;
  g.starts = a.starts;
  if (a.starts) {
    const dim3 grid((unsigned)((f.channels + 31) / 32), (unsigned)((g.groups + 31) / 32));
    block_norm_join_many_kernel<<<grid, 1024, 0, s>>>(g);
  } else {
    const dim3 grid((unsigned)((3 * f.channels + 31) / 32), (unsigned)g.groups);
    block_norm_join_kernel<<<grid, 1024, 0, s>>>(g);
  }
  SV_LAUNCH_CHECK();
  return SV_OK;
}
