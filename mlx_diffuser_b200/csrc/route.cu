// The router of a mixture of experts: each row's k best experts by their logits, the weights of their
// results, and the slots (row * k + choice) sorted by expert.
//
//     experts[n][j]: the j-th largest logit, the lower index first among equals; -1 where it is -inf
//     weights[n][j] = exp(l_j - m) / sum exp(l - m), the sum over the chosen or over all experts
//     dl_i = w_j (dw_j - sum w dw)  for the chosen, 0 elsewhere             (sum over the chosen)
//     dl_i = [i chosen] w_j dw_j - softmax_i sum w dw                       (sum over all)
//
// A warp takes a row, its logits in registers (32 L experts: L a lane). A choice is a maximum over the
// warp of the logit's bits in an order that integers have, then a minimum over the indices that have it:
// two warp reductions. NaN counts as the largest and gives NaN weights, as a softmax does.
// 40,662 rows of 64 fp32 logits, k 4, are 10 MB: HBM's 2 us are below the launches, and the selection's
// instructions (18 us) and the sort's second step (9 us) bound the call; its gradient takes 8 us. The blocks that choose also count, which is the
// sort's first step; for few rows one block does all of it.
#include <algorithm>

#include "group.h"

namespace sv {
namespace {

constexpr int ROUTE_MAX_EXPERTS = 1024;
constexpr int ROUTE_MAX_K = 32;
constexpr int ROUTE_WARPS = 8;
constexpr uint32_t TAKEN = 0u;
constexpr uint32_t MINUS_INF = 0x007fffffu;  // order_of(-inf)

// Unsigned integers in the order of the floats: zeros alike, NaN above all.
__device__ __forceinline__ uint32_t order_of(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t u = __float_as_uint(v == 0.0f ? 0.0f : v);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  if (key == 0xffffffffu) return __uint_as_float(0x7fc00000u);
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename T, int L>
__device__ __forceinline__ void load_logits(const T* row, int experts, uint32_t (&key)[L]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < L; ++i) {
    const int e = i * 32 + lane;
    key[i] = e < experts ? order_of(to_f32(row[e])) : TAKEN;
  }
}

// sum over all experts of exp(l - top), top finite or not as softmax has it.
template <int L>
__device__ __forceinline__ float total_of(const uint32_t (&key)[L], float top) {
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < L; ++i)
    if (key[i] > MINUS_INF) s += expf(value_of(key[i]) - top);
  return warp_sum(s);
}

// A row by a warp: lane j has choice j's expert (-1: none) and weight.
template <typename T, int L>
__device__ __forceinline__ void route_row(const T* row, int experts, int k, bool normalize, int& pick,
                                          float& w) {
  const int lane = threadIdx.x & 31;
  uint32_t key[L];
  load_logits<T, L>(row, experts, key);
  uint32_t mine = TAKEN;  // the lane's largest
#pragma unroll
  for (int i = 0; i < L; ++i) mine = max(mine, key[i]);
  uint32_t best = __reduce_max_sync(0xffffffffu, mine);
  const float top = best > MINUS_INF ? value_of(best) : 0.0f;
  float total = 0.0f;
  if (!normalize) total = total_of<L>(key, top);
  pick = -1;
  float value = 0.0f;
  for (int j = 0; j < k && best > MINUS_INF; ++j) {
    int at = INT32_MAX;
    if (mine == best) {
#pragma unroll
      for (int i = L - 1; i >= 0; --i)
        if (key[i] == best) at = i * 32 + lane;
    }
    const int e = __reduce_min_sync(0xffffffffu, at);
    if (lane == j) {
      pick = e;
      value = value_of(best);
    }
    if (at == e) {
      mine = TAKEN;
#pragma unroll
      for (int i = 0; i < L; ++i) {
        if (i * 32 + lane == e) key[i] = TAKEN;
        mine = max(mine, key[i]);
      }
    }
    best = __reduce_max_sync(0xffffffffu, mine);
  }
  w = pick >= 0 ? expf(value - top) : 0.0f;
  if (normalize) total = warp_sum(w);
  if (pick >= 0) w /= total;
}

// Blocks take `per` rows each and count their slots by expert for the sort's second step.
template <typename T, int L>
__global__ void __launch_bounds__(1024)
    route_kernel(const T* logits, int64_t stride, int64_t n, int64_t per, int experts, int k,
                 bool normalize, int32_t* chosen, float* weights, int32_t* counts) {
  __shared__ int32_t mine[ROUTE_MAX_EXPERTS + 1];
  const int lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i <= experts; i += 1024) mine[i] = 0;
  __syncthreads();
  const int64_t first = min(blockIdx.x * per, n), last = min(first + per, n);
  for (int64_t row = first + (threadIdx.x >> 5); row < last; row += 32) {
    int pick;
    float w;
    route_row<T, L>(logits + row * stride, experts, k, normalize, pick, w);
    if (lane < k) {
      chosen[row * k + lane] = pick;
      weights[row * k + lane] = w;
      atomicAdd(mine + (pick >= 0 ? pick : experts), 1);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i <= experts; i += 1024)
    counts[(int64_t)i * gridDim.x + blockIdx.x] = mine[i];
}

// Few rows: choices and sort in one block.
template <typename T, int L>
__global__ void __launch_bounds__(1024)
    route_small_kernel(const T* logits, int64_t stride, int n, int experts, int k, bool normalize,
                       int32_t* chosen, float* weights, int32_t* order, int32_t* offsets,
                       int32_t* place) {
  extern __shared__ int32_t counts[];
  __shared__ int32_t part[32];
  const int lane = threadIdx.x & 31;
  for (int row = threadIdx.x >> 5; row < n; row += 32) {
    int pick;
    float w;
    route_row<T, L>(logits + row * stride, experts, k, normalize, pick, w);
    if (lane < k) {
      chosen[row * k + lane] = pick;
      weights[row * k + lane] = w;
    }
  }
  __syncthreads();  // the block's choices are in memory
  group_block(chosen, 1, n * k, experts, order, offsets, place, counts, part);
}

template <typename T, int L>
__global__ void __launch_bounds__(ROUTE_WARPS * 32)
    route_backward_kernel(const T* logits, int64_t stride, int64_t n, int experts, int k,
                          bool normalize, const int32_t* chosen, const float* weights,
                          const float* dweights, T* dlogits) {
  const int lane = threadIdx.x & 31;
  const int64_t step = (int64_t)gridDim.x * ROUTE_WARPS;
  for (int64_t row = (int64_t)blockIdx.x * ROUTE_WARPS + (threadIdx.x >> 5); row < n; row += step) {
    int pick = -1;
    float w = 0.0f, dw = 0.0f;
    if (lane < k) {
      pick = chosen[row * k + lane];
      if (pick >= 0) {
        w = weights[row * k + lane];
        dw = dweights[row * k + lane];
      }
    }
    const float dot = warp_sum(w * dw);
    float d[L];
    if (normalize) {
#pragma unroll
      for (int i = 0; i < L; ++i) d[i] = 0.0f;
      dw -= dot;
    } else {
      uint32_t key[L];
      load_logits<T, L>(logits + row * stride, experts, key);
      uint32_t mine = TAKEN;
#pragma unroll
      for (int i = 0; i < L; ++i) mine = max(mine, key[i]);
      const uint32_t first = __reduce_max_sync(0xffffffffu, mine);
      const float top = first > MINUS_INF ? value_of(first) : 0.0f;
      const float total = total_of<L>(key, top);
#pragma unroll
      for (int i = 0; i < L; ++i)
        d[i] = key[i] > MINUS_INF ? -dot * (expf(value_of(key[i]) - top) / total) : 0.0f;
    }
    const float term = pick >= 0 ? w * dw : 0.0f;
    for (int j = 0; j < k; ++j) {
      const int e = __shfl_sync(0xffffffffu, pick, j);
      const float v = __shfl_sync(0xffffffffu, term, j);
#pragma unroll
      for (int i = 0; i < L; ++i)
        if (e == i * 32 + lane) d[i] += v;
    }
#pragma unroll
    for (int i = 0; i < L; ++i)
      if (i * 32 + lane < experts) dlogits[row * experts + i * 32 + lane] = from_f32<T>(d[i]);
  }
}

struct RouteArgs {
  const void* logits;
  int64_t stride, n;
  int experts, k;
  bool normalize;
  int32_t* chosen;
  float* weights;
  const float* dweights;  // the backward pass
  void* dlogits;
  int32_t *order, *offsets, *place, *counts;  // the forward pass
};

// Rows that one block chooses for: four a warp. 64 experts, k 4: 12.6 us for 128 rows, 10.0 us in two
// launches, whose second one costs the host 6 us more; 256 rows 20.6 us.
constexpr int ROUTE_SMALL = 128;
// The rows' slots are cut between the blocks at rows.
GroupPlan route_plan(int64_t n, int experts, int k) {
  GroupPlan p = group_plan(n * k, experts);
  p.small = p.small && n <= ROUTE_SMALL;
  if (p.small) return p;
  p.warps = std::max(1, std::min(16, GROUP_COUNTS / (experts + 1) - 2));
  const int64_t blocks = std::max<int64_t>(1, std::min<int64_t>((n + 31) / 32, num_sms()));
  const int64_t rows = (n + blocks - 1) / blocks;
  p.blocks = (int)blocks;
  p.per = rows * k;
  return p;
}

template <typename T, int L>
int launch_route(const RouteArgs& a, cudaStream_t s) {
  const T* x = static_cast<const T*>(a.logits);
  if (a.dlogits) {
    const unsigned blocks = (unsigned)std::min<int64_t>((a.n + ROUTE_WARPS - 1) / ROUTE_WARPS,
                                                        (int64_t)num_sms() * 8);
    route_backward_kernel<T, L><<<blocks, ROUTE_WARPS * 32, 0, s>>>(
        x, a.stride, a.n, a.experts, a.k, a.normalize, a.chosen, a.weights, a.dweights,
        static_cast<T*>(a.dlogits));
    SV_LAUNCH_CHECK();
    return SV_OK;
  }
  const GroupPlan p = route_plan(a.n, a.experts, a.k);
  if (p.small) {
    const size_t bytes = (size_t)(a.experts + 1) * 64 * sizeof(int32_t);
    route_small_kernel<T, L><<<1, 1024, bytes, s>>>(x, a.stride, (int)a.n, a.experts, a.k, a.normalize,
                                                    a.chosen, a.weights, a.order, a.offsets, a.place);
    SV_LAUNCH_CHECK();
    return SV_OK;
  }
  route_kernel<T, L><<<p.blocks, 1024, 0, s>>>(x, a.stride, a.n, p.per / a.k, a.experts, a.k,
                                               a.normalize, a.chosen, a.weights, a.counts);
  SV_LAUNCH_CHECK();
  return group_place(p, a.chosen, 1, a.n * a.k, a.experts, a.counts, a.order, a.offsets, a.place, s);
}

template <typename T>
int route_typed(const RouteArgs& a, cudaStream_t s) {
  if (a.experts <= 32) return launch_route<T, 1>(a, s);
  if (a.experts <= 64) return launch_route<T, 2>(a, s);
  if (a.experts <= 128) return launch_route<T, 4>(a, s);
  if (a.experts <= 256) return launch_route<T, 8>(a, s);
  if (a.experts <= 512) return launch_route<T, 16>(a, s);
  return launch_route<T, 32>(a, s);
}

int route_any(const RouteArgs& a, int dtype, cudaStream_t s) {
  switch (dtype) {
    case SV_FLOAT32: return route_typed<float>(a, s);
    case SV_FLOAT16: return route_typed<__half>(a, s);
    default: return route_typed<__nv_bfloat16>(a, s);
  }
}

int check_route(int64_t n, int experts, int k, int dtype, const char* what) {
  const std::string at = what;
  if (n < 0 || experts < 1 || k < 1) SV_FAIL(SV_ERR_INVALID_ARGUMENT, at + ": bad size");
  if (dtype != SV_FLOAT32 && dtype != SV_FLOAT16 && dtype != SV_BFLOAT16)
    SV_FAIL(SV_ERR_BAD_DTYPE, at + ": unknown dtype");
  if (k > experts) SV_FAIL(SV_ERR_BAD_SHAPE, at + ": more choices than experts");
  if (experts > ROUTE_MAX_EXPERTS || k > ROUTE_MAX_K)
    SV_FAIL(SV_ERR_UNSUPPORTED, at + ": at most " + std::to_string(ROUTE_MAX_EXPERTS) +
                                    " experts and " + std::to_string(ROUTE_MAX_K) + " choices");
  if (n * k > INT32_MAX - 1024) SV_FAIL(SV_ERR_UNSUPPORTED, at + ": too many rows");
  return SV_OK;
}

}  // namespace
}  // namespace sv

using namespace sv;

extern "C" size_t sv_route_workspace_bytes(int64_t n, int experts, int k) {
  if (check_route(n, experts, k, SV_FLOAT32, "sv_route") != SV_OK) return 0;
  const GroupPlan p = route_plan(n, experts, k);
  return p.small ? 0 : align_up((size_t)(experts + 1) * p.blocks * sizeof(int32_t), 256);
}

extern "C" int sv_route(const void* logits, int64_t stride, int64_t n, int experts, int k, int dtype,
                        int normalize, int32_t* chosen, float* weights, int32_t* order,
                        int32_t* offsets, int32_t* place, void* workspace, size_t workspace_bytes,
                        sv_stream_t stream) {
  const int rc = check_route(n, experts, k, dtype, "sv_route");
  if (rc != SV_OK) return rc;
  if (!offsets || (n > 0 && (!logits || !chosen || !weights || !order || !place)))
    SV_FAIL(SV_ERR_INVALID_ARGUMENT, "sv_route: null pointer");
  if (stride < experts) SV_FAIL(SV_ERR_INVALID_ARGUMENT, "sv_route: row stride below the row length");
  const size_t need = sv_route_workspace_bytes(n, experts, k);
  if (need && (!workspace || workspace_bytes < need))
    SV_FAIL(SV_ERR_WORKSPACE, "sv_route: workspace too small");
  const RouteArgs a{logits, stride, n, experts, k, normalize != 0, chosen, weights, nullptr, nullptr,
                    order, offsets, place, static_cast<int32_t*>(workspace)};
  return route_any(a, dtype, to_stream(stream));
}

extern "C" int sv_route_backward(const void* logits, int64_t stride, int64_t n, int experts, int k,
                                 int dtype, int normalize, const int32_t* chosen,
                                 const float* weights, const float* dweights, void* dlogits,
                                 sv_stream_t stream) {
  const int rc = check_route(n, experts, k, dtype, "sv_route_backward");
  if (rc != SV_OK) return rc;
  if (n == 0) return SV_OK;
  if (!logits || !chosen || !weights || !dweights || !dlogits)
    SV_FAIL(SV_ERR_INVALID_ARGUMENT, "sv_route_backward: null pointer");
  if (stride < experts)
    SV_FAIL(SV_ERR_INVALID_ARGUMENT, "sv_route_backward: row stride below the row length");
  const RouteArgs a{logits, stride, n, experts, k, normalize != 0, const_cast<int32_t*>(chosen),
                    const_cast<float*>(weights), dweights, dlogits, nullptr, nullptr, nullptr, nullptr};
  return route_any(a, dtype, to_stream(stream));
}
