// Stable counting sort of rows by a small key.
//
// Every warp takes a contiguous run of rows, ranks 32 of them at a time among those with the same key,
// and knows how many rows of each key are before its own. Nothing depends on the order of execution. Up
// to 8192 rows one block counts, scans and places; more take two launches: blocks count their rows, then
// each placing block sums the counts of the blocks before it. 20,331 rows in 2 groups: 18 us in one
// block, 8 us in two launches.
#include <algorithm>

#include "group.h"

namespace sv {
namespace {

__global__ void __launch_bounds__(1024)
    group_small_kernel(const int32_t* keys, int64_t stride, int n, int groups, int32_t* perm,
                       int32_t* offsets, int32_t* place) {
  extern __shared__ int32_t counts[];
  __shared__ int32_t part[32];
  group_block(keys, stride, n, groups, perm, offsets, place, counts, part);
}

__global__ void __launch_bounds__(512)
    group_count_kernel(const int32_t* keys, int64_t stride, int64_t n, int64_t per, int groups,
                       int32_t* counts) {
  extern __shared__ int32_t mine[];
  const int bins = groups + 1;
  for (int i = threadIdx.x; i < bins; i += 512) mine[i] = 0;
  __syncthreads();
  const int64_t a = min(blockIdx.x * per, n), b = min(a + per, n);
  for (int64_t i = a + threadIdx.x; i < b; i += 512)
    atomicAdd(mine + bin_of(keys[i * stride], groups), 1);
  __syncthreads();
  for (int i = threadIdx.x; i < bins; i += 512) counts[(int64_t)i * gridDim.x + blockIdx.x] = mine[i];
}

// `mine` [warps][bins], then each bin's total, then its rows before this block.
__global__ void __launch_bounds__(512)
    group_place_kernel(const int32_t* keys, int64_t stride, int64_t n, int64_t per, int groups,
                       const int32_t* counts, int32_t* offsets, int32_t* perm, int32_t* place) {
  extern __shared__ int32_t mine[];
  const int bins = groups + 1, warps = blockDim.x >> 5, warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31, blocks = gridDim.x;
  int32_t* total = mine + bins * warps;
  int32_t* before = total + bins;
  for (int i = threadIdx.x; i < bins * warps; i += blockDim.x) mine[i] = 0;
  __syncthreads();
  const int64_t first = min(blockIdx.x * per, n), last = min(first + per, n);
  const int64_t each = ((last - first + warps - 1) / warps + 31) / 32 * 32;
  const int64_t a = min(first + warp * each, last), b = min(a + each, last);
  count_part(keys, stride, a, b, groups, mine + warp * bins);
#pragma unroll 4
  for (int bin = warp; bin < bins; bin += warps) {
    int all = 0, prior = 0;
    for (int i = lane; i < blocks; i += 32) {
      const int c = __ldg(counts + (int64_t)bin * blocks + i);
      all += c;
      prior += i < (int)blockIdx.x ? c : 0;
    }
    all = __reduce_add_sync(0xffffffffu, all);
    prior = __reduce_add_sync(0xffffffffu, prior);
    if (lane == 0) {
      total[bin] = all;
      before[bin] = prior;
    }
  }
  __syncthreads();
  if (warp == 0) {  // the bins before each
    int sum = 0;
    for (int b0 = 0; b0 < bins; b0 += 32) {
      const int bin = b0 + lane, c = bin < bins ? total[bin] : 0;
      int upto = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      if (bin < bins) {
        before[bin] += sum + upto - c;
        if (blockIdx.x == 0) offsets[bin] = sum + upto - c;
      }
      sum += __shfl_sync(0xffffffffu, upto, 31);
    }
  }
  __syncthreads();
  for (int bin = threadIdx.x; bin < bins; bin += blockDim.x) {  // and the warps before each
    int at = before[bin];
    for (int w = 0; w < warps; ++w) {
      const int c = mine[w * bins + bin];
      mine[w * bins + bin] = at;
      at += c;
    }
  }
  __syncthreads();
  place_part(keys, stride, a, b, groups, mine + warp * bins, perm, place);
}

}  // namespace

GroupPlan group_plan(int64_t n, int groups) {
  const int bins = groups + 1;
  GroupPlan p{};
  p.small = n <= 8192 && bins * 64 + 32 <= GROUP_COUNTS;
  if (p.small) return p;
  // a placing block holds a counter a warp and bin, and two more a bin
  p.warps = std::max(1, std::min(16, GROUP_COUNTS / bins - 2));
  p.blocks = (int)std::max<int64_t>(1, std::min<int64_t>((n + 511) / 512, num_sms()));
  p.per = (n + p.blocks - 1) / p.blocks;
  return p;
}

size_t group_rows_bytes(int64_t n, int groups) {
  const GroupPlan p = group_plan(n, groups);
  return p.small ? 0 : align_up((size_t)(groups + 1) * p.blocks * sizeof(int32_t), 256);
}

int group_place(const GroupPlan& p, const int32_t* keys, int64_t stride, int64_t n, int groups,
                const int32_t* counts, int32_t* perm, int32_t* offsets, int32_t* place,
                cudaStream_t s) {
  const size_t bins = (size_t)groups + 1;
  group_place_kernel<<<p.blocks, p.warps * 32, bins * (p.warps + 2) * sizeof(int32_t), s>>>(
      keys, stride, n, p.per, groups, counts, offsets, perm, place);
  SV_LAUNCH_CHECK();
  return SV_OK;
}

int group_rows(const int32_t* keys, int64_t stride, int64_t n, int groups, int32_t* perm,
               int32_t* offsets, int32_t* place, void* workspace, cudaStream_t s) {
  if (groups + 1 > GROUP_MAX_BINS)
    SV_FAIL(SV_ERR_UNSUPPORTED, "grouping: more than " + std::to_string(GROUP_MAX_BINS - 1) + " groups");
  const GroupPlan p = group_plan(n, groups);
  const size_t bins = (size_t)groups + 1;
  if (p.small) {
    group_small_kernel<<<1, 1024, bins * 64 * sizeof(int32_t), s>>>(keys, stride, (int)n, groups, perm,
                                                                    offsets, place);
    SV_LAUNCH_CHECK();
    return SV_OK;
  }
  int32_t* counts = static_cast<int32_t*>(workspace);
  group_count_kernel<<<p.blocks, 512, bins * sizeof(int32_t), s>>>(keys, stride, n, p.per, groups,
                                                                   counts);
  SV_LAUNCH_CHECK();
  return group_place(p, keys, stride, n, groups, counts, perm, offsets, place, s);
}

}  // namespace sv
