// Stable counting sort of rows by a small key.
//
// Every warp takes a contiguous run of rows ("part"). Three steps: a histogram per part, an exclusive
// scan over each bin's parts (a bin's parts follow each other in the rows' order), and the scatter, in which a warp ranks 32 rows at a time among those with the same key.
// Nothing depends on the order of execution. Few rows take one launch of one block, more take three:
// the launches are what bounds the small ones (8 to 16 thousand rows: the block of 32 warps walks 512
// rows a warp at about 0.1 us for 32).
#include <algorithm>

#include "group.h"

namespace sv {
namespace {

constexpr int GROUP_WARPS = 8;
constexpr int SMEM_COUNTS = 12 * 1024;  // counters of a block: 48 KB of shared memory

__device__ __forceinline__ int bin_of(int32_t key, int groups) {
  return key >= 0 && key < groups ? key : groups;
}

// A warp adds its part's rows to its counters `mine` (shared memory, zeroed).
__device__ __forceinline__ void count_part(const int32_t* keys, int64_t stride, int64_t a, int64_t b,
                                           int groups, int32_t* mine) {
  const int lane = threadIdx.x & 31;
  for (int64_t i = a + lane; i < b; i += 32) atomicAdd(mine + bin_of(keys[i * stride], groups), 1);
  __syncwarp();
}

// A warp writes its part's rows to their positions; `mine`: where each bin's next row goes.
__device__ __forceinline__ void place_part(const int32_t* keys, int64_t stride, int64_t a, int64_t b,
                                           int groups, int32_t* mine, int32_t* perm,
                                           int32_t* place) {
  const int lane = threadIdx.x & 31;
  for (int64_t i0 = a; i0 < b; i0 += 32) {
    const int64_t i = i0 + lane;
    const bool in = i < b;
    const int bin = in ? bin_of(keys[i * stride], groups) : -1;
    const unsigned same = __match_any_sync(0xffffffffu, bin);
    const int rank = __popc(same & ((1u << lane) - 1u));
    int at = 0;
    if (in) at = mine[bin] + rank;
    __syncwarp();
    if (in && rank == 0) mine[bin] += __popc(same);
    __syncwarp();
    if (in) {
      perm[at] = (int32_t)i;
      if (place) place[i] = bin < groups ? at : -1;
    }
  }
}

// Exclusive sums over counts[0..total) in place, by one block of 1024 threads.
__device__ __forceinline__ void scan_block(int32_t* counts, int total, int32_t* part) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int each = (total + 1023) / 1024;
  const int a = min(tid * each, total), b = min(a + each, total);
  int sum = 0;
  for (int i = a; i < b; ++i) sum += counts[i];
  int upto = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) part[warp] = upto;
  __syncthreads();
  if (warp == 0) {
    int v = part[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    part[lane] = v;
  }
  __syncthreads();
  int at = upto - sum + (warp ? part[warp - 1] : 0);
  for (int i = a; i < b; ++i) {
    const int c = counts[i];
    counts[i] = at;
    at += c;
  }
  __syncthreads();
}

// Everything in one block; counters [bins][warps] in shared memory.
__global__ void __launch_bounds__(1024)
    group_small_kernel(const int32_t* keys, int64_t stride, int n, int groups, int32_t* perm,
                       int32_t* offsets, int32_t* place) {
  extern __shared__ int32_t counts[];
  __shared__ int32_t part[32];
  const int bins = groups + 1, tid = threadIdx.x, warp = tid >> 5;
  // warp-major while rows are counted, bin-major for the scan
  int32_t* by_warp = counts;
  int32_t* by_bin = counts + bins * 32;
  for (int i = tid; i < bins * 32; i += 1024) by_warp[i] = 0;
  __syncthreads();
  const int per = ((n + 31) / 32 + 31) / 32 * 32;
  const int a = min(warp * per, n), b = min(a + per, n);
  count_part(keys, stride, a, b, groups, by_warp + warp * bins);
  __syncthreads();
  for (int i = tid; i < bins * 32; i += 1024) by_bin[i] = by_warp[(i & 31) * bins + (i >> 5)];
  __syncthreads();
  scan_block(by_bin, bins * 32, part);
  for (int i = tid; i < bins * 32; i += 1024) by_warp[(i & 31) * bins + (i >> 5)] = by_bin[i];
  for (int g = tid; g <= groups; g += 1024) offsets[g] = by_bin[g * 32];
  __syncthreads();
  place_part(keys, stride, a, b, groups, by_warp + warp * bins, perm, place);
}

__global__ void __launch_bounds__(GROUP_WARPS * 32)
    group_count_kernel(const int32_t* keys, int64_t stride, int64_t n, int64_t per, int groups,
                       int parts, int32_t* counts) {
  extern __shared__ int32_t mine[];
  const int bins = groups + 1, warps = blockDim.x >> 5, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < bins * warps; i += blockDim.x) mine[i] = 0;
  __syncthreads();
  const int64_t p = (int64_t)blockIdx.x * warps + warp;
  const int64_t a = min(p * per, n), b = min(a + per, n);
  count_part(keys, stride, a, b, groups, mine + warp * bins);
  __syncthreads();
  for (int i = threadIdx.x; i < bins * warps; i += blockDim.x) {
    const int bin = i / warps, w = i - bin * warps;
    counts[(int64_t)bin * parts + blockIdx.x * warps + w] = mine[w * bins + bin];
  }
}

// Exclusive sums over a bin's parts in place, a block a bin, and the bin's total.
__global__ void __launch_bounds__(256) group_scan_kernel(int32_t* counts, int parts, int32_t* totals) {
  __shared__ int32_t part[8];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int32_t* mine = counts + (int64_t)blockIdx.x * parts;
  int before = 0;
  for (int i0 = 0; i0 < parts; i0 += 256) {
    const int i = i0 + tid;
    const int c = i < parts ? mine[i] : 0;
    int upto = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    __syncthreads();  // the previous round's sums have been read
    if (lane == 31) part[warp] = upto;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      if (w == warp) upto += all;
      all += part[w];
    }
    if (i < parts) mine[i] = before + upto - c;
    before += all;
  }
  if (tid == 0) totals[blockIdx.x] = before;
}

__global__ void __launch_bounds__(GROUP_WARPS * 32)
    group_place_kernel(const int32_t* keys, int64_t stride, int64_t n, int64_t per, int groups,
                       int parts, const int32_t* counts, const int32_t* totals, int32_t* offsets,
                       int32_t* perm, int32_t* place) {
  extern __shared__ int32_t mine[];
  const int bins = groups + 1, warps = blockDim.x >> 5, warp = threadIdx.x >> 5;
  int32_t* base = mine + bins * warps;  // where each bin starts
  if (warp == 0) {
    int before = 0;
    for (int b0 = 0; b0 < bins; b0 += 32) {
      const int b = b0 + (int)threadIdx.x, c = b < bins ? __ldg(totals + b) : 0;
      int upto = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if ((int)threadIdx.x >= o) upto += v;
      }
      if (b < bins) {
        base[b] = before + upto - c;
        if (blockIdx.x == 0) offsets[b] = before + upto - c;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < bins * warps; i += blockDim.x) {
    const int bin = i / warps, w = i - bin * warps;
    mine[w * bins + bin] = base[bin] + counts[(int64_t)bin * parts + blockIdx.x * warps + w];
  }
  __syncthreads();
  const int64_t p = (int64_t)blockIdx.x * warps + warp;
  const int64_t a = min(p * per, n), b = min(a + per, n);
  place_part(keys, stride, a, b, groups, mine + warp * bins, perm, place);
}

struct GroupPlan {
  bool small;
  int warps;     // a block
  int blocks;
  int64_t per;   // rows a part
};
GroupPlan group_plan(int64_t n, int groups) {
  const int bins = groups + 1;
  GroupPlan p{};
  p.small = n <= 16384 && bins * 64 + 32 <= SMEM_COUNTS;
  if (p.small) return p;
  // a block holds a counter a warp and bin, and a base a bin
  p.warps = std::max(1, std::min(GROUP_WARPS, SMEM_COUNTS / bins - 1));
  // parts of 64 rows at least, no more than a block an SM, and a megabyte of counters at most
  int64_t parts = std::min<int64_t>((n + 63) / 64, (int64_t)num_sms() * p.warps);
  parts = std::max<int64_t>(1, std::min<int64_t>(parts, (256 * 1024) / bins));
  p.blocks = (int)((parts + p.warps - 1) / p.warps);
  parts = (int64_t)p.blocks * p.warps;
  p.per = ((n + parts - 1) / parts + 31) / 32 * 32;
  return p;
}

}  // namespace

size_t group_rows_bytes(int64_t n, int groups) {
  const GroupPlan p = group_plan(n, groups);
  return p.small ? 0 : align_up((size_t)(groups + 1) * (p.blocks * p.warps + 1) * sizeof(int32_t), 256);
}

int group_rows(const int32_t* keys, int64_t stride, int64_t n, int groups, int32_t* perm,
               int32_t* offsets, int32_t* place, void* workspace, cudaStream_t s) {
  if (groups + 1 > GROUP_MAX_BINS)
    SV_FAIL(SV_ERR_UNSUPPORTED, "grouping: more than " + std::to_string(GROUP_MAX_BINS - 1) + " groups");
  const GroupPlan p = group_plan(n, groups);
  const size_t bins = (size_t)groups + 1;
  if (p.small) {
    const size_t bytes = bins * 64 * sizeof(int32_t);
    group_small_kernel<<<1, 1024, bytes, s>>>(keys, stride, (int)n, groups, perm, offsets, place);
    SV_LAUNCH_CHECK();
    return SV_OK;
  }
  int32_t* counts = static_cast<int32_t*>(workspace);
  const int parts = p.blocks * p.warps;
  int32_t* totals = counts + bins * parts;
  const size_t bytes = bins * p.warps * sizeof(int32_t);
  group_count_kernel<<<p.blocks, p.warps * 32, bytes, s>>>(keys, stride, n, p.per, groups, parts,
                                                           counts);
  SV_LAUNCH_CHECK();
  group_scan_kernel<<<(unsigned)bins, 256, 0, s>>>(counts, parts, totals);
  SV_LAUNCH_CHECK();
  group_place_kernel<<<p.blocks, p.warps * 32, bytes + bins * sizeof(int32_t), s>>>(
      keys, stride, n, p.per, groups, parts, counts, totals, offsets, perm, place);
  SV_LAUNCH_CHECK();
  return SV_OK;
}

}  // namespace sv
