// Stable grouping of rows by a key, as a counting sort on the device (group.cu): the router's slots by
// expert, and the rows of a block's modulations by batch element.
#pragma once

#include "common.cuh"

namespace sv {

constexpr int GROUP_MAX_BINS = 4096;  // groups, and one more for the rows without one
constexpr int GROUP_COUNTS = 12 * 1024;  // counters of a block: 48 KB of shared memory

// How n rows are cut: one block does everything (`small`), or `blocks` of them count their `per` rows
// into counts [groups + 1][blocks], and as many place them.
struct GroupPlan {
  bool small;
  int blocks, warps;  // warps of a placing block
  int64_t per;
};
GroupPlan group_plan(int64_t n, int groups);

// Bytes that group_rows needs for n rows and `groups` groups: the counts.
size_t group_rows_bytes(int64_t n, int groups);

// perm: the rows by group, ascending within one; those whose key is outside [0, groups) are behind the
// last group. offsets [groups + 1]. place [n], or null: a row's position in perm, or -1 for a row
// without a group. Row i's key is keys[i * stride]. n <= 2^31 - 1024.
int group_rows(const int32_t* keys, int64_t stride, int64_t n, int groups, int32_t* perm,
               int32_t* offsets, int32_t* place, void* workspace, cudaStream_t s);

// The second of its steps by itself, for a plan that is not small and counts that are there.
int group_place(const GroupPlan& plan, const int32_t* keys, int64_t stride, int64_t n, int groups,
                const int32_t* counts, int32_t* perm, int32_t* offsets, int32_t* place,
                cudaStream_t s);

#ifdef __CUDACC__
__device__ __forceinline__ int bin_of(int32_t key, int groups) {
  return key >= 0 && key < groups ? key : groups;
}

constexpr int GROUP_AHEAD = 8;  // keys of a lane that are loaded together

// A lane's bins of the GROUP_AHEAD * 32 rows from i0 on; -1 behind b.
__device__ __forceinline__ void load_bins(const int32_t* keys, int64_t stride, int64_t i0, int64_t b,
                                          int groups, int (&bins)[GROUP_AHEAD]) {
#pragma unroll
  for (int s = 0; s < GROUP_AHEAD; ++s) {
    const int64_t i = i0 + 32 * s + (threadIdx.x & 31);
    bins[s] = i < b ? bin_of(keys[i * stride], groups) : -1;
  }
}

// A warp adds rows [a, b) to its counters `mine` (shared memory, zeroed): one addition a key among 32
// rows, since neighbours often have the same one.
__device__ __forceinline__ void count_part(const int32_t* keys, int64_t stride, int64_t a, int64_t b,
                                           int groups, int32_t* mine) {
  const unsigned below = (1u << (threadIdx.x & 31)) - 1u;
  for (int64_t i0 = a; i0 < b; i0 += 32 * GROUP_AHEAD) {
    int bins[GROUP_AHEAD];
    load_bins(keys, stride, i0, b, groups, bins);
#pragma unroll
    for (int s = 0; s < GROUP_AHEAD; ++s) {
      const unsigned same = __match_any_sync(0xffffffffu, bins[s]);
      if (bins[s] >= 0 && (same & below) == 0u) atomicAdd(mine + bins[s], __popc(same));
    }
  }
  __syncwarp();
}

// A warp writes rows [a, b) to their positions, 32 at a time, ranked among those with the same key;
// `mine`: where each bin's next row goes.
__device__ __forceinline__ void place_part(const int32_t* keys, int64_t stride, int64_t a, int64_t b,
                                           int groups, int32_t* mine, int32_t* perm,
                                           int32_t* place) {
  const int lane = threadIdx.x & 31;
  for (int64_t i0 = a; i0 < b; i0 += 32 * GROUP_AHEAD) {
    int bins[GROUP_AHEAD];
    load_bins(keys, stride, i0, b, groups, bins);
#pragma unroll
    for (int s = 0; s < GROUP_AHEAD; ++s) {
      const int bin = bins[s];
      const unsigned same = __match_any_sync(0xffffffffu, bin);
      const int rank = __popc(same & ((1u << lane) - 1u));
      int at = 0;
      if (bin >= 0) at = mine[bin] + rank;
      __syncwarp();
      if (bin >= 0 && rank == 0) mine[bin] += __popc(same);
      __syncwarp();
      if (bin >= 0) {
        const int64_t i = i0 + 32 * s + lane;
        perm[at] = (int32_t)i;
        if (place) place[i] = bin < groups ? at : -1;
      }
    }
  }
}

// Exclusive sums over counts[0..total) in place, by one block of 1024 threads; part: 32 words.
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

// Everything by one block of 1024 threads. counts: shared memory, 2 x 32 (groups + 1) words; part: 32.
__device__ __forceinline__ void group_block(const int32_t* keys, int64_t stride, int n, int groups,
                                            int32_t* perm, int32_t* offsets, int32_t* place,
                                            int32_t* counts, int32_t* part) {
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

// Segments of `offsets` [groups + 1], found by a warp: offsets are taken into [0, limit] and made to rise,
// whatever they are, so that segments never overlap (an offset below one before it is that one). What
// is done for all of them is then bounded by `limit`.
struct Segment {
  int first, last;
};
__device__ __forceinline__ int inside(const int32_t* offsets, int g, int limit) {
  return min(max(__ldg(offsets + g), 0), limit);
}
__device__ __forceinline__ Segment segment_at(const int32_t* offsets, int g, int limit) {
  int first = 0;
  for (int j0 = 0; j0 <= g; j0 += 32) {
    const int j = j0 + (int)(threadIdx.x & 31);
    first = max(first, __reduce_max_sync(0xffffffffu, j <= g ? inside(offsets, j, limit) : 0));
  }
  return {first, max(first, inside(offsets, g + 1, limit))};
}
// The positions that segments have, all of them together: those before the first segment and behind the last
// one have none.
__device__ __forceinline__ Segment covered(const int32_t* offsets, int groups, int limit) {
  int last = 0;
  for (int j = threadIdx.x & 31; j <= groups; j += 32) last = max(last, inside(offsets, j, limit));
  return {inside(offsets, 0, limit), __reduce_max_sync(0xffffffffu, last)};
}
// A lane's inclusive maximum over the lanes up to it, and `before`.
__device__ __forceinline__ int rising(int v, int before) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if ((int)(threadIdx.x & 31) >= o) v = max(v, u);
  }
  return max(v, before);
}

// The segments cut into pieces of `unit` rows, in order; TAIL: the rows behind the last segment, up to
// `limit`, are segment `groups`. Piece `index` is rows [first, last) of segment `group`; group < 0:
// there are fewer pieces.
struct Piece {
  int group, first, last;
};
template <bool TAIL>
__device__ __forceinline__ Piece find_piece(const int32_t* offsets, int groups, int limit, int unit,
                                            int64_t index) {
  const int lane = threadIdx.x & 31;
  int64_t before = 0;
  int top = 0;
  for (int g0 = 0; g0 < groups + TAIL; g0 += 32) {
    const int g = g0 + lane;
    const bool in = g < groups + TAIL;
    const int a = rising(in ? inside(offsets, g, limit) : 0, top);
    const int b = !in ? a : g < groups ? max(a, inside(offsets, g + 1, limit)) : limit;
    top = __shfl_sync(0xffffffffu, a, 31);
    const int64_t count = ((int64_t)b - a + unit - 1) / unit;
    int64_t upto = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    upto += before;
    const unsigned hit = __ballot_sync(0xffffffffu, index < upto);
    if (hit) {
      const int src = __ffs(hit) - 1;
      const int64_t start = upto - count;
      const int first = a + (int)((index - start) * unit);
      Piece p{g, first, (int)min((int64_t)first + unit, (int64_t)b)};
      p.group = __shfl_sync(0xffffffffu, p.group, src);
      p.first = __shfl_sync(0xffffffffu, p.first, src);
      p.last = __shfl_sync(0xffffffffu, p.last, src);
      return p;
    }
    before = __shfl_sync(0xffffffffu, upto, 31);
  }
  return {-1, 0, 0};
}

// How many pieces there are before segment g, and of it.
__device__ __forceinline__ int2 pieces_at(const int32_t* offsets, int g, int limit, int unit) {
  const int lane = threadIdx.x & 31;
  int before = 0, top = 0;
  for (int j0 = 0; j0 < g; j0 += 32) {
    const int j = j0 + lane;
    const int a = rising(j < g ? inside(offsets, j, limit) : 0, top);
    const int b = j < g ? max(a, inside(offsets, j + 1, limit)) : a;
    top = __shfl_sync(0xffffffffu, a, 31);
    before += __reduce_add_sync(0xffffffffu, (b - a + unit - 1) / unit);
  }
  const Segment s = segment_at(offsets, g, limit);
  return make_int2(before, (s.last - s.first + unit - 1) / unit);
}
#endif

}  // namespace sv
