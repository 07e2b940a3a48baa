// Stable grouping of rows by a key, as a counting sort on the device (group.cu): the router's slots by
// expert, and the rows of a block's modulations by batch element.
#pragma once

#include "common.cuh"

namespace sv {

constexpr int GROUP_MAX_BINS = 4096;  // groups, and one more for the rows without one

// Bytes that group_rows needs for n rows and `groups` groups.
size_t group_rows_bytes(int64_t n, int groups);

// perm: the rows by group, ascending within one; those whose key is outside [0, groups) are behind the
// last group. offsets [groups + 1]. place [n], or null: a row's position in perm, or -1 for a row
// without a group. Row i's key is keys[i * stride]. n <= 2^31 - 1024.
int group_rows(const int32_t* keys, int64_t stride, int64_t n, int groups, int32_t* perm,
               int32_t* offsets, int32_t* place, void* workspace, cudaStream_t s);

#ifdef __CUDACC__
// The lanes of a warp cut the segments of `offsets` [groups + 1] into pieces of `unit` rows, in order;
// TAIL: the rows behind the last segment, up to `limit`, are segment `groups`. Piece `index` is rows
// [first, last) of segment `group`; group < 0: there are fewer pieces. Offsets are taken into
// [0, limit] and made to rise, whatever they are.
struct Piece {
  int group, first, last;
};
template <bool TAIL>
__device__ __forceinline__ Piece find_piece(const int32_t* offsets, int groups, int limit, int unit,
                                            int64_t index) {
  const int lane = threadIdx.x & 31;
  int64_t before = 0;
  for (int g0 = 0; g0 < groups + TAIL; g0 += 32) {
    const int g = g0 + lane;
    int a = 0, b = 0;
    if (g < groups + TAIL) {
      a = min(max(__ldg(offsets + g), 0), limit);
      b = g < groups ? max(min(__ldg(offsets + g + 1), limit), a) : limit;
    }
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
#endif

}  // namespace sv
