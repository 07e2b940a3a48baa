// Rows through a pipeline per warp, shared by rmsnorm.cu and blocknorm.cu: each warp keeps the next rows in
// flight by bulk copies into shared memory of its own, with no barrier between warps.
#pragma once

#include "common.cuh"

namespace sv {

constexpr int ROW_WARPS = 8;

template <typename T, int J>
struct RowRing {
  static constexpr int V = 16 / sizeof(T);
  static constexpr int ROW = 32 * J * 16;  // bytes of the widest row
  static constexpr int SMEM(int tensors, int stages) {
    return ROW_WARPS * (tensors * stages * ROW + stages * 8) + 16;
  }
};

template <typename T>
__device__ __forceinline__ void unpack(const uint4& raw, float (&v)[16 / sizeof(T)]) {
  const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
  for (int k = 0; k < 16 / (int)sizeof(T); ++k) v[k] = to_f32(e[k]);
}

// Calls row(r, k, stage, release) for the warp's rows r = first + k step below n, with their TENSORS rows in
// shared memory (base + tensor * ROW), STAGES rows ahead; it calls release() when it has read them.
// ahead(r, k): what src(t, .) wants of row r, found by all lanes when the row's copies are issued.
template <typename T, int J, int TENSORS, int STAGES, typename Ahead, typename Src, typename Row>
__device__ __forceinline__ bool run_rows(uint8_t* smem, int64_t first, int64_t step, int64_t n,
                                         uint32_t bytes, int tensors, volatile int* abort_flag,
                                         Ahead&& ahead, Src&& src, Row&& row) {
  using Ring = RowRing<T, J>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* ring = smem + warp * TENSORS * STAGES * Ring::ROW;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + ROW_WARPS * TENSORS * STAGES * Ring::ROW) +
                   warp * STAGES;
  if (lane == 0) {
    for (int s = 0; s < STAGES; ++s) mbar_init(&full[s], 1);
    fence_mbar_init();
  }
  __syncwarp();
  auto load = [&](int64_t r, int64_t k, int s) {
    if (r >= n) return;  // the same in all lanes
    const auto which = ahead(r, k);
    if (lane == 0) {
      mbar_arrive_expect_tx(&full[s], bytes * tensors);
      for (int t = 0; t < tensors; ++t)
        bulk_load(smem_u32(ring + (s * TENSORS + t) * Ring::ROW), src(t, which), bytes, &full[s]);
    }
  };
#pragma unroll
  for (int s = 0; s < STAGES; ++s) load(first + s * step, s, s);
  int s = 0, phase = 0;
  int64_t k = 0;
  for (int64_t r = first; r < n; r += step, ++k) {
    if (!__all_sync(0xffffffffu, mbar_wait_bounded(&full[s], phase, abort_flag))) {
      // the warp's copies in flight write its ring: let them land
      const uint64_t t0 = global_timer_ns();
      while (global_timer_ns() - t0 < 10000000ull) {
      }
      return false;
    }
    row(r, k, ring + s * TENSORS * Ring::ROW, [&] {
      __syncwarp();  // every lane has read the stage
      load(r + STAGES * step, k + STAGES, s);
    });
    if (++s == STAGES) {
      s = 0;
      phase ^= 1;
    }
  }
  return true;
}

}  // namespace sv
