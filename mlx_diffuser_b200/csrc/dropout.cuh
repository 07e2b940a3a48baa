// Dropout whose mask is a function of the element's number: counter-based random numbers, formed again
// wherever they are wanted, so that no mask is stored between the passes.
//
// Philox4x32 with ten rounds (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as
// 1, 2, 3", 2011): key = the seed's two words, counter = (g, subsequence) as two words each. One counter
// gives eight 16-bit numbers, those of the elements 8 g .. 8 g + 7 in row-major order, the low half of
// a word first. An element is dropped when its number is below `cut` = p 2^16 rounded, and kept
// ones are multiplied by 2^16 / (2^16 - cut), which keeps the mean exactly. 16 bits an element, since
// with 32 the generator's integer products would bound the pass and not HBM.
#pragma once

#include "common.cuh"

namespace sv {

struct Dropout {
  uint32_t cut;      // 0: nothing is dropped; 65536: everything
  float scale;       // of what is kept
  uint64_t seed;
  const uint64_t* seed_at;  // on the device, read instead of `seed`; or null
  uint64_t subsequence;
};

inline Dropout make_dropout(double p, uint64_t seed, const void* seed_at, uint64_t subsequence) {
  Dropout d;
  d.cut = (uint32_t)(p * 65536.0 + 0.5);
  d.scale = d.cut >= 65536u ? 0.0f : (float)(65536.0 / (65536.0 - d.cut));
  d.seed = seed;
  d.seed_at = static_cast<const uint64_t*>(seed_at);
  d.subsequence = subsequence;
  return d;
}

#ifdef __CUDACC__
__device__ __forceinline__ uint64_t seed_of(const Dropout& d) {
  return d.seed_at ? __ldg(reinterpret_cast<const unsigned long long*>(d.seed_at)) : d.seed;
}

// The keys of the ten rounds. held(): in registers, where a loop has 20 to spare; left to itself the
// compiler adds them up again for every counter, a sixth of its instructions.
struct PhiloxKeys {
  uint32_t low[10], high[10];
  __device__ __forceinline__ explicit PhiloxKeys(uint64_t seed) {
#pragma unroll
    for (int r = 0; r < 10; ++r) {
      low[r] = (uint32_t)seed + (uint32_t)r * 0x9E3779B9u;
      high[r] = (uint32_t)(seed >> 32) + (uint32_t)r * 0xBB67AE85u;
    }
  }
  __device__ __forceinline__ void held() {
#pragma unroll
    for (int r = 0; r < 10; ++r) asm volatile("" : "+r"(low[r]), "+r"(high[r]));
  }
};

__device__ __forceinline__ uint4 philox(uint64_t group, uint64_t subsequence, const PhiloxKeys& key) {
  uint32_t c0 = (uint32_t)group, c1 = (uint32_t)(group >> 32);
  uint32_t c2 = (uint32_t)subsequence, c3 = (uint32_t)(subsequence >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ key.low[r];
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ key.high[r];
    c3 = (uint32_t)a;
  }
  return make_uint4(c0, c1, c2, c3);
}
// Bit i: element i of the counter's eight is kept. A half is compared where it stands, in a word's upper
// half: the lower bits of the word cannot change the comparison with cut 2^16.
__device__ __forceinline__ uint32_t kept_eight(const uint4& r, const Dropout& d) {
  if (d.cut >= 65536u) return 0u;
  const uint32_t w[4] = {r.x, r.y, r.z, r.w}, cut = d.cut << 16;
  uint32_t kept = 0u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    kept |= (w[i] << 16) >= cut ? 1u << 2 * i : 0u;
    kept |= w[i] >= cut ? 2u << 2 * i : 0u;
  }
  return kept;
}

// v[0..7], the elements of one counter: scaled, or zero whatever they were.
__device__ __forceinline__ void drop_eight(float (&v)[8], const uint4& r, const Dropout& d) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
  if (d.cut >= 65536u) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    return;
  }
  const uint32_t cut = d.cut << 16;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = (w[i] << 16) >= cut ? v[2 * i] * d.scale : 0.0f;
    v[2 * i + 1] = w[i] >= cut ? v[2 * i + 1] * d.scale : 0.0f;
  }
}

// Whether element `at` by itself is kept.
__device__ __forceinline__ uint32_t kept_one(uint64_t at, const PhiloxKeys& keys, const Dropout& d) {
  return kept_eight(philox(at >> 3, d.subsequence, keys), d) >> ((uint32_t)at & 7u) & 1u;
}
#endif

}  // namespace sv
