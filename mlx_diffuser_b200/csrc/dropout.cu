// y = drop(x) + residual, element by element (dropout.cuh has the random numbers). The gradient of x is
// drop(dy), by the same numbers: one kernel serves both passes.
#include <algorithm>

#include "dropout.cuh"

namespace sv {
namespace {

template <typename T>
struct Eight {
  alignas(16) T e[8];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(e) / 16; ++i)
      reinterpret_cast<uint4*>(e)[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < (int)sizeof(e) / 16; ++i)
      reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(e)[i];
  }
};

// A thread takes AHEAD counters (eight elements each) a grid apart at a time, their loads together. WIDE:
// every pointer 16-byte aligned, and all but the last counter's elements in 16-byte accesses. A pass over
// 40,662 x 1024 bf16 is 167 MB, 25 us of HBM, and takes 31 us (38 with the keys added up for every
// counter): its instructions bound it, a counter's ten rounds 40 and the eight selections 28.
template <typename T, bool WIDE, bool RES>
__global__ void __launch_bounds__(256)
    dropout_kernel(const T* x, const T* residual, T* out, int64_t cells, Dropout d) {
  constexpr int AHEAD = 2;
  PhiloxKeys keys(seed_of(d));
  keys.held();
  const int64_t step = (int64_t)gridDim.x * 256, whole = WIDE ? cells / 8 : 0;
  int64_t g = (int64_t)blockIdx.x * 256 + threadIdx.x;
  auto work = [&](int64_t at, const Eight<T>& from, const Eight<T>& add, Eight<T>& to) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32(from.e[i]);
    if (d.cut) drop_eight(v, philox((uint64_t)at, d.subsequence, keys), d);
    if constexpr (RES) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += to_f32(add.e[i]);
    }
    pack_eight<T>(v, *reinterpret_cast<uint4(*)[sizeof(T) / 2]>(to.e));
  };
  if constexpr (WIDE) {
    for (; g + (AHEAD - 1) * step < whole; g += AHEAD * step) {
      Eight<T> from[AHEAD], add[AHEAD];
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) {
        from[a].load(x + (g + a * step) * 8);
        if constexpr (RES) add[a].load(residual + (g + a * step) * 8);
      }
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) {
        Eight<T> to;
        work(g + a * step, from[a], add[a], to);
        to.store(out + (g + a * step) * 8);
      }
    }
    for (; g < whole; g += step) {
      Eight<T> from, add, to;
      from.load(x + g * 8);
      if constexpr (RES) add.load(residual + g * 8);
      work(g, from, add, to);
      to.store(out + g * 8);
    }
  }
  for (; g * 8 < cells; g += step) {  // element by element
    Eight<T> from, add, to;
    const int64_t at = g * 8;
    const int left = (int)min((int64_t)8, cells - at);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      from.e[i] = i < left ? x[at + i] : from_f32<T>(0.0f);
      if constexpr (RES) add.e[i] = i < left ? residual[at + i] : from_f32<T>(0.0f);
    }
    work(g, from, add, to);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) out[at + i] = to.e[i];
  }
}

template <typename T>
int launch_dropout(const void* x, const void* residual, void* out, int64_t cells,
                   const Dropout& d, cudaStream_t s) {
  const bool wide = aligned16(x) && aligned16(out) && (!residual || aligned16(residual));
  const int64_t groups = (cells + 7) / 8;
  const unsigned blocks =
      (unsigned)std::min<int64_t>((groups + 255) / 256, (int64_t)num_sms() * 16);
  auto kernel = residual ? (wide ? dropout_kernel<T, true, true> : dropout_kernel<T, false, true>)
                         : (wide ? dropout_kernel<T, true, false> : dropout_kernel<T, false, false>);
  kernel<<<blocks, 256, 0, s>>>(static_cast<const T*>(x), static_cast<const T*>(residual),
                                static_cast<T*>(out), cells, d);
  SV_LAUNCH_CHECK();
  return SV_OK;
}

}  // namespace
}  // namespace sv

using namespace sv;

extern "C" int sv_dropout(const void* x, const void* residual, int64_t cells, int dtype, double p,
                          uint64_t seed, const void* seed_at, uint64_t subsequence, void* out,
                          sv_stream_t stream) {
  if (cells < 0) SV_FAIL(SV_ERR_INVALID_ARGUMENT, "sv_dropout: negative size");
  if (!(p >= 0.0 && p <= 1.0)) SV_FAIL(SV_ERR_INVALID_ARGUMENT, "sv_dropout: p outside [0, 1]");
  if (dtype != SV_FLOAT32 && dtype != SV_FLOAT16 && dtype != SV_BFLOAT16)
    SV_FAIL(SV_ERR_BAD_DTYPE, "sv_dropout: unknown dtype");
  if (cells == 0) return SV_OK;
  if (!x || !out) SV_FAIL(SV_ERR_INVALID_ARGUMENT, "sv_dropout: null pointer");
  const Dropout d = make_dropout(p, seed, seed_at, subsequence);
  cudaStream_t s = to_stream(stream);
  switch (dtype) {
    case SV_FLOAT32: return launch_dropout<float>(x, residual, out, cells, d, s);
    case SV_FLOAT16: return launch_dropout<__half>(x, residual, out, cells, d, s);
    default: return launch_dropout<__nv_bfloat16>(x, residual, out, cells, d, s);
  }
}
