// y = drop(x) + residual, element by element (dropout.cuh has the random numbers). The gradient of x is
// drop(dy), by the same numbers: one kernel serves both passes.
#include <algorithm>

#include "dropout.cuh"

namespace sv {
namespace {

template <typename T>
__device__ __forceinline__ void load_eight(const T* p, float (&v)[8]) {
  alignas(16) T e[8];
#pragma unroll
  for (int i = 0; i < (int)sizeof(e) / 16; ++i)
    reinterpret_cast<uint4*>(e)[i] = reinterpret_cast<const uint4*>(p)[i];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = to_f32(e[i]);
}

// A thread takes counters (eight elements) a grid apart. WIDE: every pointer 16-byte aligned, so that
// only the last counter is read and written element by element.
template <typename T, bool WIDE, bool RES>
__global__ void __launch_bounds__(256)
    dropout_kernel(const T* x, const T* residual, T* out,
                   int64_t cells, Dropout d) {
  const uint64_t seed = seed_of(d);
  const int64_t groups = (cells + 7) / 8, step = (int64_t)gridDim.x * 256;
#pragma unroll 2
  for (int64_t g = (int64_t)blockIdx.x * 256 + threadIdx.x; g < groups; g += step) {
    const int64_t at = g * 8;
    const int left = (int)min((int64_t)8, cells - at);
    float v[8], r[8];
    if (WIDE && left == 8) {
      load_eight(x + at, v);
      if constexpr (RES) load_eight(residual + at, r);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = i < left ? to_f32(x[at + i]) : 0.0f;
        if constexpr (RES) r[i] = i < left ? to_f32(residual[at + i]) : 0.0f;
      }
    }
    if (d.cut) drop_eight(v, philox((uint64_t)g, d.subsequence, seed), d);
    alignas(16) T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(RES ? v[i] + r[i] : v[i]);
    if (WIDE && left == 8) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(e) / 16; ++i)
        reinterpret_cast<uint4*>(out + at)[i] = reinterpret_cast<const uint4*>(e)[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < left) out[at + i] = e[i];
    }
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
