// Windowed attention with a learned relative position bias in fp32 (the formulas are attention.cu's):
// exact fp32 products and sums on the CUDA cores.
//
// A block takes up to 64 rows of one head out of the plan's list, eight warps of eight rows, and walks
// the positions that their windows cover in tiles of 32, fetched one ahead by cp.async. For the
// scores a lane holds one position's row and the warp's own rows are broadcast (one 16-byte read of
// the tile and eight of the rows for 32 fused multiply-adds); the weights then go through shared
// memory, and for the sums the lanes lie along the channels. So a row of the other side leaves HBM or
// L2 once per 64 rows and shared memory once per eight. Shared-memory reads bound it, at about one per
// three multiply-adds. 10,000 rows x 8 heads x 64, windows of 8^3: forward 204 us, dq and the table 293,
// dk and dv 275; a warp per row straight from global memory, one position a lane, was bound by L1 (32
// lines an access) and took 1,137, 1,311 and 1,461 us.
//
// The table's gradient sums in 64-bit fixed point, so that neither the order of the atomics nor
// the number of blocks changes it.
#include <limits.h>

#include <algorithm>

#include "attention.h"

namespace sv {
namespace {

constexpr int FB = 64;  // rows of a block
constexpr int FT = 32;  // positions of a tile, one a lane
constexpr int FW = 8;   // warps
constexpr int FR = FB / FW;
constexpr int F_THREADS = 32 * FW;

enum Pass { FORWARD, DQ, DKV };

// Shared memory in floats: the block's rows, two buffers of two tiles, the warps' weights (and score
// gradients), the look-up; then what F32Shared holds. Rows lie DP + 4 floats apart, so that the
// 16-byte reads of eight lanes fall into different banks.
struct alignas(16) F32Shared {
  PlanRow own[FB];
  PlanRow key[2][FT];
  float2 stats[2][FT];
  float delta[2][FT];
  int range[2];
};
template <int DP, Pass PASS>
struct F32Layout {
  static constexpr int LD = DP + 4;
  static constexpr int OWN = PASS == FORWARD ? 1 : 2;
  static constexpr int RING = OWN * FB * LD;
  static constexpr int WEIGHTS = RING + 4 * FT * LD;
  static constexpr int SHARED = WEIGHTS + (PASS == DKV ? 2 : 1) * FB * FT;
  static constexpr int LUT = SHARED + (int)sizeof(F32Shared) / 4;
  static size_t bytes(int reach) { return (LUT + 2 * (size_t)reach + 1) * 4; }
};

// `rows` rows of one head into shared memory; rows of -1 and channels past `dim` become zeros.
template <int DP, typename RowOf>
__device__ __forceinline__ void load_rows(float* tile, int rows, const float* base, int64_t stride,
                                          int dim, bool vec, RowOf&& row_of) {
  constexpr int LD = DP + 4, CH = DP / 4;
  if (vec) {
    for (int i = threadIdx.x; i < rows * CH; i += F_THREADS) {
      const int r = i / CH, c = i % CH * 4;
      const int32_t row = row_of(r);
      const bool in = row >= 0 && c < dim;
      cp_async_16(smem_u32(tile + r * LD + c), in ? base + row * stride + c : base, in ? 16u : 0u);
    }
  } else {
    for (int i = threadIdx.x; i < rows * DP; i += F_THREADS) {
      const int r = i / DP, c = i % DP;
      const int32_t row = row_of(r);
      tile[r * LD + c] = row >= 0 && c < dim ? base[row * stride + c] : 0.f;
    }
  }
}

// s[r] = the warp's row r times the lane's row of a tile.
template <int DP>
__device__ __forceinline__ void dots(const float* rows, const float* mine, float (&s)[FR]) {
  constexpr int LD = DP + 4;
#pragma unroll
  for (int r = 0; r < FR; ++r) s[r] = 0.f;
#pragma unroll 4
  for (int d = 0; d < DP; d += 4) {
    const float4 k = *reinterpret_cast<const float4*>(mine + d);
#pragma unroll
    for (int r = 0; r < FR; ++r) {
      const float4 q = *reinterpret_cast<const float4*>(rows + r * LD + d);
      s[r] = fmaf(q.x, k.x, fmaf(q.y, k.y, fmaf(q.z, k.z, fmaf(q.w, k.w, s[r]))));
    }
  }
}

// o[r] += sum over the tile's rows j of w[r][j] times row j, channels lane, lane + 32, ...
template <int DP>
__device__ __forceinline__ void add_rows(float (&o)[FR][DP / 32], const float* w,
                                         const float* tile) {
  constexpr int LD = DP + 4, CH = DP / 32;
  const int lane = threadIdx.x & 31;
#pragma unroll 2
  for (int j = 0; j < FT; j += 4) {
    float v[4][CH];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int c = 0; c < CH; ++c) v[i][c] = tile[(j + i) * LD + lane + 32 * c];
#pragma unroll
    for (int r = 0; r < FR; ++r) {
      const float4 p = *reinterpret_cast<const float4*>(w + r * FT + j);
#pragma unroll
      for (int c = 0; c < CH; ++c)
        o[r][c] = fmaf(p.x, v[0][c], fmaf(p.y, v[1][c], fmaf(p.z, v[2][c],
                                                             fmaf(p.w, v[3][c], o[r][c]))));
    }
  }
}

template <int DP, Pass PASS>
__global__ void __launch_bounds__(F_THREADS) attn_f32_kernel(AttnArgs a, bool vec) {
  using L = F32Layout<DP, PASS>;
  constexpr int LD = L::LD, CH = DP / 32;
  extern __shared__ __align__(16) float smem[];
  F32Shared& sh = *reinterpret_cast<F32Shared*>(smem + L::SHARED);
  int* lut = reinterpret_cast<int*>(smem + L::LUT);
  const PlanBlocks at = plan_blocks(a.n);
  const uint8_t* bytes = reinterpret_cast<const uint8_t*>(a.plan);
  const int2* list = reinterpret_cast<const int2*>(bytes + at.block[0]);
  const int count = (int)min((int64_t)__ldg(reinterpret_cast<const int*>(bytes + at.count)),
                             at.cap[0]);
  if ((int)blockIdx.x >= count) return;
  const int h = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row0 = warp * FR;
  const int64_t g_row = (int64_t)a.heads * a.dim;
  const float* q = static_cast<const float*>(a.q) + h * a.q_head;
  const float* k = static_cast<const float*>(a.k) + h * a.k_head;
  const float* v = static_cast<const float*>(a.v) + h * a.v_head;
  const float* g = PASS == FORWARD ? nullptr
                                   : static_cast<const float*>(a.dout) + (int64_t)h * a.dim;
  const int cells = a.nb * a.nb * a.nb;
  const float* table = static_cast<const float*>(a.table) + (int64_t)h * cells;
  for (int i = threadIdx.x; i <= 2 * a.reach; i += F_THREADS)
    lut[i] = max(0, min(a.nb - 1, __ldg(a.lut + i)));
  auto axis = [&](int d) { return lut[max(-a.reach, min(a.reach, d)) + a.reach]; };
  auto bucket = [&](const PlanRow& from, const PlanRow& to) {
    return (axis(sub_sat(to.x, from.x)) * a.nb + axis(sub_sat(to.y, from.y))) * a.nb +
           axis(sub_sat(to.z, from.z));
  };
  const int exponent = PASS == DQ && a.dtable ? dtable_exponent(a, h) : INT_MAX;
  const double unit = exponent == INT_MAX ? 0.0 : ldexp(1.0, exponent);
  float* rows_a = smem + row0 * LD;            // the warp's rows of the first own tile
  float* rows_b = rows_a + FB * LD;            // and of the second
  float* w0 = smem + L::WEIGHTS + row0 * FT;   // its weights
  float* w1 = w0 + FB * FT;                    // its score gradients (dk / dv)

  for (int block = blockIdx.x; block < count; block += gridDim.x) {
    const int2 span = __ldg(list + block);
    __syncthreads();  // the previous block is done with
    if (threadIdx.x < 2) sh.range[threadIdx.x] = threadIdx.x ? INT_MIN : INT_MAX;
    __syncthreads();
    if (threadIdx.x < FB) {
      const bool in = (int)threadIdx.x < span.y;
      PlanRow r = plan_at(a.plan, in ? span.x + threadIdx.x : span.x);
      if (!in) r.row = -1;
      if (r.row < 0) {
        r.start = r.end = 0;
      } else {
        atomicMin(&sh.range[0], r.start);
        atomicMax(&sh.range[1], r.end);
      }
      sh.own[threadIdx.x] = r;
    }
    __syncthreads();
    const int j0 = sh.range[0], j1 = sh.range[1];
    const int tiles = j1 > j0 ? (j1 - j0 + FT - 1) / FT : 0;
    auto own_row = [&](int r) { return sh.own[r].row; };
    load_rows<DP>(smem, FB, PASS == DKV ? k : q, PASS == DKV ? a.k_row : a.q_row, a.dim, vec,
                  own_row);
    if constexpr (PASS == DQ) load_rows<DP>(smem + FB * LD, FB, g, g_row, a.dim, vec, own_row);
    if constexpr (PASS == DKV) load_rows<DP>(smem + FB * LD, FB, v, a.v_row, a.dim, vec, own_row);
    auto load = [&](int t) {
      const int buf = t & 1, first = j0 + t * FT;
      float* tile = smem + L::RING + buf * 2 * FT * LD;
      auto row_of = [&](int r) { return first + r < j1 ? __ldg(&a.plan[first + r].row) : -1; };
      if constexpr (PASS == DKV) {
        load_rows<DP>(tile, FT, q, a.q_row, a.dim, vec, row_of);
        load_rows<DP>(tile + FT * LD, FT, g, g_row, a.dim, vec, row_of);
      } else {
        load_rows<DP>(tile, FT, k, a.k_row, a.dim, vec, row_of);
        load_rows<DP>(tile + FT * LD, FT, v, a.v_row, a.dim, vec, row_of);
      }
      if (threadIdx.x < FT) {
        const int j = first + threadIdx.x;
        PlanRow r{};
        r.row = -1;
        if (j < j1) r = plan_at(a.plan, j);
        sh.key[buf][threadIdx.x] = r;
        if constexpr (PASS == DKV) {
          sh.stats[buf][threadIdx.x] = r.row >= 0 ? a.stats[h * a.n + j] : make_float2(0.f, 0.f);
          sh.delta[buf][threadIdx.x] = r.row >= 0 ? a.delta[h * a.n + j] : 0.f;
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    if (tiles > 0) load(0);
    const PlanRow& some = sh.own[row0 + lane % FR];
    const int lo = __reduce_min_sync(0xffffffffu, some.row >= 0 ? some.start : INT_MAX);
    const int hi = __reduce_max_sync(0xffffffffu, some.row >= 0 ? some.end : INT_MIN);

    float first[FR], second[FR];  // forward: maximum and the lane's sum; dq: delta
    float2 stats[FR];
    float o[FR][CH], o2[FR][CH];
#pragma unroll
    for (int r = 0; r < FR; ++r) {
      first[r] = PASS == FORWARD ? -INFINITY : 0.f;
      second[r] = 0.f;
      stats[r] = make_float2(0.f, 0.f);
#pragma unroll
      for (int c = 0; c < CH; ++c) o[r][c] = o2[r][c] = 0.f;
      if constexpr (PASS == DQ) {
        const PlanRow& me = sh.own[row0 + r];
        if (me.row >= 0) {
          const int64_t p = h * a.n + span.x + row0 + r;
          const int64_t own = (me.row * (int64_t)a.heads + h) * a.dim;
          float d = 0.f;
          for (int c = lane; c < a.dim; c += 32)
            d = fmaf(static_cast<const float*>(a.dout)[own + c],
                     static_cast<const float*>(a.o)[own + c], d);
          first[r] = warp_sum(d);
          if (lane == 0) a.delta[p] = first[r];
          stats[r] = a.stats[p];
        }
      }
    }

    for (int t = 0; t < tiles; ++t) {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      __syncthreads();  // tile t is there for everybody, and nobody reads the other buffer
      if (t + 1 < tiles) load(t + 1);
      const int buf = t & 1, p0 = j0 + t * FT, j = p0 + lane;
      if (p0 >= hi || p0 + FT <= lo) continue;
      const float* tile = smem + L::RING + buf * 2 * FT * LD;
      const PlanRow key = sh.key[buf][lane];
      float s[FR], dp[FR];
      dots<DP>(rows_a, tile + lane * LD, s);
      if constexpr (PASS != FORWARD) dots<DP>(rows_b, tile + (FT + lane) * LD, dp);
      __syncwarp();  // the previous tile's weights have been read
#pragma unroll
      for (int r = 0; r < FR; ++r) {
        const PlanRow me = sh.own[row0 + r];
        const bool in = j >= me.start && j < me.end && key.row >= 0;
        const int b = in ? (PASS == DKV ? bucket(key, me) : bucket(me, key)) : 0;
        const float x = in ? fmaf(s[r], a.scale, __ldg(table + b)) : -INFINITY;
        if constexpr (PASS == FORWARD) {
          const float m = fmaxf(first[r], warp_max(x));
          const float base = m == -INFINITY ? 0.f : m;
          if (m > first[r]) {  // the same in all lanes
            const float keep = expf(first[r] - base);
            second[r] *= keep;
#pragma unroll
            for (int c = 0; c < CH; ++c) o[r][c] *= keep;
            first[r] = m;
          }
          const float e = expf(x - base);
          second[r] += e;
          w0[r * FT + lane] = e;
        } else if constexpr (PASS == DQ) {
          const bool counts = in && !lone(me);
          const float ds =
              counts ? expf(x - stats[r].x) * stats[r].y * (dp[r] - first[r]) : 0.f;
          w0[r * FT + lane] = ds;
          if (counts && a.dtable) {
            if (!(fabsf(ds) < INFINITY))
              atomicMax(a.norms + 2 * h, 0x7fffffffu);  // the head's table gradient is NaN
            else if (exponent != INT_MAX)
              atomicAdd(a.dtable + (int64_t)h * cells + b,
                        (unsigned long long)__double2ll_rn((double)ds * unit));
          }
        } else {
          const float2 st = sh.stats[buf][lane];
          const float e = in ? expf(x - st.x) * st.y : 0.f;
          w0[r * FT + lane] = e;
          w1[r * FT + lane] = in && !lone(me) ? e * (dp[r] - sh.delta[buf][lane]) : 0.f;
        }
      }
      __syncwarp();
      // forward: o += P V; dq += dS K; dv += P^T dO, dk += dS^T Q
      add_rows<DP>(o, w0, PASS == DQ ? tile : tile + FT * LD);
      if constexpr (PASS == DKV) add_rows<DP>(o2, w1, tile);
    }
    if (tiles == 0) asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();

#pragma unroll
    for (int r = 0; r < FR; ++r) {
      const PlanRow& me = sh.own[row0 + r];
      if (me.row < 0) continue;  // the same in all lanes
      const int64_t p = span.x + row0 + r;
      const int64_t own = (me.row * (int64_t)a.heads + h) * a.dim;
      float inv = a.scale;
      if constexpr (PASS == FORWARD) {
        const float sum = warp_sum(second[r]);
        inv = sum == 0.f ? 0.f : 1.f / sum;
        if (lane == 0 && a.stats) a.stats[h * a.n + p] = row_stats(first[r], sum);
      }
      bool finite = true;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int d = lane + 32 * c;
        finite = finite && fabsf(o[r][c]) < INFINITY && fabsf(o2[r][c]) < INFINITY;
        if (d >= a.dim) continue;
        if constexpr (PASS == FORWARD) static_cast<float*>(a.out)[own + d] = o[r][c] * inv;
        if constexpr (PASS == DQ) static_cast<float*>(a.dq)[own + d] = o[r][c] * inv;
        if constexpr (PASS == DKV) {
          static_cast<float*>(a.dv)[own + d] = o[r][c];
          static_cast<float*>(a.dk)[own + d] = o2[r][c] * inv;
        }
      }
      // A weight of zero does not hide a NaN or an infinity that another window's row brings into a
      // tile: such rows are computed again from their own windows alone. The weights' floats
      // are the scratch.
      if (!__all_sync(0xffffffffu, finite)) {
        if constexpr (PASS == FORWARD) row_forward<float, false>(a, p, h, w0);
        if constexpr (PASS == DQ) row_dq<float, false>(a, p, h, w0);
        if constexpr (PASS == DKV) row_dkv<float, false>(a, p, h, w0);
      }
    }
  }
}

// norms[h] = bits of the largest |dout_i|^2 and |v_j|^2 of a head. Squares are not negative, so
// their bits order like the values, and a NaN stays above everything.
__global__ void __launch_bounds__(256) attn_norms_kernel(AttnArgs a, unsigned* norms) {
  __shared__ unsigned s_top[2];
  const int h = blockIdx.y;
  if (threadIdx.x < 2) s_top[threadIdx.x] = 0u;
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int64_t r = (int64_t)blockIdx.x * 8 + warp; r < a.n; r += (int64_t)gridDim.x * 8) {
    const float* g = static_cast<const float*>(a.dout) + (r * a.heads + h) * a.dim;
    const float* v = static_cast<const float*>(a.v) + r * a.v_row + h * a.v_head;
    float g2 = 0.f, v2 = 0.f;
    for (int d = lane; d < a.dim; d += 32) {
      g2 = fmaf(g[d], g[d], g2);
      v2 = fmaf(v[d], v[d], v2);
    }
    g2 = warp_sum(g2);
    v2 = warp_sum(v2);
    if (lane == 0) {
      atomicMax(&s_top[0], __float_as_uint(g2) & 0x7fffffffu);
      atomicMax(&s_top[1], __float_as_uint(v2) & 0x7fffffffu);
    }
  }
  __syncthreads();
  if (threadIdx.x < 2) atomicMax(norms + 2 * h + threadIdx.x, s_top[threadIdx.x]);
}

__global__ void __launch_bounds__(256)
    dtable_finish_kernel(AttnArgs a, float* __restrict__ out) {
  const int64_t cells = (int64_t)a.nb * a.nb * a.nb;
  const int h = blockIdx.y;
  const int exponent = dtable_exponent(a, h);
  for (int64_t b = (int64_t)blockIdx.x * 256 + threadIdx.x; b < cells;
       b += (int64_t)gridDim.x * 256) {
    const double v = exponent == INT_MAX
                         ? __longlong_as_double(0x7ff8000000000000ll)  // the inputs were not finite
                         : ldexp((double)(long long)a.dtable[h * cells + b], -exponent);
    out[h * cells + b] = (float)v;
  }
}

bool wide(const void* p, int64_t row, int64_t head) {
  return p == nullptr || (aligned16(p) && row % 4 == 0 && head % 4 == 0);
}

template <int DP, Pass PASS>
int launch(const AttnArgs& a, cudaStream_t s) {
  const size_t bytes = F32Layout<DP, PASS>::bytes(a.reach);
  SV_CUDA_TRY(cudaFuncSetAttribute(attn_f32_kernel<DP, PASS>,
                                   cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  const bool vec = a.dim % 4 == 0 && wide(a.q, a.q_row, a.q_head) &&
                   wide(a.k, a.k_row, a.k_head) && wide(a.v, a.v_row, a.v_head) &&
                   wide(a.dout, 0, 0);
  // every CTA takes a few blocks, so that the lists' unused ends cost little
  const int64_t want = ((int64_t)num_sms() * 16 + a.heads - 1) / a.heads;
  const dim3 grid((unsigned)std::min(want, plan_blocks(a.n).cap[0]), (unsigned)a.heads);
  attn_f32_kernel<DP, PASS><<<grid, F_THREADS, bytes, s>>>(a, vec);
  SV_LAUNCH_CHECK();
  return SV_OK;
}

template <Pass PASS>
int launch_dim(const AttnArgs& a, cudaStream_t s) {
  if (a.dim <= 32) return launch<32, PASS>(a, s);
  if (a.dim <= 64) return launch<64, PASS>(a, s);
  return launch<128, PASS>(a, s);
}

}  // namespace

int attention_f32_forward(const AttnArgs& a, cudaStream_t s) { return launch_dim<FORWARD>(a, s); }

int attention_f32_backward(const AttnArgs& a, void* dtable, cudaStream_t s) {
  if (dtable) {
    const unsigned blocks = (unsigned)std::min<int64_t>((a.n + 63) / 64, 512);
    attn_norms_kernel<<<dim3(blocks, a.heads), 256, 0, s>>>(a, a.norms);
    SV_LAUNCH_CHECK();
  }
  int rc = launch_dim<DQ>(a, s);  // writes the delta that the next one reads
  if (rc == SV_OK) rc = launch_dim<DKV>(a, s);
  if (rc != SV_OK || !dtable) return rc;
  const unsigned blocks = (unsigned)((a.nb * a.nb * a.nb + 255) / 256);
  dtable_finish_kernel<<<dim3(blocks, a.heads), 256, 0, s>>>(a, static_cast<float*>(dtable));
  SV_LAUNCH_CHECK();
  return SV_OK;
}

}  // namespace sv
