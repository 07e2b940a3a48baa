// Windowed attention with a learned relative position bias in fp16 / bf16, on the tensor cores.
//
// The formulas are attention.cu's. A block takes 64 rows in window order (queries, or keys for dk and
// dv) of one head, four warps of 16, and walks the positions that any of their windows covers in
// tiles of 64: rows of several small windows share a tile, and a warp skips the tiles that none of
// its own rows' windows reach. Scores stay in registers from the product to the softmax to the next
// product (the accumulator's layout is the operand's), so the running maximum and sum are the only
// state. The gathered rows arrive by cp.async, one tile ahead.
//
// Products are warp-level mma.sync: a window of a surface holds 100-300 rows, so a tile's two
// products are a few hundred cycles, while each of its 4096 scores needs an exponential and a table
// look-up of its own. The look-up, not the product, is what a faster matrix instruction would wait
// for, and the register layout makes the bias and the softmax free of shared-memory round trips.
//
// The bucket of a pair: where the table is one entry per offset (the look-up is the identity) and
// the windows are no wider than its reach, it is linear in the coordinates and costs a subtraction;
// otherwise three look-ups.
//
// Weights and score gradients are rounded to the feature type as operands of the second products
// (half a step each, like the stored results); the softmax sums and the table's gradient use them
// unrounded.
#include <limits.h>

#include <type_traits>

#include "attention.h"

namespace sv {
namespace {

constexpr int BQ = 64;   // rows of a block
constexpr int BKV = 64;  // positions of a tile
constexpr int AT = 128;  // threads
constexpr float LOG2E = 1.4426950408889634f;

struct KeyMeta {
  int32_t x, y, z;
  int32_t pos;  // INT_MAX: no row
};

// Tiles hold DP channels a row (the head's, padded with zeros) at a stride that is an odd multiple
// of 16 bytes, so the 8 rows of a matrix fragment fall into different banks.
template <int DP>
struct Tile {
  static constexpr int STRIDE = DP * 2 + 16;
  static constexpr int BYTES = 64 * STRIDE;
};

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// 64 gathered rows of one head into a tile; rows of -1 and channels past `dim` become zeros.
template <typename T, int DP>
__device__ __forceinline__ void load_tile(uint8_t* tile, const T* base, int64_t row_stride,
                                          const int32_t* rows, int dim, bool vec) {
  constexpr int CH = DP / 8;  // 16-byte chunks of a row
  if (vec) {
    const uint32_t at = smem_u32(tile);
#pragma unroll
    for (int i = 0; i < 64 * CH / AT; ++i) {
      const int c = threadIdx.x + AT * i;
      const int r = c / CH, col = c % CH;
      const int32_t row = rows[r];
      const bool in = row >= 0 && col * 8 < dim;
      cp_async_16(at + r * Tile<DP>::STRIDE + col * 16,
                  base + (in ? (int64_t)row * row_stride + col * 8 : 0), in ? 16u : 0u);
    }
  } else {
    for (int c = threadIdx.x; c < 64 * DP; c += AT) {
      const int r = c / DP, col = c % DP;
      const int32_t row = rows[r];
      T v = from_f32<T>(0.f);
      if (row >= 0 && col < dim) v = base[(int64_t)row * row_stride + col];
      *reinterpret_cast<T*>(tile + r * Tile<DP>::STRIDE + col * 2) = v;
    }
  }
}

// A 16-row accumulator (a warp's rows of the block) through the warp's own part of a tile to the
// feature rows, in 16-byte stores.
template <typename T, int DP>
__device__ __forceinline__ void store_rows(uint8_t* tile, const float (&o)[DP / 8][4], float s0,
                                           float s1, const int32_t* rows, T* out, int heads,
                                           int head, int dim, bool vec) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c2 = 2 * (lane & 3);
  uint8_t* mine = tile + warp * 16 * Tile<DP>::STRIDE;
  __syncwarp();
#pragma unroll
  for (int n = 0; n < DP / 8; ++n) {
    *reinterpret_cast<uint32_t*>(mine + g * Tile<DP>::STRIDE + (n * 8 + c2) * 2) =
        pack2<T>(o[n][0] * s0, o[n][1] * s0);
    *reinterpret_cast<uint32_t*>(mine + (g + 8) * Tile<DP>::STRIDE + (n * 8 + c2) * 2) =
        pack2<T>(o[n][2] * s1, o[n][3] * s1);
  }
  __syncwarp();
  constexpr int CH = DP / 8;
#pragma unroll
  for (int i = 0; i < 16 * CH / 32; ++i) {
    const int c = lane + 32 * i;
    const int r = c / CH, col = c % CH;
    const int32_t row = rows[warp * 16 + r];
    if (row < 0) continue;
    T* dst = out + ((int64_t)row * heads + head) * dim + col * 8;
    const uint4 v = *reinterpret_cast<const uint4*>(mine + r * Tile<DP>::STRIDE + col * 16);
    if (vec) {
      if (col * 8 < dim) *reinterpret_cast<uint4*>(dst) = v;
    } else {
      const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (col * 8 + k < dim) dst[k] = e[k];
    }
  }
}

// What every kernel here keeps in shared memory besides its tiles.
struct alignas(16) Shared {
  KeyMeta key[3][BKV];    // ring of the other side's rows, two tiles ahead
  int32_t key_lin[3][BKV];
  int32_t key_row[3][BKV];
  float2 key_stats[3][BKV];  // their softmax and delta (dk / dv)
  float key_delta[3][BKV];
  int32_t key_bad[3][2];  // a position without a row in either half
  PlanRow own[BQ];
  int32_t own_row[BQ];
  int32_t range[2];
};

template <typename T, int DP>
struct Block {
  const AttnArgs& a;
  Shared& s;
  float* table;      // [nb^3] fp32
  int16_t* lut;      // [2 reach + 1]
  int head;
  bool lut_linear;
  // set per 64 rows
  bool linear;
  int j0, tiles;

  __device__ __forceinline__ int cells() const { return a.nb * a.nb * a.nb; }

  __device__ __forceinline__ int lin(const PlanRow& r) const {
    return (int)(((unsigned)r.x * a.nb + (unsigned)r.y) * a.nb + (unsigned)r.z);
  }

  __device__ void stage_tables() {
    const T* src = static_cast<const T*>(a.table) + (int64_t)head * cells();
    for (int i = threadIdx.x; i < cells(); i += AT) table[i] = to_f32(src[i]);
    bool same = a.nb == 2 * a.reach + 1;
    for (int i = threadIdx.x; i < 2 * a.reach + 1; i += AT) {
      const int v = max(0, min(a.nb - 1, __ldg(a.lut + i)));
      lut[i] = (int16_t)v;
      same = same && v == i;
    }
    lut_linear = __syncthreads_and(same);
  }

  // The block's rows and the positions their windows cover.
  __device__ void begin(int64_t p0) {
    if (threadIdx.x < 2) s.range[threadIdx.x] = threadIdx.x ? INT_MIN : INT_MAX;
    __syncthreads();
    bool narrow = true;
    if (threadIdx.x < BQ) {
      const int64_t p = p0 + threadIdx.x;
      PlanRow r{};
      r.row = -1;
      if (p < a.n) {
        const int4* src = reinterpret_cast<const int4*>(a.plan + p);
        *reinterpret_cast<int4*>(&r) = __ldg(src);
        *(reinterpret_cast<int4*>(&r) + 1) = __ldg(src + 1);
      }
      if (r.row < 0) {
        r.start = r.end = 0;
      } else {
        atomicMin(&s.range[0], r.start);
        atomicMax(&s.range[1], r.end);
        narrow = r.span <= a.reach;
      }
      s.own[threadIdx.x] = r;
      s.own_row[threadIdx.x] = r.row;
    }
    linear = __syncthreads_and(narrow) && lut_linear;
    j0 = s.range[0];
    tiles = s.range[1] > j0 ? (s.range[1] - j0 + BKV - 1) / BKV : 0;
  }

  template <bool STATS>
  __device__ void stage_meta(int t) {
    const int slot = t % 3;
    const int i = threadIdx.x;
    bool bad = false;
    if (i < BKV) {
      const int j = j0 + t * BKV + i;
      KeyMeta m{0, 0, 0, INT_MAX};
      int32_t row = -1, l = 0;
      float2 x = make_float2(0.f, 0.f);
      float y = 0.f;
      if (j < s.range[1]) {
        const int4* src = reinterpret_cast<const int4*>(a.plan + j);
        const int4 c = __ldg(src);
        row = c.w;
        if (row >= 0) {
          PlanRow r;
          r.x = c.x; r.y = c.y; r.z = c.z;
          l = lin(r);
          m = KeyMeta{c.x, c.y, c.z, j};
          if constexpr (STATS) {
            x = a.stats[head * a.n + j];
            y = a.delta[head * a.n + j];
          }
        }
      }
      bad = row < 0;
      s.key[slot][i] = m;
      s.key_lin[slot][i] = l;
      s.key_row[slot][i] = row;
      if constexpr (STATS) {
        s.key_stats[slot][i] = x;
        s.key_delta[slot][i] = y;
      }
      const unsigned any = __ballot_sync(0xffffffffu, bad);
      if ((i & 31) == 0) s.key_bad[slot][i >> 5] = any != 0;
    }
  }

  // Bucket of (query, key): `query` and `key` as linear coordinates, or by the look-up.
  __device__ __forceinline__ int bucket(int qx, int qy, int qz, int kx, int ky, int kz) const {
    const int R = a.reach;
    const int x = lut[max(-R, min(R, sub_sat(kx, qx))) + R];
    const int y = lut[max(-R, min(R, sub_sat(ky, qy))) + R];
    const int z = lut[max(-R, min(R, sub_sat(kz, qz))) + R];
    return (x * a.nb + y) * a.nb + z;
  }
};

// Buckets of a thread's 32 pairs: rows g and g + 8 of the warp's 16, columns 8 n + 2 (lane % 4) + {0,
// 1}. FLIP: the rows are keys and the columns queries.
template <typename T, int DP, bool FLIP>
__device__ __forceinline__ void buckets(const Block<T, DP>& b, int slot, const PlanRow (&own)[2],
                                        int (&idx)[8][4]) {
  const int c2 = 2 * (threadIdx.x & 3);
  if (b.linear) {
    // inside a window every index is in the table; across windows (masked later) it is clamped
    const unsigned top = (unsigned)b.cells() - 1u;
    const int mid = (int)(top / 2);
    const int l0 = b.lin(own[0]), l1 = b.lin(own[1]);
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const int2 l = *reinterpret_cast<const int2*>(&b.s.key_lin[slot][n * 8 + c2]);
      const int d[4] = {l.x - l0, l.y - l0, l.x - l1, l.y - l1};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        idx[n][e] = (int)min((unsigned)((FLIP ? -d[e] : d[e]) + mid), top);
    }
  } else {
#pragma unroll
    for (int n = 0; n < 8; ++n) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const KeyMeta k = b.s.key[slot][n * 8 + c2 + c];
#pragma unroll
        for (int r = 0; r < 2; ++r)
          idx[n][2 * r + c] =
              FLIP ? b.bucket(k.x, k.y, k.z, own[r].x, own[r].y, own[r].z)
                   : b.bucket(own[r].x, own[r].y, own[r].z, k.x, k.y, k.z);
      }
    }
  }
}

// acc[n] += rows (operand fragments in registers) x tile^T over DP channels: 16 x 64 products.
template <typename T, int DP>
__device__ __forceinline__ void mma_nt(float (&acc)[8][4], const uint32_t (&frag)[DP / 16][4],
                                       uint32_t tile) {
  const int lane = threadIdx.x & 31;
  const uint32_t at = tile + ((lane & 7) + (lane >> 4) * 8) * Tile<DP>::STRIDE +
                      ((lane >> 3) & 1) * 16;
#pragma unroll
  for (int k = 0; k < DP / 16; ++k) {
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      uint32_t b[4];
      ldsm4(at + n * 16 * Tile<DP>::STRIDE + k * 32, b);
      mma<T>(acc[2 * n], frag[k], b[0], b[1]);
      mma<T>(acc[2 * n + 1], frag[k], b[2], b[3]);
    }
  }
}

// out += w (16 x 64, packed as operand fragments) x tile (64 x DP).
template <typename T, int DP>
__device__ __forceinline__ void mma_nn(float (&out)[DP / 8][4], const uint32_t (&w)[4][4],
                                       uint32_t tile) {
  const int lane = threadIdx.x & 31;
  const uint32_t at = tile + ((lane & 7) + ((lane >> 3) & 1) * 8) * Tile<DP>::STRIDE +
                      (lane >> 4) * 16;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
#pragma unroll
    for (int n = 0; n < DP / 16; ++n) {
      uint32_t b[4];
      ldsm4_t(at + k * 16 * Tile<DP>::STRIDE + n * 32, b);
      mma<T>(out[2 * n], w[k], b[0], b[1]);
      mma<T>(out[2 * n + 1], w[k], b[2], b[3]);
    }
  }
}

template <typename T>
__device__ __forceinline__ void pack_rows(const float (&s)[8][4], uint32_t (&w)[4][4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    w[k][0] = pack2<T>(s[2 * k][0], s[2 * k][1]);
    w[k][1] = pack2<T>(s[2 * k][2], s[2 * k][3]);
    w[k][2] = pack2<T>(s[2 * k + 1][0], s[2 * k + 1][1]);
    w[k][3] = pack2<T>(s[2 * k + 1][2], s[2 * k + 1][3]);
  }
}

template <int DP>
__device__ __forceinline__ void load_frags(uint32_t tile, uint32_t (&f)[DP / 16][4]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t at = tile + (warp * 16 + (lane & 15)) * Tile<DP>::STRIDE + (lane >> 4) * 16;
#pragma unroll
  for (int k = 0; k < DP / 16; ++k) ldsm4(at + k * 32, f[k]);
}

template <int W>
__device__ __forceinline__ void zero(float (&x)[W][4]) {
#pragma unroll
  for (int i = 0; i < W; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) x[i][e] = 0.f;
}

// Which of the warp's rows see column `pos`: both bounds of a row's window.
__device__ __forceinline__ bool sees(const PlanRow& r, int pos) {
  return pos >= r.start && pos < r.end;
}

// Positions that any of the warp's 16 rows sees, and those that all of them do.
struct Reach {
  int lo, hi, all_lo, all_hi;
};
__device__ __forceinline__ Reach warp_reach(const PlanRow (&own)[2]) {
  Reach w;
  int lo = INT_MAX, hi = INT_MIN;
#pragma unroll
  for (int r = 0; r < 2; ++r)
    if (own[r].end > own[r].start) {
      lo = min(lo, own[r].start);
      hi = max(hi, own[r].end);
    }
  w.lo = __reduce_min_sync(0xffffffffu, lo);
  w.hi = __reduce_max_sync(0xffffffffu, hi);
  w.all_lo = __reduce_max_sync(0xffffffffu, max(own[0].start, own[1].start));
  w.all_hi = __reduce_min_sync(0xffffffffu, min(own[0].end, own[1].end));
  return w;
}

// A weight of zero does not hide a NaN or an infinity that another window's row brings into a tile,
// and fp16 score gradients can overflow where their sums do not. So rows that come out not finite
// are computed again, one at a time, from their own windows alone.
template <int DP>
__device__ __forceinline__ uint32_t not_finite(const float (&o)[DP / 8][4]) {
  bool bad[2] = {false, false};
#pragma unroll
  for (int n = 0; n < DP / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) bad[e >> 1] = bad[e >> 1] || !(fabsf(o[n][e]) < INFINITY);
  const unsigned b0 = __ballot_sync(0xffffffffu, bad[0]);
  const unsigned b1 = __ballot_sync(0xffffffffu, bad[1]);
  uint32_t rows = 0;  // bit r: row r of the warp's 16
  for (int g = 0; g < 8; ++g) {
    if (b0 >> (4 * g) & 15u) rows |= 1u << g;
    if (b1 >> (4 * g) & 15u) rows |= 1u << (g + 8);
  }
  return rows;
}

template <typename T, typename F>
__device__ __forceinline__ void again(uint32_t rows, int64_t p0, uint8_t* scratch, F&& row) {
  while (rows) {  // the same in all lanes
    const int r = __ffs(rows) - 1;
    rows &= rows - 1;
    __syncwarp();
    row(p0 + r, reinterpret_cast<float*>(scratch));
  }
}

template <typename T>
__device__ __noinline__ void again_forward(AttnArgs a, int64_t p, int h, float* s) {
  row_forward<T>(a, p, h, s);
}
template <typename T>
__device__ __noinline__ void again_dq(AttnArgs a, int64_t p, int h, float* s) {
  row_dq<T, false>(a, p, h, s);
}
template <typename T>
__device__ __noinline__ void again_dkv(AttnArgs a, int64_t p, int h, float* s) {
  row_dkv<T>(a, p, h, s);
}

template <int DP, int TILES>
struct SmemLayout {
  static constexpr int SHARED = TILES * Tile<DP>::BYTES;
  static constexpr int TABLE = (SHARED + (int)sizeof(Shared) + 15) / 16 * 16;
};

__host__ __device__ inline size_t table_bytes(int nb, int words) { return (size_t)nb * nb * nb * 4 * words; }
inline size_t lut_bytes(int reach) { return align_up((size_t)(2 * reach + 1) * 2, 16); }

template <typename T, int DP>
__global__ void __launch_bounds__(AT) attn_tc_kernel(AttnArgs a, int per_block, bool vec) {
  using L = SmemLayout<DP, 5>;
  extern __shared__ __align__(16) uint8_t smem[];
  uint8_t* s_q = smem;
  uint8_t* s_kv = smem + Tile<DP>::BYTES;  // two buffers of k and v
  Shared& sh = *reinterpret_cast<Shared*>(smem + L::SHARED);
  float* table = reinterpret_cast<float*>(smem + L::TABLE);
  const int head = blockIdx.y;
  Block<T, DP> b{a, sh, table,
                 reinterpret_cast<int16_t*>(smem + L::TABLE + table_bytes(a.nb, 1)), head};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c2 = 2 * (lane & 3);
  const T* q = static_cast<const T*>(a.q) + head * a.q_head;
  const T* k = static_cast<const T*>(a.k) + head * a.k_head;
  const T* v = static_cast<const T*>(a.v) + head * a.v_head;
  b.stage_tables();
  const int64_t first = (int64_t)blockIdx.x * per_block;
  for (int64_t t64 = first; t64 < first + per_block && t64 * BQ < a.n; ++t64) {
    b.begin(t64 * BQ);
    load_tile<T, DP>(s_q, q, a.q_row, sh.own_row, a.dim, vec);
    b.template stage_meta<false>(0);
    __syncthreads();
    if (b.tiles > 0) {
      load_tile<T, DP>(s_kv, k, a.k_row, sh.key_row[0], a.dim, vec);
      load_tile<T, DP>(s_kv + Tile<DP>::BYTES, v, a.v_row, sh.key_row[0], a.dim, vec);
    }
    cp_commit();
    b.template stage_meta<false>(1);
    const PlanRow own[2] = {sh.own[warp * 16 + g], sh.own[warp * 16 + g + 8]};
    const Reach w = warp_reach(own);
    uint32_t fq[DP / 16][4];
    float o[DP / 8][4], top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
    zero(o);
    for (int t = 0; t < b.tiles; ++t) {
      __syncthreads();  // the other buffer's readers are done; the next tile's rows are known
      uint8_t* tile = s_kv + (t & 1) * 2 * Tile<DP>::BYTES;
      if (t + 1 < b.tiles) {
        uint8_t* next = s_kv + ((t + 1) & 1) * 2 * Tile<DP>::BYTES;
        load_tile<T, DP>(next, k, a.k_row, sh.key_row[(t + 1) % 3], a.dim, vec);
        load_tile<T, DP>(next + Tile<DP>::BYTES, v, a.v_row, sh.key_row[(t + 1) % 3], a.dim, vec);
        cp_commit();
        cp_wait<1>();
      } else {
        cp_wait<0>();
      }
      __syncthreads();
      if (t + 2 < b.tiles) b.template stage_meta<false>(t + 2);
      if (t == 0) load_frags<DP>(smem_u32(s_q), fq);
      const int p0 = b.j0 + t * BKV;
      if (p0 >= w.hi || p0 + BKV <= w.lo) continue;
      float s[8][4];
      zero(s);
      mma_nt<T, DP>(s, fq, smem_u32(tile));
      const int slot = t % 3;
      int idx[8][4];
      buckets<T, DP, false>(b, slot, own, idx);
      const bool whole = p0 >= w.all_lo && p0 + BKV <= w.all_hi && !sh.key_bad[slot][0] && !sh.key_bad[slot][1];
      float m[2] = {top[0], top[1]};
#pragma unroll
      for (int n = 0; n < 8; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = fmaf(s[n][e], a.scale, table[idx[n][e]]);
        if (!whole) {
          const int pos0 = sh.key[slot][n * 8 + c2].pos, pos1 = sh.key[slot][n * 8 + c2 + 1].pos;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!sees(own[e >> 1], e & 1 ? pos1 : pos0)) s[n][e] = -INFINITY;
        }
        m[0] = fmaxf(m[0], fmaxf(s[n][0], s[n][1]));
        m[1] = fmaxf(m[1], fmaxf(s[n][2], s[n][3]));
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        m[r] = fmaxf(m[r], __shfl_xor_sync(0xffffffffu, m[r], 1));
        m[r] = fmaxf(m[r], __shfl_xor_sync(0xffffffffu, m[r], 2));
        const float base = m[r] == -INFINITY ? 0.f : m[r];
        const float keep = exp2_fast((top[r] - base) * LOG2E);
        top[r] = m[r];
        sum[r] *= keep;
#pragma unroll
        for (int n = 0; n < 8; ++n) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            // subtracted before it is scaled: the type's lowest value times log2(e) overflows
            const float e = exp2_fast((s[n][2 * r + c] - base) * LOG2E);
            s[n][2 * r + c] = e;
            sum[r] += e;
          }
        }
#pragma unroll
        for (int n = 0; n < DP / 8; ++n) {
          o[n][2 * r] *= keep;
          o[n][2 * r + 1] *= keep;
        }
      }
      uint32_t p[4][4];
      pack_rows<T>(s, p);
      mma_nn<T, DP>(o, p, smem_u32(tile + Tile<DP>::BYTES));
    }
    float inv[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
      sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
      const float2 st = row_stats(top[r], sum[r]);
      inv[r] = st.y;
      if (a.stats && c2 == 0 && own[r].row >= 0)
        a.stats[head * a.n + t64 * BQ + warp * 16 + g + 8 * r] = st;
    }
    __syncthreads();
    store_rows<T, DP>(s_q, o, inv[0], inv[1], sh.own_row, static_cast<T*>(a.out), a.heads, head,
                      a.dim, vec);
    again<T>(not_finite<DP>(o), t64 * BQ + warp * 16, s_q + warp * 16 * Tile<DP>::STRIDE,
             [&](int64_t p, float* f) { if (p < a.n) again_forward<T>(a, p, head, f); });
    __syncthreads();
  }
}

// delta_i = dout_i . o_i by position, and the largest |dout_i|^2 and |v_j|^2 of a head (bits order
// like the values of these non-negative numbers, a NaN above everything).
template <typename T>
__global__ void __launch_bounds__(256) attn_prepare_kernel(AttnArgs a) {
  __shared__ unsigned s_top[2];
  const int h = blockIdx.y;
  if (threadIdx.x < 2) s_top[threadIdx.x] = 0u;
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  unsigned g_top = 0u, v_top = 0u;
  for (int64_t p = (int64_t)blockIdx.x * 8 + warp; p < a.n; p += (int64_t)gridDim.x * 8) {
    const int32_t row = __ldg(&a.plan[p].row);
    if (row < 0) continue;
    const int64_t at = ((int64_t)row * a.heads + h) * a.dim;
    const T* g = static_cast<const T*>(a.dout) + at;
    const T* o = static_cast<const T*>(a.o) + at;
    const T* v = static_cast<const T*>(a.v) + row * a.v_row + h * a.v_head;
    float g2 = 0.f, v2 = 0.f, d = 0.f;
    for (int c = lane; c < a.dim; c += 32) {
      const float x = to_f32(g[c]), y = to_f32(v[c]);
      g2 = fmaf(x, x, g2);
      v2 = fmaf(y, y, v2);
      d = fmaf(x, to_f32(o[c]), d);
    }
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) {
      g2 += __shfl_xor_sync(0xffffffffu, g2, s);
      v2 += __shfl_xor_sync(0xffffffffu, v2, s);
      d += __shfl_xor_sync(0xffffffffu, d, s);
    }
    if (lane == 0) a.delta[h * a.n + p] = d;
    g_top = max(g_top, __float_as_uint(g2) & 0x7fffffffu);
    v_top = max(v_top, __float_as_uint(v2) & 0x7fffffffu);
  }
  if (lane == 0) {
    atomicMax(&s_top[0], g_top);
    atomicMax(&s_top[1], v_top);
  }
  __syncthreads();
  if (threadIdx.x < 2 && a.dtable) atomicMax(a.norms + 2 * h + threadIdx.x, s_top[threadIdx.x]);
}

// A block's share of the table's gradient sums in two 32-bit words a bucket: whole units, and the
// rest in 2^-12 of one. |dS| over a row sums to at most 2 max|dout| max|v| (attention.h), so
// `rows` of them stay below 2^30 units, and 2^19 remainders of at most half a unit fit the other
// word (a block meets fewer pairs of one bucket: it empties the words every 2^19 / 64 positions).
__device__ __forceinline__ int block_exponent(const AttnArgs& a, int head, int rows) {
  const float g2 = __uint_as_float(a.norms[2 * head]), v2 = __uint_as_float(a.norms[2 * head + 1]);
  const double bound = 2.0 * sqrt((double)g2) * sqrt((double)v2) * (double)rows;
  if (!(bound < 1e300)) return INT_MAX;
  if (bound == 0.0) return 0;
  int e;
  frexp(bound, &e);
  return max(-120, min(100, 29 - e));  // a factor of two left for the products' rounding
}

// dq and the table's gradient.
template <typename T, int DP, bool TABLE>
__global__ void __launch_bounds__(AT) attn_dq_tc_kernel(AttnArgs a, int per_block, bool vec) {
  using L = SmemLayout<DP, 6>;
  extern __shared__ __align__(16) uint8_t smem[];
  uint8_t* s_q = smem;
  uint8_t* s_g = smem + Tile<DP>::BYTES;
  uint8_t* s_kv = smem + 2 * Tile<DP>::BYTES;
  Shared& sh = *reinterpret_cast<Shared*>(smem + L::SHARED);
  float* table = reinterpret_cast<float*>(smem + L::TABLE);
  const int cells = a.nb * a.nb * a.nb;
  int* s_hi = reinterpret_cast<int*>(table + cells);
  int* s_lo = s_hi + cells;
  const int head = blockIdx.y;
  Block<T, DP> b{a, sh, table,
                 reinterpret_cast<int16_t*>(smem + L::TABLE + table_bytes(a.nb, TABLE ? 3 : 1)),
                 head};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c2 = 2 * (lane & 3);
  const T* q = static_cast<const T*>(a.q) + head * a.q_head;
  const T* k = static_cast<const T*>(a.k) + head * a.k_head;
  const T* v = static_cast<const T*>(a.v) + head * a.v_head;
  const T* dout = static_cast<const T*>(a.dout) + (int64_t)head * a.dim;
  const int64_t g_row = (int64_t)a.heads * a.dim;
  const int exponent = TABLE ? block_exponent(a, head, per_block * BQ) : INT_MAX;
  const float unit = exponent == INT_MAX ? 0.f : ldexpf(1.f, exponent);
  if constexpr (TABLE) {
    for (int i = threadIdx.x; i < 2 * cells; i += AT) s_hi[i] = 0;
  }
  b.stage_tables();
  auto flush = [&] {
    if constexpr (TABLE) {
      __syncthreads();
      for (int i = threadIdx.x; i < cells; i += AT) {
        const long long add = ((long long)s_hi[i] << 12) + s_lo[i];
        if (add != 0)
          atomicAdd(a.dtable + (int64_t)head * cells + i, (unsigned long long)add);
        s_hi[i] = 0;
        s_lo[i] = 0;
      }
      __syncthreads();
    }
  };
  int since = 0;  // tiles of pairs since the words were emptied
  const int64_t first = (int64_t)blockIdx.x * per_block;
  for (int64_t t64 = first; t64 < first + per_block && t64 * BQ < a.n; ++t64) {
    b.begin(t64 * BQ);
    load_tile<T, DP>(s_q, q, a.q_row, sh.own_row, a.dim, vec);
    load_tile<T, DP>(s_g, dout, g_row, sh.own_row, a.dim, vec);
    b.template stage_meta<false>(0);
    __syncthreads();
    if (b.tiles > 0) {
      load_tile<T, DP>(s_kv, k, a.k_row, sh.key_row[0], a.dim, vec);
      load_tile<T, DP>(s_kv + Tile<DP>::BYTES, v, a.v_row, sh.key_row[0], a.dim, vec);
    }
    cp_commit();
    b.template stage_meta<false>(1);
    const PlanRow own[2] = {sh.own[warp * 16 + g], sh.own[warp * 16 + g + 8]};
    const Reach w = warp_reach(own);
    float2 stats[2];
    float delta[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int64_t p = t64 * BQ + warp * 16 + g + 8 * r;
      stats[r] = own[r].row >= 0 ? a.stats[head * a.n + p] : make_float2(0.f, 0.f);
      delta[r] = own[r].row >= 0 ? a.delta[head * a.n + p] : 0.f;
    }
    float dq[DP / 8][4];
    zero(dq);
    for (int t = 0; t < b.tiles; ++t) {
      __syncthreads();
      uint8_t* tile = s_kv + (t & 1) * 2 * Tile<DP>::BYTES;
      if (t + 1 < b.tiles) {
        uint8_t* next = s_kv + ((t + 1) & 1) * 2 * Tile<DP>::BYTES;
        load_tile<T, DP>(next, k, a.k_row, sh.key_row[(t + 1) % 3], a.dim, vec);
        load_tile<T, DP>(next + Tile<DP>::BYTES, v, a.v_row, sh.key_row[(t + 1) % 3], a.dim, vec);
        cp_commit();
        cp_wait<1>();
      } else {
        cp_wait<0>();
      }
      __syncthreads();
      if (t + 2 < b.tiles) b.template stage_meta<false>(t + 2);
      if constexpr (TABLE) {
        if (++since > (1 << 19) / BKV / BQ) {  // 64 x 64 pairs a tile
          flush();
          since = 1;
        }
      }
      const int p0 = b.j0 + t * BKV;
      if (p0 >= w.hi || p0 + BKV <= w.lo) continue;
      float s[8][4], dp[8][4];
      zero(s);
      zero(dp);
      {
        uint32_t f[DP / 16][4];
        load_frags<DP>(smem_u32(s_q), f);
        mma_nt<T, DP>(s, f, smem_u32(tile));
        load_frags<DP>(smem_u32(s_g), f);
        mma_nt<T, DP>(dp, f, smem_u32(tile + Tile<DP>::BYTES));
      }
      const int slot = t % 3;
      int idx[8][4];
      buckets<T, DP, false>(b, slot, own, idx);
      const bool whole = p0 >= w.all_lo && p0 + BKV <= w.all_hi && !sh.key_bad[slot][0] && !sh.key_bad[slot][1];
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const int pos0 = sh.key[slot][n * 8 + c2].pos, pos1 = sh.key[slot][n * 8 + c2 + 1].pos;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = e >> 1;
          const float x = fmaf(s[n][e], a.scale, table[idx[n][e]]);
          float ds = exp2_fast((x - stats[r].x) * LOG2E) * stats[r].y * (dp[n][e] - delta[r]);
          const bool in = whole || sees(own[r], e & 1 ? pos1 : pos0);
          if (!in) ds = 0.f;
          s[n][e] = ds;
          if constexpr (TABLE) {
            if (in && exponent != INT_MAX) {
              if (fabsf(ds) < INFINITY) {
                const float f = ds * unit;
                const float whole_units = rintf(f);
                atomicAdd(s_hi + idx[n][e], __float2int_rn(whole_units));
                atomicAdd(s_lo + idx[n][e], __float2int_rn((f - whole_units) * 4096.f));
              } else {
                atomicMax(a.norms + 2 * head, 0x7fffffffu);  // the head's table gradient is NaN
              }
            }
          }
        }
      }
      uint32_t p[4][4];
      pack_rows<T>(s, p);
      mma_nn<T, DP>(dq, p, smem_u32(tile));
    }
    __syncthreads();
    store_rows<T, DP>(s_q, dq, a.scale, a.scale, sh.own_row, static_cast<T*>(a.dq), a.heads, head,
                      a.dim, vec);
    again<T>(not_finite<DP>(dq), t64 * BQ + warp * 16, s_q + warp * 16 * Tile<DP>::STRIDE,
             [&](int64_t p, float* f) { if (p < a.n) again_dq<T>(a, p, head, f); });
    __syncthreads();
  }
  flush();
}

// dk and dv: the block's rows are keys, the tiles queries.
template <typename T, int DP>
__global__ void __launch_bounds__(AT) attn_dkv_tc_kernel(AttnArgs a, int per_block, bool vec) {
  using L = SmemLayout<DP, 6>;
  extern __shared__ __align__(16) uint8_t smem[];
  uint8_t* s_k = smem;
  uint8_t* s_v = smem + Tile<DP>::BYTES;
  uint8_t* s_qg = smem + 2 * Tile<DP>::BYTES;
  Shared& sh = *reinterpret_cast<Shared*>(smem + L::SHARED);
  float* table = reinterpret_cast<float*>(smem + L::TABLE);
  const int head = blockIdx.y;
  Block<T, DP> b{a, sh, table,
                 reinterpret_cast<int16_t*>(smem + L::TABLE + table_bytes(a.nb, 1)), head};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c2 = 2 * (lane & 3);
  const T* q = static_cast<const T*>(a.q) + head * a.q_head;
  const T* k = static_cast<const T*>(a.k) + head * a.k_head;
  const T* v = static_cast<const T*>(a.v) + head * a.v_head;
  const T* dout = static_cast<const T*>(a.dout) + (int64_t)head * a.dim;
  const int64_t g_row = (int64_t)a.heads * a.dim;
  b.stage_tables();
  const int64_t first = (int64_t)blockIdx.x * per_block;
  for (int64_t t64 = first; t64 < first + per_block && t64 * BQ < a.n; ++t64) {
    b.begin(t64 * BQ);
    load_tile<T, DP>(s_k, k, a.k_row, sh.own_row, a.dim, vec);
    load_tile<T, DP>(s_v, v, a.v_row, sh.own_row, a.dim, vec);
    b.template stage_meta<true>(0);
    __syncthreads();
    if (b.tiles > 0) {
      load_tile<T, DP>(s_qg, q, a.q_row, sh.key_row[0], a.dim, vec);
      load_tile<T, DP>(s_qg + Tile<DP>::BYTES, dout, g_row, sh.key_row[0], a.dim, vec);
    }
    cp_commit();
    b.template stage_meta<true>(1);
    const PlanRow own[2] = {sh.own[warp * 16 + g], sh.own[warp * 16 + g + 8]};
    const Reach w = warp_reach(own);
    float dk[DP / 8][4], dv[DP / 8][4];
    zero(dk);
    zero(dv);
    for (int t = 0; t < b.tiles; ++t) {
      __syncthreads();
      uint8_t* tile = s_qg + (t & 1) * 2 * Tile<DP>::BYTES;
      if (t + 1 < b.tiles) {
        uint8_t* next = s_qg + ((t + 1) & 1) * 2 * Tile<DP>::BYTES;
        load_tile<T, DP>(next, q, a.q_row, sh.key_row[(t + 1) % 3], a.dim, vec);
        load_tile<T, DP>(next + Tile<DP>::BYTES, dout, g_row, sh.key_row[(t + 1) % 3], a.dim, vec);
        cp_commit();
        cp_wait<1>();
      } else {
        cp_wait<0>();
      }
      __syncthreads();
      if (t + 2 < b.tiles) b.template stage_meta<true>(t + 2);
      const int p0 = b.j0 + t * BKV;
      if (p0 >= w.hi || p0 + BKV <= w.lo) continue;
      const int slot = t % 3;
      float s[8][4], dp[8][4];
      zero(s);
      {
        uint32_t f[DP / 16][4];
        load_frags<DP>(smem_u32(s_k), f);
        mma_nt<T, DP>(s, f, smem_u32(tile));
      }
      {
        int idx[8][4];
        buckets<T, DP, true>(b, slot, own, idx);
        const bool whole = p0 >= w.all_lo && p0 + BKV <= w.all_hi && !sh.key_bad[slot][0] && !sh.key_bad[slot][1];
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          const int pos0 = sh.key[slot][n * 8 + c2].pos, pos1 = sh.key[slot][n * 8 + c2 + 1].pos;
          // {maximum, 1 / sum} of the two queries
          const float4 st = *reinterpret_cast<const float4*>(&sh.key_stats[slot][n * 8 + c2]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = fmaf(s[n][e], a.scale, table[idx[n][e]]);
            s[n][e] = exp2_fast((x - (e & 1 ? st.z : st.x)) * LOG2E) * (e & 1 ? st.w : st.y);
            if (!whole && !sees(own[e >> 1], e & 1 ? pos1 : pos0)) s[n][e] = 0.f;
          }
        }
      }
      {
        uint32_t p[4][4];
        pack_rows<T>(s, p);
        mma_nn<T, DP>(dv, p, smem_u32(tile + Tile<DP>::BYTES));
      }
      zero(dp);
      {
        uint32_t f[DP / 16][4];
        load_frags<DP>(smem_u32(s_v), f);
        mma_nt<T, DP>(dp, f, smem_u32(tile + Tile<DP>::BYTES));
      }
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const float2 delta = *reinterpret_cast<const float2*>(&sh.key_delta[slot][n * 8 + c2]);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          // a weight of zero may stand for a row of another window, which may hold anything
          dp[n][e] = s[n][e] == 0.f ? 0.f : s[n][e] * (dp[n][e] - (e & 1 ? delta.y : delta.x));
      }
      uint32_t p[4][4];
      pack_rows<T>(dp, p);
      mma_nn<T, DP>(dk, p, smem_u32(tile));
    }
    __syncthreads();
    store_rows<T, DP>(s_k, dk, a.scale, a.scale, sh.own_row, static_cast<T*>(a.dk), a.heads, head,
                      a.dim, vec);
    store_rows<T, DP>(s_v, dv, 1.f, 1.f, sh.own_row, static_cast<T*>(a.dv), a.heads, head, a.dim,
                      vec);
    again<T>(not_finite<DP>(dk) | not_finite<DP>(dv), t64 * BQ + warp * 16,
             s_k + warp * 16 * Tile<DP>::STRIDE,
             [&](int64_t p, float* f) { if (p < a.n) again_dkv<T>(a, p, head, f); });
    __syncthreads();
  }
}

template <typename T>
__global__ void __launch_bounds__(256)
    dtable_tc_finish_kernel(AttnArgs a, int rows, T* __restrict__ out) {
  const int cells = a.nb * a.nb * a.nb;
  const int h = blockIdx.y;
  const int exponent = block_exponent(a, h, rows);
  for (int b = blockIdx.x * 256 + threadIdx.x; b < cells; b += gridDim.x * 256) {
    const int64_t at = (int64_t)h * cells + b;
    const double v = exponent == INT_MAX
                         ? __longlong_as_double(0x7ff8000000000000ll)  // the inputs were not finite
                         : ldexp((double)(long long)a.dtable[at], -exponent - 12);
    out[at] = from_f32<T>((float)v);
  }
}

bool wide(const void* p, int64_t row, int64_t head) {
  return p == nullptr || (aligned16(p) && row % 8 == 0 && head % 8 == 0);
}

// Whether rows move in 16-byte pieces: tensors that are sliced off a boundary or have odd heads go
// element by element.
bool wide_rows(const AttnArgs& a) {
  const int64_t head = a.dim, row = (int64_t)a.heads * a.dim;
  return a.dim % 8 == 0 && wide(a.q, a.q_row, a.q_head) && wide(a.k, a.k_row, a.k_head) &&
         wide(a.v, a.v_row, a.v_head) && wide(a.out, row, head) && wide(a.dout, row, head) &&
         wide(a.dq, row, head) && wide(a.dk, row, head) && wide(a.dv, row, head);
}

// 64-row tiles of one head that a block takes in turn, so that it stages the table (and adds up its
// gradient) once: as many as still leave `waves` blocks for each of an SM's places.
int tiles_per_block(const AttnArgs& a, int waves) {
  const int64_t tiles = (a.n + BQ - 1) / BQ;
  const int64_t per = tiles * a.heads / ((int64_t)num_sms() * waves);
  return (int)(per < 1 ? 1 : (per > 16 ? 16 : per));
}

template <typename K>
int allow_smem(K kernel, size_t bytes) {
  SV_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   (int)bytes));
  return SV_OK;
}

template <int DP, int TILES>
size_t smem_bytes(const AttnArgs& a, int words) {
  return SmemLayout<DP, TILES>::TABLE + table_bytes(a.nb, words) + lut_bytes(a.reach);
}

template <typename T, int DP>
int forward(const AttnArgs& a, cudaStream_t s) {
  const size_t bytes = smem_bytes<DP, 5>(a, 1);
  const int rc = allow_smem(attn_tc_kernel<T, DP>, bytes);
  if (rc != SV_OK) return rc;
  const int per = tiles_per_block(a, 12);
  const int64_t blocks = ((a.n + BQ - 1) / BQ + per - 1) / per;
  attn_tc_kernel<T, DP><<<dim3((unsigned)blocks, a.heads), AT, bytes, s>>>(a, per, wide_rows(a));
  SV_LAUNCH_CHECK();
  return SV_OK;
}

template <typename T, int DP>
int backward(const AttnArgs& a, void* dtable, cudaStream_t s) {
  const unsigned prep = (unsigned)((a.n + 63) / 64 < 512 ? (a.n + 63) / 64 : 512);
  attn_prepare_kernel<T><<<dim3(prep, a.heads), 256, 0, s>>>(a);
  SV_LAUNCH_CHECK();
  const bool vec = wide_rows(a);
  const int per = tiles_per_block(a, 6);
  const dim3 grid((unsigned)(((a.n + BQ - 1) / BQ + per - 1) / per), a.heads);
  size_t bytes = smem_bytes<DP, 6>(a, dtable ? 3 : 1);
  int rc = dtable ? allow_smem(attn_dq_tc_kernel<T, DP, true>, bytes)
                  : allow_smem(attn_dq_tc_kernel<T, DP, false>, bytes);
  if (rc != SV_OK) return rc;
  if (dtable)
    attn_dq_tc_kernel<T, DP, true><<<grid, AT, bytes, s>>>(a, per, vec);
  else
    attn_dq_tc_kernel<T, DP, false><<<grid, AT, bytes, s>>>(a, per, vec);
  SV_LAUNCH_CHECK();
  if (dtable) {
    const unsigned blocks = (unsigned)((a.nb * a.nb * a.nb + 255) / 256);
    dtable_tc_finish_kernel<T><<<dim3(blocks, a.heads), 256, 0, s>>>(a, per * BQ,
                                                                     static_cast<T*>(dtable));
    SV_LAUNCH_CHECK();
  }
  bytes = smem_bytes<DP, 6>(a, 1);
  rc = allow_smem(attn_dkv_tc_kernel<T, DP>, bytes);
  if (rc != SV_OK) return rc;
  attn_dkv_tc_kernel<T, DP><<<grid, AT, bytes, s>>>(a, per, vec);
  SV_LAUNCH_CHECK();
  return SV_OK;
}

template <typename T>
int forward_typed(const AttnArgs& a, cudaStream_t s) {
  if (a.dim <= 32) return forward<T, 32>(a, s);
  if (a.dim <= 64) return forward<T, 64>(a, s);
  return forward<T, 128>(a, s);
}

template <typename T>
int backward_typed(const AttnArgs& a, void* dtable, cudaStream_t s) {
  if (a.dim <= 32) return backward<T, 32>(a, dtable, s);
  if (a.dim <= 64) return backward<T, 64>(a, dtable, s);
  return backward<T, 128>(a, dtable, s);
}

}  // namespace

int attention_tc_forward(const AttnArgs& a, bool bf16, cudaStream_t s) {
  return bf16 ? forward_typed<__nv_bfloat16>(a, s) : forward_typed<__half>(a, s);
}

int attention_tc_backward(const AttnArgs& a, bool bf16, void* dtable, cudaStream_t s) {
  return bf16 ? backward_typed<__nv_bfloat16>(a, dtable, s) : backward_typed<__half>(a, dtable, s);
}

}  // namespace sv
