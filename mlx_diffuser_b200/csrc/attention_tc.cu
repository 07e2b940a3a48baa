// Windowed attention with a learned relative position bias in fp16 / bf16, on the tensor cores.
//
// The formulas are attention.cu's. A block takes up to 128 rows (queries; 64 in the backward pass, keys
// for dk and dv) of one head out of the plan's list, four warps of 32 or 16, and walks the positions
// that any of their windows covers in tiles of 32: rows of several small windows share a tile, and a
// warp skips the tiles that none of its own rows' windows reach. Scores stay in registers from the
// product to the softmax to the next product (the accumulator's layout is the operand's), so the
// running maximum and sum are the only state. The gathered rows arrive by cp.async, one or two tiles
// ahead.
//
// Products are warp-level mma.sync: a window of a surface holds 100-300 rows, so a tile's two
// products are a few hundred cycles, while each of its scores needs an exponential and a table
// look-up of its own. The register layout makes the bias and the softmax free of shared-memory round
// trips. A form with the scores in TMEM (tcgen05, four row warps a block) was slower: 332 against
// 279 us forward, 398 + 305 against 308 + 276 us backward, its warps waiting for each other between
// tiles that short; it won only for windows of 4,096 rows (590 against 678 us, before that walk was
// split).
//
// Latency bounds these kernels: with the 168 registers of a thread three blocks fit an SM, 2.8 warps a
// scheduler that issue an instruction every 2.6 cycles (a quarter of the stalls at the tile's barrier,
// a fifth fixed latencies). bf16, 64 channels:
//   forward   40,662 x 12 heads, windows of 8^3 (95 M pairs): 239 us; 20,331 x 16 (63 M): 225 us with
//             what training adds, 41 MB of rests and a second product
//   backward  20,331 x 16: delta 26 us, dk and dv with each bucket's largest term 371 us, dq and the
//             table's gradient 328 us; 282 and 226 where no table gradient is wanted (fp16, whose score
//             gradients are raised row by row, 306 and 246)
//   forward   8,192 x 6 x 128 in two windows (201 M pairs), three parts: 495 us and 28 us to join
// Two row parts a warp in the dk / dv pass halve its fragment loads but leave two blocks an SM: 328 us
// where one took 268.
//
// The bucket of a pair: where the table is one entry per offset (the look-up is the identity) and
// the windows are no wider than its reach, it is linear in the coordinates and costs a subtraction;
// otherwise three look-ups.
//
// Weights and score gradients are rounded to the feature type as operands of the second products
// (half a step each, like the stored results: 0.0022 against the 0.0017 of the result's own rounding over
// the outputs of 40,662 x 12 x 64 bf16); the softmax sums and the table's gradient use them unrounded.
// The forward pass of training adds a second product for what rounding the weights leaves
// out: delta, which dS is a small difference with, comes from its output (dq and dk off by 1.42 times
// the plain form's error instead of up to 1.55, for 22 us of 225 at 20,331 x 16 x 64).
//
// In fp16 these operands, and what rounding the output leaves out, are raised by powers of two that the
// result's factor takes back: below 2^-14 a half has no 11 bits, below 2^-25 it is zero, and the weights
// of long windows and the score gradients of a mean loss lie there (unraised, dq of 4,096 rows was off by
// 8 times the result's rounding at output gradients of 1e-3). Weights by fixed powers, score gradients by
// one for each row, lowered when a larger one comes.
#include <limits.h>

#include <algorithm>
#include <type_traits>

#include "attention.h"

namespace sv {
namespace {

// CTAs an SM over a call's course (three run at a time). 5: 265 us forward and 308 + 289 us backward; 9:
// 238 and 284 + 266; 16: 233 and 288 + 269, whose staging of the table counts in the backward pass
// (before that one's units for each bucket).
constexpr int WAVES = 9;
constexpr int AT = 128;   // threads: four warps of 16 rows, or of 32
constexpr int KB = 32;   // positions of a tile
// Rows of a block in the forward pass: two 16-row parts a warp, whose products share the tile's
// fragments (8,192 x 6 x 128 fp16: 678 us with one, 651 with two).
constexpr int FORWARD_ROWS = 128;

template <typename T>
constexpr bool IS_HALF = std::is_same<T, __half>::value;
// The dk / dv pass's weights, at most 1, as operands: raised by this.
template <typename T>
constexpr float RAISE = IS_HALF<T> ? 32768.f : 1.f;

// Tiles hold DP channels a row (the head's, padded with zeros) at a stride that is an odd multiple
// of 16 bytes, so the 8 rows of a matrix fragment fall into different banks.
template <int DP>
constexpr int STRIDE = DP * 2 + 16;

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

// What pack2 left out of two numbers, rounded in turn.
template <typename T>
__device__ __forceinline__ uint32_t rest2(uint32_t packed, float lo, float hi) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    return pack2<T>(lo - __uint_as_float(packed << 16), hi - __uint_as_float(packed & 0xffff0000u));
  } else {
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&packed));
    return pack2<T>(lo - v.x, hi - v.y);
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

// max that keeps a NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}

// R gathered rows of one head into a tile; rows of -1 and channels past `dim` become zeros.
template <typename T, int DP, int R>
__device__ __forceinline__ void load_tile(uint8_t* tile, const T* base, int row_stride,
                                          const int32_t* rows, int dim, bool vec) {
  constexpr int CH = DP / 8;  // 16-byte chunks of a row; a thread copies the same one of every row
  static_assert(AT % CH == 0 && R * CH % AT == 0, "whole rounds");
  if (vec) {
    const int col = threadIdx.x % CH, r0 = threadIdx.x / CH;
    const uint32_t at = smem_u32(tile) + r0 * STRIDE<DP> + col * 16;
    const bool in_row = col * 8 < dim;
    const T* from = base + (in_row ? col * 8 : 0);
#pragma unroll
    for (int i = 0; i < R * CH / AT; ++i) {
      const int32_t row = rows[r0 + i * (AT / CH)];
      cp_async_16(at + i * (AT / CH) * STRIDE<DP>, from + (int64_t)max(row, 0) * row_stride,
                  row >= 0 && in_row ? 16u : 0u);
    }
  } else {
    for (int c = threadIdx.x; c < R * DP; c += AT) {
      const int r = c / DP, col = c % DP;
      const int32_t row = rows[r];
      T v = from_f32<T>(0.f);
      if (row >= 0 && col < dim) v = base[(int64_t)row * row_stride + col];
      *reinterpret_cast<T*>(tile + r * STRIDE<DP> + col * 2) = v;
    }
  }
}

// A 16-row accumulator into the warp's own part of a tile (`mine`), rounded to T, or with REST what
// that rounding leaves out.
template <typename T, int DP, bool REST = false>
__device__ __forceinline__ void put_rows(uint8_t* mine, const float (&o)[DP / 8][4], float s0,
                                         float s1) {
  const int lane = threadIdx.x & 31;
  const int g = lane >> 2, c2 = 2 * (lane & 3);
  auto pack = [](float x, float y) {
    return REST ? pack2<T>(rest_of<T>(x), rest_of<T>(y)) : pack2<T>(x, y);
  };
#pragma unroll
  for (int n = 0; n < DP / 8; ++n) {
    *reinterpret_cast<uint32_t*>(mine + g * STRIDE<DP> + (n * 8 + c2) * 2) =
        pack(o[n][0] * s0, o[n][1] * s0);
    *reinterpret_cast<uint32_t*>(mine + (g + 8) * STRIDE<DP> + (n * 8 + c2) * 2) =
        pack(o[n][2] * s1, o[n][3] * s1);
  }
}

// Those 16 rows to the feature rows `rows`, in 16-byte stores.
template <typename T, int DP>
__device__ __forceinline__ void send_rows(const uint8_t* mine, const int32_t* rows, T* out,
                                          int heads, int head, int dim, bool vec) {
  constexpr int CH = DP / 8;
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 16 * CH / 32; ++i) {
    const int c = lane + 32 * i;
    const int r = c / CH, col = c % CH;
    const int32_t row = rows[r];
    if (row < 0) continue;
    T* dst = out + ((int64_t)row * heads + head) * dim + col * 8;
    const uint4 v = *reinterpret_cast<const uint4*>(mine + r * STRIDE<DP> + col * 16);
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

template <typename T, int DP>
__device__ __forceinline__ void store_rows(uint8_t* mine, const float (&o)[DP / 8][4], float s0,
                                           float s1, const int32_t* rows, T* out, int heads,
                                           int head, int dim, bool vec) {
  __syncwarp();
  put_rows<T, DP>(mine, o, s0, s1);
  __syncwarp();
  send_rows<T, DP>(mine, rows, out, heads, head, dim, vec);
}

struct KeyMeta {
  int32_t x, y, z, row;  // row -1: no row
};

constexpr int SLOTS = 4;  // tiles whose rows are known: the one worked on and three ahead

// What every kernel here keeps in shared memory besides its tiles; BQ rows of the block's own.
template <int BQ>
struct alignas(16) Shared {
  KeyMeta key[SLOTS][KB];       // the other side's rows
  int2 key_lin[SLOTS][KB];      // their linear coordinates (Block::lin)
  int32_t key_row[SLOTS][KB];
  float2 key_stats[SLOTS][KB];  // their softmax, the weights raised by RAISE, and delta (dk / dv)
  float key_delta[SLOTS][KB];
  int32_t key_bad[SLOTS];       // whether a position has no row
  PlanRow own[BQ];
  int32_t own_row[BQ];
  int32_t range[2];
};

// How a pair's bucket is found. LINEAR: the look-up is the identity and the windows are within the
// table's reach, so the bucket is a difference of linear coordinates. JOINT: within the reach, and
// the look-ups of x and y are joined in one table of all their offsets. GENERAL: any. All indexes are
// kept as byte offsets.
enum { GENERAL = 0, JOINT = 1, LINEAR = 2 };
constexpr int JOINT_MAX = 4096;

__device__ __forceinline__ float lds_f32(uint32_t at) {
  float v;
  asm("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at));
  return v;
}
__device__ __forceinline__ uint32_t lds_u8(uint32_t at) {
  uint32_t v;
  asm("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(at));
  return v;
}
__device__ __forceinline__ uint32_t lds_u16(uint32_t at) {
  uint16_t v;
  asm("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at));
  return v;
}

template <typename T, int BQ>
struct Block {
  const AttnArgs& a;
  Shared<BQ>& s;
  float* table;      // [nb^3] times log2(e)
  uint16_t* lut;     // [2 reach + 1], times 4
  uint16_t* joint;   // [(2 reach + 1)^2]: x and y buckets' offset in the table, or null
  int head;
  bool identity;
  // set per BQ rows
  int mode;
  int j0, tiles;

  __device__ __forceinline__ int cells() const { return a.nb * a.nb * a.nb; }
  __device__ __forceinline__ int width() const { return 2 * a.reach + 1; }

  // LINEAR: 4 ((x nb + y) nb + z); JOINT: 2 (x width + y) and 2 z. Wrap-around is harmless: only
  // differences inside a window are used.
  __device__ __forceinline__ int2 lin(int x, int y, int z) const {
    if (mode == LINEAR)
      return make_int2((int)((((unsigned)x * a.nb + (unsigned)y) * a.nb + (unsigned)z) * 4u), 0);
    return make_int2((int)(((unsigned)x * width() + (unsigned)y) * 2u), (int)((unsigned)z * 2u));
  }

  __device__ void stage_tables() {
    const T* src = static_cast<const T*>(a.table) + (int64_t)head * cells();
#pragma unroll 8
    for (int i = threadIdx.x; i < cells(); i += AT) table[i] = times_log2e(to_f32(src[i]));
    bool same = a.nb == width();
    for (int i = threadIdx.x; i < width(); i += AT) {
      const int v = max(0, min(a.nb - 1, __ldg(a.lut + i)));
      lut[i] = (uint16_t)(4 * v);
      same = same && v == i;
    }
    identity = __syncthreads_and(same);
    if (!identity && joint != nullptr)
      for (int i = threadIdx.x; i < width() * width(); i += AT)
        joint[i] = (uint16_t)((lut[i / width()] * a.nb + lut[i % width()]) * a.nb);
  }

  // The block's rows, `count` from position p0 on, and the positions their windows cover, of which part
  // `part` of `parts` is walked. STAND_IN: rows behind the last see what the first one does, so that
  // they cost no mask; nothing of theirs is stored. Without it they see nothing, as the backward
  // pass needs them to, which takes sums and maxima over all of a warp's pairs.
  // LONE: rows that see one position see nothing (dq).
  template <bool STAND_IN, bool LONE = false>
  __device__ void begin(int p0, int count, int part = 0, int parts = 1) {
    if (threadIdx.x < 2) s.range[threadIdx.x] = threadIdx.x ? INT_MIN : INT_MAX;
    __syncthreads();
    bool narrow = true;
    if (threadIdx.x < BQ) {
      const bool in = (int)threadIdx.x < count;
      PlanRow r = plan_at(a.plan, in ? p0 + threadIdx.x : p0);
      if (r.row < 0 || (LONE && lone(r))) {
        r.start = r.end = 0;
        if (!in) r.row = -1;
      } else {
        narrow = r.span <= a.reach;
        if (in) {
          atomicMin(&s.range[0], r.start);
          atomicMax(&s.range[1], r.end);
        } else {
          r.row = -1;
          if (!STAND_IN) r.start = r.end = 0;
        }
      }
      s.own[threadIdx.x] = r;
      s.own_row[threadIdx.x] = r.row;
    }
    narrow = __syncthreads_and(narrow);
    mode = !narrow ? GENERAL : (identity ? LINEAR : (joint != nullptr ? JOINT : GENERAL));
    j0 = s.range[0];
    tiles = s.range[1] > j0 ? (s.range[1] - j0 + KB - 1) / KB : 0;
    if (parts > 1) {
      const int per = (tiles + parts - 1) / parts;
      j0 += part * per * KB;
      tiles = max(0, min(per, tiles - part * per));
    }
  }

  // By one warp: a position a lane.
  template <bool STATS>
  __device__ void stage_meta(int t) {
    static_assert(KB == 32, "a position a lane");
    const int slot = t % SLOTS;
    const int i = threadIdx.x & 31;
    const int j = j0 + t * KB + i;
    KeyMeta m{0, 0, 0, -1};
    if (j < s.range[1])
      *reinterpret_cast<int4*>(&m) = __ldg(reinterpret_cast<const int4*>(a.plan + j));
    if constexpr (STATS) {
      float2 st = make_float2(0.f, 0.f);
      float d = 0.f;
      if (m.row >= 0) {
        st = a.stats[head * a.n + j];
        st.y *= RAISE<T>;
        d = a.delta[head * a.n + j];
      }
      s.key_stats[slot][i] = st;
      s.key_delta[slot][i] = d;
    }
    const unsigned bad = __ballot_sync(0xffffffffu, j < s.range[1] && m.row < 0);
    if (i == 0) s.key_bad[slot] = bad != 0;
    s.key[slot][i] = m;
    s.key_lin[slot][i] = lin(m.x, m.y, m.z);
    s.key_row[slot][i] = m.row;
  }

  __device__ __forceinline__ uint32_t bucket(int qx, int qy, int qz, int kx, int ky, int kz) const {
    const int R = a.reach;
    const int x = lut[max(-R, min(R, sub_sat(kx, qx))) + R];
    const int y = lut[max(-R, min(R, sub_sat(ky, qy))) + R];
    const int z = lut[max(-R, min(R, sub_sat(kz, qz))) + R];
    return (uint32_t)((x * a.nb + y) * a.nb + z);
  }
};

// Calls use(n, e, at) for a thread's pairs with the pair's byte offset in the table: element e of
// fragment n is row g + 8 (e / 2) of 16 and column 8 n + 2 (lane % 4) + e % 2. FLIP: the rows are
// keys and the columns queries. WHOLE: all pairs are inside a window; otherwise the offsets of the
// others (masked) are clamped.
template <bool FLIP, bool WHOLE, typename T, int BQ, typename F>
__device__ __forceinline__ void each_pair(const Block<T, BQ>& b, int slot, const PlanRow* own,
                                          F&& use) {
  const int c2 = 2 * (threadIdx.x & 3);
  auto within = [](int v, uint32_t top) -> uint32_t {
    return WHOLE ? (uint32_t)v : min((uint32_t)v, top);
  };
  if (b.mode == LINEAR) {
    const uint32_t top = (uint32_t)b.cells() * 4u - 4u;
    const int mid = FLIP ? (int)(top / 2) : -(int)(top / 2);
    const int l[2] = {b.lin(own[0].x, own[0].y, own[0].z).x + mid,
                      b.lin(own[8].x, own[8].y, own[8].z).x + mid};
#pragma unroll
    for (int n = 0; n < KB / 8; ++n) {
      // the linear coordinates of two neighbours: .x and .z
      const int4 k = *reinterpret_cast<const int4*>(&b.s.key_lin[slot][n * 8 + c2]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = e & 1 ? k.z : k.x;
        use(n, e, within(FLIP ? l[e >> 1] - c : c - l[e >> 1], top));
      }
    }
  } else if (b.mode == JOINT) {
    const uint32_t joint = smem_u32(b.joint), lut = smem_u32(b.lut);
    const uint32_t top = (uint32_t)(b.width() * b.width()) * 2u - 2u;
    const uint32_t ztop = (uint32_t)b.width() * 2u - 2u;
    const int mid = FLIP ? (int)(top / 2) : -(int)(top / 2);
    const int zmid = FLIP ? 2 * b.a.reach : -2 * b.a.reach;
    int2 l[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] = b.lin(own[8 * r].x, own[8 * r].y, own[8 * r].z);
      l[r].x += mid;
      l[r].y += zmid;
    }
#pragma unroll
    for (int n = 0; n < KB / 8; ++n) {
      const int4 k = *reinterpret_cast<const int4*>(&b.s.key_lin[slot][n * 8 + c2]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = e & 1 ? k.z : k.x, z = e & 1 ? k.w : k.y;
        const uint32_t xy = within(FLIP ? l[e >> 1].x - c : c - l[e >> 1].x, top);
        const uint32_t dz = within(FLIP ? l[e >> 1].y - z : z - l[e >> 1].y, ztop);
        use(n, e, lds_u16(joint + xy) + lds_u16(lut + dz));
      }
    }
  } else {
#pragma unroll
    for (int n = 0; n < KB / 8; ++n) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const KeyMeta k = b.s.key[slot][n * 8 + c2 + c];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const PlanRow& o = own[8 * r];
          use(n, 2 * r + c, FLIP ? b.bucket(k.x, k.y, k.z, o.x, o.y, o.z)
                                 : b.bucket(o.x, o.y, o.z, k.x, k.y, k.z));
        }
      }
    }
  }
}

// acc += rows x tile^T over DP channels, 16 MR rows by KB columns; the rows' fragments come from
// `rows` (the warp's rows of a tile).
template <typename T, int DP, int MR>
__device__ __forceinline__ void mma_nt(float (&acc)[MR][KB / 8][4], uint32_t rows, uint32_t tile) {
  const int lane = threadIdx.x & 31;
  const uint32_t from = rows + (lane & 15) * STRIDE<DP> + (lane >> 4) * 16;
  const uint32_t at = tile + ((lane & 7) + (lane >> 4) * 8) * STRIDE<DP> + ((lane >> 3) & 1) * 16;
#pragma unroll
  for (int k = 0; k < DP / 16; ++k) {
    uint32_t f[MR][4];
#pragma unroll
    for (int m = 0; m < MR; ++m) ldsm4(from + m * 16 * STRIDE<DP> + k * 32, f[m]);
#pragma unroll
    for (int n = 0; n < KB / 16; ++n) {
      uint32_t b[4];
      ldsm4(at + n * 16 * STRIDE<DP> + k * 32, b);
#pragma unroll
      for (int m = 0; m < MR; ++m) {
        mma<T>(acc[m][2 * n], f[m], b[0], b[1]);
        mma<T>(acc[m][2 * n + 1], f[m], b[2], b[3]);
      }
    }
  }
}

// out += w (16 MR x KB sums, rounded to T as operand fragments) x tile (KB x DP). SPLIT: with a second
// product for what the rounding leaves out.
template <typename T, int DP, int MR, bool SPLIT = false>
__device__ __forceinline__ void mma_nn(float (&out)[MR][DP / 8][4],
                                       const float (&w)[MR][KB / 8][4], uint32_t tile) {
  const int lane = threadIdx.x & 31;
  const uint32_t at = tile + ((lane & 7) + ((lane >> 3) & 1) * 8) * STRIDE<DP> + (lane >> 4) * 16;
#pragma unroll
  for (int k = 0; k < KB / 16; ++k) {
    uint32_t f[MR][4];
#pragma unroll
    for (int m = 0; m < MR; ++m) {
      f[m][0] = pack2<T>(w[m][2 * k][0], w[m][2 * k][1]);
      f[m][1] = pack2<T>(w[m][2 * k][2], w[m][2 * k][3]);
      f[m][2] = pack2<T>(w[m][2 * k + 1][0], w[m][2 * k + 1][1]);
      f[m][3] = pack2<T>(w[m][2 * k + 1][2], w[m][2 * k + 1][3]);
    }
    uint32_t low[MR][4];
    if constexpr (SPLIT) {
#pragma unroll
      for (int m = 0; m < MR; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          low[m][i] = rest2<T>(f[m][i], w[m][2 * k + i / 2][i % 2 * 2],
                               w[m][2 * k + i / 2][i % 2 * 2 + 1]);
    }
#pragma unroll
    for (int n = 0; n < DP / 16; ++n) {
      uint32_t b[4];
      ldsm4_t(at + k * 16 * STRIDE<DP> + n * 32, b);
#pragma unroll
      for (int m = 0; m < MR; ++m) {
        mma<T>(out[m][2 * n], f[m], b[0], b[1]);
        mma<T>(out[m][2 * n + 1], f[m], b[2], b[3]);
        if constexpr (SPLIT) {
          mma<T>(out[m][2 * n], low[m], b[0], b[1]);
          mma<T>(out[m][2 * n + 1], low[m], b[2], b[3]);
        }
      }
    }
  }
}

template <int W>
__device__ __forceinline__ void zero(float (&x)[W][4]) {
#pragma unroll
  for (int i = 0; i < W; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) x[i][e] = 0.f;
}

// Positions that any of a warp's ROWS rows sees, and those that all of them do.
struct Reach {
  int lo, hi, all_lo, all_hi;
};
template <int ROWS>
__device__ __forceinline__ Reach warp_reach(const PlanRow* own) {
  const int lane = threadIdx.x & 31;
  const PlanRow& r = own[lane % ROWS];
  const bool any = r.row >= 0 && r.end > r.start;
  Reach w;
  w.lo = __reduce_min_sync(0xffffffffu, any ? r.start : INT_MAX);
  w.hi = __reduce_max_sync(0xffffffffu, any ? r.end : INT_MIN);
  w.all_lo = __reduce_max_sync(0xffffffffu, r.start);
  w.all_hi = __reduce_min_sync(0xffffffffu, r.end);
  return w;
}

// The columns of a thread's fragments that the rows g and g + 8 see, relative to its own first
// column: element (n, e) is column 8 n + e % 2 of row e / 2.
struct Sight {
  int lo[2], hi[2];
};
__device__ __forceinline__ Sight sight(const PlanRow* own, int p0) {
  const int c2 = 2 * (threadIdx.x & 3);
  Sight v;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    v.lo[r] = own[8 * r].start - p0 - c2;
    v.hi[r] = own[8 * r].end - p0 - c2;
  }
  return v;
}
// `bad`: some column has no row.
template <int BQ>
__device__ __forceinline__ bool hidden(const Sight& v, int n, int e, bool bad, const Shared<BQ>& s,
                                       int slot) {
  const int col = 8 * n + (e & 1);
  bool out = (col < v.lo[e >> 1]) | (col >= v.hi[e >> 1]);
  if (bad) out |= s.key_row[slot][col + 2 * (threadIdx.x & 3)] < 0;
  return out;
}

// A weight of zero does not hide a NaN or an infinity that another window's row brings into a tile. So
// rows that come out not finite are computed again, one at a time, from their own windows alone.
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

template <typename F>
__device__ __forceinline__ void again(uint32_t rows, int first, uint8_t* scratch, F&& row) {
  while (rows) {  // the same in all lanes
    const int r = __ffs(rows) - 1;
    rows &= rows - 1;
    __syncwarp();
    row(first + r, reinterpret_cast<float*>(scratch));
  }
}

template <typename T>
__device__ __noinline__ void again_forward(AttnArgs a, int64_t p, int h, float* s) {
  row_forward<T, true>(a, p, h, s);
}
template <typename T>
__device__ __noinline__ void again_dq(AttnArgs a, int64_t p, int h, float* s) {
  row_dq<T, true>(a, p, h, s);
}
template <typename T>
__device__ __noinline__ void again_dkv(AttnArgs a, int64_t p, int h, float* s) {
  row_dkv<T, true>(a, p, h, s);
}

// Shared memory: OWN tiles of the block's BQ rows, STAGES buffers of two tiles of KB positions, then
// the tables.
template <int DP, int BQ, int OWN, int STAGES>
struct Layout {
  static constexpr int OWN_TILE = BQ * STRIDE<DP>;
  static constexpr int TILE = KB * STRIDE<DP>;
  static constexpr int RING = OWN * OWN_TILE;
  static constexpr int SHARED = RING + STAGES * 2 * TILE;
  static constexpr int TABLE = (SHARED + (int)sizeof(Shared<BQ>) + 15) / 16 * 16;
};

struct Tables {
  int words, units, lut, joint, total;  // byte offsets behind Layout::TABLE; joint < 0: none
};
// `words`: one 32-bit word a bucket beside the bias; `units`: and one byte.
__host__ __device__ inline Tables tables(const AttnArgs& a, bool words, bool units) {
  const int cells = a.nb * a.nb * a.nb, width = 2 * a.reach + 1;
  Tables t;
  t.words = cells * 4;
  t.units = t.words + (words ? cells * 4 : 0);
  t.lut = (t.units + (units ? cells : 0) + 15) / 16 * 16;
  t.joint = -1;
  t.total = t.lut + (width * 2 + 15) / 16 * 16;
  if (width * width <= JOINT_MAX) {
    t.joint = t.total;
    t.total += width * width * 2;
  }
  return t;
}

// The plan's list of blocks of BQ positions.
struct BlockList {
  const int2* at;
  int count;
};
template <int BQ>
__device__ __forceinline__ BlockList block_list(const AttnArgs& a) {
  static_assert(BQ == 64 || BQ == 128, "the plan's sizes");
  constexpr int which = BQ == 128;
  const PlanBlocks b = plan_blocks(a.n);
  const uint8_t* plan = reinterpret_cast<const uint8_t*>(a.plan);
  const int count = __ldg(reinterpret_cast<const int*>(plan + b.count) + which);
  return {reinterpret_cast<const int2*>(plan + b.block[which]),
          (int)min((int64_t)count, b.cap[which])};
}

template <typename T, int BQ>
__device__ __forceinline__ Block<T, BQ> make_block(const AttnArgs& a, uint8_t* smem, int shared,
                                                   int table, bool words, bool units) {
  const Tables t = tables(a, words, units);
  return Block<T, BQ>{a, *reinterpret_cast<Shared<BQ>*>(smem + shared),
                      reinterpret_cast<float*>(smem + table),
                      reinterpret_cast<uint16_t*>(smem + table + t.lut),
                      t.joint < 0 ? nullptr : reinterpret_cast<uint16_t*>(smem + table + t.joint),
                      (int)blockIdx.y, false};
}

// The tiles of one block: load(buffer, rows) fetches a tile's rows, STAGES - 1 tiles ahead (the
// block's own rows, loaded before, are in the first group), and body(t, buffer) works on tile t.
// One barrier a tile: behind it the tile has landed, the readers of the buffer that is filled next
// are done, and the rows of the tile that fills it are known. ask() is asked at the barrier, by
// every thread, and flush() done before the tile if any said yes.
template <bool STATS, int STAGES, typename B, typename Load, typename Body, typename Ask,
          typename Flush>
__device__ __forceinline__ void walk(B& b, Load&& load, Body&& body, Ask&& ask, Flush&& flush) {
  static_assert(STAGES + 1 <= SLOTS, "rows known ahead");
  const int warp = threadIdx.x >> 5;
  if (warp < STAGES) b.template stage_meta<STATS>(warp);
  __syncthreads();
#pragma unroll
  for (int t = 0; t < STAGES - 1; ++t) {
    if (t < b.tiles) load(t, b.s.key_row[t]);
    cp_commit();
  }
  int buf = 0, fill = STAGES - 1;
  for (int t = 0; t < b.tiles; ++t) {
    cp_wait<STAGES - 2>();
    if (__syncthreads_or(ask())) flush();
    if (t + STAGES - 1 < b.tiles) load(fill, b.s.key_row[(t + STAGES - 1) % SLOTS]);
    cp_commit();
    // by another warp each time
    if (t + STAGES < b.tiles && warp == (t & 3)) b.template stage_meta<STATS>(t + STAGES);
    body(t, buf);
    buf = buf + 1 == STAGES ? 0 : buf + 1;
    fill = fill + 1 == STAGES ? 0 : fill + 1;
  }
  cp_wait<0>();
  __syncthreads();
}

// The running base lies LIFT below the largest score that it was set by, so that weights start at
// 2^LIFT, and scores may pass that by SLACK (all in powers of two) before the sums are rescaled, so most
// tiles skip it. bf16: weights of 1 to 2^8, which neither the type nor the fp32 sums notice. fp16: up
// to 2^15, so that weights 2^-27 of the largest still have all their bits.
template <typename T>
constexpr float LIFT = IS_HALF<T> ? 13.f : 0.f;
template <typename T>
constexpr float SLACK = IS_HALF<T> ? 2.f : 8.f;

// MR: 16-row parts of a warp, whose products share the tile's fragments. TRAIN: the backward pass's
// inputs are kept too.
template <typename T, int DP, int MR, int STAGES, bool TRAIN>
__global__ void __launch_bounds__(AT, DP <= 64 ? 3 : 2)
    attn_tc_kernel(AttnArgs a, bool vec) {
  constexpr int BQ = 64 * MR;
  using L = Layout<DP, BQ, 1, STAGES>;
  extern __shared__ __align__(16) uint8_t smem[];
  const BlockList list = block_list<BQ>(a);
  if ((int)blockIdx.x >= list.count) return;
  Block<T, BQ> b = make_block<T, BQ>(a, smem, L::SHARED, L::TABLE, false, false);
  Shared<BQ>& sh = b.s;
  const int head = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c2 = 2 * (lane & 3);
  const int row0 = warp * 16 * MR;            // the warp's rows of the block
  uint8_t* mine = smem + row0 * STRIDE<DP>;   // and of q
  const T* q = static_cast<const T*>(a.q) + head * a.q_head;
  const T* k = static_cast<const T*>(a.k) + head * a.k_head;
  const T* v = static_cast<const T*>(a.v) + head * a.v_head;
  const float scale = a.scale * ATTN_LOG2E;
  const uint32_t table = smem_u32(b.table);
  b.stage_tables();
  for (int block = blockIdx.x; block < list.count; block += gridDim.x) {
    const int2 at = __ldg(list.at + block);
    b.template begin<true>(at.x, at.y, blockIdx.z, a.parts);
    load_tile<T, DP, BQ>(smem, q, (int)a.q_row, sh.own_row, a.dim, vec);
    const PlanRow* own = sh.own + row0 + g;
    const Reach w = warp_reach<16 * MR>(sh.own + row0);
    float o[MR][DP / 8][4], base[MR][2], sum[MR][2];
#pragma unroll
    for (int m = 0; m < MR; ++m) {
      zero(o[m]);
      base[m][0] = base[m][1] = -3.402823466e38f;
      sum[m][0] = sum[m][1] = 0.f;
    }
    auto body = [&](int t, int buf) {
      const int p0 = b.j0 + t * KB;
      if (p0 >= w.hi || p0 + KB <= w.lo) return;
      const uint32_t tile = smem_u32(smem + L::RING + buf * 2 * L::TILE);
      const int slot = t % SLOTS;
      const bool bad = sh.key_bad[slot];
      const bool whole = p0 >= w.all_lo && p0 + KB <= w.all_hi && !bad;
      float s[MR][KB / 8][4];
#pragma unroll
      for (int m = 0; m < MR; ++m) zero(s[m]);
      mma_nt<T, DP, MR>(s, smem_u32(mine), tile);
#pragma unroll
      for (int m = 0; m < MR; ++m) {
        auto score = [&](int n, int e, uint32_t at) {
          s[m][n][e] = fmaf(s[m][n][e], scale, lds_f32(table + at));
        };
        if (whole) {
          each_pair<false, true>(b, slot, own + 16 * m, score);
        } else {
          each_pair<false, false>(b, slot, own + 16 * m, score);
          const Sight seen = sight(own + 16 * m, p0);
#pragma unroll
          for (int n = 0; n < KB / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (hidden(seen, n, e, bad, sh, slot)) s[m][n][e] = -INFINITY;
        }
      }
      float top[MR][2];
      bool over = false;
#pragma unroll
      for (int m = 0; m < MR; ++m) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float x = fmaxf(s[m][0][2 * r], s[m][0][2 * r + 1]);
#pragma unroll
          for (int n = 1; n < KB / 8; ++n) x = fmaxf(x, fmaxf(s[m][n][2 * r], s[m][n][2 * r + 1]));
          top[m][r] = x;
          over = over || x > base[m][r] + (LIFT<T> + SLACK<T>);
        }
      }
      if (__any_sync(0xffffffffu, over)) {
#pragma unroll
        for (int m = 0; m < MR; ++m) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float x = top[m][r];
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
            x = fmaxf(x - LIFT<T>, base[m][r]);
            const float keep = exp2_fast(base[m][r] - x);
            base[m][r] = x;
            sum[m][r] *= keep;
#pragma unroll
            for (int n = 0; n < DP / 8; ++n) {
              o[m][n][2 * r] *= keep;
              o[m][n][2 * r + 1] *= keep;
            }
          }
        }
      }
#pragma unroll
      for (int m = 0; m < MR; ++m)
#pragma unroll
        for (int n = 0; n < KB / 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[m][n][e] = exp2_fast(s[m][n][e] - base[m][e >> 1]);
            sum[m][e >> 1] += s[m][n][e];
          }
      mma_nn<T, DP, MR, TRAIN>(o, s, tile + L::TILE);
    };
    walk<false, STAGES>(
        b,
        [&](int buf, const int32_t* rows) {
          uint8_t* tile = smem + L::RING + buf * 2 * L::TILE;
          load_tile<T, DP, KB>(tile, k, (int)a.k_row, rows, a.dim, vec);
          load_tile<T, DP, KB>(tile + L::TILE, v, (int)a.v_row, rows, a.dim, vec);
        },
        body, [] { return false; }, [] {});
    if (a.parts > 1) {
      const int64_t first = ((int64_t)blockIdx.z * a.heads + head) * a.n + at.x;
#pragma unroll
      for (int m = 0; m < MR; ++m) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float x = sum[m][r];
          x += __shfl_xor_sync(0xffffffffu, x, 1);
          x += __shfl_xor_sync(0xffffffffu, x, 2);
          const int i = row0 + 16 * m + g + 8 * r;
          if (sh.own_row[i] < 0) continue;
          if (c2 == 0) a.part_stats[first + i] = make_float2(base[m][r], x);
          float* dst = a.part_out + (first + i) * a.dim;
#pragma unroll
          for (int n = 0; n < DP / 8; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (n * 8 + c2 + e < a.dim) dst[n * 8 + c2 + e] = o[m][n][2 * r + e];
        }
      }
      __syncthreads();
      continue;
    }
    // the ring is free: the rests go there, a stretch a warp
    static_assert(4 * MR * 16 * STRIDE<DP> <= STAGES * 2 * L::TILE, "room for the rests");
    uint8_t* rest = smem + L::RING + row0 * STRIDE<DP>;
    uint32_t redo = 0;
#pragma unroll
    for (int m = 0; m < MR; ++m) {
      float inv[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float x = sum[m][r];
        x += __shfl_xor_sync(0xffffffffu, x, 1);
        x += __shfl_xor_sync(0xffffffffu, x, 2);
        const float2 st = row_stats(base[m][r], x);
        inv[r] = st.y;
        const int i = row0 + 16 * m + g + 8 * r;
        if (TRAIN && a.stats && c2 == 0 && sh.own_row[i] >= 0)
          a.stats[head * a.n + at.x + i] = st;
      }
      put_rows<T, DP>(mine + 16 * m * STRIDE<DP>, o[m], inv[0], inv[1]);
      if constexpr (TRAIN)
        put_rows<T, DP, true>(rest + 16 * m * STRIDE<DP>, o[m], inv[0], inv[1]);
      redo |= not_finite<DP>(o[m]) << (16 * m);
    }
    __syncwarp();
#pragma unroll
    for (int m = 0; m < MR; ++m) {
      const int32_t* rows = sh.own_row + row0 + 16 * m;
      send_rows<T, DP>(mine + 16 * m * STRIDE<DP>, rows, static_cast<T*>(a.out), a.heads, head,
                       a.dim, vec);
      if (TRAIN && a.out_rest)
        send_rows<T, DP>(rest + 16 * m * STRIDE<DP>, rows, static_cast<T*>(a.out_rest), a.heads,
                         head, a.dim, vec);
    }
    again(redo, row0, mine, [&](int i, float* f) {
      if (sh.own_row[i] >= 0) again_forward<T>(a, at.x + i, head, f);
    });
    __syncthreads();
  }
}

// The parts of a split walk, joined in order: a warp per row and head. Rows that come out not finite
// are computed again, as in the kernel above.
constexpr int JOIN_WARPS = 8;
template <typename T>
__global__ void __launch_bounds__(32 * JOIN_WARPS) attn_join_kernel(AttnArgs a) {
  __shared__ float scratch[JOIN_WARPS][ATTN_MAX_DIM];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, h = blockIdx.y;
  const int64_t p = (int64_t)blockIdx.x * JOIN_WARPS + warp;
  if (p >= a.n) return;
  const int32_t row = __ldg(&a.plan[p].row);
  if (row < 0) return;
  float top = -3.402823466e38f, sum = 0.f, o[ATTN_CH] = {};
  for (int z = 0; z < a.parts; ++z)
    top = fmaxf(top, a.part_stats[((int64_t)z * a.heads + h) * a.n + p].x);
  for (int z = 0; z < a.parts; ++z) {
    const int64_t at = ((int64_t)z * a.heads + h) * a.n + p;
    const float2 st = a.part_stats[at];
    const float w = exp2f(st.x - top);
    sum = fmaf(w, st.y, sum);
#pragma unroll
    for (int c = 0; c < ATTN_CH; ++c)
      if (lane + 32 * c < a.dim) o[c] = fmaf(w, a.part_out[at * a.dim + lane + 32 * c], o[c]);
  }
  bool finite = true;
#pragma unroll
  for (int c = 0; c < ATTN_CH; ++c) finite = finite && fabsf(o[c]) < INFINITY;
  if (!__all_sync(0xffffffffu, finite)) {
    again_forward<T>(a, p, h, scratch[warp]);
    return;
  }
  const float2 st = row_stats(top, sum);
  const int64_t own = ((int64_t)row * a.heads + h) * a.dim;
#pragma unroll
  for (int c = 0; c < ATTN_CH; ++c) {
    const int d = lane + 32 * c;
    if (d >= a.dim) continue;
    const float x = o[c] * st.y;
    static_cast<T*>(a.out)[own + d] = from_f32<T>(x);
    if (a.out_rest) static_cast<T*>(a.out_rest)[own + d] = from_f32<T>(rest_of<T>(x));
  }
  if (lane == 0 && a.stats) a.stats[h * a.n + p] = st;
}

// delta_i = dout_i . o_i by position: eight lanes a row and head, a warp four heads of a row, a block
// eight positions. o is taken with what its rounding left out: dS = P (dP - delta) is small next to
// delta where a window has few rows, so half a step of o would be several of dS.
template <typename T>
__global__ void __launch_bounds__(256) attn_delta_kernel(AttnArgs a, bool vec) {
  const int sub = threadIdx.x & 7;
  const int64_t p = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int h = blockIdx.y * 4 + ((threadIdx.x >> 3) & 3);
  const bool live = p < a.n && h < a.heads;
  const int32_t row = live ? __ldg(&a.plan[p].row) : -1;
  float d = 0.f;
  if (row >= 0) {
    const int64_t from = ((int64_t)row * a.heads + h) * a.dim;
    const T* g = static_cast<const T*>(a.dout) + from;
    const T* o = static_cast<const T*>(a.o) + from;
    const T* rest = a.o_rest ? static_cast<const T*>(a.o_rest) + from : nullptr;
    if (vec) {
#pragma unroll
      for (int i = 0; i < ATTN_MAX_DIM / 64; ++i) {
        const int c = sub * 8 + i * 64;
        if (c >= a.dim) break;
        const uint4 x = *reinterpret_cast<const uint4*>(g + c);
        const uint4 y = *reinterpret_cast<const uint4*>(o + c);
        const uint4 z = rest ? *reinterpret_cast<const uint4*>(rest + c) : make_uint4(0, 0, 0, 0);
        const T* xe = reinterpret_cast<const T*>(&x);
        const T* ye = reinterpret_cast<const T*>(&y);
        const T* ze = reinterpret_cast<const T*>(&z);
#pragma unroll
        for (int k = 0; k < 8; ++k) d = fmaf(to_f32(xe[k]), whole_of(ye[k], ze[k]), d);
      }
    } else {
      for (int c = sub; c < a.dim; c += 8)
        d = fmaf(to_f32(g[c]), rest ? whole_of(o[c], rest[c]) : to_f32(o[c]), d);
    }
  }
#pragma unroll
  for (int s = 4; s > 0; s >>= 1) d += __shfl_xor_sync(0xffffffffu, d, s);
  if (sub == 0 && live) a.delta[h * a.n + p] = d;
}

// Raises score gradients `ds` of a thread's two rows (g and g + 8; the four lanes of a row agree) so that
// their largest lies below 2^15, and lowers the sums formed so far with them: `by` is a power of two
// for each row, no larger than it was.
constexpr float RAISE_START = 0x1p100f;
template <int DP>
__device__ __forceinline__ void raise_rows(float (&ds)[KB / 8][4], float (&by)[2],
                                           float (&sums)[DP / 8][4]) {
  float top[2] = {0.f, 0.f};
#pragma unroll
  for (int n = 0; n < KB / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) top[e >> 1] = fmaxf(top[e >> 1], fabsf(ds[n][e]));
  constexpr float LIMIT = 32768.f;
  if (__any_sync(0xffffffffu, top[0] * by[0] > LIMIT || top[1] * by[1] > LIMIT)) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float x = top[r];
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
      // an infinity stays one, and its row is computed again
      if (x * by[r] > LIMIT && x < INFINITY) {
        const float to = __uint_as_float((268u - (__float_as_uint(x) >> 23)) << 23);  // x to = 2^14 ..
        const float keep = to / by[r];
        by[r] = to;
#pragma unroll
        for (int n = 0; n < DP / 8; ++n) {
          sums[n][2 * r] *= keep;
          sums[n][2 * r + 1] *= keep;
        }
      }
    }
  }
#pragma unroll
  for (int n = 0; n < KB / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) ds[n][e] *= by[e >> 1];
}

// The table's gradient in fixed point, with a unit for each bucket: a score gradient is at most 2^18 of
// its bucket's units (the bucket's largest is known from the dk / dv pass), so every pair keeps 2^-18 of
// its own bucket's largest however far another bucket's or row's lie above it. (One unit for a head
// left exact zeros in 62% of the buckets of a table that falls by 1.5 a voxel.) The pairs sum to a
// 32-bit word per bucket in shared memory. A thread counts the units it has added; the block empties its
// words into the 64-bit sums in global memory before any thread's count can pass 2^24, so 128 threads
// cannot overflow a word.
constexpr int UNIT_BITS = 18;
constexpr float UNIT_TOP = (float)(1 << UNIT_BITS);
// Exponent of a bucket's reciprocal unit; INT_MAX when a score gradient of the bucket was not finite.
__device__ __forceinline__ int unit_exponent(unsigned bits) {
  const float top = __uint_as_float(bits);
  if (!(top < INFINITY)) return INT_MAX;
  if (top == 0.f) return 120;
  int e;
  frexpf(top, &e);                      // top < 2^e
  return min(UNIT_BITS - 1 - e, 120);   // the two passes round their products differently
}

// dq and the table's gradient.
template <typename T, int DP, int STAGES, bool TABLE>
__global__ void __launch_bounds__(AT, DP <= 64 ? 3 : 2)
    attn_dq_tc_kernel(AttnArgs a, bool vec) {
  constexpr int BQ = 64;
  using L = Layout<DP, BQ, 2, STAGES>;
  extern __shared__ __align__(16) uint8_t smem[];
  const BlockList list = block_list<BQ>(a);
  if ((int)blockIdx.x >= list.count) return;
  Block<T, BQ> b = make_block<T, BQ>(a, smem, L::SHARED, L::TABLE, TABLE, TABLE);
  Shared<BQ>& sh = b.s;
  const int cells = b.cells();
  const Tables extra = tables(a, TABLE, TABLE);
  int* s_grad = reinterpret_cast<int*>(smem + L::TABLE + extra.words);
  uint8_t* s_unit = smem + L::TABLE + extra.units;  // the units' reciprocals: their exponent fields
  const uint32_t table = smem_u32(b.table), grads = smem_u32(s_grad), units = smem_u32(s_unit);
  const int head = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2;
  uint8_t* mine = smem + warp * 16 * STRIDE<DP>;
  const T* q = static_cast<const T*>(a.q) + head * a.q_head;
  const T* k = static_cast<const T*>(a.k) + head * a.k_head;
  const T* v = static_cast<const T*>(a.v) + head * a.v_head;
  const T* dout = static_cast<const T*>(a.dout) + (int64_t)head * a.dim;
  const int g_row = a.heads * a.dim;
  const float scale = a.scale * ATTN_LOG2E;
  // a thread adds KB / 2 pairs a tile; half a unit each for rounding to an integer and as much for
  // rounding the count itself
  constexpr float LIMIT = 16777216.f - 2 * KB - (KB / 2) * UNIT_TOP;
  float spent = 0.f;  // units added since the words were emptied
  if constexpr (TABLE) {
    const unsigned* tops = a.tops + (int64_t)head * cells;
    for (int i = threadIdx.x; i < cells; i += AT) {
      const int e = unit_exponent(__ldg(tops + i));
      s_grad[i] = 0;
      s_unit[i] = (uint8_t)(e == INT_MAX ? 0 : 127 + e);  // 0: nothing of the bucket counts
    }
  }
  b.stage_tables();
  auto flush = [&] {
    if constexpr (TABLE) {
      for (int i = threadIdx.x; i < cells; i += AT) {
        const int add = s_grad[i];
        s_grad[i] = 0;
        if (add != 0)
          atomicAdd(a.dtable + (int64_t)head * cells + i, (unsigned long long)(long long)add);
      }
      spent = 0.f;
      __syncthreads();
    }
  };
  for (int block = blockIdx.x; block < list.count; block += gridDim.x) {
    const int2 at = __ldg(list.at + block);
    b.template begin<false, true>(at.x, at.y);
    load_tile<T, DP, BQ>(smem, q, (int)a.q_row, sh.own_row, a.dim, vec);
    load_tile<T, DP, BQ>(smem + L::OWN_TILE, dout, g_row, sh.own_row, a.dim, vec);
    const PlanRow* own = sh.own + warp * 16 + g;
    const Reach w = warp_reach<16>(sh.own + warp * 16);
    float top[2], inv[2], delta[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const bool live = own[8 * r].row >= 0;
      const int64_t p = head * a.n + at.x + warp * 16 + g + 8 * r;
      const float2 st = live ? a.stats[p] : make_float2(0.f, 0.f);
      top[r] = st.x;
      inv[r] = st.y;
      delta[r] = live ? a.delta[p] : 0.f;
    }
    float dq[1][DP / 8][4], by[2] = {1.f, 1.f};
    zero(dq[0]);
    if constexpr (IS_HALF<T>) by[0] = by[1] = RAISE_START;
    auto body = [&](int t, int buf) {
      const int p0 = b.j0 + t * KB;
      if (p0 >= w.hi || p0 + KB <= w.lo) return;
      const uint32_t tile = smem_u32(smem + L::RING + buf * 2 * L::TILE);
      const int slot = t % SLOTS;
      float s[1][KB / 8][4], dp[1][KB / 8][4];
      zero(s[0]);
      mma_nt<T, DP, 1>(s, smem_u32(mine), tile);
#pragma unroll
      for (int n = 0; n < KB / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) dp[0][n][e] = -delta[e >> 1];
      mma_nt<T, DP, 1>(dp, smem_u32(mine + L::OWN_TILE), tile + L::TILE);
      const bool bad = sh.key_bad[slot];
      if constexpr (TABLE) spent += KB / 2;
      auto grad = [&](int n, int e, uint32_t at, bool in) {
        const int r = e >> 1;
        const float x = fmaf(s[0][n][e], scale, lds_f32(table + at));
        const float ds = exp2_fast(x - top[r]) * (inv[r] * dp[0][n][e]);
        s[0][n][e] = in ? ds : 0.f;
        if constexpr (TABLE) {
          if (in) {
            // The two passes round dp - delta differently: where that is all a bucket's terms are, this
            // one may find a larger term. A NaN counts as a number, and its bucket ends as NaN.
            const float unit = __uint_as_float(lds_u8(units + (at >> 2)) << 23);
            const float u = fminf(fmaxf(ds * unit, -UNIT_TOP), UNIT_TOP);
            spent += fabsf(u);
            // 1.5 * 2^23: the sum's low bits are the rounded integer
            asm volatile("red.shared.add.s32 [%0], %1;" ::"r"(grads + at),
                         "r"(__float_as_int(u + 12582912.f) - 0x4b400000));
          }
        }
      };
      if (p0 >= w.all_lo && p0 + KB <= w.all_hi && !bad) {
        each_pair<false, true>(b, slot, own,
                               [&](int n, int e, uint32_t at) { grad(n, e, at, true); });
      } else {
        const Sight seen = sight(own, p0);
        each_pair<false, false>(b, slot, own, [&](int n, int e, uint32_t at) {
          grad(n, e, at, !hidden(seen, n, e, bad, sh, slot));
        });
      }
      if constexpr (IS_HALF<T>) raise_rows<DP>(s[0], by, dq[0]);
      mma_nn<T, DP, 1>(dq, s, tile);
    };
    walk<false, STAGES>(
        b,
        [&](int buf, const int32_t* rows) {
          uint8_t* tile = smem + L::RING + buf * 2 * L::TILE;
          load_tile<T, DP, KB>(tile, k, (int)a.k_row, rows, a.dim, vec);
          load_tile<T, DP, KB>(tile + L::TILE, v, (int)a.v_row, rows, a.dim, vec);
        },
        body, [&] { return TABLE && spent > LIMIT; }, flush);
    store_rows<T, DP>(mine, dq[0], a.scale / by[0], a.scale / by[1], sh.own_row + warp * 16,
                      static_cast<T*>(a.dq), a.heads, head, a.dim, vec);
    again(not_finite<DP>(dq[0]), warp * 16, mine, [&](int i, float* f) {
      if (sh.own_row[i] >= 0) again_dq<T>(a, at.x + i, head, f);
    });
    __syncthreads();
  }
  flush();
}

// dk and dv, and the largest |dS| of every bucket: the block's rows are keys, the tiles queries.
template <typename T, int DP, int STAGES, bool TABLE>
__global__ void __launch_bounds__(AT, DP <= 64 ? 3 : 2)
    attn_dkv_tc_kernel(AttnArgs a, bool vec) {
  constexpr int BQ = 64;
  using L = Layout<DP, BQ, 2, STAGES>;
  extern __shared__ __align__(16) uint8_t smem[];
  const BlockList list = block_list<BQ>(a);
  if ((int)blockIdx.x >= list.count) return;
  Block<T, BQ> b = make_block<T, BQ>(a, smem, L::SHARED, L::TABLE, TABLE, false);
  Shared<BQ>& sh = b.s;
  const int cells = b.cells();
  unsigned* s_top = reinterpret_cast<unsigned*>(smem + L::TABLE + tables(a, TABLE, false).words);
  const uint32_t table = smem_u32(b.table), tops = smem_u32(s_top);
  const int head = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c2 = 2 * (lane & 3);
  uint8_t* mine = smem + warp * 16 * STRIDE<DP>;
  const T* q = static_cast<const T*>(a.q) + head * a.q_head;
  const T* k = static_cast<const T*>(a.k) + head * a.k_head;
  const T* v = static_cast<const T*>(a.v) + head * a.v_head;
  const T* dout = static_cast<const T*>(a.dout) + (int64_t)head * a.dim;
  const int g_row = a.heads * a.dim;
  const float scale = a.scale * ATTN_LOG2E;
  if constexpr (TABLE) {
    for (int i = threadIdx.x; i < cells; i += AT) s_top[i] = 0u;
  }
  b.stage_tables();
  for (int block = blockIdx.x; block < list.count; block += gridDim.x) {
    const int2 at = __ldg(list.at + block);
    b.template begin<false>(at.x, at.y);
    load_tile<T, DP, BQ>(smem, k, (int)a.k_row, sh.own_row, a.dim, vec);
    load_tile<T, DP, BQ>(smem + L::OWN_TILE, v, (int)a.v_row, sh.own_row, a.dim, vec);
    const PlanRow* own = sh.own + warp * 16 + g;
    const Reach w = warp_reach<16>(sh.own + warp * 16);
    const bool solo[2] = {lone(own[0]), lone(own[8])};
    float dk[1][DP / 8][4], dv[1][DP / 8][4], by[2] = {1.f, 1.f};
    if constexpr (IS_HALF<T>) by[0] = by[1] = RAISE_START;
    zero(dk[0]);
    zero(dv[0]);
    auto body = [&](int t, int buf) {
      const int p0 = b.j0 + t * KB;
      if (p0 >= w.hi || p0 + KB <= w.lo) return;
      const uint32_t tile = smem_u32(smem + L::RING + buf * 2 * L::TILE);
      const int slot = t % SLOTS;
      const bool bad = sh.key_bad[slot];
      const bool whole = p0 >= w.all_lo && p0 + KB <= w.all_hi && !bad;
      float s[1][KB / 8][4], dp[1][KB / 8][4];
      zero(s[0]);
      mma_nt<T, DP, 1>(s, smem_u32(mine), tile);
      auto form_dp = [&] {
#pragma unroll
        for (int n = 0; n < KB / 8; ++n) {
          const float2 delta = *reinterpret_cast<const float2*>(&sh.key_delta[slot][n * 8 + c2]);
          dp[0][n][0] = dp[0][n][2] = -delta.x;
          dp[0][n][1] = dp[0][n][3] = -delta.y;
        }
        mma_nt<T, DP, 1>(dp, smem_u32(mine + L::OWN_TILE), tile + L::TILE);
      };
      // A bucket's largest term wants dP while its word is known; without a table gradient dP comes after
      // dv's product, which spares its registers there (282 against 291 us).
      if constexpr (TABLE) form_dp();
      auto grad = [&](int n, int e, uint32_t at, bool in, bool counts) {
        const float2 st = sh.key_stats[slot][n * 8 + c2 + (e & 1)];
        const float w = exp2_fast(fmaf(s[0][n][e], scale, lds_f32(table + at)) - st.x) * st.y;
        s[0][n][e] = in ? w : 0.f;
        if constexpr (TABLE) {
          // a pair out of sight may be with a row that holds anything
          dp[0][n][e] = in ? w * dp[0][n][e] : 0.f;
          // bits of numbers that are not negative order like the numbers, a NaN's above all
          asm volatile("red.shared.max.u32 [%0], %1;" ::"r"(tops + at),
                       "r"(counts ? __float_as_uint(dp[0][n][e]) & 0x7fffffffu : 0u));
        }
      };
      if (whole) {
        each_pair<true, true>(b, slot, own,
                              [&](int n, int e, uint32_t at) { grad(n, e, at, true, true); });
      } else {
        const Sight seen = sight(own, p0);
        each_pair<true, false>(b, slot, own, [&](int n, int e, uint32_t at) {
          grad(n, e, at, !hidden(seen, n, e, bad, sh, slot), !solo[e >> 1]);
        });
      }
      mma_nn<T, DP, 1>(dv, s, tile + L::TILE);
      if constexpr (!TABLE) {
        form_dp();
#pragma unroll
        for (int n = 0; n < KB / 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            // here a weight of zero stands for a pair out of sight
            dp[0][n][e] = !whole && s[0][n][e] == 0.f ? 0.f : s[0][n][e] * dp[0][n][e];
      }
      if constexpr (IS_HALF<T>) raise_rows<DP>(dp[0], by, dk[0]);
      mma_nn<T, DP, 1>(dk, dp, tile);
    };
    walk<true, STAGES>(
        b,
        [&](int buf, const int32_t* rows) {
          uint8_t* tile = smem + L::RING + buf * 2 * L::TILE;
          load_tile<T, DP, KB>(tile, q, (int)a.q_row, rows, a.dim, vec);
          load_tile<T, DP, KB>(tile + L::TILE, dout, g_row, rows, a.dim, vec);
        },
        body, [] { return false; }, [] {});
    // a power of two, and the quotient exact
    const float down[2] = {a.scale / RAISE<T> / by[0], a.scale / RAISE<T> / by[1]};
    store_rows<T, DP>(mine, dk[0], solo[0] ? 0.f : down[0], solo[1] ? 0.f : down[1], sh.own_row + warp * 16, static_cast<T*>(a.dk), a.heads, head, a.dim, vec);
    store_rows<T, DP>(mine + L::OWN_TILE, dv[0], 1.f / RAISE<T>, 1.f / RAISE<T>, sh.own_row + warp * 16,
                      static_cast<T*>(a.dv), a.heads, head, a.dim, vec);
    again(not_finite<DP>(dk[0]) | not_finite<DP>(dv[0]), warp * 16, mine, [&](int i, float* f) {
      if (sh.own_row[i] >= 0) again_dkv<T>(a, at.x + i, head, f);
    });
    __syncthreads();
  }
  if constexpr (TABLE) {  // behind the last block's barrier
    unsigned* to = a.tops + (int64_t)head * cells;
    for (int i = threadIdx.x; i < cells; i += AT)
      if (s_top[i] != 0u)
        atomicMax(to + i, __float_as_uint(__uint_as_float(s_top[i]) / RAISE<T>));
  }
}

template <typename T>
__global__ void __launch_bounds__(256) dtable_tc_finish_kernel(AttnArgs a, T* __restrict__ out) {
  const int cells = a.nb * a.nb * a.nb;
  const int h = blockIdx.y;
  for (int b = blockIdx.x * 256 + threadIdx.x; b < cells; b += gridDim.x * 256) {
    const int64_t at = (int64_t)h * cells + b;
    const int exponent = unit_exponent(a.tops[at]);
    const double v = exponent == INT_MAX
                         ? __longlong_as_double(0x7ff8000000000000ll)  // something was not finite
                         : ldexp((double)(long long)a.dtable[at], -exponent);
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
         wide(a.v, a.v_row, a.v_head) && wide(a.out, row, head) && wide(a.out_rest, row, head) &&
         wide(a.o, row, head) && wide(a.o_rest, row, head) && wide(a.dout, row, head) &&
         wide(a.dq, row, head) && wide(a.dk, row, head) && wide(a.dv, row, head);
}

// CTAs of one head: each takes every that-many-th block, so that it stages the table (and adds up its
// gradient) once. `waves` for each SM over all heads; the list is at most `cap` long.
unsigned ctas_of(const AttnArgs& a, int bq, int waves) {
  const int64_t want = ((int64_t)num_sms() * waves + a.heads - 1) / a.heads;
  return (unsigned)std::min(want, plan_blocks(a.n).cap[bq == 128]);
}

template <typename K>
int allow_smem(K kernel, size_t bytes) {
  SV_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   (int)bytes));
  return SV_OK;
}

template <typename T, int DP, bool TRAIN>
int forward(const AttnArgs& a, cudaStream_t s) {
  constexpr int MR = FORWARD_ROWS / 64, STAGES = DP <= 64 ? 3 : 2;
  const size_t bytes = Layout<DP, 64 * MR, 1, STAGES>::TABLE + tables(a, false, false).total;
  const int rc = allow_smem(attn_tc_kernel<T, DP, MR, STAGES, TRAIN>, bytes);
  if (rc != SV_OK) return rc;
  attn_tc_kernel<T, DP, MR, STAGES, TRAIN>
      <<<dim3(ctas_of(a, 64 * MR, WAVES), a.heads, a.parts), AT, bytes, s>>>(a, wide_rows(a));
  SV_LAUNCH_CHECK();
  if (a.parts > 1) {
    attn_join_kernel<T><<<dim3((unsigned)((a.n + JOIN_WARPS - 1) / JOIN_WARPS), a.heads),
                          32 * JOIN_WARPS, 0, s>>>(a);
    SV_LAUNCH_CHECK();
  }
  return SV_OK;
}

template <typename T, int DP, bool TABLE>
int backward(const AttnArgs& a, void* dtable, cudaStream_t s) {
  constexpr int STAGES = 2;
  using L = Layout<DP, 64, 2, STAGES>;
  const bool vec = wide_rows(a);
  attn_delta_kernel<T>
      <<<dim3((unsigned)((a.n + 7) / 8), (unsigned)((a.heads + 3) / 4)), 256, 0, s>>>(a, vec);
  SV_LAUNCH_CHECK();
  const dim3 grid(ctas_of(a, 64, WAVES), a.heads);
  size_t bytes = L::TABLE + tables(a, TABLE, false).total;
  int rc = allow_smem(attn_dkv_tc_kernel<T, DP, STAGES, TABLE>, bytes);
  if (rc != SV_OK) return rc;
  attn_dkv_tc_kernel<T, DP, STAGES, TABLE><<<grid, AT, bytes, s>>>(a, vec);
  SV_LAUNCH_CHECK();
  bytes = L::TABLE + tables(a, TABLE, TABLE).total;
  rc = allow_smem(attn_dq_tc_kernel<T, DP, STAGES, TABLE>, bytes);
  if (rc != SV_OK) return rc;
  attn_dq_tc_kernel<T, DP, STAGES, TABLE><<<grid, AT, bytes, s>>>(a, vec);
  SV_LAUNCH_CHECK();
  if constexpr (TABLE) {
    const unsigned blocks = (unsigned)((a.nb * a.nb * a.nb + 255) / 256);
    dtable_tc_finish_kernel<T><<<dim3(blocks, a.heads), 256, 0, s>>>(a, static_cast<T*>(dtable));
    SV_LAUNCH_CHECK();
  }
  return SV_OK;
}

template <typename T, bool TRAIN>
int forward_dim(const AttnArgs& a, cudaStream_t s) {
  if (a.dim <= 32) return forward<T, 32, TRAIN>(a, s);
  if (a.dim <= 64) return forward<T, 64, TRAIN>(a, s);
  return forward<T, 128, TRAIN>(a, s);
}

template <typename T>
int forward_typed(const AttnArgs& a, cudaStream_t s) {
  return a.stats || a.out_rest ? forward_dim<T, true>(a, s) : forward_dim<T, false>(a, s);
}

template <typename T>
int backward_typed(const AttnArgs& a, void* dtable, cudaStream_t s) {
  if (a.dim <= 32)
    return dtable ? backward<T, 32, true>(a, dtable, s) : backward<T, 32, false>(a, dtable, s);
  if (a.dim <= 64)
    return dtable ? backward<T, 64, true>(a, dtable, s) : backward<T, 64, false>(a, dtable, s);
  return dtable ? backward<T, 128, true>(a, dtable, s) : backward<T, 128, false>(a, dtable, s);
}

}  // namespace

// Parts of every block's positions in the forward pass. Few blocks of long windows leave CTAs idle (8,192
// rows of 6 heads x 128 in two windows are 384 blocks for 296 resident CTAs: two rounds, the second a
// third full), so the walk is split where that shortens the estimated time: rounds of CTAs, each as
// many tiles long, against a pass that joins the parts' fp32 sums. Windows of a few tiles are left
// whole. Estimates in us: a tile of 32 positions 1 + dim / 85, the join 4 and 4 MB of sums a us.
int attention_tc_parts(int64_t n, int heads, int dim, int64_t windows) {
  if (n <= 0 || heads <= 0 || windows <= 0) return 1;
  const int64_t tiles = n / windows / KB, blocks = (n / FORWARD_ROWS + 1) * heads;
  const int64_t slots = (int64_t)num_sms() * (dim <= 64 ? 3 : 2);
  const double tile_us = 1.0 + dim / 85.0, mb = 8e-6 * n * heads * dim;
  int best = 1;
  double least = 0;
  for (int parts = 1; parts <= 16 && (parts == 1 || tiles / parts >= 4); ++parts) {
    const int64_t rounds = (blocks * parts + slots - 1) / slots;
    double us = tile_us * rounds * ((tiles + parts - 1) / parts + 2);
    if (parts > 1) us += 4 + mb * parts / 4;
    if (parts == 1 || us < least) {
      least = us;
      best = parts;
    }
  }
  return mb * best > 1024 ? 1 : best;
}

int attention_tc_forward(const AttnArgs& a, bool bf16, cudaStream_t s) {
  return bf16 ? forward_typed<__nv_bfloat16>(a, s) : forward_typed<__half>(a, s);
}

int attention_tc_backward(const AttnArgs& a, bool bf16, void* dtable, cudaStream_t s) {
  return bf16 ? backward_typed<__nv_bfloat16>(a, dtable, s) : backward_typed<__half>(a, dtable, s);
}

}  // namespace sv
