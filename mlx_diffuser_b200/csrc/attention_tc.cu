// Windowed attention with a learned relative position bias in fp16 / bf16, on the 5th-generation
// tensor cores.
//
// The formulas are attention.cu's. A CTA takes 128 rows in window order (queries, or keys for dk and
// dv) of one head and walks the positions that any of their windows covers in tiles of KB: rows of
// several small windows share a tile. The scores of a tile are one product into TMEM; a thread owns a row
// of them, so the softmax needs no exchange between lanes, and writes the weights back to TMEM, where
// they are the left operand of the second product:
//   forward   S = Q K^T            o  += P V
//   dq        S = Q K^T, D = dO V^T     dq += dS K, and the table's gradient
//   dk, dv    S = K Q^T, D = V dO^T     dv += P dO, dk += dS Q   (transposed: rows are keys)
// The right operands of the second products are the tiles of the first, read along the other axis.
//
// What bounds it is the work a score needs besides the products: its bucket, the look-up, an
// exponential, the running sums, about ten instructions; the products are a tenth of that time on
// tcgen05. Fragments of warp-level mma.sync instead took 37 instructions a score for loads,
// conversions and exchanges (40,662 voxels x 768 channels, 8^3 windows, bf16: 279 us).
//
// The bucket of a pair: where the table is one entry per offset (the look-up is the identity) and
// the windows are no wider than its reach, it is linear in the coordinates and costs a subtraction;
// within the reach the look-ups of x and y are joined in one; otherwise three look-ups.
//
// Warp roles (224 threads, two CTAs an SM where shared memory and TMEM allow it):
//   warps 0-3   a row a thread: scores, softmax, score gradients, results;
//   warp 4      TMEM allocator and the tcgen05.mma issuer;
//   warps 5, 6  gather the rows of the block and of the tiles by cp.async into 128-byte-swizzled
//               panels of 64 channels, a few tiles ahead.
// Every wait is bounded (2 s, CTA abort flag); on expiry SV_DEVICE_WAIT_TIMEOUT is reported.
//
// Weights and score gradients are rounded to the feature type as operands of the second products
// (half a step each, like the stored results); the softmax sums and the table's gradient use them
// unrounded.
#include <limits.h>

#include <type_traits>

#include "attention.h"

namespace sv {
namespace {

constexpr int BQ = 128;        // rows of a block: the TMEM lanes
constexpr int AT = 224;        // threads: with seven warps a CTA, two CTAs get 128 registers a thread
constexpr int LOADERS = 64;    // of them, warps 5 and 6
constexpr int PANEL = 128;     // bytes of a row in a panel: 64 channels

enum { FWD = 0, DQ = 1, DKV = 2 };

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// max that keeps a NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}
__device__ __forceinline__ float lds_f32(uint32_t at) {
  float v;
  asm("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at));
  return v;
}
__device__ __forceinline__ uint32_t lds_u16(uint32_t at) {
  uint16_t v;
  asm("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at));
  return v;
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

__device__ __forceinline__ void arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// D[tmem] (+)= A[tmem] * B[smem]^T.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                       uint32_t more) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(more)
      : "memory");
}

// 32 lanes x 16 / 8 consecutive 32-bit columns from registers.
__device__ __forceinline__ void tmem_st_x16(uint32_t at, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0],"
      " {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_x8(uint32_t at, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(at),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]),
               "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

constexpr int CH = 16;  // columns of scores a row thread works on at a time: code that stays in the
                        // instruction cache, where whole tiles unrolled starved on fetches

template <typename T>
__device__ __forceinline__ void store_weights(uint32_t at, const float (&v)[CH]) {
  uint32_t r[CH / 2];
#pragma unroll
  for (int i = 0; i < CH / 2; ++i) r[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
  tmem_st_x8(at, r);
}

// The other side's rows of a tile, as the row threads read them.
template <int KB>
struct alignas(16) Meta {
  int32_t lin[KB];     // LINEAR: 4 ((x nb + y) nb + z)
  int2 joint[KB];      // JOINT: 2 (x width + y), 2 z
  int4 xyzr[KB];       // coordinates and row (-1: none)
  float top[KB], inv[KB], delta[KB];  // their softmax and delta (dk / dv)
  uint32_t rows[KB / 32];              // bit c: position c of 32 has a row
};

// How a pair's bucket is found; all indexes are byte offsets.
enum { GENERAL = 0, JOINT = 1, LINEAR = 2 };
constexpr int JOINT_MAX = 4096;

struct Tables {
  int grad, lut, joint, total;  // byte offsets behind the table; joint < 0: none
};
__host__ __device__ inline Tables tables(const AttnArgs& a, bool grad) {
  const int cells = a.nb * a.nb * a.nb, width = 2 * a.reach + 1;
  Tables t;
  t.grad = cells * 4;
  t.lut = t.grad + (grad ? cells * 4 : 0);
  t.joint = -1;
  t.total = t.lut + (width * 2 + 15) / 16 * 16;
  if (width * width <= JOINT_MAX) {
    t.joint = t.total;
    t.total += width * width * 2;
  }
  return t;
}

// Shared memory and TMEM of one kernel. PANELS of 64 channels a row; TILES of the block's own rows.
template <int MODE, int PANELS, int KB>
struct Plan {
  static constexpr int OWN = MODE == FWD ? 1 : 2;
  static constexpr int STAGES = MODE == FWD && PANELS == 1 ? 3 : 2;
  static constexpr int BUFS = MODE == FWD ? 2 : 1;  // score buffers in TMEM
  static constexpr int OWN_PANEL = BQ * PANEL;
  static constexpr int OWN_TILE = PANELS * OWN_PANEL;
  static constexpr int TILE_PANEL = KB * PANEL;
  static constexpr int TILE = PANELS * TILE_PANEL;
  static constexpr int RING = OWN * OWN_TILE;
  static constexpr int META = RING + STAGES * 2 * TILE;
  static constexpr int SCRATCH = META + STAGES * (int)sizeof(Meta<KB>);
  static constexpr int MISC = SCRATCH + 4 * 2 * ATTN_MAX_DIM * 4;
  static constexpr int NUM_BARS = 2 * STAGES + 3 * BUFS + 3;
  static constexpr int TABLE = (MISC + 32 + NUM_BARS * 8 + 15) / 16 * 16;
  // TMEM columns: sums, then the score buffers
  static constexpr int ACC = 64 * PANELS;
  static constexpr int SCORES = (MODE == DKV ? 2 : 1) * ACC;
  // A buffer: S and, forward, the weights beside it (a tile may be done again with another base);
  // else S and D, whose weights and gradients take their place as they are read.
  static constexpr int SCORE_COLS = MODE == FWD ? KB + KB / 2 : 2 * KB;
  static constexpr int WEIGHTS = MODE == FWD ? KB : 0;
  static constexpr int USED = SCORES + BUFS * SCORE_COLS;
  static constexpr int COLS = USED <= 256 ? 256 : 512;
  static_assert(USED <= 512, "TMEM columns");
  static constexpr int CTAS = COLS == 256 ? 2 : 1;
};

// A row thread's own row and how it finds buckets.
struct Own {
  PlanRow p;
  int lin, joint_xy, joint_z;
};

struct Look {
  uint32_t table, lut, joint;  // shared-memory addresses
  int nb, reach, mode;
  uint32_t top, joint_top, z_top;  // largest byte offsets
};

__device__ __forceinline__ uint32_t bucket3(const Look& l, int qx, int qy, int qz, int kx, int ky,
                                            int kz) {
  const int R = l.reach;
  const int x = lds_u16(l.lut + 2 * (max(-R, min(R, sub_sat(kx, qx))) + R));
  const int y = lds_u16(l.lut + 2 * (max(-R, min(R, sub_sat(ky, qy))) + R));
  const int z = lds_u16(l.lut + 2 * (max(-R, min(R, sub_sat(kz, qz))) + R));
  return (uint32_t)((x * l.nb + y) * l.nb + z);
}

// The pairs' byte offsets in the table for the CH columns c0 .. of a tile. FLIP: the thread's row is
// the key and the columns are queries. Outside a window (masked later) they are clamped; inside, the
// clamp changes nothing.
template <bool FLIP, int KB>
__device__ __forceinline__ void buckets(const Look& l, const Meta<KB>& m, const Own& o, int c0,
                                        uint32_t (&at)[CH]) {
  if (l.mode == LINEAR) {
#pragma unroll
    for (int c = 0; c < CH; c += 4) {
      const int4 k = *reinterpret_cast<const int4*>(&m.lin[c0 + c]);
      const int v[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        at[c + e] = min((uint32_t)(FLIP ? o.lin - v[e] : v[e] - o.lin), l.top);
    }
  } else if (l.mode == JOINT) {
#pragma unroll
    for (int c = 0; c < CH; c += 2) {
      const int4 k = *reinterpret_cast<const int4*>(&m.joint[c0 + c]);
      const int xy[2] = {k.x, k.z}, z[2] = {k.y, k.w};
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t dxy = (uint32_t)(FLIP ? o.joint_xy - xy[e] : xy[e] - o.joint_xy);
        const uint32_t dz = (uint32_t)(FLIP ? o.joint_z - z[e] : z[e] - o.joint_z);
        at[c + e] = lds_u16(l.joint + min(dxy, l.joint_top)) + lds_u16(l.lut + min(dz, l.z_top));
      }
    }
  } else {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int4 k = m.xyzr[c0 + c];
      at[c] = FLIP ? bucket3(l, k.x, k.y, k.z, o.p.x, o.p.y, o.p.z)
                   : bucket3(l, o.p.x, o.p.y, o.p.z, k.x, k.y, k.z);
    }
  }
}

// Bits of the CH columns c0 .. that a row with columns lo .. hi - 1 in its window sees.
constexpr uint32_t ALL_SEEN = (1u << CH) - 1u;
__device__ __forceinline__ uint32_t seen_bits(int lo, int hi, int c0) {
  const int l = max(0, min(CH, lo - c0)), h = max(0, min(CH, hi - c0));
  return ((1u << h) - 1u) & ~((1u << l) - 1u);
}

template <typename T>
__device__ __noinline__ void again_forward(AttnArgs a, int64_t p, int h, float* s) {
  row_forward<T, true>(a, p, h, s);
}
template <typename T>
__device__ __noinline__ void again_dq(AttnArgs a, int64_t p, int h, float* s) {
  row_dq<T, true, false>(a, p, h, s);
}
template <typename T>
__device__ __noinline__ void again_dkv(AttnArgs a, int64_t p, int h, float* s) {
  row_dkv<T, true>(a, p, h, s);
}

// The table's gradient in fixed point: a score gradient is at most 2^17 units (the head's largest is
// known from the dk / dv pass), and sums to a 32-bit word per bucket in shared memory. A thread
// counts the units it has added; its warp moves the words into the 64-bit sums in global memory
// before the count can pass 2^24, so the 128 threads cannot overflow a word. INT_MAX when a score
// gradient was not finite.
constexpr int UNIT_BITS = 17;
__device__ __forceinline__ int unit_exponent(const AttnArgs& a, int head) {
  const float top = __uint_as_float(a.norms[2 * head]);
  if (!(top < INFINITY)) return INT_MAX;
  if (top == 0.f) return 0;
  int e;
  frexpf(top, &e);                      // top < 2^e
  return min(UNIT_BITS - 1 - e, 120);   // the two passes round their products differently
}

// The running maximum of the softmax is only kept within this many powers of two: a row starts with
// a base of 0, and its sums are rescaled (and the tile done again) when a score passes the base by
// more, or when the first scores it sees are all that far below. Weights are then between 2^-8 and 2^8 of
// the usual ones, which neither type nor the fp32 sums notice.
constexpr float SLACK = 8.f;

// Range of positions that the block's rows see: by every warp for itself, from the plan.
struct Range {
  int lo, tiles;
};
template <int KB>
__device__ __forceinline__ Range block_range(const AttnArgs& a, int64_t p0) {
  const int lane = threadIdx.x & 31;
  int lo = INT_MAX, hi = INT_MIN;
#pragma unroll
  for (int i = 0; i < BQ / 32; ++i) {
    const int64_t p = p0 + lane + 32 * i;
    if (p < a.n) {
      const int4 r = __ldg(reinterpret_cast<const int4*>(a.plan + p) + 1);  // start, end, span
      if (__ldg(&a.plan[p].row) >= 0) {
        lo = min(lo, r.x);
        hi = max(hi, r.y);
      }
    }
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  return Range{lo, hi > lo ? (hi - lo + KB - 1) / KB : 0};
}

template <typename T, int MODE, int PANELS, int KB, bool TABLE>
__global__ void __launch_bounds__(AT, Plan<MODE, PANELS, KB>::CTAS)
    attn_tc_kernel(AttnArgs a, int per_cta, bool vec, int32_t* status) {
  using P = Plan<MODE, PANELS, KB>;
  constexpr int ST = P::STAGES, NB = P::BUFS;
  constexpr bool kBF16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  Meta<KB>* metas = reinterpret_cast<Meta<KB>*>(smem + P::META);
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(smem + P::MISC);
  volatile int* s_abort = reinterpret_cast<volatile int*>(smem + P::MISC + 4);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + P::MISC + 32);  // a tile has landed
  uint64_t* empty = full + ST;        // a tile's products are done
  uint64_t* s_full = empty + ST;      // scores are in TMEM
  uint64_t* p_full = s_full + NB;     // weights are in TMEM
  uint64_t* acc_done = p_full + NB;   // a tile's second products are done (one a buffer: a wait by
                                      // parity tells a phase from the next only)
  uint64_t* acc_free = acc_done + NB;  // the block's results have been read
  uint64_t* own_full = acc_free + 1;
  uint64_t* own_empty = own_full + 1;
  const Tables tb = tables(a, TABLE && MODE == DQ);
  float* table = reinterpret_cast<float*>(smem + P::TABLE);
  int* s_grad = reinterpret_cast<int*>(smem + P::TABLE + tb.grad);
  uint16_t* lut = reinterpret_cast<uint16_t*>(smem + P::TABLE + tb.lut);
  uint16_t* joint =
      tb.joint < 0 ? nullptr : reinterpret_cast<uint16_t*>(smem + P::TABLE + tb.joint);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int head = blockIdx.y;
  const int cells = a.nb * a.nb * a.nb, width = 2 * a.reach + 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(&full[s], 2 * LOADERS);  // each loader: its copies, and its plain stores
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < NB; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&p_full[s], 4);
      mbar_init(&acc_done[s], 1);
    }
    mbar_init(acc_free, 4);
    mbar_init(own_full, 2 * LOADERS);
    mbar_init(own_empty, 1);
    *s_abort = 0;
    fence_mbar_init();
  }
  if (warp == 4) {
    tmem_alloc(s_tmem, P::COLS);
    tmem_relinquish();
  }
  {
    const T* src = static_cast<const T*>(a.table) + (int64_t)head * cells;
#pragma unroll 4
    for (int i = threadIdx.x; i < cells; i += AT) table[i] = times_log2e(to_f32(src[i]));
    if constexpr (TABLE && MODE == DQ)
      for (int i = threadIdx.x; i < cells; i += AT) s_grad[i] = 0;
  }
  bool same = a.nb == width;
  for (int i = threadIdx.x; i < width; i += AT) {
    const int v = max(0, min(a.nb - 1, __ldg(a.lut + i)));
    lut[i] = (uint16_t)(4 * v);
    same = same && v == i;
  }
  tc_fence_before();
  const bool identity = __syncthreads_and(same);
  tc_fence_after();
  if (!identity && joint != nullptr) {
    for (int i = threadIdx.x; i < width * width; i += AT)
      joint[i] = (uint16_t)((lut[i / width] * a.nb + lut[i % width]) * a.nb);
    __syncthreads();
  }
  const uint32_t tmem = *s_tmem;
  const int64_t blocks = (a.n + BQ - 1) / BQ;
  const int64_t first = (int64_t)blockIdx.x * per_cta;
  const int64_t last = first + per_cta < blocks ? first + per_cta : blocks;
  const int ksteps = (a.dim + 15) / 16;  // of 16 channels
  bool ok = true;

  if (warp >= 5) {
    // ---- loaders ----
    const int tid = threadIdx.x - 160;
    const T* q = static_cast<const T*>(a.q) + head * a.q_head;
    const T* k = static_cast<const T*>(a.k) + head * a.k_head;
    const T* v = static_cast<const T*>(a.v) + head * a.v_head;
    const T* g = static_cast<const T*>(a.dout) + (int64_t)head * a.dim;
    const int g_row = a.heads * a.dim;
    const T* own0 = MODE == DKV ? k : q;
    const T* own1 = MODE == DKV ? v : g;
    const int own0_row = (int)(MODE == DKV ? a.k_row : a.q_row);
    const int own1_row = MODE == DKV ? (int)a.v_row : g_row;
    const T* tile0 = MODE == DKV ? q : k;
    const T* tile1 = MODE == DKV ? g : v;
    const int tile0_row = (int)(MODE == DKV ? a.q_row : a.k_row);
    const int tile1_row = MODE == DKV ? g_row : (int)a.v_row;
    const int chunks = 2 * ksteps;  // 16-byte pieces of a row that the products read
    // Rows p .. p + ROWS - 1 (positions below `end`) of one or two tensors. A thread takes one piece
    // of every (128 / PIECES)th row.
    constexpr int PIECES = 8 * PANELS;
    auto gather = [&](uint8_t* dst0, uint8_t* dst1, const T* src0, const T* src1, int row0, int row1,
                      int64_t p, int64_t end, auto rows_c) {
      constexpr int ROWS = decltype(rows_c)::value;
      constexpr int STEP = LOADERS / PIECES;
      const int c = tid % PIECES;
      const uint32_t panel = (uint32_t)(c / 8) * (ROWS * PANEL);
      int32_t idx[ROWS / STEP];
#pragma unroll
      for (int i = 0; i < ROWS / STEP; ++i) {
        const int64_t at = p + tid / PIECES + i * STEP;
        idx[i] = at < end ? __ldg(&a.plan[at].row) : -1;
      }
      if (c < chunks) {
#pragma unroll
        for (int i = 0; i < ROWS / STEP; ++i) {
          const int r = tid / PIECES + i * STEP;
          const uint32_t at = panel + r * PANEL + (((c & 7) ^ (r & 7)) << 4);
          const int64_t row = max(idx[i], 0);
          if (vec) {
            const bool in = idx[i] >= 0 && c * 8 < a.dim;
            const int from = in ? c * 8 : 0;
            cp_async_16(smem_u32(dst0) + at, src0 + row * row0 + from, in ? 16u : 0u);
            if (dst1) cp_async_16(smem_u32(dst1) + at, src1 + row * row1 + from, in ? 16u : 0u);
          } else {
            for (int d = 0; d < (dst1 ? 2 : 1); ++d) {
              T e[8];
#pragma unroll
              for (int x = 0; x < 8; ++x) {
                e[x] = from_f32<T>(0.f);
                if (idx[i] >= 0 && c * 8 + x < a.dim)
                  e[x] = d ? src1[row * row1 + c * 8 + x] : src0[row * row0 + c * 8 + x];
              }
              *reinterpret_cast<uint4*>((d ? dst1 : dst0) + at) = *reinterpret_cast<uint4*>(e);
            }
          }
        }
      }
    };
    // Arrives for the copies when they land, and for the plain stores now.
    auto landed = [](uint64_t* bar) {
      fence_proxy_async_smem();
      cp_async_arrive_noinc(bar);
      arrive(bar);
    };
    int it = 0, local = 0;
    float delta_top = 0.f;
    for (int64_t block = first; block < last && ok; ++block, ++local) {
      const Range range = block_range<KB>(a, block * BQ);
      if (!mbar_wait_bounded(own_empty, (local & 1) ^ 1, s_abort)) {
        ok = false;
        break;
      }
      gather(smem, P::OWN == 2 ? smem + P::OWN_TILE : nullptr, own0, own1, own0_row, own1_row,
             block * BQ, a.n, std::integral_constant<int, BQ>{});
      landed(own_full);
      for (int t = 0; t < range.tiles; ++t, ++it) {
        const int s = it % ST;
        const int64_t p0 = (int64_t)range.lo + t * KB;
        const int64_t end = min(a.n, p0 + KB);
        if (!mbar_wait_bounded(&empty[s], ((it / ST) & 1) ^ 1, s_abort)) {
          ok = false;
          break;
        }
        uint8_t* dst = smem + P::RING + s * 2 * P::TILE;
        gather(dst, dst + P::TILE, tile0, tile1, tile0_row, tile1_row, p0, end,
               std::integral_constant<int, KB>{});
        if (tid < KB) {
          Meta<KB>& m = metas[s];
          int4 r = make_int4(0, 0, 0, -1);
          if (p0 + tid < end) r = __ldg(reinterpret_cast<const int4*>(a.plan + p0 + tid));
          m.xyzr[tid] = r;
          m.lin[tid] = (int)((((unsigned)r.x * a.nb + (unsigned)r.y) * a.nb + (unsigned)r.z) * 4u);
          m.joint[tid] = make_int2((int)(((unsigned)r.x * width + (unsigned)r.y) * 2u),
                                   (int)((unsigned)r.z * 2u));
          if constexpr (MODE == DKV) {
            float2 st = make_float2(0.f, 0.f);
            float d = 0.f;
            if (r.w >= 0) {
              st = a.stats[head * a.n + p0 + tid];
              d = a.delta[head * a.n + p0 + tid];
            }
            m.top[tid] = st.x;
            m.inv[tid] = st.y;
            m.delta[tid] = d;
            delta_top = max_nan(delta_top, fabsf(d));
          }
          const unsigned rows = __ballot_sync(0xffffffffu, r.w >= 0);
          if (lane == 0) m.rows[tid / 32] = rows;
        }
        landed(&full[s]);
      }
    }
    if (!ok) report(status, SV_DEVICE_WAIT_TIMEOUT);
    cp_async_wait_all();
    if constexpr (MODE == DKV && TABLE) {
      // The two passes round dp - delta differently, by up to 2^-17 |delta| or so; a head whose score
      // gradients are nothing but that must not get a unit so small that the other pass overflows it.
      const unsigned top =
          __reduce_max_sync(0xffffffffu, __float_as_uint(delta_top * 0x1p-14f) & 0x7fffffffu);
      if (lane == 0 && top) atomicMax(a.norms + 2 * head, top);
    }
  } else if (warp == 4) {
    // ---- products ----
    const uint32_t id_nt = idesc_f16(kBF16, BQ, KB);
    const uint32_t id_nn = idesc_f16_major(kBF16, BQ, 16 * ksteps, false, true);
    int it = 0, local = 0;
    for (int64_t block = first; block < last && ok; ++block, ++local) {
      const Range range = block_range<KB>(a, block * BQ);
      if (lane == 0) {
        const uint32_t own = smem_u32(smem);
        auto stage = [&](int i) { return smem_u32(smem + P::RING + (i % ST) * 2 * P::TILE); };
        // Scores of tile i: A = the block's rows, B = the tile's, both along the channels. `after`:
        // the tile of the block whose weights were in the buffer, to be multiplied first (-1: none).
        auto scores = [&](int i, int after) {
          if (!mbar_wait_bounded(&full[i % ST], (i / ST) & 1, s_abort)) return false;
          if (after >= 0 &&
              !mbar_wait_bounded(&acc_done[after % NB], (after / NB) & 1, s_abort))
            return false;
          tc_fence_after();
          fence_proxy_async_smem();
          const uint32_t d = tmem + P::SCORES + (i % NB) * P::SCORE_COLS;
          for (int x = 0; x < (MODE == FWD ? 1 : 2); ++x) {
            for (int j = 0; j < ksteps; ++j) {
              const uint32_t at = (j % 4) * 32;
              tc_mma_f16(d + x * KB,
                         smem_desc_sw128(own + x * P::OWN_TILE + (j / 4) * P::OWN_PANEL + at),
                         smem_desc_sw128(stage(i) + x * P::TILE + (j / 4) * P::TILE_PANEL + at),
                         id_nt, j > 0);
            }
          }
          tc_commit(&s_full[i % NB]);
          return true;
        };
        if (range.tiles > 0) {
          ok = mbar_wait_bounded(own_full, local & 1, s_abort) &&
               (local == 0 || mbar_wait_bounded(acc_free, (local - 1) & 1, s_abort));
          if (ok) ok = scores(it, -1);
        }
        for (int t = 0; t < range.tiles && ok; ++t) {
          const int i = it + t;
          if (NB == 2 && t + 1 < range.tiles && !(ok = scores(i + 1, t > 0 ? i - 1 : -1))) break;
          if (!(ok = mbar_wait_bounded(&p_full[i % NB], (i / NB) & 1, s_abort))) break;
          tc_fence_after();
          const uint32_t s = tmem + P::SCORES + (i % NB) * P::SCORE_COLS;
          // sums += weights x tile, the tile read along its rows
          for (int j = 0; j < KB / 16; ++j) {
            auto tile = [&](int x) {
              return smem_desc_mn_sw128(stage(i) + x * P::TILE + j * 16 * PANEL, P::TILE_PANEL,
                                        8 * PANEL);
            };
            const uint32_t more = t > 0 || j > 0;
            if constexpr (MODE == FWD) mma_ts(tmem, s + P::WEIGHTS + j * 8, tile(1), id_nn, more);
            if constexpr (MODE == DQ) mma_ts(tmem, s + j * 8, tile(0), id_nn, more);
            if constexpr (MODE == DKV) {
              mma_ts(tmem, s + KB + j * 8, tile(0), id_nn, more);      // dk += dS Q
              mma_ts(tmem + P::ACC, s + j * 8, tile(1), id_nn, more);  // dv += P dO
            }
          }
          tc_commit(&empty[i % ST]);
          tc_commit(&acc_done[i % NB]);
          if (t + 1 == range.tiles) tc_commit(own_empty);
          if (NB == 1 && t + 1 < range.tiles && !(ok = scores(i + 1, i))) break;
        }
        if (range.tiles == 0) {
          // nothing reads the block's rows; keep the barriers' phases in step
          ok = mbar_wait_bounded(own_full, local & 1, s_abort) &&
               (local == 0 || mbar_wait_bounded(acc_free, (local - 1) & 1, s_abort));
          arrive(own_empty);
        }
      }
      ok = __all_sync(0xffffffffu, ok);
      it += range.tiles;
    }
    if (lane == 0) {
      // The last commit's arrival, and after a wait that ran out the products in flight, use this
      // CTA's shared memory and TMEM: let them finish.
      if (ok) ok = mbar_wait_bounded(own_empty, (local - 1) & 1, s_abort);
      if (!ok) {
        report(status, SV_DEVICE_WAIT_TIMEOUT);
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 10000000ull) {
        }
      }
    }
  } else {
    // ---- a row a thread ----
    const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
    float* scratch = reinterpret_cast<float*>(smem + P::SCRATCH) + warp * 2 * ATTN_MAX_DIM;
    const float scale = a.scale * ATTN_LOG2E;
    Look look{smem_u32(table), smem_u32(lut), joint ? smem_u32(joint) : 0u, a.nb, a.reach, GENERAL,
              (uint32_t)cells * 4u - 4u, (uint32_t)(width * width) * 2u - 2u,
              (uint32_t)width * 2u - 2u};
    const uint32_t grads = smem_u32(s_grad);
    const int exponent = TABLE && MODE == DQ ? unit_exponent(a, head) : INT_MAX;
    const float unit = exponent == INT_MAX ? 0.f : ldexpf(1.f, exponent);
    constexpr float LIMIT = 16777216.f - CH * (float)(1 << UNIT_BITS);  // CH pairs between checks
    float spent = 0.f;  // sum of |dS| since this warp emptied the words
    float most = 0.f;
    auto flush = [&] {
      for (int i = lane; i < cells; i += 32) {
        const int add = atomicExch(s_grad + i, 0);
        if (add != 0)
          atomicAdd(a.dtable + (int64_t)head * cells + i, (unsigned long long)(long long)add);
      }
      spent = 0.f;
    };
    auto wait = [&](uint64_t* bar, int phase) {
      return (bool)__all_sync(0xffffffffu, mbar_wait_bounded(bar, phase & 1, s_abort));
    };
    int it = 0;
    for (int64_t block = first; block < last && ok; ++block) {
      const Range range = block_range<KB>(a, block * BQ);
      const int64_t pos = block * BQ + warp * 32 + lane;
      Own own;
      own.p = PlanRow{};
      own.p.row = -1;
      if (pos < a.n) own.p = plan_at(a.plan, pos);
      const bool live = own.p.row >= 0;
      if (!live) own.p.start = own.p.end = 0;
      const bool narrow = __all_sync(0xffffffffu, !live || own.p.span <= a.reach);
      look.mode = !narrow ? GENERAL : (identity ? LINEAR : (joint ? JOINT : GENERAL));
      // the middle of the tables is folded into the row's side
      const int sign = MODE == DKV ? 1 : -1;
      own.lin = (int)((((unsigned)own.p.x * a.nb + (unsigned)own.p.y) * a.nb + (unsigned)own.p.z) *
                      4u) + sign * (int)(look.top / 2);
      own.joint_xy = (int)(((unsigned)own.p.x * width + (unsigned)own.p.y) * 2u) +
                     sign * (int)(look.joint_top / 2);
      own.joint_z = (int)((unsigned)own.p.z * 2u) + sign * 2 * a.reach;
      float base = 0.f, sum = 0.f;                     // forward
      bool fresh = true;                               // no score seen yet
      float top = 0.f, inv = 0.f, shift = 0.f;         // dq
      if constexpr (MODE == DQ) {
        if (live) {
          const float2 st = a.stats[head * a.n + pos];
          top = st.x;
          inv = st.y;
          shift = -st.y * a.delta[head * a.n + pos];
        }
      }
      for (int t = 0; t < range.tiles && ok; ++t, ++it) {
        const int p0 = range.lo + t * KB;
        const int buf = it % NB;
        const Meta<KB>& m = metas[it % ST];
        const uint32_t at = lanes + P::SCORES + buf * P::SCORE_COLS;
        if (!wait(&full[it % ST], it / ST) || !wait(&s_full[buf], it / NB)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const int lo = own.p.start - p0, hi = own.p.end - p0;
        // Bits of the columns c0 .. that the row sees.
        auto seen_at = [&](int c0) {
          return seen_bits(lo, hi, c0) & (m.rows[c0 / 32] >> (c0 % 32));
        };
        if constexpr (MODE == FWD) {
          for (bool again = false;; again = true) {
            float high = -INFINITY, part = 0.f;
#pragma unroll 1
            for (int c0 = 0; c0 < KB; c0 += CH) {
              const uint32_t seen = seen_at(c0);
              float v[CH];
              if (!__any_sync(0xffffffffu, seen)) {
#pragma unroll
                for (int c = 0; c < CH; ++c) v[c] = 0.f;
              } else {
                uint32_t r[CH], off[CH];
                tmem_ld_32x32b_x16(at + c0, r);
                buckets<false>(look, m, own, c0, off);
                tc_wait_ld();
#pragma unroll
                for (int c = 0; c < CH; ++c)
                  v[c] = fmaf(__uint_as_float(r[c]), scale, lds_f32(look.table + off[c]));
                if (!__all_sync(0xffffffffu, seen == ALL_SEEN)) {
#pragma unroll
                  for (int c = 0; c < CH; ++c)
                    if (!(seen & (1u << c))) v[c] = -INFINITY;
                }
#pragma unroll
                for (int c = 0; c < CH; c += 2) high = fmaxf(high, fmaxf(v[c], v[c + 1]));
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                  v[c] = exp2_fast(v[c] - base);
                  part += v[c];
                }
              }
              __syncwarp();
              store_weights<T>(at + P::WEIGHTS + c0 / 2, v);
            }
            const bool off_base =
                high > base + SLACK || (fresh && high > -INFINITY && high < base - SLACK);
            if (again || !__any_sync(0xffffffffu, off_base)) {
              sum += part;
              fresh = fresh && high == -INFINITY;
              break;
            }
            // lanes whose base stays keep it: their weights come out the same again
            const float keep = off_base ? exp2_fast(base - high) : 1.f;
            if (off_base) base = high;
            sum = fresh ? 0.f : sum * keep;
            if (t > 0) {
              if (!wait(&acc_done[(it - 1) % NB], (it - 1) / NB)) {
                ok = false;
                break;
              }
              tc_fence_after();
              for (int c = 0; c < 16 * ksteps; c += 16) {
                uint32_t r[16];
                tmem_ld_32x32b_x16(lanes + c, r);
                tc_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i)
                  r[i] = fresh ? 0u : __float_as_uint(__uint_as_float(r[i]) * keep);
                tmem_st_x16(lanes + c, r);
              }
            }
            tmem_wait_st();
          }
          if (!ok) break;
        } else {
#pragma unroll 1
          for (int c0 = 0; c0 < KB; c0 += CH) {
            const uint32_t seen = seen_at(c0);
            float s[CH], d[CH];
            if (!__any_sync(0xffffffffu, seen)) {
#pragma unroll
              for (int c = 0; c < CH; ++c) s[c] = d[c] = 0.f;
            } else {
              uint32_t rs[CH], rd[CH], off[CH];
              tmem_ld_32x32b_x16(at + c0, rs);
              tmem_ld_32x32b_x16(at + KB + c0, rd);
              buckets<MODE == DKV>(look, m, own, c0, off);
              tc_wait_ld();
#pragma unroll
              for (int c = 0; c < CH; ++c) {
                s[c] = fmaf(__uint_as_float(rs[c]), scale, lds_f32(look.table + off[c]));
                d[c] = __uint_as_float(rd[c]);
              }
              const bool whole = __all_sync(0xffffffffu, seen == ALL_SEEN);
              if constexpr (MODE == DQ) {
#pragma unroll
                for (int c = 0; c < CH; ++c)
                  s[c] = exp2_fast(s[c] - top) * fmaf(d[c], inv, shift);
                if (!whole) {
#pragma unroll
                  for (int c = 0; c < CH; ++c)
                    if (!(seen & (1u << c))) s[c] = 0.f;
                }
                if constexpr (TABLE) {
#pragma unroll
                  for (int c = 0; c < CH; ++c) {
                    spent += fabsf(s[c]);
                    // 1.5 * 2^23: the sum's low bits are the rounded integer
                    const float f = fmaf(s[c], unit, 12582912.f);
                    const int add = __float_as_int(f) - 0x4b400000;
                    if (add != 0)
                      asm volatile("red.shared.add.s32 [%0], %1;" ::"r"(grads + off[c]), "r"(add)
                                   : "memory");
                  }
                }
              } else {
#pragma unroll
                for (int c = 0; c < CH; c += 4) {
                  const float4 tp = *reinterpret_cast<const float4*>(&m.top[c0 + c]);
                  const float4 iv = *reinterpret_cast<const float4*>(&m.inv[c0 + c]);
                  const float4 dl = *reinterpret_cast<const float4*>(&m.delta[c0 + c]);
                  const float tops[4] = {tp.x, tp.y, tp.z, tp.w}, invs[4] = {iv.x, iv.y, iv.z, iv.w},
                              dels[4] = {dl.x, dl.y, dl.z, dl.w};
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    s[c + e] = exp2_fast(s[c + e] - tops[e]) * invs[e];
                    d[c + e] -= dels[e];
                  }
                }
                if (!whole) {  // another window's row may hold anything
#pragma unroll
                  for (int c = 0; c < CH; ++c)
                    if (!(seen & (1u << c))) s[c] = d[c] = 0.f;
                }
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                  d[c] *= s[c];
                  if constexpr (TABLE) most = max_nan(most, fabsf(d[c]));
                }
              }
            }
            __syncwarp();
            store_weights<T>(at + c0 / 2, s);
            if constexpr (MODE == DKV) store_weights<T>(at + KB + c0 / 2, d);
            if constexpr (TABLE && MODE == DQ) {
              if (__any_sync(0xffffffffu, spent * unit > LIMIT)) flush();
            }
          }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive(&p_full[buf]);
      }
      if (!ok) break;
      // ---- results ----
      if (range.tiles > 0) {
        if (!wait(&acc_done[(it - 1) % NB], (it - 1) / NB)) {
          ok = false;
          break;
        }
        tc_fence_after();
      }
      float by = a.scale;  // dq, dk
      if constexpr (MODE == FWD) {
        const float2 st = row_stats(base, sum);
        by = st.y;
        if (a.stats && live) a.stats[head * a.n + pos] = st;
      }
      bool finite = true;
      const int64_t out_row = ((int64_t)max(own.p.row, 0) * a.heads + head) * a.dim;
#pragma unroll 1
      for (int x = 0; x < (MODE == DKV ? 2 : 1); ++x) {
        T* out = static_cast<T*>(MODE == FWD ? a.out : MODE == DQ ? a.dq : x ? a.dv : a.dk);
        const float f = MODE == DKV && x ? 1.f : by;
#pragma unroll 1
        for (int c = 0; c < 16 * ksteps && range.tiles > 0; c += 16) {
          uint32_t r[16];
          __syncwarp();  // lanes without a row skip the rest of a round
          tmem_ld_32x32b_x16(lanes + x * P::ACC + c, r);
          tc_wait_ld();
          if (!live) continue;
          float o[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            o[i] = __uint_as_float(r[i]) * f;
            finite = finite && fabsf(o[i]) < INFINITY;
          }
          T* dst = out + out_row + c;
          if (vec) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
              if (c + 8 * i < a.dim)
                reinterpret_cast<uint4*>(dst)[i] =
                    make_uint4(pack2<T>(o[8 * i], o[8 * i + 1]), pack2<T>(o[8 * i + 2], o[8 * i + 3]),
                               pack2<T>(o[8 * i + 4], o[8 * i + 5]),
                               pack2<T>(o[8 * i + 6], o[8 * i + 7]));
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (c + i < a.dim) dst[i] = from_f32<T>(o[i]);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive(acc_free);
      // A weight of zero does not hide a NaN or an infinity that another window's row brings into a
      // tile, and fp16 score gradients can overflow where their sums do not. So rows that come out
      // not finite are computed again, one at a time, from their own windows alone.
      unsigned redo = __ballot_sync(0xffffffffu, live && !finite);
      while (redo) {  // the same in all lanes
        const int64_t p = block * BQ + warp * 32 + __ffs(redo) - 1;
        redo &= redo - 1;
        __syncwarp();
        if constexpr (MODE == FWD) again_forward<T>(a, p, head, scratch);
        if constexpr (MODE == DQ) again_dq<T>(a, p, head, scratch);
        if constexpr (MODE == DKV) again_dkv<T>(a, p, head, scratch);
      }
    }
    if (!ok) report(status, SV_DEVICE_WAIT_TIMEOUT);
    if constexpr (TABLE && MODE == DKV) {
      // bits of non-negative numbers order like the numbers, a NaN's above all
      const unsigned high = __reduce_max_sync(0xffffffffu, __float_as_uint(most) & 0x7fffffffu);
      if (lane == 0 && high) atomicMax(a.norms + 2 * head, high);
    }
    if constexpr (TABLE && MODE == DQ) flush();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 4) {
    tc_fence_after();
    tmem_dealloc(tmem, P::COLS);
  }
}

// delta_i = dout_i . o_i by position: eight lanes a row and head.
template <typename T>
__global__ void __launch_bounds__(256) attn_delta_kernel(AttnArgs a, bool vec) {
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) / 8;  // head * n + position
  const int sub = threadIdx.x & 7;
  float d = 0.f;
  if (at < a.n * a.heads) {
    const int64_t h = at / a.n, p = at - h * a.n;
    const int32_t row = __ldg(&a.plan[p].row);
    if (row >= 0) {
      const int64_t from = ((int64_t)row * a.heads + h) * a.dim;
      const T* g = static_cast<const T*>(a.dout) + from;
      const T* o = static_cast<const T*>(a.o) + from;
      if (vec) {
        for (int c = sub * 8; c < a.dim; c += 64) {
          const uint4 x = *reinterpret_cast<const uint4*>(g + c);
          const uint4 y = *reinterpret_cast<const uint4*>(o + c);
          const T* xe = reinterpret_cast<const T*>(&x);
          const T* ye = reinterpret_cast<const T*>(&y);
#pragma unroll
          for (int k = 0; k < 8; ++k) d = fmaf(to_f32(xe[k]), to_f32(ye[k]), d);
        }
      } else {
        for (int c = sub; c < a.dim; c += 8) d = fmaf(to_f32(g[c]), to_f32(o[c]), d);
      }
    }
  }
#pragma unroll
  for (int s = 4; s > 0; s >>= 1) d += __shfl_xor_sync(0xffffffffu, d, s);
  if (sub == 0 && at < a.n * a.heads) a.delta[at] = d;
}

template <typename T>
__global__ void __launch_bounds__(256) dtable_tc_finish_kernel(AttnArgs a, T* __restrict__ out) {
  const int cells = a.nb * a.nb * a.nb;
  const int h = blockIdx.y;
  const int exponent = unit_exponent(a, h);
  for (int b = blockIdx.x * 256 + threadIdx.x; b < cells; b += gridDim.x * 256) {
    const int64_t at = (int64_t)h * cells + b;
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
         wide(a.v, a.v_row, a.v_head) && wide(a.out, row, head) && wide(a.dout, row, head) &&
         wide(a.dq, row, head) && wide(a.dk, row, head) && wide(a.dv, row, head);
}

// Blocks of one head that a CTA takes in turn, so that it stages the table (and adds up its gradient)
// once: as many as still leave `waves` CTAs for each SM.
int blocks_per_cta(const AttnArgs& a, int waves) {
  const int64_t blocks = (a.n + BQ - 1) / BQ;
  const int64_t per = blocks * a.heads / ((int64_t)num_sms() * waves);
  return (int)(per < 1 ? 1 : (per > 16 ? 16 : per));
}

template <typename K>
int allow_smem(K kernel, size_t bytes) {
  SV_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   (int)bytes));
  return SV_OK;
}

template <typename T, int MODE, int PANELS, bool TABLE>
int launch(const AttnArgs& a, int32_t* status, cudaStream_t s) {
  constexpr int KB = PANELS == 1 ? 64 : 32;  // positions of a tile: two CTAs fit an SM
  auto kernel = attn_tc_kernel<T, MODE, PANELS, KB, TABLE>;
  const size_t bytes =
      Plan<MODE, PANELS, KB>::TABLE + tables(a, TABLE && MODE == DQ).total + 1024;
  const int rc = allow_smem(kernel, bytes);
  if (rc != SV_OK) return rc;
  const int per = blocks_per_cta(a, MODE == FWD ? 8 : 8);
  const int64_t ctas = ((a.n + BQ - 1) / BQ + per - 1) / per;
  kernel<<<dim3((unsigned)ctas, a.heads), AT, bytes, s>>>(a, per, wide_rows(a), status);
  SV_LAUNCH_CHECK();
  return SV_OK;
}

template <typename T, int PANELS, bool TABLE>
int backward(const AttnArgs& a, void* dtable, int32_t* status, cudaStream_t s) {
  attn_delta_kernel<T><<<(unsigned)((a.n * a.heads + 31) / 32), 256, 0, s>>>(
      a, wide_rows(a) && aligned16(a.o));
  SV_LAUNCH_CHECK();
  int rc = launch<T, DKV, PANELS, TABLE>(a, status, s);
  if (rc == SV_OK) rc = launch<T, DQ, PANELS, TABLE>(a, status, s);
  if (rc != SV_OK) return rc;
  if constexpr (TABLE) {
    const unsigned blocks = (unsigned)((a.nb * a.nb * a.nb + 255) / 256);
    dtable_tc_finish_kernel<T><<<dim3(blocks, a.heads), 256, 0, s>>>(a, static_cast<T*>(dtable));
    SV_LAUNCH_CHECK();
  }
  return SV_OK;
}

template <typename T>
int forward_typed(const AttnArgs& a, int32_t* status, cudaStream_t s) {
  return a.dim <= 64 ? launch<T, FWD, 1, false>(a, status, s)
                     : launch<T, FWD, 2, false>(a, status, s);
}

template <typename T>
int backward_typed(const AttnArgs& a, void* dtable, int32_t* status, cudaStream_t s) {
  if (a.dim <= 64)
    return dtable ? backward<T, 1, true>(a, dtable, status, s)
                  : backward<T, 1, false>(a, dtable, status, s);
  return dtable ? backward<T, 2, true>(a, dtable, status, s)
                : backward<T, 2, false>(a, dtable, status, s);
}

}  // namespace

int attention_tc_forward(const AttnArgs& a, bool bf16, int32_t* status, cudaStream_t s) {
  return bf16 ? forward_typed<__nv_bfloat16>(a, status, s) : forward_typed<__half>(a, status, s);
}

int attention_tc_backward(const AttnArgs& a, bool bf16, void* dtable, int32_t* status,
                          cudaStream_t s) {
  return bf16 ? backward_typed<__nv_bfloat16>(a, dtable, status, s)
              : backward_typed<__half>(a, dtable, status, s);
}

}  // namespace sv
