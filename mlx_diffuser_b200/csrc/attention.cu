// Self-attention inside coordinate windows with a learned relative position bias, and its
// gradients.
//
//     s_ij = scale * q_i . k_j + T[h][L[x_j - x_i]][L[y_j - y_i]][L[z_j - z_i]]   (i, j in a window)
//     p_ij = softmax_j(s_ij),  o_i = sum_j p_ij v_j
//     dv_j = sum_i p_ij do_i,  ds_ij = p_ij (do_i . v_j - delta_i),  delta_i = do_i . o_i
//     dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dT[h][b] = sum of ds over b's pairs
//
// L maps an offset along an axis, clamped to the table's reach, to a bucket. The windows come as a
// plan: rows in window order with each window's range of positions (sv_window_plan).
//
// fp32 runs on attention_f32.cu, fp16 and bf16 on attention_tc.cu; the plan and the entry points are
// here.
#include "attention.h"

namespace sv {
namespace {

// Every row's window extent: a block per window.
__global__ void __launch_bounds__(128)
    window_span_kernel(const int32_t* __restrict__ offsets, int64_t groups, int64_t n,
                       PlanRow* __restrict__ plan) {
  __shared__ int s_low[3], s_high[3];
  const int64_t g = blockIdx.x;
  const int64_t start = max(0, __ldg(offsets + g)), end = min((int64_t)__ldg(offsets + g + 1), n);
  if (threadIdx.x < 3) {
    s_low[threadIdx.x] = INT_MAX;
    s_high[threadIdx.x] = INT_MIN;
  }
  __syncthreads();
  int low[3] = {INT_MAX, INT_MAX, INT_MAX}, high[3] = {INT_MIN, INT_MIN, INT_MIN};
  for (int64_t p = start + threadIdx.x; p < end; p += 128) {
    const PlanRow& r = plan[p];
    if (r.row < 0) continue;
    low[0] = min(low[0], r.x); high[0] = max(high[0], r.x);
    low[1] = min(low[1], r.y); high[1] = max(high[1], r.y);
    low[2] = min(low[2], r.z); high[2] = max(high[2], r.z);
  }
#pragma unroll
  for (int c = 0; c < 3; ++c) {
    const int l = __reduce_min_sync(0xffffffffu, low[c]);
    const int h = __reduce_max_sync(0xffffffffu, high[c]);
    if ((threadIdx.x & 31) == 0) {
      atomicMin(&s_low[c], l);
      atomicMax(&s_high[c], h);
    }
  }
  __syncthreads();
  int span = 0;
#pragma unroll
  for (int c = 0; c < 3; ++c)
    if (s_high[c] >= s_low[c]) span = max(span, sub_sat(s_high[c], s_low[c]));
  for (int64_t p = start + threadIdx.x; p < end; p += 128)
    if (plan[p].row >= 0) plan[p].span = span;
}

__global__ void __launch_bounds__(256)
    window_plan_kernel(const int32_t* __restrict__ coords, const int32_t* __restrict__ perm,
                       const int32_t* __restrict__ offsets, int64_t groups, int64_t n,
                       PlanRow* __restrict__ plan, int32_t* status) {
  const int64_t p = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (p >= n) return;
  int64_t lo = 0, hi = groups;  // offsets[lo] <= p < offsets[hi]
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) / 2;
    if (__ldg(offsets + mid) <= p) lo = mid; else hi = mid;
  }
  PlanRow r{};
  const int32_t start = __ldg(offsets + lo), end = __ldg(offsets + lo + 1);
  r.row = __ldg(perm + p);
  if (r.row < 0 || r.row >= n || start > p || end <= p || start < 0 || end > n) {
    report(status, SV_DEVICE_BAD_INDEX);
    r.row = -1;
    r.start = r.end = (int32_t)p;
  } else {
    const int4 c = __ldg(reinterpret_cast<const int4*>(coords) + r.row);
    r.x = c.y;
    r.y = c.z;
    r.z = c.w;
    r.start = start;
    r.end = end;
  }
  plan[p] = r;
}

// The blocks of the plan: a thread per window, blockIdx.y for the two sizes.
__global__ void __launch_bounds__(128)
    window_blocks_kernel(const int32_t* __restrict__ offsets, int64_t groups, int64_t n,
                         uint8_t* __restrict__ plan, int32_t* status) {
  const int64_t g = (int64_t)blockIdx.x * 128 + threadIdx.x;
  if (g >= groups) return;
  const int which = blockIdx.y, size = which ? 128 : 64, half = size / 2;
  const PlanBlocks at = plan_blocks(n);
  int2* blocks = reinterpret_cast<int2*>(plan + at.block[which]);
  auto bound = [&](int64_t i) { return max(0, min((int)n, __ldg(offsets + i))); };
  const int start = bound(g), end = bound(g + 1), rows = end - start;
  if (rows <= 0) return;
  int stop = end;
  if (rows <= half) {
    // The first small window of its stretch takes the others along. Empty windows between them are
    // passed over, though not without end; both loops go by the same rule.
    constexpr int GAP = 64;
    for (int64_t i = g - 1, gap = 0; i >= 0 && gap <= GAP; --i, ++gap) {
      const int s = bound(i), e = bound(i + 1);
      if (e <= s) continue;
      if (e == start && e - s <= half && s / half == start / half) return;
      break;
    }
    for (int64_t i = g + 1, gap = 0; i < groups && gap <= GAP; ++i, ++gap) {
      const int s = bound(i), e = bound(i + 1);
      if (e <= s) continue;
      if (s != stop || e - s > half || s / half != start / half) break;
      stop = e;
      gap = -1;
    }
  }
  const int pieces = (stop - start + size - 1) / size;
  const int first = atomicAdd(reinterpret_cast<int*>(plan + at.count) + which, pieces);
  for (int i = 0; i < pieces; ++i) {
    if (first + i >= at.cap[which]) {  // windows that overlap
      report(status, SV_DEVICE_BAD_INDEX);
      return;
    }
    const int p = start + i * size;
    blocks[first + i] = make_int2(p, min(size, stop - p));
  }
}

bool float_type(int d) { return d == SV_FLOAT32 || d == SV_FLOAT16 || d == SV_BFLOAT16; }

int check(int64_t n, int heads, int dim, int dtype, int nb, int reach, const char* what) {
  if (!float_type(dtype))
    SV_FAIL(SV_ERR_BAD_DTYPE, std::string(what) + ": unknown dtype");
  if (n < 0 || heads < 0 || dim < 0 || nb < 1 || reach < 0)
    SV_FAIL(SV_ERR_INVALID_ARGUMENT, std::string(what) + ": negative size");
  if (n > (1 << 25) || heads > ATTN_MAX_HEADS || dim > ATTN_MAX_DIM || nb > ATTN_MAX_BUCKETS ||
      reach > ATTN_MAX_REACH)
    SV_FAIL(SV_ERR_UNSUPPORTED,
            std::string(what) +
                ": at most 2^25 rows, 65535 heads, 128 channels a head, 25 buckets an axis and a "
                "reach of 1023");
  return SV_OK;
}

int check_strides(const int64_t* strides, const char* what) {
  for (int i = 0; i < 6; ++i)
    if (strides[i] < 0 || strides[i] > (1 << 30))
      SV_FAIL(SV_ERR_UNSUPPORTED, std::string(what) + ": strides must be between 0 and 2^30");
  return SV_OK;
}

// Workspace of a split forward pass: the parts' sums.
struct PartLayout {
  int parts;
  size_t stats, total;  // the sums are at the start
};
PartLayout part_layout(int64_t n, int heads, int dim, int dtype, int64_t windows) {
  PartLayout l{1, 0, 0};
  if (dtype != SV_FLOAT32) l.parts = attention_tc_parts(n, heads, dim, windows);
  if (l.parts == 1) return l;
  const size_t rows = (size_t)l.parts * heads * n;
  l.stats = align_up(rows * dim * 4, 256);
  l.total = l.stats + align_up(rows * 8, 256);
  return l;
}

// Workspace of the backward pass: fixed-point table, norms, the buckets' largest terms, delta.
struct Layout {
  size_t table, norms, tops, delta, total;
};
Layout layout(int64_t n, int heads, int nb) {
  Layout l;
  l.table = 0;
  l.norms = l.table + align_up((size_t)heads * nb * nb * nb * 8, 256);
  l.tops = l.norms + align_up((size_t)heads * 8, 256);
  l.delta = l.tops + align_up((size_t)heads * nb * nb * nb * 4, 256);
  l.total = l.delta + align_up((size_t)heads * n * 4, 256);
  return l;
}

}  // namespace
}  // namespace sv

using namespace sv;

extern "C" size_t sv_window_plan_bytes(int64_t n) {
  return n > 0 && n <= (1 << 25) ? (size_t)plan_blocks(n).total : 0;
}

extern "C" int sv_window_plan(const int32_t* coords, const int32_t* perm, const int32_t* offsets,
                              int64_t groups, int64_t n, void* plan, int32_t* status,
                              sv_stream_t stream) {
  if (n < 0 || groups < 0) SV_FAIL(SV_ERR_INVALID_ARGUMENT, "sv_window_plan: negative size");
  if (n > (1 << 25)) SV_FAIL(SV_ERR_UNSUPPORTED, "sv_window_plan: at most 2^25 rows");
  if (n == 0) return SV_OK;
  if (!coords || !perm || !offsets || !plan || groups < 1 || groups > n || !aligned16(coords) ||
      !aligned16(plan))
    SV_FAIL(SV_ERR_INVALID_ARGUMENT,
            "sv_window_plan: null or misaligned pointer, or not 1 to n groups");
  uint8_t* bytes = static_cast<uint8_t*>(plan);
  SV_CUDA_TRY(cudaMemsetAsync(bytes + plan_blocks(n).count, 0, 16, to_stream(stream)));
  window_plan_kernel<<<(unsigned)((n + 255) / 256), 256, 0, to_stream(stream)>>>(
      coords, perm, offsets, groups, n, static_cast<PlanRow*>(plan), status);
  SV_LAUNCH_CHECK();
  window_span_kernel<<<(unsigned)groups, 128, 0, to_stream(stream)>>>(
      offsets, groups, n, static_cast<PlanRow*>(plan));
  SV_LAUNCH_CHECK();
  window_blocks_kernel<<<dim3((unsigned)((groups + 127) / 128), 2), 128, 0, to_stream(stream)>>>(
      offsets, groups, n, bytes, status);
  SV_LAUNCH_CHECK();
  return SV_OK;
}

extern "C" size_t sv_window_attention_workspace_bytes(int64_t n, int heads, int dim, int dtype,
                                                      int64_t windows) {
  if (n < 0 || heads < 0 || dim < 0 || dim > ATTN_MAX_DIM || !float_type(dtype)) return 0;
  return part_layout(n, heads, dim, dtype, windows).total;
}

extern "C" int sv_window_attention(const void* q, const void* k, const void* v,
                                   const int64_t* strides, int64_t n, int heads, int dim,
                                   int dtype, const void* plan, int64_t windows,
                                   const void* table, int buckets, const int32_t* lut, int reach,
                                   float scale, void* out, void* out_rest, float* stats,
                                   void* workspace, size_t workspace_bytes, sv_stream_t stream) {
  const int rc = check(n, heads, dim, dtype, buckets, reach, "sv_window_attention");
  if (rc != SV_OK) return rc;
  if (n == 0 || heads == 0 || dim == 0) return SV_OK;
  if (!q || !k || !v || !strides || !plan || !table || !lut || !out || !aligned16(plan))
    SV_FAIL(SV_ERR_INVALID_ARGUMENT, "sv_window_attention: null pointer");
  const int bad = check_strides(strides, "sv_window_attention");
  if (bad != SV_OK) return bad;
  AttnArgs a{};
  a.q = q; a.k = k; a.v = v; a.out = out; a.out_rest = dtype == SV_FLOAT32 ? nullptr : out_rest;
  a.q_row = strides[0]; a.q_head = strides[1];
  a.k_row = strides[2]; a.k_head = strides[3];
  a.v_row = strides[4]; a.v_head = strides[5];
  a.plan = static_cast<const PlanRow*>(plan);
  a.table = table; a.lut = lut; a.stats = reinterpret_cast<float2*>(stats);
  a.n = n; a.heads = heads; a.dim = dim; a.nb = buckets; a.reach = reach; a.scale = scale;
  cudaStream_t s = to_stream(stream);
  const PartLayout l = part_layout(n, heads, dim, dtype, windows);
  a.parts = l.parts;
  if (l.parts > 1) {
    if (!workspace || workspace_bytes < l.total || !aligned16(workspace))
      SV_FAIL(SV_ERR_WORKSPACE, "sv_window_attention: workspace too small or unaligned");
    a.part_out = static_cast<float*>(workspace);
    a.part_stats = reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace) + l.stats);
  }
  if (dtype != SV_FLOAT32) return attention_tc_forward(a, dtype == SV_BFLOAT16, s);
  return attention_f32_forward(a, s);
}

extern "C" size_t sv_window_attention_backward_workspace_bytes(int64_t n, int heads, int buckets) {
  if (n < 0 || heads < 0 || buckets < 1 || buckets > ATTN_MAX_BUCKETS) return 0;
  return layout(n, heads, buckets).total;
}

extern "C" int sv_window_attention_backward(
    const void* q, const void* k, const void* v, const int64_t* strides, const void* o,
    const void* o_rest, const void* dout, const float* stats, int64_t n, int heads, int dim,
    int dtype, const void* plan, const void* table, int buckets, const int32_t* lut, int reach,
    float scale, void* dq, void* dk, void* dv, void* dtable, void* workspace,
    size_t workspace_bytes, sv_stream_t stream) {
  const int rc = check(n, heads, dim, dtype, buckets, reach, "sv_window_attention_backward");
  if (rc != SV_OK) return rc;
  cudaStream_t s = to_stream(stream);
  const size_t cells = (size_t)heads * buckets * buckets * buckets;
  if (n == 0 || heads == 0 || dim == 0) {
    if (dtable && cells) SV_CUDA_TRY(cudaMemsetAsync(dtable, 0, cells * dtype_size(dtype), s));
    return SV_OK;
  }
  if (!q || !k || !v || !strides || !o || !dout || !stats || !plan || !table || !lut || !dq || !dk ||
      !dv || !aligned16(plan))
    SV_FAIL(SV_ERR_INVALID_ARGUMENT, "sv_window_attention_backward: null pointer");
  const int bad = check_strides(strides, "sv_window_attention_backward");
  if (bad != SV_OK) return bad;
  const Layout l = layout(n, heads, buckets);
  if (!workspace || workspace_bytes < l.total || !aligned16(workspace))
    SV_FAIL(SV_ERR_WORKSPACE, "sv_window_attention_backward: workspace too small or unaligned");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  AttnArgs a{};
  a.q = q; a.k = k; a.v = v; a.o = o; a.dout = dout;
  a.o_rest = dtype == SV_FLOAT32 ? nullptr : o_rest;
  a.q_row = strides[0]; a.q_head = strides[1];
  a.k_row = strides[2]; a.k_head = strides[3];
  a.v_row = strides[4]; a.v_head = strides[5];
  a.dq = dq; a.dk = dk; a.dv = dv;
  a.plan = static_cast<const PlanRow*>(plan);
  a.table = table; a.lut = lut;
  a.stats = reinterpret_cast<float2*>(const_cast<float*>(stats));
  a.delta = reinterpret_cast<float*>(ws + l.delta);
  a.n = n; a.heads = heads; a.dim = dim; a.nb = buckets; a.reach = reach; a.scale = scale;
  a.norms = reinterpret_cast<unsigned*>(ws + l.norms);
  a.tops = reinterpret_cast<unsigned*>(ws + l.tops);
  if (dtable) {
    a.dtable = reinterpret_cast<unsigned long long*>(ws + l.table);
    SV_CUDA_TRY(cudaMemsetAsync(ws, 0, l.delta, s));  // the table, the norms and the buckets' largest terms
  }
  if (dtype == SV_FLOAT32) return attention_f32_backward(a, dtable, s);
  return attention_tc_backward(a, dtype == SV_BFLOAT16, dtable, s);
}
