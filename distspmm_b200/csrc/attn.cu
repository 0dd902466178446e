// attn.cu — attention over the entries of a CSR pattern, and over cache rows listed by a CSR in device memory.
//
//   u_ij = cap tanh(scale q_i.k_j / cap) - slope |i + row_offset - j|     for the entries (i, j) of row i
//   o_i = sum_j p_ij v_j,  p_ij = exp(u_ij - lse_i),  lse_i = log sum_j exp(u_ij)
//   delta_i = dout_i.o_i,  ds_ij = p_ij (dout_i.v_j - delta_i) (1 - tanh^2) scale
//   dq_i = sum_j ds_ij k_j,  dk_j = sum_i ds_ij q_i,  dv_j = sum_i p_ij dout_i
//
// These kernels gather: for each entry and head one row of k and one of v (or of q and dout, by columns) come out of L2, two
// operations per element read. What bounds them is issue (68 % of the slots in the forward of R-MAT 14, fp32, 4 heads of 32; L1 31 %): dot
// products by shuffles, and the ends of short rows. A warp owns one chunk of entries (pattern.h) and one head; LPR lanes
// hold a head's row in vectors of VE elements, so 32 / LPR entries are in work side by side, each with its own running
// maximum and sum, merged when the row ends. Only listed entries are read: what other rows of k and v hold, NaN included,
// cannot reach a row that does not list them.
#include <algorithm>
#include <type_traits>

#include "attn_row.cuh"
#include "attn_decode.h"
#include "attn_graph.h"
#include "attn_tile.h"

namespace dsp {
namespace {

constexpr int kThreads = 256;

// Rows r0 .. r1 and entries p0 .. p1 of a chunk, for head h.
template <class T, int VE, int LPR, int VPL, class Rows>
__device__ __forceinline__ void chunk_rows(const Rows &d, const AttnArgs &a, int64_t chunk, int h, typename Rows::Index r0,
                                           typename Rows::Index r1, typename Rows::Index p0, typename Rows::Index p1) {
  using H = HeadRow<T, VE, LPR, VPL>;
  using I = typename Rows::Index;
  const int lane = threadIdx.x % LPR, g = (threadIdx.x & 31) / LPR;
  const bool head_cut = p0 > d.ptr(r0);
  I p = p0;
  for (I row = r0; row <= r1; ++row) {
    if (row == r1 && (p >= p1 || row >= d.n())) break;
    const I end = d.ptr(row + 1), pe = row < r1 ? end : p1;
    float acc[VPL][VE], m, l;
    attend<H, LPR>(d, a, row, h, p, pe, end, m, l, acc);
    const bool cut_head = row == r0 && head_cut;
    if (cut_head || row == r1) {
      const int64_t slot = (cut_head ? 2 * chunk : 2 * chunk + 1) * a.heads + h;
      if (g == 0) H::store_f32(a.slots + slot * a.dim, lane, a.dim, acc);
      if ((threadIdx.x & 31) == 0) a.slot_ml[2 * slot] = m, a.slot_ml[2 * slot + 1] = l;
    } else {
      put_row<H, LPR>(a, row, h, m, l, acc);
    }
    p = pe;
  }
}

template <class Rows, class T, int VE, int LPR, int VPL>
__global__ void __launch_bounds__(kThreads, VPL == 1 ? 3 : 2) attn_rows_kernel(const Rows d, const AttnArgs a) {
  const int64_t item = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> 5;
  const int64_t chunk = item / a.heads;
  const int h = (int)(item - chunk * a.heads);
  if (chunk >= d.chunks()) return;
  if constexpr (std::is_same<Rows, PlanRows>::value) {
    __shared__ ChunkLists lists[kThreads / 32];
    const StagedRows s(d, chunk, lists[threadIdx.x >> 5]);
    chunk_rows<T, VE, LPR, VPL>(s, a, chunk, h, s.r0, s.r1, s.p0, s.p1);
  } else {
    int64_t r0, r1, p0, p1;
    d.chunk(chunk, r0, r1, p0, p1);
    chunk_rows<T, VE, LPR, VPL>(d, a, chunk, h, r0, r1, p0, p1);
  }
}

// dq and delta of the pattern's rows.
template <class T, int VE, int LPR, int VPL>
__global__ void __launch_bounds__(kThreads, VPL == 1 ? 3 : 2) attn_dq_kernel(const PlanRows rows, const AttnArgs a) {
  using H = HeadRow<T, VE, LPR, VPL>;
  const int64_t item = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> 5;
  const int64_t chunk = item / a.heads;
  const int h = (int)(item - chunk * a.heads);
  if (chunk >= rows.chunks()) return;
  const int lane = threadIdx.x % LPR, g = (threadIdx.x & 31) / LPR;
  __shared__ ChunkLists lists[kThreads / 32];
  const StagedRows d(rows, chunk, lists[threadIdx.x >> 5]);
  const int32_t r0 = d.r0, r1 = d.r1, p1 = d.p1;
  int32_t p = d.p0;
  const bool head_cut = p > d.ptr(r0);
  for (int32_t row = r0; row <= r1; ++row) {
    if (row == r1 && p >= p1) break;
    const int32_t pe = row < r1 ? d.ptr(row + 1) : p1;
    float gap, delta0, x[VPL][VE], y[VPL][VE];
    attend_dq<H, LPR>(d, a, row, h, p, pe, gap, delta0, x, y);
    const bool cut_head = row == r0 && head_cut;
    if (cut_head || row == r1) {
      const int64_t slot = (cut_head ? 2 * chunk : 2 * chunk + 1) * a.heads + h;
      if (g == 0) {
        H::store_f32(a.slots + slot * 2 * a.dim, lane, a.dim, x);
        H::store_f32(a.slots + slot * 2 * a.dim + a.dim, lane, a.dim, y);
      }
      if ((threadIdx.x & 31) == 0) a.slot_ml[2 * slot] = gap, a.slot_ml[2 * slot + 1] = delta0;
    } else {
#pragma unroll
      for (int w = 0; w < VPL; ++w)
#pragma unroll
        for (int i = 0; i < VE; ++i) x[w][i] = (x[w][i] - gap * y[w][i]) * a.scale;
      if (g == 0) H::store(a.dq, row, h, lane, a.dim, x);
      if ((threadIdx.x & 31) == 0) a.delta[(int64_t)row * a.heads + h] = delta0 + gap;
    }
    p = pe;
  }
}

// dk and dv of the pattern's columns (d: the transposed pattern), one key/value head.
template <class T, int VE, int LPR, int VPL>
__global__ void __launch_bounds__(kThreads, VPL == 1 ? 3 : 2) attn_dkv_kernel(const PlanRows rows, const AttnArgs a) {
  using H = HeadRow<T, VE, LPR, VPL>;
  const int kv_heads = a.heads / a.group;
  const int64_t item = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> 5;
  const int64_t chunk = item / kv_heads;
  const int hk = (int)(item - chunk * kv_heads);
  if (chunk >= rows.chunks()) return;
  const int lane = threadIdx.x % LPR, g = (threadIdx.x & 31) / LPR;
  __shared__ ChunkLists lists[kThreads / 32];
  const StagedRows d(rows, chunk, lists[threadIdx.x >> 5]);
  const int32_t r0 = d.r0, r1 = d.r1, p1 = d.p1;
  int32_t p = d.p0;
  const bool head_cut = p > d.ptr(r0);
  for (int32_t row = r0; row <= r1; ++row) {  // a row here is a column of A
    if (row == r1 && p >= p1) break;
    const int32_t pe = row < r1 ? d.ptr(row + 1) : p1;
    float dk[VPL][VE], dv[VPL][VE];
    attend_dkv<H, LPR>(d, a, row, hk, p, pe, dk, dv);
    const bool cut_head = row == r0 && head_cut;
    if (g == 0) {
      if (cut_head || row == r1) {
        float *dst = a.slots + ((cut_head ? 2 * chunk : 2 * chunk + 1) * kv_heads + hk) * 2 * a.dim;
        H::store_f32(dst, lane, a.dim, dk);
        H::store_f32(dst + a.dim, lane, a.dim, dv);
      } else {
        H::store(a.dk, row, hk, lane, a.dim, dk);
        H::store(a.dv, row, hk, lane, a.dim, dv);
      }
    }
    p = pe;
  }
}

// A cut row of the list and the warps that join it: a block for each long one (warp w takes slots w, w + 8, ...), a warp for each
// other. join_blocks(d) blocks of 8 warps.
struct CutRow {
  int64_t row, c0, c1;
  bool wide;
  __device__ __forceinline__ bool find(const DirView &d) {
    wide = (int)blockIdx.x < d.n_long;
    const int at = wide ? (int)blockIdx.x : d.n_long + ((int)blockIdx.x - d.n_long) * 8 + (threadIdx.x >> 5);
    if (at >= d.n_split) return false;
    row = __ldg(d.split_row + at);
    c0 = row_start(row, __ldg(d.ptr + row)) / d.L, c1 = row_start(row, __ldg(d.ptr + row + 1)) / d.L;
    return true;
  }
  __device__ __forceinline__ int64_t slot(int64_t c) const { return c == c0 ? 2 * c + 1 : 2 * c; }
};

// Where attn_graph.cu left the partials of type T, an infinity in them may have become NaN: the row, or key, again by gather.
template <class T>
__device__ __forceinline__ void row_again(const DirView &d, const AttnArgs &a, int64_t row, int h) {
  if constexpr (sizeof(T) == 2) {
    if (a.dim == 32) attend_again<T, 32>(PlanRows{d}, a, row, h);
    else if (a.dim == 64) attend_again<T, 64>(PlanRows{d}, a, row, h);
    else if (a.dim == 128) attend_again<T, 128>(PlanRows{d}, a, row, h);
  }
}
template <class T>
__device__ __forceinline__ void key_again(const DirView &d, const AttnArgs &a, int64_t row, int hk) {
  if constexpr (sizeof(T) == 2) {
    if (a.dim == 32) attend_dkv_again<T, 32>(PlanRows{d}, a, row, hk);
    else if (a.dim == 64) attend_dkv_again<T, 64>(PlanRows{d}, a, row, hk);
    else if (a.dim == 128) attend_dkv_again<T, 128>(PlanRows{d}, a, row, hk);
  }
}

// Partials of cut rows (forward), merged in a fixed order. blockIdx.y: head. Lane l holds columns l, l + 32, ...
template <class T>
__global__ void __launch_bounds__(kThreads, 5) attn_join_kernel(const __grid_constant__ DirView d, const __grid_constant__ AttnArgs a) {
  __shared__ float part[8][256], part_ml[8][2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, h = blockIdx.y;
  CutRow r;
  if (!r.find(d)) return;  // whole warps of a block without barriers
  float m = -INFINITY, l = 0.f, acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.f;
  auto merge = [&](float m2, float l2, const float *src) {
    const float top = fmaxf(m, m2), base = top == -INFINITY ? 0.f : top;
    const float f1 = exp2_approx(m - base), f2 = exp2_approx(m2 - base);
    l = l * f1 + l2 * f2;
    m = top;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < a.dim) acc[i] = acc[i] * f1 + src[lane + 32 * i] * f2;
  };
#pragma unroll 4
  for (int64_t c = r.c0 + (r.wide ? warp : 0); c <= r.c1; c += r.wide ? 8 : 1) {
    const int64_t slot = r.slot(c) * a.heads + h;
    merge(a.slot_ml[2 * slot], a.slot_ml[2 * slot + 1], a.slots + slot * a.dim);
  }
  if (r.wide) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < a.dim) part[warp][lane + 32 * i] = acc[i];
    if (lane == 0) part_ml[warp][0] = m, part_ml[warp][1] = l;
    __syncthreads();
    if (warp > 0) return;
    for (int w = 1; w < 8; ++w) merge(part_ml[w][0], part_ml[w][1], part[w]);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  float zero = 0.f;
  T *dst = (T *)a.out.p + r.row * a.out.row + h * a.out.head;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (lane + 32 * i < a.dim) {
      dst[lane + 32 * i] = T(acc[i] * inv);
      zero = fmaf(acc[i] * inv, 0.f, zero);
    }
  if (a.lse && lane == 0) a.lse[r.row * a.heads + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
  if (__any_sync(0xffffffffu, zero != 0.f) && l == l) row_again<T>(d, a, r.row, h);
}

// Partials of cut rows (gradients), 2 dim floats per slot and head, summed in a fixed order. DQ: the sums x and y of a row, its
// delta - delta0 and delta0 (attend_dq); else dk and dv of a key.
template <class T, bool DQ>
__global__ void __launch_bounds__(kThreads, 4) attn_sum_kernel(const __grid_constant__ DirView d, int n_heads, const __grid_constant__ AttnArgs a) {
  __shared__ float part[8][512], part_delta[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, h = blockIdx.y;
  CutRow r;
  if (!r.find(d)) return;
  const int64_t first = r.c0 + (r.wide ? warp : 0);
  const int step = r.wide ? 8 : 1;
  float delta = 0.f, x[8], y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = y[i] = 0.f;
#pragma unroll 4
  for (int64_t c = first; c <= r.c1; c += step) {
    const int64_t slot = r.slot(c) * n_heads + h;
    const float *src = a.slots + slot * 2 * a.dim + lane;
    if (DQ) delta += a.slot_ml[2 * slot];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < a.dim) x[i] += src[32 * i], y[i] += src[a.dim + 32 * i];
  }
  if (r.wide) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < a.dim) part[warp][lane + 32 * i] = x[i], part[warp][256 + lane + 32 * i] = y[i];
    if (lane == 0) part_delta[warp] = delta;
    __syncthreads();
    if (warp > 0) return;
    for (int w = 1; w < 8; ++w) {
      delta += part_delta[w];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (lane + 32 * i < a.dim) x[i] += part[w][lane + 32 * i], y[i] += part[w][256 + lane + 32 * i];
    }
  }
  if (DQ && lane == 0) {
    const float lse = a.lse[r.row * a.heads + h], whole = delta + a.slot_ml[2 * (r.slot(r.c0) * n_heads + h) + 1];
    if (a.stats) a.stats[r.row * a.heads + h] = make_float2(lse == -INFINITY ? INFINITY : lse * kLog2e, whole);
    else a.delta[r.row * a.heads + h] = whole;
  }
  float zero = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int col = lane + 32 * i;
    if (col >= a.dim) continue;
    zero = fmaf(x[i], 0.f, fmaf(y[i], 0.f, zero));
    if (DQ) {
      ((T *)a.dq.p)[r.row * a.dq.row + h * a.dq.head + col] = T((x[i] - delta * y[i]) * a.scale);
    } else {
      ((T *)a.dk.p)[r.row * a.dk.row + h * a.dk.head + col] = T(x[i]);
      ((T *)a.dv.p)[r.row * a.dv.row + h * a.dv.head + col] = T(y[i]);
    }
  }
  if constexpr (!DQ) {
    if (__any_sync(0xffffffffu, zero != 0.f)) key_again<T>(d, a, r.row, h);
  }
}

// ------------------------------------------------------------------------------------------------ launches

int64_t up256(int64_t x) { return (x + 255) / 256 * 256; }

int status(const char *who) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? DSP_OK : fail(DSP_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
}

unsigned warps_grid(int64_t warps) { return (unsigned)((warps + kThreads / 32 - 1) / (kThreads / 32)); }

template <class Rows, class T, int VE, int LPR, int VPL>
void launch_shape(AttnPass pass, const Rows &rows, const AttnArgs &a, int64_t n_chunks, cudaStream_t s) {
  const int64_t warps = n_chunks * (pass == kDkv ? a.heads / a.group : a.heads);
  if (pass == kForward) {
    attn_rows_kernel<Rows, T, VE, LPR, VPL><<<warps_grid(warps), kThreads, 0, s>>>(rows, a);
  } else if constexpr (std::is_same<Rows, PlanRows>::value) {
    if (pass == kDq) attn_dq_kernel<T, VE, LPR, VPL><<<warps_grid(warps), kThreads, 0, s>>>(rows, a);
    else attn_dkv_kernel<T, VE, LPR, VPL><<<warps_grid(warps), kThreads, 0, s>>>(rows, a);
  }
}

template <class Rows, class T>
void launch_pass(AttnPass pass, const Rows &rows, const AttnArgs &a, int64_t n_chunks, cudaStream_t s) {
  if (n_chunks == 0) return;
  if constexpr (sizeof(T) == 2) {
    if (a.dim <= 32) launch_shape<Rows, T, 8, 4, 1>(pass, rows, a, n_chunks, s);
    else if (a.dim <= 64) launch_shape<Rows, T, 8, 8, 1>(pass, rows, a, n_chunks, s);
    else if (a.dim <= 128) launch_shape<Rows, T, 8, 16, 1>(pass, rows, a, n_chunks, s);
    else launch_shape<Rows, T, 8, 32, 1>(pass, rows, a, n_chunks, s);
  } else {
    if (a.dim <= 32) launch_shape<Rows, T, 4, 8, 1>(pass, rows, a, n_chunks, s);
    else if (a.dim <= 64) launch_shape<Rows, T, 4, 16, 1>(pass, rows, a, n_chunks, s);
    else if (a.dim <= 128) launch_shape<Rows, T, 4, 32, 1>(pass, rows, a, n_chunks, s);
    else launch_shape<Rows, T, 4, 32, 2>(pass, rows, a, n_chunks, s);
  }
}

AttnArgs args_of(const dsp_attn_desc *d) {
  AttnArgs a = {};
  a.heads = d->heads, a.group = d->heads / d->kv_heads, a.dim = d->dim;
  a.scale = d->scale, a.cap = d->softcap, a.slopes = d->slopes, a.row_offset = d->row_offset;
  a.q = {d->q, d->q_row, d->q_head};
  a.k = {d->k, d->k_row, d->k_head};
  a.v = {d->v, d->v_row, d->v_head};
  a.out = {d->out, d->out_row, d->out_head};
  a.o = {d->out, d->out_row, d->out_head};
  a.lse = d->lse;
  return a;
}

struct ForwardPlan {
  int64_t slots, ml, total;
};
ForwardPlan forward_plan(int64_t n_chunks, bool cut, int heads, int dim) {
  ForwardPlan f = {};
  f.ml = cut ? up256(8 * n_chunks * heads * dim) : 0;
  f.total = f.ml + (cut ? up256(16 * n_chunks * heads) : 0);
  return f;
}

struct GradPlan {
  int64_t slots, ml, total;
};
GradPlan grad_plan(const dsp_pattern *p, const dsp_attn_desc *d) {
  GradPlan g = {};
  g.slots = up256(8 * p->rows * d->heads);  // delta, or stats, lie before them
  const int64_t q = p->a.n_split ? 16ll * p->a.n_chunks * d->heads * d->dim : 0;
  const int64_t kv = p->t.n_split ? 16ll * p->t.n_chunks * d->kv_heads * d->dim : 0;
  g.ml = g.slots + up256(std::max(q, kv));  // dq's partials are joined before dk's and dv's are written
  g.total = g.ml + (p->a.n_split ? up256(16ll * p->a.n_chunks * d->heads) : 0);
  return g;
}

template <class T>
int forward(const dsp_pattern *p, const dsp_attn_desc *d, char *ws, cudaStream_t s) {
  AttnArgs a = args_of(d);
  const ForwardPlan f = forward_plan(p->a.n_chunks, p->a.n_split > 0, d->heads, d->dim);
  a.slots = (float *)ws;
  a.slot_ml = (float *)(ws + f.ml);
  const PlanRows rows = {view(p->a)};
  if (graph_on_tensor_cores(d->dtype, d->dim)) graph_pass(kForward, rows.d, a, d->dtype, s);
  else launch_pass<PlanRows, T>(kForward, rows, a, p->a.n_chunks, s);
  if (p->a.n_split)
    attn_join_kernel<T><<<dim3((unsigned)join_blocks(rows.d), (unsigned)d->heads), kThreads, 0, s>>>(rows.d, a);
  return status("dsp_attn");
}

AttnArgs grad_args(const dsp_attn_grad_desc *g) {
  AttnArgs a = args_of(&g->fwd);
  a.dout = {g->dout, g->dout_row, g->dout_head};
  a.dq = {g->dq, g->dq_row, g->dq_head};
  a.dk = {g->dk, g->dk_row, g->dk_head};
  a.dv = {g->dv, g->dv_row, g->dv_head};
  return a;
}

template <class T>
int gradients(const dsp_pattern *p, const dsp_attn_grad_desc *g, char *ws, cudaStream_t s) {
  const dsp_attn_desc *d = &g->fwd;
  AttnArgs a = grad_args(g);
  const GradPlan f = grad_plan(p, d);
  a.delta = (float *)ws;
  a.slots = (float *)(ws + f.slots);
  a.slot_ml = (float *)(ws + f.ml);
  const PlanRows ra = {view(p->a)}, rt = {view(p->t)};
  const bool tensor = graph_on_tensor_cores(d->dtype, d->dim);
  if (tensor) a.stats = (float2 *)ws;
  if (tensor) graph_pass(kDq, ra.d, a, d->dtype, s);
  else launch_pass<PlanRows, T>(kDq, ra, a, ra.d.n_chunks, s);
  if (ra.d.n_split)
    attn_sum_kernel<T, true><<<dim3((unsigned)join_blocks(ra.d), (unsigned)d->heads), kThreads, 0, s>>>(ra.d, d->heads, a);
  if (tensor) graph_pass(kDkv, rt.d, a, d->dtype, s);
  else launch_pass<PlanRows, T>(kDkv, rt, a, rt.d.n_chunks, s);
  if (rt.d.n_split)
    attn_sum_kernel<T, false>
        <<<dim3((unsigned)join_blocks(rt.d), (unsigned)d->kv_heads), kThreads, 0, s>>>(rt.d, d->kv_heads, a);
  return status("dsp_attn_grad");
}

template <class T>
int decode(const dsp_attn_decode_desc *g, char *ws, cudaStream_t s) {
  const dsp_attn_desc *d = &g->fwd;
  AttnArgs a = args_of(d);
  const bool tensor = decode_on_tensor_cores(d->dtype, d->dim);
  ListRows rows = {g->indptr, g->indices, g->rows, g->nnz, g->keys, 0, decode_units(g->rows, g->nnz, d->heads, d->kv_heads, tensor)};
  rows.n_chunks = (int32_t)((row_start(g->rows, g->nnz) + rows.L - 1) / rows.L);
  const ForwardPlan f = forward_plan(rows.n_chunks, true, d->heads, d->dim);
  a.slots = (float *)ws;
  a.slot_ml = (float *)(ws + f.ml);
  if (tensor) return decode_tensor(rows, a, d->dtype, s);
  launch_pass<ListRows, T>(kForward, rows, a, rows.n_chunks, s);
  return decode_join(rows, a, d->dtype, s);
}

int check_heads(const char *who, const char *name, const void *p, int64_t row, int64_t head, int dtype) {
  const int64_t e = dtype == DSP_F32 ? 4 : 2;
  DSP_TRY_ARG(p, "%s: %s is null", who, name);
  DSP_TRY_ARG(((uintptr_t)p & 15) == 0 && row * e % 16 == 0 && head * e % 16 == 0,
              "%s: %s and its strides (%lld, %lld) must be multiples of 16 bytes", who, name, (long long)row, (long long)head);
  DSP_TRY_ARG(row >= 0 && head >= 0, "%s: %s with strides (%lld, %lld)", who, name, (long long)row, (long long)head);
  if (row >= (1ll << 30))
    return fail(DSP_ERR_UNSUPPORTED, "%s: %s with a row stride of %lld: less than 2^30 is wanted", who, name, (long long)row);
  return DSP_OK;
}

// Grids count warps, one for each chunk and head, in 32 bits; tiles in CTAs.
int check_grid(const char *who, int64_t chunks, int64_t heads, int64_t tiles) {
  if (chunks * heads > (1ll << 32) || tiles * heads >= (1ll << 31))
    return fail(DSP_ERR_UNSUPPORTED, "%s: %lld chunks of entries for %lld heads", who, (long long)chunks, (long long)heads);
  return DSP_OK;
}

int check_workspace(const char *who, const void *ws, int64_t have, int64_t need) {
  if (need == 0) return DSP_OK;
  DSP_TRY_ARG(ws && have >= need, "%s: workspace of %lld bytes, %lld needed", who, (long long)(ws ? have : 0), (long long)need);
  DSP_TRY_ARG(((uintptr_t)ws & 255) == 0, "%s: the workspace must be 256-byte aligned", who);
  return DSP_OK;
}

}  // namespace

int check_attn(const char *who, const dsp_attn_desc *d, int64_t rows, int64_t keys) {
  DSP_TRY_ARG(d->dtype >= DSP_F32 && d->dtype <= DSP_F16, "%s: dtype %d", who, d->dtype);
  DSP_TRY_ARG(d->heads > 0 && d->heads <= 65535 && d->kv_heads > 0 && d->heads % d->kv_heads == 0,
              "%s: %d query heads, %d key/value heads", who, d->heads, d->kv_heads);
  if (d->dim <= 0 || d->dim > 256 || d->dim % 8)
    return fail(DSP_ERR_UNSUPPORTED, "%s: dim %d: a multiple of 8 up to 256 is wanted", who, d->dim);
  DSP_TRY_ARG(fabsf(d->scale) < INFINITY && (d->softcap == 0.f || (d->softcap >= 1e-6f && d->softcap < INFINITY)),
              "%s: scale %g, softcap %g", who, d->scale, d->softcap);
  int rc;
  if (rows > 0 && ((rc = check_heads(who, "q", d->q, d->q_row, d->q_head, d->dtype)) ||
                   (rc = check_heads(who, "out", d->out, d->out_row, d->out_head, d->dtype))))
    return rc;
  if (keys > 0 && ((rc = check_heads(who, "k", d->k, d->k_row, d->k_head, d->dtype)) ||
                   (rc = check_heads(who, "v", d->v, d->v_row, d->v_head, d->dtype))))
    return rc;
  return DSP_OK;
}

}  // namespace dsp

using namespace dsp;

static bool usable(const dsp_attn_desc *d) {
  return d && d->heads > 0 && d->heads <= 65535 && d->kv_heads > 0 && d->heads % d->kv_heads == 0 && d->dim > 0 && d->dim <= 256;
}

extern "C" int64_t dsp_attn_workspace(const dsp_pattern *p, const dsp_attn_desc *d) {
  if (!p || !usable(d)) return 0;
  if (tile_form(p, d)) return tile_forward_bytes(p, d);
  return forward_plan(p->a.n_chunks, p->a.n_split > 0, d->heads, d->dim).total;
}

extern "C" int dsp_attn(const dsp_pattern *p, const dsp_attn_desc *d, void *workspace, int64_t workspace_bytes, void *stream) {
  const char *who = "dsp_attn";
  DSP_TRY_ARG(p && d, "%s: null argument", who);
  if (!(p->flags & DSP_PATTERN_ATTENTION)) return fail(DSP_ERR_STATE, "%s: needs a pattern with DSP_PATTERN_ATTENTION", who);
  int rc = check_attn(who, d, p->rows, p->nnz ? p->cols : 0);
  if (rc) return rc;
  if (p->rows == 0) return DSP_OK;
  if ((rc = check_grid(who, p->a.n_chunks, d->heads, p->at.n))) return rc;
  rc = check_workspace(who, workspace, workspace_bytes, dsp_attn_workspace(p, d));
  if (rc) return rc;
  DeviceGuard g(p->device);
  if (g.err != cudaSuccess) return fail(DSP_ERR_CUDA, "%s: %s", who, cudaGetErrorString(g.err));
  if (tile_form(p, d)) return tile_forward(p, args_of(d), d->dtype, workspace, (cudaStream_t)stream);
  if (d->dtype == DSP_F32) return forward<float>(p, d, (char *)workspace, (cudaStream_t)stream);
  if (d->dtype == DSP_BF16) return forward<__nv_bfloat16>(p, d, (char *)workspace, (cudaStream_t)stream);
  return forward<__half>(p, d, (char *)workspace, (cudaStream_t)stream);
}

extern "C" int64_t dsp_attn_grad_workspace(const dsp_pattern *p, const dsp_attn_desc *d) {
  if (!p || !usable(d)) return 0;
  if (tile_form(p, d)) return tile_grad_bytes(p, d);
  return grad_plan(p, d).total;
}

extern "C" int dsp_attn_grad(const dsp_pattern *p, const dsp_attn_grad_desc *g, void *workspace, int64_t workspace_bytes,
                             void *stream) {
  const char *who = "dsp_attn_grad";
  DSP_TRY_ARG(p && g, "%s: null argument", who);
  const int both = DSP_PATTERN_ATTENTION | DSP_PATTERN_GRAD;
  if ((p->flags & both) != both)
    return fail(DSP_ERR_STATE, "%s: needs a pattern with DSP_PATTERN_ATTENTION and DSP_PATTERN_GRAD", who);
  const dsp_attn_desc *d = &g->fwd;
  int rc = check_attn(who, d, p->rows, p->cols);
  if (rc) return rc;
  if (p->rows > 0) {
    DSP_TRY_ARG(d->lse, "%s: lse is null", who);
    DSP_TRY_ARG((p->rows == 1 || g->dout_row > 0) && (d->heads == 1 || g->dout_head > 0), "%s: dout with strides (%lld, %lld)", who,
                (long long)g->dout_row, (long long)g->dout_head);
    if ((rc = check_heads(who, "dout", g->dout, g->dout_row, g->dout_head, d->dtype)) ||
        (rc = check_heads(who, "dq", g->dq, g->dq_row, g->dq_head, d->dtype)))
      return rc;
  }
  if (p->cols > 0 && ((rc = check_heads(who, "dk", g->dk, g->dk_row, g->dk_head, d->dtype)) ||
                      (rc = check_heads(who, "dv", g->dv, g->dv_row, g->dv_head, d->dtype))))
    return rc;
  if ((rc = check_grid(who, std::max(p->a.n_chunks, p->t.n_chunks), d->heads, std::max(p->at.n, p->tt.n)))) return rc;
  rc = check_workspace(who, workspace, workspace_bytes, dsp_attn_grad_workspace(p, d));
  if (rc) return rc;
  DeviceGuard dg(p->device);
  if (dg.err != cudaSuccess) return fail(DSP_ERR_CUDA, "%s: %s", who, cudaGetErrorString(dg.err));
  if (tile_form(p, d)) return tile_gradients(p, grad_args(g), d->dtype, workspace, (cudaStream_t)stream);
  if (d->dtype == DSP_F32) return gradients<float>(p, g, (char *)workspace, (cudaStream_t)stream);
  if (d->dtype == DSP_BF16) return gradients<__nv_bfloat16>(p, g, (char *)workspace, (cudaStream_t)stream);
  return gradients<__half>(p, g, (char *)workspace, (cudaStream_t)stream);
}

extern "C" int64_t dsp_attn_decode_workspace(const dsp_attn_decode_desc *g) {
  if (!g || !usable(&g->fwd) || g->rows < 0 || g->nnz < 0) return 0;
  const int64_t L = decode_units(g->rows, g->nnz, g->fwd.heads, g->fwd.kv_heads, decode_on_tensor_cores(g->fwd.dtype, g->fwd.dim));
  return forward_plan((row_start(g->rows, g->nnz) + L - 1) / L, true, g->fwd.heads, g->fwd.dim).total;
}

extern "C" int dsp_attn_decode(const dsp_attn_decode_desc *g, void *workspace, int64_t workspace_bytes, void *stream) {
  const char *who = "dsp_attn_decode";
  DSP_TRY_ARG(g, "%s: null argument", who);
  DSP_TRY_ARG(g->rows >= 0 && g->nnz >= 0 && g->keys >= 0, "%s: negative size", who);
  if (g->rows > (1 << 24) || g->nnz >= INT32_MAX || g->keys > INT32_MAX)
    return fail(DSP_ERR_UNSUPPORTED, "%s: %lld rows, %lld entries, %lld keys", who, (long long)g->rows, (long long)g->nnz, (long long)g->keys);
  int rc = check_attn(who, &g->fwd, g->rows, g->keys);
  if (rc) return rc;
  if (g->rows == 0) return DSP_OK;
  DSP_TRY_ARG(g->indptr && (g->indices || g->nnz == 0), "%s: null index list", who);
  const int64_t units = decode_units(g->rows, g->nnz, g->fwd.heads, g->fwd.kv_heads, decode_on_tensor_cores(g->fwd.dtype, g->fwd.dim));
  if ((rc = check_grid(who, (row_start(g->rows, g->nnz) + units - 1) / units, g->fwd.heads, 0))) return rc;
  rc = check_workspace(who, workspace, workspace_bytes, dsp_attn_decode_workspace(g));
  if (rc) return rc;
  DeviceGuard dg(g->device);
  if (dg.err != cudaSuccess) return fail(DSP_ERR_CUDA, "%s: %s", who, cudaGetErrorString(dg.err));
  if (g->fwd.dtype == DSP_F32) return decode<float>(g, (char *)workspace, (cudaStream_t)stream);
  if (g->fwd.dtype == DSP_BF16) return decode<__nv_bfloat16>(g, (char *)workspace, (cudaStream_t)stream);
  return decode<__half>(g, (char *)workspace, (cudaStream_t)stream);
}
