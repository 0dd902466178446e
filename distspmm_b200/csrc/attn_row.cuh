// attn_row.cuh — one query row, or one key column, of attention by one warp: gathers of listed entries.
#pragma once
#include "attn.h"
#include "rowvec.cuh"

namespace dsp {

// Rows and entries of a prepared pattern.
struct PlanRows {
  using Index = int32_t;
  DirView d;
  __device__ int64_t chunks() const { return d.n_chunks; }
  __device__ void chunk(int64_t c, int64_t &r0, int64_t &r1, int64_t &p0, int64_t &p1) const {
    r0 = __ldg(d.row0 + c), r1 = __ldg(d.row0 + c + 1), p0 = __ldg(d.nz0 + c), p1 = __ldg(d.nz0 + c + 1);
  }
  __device__ int64_t n() const { return d.n; }
  __device__ int64_t ptr(int64_t r) const { return __ldg(d.ptr + r); }
  __device__ int64_t col(int64_t p) const { return __ldg(d.cols + p); }
  __device__ float distance(const AttnArgs &a, int64_t row, int64_t, int64_t, int64_t col) const {
    return fabsf((float)(row + a.row_offset - col));
  }
  __device__ bool in_range(int64_t) const { return true; }
};

// A chunk of a prepared pattern with its lists in shared memory: one coalesced read instead of a wait for each step.
struct ChunkLists {
  int32_t cols[kMaxUnits];
  int32_t ptr[kMaxUnits / kRowUnits + 4];
};
struct StagedRows : PlanRows {
  const int32_t *cols_, *ptr_;
  int32_t r0, r1, p0, p1;
  __device__ __forceinline__ StagedRows(const PlanRows &rows, int64_t c, ChunkLists &list) : PlanRows(rows) {
    const int lane = threadIdx.x & 31;
    r0 = __ldg(d.row0 + c), r1 = __ldg(d.row0 + c + 1), p0 = __ldg(d.nz0 + c), p1 = __ldg(d.nz0 + c + 1);
    for (int i = lane; i <= r1 - r0 + 1; i += 32)
      if (r0 + i <= d.n) list.ptr[i] = __ldg(d.ptr + r0 + i);
#pragma unroll 4
    for (int i = lane; i < p1 - p0; i += 32) list.cols[i] = __ldg(d.cols + p0 + i);
    __syncwarp();
    cols_ = list.cols - p0, ptr_ = list.ptr - r0;
  }
  __device__ int32_t ptr(int32_t r) const { return ptr_[r]; }
  __device__ int32_t col(int32_t p) const { return cols_[p]; }
};

// A head's row in the lanes of a group: VPL vectors of VE elements.
template <class T, int VE, int LPR, int VPL>
struct HeadRow {
  using V = RowVec<T, VE>;
  using Raw = typename V::Raw;
  static __device__ __forceinline__ void fetch(const Heads &x, int64_t row, int head, int lane, int dim, bool on, Raw (&r)[VPL]) {
    const T *src = (const T *)x.p + row * x.row + head * x.head + lane * VE;
#pragma unroll
    for (int w = 0; w < VPL; ++w) r[w] = on && (lane + w * LPR) * VE < dim ? V::ldg(src + w * LPR * VE) : V::zero();
  }
  static __device__ __forceinline__ void widen(const Raw (&r)[VPL], float (&f)[VPL][VE]) {
#pragma unroll
    for (int w = 0; w < VPL; ++w) V::widen(r[w], f[w]);
  }
  static __device__ __forceinline__ float dot(const float (&x)[VPL][VE], const Raw (&r)[VPL]) {
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int w = 0; w < VPL; ++w) dot_row<T, VE>(s, x[w], r[w]);
    return s[0] + s[1];
  }
  static __device__ __forceinline__ void add(float (&acc)[VPL][VE], float x, const Raw (&r)[VPL]) {
#pragma unroll
    for (int w = 0; w < VPL; ++w) fma_row<T, VE>(acc[w], x, r[w]);
  }
  static __device__ __forceinline__ void store(const HeadsOut &x, int64_t row, int head, int lane, int dim, const float (&f)[VPL][VE]) {
    T *dst = (T *)x.p + row * x.row + head * x.head + lane * VE;
#pragma unroll
    for (int w = 0; w < VPL; ++w)
      if ((lane + w * LPR) * VE < dim) V::st(dst + w * LPR * VE, f[w]);
  }
  static __device__ __forceinline__ void store_f32(float *dst, int lane, int dim, const float (&f)[VPL][VE]) {
#pragma unroll
    for (int w = 0; w < VPL; ++w)
      if ((lane + w * LPR) * VE < dim) st_f32<VE>(dst + (lane + w * LPR) * VE, f[w]);
  }
};

template <int LPR>
__device__ __forceinline__ float group_sum(float x) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// u_ij in units of log 2, and the capped score's tanh (tanhf: fp32 results are held to fp32's rounding).
__device__ __forceinline__ float score2(const AttnArgs &a, float dot, float inv_cap, float slope, float dist, float &th) {
  float s = dot * a.scale;
  if (a.cap > 0.f) {
    th = tanhf(s * inv_cap);
    s = a.cap * th;
  }
  return (s - slope * dist) * kLog2e;
}

// The entries [p, pe) of a row (which ends at `end`) for head h: running maximum m, sum l and weighted sum acc, over all
// lanes of the warp. q: the row's query in the lanes of each group.
template <class H, int LPR, class Rows, int VPL, int VE>
__device__ __forceinline__ void attend(const Rows &d, const AttnArgs &a, int64_t row, int h, typename Rows::Index p,
                                       typename Rows::Index pe, typename Rows::Index end,
                                       float &m, float &l, float (&acc)[VPL][VE]) {
  constexpr int G = 32 / LPR, U = 4;
  const int lane = threadIdx.x % LPR, g = (threadIdx.x & 31) / LPR;
  const float slope = a.slopes ? __ldg(a.slopes + h) : 0.f, inv_cap = a.cap > 0.f ? 1.f / a.cap : 0.f;
  float q[VPL][VE];
  typename H::Raw raw[VPL];
  H::fetch(a.q, row, h, lane, a.dim, true, raw);
  H::widen(raw, q);
  m = -INFINITY, l = 0.f;
#pragma unroll
  for (int w = 0; w < VPL; ++w)
#pragma unroll
    for (int i = 0; i < VE; ++i) acc[w][i] = 0.f;
  for (typename Rows::Index b = p; b < pe; b += G * U) {
    typename H::Raw k[U][VPL], v[U][VPL];
    typename Rows::Index c[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const typename Rows::Index at = b + u * G + g;
      c[u] = at < pe ? d.col(at) : -1;
      const bool on = at < pe && d.in_range(c[u]);
      H::fetch(a.k, on ? c[u] : 0, h / a.group, lane, a.dim, on, k[u]);
      H::fetch(a.v, on ? c[u] : 0, h / a.group, lane, a.dim, on, v[u]);
    }
    float s[U], top = m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const typename Rows::Index at = b + u * G + g;
      float th;
      s[u] = score2(a, group_sum<LPR>(H::dot(q, k[u])), inv_cap, slope, d.distance(a, row, end, at, c[u]), th);
      if (!d.in_range(c[u])) s[u] = NAN;  // a key that does not exist: the row shows it
      if (at >= pe) s[u] = -INFINITY;
      top = fmaxf(top, s[u]);
    }
    const float base = top == -INFINITY ? 0.f : top, keep = exp2_approx(m - base);
    m = top;
    l *= keep;
#pragma unroll
    for (int w = 0; w < VPL; ++w)
#pragma unroll
      for (int i = 0; i < VE; ++i) acc[w][i] *= keep;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (b + u * G + g < pe) {
        const float x = exp2_approx(s[u] - base);
        l += x;
        H::add(acc, x, v[u]);
      }
    }
  }
  // the groups' shares of the row
#pragma unroll
  for (int o = LPR; o < 32; o <<= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), l2 = __shfl_xor_sync(0xffffffffu, l, o);
    const float top = fmaxf(m, m2), base = top == -INFINITY ? 0.f : top;
    const float f1 = exp2_approx(m - base), f2 = exp2_approx(m2 - base);
    l = l * f1 + l2 * f2;
#pragma unroll
    for (int w = 0; w < VPL; ++w)
#pragma unroll
      for (int i = 0; i < VE; ++i) acc[w][i] = acc[w][i] * f1 + __shfl_xor_sync(0xffffffffu, acc[w][i], o) * f2;
    m = top;
  }
}

// The finished row: out and lse. A row without entries gives 0 and -infinity.
template <class H, int LPR, int VPL, int VE>
__device__ __forceinline__ void put_row(const AttnArgs &a, int64_t row, int h, float m, float l, float (&acc)[VPL][VE]) {
  const int lane = threadIdx.x % LPR, g = (threadIdx.x & 31) / LPR;
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int w = 0; w < VPL; ++w)
#pragma unroll
    for (int i = 0; i < VE; ++i) acc[w][i] *= inv;
  if (g == 0) H::store(a.out, row, h, lane, a.dim, acc);
  if (a.lse && (threadIdx.x & 31) == 0) a.lse[row * a.heads + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

// A whole row once more, for head h: where products of hi + lo parts met an infinity (lo x infinity), which here stays one.
template <class T, int D, class Rows>
__device__ __noinline__ void attend_again(const Rows &d, const AttnArgs &a, int64_t row, int h) {
  using H = HeadRow<T, 8, D / 8, 1>;
  float y[1][8], m, l;
  const typename Rows::Index p = d.ptr(row), pe = d.ptr(row + 1);
  __syncwarp();  // the first result was written by other lanes than will write it now
  attend<H, D / 8>(d, a, row, h, p, pe, pe, m, l, y);
  put_row<H, D / 8>(a, row, h, m, l, y);
}

// The entries [p, pe) of a row for head h, for dq. With c = 1 - tanh^2 and delta0 = dout . out (out may be rounded): gap = sum p (dp -
// delta0) = delta - delta0, x = sum p c (dp - delta0) k, y = sum p c k, so that dq = scale (x - gap y) needs one pass. Differences from
// delta0 are as small as ds itself: what the weights are off together (lse is rounded, by 2^-24 of its size) scales dq, and
// leaves nothing of delta in it.
template <class H, int LPR, class Rows, int VPL, int VE>
__device__ __forceinline__ void attend_dq(const Rows &d, const AttnArgs &a, int64_t row, int h, int32_t p, int32_t pe,
                                          float &gap, float &delta0, float (&x)[VPL][VE], float (&y)[VPL][VE]) {
  constexpr int G = 32 / LPR, U = 4;
  const int lane = threadIdx.x % LPR, g = (threadIdx.x & 31) / LPR;
  const float slope = a.slopes ? __ldg(a.slopes + h) : 0.f, inv_cap = a.cap > 0.f ? 1.f / a.cap : 0.f;
  float q[VPL][VE], dout[VPL][VE];
  typename H::Raw raw[VPL];
  H::fetch(a.q, row, h, lane, a.dim, true, raw);
  H::widen(raw, q);
  H::fetch(a.dout, row, h, lane, a.dim, true, raw);
  H::widen(raw, dout);
  H::fetch(a.o, row, h, lane, a.dim, true, raw);
  delta0 = group_sum<LPR>(H::dot(dout, raw));
  const float lse2 = a.lse[row * a.heads + h] * kLog2e;
  gap = 0.f;
#pragma unroll
  for (int w = 0; w < VPL; ++w)
#pragma unroll
    for (int i = 0; i < VE; ++i) x[w][i] = y[w][i] = 0.f;
  for (int32_t b = p; b < pe; b += G * U) {
    typename H::Raw k[U][VPL], v[U][VPL];
    int32_t c[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int32_t at = b + u * G + g;
      c[u] = at < pe ? d.col(at) : 0;
      H::fetch(a.k, c[u], h / a.group, lane, a.dim, at < pe, k[u]);
      H::fetch(a.v, c[u], h / a.group, lane, a.dim, at < pe, v[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float th = 0.f;
      const float s = score2(a, group_sum<LPR>(H::dot(q, k[u])), inv_cap, slope, d.distance(a, row, 0, 0, c[u]), th);
      const float dp = group_sum<LPR>(H::dot(dout, v[u])) - delta0;
      if (b + u * G + g < pe) {
        const float w = lse2 == -INFINITY ? 0.f : exp2_approx(s - lse2), wc = w * (1.f - th * th);
        gap = fmaf(w, dp, gap);
        H::add(x, wc * dp, k[u]);
        H::add(y, wc, k[u]);
      }
    }
  }
#pragma unroll
  for (int o = LPR; o < 32; o <<= 1) {
    gap += __shfl_xor_sync(0xffffffffu, gap, o);
#pragma unroll
    for (int w = 0; w < VPL; ++w)
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        x[w][i] += __shfl_xor_sync(0xffffffffu, x[w][i], o);
        y[w][i] += __shfl_xor_sync(0xffffffffu, y[w][i], o);
      }
  }
}

// The entries [p, pe) of key `row` (d: the transposed pattern) for key/value head hk: dk and dv over the query heads of its
// group, one after another in the same sums.
template <class H, int LPR, class Rows, int VPL, int VE>
__device__ __forceinline__ void attend_dkv(const Rows &d, const AttnArgs &a, int64_t row, int hk, int32_t p, int32_t pe,
                                           float (&dk)[VPL][VE], float (&dv)[VPL][VE]) {
  constexpr int G = 32 / LPR, U = 4;
  const int lane = threadIdx.x % LPR, g = (threadIdx.x & 31) / LPR;
  const float inv_cap = a.cap > 0.f ? 1.f / a.cap : 0.f;
  float k[VPL][VE], v[VPL][VE];
  typename H::Raw raw[VPL];
  H::fetch(a.k, row, hk, lane, a.dim, true, raw);
  H::widen(raw, k);
  H::fetch(a.v, row, hk, lane, a.dim, true, raw);
  H::widen(raw, v);
#pragma unroll
  for (int w = 0; w < VPL; ++w)
#pragma unroll
    for (int i = 0; i < VE; ++i) dk[w][i] = dv[w][i] = 0.f;
  for (int h = hk * a.group; h < (hk + 1) * a.group; ++h) {
    const float slope = a.slopes ? __ldg(a.slopes + h) : 0.f;
    for (int32_t b = p; b < pe; b += G * U) {
      typename H::Raw q[U][VPL], dout[U][VPL];
      int32_t c[U];
      float lse2[U], delta[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int32_t at = b + u * G + g;
        c[u] = at < pe ? d.col(at) : 0;
        H::fetch(a.q, c[u], h, lane, a.dim, at < pe, q[u]);
        H::fetch(a.dout, c[u], h, lane, a.dim, at < pe, dout[u]);
        lse2[u] = at < pe ? a.lse[(int64_t)c[u] * a.heads + h] * kLog2e : -INFINITY;
        delta[u] = at >= pe ? 0.f : a.stats ? a.stats[(int64_t)c[u] * a.heads + h].y : a.delta[(int64_t)c[u] * a.heads + h];
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float th = 0.f;
        const float s = score2(a, group_sum<LPR>(H::dot(k, q[u])), inv_cap, slope,
                               fabsf((float)(c[u] + a.row_offset - row)), th);
        const float dp = group_sum<LPR>(H::dot(v, dout[u]));
        if (b + u * G + g < pe) {
          const float x = lse2[u] == -INFINITY ? 0.f : exp2_approx(s - lse2[u]);
          H::add(dv, x, dout[u]);
          H::add(dk, x * (dp - delta[u]) * (1.f - th * th) * a.scale, q[u]);
        }
      }
    }
  }
#pragma unroll
  for (int o = LPR; o < 32; o <<= 1)
#pragma unroll
    for (int w = 0; w < VPL; ++w)
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        dk[w][i] += __shfl_xor_sync(0xffffffffu, dk[w][i], o);
        dv[w][i] += __shfl_xor_sync(0xffffffffu, dv[w][i], o);
      }
}

// As attend_again, of a key.
template <class T, int D>
__device__ __noinline__ void attend_dkv_again(const PlanRows &d, const AttnArgs &a, int64_t row, int hk) {
  using H = HeadRow<T, 8, D / 8, 1>;
  float dk[1][8], dv[1][8];
  __syncwarp();
  attend_dkv<H, D / 8>(d, a, row, hk, (int32_t)d.ptr(row), (int32_t)d.ptr(row + 1), dk, dv);
  if ((threadIdx.x & 31) < D / 8) {
    H::store(a.dk, row, hk, threadIdx.x & 31, D, dk);
    H::store(a.dv, row, hk, threadIdx.x & 31, D, dv);
  }
}

}  // namespace dsp
