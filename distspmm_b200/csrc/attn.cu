// attn.cu — attention over the entries of a CSR pattern, and over cache rows listed by a CSR in device memory.
//
//   u_ij = cap tanh(scale q_i.k_j / cap) - slope |i + row_offset - j|     for the entries (i, j) of row i
//   o_i = sum_j p_ij v_j,  p_ij = exp(u_ij - lse_i),  lse_i = log sum_j exp(u_ij)
//   delta_i = dout_i.o_i,  ds_ij = p_ij (dout_i.v_j - delta_i) (1 - tanh^2) scale
//   dq_i = sum_j ds_ij k_j,  dk_j = sum_i ds_ij q_i,  dv_j = sum_i p_ij dout_i
//
// These kernels gather: for each entry and head one row of k and one of v (or of q and dout, by columns) come out of L2, two
// operations per element read, so L2's rate bounds them. A warp owns one chunk of entries (pattern.h) and one head; LPR lanes
// hold a head's row in vectors of VE elements, so 32 / LPR entries are in work side by side, each with its own running
// maximum and sum, merged when the row ends. Only listed entries are read: what other rows of k and v hold, NaN included,
// cannot reach a row that does not list them.
#include <algorithm>
#include <type_traits>

#include "attn.h"
#include "rowvec.cuh"

namespace dsp {
namespace {

constexpr int kThreads = 256;

// Rows and entries of a prepared pattern.
struct PlanRows {
  DirView d;
  __device__ int64_t chunks() const { return d.n_chunks; }
  __device__ void chunk(int64_t c, int64_t &r0, int64_t &r1, int64_t &p0, int64_t &p1) const {
    r0 = __ldg(d.row0 + c), r1 = __ldg(d.row0 + c + 1), p0 = __ldg(d.nz0 + c), p1 = __ldg(d.nz0 + c + 1);
  }
  __device__ int64_t n() const { return d.n; }
  __device__ int64_t ptr(int64_t r) const { return __ldg(d.ptr + r); }
  __device__ int64_t col(int64_t p) const { return __ldg(d.cols + p); }
  __device__ float distance(const AttnArgs &a, int64_t row, int64_t end, int64_t p, int64_t col) const {
    (void)end, (void)p;
    return fabsf((float)(row + a.row_offset - col));
  }
  __device__ bool in_range(int64_t) const { return true; }
  __device__ int32_t units() const { return d.L; }
};

// Rows listed by a CSR in device memory that nothing has validated: every value read from it is bounded before it is used,
// so that no list can make the kernel leave its operands.
struct ListRows {
  const int64_t *indptr, *indices;
  int64_t rows, nnz, keys;
  int32_t n_chunks, L;
  __device__ int64_t chunks() const { return n_chunks; }
  __device__ int64_t n() const { return rows; }
  __device__ int64_t ptr(int64_t r) const { return min(max(__ldg(indptr + r), (int64_t)0), nnz); }
  __device__ void at(int64_t x, int64_t &r, int64_t &p) const {
    int64_t lo = 0, hi = rows;
    while (lo < hi) {
      const int64_t m = (lo + hi) / 2;
      if (row_start(m, ptr(m + 1)) < x) lo = m + 1;
      else hi = m;
    }
    r = lo;
    p = lo < rows ? min(max(x - row_start(lo, 0), ptr(lo)), nnz) : ptr(rows);  // no entry behind the last row's end
  }
  __device__ void chunk(int64_t c, int64_t &r0, int64_t &r1, int64_t &p0, int64_t &p1) const {
    at(c * L, r0, p0);
    at(min((c + 1) * L, row_start(rows, nnz)), r1, p1);
  }
  __device__ int64_t col(int64_t p) const { return __ldg(indices + p); }
  __device__ float distance(const AttnArgs &, int64_t, int64_t end, int64_t p, int64_t) const { return (float)(end - 1 - p); }
  __device__ bool in_range(int64_t c) const { return c >= 0 && c < keys; }
  __device__ int32_t units() const { return L; }
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
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < VPL; ++w) {
      float f[VE];
      V::widen(r[w], f);
#pragma unroll
      for (int i = 0; i < VE; ++i) s = fmaf(x[w][i], f[i], s);
    }
    return s;
  }
  static __device__ __forceinline__ void add(float (&acc)[VPL][VE], float x, const Raw (&r)[VPL]) {
#pragma unroll
    for (int w = 0; w < VPL; ++w) {
      float f[VE];
      V::widen(r[w], f);
#pragma unroll
      for (int i = 0; i < VE; ++i) acc[w][i] = fmaf(x, f[i], acc[w][i]);
    }
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

// u_ij in units of log 2, and the capped score's tanh.
__device__ __forceinline__ float score2(const AttnArgs &a, float dot, float inv_cap2, float slope, float dist, float &th) {
  float s = dot * a.scale;
  if (a.cap > 0.f) s = capped(s, a.cap, inv_cap2, th);
  return (s - slope * dist) * kLog2e;
}

template <class Rows, class T, int VE, int LPR, int VPL>
__global__ void __launch_bounds__(kThreads) attn_rows_kernel(const Rows d, const AttnArgs a) {
  using H = HeadRow<T, VE, LPR, VPL>;
  constexpr int G = 32 / LPR, U = 4;
  const int64_t item = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> 5;
  const int64_t chunk = item / a.heads;
  const int h = (int)(item - chunk * a.heads);
  if (chunk >= d.chunks()) return;
  const int lane = threadIdx.x % LPR, g = (threadIdx.x & 31) / LPR;
  const float slope = a.slopes ? __ldg(a.slopes + h) : 0.f, inv_cap2 = a.cap > 0.f ? 2.f * kLog2e / a.cap : 0.f;
  int64_t r0, r1, p0, p1;
  d.chunk(chunk, r0, r1, p0, p1);
  const bool head_cut = p0 > d.ptr(r0);
  int64_t p = p0;
  for (int64_t row = r0; row <= r1; ++row) {
    if (row == r1 && (p >= p1 || row >= d.n())) break;
    const int64_t end = d.ptr(row + 1), pe = row < r1 ? end : p1;
    float q[VPL][VE], acc[VPL][VE], m = -INFINITY, l = 0.f;
    typename H::Raw raw[VPL];
    H::fetch(a.q, row, h, lane, a.dim, true, raw);
    H::widen(raw, q);
#pragma unroll
    for (int w = 0; w < VPL; ++w)
#pragma unroll
      for (int i = 0; i < VE; ++i) acc[w][i] = 0.f;
    for (int64_t b = p; b < pe; b += G * U) {
      typename H::Raw k[U][VPL], v[U][VPL];
      int64_t c[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t at = b + u * G + g;
        c[u] = at < pe ? d.col(at) : -1;
        const bool on = at < pe && d.in_range(c[u]);
        H::fetch(a.k, on ? c[u] : 0, h / a.group, lane, a.dim, on, k[u]);
        H::fetch(a.v, on ? c[u] : 0, h / a.group, lane, a.dim, on, v[u]);
      }
      float s[U], top = m;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t at = b + u * G + g;
        float th;
        s[u] = score2(a, group_sum<LPR>(H::dot(q, k[u])), inv_cap2, slope, d.distance(a, row, end, at, c[u]), th);
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
    const bool cut_head = row == r0 && head_cut;
    if (cut_head || row == r1) {
      const int64_t slot = (cut_head ? 2 * chunk : 2 * chunk + 1) * a.heads + h;
      if (g == 0) H::store_f32(a.slots + slot * a.dim, lane, a.dim, acc);
      if ((threadIdx.x & 31) == 0) a.slot_ml[2 * slot] = m, a.slot_ml[2 * slot + 1] = l;
    } else {
      const float inv = l == 0.f ? 0.f : 1.f / l;  // a row without entries gives 0
#pragma unroll
      for (int w = 0; w < VPL; ++w)
#pragma unroll
        for (int i = 0; i < VE; ++i) acc[w][i] *= inv;
      if (g == 0) H::store(a.out, row, h, lane, a.dim, acc);
      if (a.lse && (threadIdx.x & 31) == 0) a.lse[row * a.heads + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
    }
    p = pe;
  }
}

// dq of the pattern's rows.
template <class T, int VE, int LPR, int VPL>
__global__ void __launch_bounds__(kThreads) attn_dq_kernel(const DirView d, const AttnArgs a) {
  using H = HeadRow<T, VE, LPR, VPL>;
  constexpr int G = 32 / LPR, U = 4;
  const int64_t item = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> 5;
  const int64_t chunk = item / a.heads;
  const int h = (int)(item - chunk * a.heads);
  if (chunk >= d.n_chunks) return;
  const int lane = threadIdx.x % LPR, g = (threadIdx.x & 31) / LPR;
  const float slope = a.slopes ? __ldg(a.slopes + h) : 0.f, inv_cap2 = a.cap > 0.f ? 2.f * kLog2e / a.cap : 0.f;
  const int32_t r0 = __ldg(d.row0 + chunk), r1 = __ldg(d.row0 + chunk + 1);
  const int32_t p1 = __ldg(d.nz0 + chunk + 1);
  int32_t p = __ldg(d.nz0 + chunk);
  const bool head_cut = p > __ldg(d.ptr + r0);
  for (int32_t row = r0; row <= r1; ++row) {
    const int32_t pe = row < r1 ? __ldg(d.ptr + row + 1) : p1;
    if (row == r1 && p >= pe) break;
    float q[VPL][VE], dout[VPL][VE], acc[VPL][VE];
    typename H::Raw raw[VPL];
    H::fetch(a.q, row, h, lane, a.dim, true, raw);
    H::widen(raw, q);
    H::fetch(a.dout, row, h, lane, a.dim, true, raw);
    H::widen(raw, dout);
    const float lse2 = a.lse[(int64_t)row * a.heads + h] * kLog2e, delta = a.delta[(int64_t)row * a.heads + h];
#pragma unroll
    for (int w = 0; w < VPL; ++w)
#pragma unroll
      for (int i = 0; i < VE; ++i) acc[w][i] = 0.f;
    for (int32_t b = p; b < pe; b += G * U) {
      typename H::Raw k[U][VPL], v[U][VPL];
      int32_t c[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int32_t at = b + u * G + g;
        c[u] = at < pe ? __ldg(d.cols + at) : 0;
        H::fetch(a.k, c[u], h / a.group, lane, a.dim, at < pe, k[u]);
        H::fetch(a.v, c[u], h / a.group, lane, a.dim, at < pe, v[u]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float th = 0.f;
        const float s = score2(a, group_sum<LPR>(H::dot(q, k[u])), inv_cap2, slope,
                               fabsf((float)((int64_t)row + a.row_offset - c[u])), th);
        const float dp = group_sum<LPR>(H::dot(dout, v[u]));
        if (b + u * G + g < pe) {
          const float x = lse2 == -INFINITY ? 0.f : exp2_approx(s - lse2);
          H::add(acc, x * (dp - delta) * (1.f - th * th) * a.scale, k[u]);
        }
      }
    }
#pragma unroll
    for (int o = LPR; o < 32; o <<= 1)
#pragma unroll
      for (int w = 0; w < VPL; ++w)
#pragma unroll
        for (int i = 0; i < VE; ++i) acc[w][i] += __shfl_xor_sync(0xffffffffu, acc[w][i], o);
    const bool cut_head = row == r0 && head_cut;
    if (g == 0) {
      if (cut_head || row == r1)
        H::store_f32(a.slots + ((cut_head ? 2 * chunk : 2 * chunk + 1) * a.heads + h) * a.dim, lane, a.dim, acc);
      else
        H::store(a.dq, row, h, lane, a.dim, acc);
    }
    p = pe;
  }
}

// dk and dv of the pattern's columns (d: the transposed pattern), one key/value head: the query heads of its group follow one
// another in the same sums.
template <class T, int VE, int LPR, int VPL>
__global__ void __launch_bounds__(kThreads) attn_dkv_kernel(const DirView d, const AttnArgs a) {
  using H = HeadRow<T, VE, LPR, VPL>;
  constexpr int G = 32 / LPR, U = 4;
  const int kv_heads = a.heads / a.group;
  const int64_t item = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> 5;
  const int64_t chunk = item / kv_heads;
  const int hk = (int)(item - chunk * kv_heads);
  if (chunk >= d.n_chunks) return;
  const int lane = threadIdx.x % LPR, g = (threadIdx.x & 31) / LPR;
  const float inv_cap2 = a.cap > 0.f ? 2.f * kLog2e / a.cap : 0.f;
  const int32_t r0 = __ldg(d.row0 + chunk), r1 = __ldg(d.row0 + chunk + 1);
  const int32_t p1 = __ldg(d.nz0 + chunk + 1);
  int32_t p = __ldg(d.nz0 + chunk);
  const bool head_cut = p > __ldg(d.ptr + r0);
  for (int32_t row = r0; row <= r1; ++row) {  // a row here is a column of A
    const int32_t pe = row < r1 ? __ldg(d.ptr + row + 1) : p1;
    if (row == r1 && p >= pe) break;
    float k[VPL][VE], v[VPL][VE], dk[VPL][VE], dv[VPL][VE];
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
          c[u] = at < pe ? __ldg(d.cols + at) : 0;
          H::fetch(a.q, c[u], h, lane, a.dim, at < pe, q[u]);
          H::fetch(a.dout, c[u], h, lane, a.dim, at < pe, dout[u]);
          lse2[u] = at < pe ? a.lse[(int64_t)c[u] * a.heads + h] * kLog2e : -INFINITY;
          delta[u] = at < pe ? a.delta[(int64_t)c[u] * a.heads + h] : 0.f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float th = 0.f;
          const float s = score2(a, group_sum<LPR>(H::dot(k, q[u])), inv_cap2, slope,
                                 fabsf((float)((int64_t)c[u] + a.row_offset - row)), th);
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

// delta_i = dout_i . out_i of each row and head, a warp each.
template <class T>
__global__ void __launch_bounds__(kThreads) attn_delta_kernel(int64_t rows, const AttnArgs a) {
  const int64_t item = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> 5;
  const int64_t row = item / a.heads;
  const int h = (int)(item - row * a.heads), lane = threadIdx.x & 31;
  if (row >= rows) return;
  const T *x = (const T *)a.dout.p + row * a.dout.row + h * a.dout.head, *y = (const T *)a.o.p + row * a.o.row + h * a.o.head;
  float s = 0.f;
  for (int i = lane; i < a.dim; i += 32) s = fmaf((float)x[i], (float)y[i], s);
  s = group_sum<32>(s);
  if (lane == 0) a.delta[item] = s;
}

// Partials of cut rows (forward): merged in chunk order. blockIdx.y: head. Lane l holds columns l, l + 32, ...
template <class Rows, class T>
__global__ void __launch_bounds__(kThreads) attn_join_kernel(const Rows d, const int32_t *split_row, int n_split, const AttnArgs a) {
  const int lane = threadIdx.x & 31, h = blockIdx.y;
  const int64_t at = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (at >= n_split) return;
  const int64_t r = split_row ? __ldg(split_row + at) : at;
  const int64_t L = d.units(), last = d.chunks() - 1;
  const int64_t c0 = row_start(r, d.ptr(r)) / L, c1 = min(row_start(r, d.ptr(r + 1)) / L, last);
  if (c0 >= c1) return;  // not cut
  float m = -INFINITY, l = 0.f, acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.f;
#pragma unroll 4
  for (int64_t c = c0; c <= c1; ++c) {
    const int64_t slot = (c == c0 ? 2 * c + 1 : 2 * c) * a.heads + h;
    const float m2 = a.slot_ml[2 * slot], l2 = a.slot_ml[2 * slot + 1];
    const float top = fmaxf(m, m2), base = top == -INFINITY ? 0.f : top;
    const float f1 = exp2_approx(m - base), f2 = exp2_approx(m2 - base);
    l = l * f1 + l2 * f2;
    m = top;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < a.dim) acc[i] = acc[i] * f1 + a.slots[slot * a.dim + lane + 32 * i] * f2;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T *dst = (T *)a.out.p + r * a.out.row + h * a.out.head;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (lane + 32 * i < a.dim) dst[lane + 32 * i] = T(acc[i] * inv);
  if (a.lse && lane == 0) a.lse[r * a.heads + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

// Partials of cut rows (gradients): sums in chunk order. n_heads x width floats per slot; the first dim columns go to x, the
// others to y.
template <class T>
__global__ void __launch_bounds__(kThreads) attn_sum_kernel(const DirView d, const float *slots, int n_heads, int width, int dim,
                                                            HeadsOut x, HeadsOut y) {
  const int lane = threadIdx.x & 31, h = blockIdx.y;
  const int64_t at = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (at >= d.n_split) return;
  const int64_t r = __ldg(d.split_row + at);
  const int64_t c0 = row_start(r, __ldg(d.ptr + r)) / d.L, c1 = row_start(r, __ldg(d.ptr + r + 1)) / d.L;
  for (int col = lane; col < width; col += 32) {
    float s = 0.f;
#pragma unroll 4
    for (int64_t c = c0; c <= c1; ++c) s += slots[((c == c0 ? 2 * c + 1 : 2 * c) * n_heads + h) * width + col];
    if (col < dim) ((T *)x.p)[r * x.row + h * x.head + col] = T(s);
    else ((T *)y.p)[r * y.row + h * y.head + col - dim] = T(s);
  }
}

// ------------------------------------------------------------------------------------------------ launches

int64_t up256(int64_t x) { return (x + 255) / 256 * 256; }

int status(const char *who) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? DSP_OK : fail(DSP_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
}

unsigned warps_grid(int64_t warps) { return (unsigned)((warps + kThreads / 32 - 1) / (kThreads / 32)); }

enum Pass { kForward, kDq, kDkv };

template <class Rows, class T, int VE, int LPR, int VPL>
void launch_shape(Pass pass, const Rows &rows, const DirView &d, const AttnArgs &a, int64_t n_chunks, cudaStream_t s) {
  const int64_t warps = n_chunks * (pass == kDkv ? a.heads / a.group : a.heads);
  if (pass == kForward) {
    attn_rows_kernel<Rows, T, VE, LPR, VPL><<<warps_grid(warps), kThreads, 0, s>>>(rows, a);
  } else if constexpr (std::is_same<Rows, PlanRows>::value) {
    if (pass == kDq) attn_dq_kernel<T, VE, LPR, VPL><<<warps_grid(warps), kThreads, 0, s>>>(d, a);
    else attn_dkv_kernel<T, VE, LPR, VPL><<<warps_grid(warps), kThreads, 0, s>>>(d, a);
  }
}

template <class Rows, class T>
void launch_pass(Pass pass, const Rows &rows, const DirView &d, const AttnArgs &a, int64_t n_chunks, cudaStream_t s) {
  if (n_chunks == 0) return;
  if constexpr (sizeof(T) == 2) {
    if (a.dim <= 32) launch_shape<Rows, T, 8, 4, 1>(pass, rows, d, a, n_chunks, s);
    else if (a.dim <= 64) launch_shape<Rows, T, 8, 8, 1>(pass, rows, d, a, n_chunks, s);
    else if (a.dim <= 128) launch_shape<Rows, T, 8, 16, 1>(pass, rows, d, a, n_chunks, s);
    else launch_shape<Rows, T, 8, 32, 1>(pass, rows, d, a, n_chunks, s);
  } else {
    if (a.dim <= 32) launch_shape<Rows, T, 4, 8, 1>(pass, rows, d, a, n_chunks, s);
    else if (a.dim <= 64) launch_shape<Rows, T, 4, 16, 1>(pass, rows, d, a, n_chunks, s);
    else if (a.dim <= 128) launch_shape<Rows, T, 4, 32, 1>(pass, rows, d, a, n_chunks, s);
    else launch_shape<Rows, T, 4, 32, 2>(pass, rows, d, a, n_chunks, s);
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
  int64_t delta, slots, total;
};
GradPlan grad_plan(const dsp_pattern *p, const dsp_attn_desc *d) {
  GradPlan g = {};
  g.slots = up256(4 * p->rows * d->heads);
  const int64_t q = p->a.n_split ? 8ll * p->a.n_chunks * d->heads * d->dim : 0;
  const int64_t kv = p->t.n_split ? 16ll * p->t.n_chunks * d->kv_heads * d->dim : 0;
  g.total = g.slots + up256(std::max(q, kv));  // dq's partials are joined before dk's and dv's are written
  return g;
}

template <class T>
int forward(const dsp_pattern *p, const dsp_attn_desc *d, char *ws, cudaStream_t s) {
  AttnArgs a = args_of(d);
  const ForwardPlan f = forward_plan(p->a.n_chunks, p->a.n_split > 0, d->heads, d->dim);
  a.slots = (float *)ws;
  a.slot_ml = (float *)(ws + f.ml);
  const PlanRows rows = {view(p->a)};
  launch_pass<PlanRows, T>(kForward, rows, rows.d, a, p->a.n_chunks, s);
  if (p->a.n_split)
    attn_join_kernel<PlanRows, T>
        <<<dim3((unsigned)((p->a.n_split + 7) / 8), (unsigned)d->heads), kThreads, 0, s>>>(rows, p->a.split_row, p->a.n_split, a);
  return status("dsp_attn");
}

template <class T>
int gradients(const dsp_pattern *p, const dsp_attn_grad_desc *g, char *ws, cudaStream_t s) {
  const dsp_attn_desc *d = &g->fwd;
  AttnArgs a = args_of(d);
  const GradPlan f = grad_plan(p, d);
  a.dout = {g->dout, g->dout_row, g->dout_head};
  a.dq = {g->dq, g->dq_row, g->dq_head};
  a.dk = {g->dk, g->dk_row, g->dk_head};
  a.dv = {g->dv, g->dv_row, g->dv_head};
  a.delta = (float *)ws;
  a.slots = (float *)(ws + f.slots);
  if (p->rows) attn_delta_kernel<T><<<warps_grid(p->rows * d->heads), kThreads, 0, s>>>(p->rows, a);
  const DirView va = view(p->a), vt = view(p->t);
  launch_pass<PlanRows, T>(kDq, PlanRows{va}, va, a, va.n_chunks, s);
  if (va.n_split)
    attn_sum_kernel<T><<<dim3((unsigned)((va.n_split + 7) / 8), (unsigned)d->heads), kThreads, 0, s>>>(va, a.slots, d->heads, d->dim,
                                                                                                     d->dim, a.dq, a.dq);
  launch_pass<PlanRows, T>(kDkv, PlanRows{vt}, vt, a, vt.n_chunks, s);
  if (vt.n_split)
    attn_sum_kernel<T><<<dim3((unsigned)((vt.n_split + 7) / 8), (unsigned)d->kv_heads), kThreads, 0, s>>>(
        vt, a.slots, d->kv_heads, 2 * d->dim, d->dim, a.dk, a.dv);
  return status("dsp_attn_grad");
}

// Units of a chunk for a list of nnz entries: some 16 warps for every SM over all heads.
int32_t list_units(int64_t rows, int64_t nnz, int heads) {
  const int64_t l = (row_start(rows, nnz) * heads + 148 * 16 - 1) / (148 * 16);
  return (int32_t)std::min<int64_t>(1024, std::max<int64_t>(64, (l + 31) / 32 * 32));
}

template <class T>
int decode(const dsp_attn_decode_desc *g, char *ws, cudaStream_t s) {
  const dsp_attn_desc *d = &g->fwd;
  AttnArgs a = args_of(d);
  ListRows rows = {g->indptr, g->indices, g->rows, g->nnz, g->keys, 0, list_units(g->rows, g->nnz, d->heads)};
  rows.n_chunks = (int32_t)((row_start(g->rows, g->nnz) + rows.L - 1) / rows.L);
  const ForwardPlan f = forward_plan(rows.n_chunks, true, d->heads, d->dim);
  a.slots = (float *)ws;
  a.slot_ml = (float *)(ws + f.ml);
  launch_pass<ListRows, T>(kForward, rows, DirView{}, a, rows.n_chunks, s);
  attn_join_kernel<ListRows, T>
      <<<dim3((unsigned)((g->rows + 7) / 8), (unsigned)d->heads), kThreads, 0, s>>>(rows, nullptr, (int)g->rows, a);
  return status("dsp_attn_decode");
}

int check_heads(const char *who, const char *name, const void *p, int64_t row, int64_t head, int dtype) {
  const int64_t e = dtype == DSP_F32 ? 4 : 2;
  DSP_TRY_ARG(p, "%s: %s is null", who, name);
  DSP_TRY_ARG(((uintptr_t)p & 15) == 0 && row * e % 16 == 0 && head * e % 16 == 0,
              "%s: %s and its strides (%lld, %lld) must be multiples of 16 bytes", who, name, (long long)row, (long long)head);
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
  DSP_TRY_ARG(d->scale == d->scale && d->softcap >= 0.f && d->softcap < INFINITY, "%s: scale %g, softcap %g", who, d->scale, d->softcap);
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
  return forward_plan(p->a.n_chunks, p->a.n_split > 0, d->heads, d->dim).total;
}

extern "C" int dsp_attn(const dsp_pattern *p, const dsp_attn_desc *d, void *workspace, int64_t workspace_bytes, void *stream) {
  const char *who = "dsp_attn";
  DSP_TRY_ARG(p && d, "%s: null argument", who);
  if (!(p->flags & DSP_PATTERN_ATTENTION)) return fail(DSP_ERR_STATE, "%s: needs a pattern with DSP_PATTERN_ATTENTION", who);
  int rc = check_attn(who, d, p->rows, p->nnz ? p->cols : 0);
  if (rc) return rc;
  if (p->rows == 0) return DSP_OK;
  rc = check_workspace(who, workspace, workspace_bytes, dsp_attn_workspace(p, d));
  if (rc) return rc;
  DeviceGuard g(p->device);
  if (g.err != cudaSuccess) return fail(DSP_ERR_CUDA, "%s: %s", who, cudaGetErrorString(g.err));
  if (d->dtype == DSP_F32) return forward<float>(p, d, (char *)workspace, (cudaStream_t)stream);
  if (d->dtype == DSP_BF16) return forward<__nv_bfloat16>(p, d, (char *)workspace, (cudaStream_t)stream);
  return forward<__half>(p, d, (char *)workspace, (cudaStream_t)stream);
}

extern "C" int64_t dsp_attn_grad_workspace(const dsp_pattern *p, const dsp_attn_desc *d) {
  if (!p || !usable(d)) return 0;
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
    if ((rc = check_heads(who, "dout", g->dout, g->dout_row, g->dout_head, d->dtype)) ||
        (rc = check_heads(who, "dq", g->dq, g->dq_row, g->dq_head, d->dtype)))
      return rc;
  }
  if (p->cols > 0 && ((rc = check_heads(who, "dk", g->dk, g->dk_row, g->dk_head, d->dtype)) ||
                      (rc = check_heads(who, "dv", g->dv, g->dv_row, g->dv_head, d->dtype))))
    return rc;
  rc = check_workspace(who, workspace, workspace_bytes, dsp_attn_grad_workspace(p, d));
  if (rc) return rc;
  DeviceGuard dg(p->device);
  if (dg.err != cudaSuccess) return fail(DSP_ERR_CUDA, "%s: %s", who, cudaGetErrorString(dg.err));
  if (d->dtype == DSP_F32) return gradients<float>(p, g, (char *)workspace, (cudaStream_t)stream);
  if (d->dtype == DSP_BF16) return gradients<__nv_bfloat16>(p, g, (char *)workspace, (cudaStream_t)stream);
  return gradients<__half>(p, g, (char *)workspace, (cudaStream_t)stream);
}

extern "C" int64_t dsp_attn_decode_workspace(const dsp_attn_decode_desc *g) {
  if (!g || !usable(&g->fwd) || g->rows < 0 || g->nnz < 0) return 0;
  const int64_t L = list_units(g->rows, g->nnz, g->fwd.heads);
  return forward_plan((row_start(g->rows, g->nnz) + L - 1) / L, true, g->fwd.heads, g->fwd.dim).total;
}

extern "C" int dsp_attn_decode(const dsp_attn_decode_desc *g, void *workspace, int64_t workspace_bytes, void *stream) {
  const char *who = "dsp_attn_decode";
  DSP_TRY_ARG(g, "%s: null argument", who);
  DSP_TRY_ARG(g->rows >= 0 && g->nnz >= 0 && g->keys >= 0, "%s: negative size", who);
  if (g->rows > (1 << 24) || g->nnz >= INT32_MAX) return fail(DSP_ERR_UNSUPPORTED, "%s: %lld rows, %lld entries", who, (long long)g->rows, (long long)g->nnz);
  int rc = check_attn(who, &g->fwd, g->rows, g->keys);
  if (rc) return rc;
  if (g->rows == 0) return DSP_OK;
  DSP_TRY_ARG(g->indptr && (g->indices || g->nnz == 0), "%s: null index list", who);
  rc = check_workspace(who, workspace, workspace_bytes, dsp_attn_decode_workspace(g));
  if (rc) return rc;
  if (g->fwd.dtype == DSP_F32) return decode<float>(g, (char *)workspace, (cudaStream_t)stream);
  if (g->fwd.dtype == DSP_BF16) return decode<__nv_bfloat16>(g, (char *)workspace, (cudaStream_t)stream);
  return decode<__half>(g, (char *)workspace, (cudaStream_t)stream);
}
