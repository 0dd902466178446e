// attn_graph.cu — attention over a pattern's entries, row by row, 16-bit operands of dim 32, 64 or 128: forward, dq, and dk, dv.
//
// For patterns too thin for tiles (a graph's edges). The formulas are those of attn.cu; what bounds both is the gather of a row
// of k and one of v (q and dout, by columns) for each entry and head out of L2. Here the arithmetic is given to mma.sync, though
// an entry has but one query to be multiplied with (of m16n8k16 products, 16 rows are entries and 1 to 8 columns are query
// heads): 16 entries of dim 64 take some 120 instructions where dot products by shuffles took 780 (R-MAT 15, 8 heads of 64).
//
//   pass      rows of 16 entries      columns                      then, turned
//   forward   k                       q of up to 8 heads           v   x weights
//   dq        k, v                    q, dout of up to 4 heads,    k   x [p c dp | p c]   (x and y of attn_row.cuh)
//                                     twice
//   dk, dv    q, dout of one head     k, v (one key, twice)        dout x p, q x p c (dp - delta): hi and lo parts in the columns
//
// A warp owns a chunk (pattern.h) and a head or group; its column ids and row pointers are staged in shared memory, and the walk
// over 16-entry steps runs on across rows: the next step's rows are requested as soon as the present ones are in the products,
// so a short row costs no wait. Weights enter the second product as hi + lo, as exact as fp32.
#include <algorithm>
#include <type_traits>

#include "attn_graph.h"
#include "frag.cuh"

namespace dsp {
namespace {

constexpr int kThreads = 128;

struct Lists {
  int32_t cols[kMaxUnits];
  int32_t ptr[kMaxUnits / kRowUnits + 4];
};

// A step: 16 entries from b on, of a row whose entries in this chunk end at pe, for query head number h of the group (dk, dv).
struct Step {
  int32_t row, b, pe, h;
};

template <class T, int D, AttnPass M>
__global__ void __launch_bounds__(kThreads, D == 128 ? (M == kDkv ? 2 : 3) : (M == kDkv ? 3 : 4))
    attn_graph_kernel(const DirView d, const AttnArgs a, int head_tiles) {
  constexpr int VR = D / 32, VT = kTurned<D>, NT = kTiles<D>;
  constexpr int kWidth = M == kForward ? 8 : M == kDq ? 4 : 1;  // query heads of a warp's columns
  __shared__ Lists all_lists[kThreads / 32];
  const int lane = threadIdx.x & 31, t = lane & 3, n8 = lane >> 2;
  const int kv_heads = a.heads / a.group, per_chunk = kv_heads * head_tiles;
  const int64_t item = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> 5;
  const int64_t chunk = item / per_chunk;
  if (chunk >= d.n_chunks) return;
  const int hk = (int)(item - chunk * per_chunk) / head_tiles, h0 = hk * a.group + (int)(item % head_tiles) * kWidth;
  const int live = M == kDkv ? 1 : min(kWidth, (hk + 1) * a.group - h0);  // query heads h0 .. h0 + live - 1
  Lists &list = all_lists[threadIdx.x >> 5];
  const int32_t r0 = __ldg(d.row0 + chunk), r1 = __ldg(d.row0 + chunk + 1), p0 = __ldg(d.nz0 + chunk), p1 = __ldg(d.nz0 + chunk + 1);
  for (int i = lane; i <= r1 - r0 + 1; i += 32)
    if (r0 + i <= d.n) list.ptr[i] = __ldg(d.ptr + r0 + i);
#pragma unroll 4
  for (int i = lane; i < p1 - p0; i += 32) list.cols[i] = __ldg(d.cols + p0 + i);
  __syncwarp();
  const int32_t *cols = list.cols - p0;
  const bool head_cut = p0 > list.ptr[0];
  constexpr bool kHalf = std::is_same<T, __half>::value;
  // fp16: score gradients carry the factor up, weights of dk, dv 2^12; both come off at the row's end
  const float up = kHalf && M != kForward ? dout_scale(a.dout_max) : 1.f, down = 1.f / up;
  constexpr float kUp = kHalf && M == kDkv ? 4096.f : 1.f;
  const float inv_cap2 = a.cap > 0.f ? 2.f * kLog2e / a.cap : 0.f, scale2 = a.scale * kLog2e;

  // places this lane's columns 2 t, 2 t + 1 have among the heads
  auto head_of = [&](int j) { return M == kForward ? 2 * t + j : M == kDq ? (2 * t + j) & 3 : 0; };
  float slope2[2];
#pragma unroll
  for (int j = 0; j < 2; ++j)
    slope2[j] = M != kDkv && a.slopes && head_of(j) < live ? __ldg(a.slopes + h0 + head_of(j)) * kLog2e : 0.f;

  auto first_of = [&](Step s) {  // the first row from s.row on with entries in this chunk; row r1 + 1: none
    for (; s.row <= r1; ++s.row) {
      s.pe = s.row < r1 ? list.ptr[s.row - r0 + 1] : p1;
      if (s.pe > s.b) break;
    }
    s.h = 0;
    return s;
  };
  auto next_of = [&](const Step &s) {
    Step n = s;
    n.b += 16;
    if (n.b < s.pe) return n;
    if (M == kDkv && s.h + 1 < a.group) {
      n.b = s.row == r0 ? p0 : list.ptr[s.row - r0];
      ++n.h;
      return n;
    }
    n.b = s.pe;
    ++n.row;
    return first_of(n);
  };
  // rows from .. to - 1 have no entry here: zeros, or an empty share of a row cut before this chunk
  auto idle = [&](int32_t from, int32_t to) {
    for (int32_t row = from; row < min(to, r1); ++row) {
      const bool cut = row == r0 && head_cut;
      const uint4 zero = make_uint4(0, 0, 0, 0);
      if (M == kDkv) {
        if (cut) {
          float *dst = a.slots + (2 * chunk * kv_heads + hk) * 2 * D;
          for (int i = lane; i < D / 2; i += 32) reinterpret_cast<uint4 *>(dst)[i] = zero;
        } else if (lane < D / 8) {
          *reinterpret_cast<uint4 *>((T *)a.dk.p + (int64_t)row * a.dk.row + (int64_t)hk * a.dk.head + 8 * lane) = zero;
          *reinterpret_cast<uint4 *>((T *)a.dv.p + (int64_t)row * a.dv.row + (int64_t)hk * a.dv.head + 8 * lane) = zero;
        }
        continue;
      }
      for (int j = 0; j < live; ++j) {
        const int h = h0 + j;
        const int64_t slot = 2 * chunk * a.heads + h;
        if (cut) {
          constexpr int width = M == kForward ? D : 2 * D;
          for (int i = lane; i < width / 4; i += 32) reinterpret_cast<uint4 *>(a.slots + slot * width)[i] = zero;
          if (lane == 0 && M == kForward) a.slot_ml[2 * slot] = -INFINITY, a.slot_ml[2 * slot + 1] = 0.f;
          if (lane == 0 && M == kDq) a.slot_ml[slot] = 0.f;
        } else {
          const HeadsOut &o = M == kForward ? a.out : a.dq;
          if (lane < D / 8) *reinterpret_cast<uint4 *>((T *)o.p + (int64_t)row * o.row + (int64_t)h * o.head + 8 * lane) = zero;
          if (lane == 0 && M == kForward && a.lse) a.lse[(int64_t)row * a.heads + h] = -INFINITY;
          if (lane == 0 && M == kDq) a.delta[(int64_t)row * a.heads + h] = 0.f;
        }
      }
    }
  };

  // gathers: rows n8, n8 + 8 of a step; turned rows
  auto load_rows = [&](uint4(&x)[2][VR], const Heads &m, const Step &s, int head) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int32_t at = s.b + n8 + 8 * j;
      const bool on = at < s.pe;
      const T *src = (const T *)m.p + (int64_t)cols[on ? at : s.b] * m.row + (int64_t)head * m.head + t * 8;
#pragma unroll
      for (int i = 0; i < VR; ++i) x[j][i] = on ? __ldg(reinterpret_cast<const uint4 *>(src + 32 * i)) : make_uint4(0, 0, 0, 0);
    }
  };
  auto load_turned = [&](uint4(&x)[4][VT], const Heads &m, const Step &s, int head) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int32_t at = s.b + 2 * t + (j & 1) + 8 * (j >> 1);
      const bool on = at < s.pe && (D >= 64 || n8 < D / 8);
      const T *src = (const T *)m.p + (int64_t)cols[at < s.pe ? at : s.b] * m.row + (int64_t)head * m.head + n8 * 8;
#pragma unroll
      for (int i = 0; i < VT; ++i) x[j][i] = on ? __ldg(reinterpret_cast<const uint4 *>(src + 64 * i)) : make_uint4(0, 0, 0, 0);
    }
  };
  auto head_at = [&](const Step &s) { return M == kDkv ? hk * a.group + s.h : hk; };

  // element values of this lane's columns of a 16 x 8-column result: f[8] of vector n8 + 8 i for column j
  auto elements = [&](const float(&acc)[NT][4], int i, int j, float(&f)[8]) {
#pragma unroll
    for (int c = 0; c < 4; ++c) f[2 * c] = acc[4 * i + c][j], f[2 * c + 1] = acc[4 * i + c][2 + j];
  };

  Step now = first_of({r0, p0, 0, 0});
  idle(r0, now.row);
  if (now.row > r1) return;

  uint4 x0[2][VR], x1[M == kForward ? 1 : 2][VR];  // k; v    (dk, dv: q; dout)
  uint4 xt[4][VT];                                 // forward: v turned, requested ahead; else loaded in its place
  load_rows(x0, M == kDkv ? a.q : a.k, now, head_at(now));
  if constexpr (M != kForward) load_rows(x1, M == kDkv ? a.dout : a.v, now, head_at(now));
  else load_turned(xt, a.v, now, hk);
  float lse_e[2] = {0.f, 0.f}, delta_e[2] = {0.f, 0.f};  // dk, dv: of the queries n8, n8 + 8
  auto load_stats = [&](const Step &s) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int32_t at = s.b + n8 + 8 * j;
      const int64_t i = (int64_t)cols[at < s.pe ? at : s.b] * a.heads + head_at(s);
      lse_e[j] = __ldg(a.lse + i);
      delta_e[j] = a.delta[i];
    }
  };
  if (M == kDkv) load_stats(now);

  int32_t row = -1;
  uint32_t c0[D / 16][2], c1[M == kForward ? 1 : D / 16][2];  // columns: q; dout    (dk, dv: k; v)
  float acc[NT][4], acc2[M == kDkv ? NT : 1][4];
  float m[2], l[2], lse2[2];  // forward: maximum, sum; dq: l is delta

#pragma unroll 1
  while (true) {
    if (now.row != row) {
      row = now.row;
      if (M == kDkv) {
        load_column<T, D>(c0, (const T *)a.k.p + (int64_t)row * a.k.row + (int64_t)hk * a.k.head, n8 < 2);
        if constexpr (M != kForward) load_column<T, D>(c1, (const T *)a.v.p + (int64_t)row * a.v.row + (int64_t)hk * a.v.head, n8 < 2);
      } else {
        const int h = M == kForward ? n8 : n8 & 3;
        load_column<T, D>(c0, (const T *)a.q.p + (int64_t)row * a.q.row + (int64_t)(h0 + h) * a.q.head, h < live);
        if constexpr (M == kDq) {
          load_column<T, D>(c1, (const T *)a.dout.p + (int64_t)row * a.dout.row + (int64_t)(h0 + h) * a.dout.head, h < live);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            lse2[j] = head_of(j) < live ? __ldg(a.lse + (int64_t)row * a.heads + h0 + head_of(j)) * kLog2e : 0.f;
            if (lse2[j] == -INFINITY) lse2[j] = INFINITY;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          acc[i][j] = 0.f;
          if constexpr (M == kDkv) acc2[i][j] = 0.f;
        }
      m[0] = m[1] = -INFINITY, l[0] = l[1] = 0.f;
    }
    const Step next = next_of(now);
    const bool more = next.row <= r1;
    float s[4] = {0.f, 0.f, 0.f, 0.f}, dp[4] = {0.f, 0.f, 0.f, 0.f};
    rows_times<T, D>(s, x0, c0);
    if constexpr (M != kForward) rows_times<T, D>(dp, x1, c1);
    float lse_n[2] = {lse_e[0], lse_e[1]}, delta_n[2] = {delta_e[0], delta_e[1]};
    // the next step's rows; of this one the turned rows, which the first product has brought to L1
    if constexpr (M == kDq) load_turned(xt, a.k, now, hk);
    if constexpr (M == kDkv) load_turned(xt, a.dout, now, head_at(now));
    if (more) {
      load_rows(x0, M == kDkv ? a.q : a.k, next, head_at(next));
      if constexpr (M != kForward) load_rows(x1, M == kDkv ? a.dout : a.v, next, head_at(next));
      if (M == kDkv) load_stats(next);
    }
    // scores, base 2, of entries n8 (s[0], s[1]) and n8 + 8
    float th[4];
    bool on[2];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int32_t at = now.b + n8 + 8 * (j >> 1);
      on[j >> 1] = at < now.pe;
      float u = s[j];
      th[j] = 0.f;
      if (a.cap > 0.f) u = capped(u * a.scale, a.cap, inv_cap2, th[j]) * kLog2e;
      else u *= scale2;
      if (a.slopes) {
        const int32_t c = cols[on[j >> 1] ? at : now.b];
        const int64_t dist = M == kDkv ? c + a.row_offset - row : row + a.row_offset - c;
        const float sl = M == kDkv ? __ldg(a.slopes + head_at(now)) * kLog2e : slope2[j & 1];
        u = fmaf(-sl, fabsf((float)dist), u);
      }
      s[j] = u;
    }
    uint32_t parts[2][2];
    if constexpr (M == kForward) {
      float top[2] = {m[0], m[1]}, base[2];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (!on[j >> 1]) s[j] = -INFINITY;
        top[j & 1] = fmaxf(top[j & 1], s[j]);
      }
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], o));
        top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], o));
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        base[j] = top[j] == -INFINITY ? 0.f : top[j];
        const float keep = exp2_approx(m[j] - base[j]);
        m[j] = top[j];
        l[j] *= keep;
#pragma unroll
        for (int i = 0; i < NT; ++i) acc[i][j] *= keep, acc[i][2 + j] *= keep;
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float pa = exp2_approx(s[2 * j] - base[0]), pb = exp2_approx(s[2 * j + 1] - base[1]);
        l[0] += pa;
        l[1] += pb;
        uint32_t hi, lo;
        split2<T>(pa, pb, hi, lo);
        parts[0][j] = transpose8x8(hi);
        parts[1][j] = transpose8x8(lo);
      }
      turned_times<T, D, 2>(acc, xt, parts);
      if (more) load_turned(xt, a.v, next, hk);
    } else if constexpr (M == kDq) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float v[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int e = 2 * j + k;
          const float w = on[j] ? exp2_approx(s[e] - lse2[k]) : 0.f, wc = w * (1.f - th[e] * th[e]);
          if (on[j]) l[k] = fmaf(w, dp[e], l[k]);
          v[k] = t < 2 ? (on[j] ? wc * dp[e] * up : 0.f) : wc;
        }
        uint32_t hi, lo;
        split2<T>(v[0], v[1], hi, lo);
        parts[0][j] = transpose8x8(hi);
        parts[1][j] = transpose8x8(lo);
      }
      turned_times<T, D, 2>(acc, xt, parts);
    } else {
      // column 0: the value rounded, column 1: what rounding took (lanes of t = 0 hold both)
      uint32_t wp[1][2], wd[1][2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float lse = lse_n[j] * kLog2e;
        const float w = on[j] && lse_n[j] != -INFINITY ? exp2_approx(s[2 * j] - lse) : 0.f;
        const float g = on[j] ? w * (dp[2 * j] - delta_n[j]) * (1.f - th[2 * j] * th[2 * j]) * up : 0.f;
        const float wk = w * kUp, w_hi = unpack2<T>(pack2<T>(wk, 0.f)).x, g_hi = unpack2<T>(pack2<T>(g, 0.f)).x;
        wp[0][j] = transpose8x8(pack2<T>(wk, wk - w_hi));
        wd[0][j] = transpose8x8(pack2<T>(g, g - g_hi));
      }
      turned_times<T, D, 1>(acc, xt, wp);
      load_turned(xt, a.q, now, head_at(now));
      turned_times<T, D, 1>(acc2, xt, wd);
    }
    if (more && next.row == row) {
      now = next;
      continue;
    }
    // the row ends here
    const bool cut_head = row == r0 && head_cut, cut = cut_head || row == r1;
    const int64_t slot = cut_head ? 2 * chunk : 2 * chunk + 1;
    if constexpr (M != kDkv) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        l[0] += __shfl_xor_sync(0xffffffffu, l[0], o);
        l[1] += __shfl_xor_sync(0xffffffffu, l[1], o);
      }
    }
    const bool writes = D >= 64 || n8 < D / 8;
    if constexpr (M == kForward) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int h = h0 + 2 * t + j;
        if (2 * t + j >= live) continue;
        const float inv = l[j] == 0.f ? 0.f : 1.f / l[j];
#pragma unroll
        for (int i = 0; i < VT; ++i) {
          float f[8];
          elements(acc, i, j, f);
          const int col = (n8 + 8 * i) * 8;
          if (!writes) continue;
          if (cut) {
            st_f32<8>(a.slots + (slot * a.heads + h) * D + col, f);
          } else {
#pragma unroll
            for (int c = 0; c < 8; ++c) f[c] *= inv;
            RowVec<T, 8>::st((T *)a.out.p + (int64_t)row * a.out.row + (int64_t)h * a.out.head + col, f);
          }
        }
        if (n8 == 0) {
          if (cut) a.slot_ml[2 * (slot * a.heads + h)] = m[j], a.slot_ml[2 * (slot * a.heads + h) + 1] = l[j];
          else if (a.lse) a.lse[(int64_t)row * a.heads + h] = l[j] == 0.f ? -INFINITY : (m[j] + log2f(l[j])) * kLn2;
        }
      }
    } else if constexpr (M == kDq) {
      // x of heads 2 t, 2 t + 1 in lanes t < 2, their y in lanes t + 2
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int h = h0 + head_of(j);
        const bool own = head_of(j) < live && writes;
#pragma unroll
        for (int i = 0; i < VT; ++i) {
          float f[8], g[8];
          elements(acc, i, j, f);
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            if (t < 2) f[c] *= down;
            g[c] = __shfl_xor_sync(0xffffffffu, f[c], 2);
          }
          const int col = (n8 + 8 * i) * 8;
          if (!own) continue;
          if (cut) {
            st_f32<8>(a.slots + (slot * a.heads + h) * 2 * D + (t < 2 ? 0 : D) + col, f);
          } else if (t < 2) {
#pragma unroll
            for (int c = 0; c < 8; ++c) f[c] = (f[c] - l[j] * g[c]) * a.scale;
            RowVec<T, 8>::st((T *)a.dq.p + (int64_t)row * a.dq.row + (int64_t)h * a.dq.head + col, f);
          }
        }
        if (n8 == 0 && t < 2 && head_of(j) < live) {
          if (cut) a.slot_ml[slot * a.heads + h] = l[j];
          else a.delta[(int64_t)row * a.heads + h] = l[j];
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < VT; ++i) {
        float f[8], f1[8], g[8], g1[8];
        elements(acc2, i, 0, f);
        elements(acc2, i, 1, f1);
        elements(acc, i, 0, g);
        elements(acc, i, 1, g1);
#pragma unroll
        for (int c = 0; c < 8; ++c) f[c] = (f[c] + f1[c]) * (a.scale * down), g[c] = (g[c] + g1[c]) * (1.f / kUp);
        const int col = (n8 + 8 * i) * 8;
        if (t != 0 || !writes) continue;
        if (cut) {
          float *dst = a.slots + (slot * kv_heads + hk) * 2 * D + col;
          st_f32<8>(dst, f);
          st_f32<8>(dst + D, g);
        } else {
          RowVec<T, 8>::st((T *)a.dk.p + (int64_t)row * a.dk.row + (int64_t)hk * a.dk.head + col, f);
          RowVec<T, 8>::st((T *)a.dv.p + (int64_t)row * a.dv.row + (int64_t)hk * a.dv.head + col, g);
        }
      }
    }
    idle(row + 1, more ? next.row : r1);
    if (!more) break;
    now = next;
  }
}

__global__ void __launch_bounds__(256) dout_max_kernel(Heads x, int64_t rows, int heads, int dim, uint32_t *out) {
  const int per = dim / 8;
  const int64_t n = rows * heads * per;
  float top = 0.f;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t item = i / per, row = item / heads;
    float f[8];
    RowVec<__half, 8>::widen(RowVec<__half, 8>::ldg((const __half *)x.p + row * x.row + (item - row * heads) * x.head + (i - item * per) * 8), f);
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (isfinite(f[c])) top = fmaxf(top, fabsf(f[c]));
  }
  const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
  if ((threadIdx.x & 31) == 0 && bits > 0) atomicMax(out, bits);  // a maximum does not depend on the order
}

template <class T, int D>
void run(AttnPass pass, const DirView &d, const AttnArgs &a, cudaStream_t s) {
  const int kv_heads = a.heads / a.group, width = pass == kForward ? 8 : pass == kDq ? 4 : a.group;
  const int head_tiles = (a.group + width - 1) / width;
  const unsigned blocks = (unsigned)(((int64_t)d.n_chunks * kv_heads * head_tiles + kThreads / 32 - 1) / (kThreads / 32));
  if (pass == kForward) attn_graph_kernel<T, D, kForward><<<blocks, kThreads, 0, s>>>(d, a, head_tiles);
  else if (pass == kDq) attn_graph_kernel<T, D, kDq><<<blocks, kThreads, 0, s>>>(d, a, head_tiles);
  else attn_graph_kernel<T, D, kDkv><<<blocks, kThreads, 0, s>>>(d, a, head_tiles);
}

template <class T>
void pick(AttnPass pass, const DirView &d, const AttnArgs &a, cudaStream_t s) {
  if (a.dim == 32) run<T, 32>(pass, d, a, s);
  else if (a.dim == 64) run<T, 64>(pass, d, a, s);
  else run<T, 128>(pass, d, a, s);
}

}  // namespace

bool graph_on_tensor_cores(int dtype, int dim) { return dtype != DSP_F32 && (dim == 32 || dim == 64 || dim == 128); }

int graph_dout_max(const Heads &dout, int64_t rows, int heads, int dim, uint32_t *out, cudaStream_t s) {
  const cudaError_t e = cudaMemsetAsync(out, 0, 4, s);
  if (e != cudaSuccess) return fail(DSP_ERR_CUDA, "dsp_attn_grad: %s", cudaGetErrorString(e));
  const int64_t n = rows * heads * (dim / 8);
  if (n > 0) dout_max_kernel<<<(unsigned)std::min<int64_t>(148 * 8, (n + 255) / 256), 256, 0, s>>>(dout, rows, heads, dim, out);
  return DSP_OK;
}

void graph_pass(AttnPass pass, const DirView &d, const AttnArgs &a, int dtype, cudaStream_t s) {
  if (d.n_chunks == 0) return;
  if (dtype == DSP_BF16) pick<__nv_bfloat16>(pass, d, a, s);
  else pick<__half>(pass, d, a, s);
}

}  // namespace dsp
