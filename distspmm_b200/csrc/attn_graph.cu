// attn_graph.cu — attention over a pattern's entries, row by row, 16-bit operands of dim 32, 64 or 128: forward, dq, and dk, dv.
//
// For patterns too thin for tiles (a graph's edges). The formulas are those of attn.cu; what bounds both is the gather of a row
// of k and one of v (q and dout, by columns) for each entry and head out of L2. Here the arithmetic is given to mma.sync, though
// an entry has but one query for each head to be multiplied with (of m16n8k16 products, 8 columns are entries and 1 to 8 rows
// query heads): R-MAT 15, 8 heads of 64, bf16: forward 577 -> 377 us, dq 632 -> 468,
// dk and dv 681 -> 597 against dot products by shuffles.
//
//   pass      16 entries as columns   rows                         then, entries turned
//   forward   k                       q of up to 8 heads           v   x weights
//   dq        k, v                    q, dout of up to 4 heads,    k   x [p c (dp - delta0) | p c]   (x and y of attn_row.cuh)
//                                     twice
//   dk, dv    q, dout of one head     k, v (one key, twice)        dout x p, q x p c (dp - delta): hi and lo parts in the columns
//
// A warp owns a chunk (pattern.h) and a head or group; its column ids and row pointers are staged in shared memory, and the walk
// over 16-entry steps runs on across rows: the next step's rows are requested as soon as the present ones are in the products,
// so a short row costs no wait. Weights enter the second product as hi + lo (2^-16 of a weight is lost at most). So dq takes its
// differences dp - delta from delta0 = dout . out, within out's rounding of delta, before they are split, and the rest off after the
// products: dq = scale (x - g y) with g = delta - delta0 = sum p (dp - delta0). An infinity that is listed would meet lo parts of 0 or of
// the other sign: rows whose result is not finite are done again by attn_row.cuh's gather (dq: any such row is NaN by the formula).
#include <algorithm>
#include <type_traits>

#include "attn_graph.h"
#include "attn_row.cuh"
#include "frag.cuh"

namespace dsp {
namespace {

constexpr int kThreads = 128;
constexpr float kSlack = 8.f;

// A step: 16 entries from b on, of a row whose entries in this chunk end at pe, for query head number h of the group (dk, dv).
struct Step {
  int32_t row, b, pe, h;
};

// fp16 has few exponents: a column of the second product's weights is carried with a power of two, the same from one step to the next
// while the largest weight stays between 2^0 (in a row's first step that has any) and 2^15, else that which brings it to 2^10 (what the sums
// hold is then scaled by the same). So nothing overflows, and hi + lo are within 2^-25 where the largest is 1 or more.
__device__ __forceinline__ bool out_of_place(float top, float carry, bool fresh) {
  const float x = top * carry;
  return x > 32768.f || (fresh && x < 1.f && top > 0.f);
}
// The new carry, and what the sums are to be multiplied with.
__device__ __forceinline__ float renew(float top, float &carry, bool fresh) {
  const int e = (int)(__float_as_uint(top) >> 23);  // 255: not finite, and nothing will help
  if (!out_of_place(top, carry, fresh) || e == 255) return 1.f;
  const float now = __uint_as_float((uint32_t)min(max(127 + 10 - (e - 127), 1), 254) << 23), keep = fresh ? 1.f : now / carry;
  carry = now;
  return keep;
}
__device__ __forceinline__ float largest(const float (&x)[4]) {
  return fmaxf(max3(fabsf(x[0]), fabsf(x[1]), fabsf(x[2])), fabsf(x[3]));
}

template <class T, int D, AttnPass M>
__global__ void __launch_bounds__(kThreads, D == 128 ? (M == kDkv ? 2 : 3) : (M == kDkv ? 3 : 4))
    attn_graph_kernel(const __grid_constant__ DirView d, const __grid_constant__ AttnArgs a, int head_tiles) {
  constexpr int VR = D / 32, VT = kTurned<D>, NT = kTiles<D>;
  constexpr int kWidth = M == kForward ? 8 : M == kDq ? 4 : 1;  // query heads of a warp's columns
  __shared__ ChunkLists all_lists[kThreads / 32];
  __shared__ uint8_t all_bad[kThreads / 32][kMaxUnits / kRowUnits + 4];  // heads of the chunk's rows to be done again
  const int lane = threadIdx.x & 31, t = lane & 3, n8 = lane >> 2;
  const int kv_heads = a.heads / a.group, per_chunk = kv_heads * head_tiles;
  const int64_t item = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> 5;
  const int64_t chunk = item / per_chunk;
  if (chunk >= d.n_chunks) return;
  const int hk = (int)(item - chunk * per_chunk) / head_tiles, h0 = hk * a.group + (int)(item % head_tiles) * kWidth;
  const int live = M == kDkv ? 1 : min(kWidth, (hk + 1) * a.group - h0);  // query heads h0 .. h0 + live - 1
  ChunkLists &list = all_lists[threadIdx.x >> 5];
  const int32_t r0 = __ldg(d.row0 + chunk), r1 = __ldg(d.row0 + chunk + 1), p0 = __ldg(d.nz0 + chunk), p1 = __ldg(d.nz0 + chunk + 1);
  uint8_t *bad_rows = all_bad[threadIdx.x >> 5];
  for (int i = lane; i <= r1 - r0 + 1; i += 32) {
    if (r0 + i <= d.n) list.ptr[i] = __ldg(d.ptr + r0 + i);
    bad_rows[i] = 0;
  }
#pragma unroll 4
  for (int i = lane; i < p1 - p0; i += 32) list.cols[i] = __ldg(d.cols + p0 + i);
  __syncwarp();
  const int32_t *cols = list.cols - p0;
  const bool head_cut = p0 > list.ptr[0];
  constexpr bool kHalf = std::is_same<T, __half>::value;
  // fp16: what the columns of the second products carry (dq: this lane's column; dk, dv: the weights, the score gradients)
  float carry = 1.f, carry2 = 1.f;
  const float inv_cap2 = a.cap > 0.f ? 2.f * kLog2e / a.cap : 0.f, scale2 = a.scale * kLog2e;

  // a lane has the scores of column n8, a query head (dk, dv: the key, in columns 0 and 1), for the entries 2 t, 2 t + 1, 2 t + 8,
  // 2 t + 9 of a step: as they enter the second product
  bool fresh = false, fresh2 = false;  // the row's sums are still 0
  const int head = M == kForward ? n8 : M == kDq ? n8 & 3 : 0;
  const float slope2 = M != kDkv && a.slopes && head < live ? __ldg(a.slopes + h0 + head) * kLog2e : 0.f;
  auto entry = [&](int j) { return 2 * t + (j & 1) + 8 * (j >> 1); };

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
          if (lane == 0 && M == kDq) a.slot_ml[2 * slot] = a.slot_ml[2 * slot + 1] = 0.f;
        } else {
          const HeadsOut &o = M == kForward ? a.out : a.dq;
          if (lane < D / 8) *reinterpret_cast<uint4 *>((T *)o.p + (int64_t)row * o.row + (int64_t)h * o.head + 8 * lane) = zero;
          if (lane == 0 && M == kForward && a.lse) a.lse[(int64_t)row * a.heads + h] = -INFINITY;
          if (lane == 0 && M == kDq) a.stats[(int64_t)row * a.heads + h] = make_float2(INFINITY, 0.f);
        }
      }
    }
  };

  // gathers: rows n8, n8 + 8 of a step; turned rows. Entries behind the row's end are read as its last one; their weights are 0.
  auto at_row = [](const Heads &m, int head, int vec) { return (const char *)((const T *)m.p + (int64_t)head * m.head + vec * 8); };
  auto load_rows = [&](uint4(&x)[2][VR], const Heads &m, const Step &s, int head) {
    const char *base = at_row(m, head, t);
    const uint32_t stride = (uint32_t)m.row * (uint32_t)sizeof(T);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const char *src = base + (uint64_t)(uint32_t)cols[min(s.b + n8 + 8 * j, s.pe - 1)] * stride;
#pragma unroll
      for (int i = 0; i < VR; ++i) x[j][i] = __ldg(reinterpret_cast<const uint4 *>(src + 64 * i));
    }
  };
  auto load_turned = [&](uint4(&x)[4][VT], const Heads &m, const Step &s, int head) {
    const char *base = at_row(m, head, D >= 64 ? n8 : min(n8, D / 8 - 1));
    const uint32_t stride = (uint32_t)m.row * (uint32_t)sizeof(T);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const char *src = base + (uint64_t)(uint32_t)cols[min(s.b + entry(j), s.pe - 1)] * stride;
#pragma unroll
      for (int i = 0; i < VT; ++i) x[j][i] = __ldg(reinterpret_cast<const uint4 *>(src + 128 * i));
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
  float2 stat_e[4] = {};  // dk, dv: of this lane's queries (columns 0 and 1 need them)
  auto load_stats = [&](const Step &s) {
    if (n8 >= 2) return;
#pragma unroll
    for (int j = 0; j < 4; ++j) stat_e[j] = a.stats[(int64_t)cols[min(s.b + entry(j), s.pe - 1)] * a.heads + head_at(s)];
  };
  if (M == kDkv) load_stats(now);

  int32_t row = -1;
  uint32_t pair[D / 16][4];  // q over dout (dk, dv: k over v)
  float acc[NT][4], acc2[M == kDkv ? NT : 1][4];
  float m = -INFINITY, l = 0.f, lse2 = 0.f, delta0 = 0.f;  // forward: maximum, sum; dq: l is delta - delta0

#pragma unroll 1
  while (true) {
    if (now.row != row) {
      row = now.row;
      if (M == kDkv) {
        load_pair<T, D>(pair, (const T *)a.k.p + (int64_t)row * a.k.row + (int64_t)hk * a.k.head, n8 < 2,
                        (const T *)a.v.p + (int64_t)row * a.v.row + (int64_t)hk * a.v.head, n8 < 2);
      } else {
        load_pair<T, D>(pair, (const T *)a.q.p + (int64_t)row * a.q.row + (int64_t)(h0 + head) * a.q.head, head < live,
                        (const T *)a.dout.p + (int64_t)row * a.dout.row + (int64_t)(h0 + head) * a.dout.head, M == kDq && head < live);
        if constexpr (M == kDq) {
          lse2 = head < live ? __ldg(a.lse + (int64_t)row * a.heads + h0 + head) * kLog2e : 0.f;
          if (lse2 == -INFINITY) lse2 = INFINITY;
          delta0 = 0.f;
          if (head < live) {
            const T *o = (const T *)a.o.p + (int64_t)row * a.o.row + (int64_t)(h0 + head) * a.o.head + t * 8;
#pragma unroll
            for (int i = 0; i < VR; ++i) {
              const uint4 w = __ldg(reinterpret_cast<const uint4 *>(o + 32 * i));
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                const float2 x = unpack2<T>(word(w, c)), y = unpack2<T>(pair[2 * i + c / 2][1 + 2 * (c & 1)]);
                delta0 = fmaf(x.x, y.x, fmaf(x.y, y.y, delta0));
              }
            }
          }
          delta0 += __shfl_xor_sync(0xffffffffu, delta0, 1);
          delta0 += __shfl_xor_sync(0xffffffffu, delta0, 2);
        }
      }
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          acc[i][j] = 0.f;
          if constexpr (M == kDkv) acc2[i][j] = 0.f;
        }
      m = -INFINITY, l = 0.f;
      fresh = fresh2 = true;
    }
    const Step next = next_of(now);
    const bool more = next.row <= r1;
    float s[4], dp[4];
    pair_times<T, D, false>(s, pair, x0);
    if constexpr (M != kForward) pair_times<T, D, true>(dp, pair, x1);
    float2 stat[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) stat[j] = stat_e[j];
    // the next step's rows; of this one the turned rows, which the first product has brought to L1
    if constexpr (M == kDq) load_turned(xt, a.k, now, hk);
    if constexpr (M == kDkv) load_turned(xt, a.dout, now, head_at(now));
    if (more) {
      load_rows(x0, M == kDkv ? a.q : a.k, next, head_at(next));
      if constexpr (M != kForward) load_rows(x1, M == kDkv ? a.dout : a.v, next, head_at(next));
      if (M == kDkv) load_stats(next);
    }
    // scores, base 2
    float th[4];
    bool on[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int32_t at = now.b + entry(j);
      on[j] = at < now.pe;
      float u = s[j];
      th[j] = 0.f;
      if (a.cap > 0.f) u = capped(u * a.scale, a.cap, inv_cap2, th[j]) * kLog2e;
      else u *= scale2;
      if (a.slopes) {
        const int32_t c = cols[min(at, now.pe - 1)];
        const int64_t dist = M == kDkv ? c + a.row_offset - row : row + a.row_offset - c;
        const float sl = M == kDkv ? __ldg(a.slopes + head_at(now)) * kLog2e : slope2;
        u = fmaf(-sl, fabsf((float)dist), u);
      }
      s[j] = u;
    }
    uint32_t parts[2][2];
    if constexpr (M == kForward) {
      // m: a maximum of the row that the column's lanes agree on; renewed when a score is above it by more than 2^kSlack
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (!on[j]) s[j] = -INFINITY;
        top = fmaxf(top, s[j]);
      }
      if (__any_sync(0xffffffffu, top > m + kSlack)) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float m2 = fmaxf(m, top), keep = m2 == -INFINITY ? 0.f : exp2_approx(m - m2);
        m = m2;
        l *= keep;
        // the sums' columns are heads 2 t and 2 t + 1
        const float k0 = __shfl_sync(0xffffffffu, keep, 8 * t), k1 = __shfl_sync(0xffffffffu, keep, 8 * t + 4);
#pragma unroll
        for (int i = 0; i < NT; ++i) acc[i][0] *= k0, acc[i][2] *= k0, acc[i][1] *= k1, acc[i][3] *= k1;
      }
      const float base = m == -INFINITY ? 0.f : m;
      float w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[j] = exp2_approx(s[j] - base);
        l += w[j];
      }
      split2<T>(w[0], w[1], parts[0][0], parts[1][0]);
      split2<T>(w[2], w[3], parts[0][1], parts[1][1]);
      turned_times<T, D, 2>(acc, xt, parts);
      if (more) load_turned(xt, a.v, next, hk);
    } else if constexpr (M == kDq) {
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float w = on[j] ? exp2_approx(s[j] - lse2) : 0.f, wc = w * (1.f - th[j] * th[j]), gap = dp[j] - delta0;
        l = fmaf(w, gap, l);
        v[j] = n8 < 4 ? wc * gap : wc;
      }
      if constexpr (kHalf) {
        float top = largest(v);
        const uint32_t filled = __ballot_sync(0xffffffffu, top > 0.f) >> (lane & 28) & 15;  // of this lane's column
        if (__any_sync(0xffffffffu, out_of_place(top, carry, fresh))) {
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const float keep = renew(top, carry, fresh);
          const float k0 = __shfl_sync(0xffffffffu, keep, 8 * t), k1 = __shfl_sync(0xffffffffu, keep, 8 * t + 4);
#pragma unroll
          for (int i = 0; i < NT; ++i) acc[i][0] *= k0, acc[i][2] *= k0, acc[i][1] *= k1, acc[i][3] *= k1;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] *= carry;
        fresh = fresh && filled == 0;
      }
      split2<T>(v[0], v[1], parts[0][0], parts[1][0]);
      split2<T>(v[2], v[3], parts[0][1], parts[1][1]);
      turned_times<T, D, 2>(acc, xt, parts);
    } else {
      // column 0: the value rounded, column 1: what rounding took
      uint32_t wp[1][2], wd[1][2];
      float w[4], g[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[j] = on[j] ? exp2_approx(s[j] - stat[j].x) : 0.f;
        g[j] = w[j] * (dp[j] - stat[j].y) * (1.f - th[j] * th[j]);
      }
      if constexpr (kHalf) {
        float top = n8 == 0 ? largest(w) : 0.f, top2 = n8 == 0 ? largest(g) : 0.f;
        const bool filled = __any_sync(0xffffffffu, top > 0.f), filled2 = __any_sync(0xffffffffu, top2 > 0.f);
        if (__any_sync(0xffffffffu, out_of_place(top, carry, fresh) || out_of_place(top2, carry2, fresh2))) {
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            top2 = fmaxf(top2, __shfl_xor_sync(0xffffffffu, top2, o));
          }
          const float keep = renew(top, carry, fresh), keep2 = renew(top2, carry2, fresh2);
#pragma unroll
          for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] *= keep, acc2[i][j] *= keep2;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] *= carry, g[j] *= carry2;
        fresh = fresh && !filled, fresh2 = fresh2 && !filled2;
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t hi, lo;
        split2<T>(w[2 * j], w[2 * j + 1], hi, lo);
        wp[0][j] = n8 == 0 ? hi : lo;
        split2<T>(g[2 * j], g[2 * j + 1], hi, lo);
        wd[0][j] = n8 == 0 ? hi : lo;
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
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
    }
    // of the heads 2 t, 2 t + 1 (dq: 2 t & 3, ...) whose sums this lane holds
    const float l2[2] = {__shfl_sync(0xffffffffu, l, 8 * t), __shfl_sync(0xffffffffu, l, 8 * t + 4)};
    const bool writes = D >= 64 || n8 < D / 8;
    if constexpr (M == kForward) {
      uint32_t bad = 0;  // heads with a result that is not finite, though the weights are
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int h = h0 + 2 * t + j;
        if (2 * t + j >= live) continue;
        const float inv = l2[j] == 0.f ? 0.f : 1.f / l2[j];
        float zero = 0.f;
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
            for (int c = 0; c < 8; ++c) f[c] *= inv, zero = fmaf(f[c], 0.f, zero);
            RowVec<T, 8>::st((T *)a.out.p + (int64_t)row * a.out.row + (int64_t)h * a.out.head + col, f);
          }
        }
        if (zero != 0.f && l2[j] == l2[j]) bad |= 1u << (2 * t + j);
      }
      if (t == 0 && n8 < live) {
        const int64_t at = slot * a.heads + h0 + n8;
        if (cut) a.slot_ml[2 * at] = m, a.slot_ml[2 * at + 1] = l;
        else if (a.lse) a.lse[(int64_t)row * a.heads + h0 + n8] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
      }
      if (__any_sync(0xffffffffu, bad != 0)) bad_rows[row - r0] = (uint8_t)__reduce_or_sync(0xffffffffu, bad);
    } else if constexpr (M == kDq) {
      // x of heads 2 t, 2 t + 1 in lanes t < 2, their y in lanes t + 2
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int hh = (2 * t + j) & 3, h = h0 + hh;
        const bool own = hh < live && writes;
        const float down = kHalf ? 1.f / __shfl_sync(0xffffffffu, carry, 8 * t + 4 * j) : 1.f;
#pragma unroll
        for (int i = 0; i < VT; ++i) {
          float f[8], g[8];
          elements(acc, i, j, f);
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            if (kHalf) f[c] *= down;
            g[c] = __shfl_xor_sync(0xffffffffu, f[c], 2);
          }
          const int col = (n8 + 8 * i) * 8;
          if (!own) continue;
          if (cut) {
            st_f32<8>(a.slots + (slot * a.heads + h) * 2 * D + (t < 2 ? 0 : D) + col, f);
          } else if (t < 2) {
#pragma unroll
            for (int c = 0; c < 8; ++c) f[c] = (f[c] - l2[j] * g[c]) * a.scale;
            RowVec<T, 8>::st((T *)a.dq.p + (int64_t)row * a.dq.row + (int64_t)h * a.dq.head + col, f);
          }
        }
      }
      if (t == 0 && n8 < live) {
        const int64_t at = 2 * (slot * a.heads + h0 + n8);
        if (cut) a.slot_ml[at] = l, a.slot_ml[at + 1] = delta0;
        else a.stats[(int64_t)row * a.heads + h0 + n8] = make_float2(lse2, delta0 + l);
      }
    } else {
      float zero = 0.f;
#pragma unroll
      for (int i = 0; i < VT; ++i) {
        float f[8], f1[8], g[8], g1[8];
        elements(acc2, i, 0, f);
        elements(acc2, i, 1, f1);
        elements(acc, i, 0, g);
        elements(acc, i, 1, g1);
#pragma unroll
        for (int c = 0; c < 8; ++c) f[c] = (f[c] + f1[c]) * (a.scale / carry2), g[c] = (g[c] + g1[c]) * (1.f / carry);
        const int col = (n8 + 8 * i) * 8;
        if (t != 0 || !writes) continue;
        if (cut) {
          float *dst = a.slots + (slot * kv_heads + hk) * 2 * D + col;
          st_f32<8>(dst, f);
          st_f32<8>(dst + D, g);
        } else {
          RowVec<T, 8>::st((T *)a.dk.p + (int64_t)row * a.dk.row + (int64_t)hk * a.dk.head + col, f);
          RowVec<T, 8>::st((T *)a.dv.p + (int64_t)row * a.dv.row + (int64_t)hk * a.dv.head + col, g);
#pragma unroll
          for (int c = 0; c < 8; ++c) zero = fmaf(f[c], 0.f, fmaf(g[c], 0.f, zero));
        }
      }
      if (__any_sync(0xffffffffu, zero != 0.f)) bad_rows[row - r0] = 1;
    }
    idle(row + 1, more ? next.row : r1);
    if (!more) break;
    now = next;
  }
  if constexpr (M != kDq) {
    __syncwarp();
#pragma unroll 1
    for (int i = 0; i < r1 - r0; ++i) {  // after the loop: a call within it would cost its registers
      if constexpr (M == kDkv) {
        if (bad_rows[i]) attend_dkv_again<T, D>(PlanRows{d}, a, r0 + i, hk);
      } else {
#pragma unroll 1
        for (uint32_t bad = bad_rows[i]; bad; bad &= bad - 1) attend_again<T, D>(PlanRows{d}, a, r0 + i, h0 + __ffs(bad) - 1);
      }
    }
  }
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

void graph_pass(AttnPass pass, const DirView &d, const AttnArgs &a, int dtype, cudaStream_t s) {
  if (d.n_chunks == 0) return;
  if (dtype == DSP_BF16) pick<__nv_bfloat16>(pass, d, a, s);
  else pick<__half>(pass, d, a, s);
}

}  // namespace dsp
