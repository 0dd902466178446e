// frag.cuh — gathered rows as operands of mma.sync m16n8k16 (bf16, fp16), straight from global memory.
//
// The order of a sum is free, so the places of a row's elements in the fragments are chosen such that every lane's part of a
// row is whole 16-byte vectors and neighbouring lanes read neighbouring vectors: no shared memory, no shuffles. With t = lane %
// 4 and n8 = lane / 4:
//   Rows  (A = 16 rows x dim, a product over dim): rows n8 and n8 + 8, of each the vectors t + 4 i
//   Turned (A = dim x 16 rows, a product over rows): rows 2 t, 2 t + 1, 2 t + 8, 2 t + 9, of each the vectors n8 + 8 i; pairs of
//          rows are interleaved by a byte permute. Row n8 (n8 + 8) of the 16 x 8 result tile 4 i + c is element 2 c (2 c + 1) of
//          vector n8 + 8 i.
//   column (B = dim x 8): the vectors t + 4 i of the row that is column n8
#pragma once
#include "rowvec.cuh"

namespace dsp {

template <class T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// An 8 x 8 block of 16-bit elements, row n8 with columns 2 t, 2 t + 1 in a lane, transposed.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <class T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const __nv_bfloat162 x = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&x);
  } else {
    const __half2 x = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&x);
  }
}
template <class T>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  else return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
// Two values as rounded parts and what rounding took.
template <class T>
__device__ __forceinline__ void split2(float x, float y, uint32_t &hi, uint32_t &lo) {
  hi = pack2<T>(x, y);
  const float2 f = unpack2<T>(hi);
  lo = pack2<T>(x - f.x, y - f.y);
}

__device__ __forceinline__ uint32_t word(const uint4 &x, int i) { return i == 0 ? x.x : i == 1 ? x.y : i == 2 ? x.z : x.w; }

// s (+)= rows . columns: 16 x 8
template <class T, int D>
__device__ __forceinline__ void rows_times(float (&s)[4], const uint4 (&k)[2][D / 32], const uint32_t (&q)[D / 16][2]) {
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t w[4] = {word(k[0][i], 2 * j), word(k[1][i], 2 * j), word(k[0][i], 2 * j + 1), word(k[1][i], 2 * j + 1)};
      mma16816<T>(s, w, q[2 * i + j][0], q[2 * i + j][1]);
    }
}
// Fragments of the columns from one row per lane group; zeros where !on.
template <class T, int D>
__device__ __forceinline__ void load_column(uint32_t (&q)[D / 16][2], const T *row, bool on) {
  const int t = threadIdx.x & 3;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    const uint4 w = on ? __ldg(reinterpret_cast<const uint4 *>(row + t * 8 + 32 * i)) : make_uint4(0, 0, 0, 0);
    q[2 * i][0] = w.x, q[2 * i][1] = w.y, q[2 * i + 1][0] = w.z, q[2 * i + 1][1] = w.w;
  }
}
// The other way round: 16 gathered rows as the 8 columns of two products, so that a row's vectors are operands as they are
// loaded. Of A, rows 0 to 7 are `low`, rows 8 to 15 `high` (one row per lane group n8 each).
template <class T, int D>
__device__ __forceinline__ void load_pair(uint32_t (&q)[D / 16][4], const T *low, bool low_on, const T *high, bool high_on) {
  const int t = threadIdx.x & 3;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    const uint4 zero = make_uint4(0, 0, 0, 0);
    const uint4 w = low_on ? __ldg(reinterpret_cast<const uint4 *>(low + t * 8 + 32 * i)) : zero;
    const uint4 v = high_on ? __ldg(reinterpret_cast<const uint4 *>(high + t * 8 + 32 * i)) : zero;
    q[2 * i][0] = w.x, q[2 * i][2] = w.y, q[2 * i + 1][0] = w.z, q[2 * i + 1][2] = w.w;
    q[2 * i][1] = v.x, q[2 * i][3] = v.y, q[2 * i + 1][1] = v.z, q[2 * i + 1][3] = v.w;
  }
}
// s[0], s[1]: row n8 of low (HIGH: high) . gathered rows 2 t, 2 t + 1; s[2], s[3]: . rows 2 t + 8, 2 t + 9.
template <class T, int D, bool HIGH>
__device__ __forceinline__ void pair_times(float (&s)[4], const uint32_t (&q)[D / 16][4], const uint4 (&k)[2][D / 32]) {
  float c[2][4];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c[j][i] = 0.f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      mma16816<T>(c[j], q[2 * i], k[j][i].x, k[j][i].y);
      mma16816<T>(c[j], q[2 * i + 1], k[j][i].z, k[j][i].w);
    }
    s[2 * j] = c[j][HIGH ? 2 : 0], s[2 * j + 1] = c[j][HIGH ? 3 : 1];
  }
}

// vectors of a turned row per lane, result tiles
template <int D>
constexpr int kTurned = D >= 64 ? D / 64 : 1;
template <int D>
constexpr int kTiles = 4 * kTurned<D>;

// acc += turned rows . weights (hi and lo parts), 16-bit pairs of rows in b
template <class T, int D, int PARTS>
__device__ __forceinline__ void turned_times(float (&acc)[kTiles<D>][4], const uint4 (&v)[4][kTurned<D>], const uint32_t (&b)[PARTS][2]) {
#pragma unroll
  for (int i = 0; i < kTurned<D>; ++i)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint32_t k0 = word(v[0][i], c), k1 = word(v[1][i], c), k2 = word(v[2][i], c), k3 = word(v[3][i], c);
      const uint32_t w[4] = {__byte_perm(k0, k1, 0x5410), __byte_perm(k0, k1, 0x7632), __byte_perm(k2, k3, 0x5410),
                             __byte_perm(k2, k3, 0x7632)};
#pragma unroll
      for (int p = 0; p < PARTS; ++p) mma16816<T>(acc[4 * i + c], w, b[p][0], b[p][1]);
    }
}

}  // namespace dsp
