// rowvec.cuh — vectors of a dense row in fp32, bf16 or fp16, widened to fp32 in registers.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace dsp {

template <int BYTES>
struct RawOf;
template <>
struct RawOf<16> {
  using type = uint4;
};
template <>
struct RawOf<8> {
  using type = uint2;
};
template <>
struct RawOf<4> {
  using type = uint32_t;
};
template <>
struct RawOf<2> {
  using type = uint16_t;
};

// VE elements of T in one register vector.
template <class T, int VE>
struct RowVec {
  using Raw = typename RawOf<(int)sizeof(T) * VE>::type;
  union U {
    Raw raw;
    T e[VE];
    uint32_t w[(sizeof(T) * VE + 3) / 4];
    __device__ U() {}
  };
  static __device__ __forceinline__ Raw zero() {
    U u;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) * VE + 3) / 4; ++i) u.w[i] = 0;
    return u.raw;
  }
  static __device__ __forceinline__ Raw ldg(const T *p) { return __ldg(reinterpret_cast<const Raw *>(p)); }
  static __device__ __forceinline__ Raw ld(const T *p) { return *reinterpret_cast<const Raw *>(p); }
  static __device__ __forceinline__ void widen(Raw r, float (&f)[VE]) {
    U u;
    u.raw = r;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < VE; ++i) f[i] = (float)u.e[i];
    } else if constexpr (VE == 1) {
      f[0] = (float)u.e[0];
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
      for (int i = 0; i < VE / 2; ++i) {  // bf16 is the upper half of an fp32
        f[2 * i] = __uint_as_float(u.w[i] << 16);
        f[2 * i + 1] = __uint_as_float(u.w[i] & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int i = 0; i < VE / 2; ++i) {
        const float2 x = __half22float2(*reinterpret_cast<const __half2 *>(&u.w[i]));
        f[2 * i] = x.x;
        f[2 * i + 1] = x.y;
      }
    }
  }
  static __device__ __forceinline__ Raw narrow(const float (&f)[VE]) {  // round to nearest
    U u;
#pragma unroll
    for (int i = 0; i < VE; ++i) u.e[i] = T(f[i]);
    return u.raw;
  }
  static __device__ __forceinline__ void st(T *p, const float (&f)[VE]) { *reinterpret_cast<Raw *>(p) = narrow(f); }
  static __device__ __forceinline__ void st_stream(T *p, const float (&f)[VE]) {
    __stcs(reinterpret_cast<Raw *>(p), narrow(f));
  }
};

// Two fused multiply-adds in one instruction, each rounded as fmaf.
__device__ __forceinline__ void fma2(float &c0, float &c1, float a0, float a1, float b0, float b1) {
  asm("{\n .reg .b64 a, b, c;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mov.b64 c, {%0, %1};\n fma.rn.f32x2 c, a, b, c;\n "
      "mov.b64 {%0, %1}, c;\n}"
      : "+f"(c0), "+f"(c1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}
// d = a b + c of pairs (a c that is used again, such as a constant, needs no copy).
__device__ __forceinline__ void fma2(float &d0, float &d1, float a0, float a1, float b0, float b1, float c0, float c1) {
  asm("{\n .reg .b64 a, b, c, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mov.b64 c, {%6, %7};\n fma.rn.f32x2 d, a, b, c;\n "
      "mov.b64 {%0, %1}, d;\n}"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}
// c = a + b, c = a b of pairs.
__device__ __forceinline__ void add2(float &c0, float &c1, float a0, float a1, float b0, float b1) {
  asm("{\n .reg .b64 a, b, c;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n add.rn.f32x2 c, a, b;\n mov.b64 {%0, %1}, c;\n}"
      : "=f"(c0), "=f"(c1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}
__device__ __forceinline__ void mul2(float &c0, float &c1, float a0, float a1, float b0, float b1) {
  asm("{\n .reg .b64 a, b, c;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mul.rn.f32x2 c, a, b;\n mov.b64 {%0, %1}, c;\n}"
      : "=f"(c0), "=f"(c1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// acc += x * row
template <class T, int VE>
__device__ __forceinline__ void fma_row(float (&acc)[VE], float x, typename RowVec<T, VE>::Raw r) {
  float f[VE];
  RowVec<T, VE>::widen(r, f);
  if constexpr (VE % 2 == 0) {
#pragma unroll
    for (int i = 0; i < VE; i += 2) fma2(acc[i], acc[i + 1], f[i], f[i + 1], x, x);
  } else {
#pragma unroll
    for (int i = 0; i < VE; ++i) acc[i] = fmaf(x, f[i], acc[i]);
  }
}
// s += x . row, in two interleaved sums where VE is even
template <class T, int VE>
__device__ __forceinline__ void dot_row(float (&s)[2], const float (&x)[VE], typename RowVec<T, VE>::Raw r) {
  float f[VE];
  RowVec<T, VE>::widen(r, f);
  if constexpr (VE % 2 == 0) {
#pragma unroll
    for (int i = 0; i < VE; i += 2) fma2(s[0], s[1], f[i], f[i + 1], x[i], x[i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < VE; ++i) s[0] = fmaf(x[i], f[i], s[0]);
  }
}

// fp32 rows beside rows of T (pre-activations, partial sums): VE floats as float4s, or one by one.
template <int VE>
__device__ __forceinline__ void ld_f32(const float *p, float (&f)[VE]) {
  if constexpr (VE % 4 == 0) {
#pragma unroll
    for (int i = 0; i < VE / 4; ++i) {
      const float4 x = __ldg(reinterpret_cast<const float4 *>(p) + i);
      f[4 * i] = x.x, f[4 * i + 1] = x.y, f[4 * i + 2] = x.z, f[4 * i + 3] = x.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < VE; ++i) f[i] = __ldg(p + i);
  }
}
template <int VE>
__device__ __forceinline__ void st_f32(float *p, const float (&f)[VE]) {
  if constexpr (VE % 4 == 0) {
#pragma unroll
    for (int i = 0; i < VE / 4; ++i)
      __stcs(reinterpret_cast<float4 *>(p) + i, make_float4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]));
  } else {
#pragma unroll
    for (int i = 0; i < VE; ++i) p[i] = f[i];
  }
}

}  // namespace dsp
