// attn.h — arguments shared by the attention kernels.
#pragma once
#include "pattern.h"

namespace dsp {

// Strides are in elements; a head's dim values are contiguous.
struct Heads {
  const void *p;
  int64_t row, head;
};
struct HeadsOut {
  void *p;
  int64_t row, head;
};

struct AttnArgs {
  int heads, group, dim;  // group: query heads of one key/value head
  float scale, cap;       // cap = 0: none
  const float *slopes;    // [heads] or nullptr
  int64_t row_offset;
  int64_t n_queries;      // rows of q (tile form of dk, dv)
  Heads q, k, v, dout, o;
  HeadsOut out, dq, dk, dv;
  float *lse;        // [rows][heads]
  float *delta;      // [rows][heads] dout . out
  float2 *stats;     // [rows][heads] lse in base 2 (+infinity: a row without entries) and delta, for attn_graph.cu's dk, dv
  const uint32_t *dout_max;  // [heads][rows] bits of the largest finite |dout| (fp16 gradients by tiles)
  float *slots;      // partials of cut rows: [2 n_chunks][heads][width]
  float *slot_ml;    // [2 n_chunks][heads][2] running maximum and sum (forward), delta - delta0 and delta0 (dq)
};

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// cap tanh x, x = s / cap, inv_cap2 = 2 log2(e) / cap. From 1/2 on through one exponential: tanh x = 1 - 2 / (e^2x + 1), within 2^-22
// (tanh.approx is within 2^-11 of the value: a cap of 50 would shift scores by 0.02). Below, where that difference cancels (a cap
// of 10^8 would leave 0 of any score), x P(x^2), P of degree 4 through Chebyshev nodes, within 1.2e-7 of the value. th: tanh itself, for
// the gradient.
constexpr float kTanh0 = 0.999999987f, kTanh1 = -0.333330719f, kTanh2 = 0.13324829f, kTanh3 = -0.0529892412f, kTanh4 = 0.017141319f;
__device__ __forceinline__ float capped(float s, float cap, float inv_cap2, float &th) {
  const float two = s * inv_cap2, x = two * (0.5f * kLn2), y = x * x;
  const float p = fmaf(fmaf(fmaf(fmaf(kTanh4, y, kTanh3), y, kTanh2), y, kTanh1), y, kTanh0);
  th = 1.f - __fdividef(2.f, exp2_approx(two) + 1.f);  // 2 / inf = 0
  th = y < 0.25f ? x * p : th;
  return cap * th;
}

// fp16 has few exponents: gradients of scores are carried with a power of two that brings the largest |dout| near 16.
__device__ __forceinline__ float dout_scale(uint32_t dout_max) {
  const int e = (int)(dout_max >> 23);  // biased exponent; 255: not finite
  return e > 0 && e < 255 ? __uint_as_float((uint32_t)min(max(127 + 4 - (e - 127), 1), 254) << 23) : 1.f;
}

int check_attn(const char *who, const dsp_attn_desc *d, int64_t rows, int64_t keys);

}  // namespace dsp
