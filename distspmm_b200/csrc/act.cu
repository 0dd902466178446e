// act.cu — out = act(A.B + bias) + residual and its gradients.
//
//   z_i = sum over the entries p of row i of a_p B[c_p] + bias,   out_i = act(z_i) + residual_i
//   dz_i = dout_i act'(z_i),   dB = A^T dz,   da_p = dz_{r_p} . B[c_p],   dbias = sum_i dz_i
//
// The work is a gather of one row of B (or dz) per entry; the arithmetic is two operations per element read, so the kernels
// are bound by how fast rows come out of L2 (or HBM, once B is larger than the 126 MB L2). What the design does about it:
// 16-bit rows stay 16-bit until they are in registers, the epilogue adds no pass over the result, and work is cut into
// chunks of equal entries + row ends, so that hub rows and runs of empty rows are spread evenly. A warp owns a chunk; a row
// is read in 16-byte vectors by as many lanes as it has, several rows side by side where it has fewer than 32. Measured, R-MAT
// 18 (7.6 M entries), N = 128, bf16: 199 us without an epilogue (9.8 TB/s gathered), 234 with bias, gelu and residual.
#include <algorithm>
#include <type_traits>

#include "pattern.h"
#include "rowvec.cuh"

namespace dsp {
namespace {

constexpr int kThreads = 256;

struct ActArgs {
  int act, N;
  const float *values;
  const void *B;
  uint32_t ldb_bytes;
  const float *bias;
  const void *residual;
  int64_t ldr;
  void *out;
  int64_t ldo;
  float *pre;
  int64_t ldp;
  float *slots;  // [2 n_chunks][N] partial rows
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Phi(z) (the normal distribution) and exp(-z^2 / 2) of two values. With x = |z| / sqrt 2 and t = 1 / (1 + 0.45 x):
// erfc(x) = t exp(-x^2) Q(t), Q the polynomial of degree 9 through erfcx(x) / t at Chebyshev nodes of (0, 1]; it is within 4e-8
// of it. In fp32 the whole is within 2^-20 + z^2 2^-24 relative to erfc itself: z^2 is rounded before the exponential (4e-7 at |z| < 1,
// 7e-7 at 3, 8e-6 at 12). (erfcf costs five times the instructions: 50 of 272 us of an R-MAT 18 product with gelu.)
__device__ __forceinline__ void normal2(float z0, float z1, float &c0, float &c1, float &e0, float &e1) {
  constexpr float Q[10] = {0.253885329f, 0.253883481f, 0.228263408f, 0.175332934f, 0.119559288f, -0.021311678f, 0.140786096f, -0.299159557f, 0.190028757f, -0.041268073f};
  const float t0 = __fdividef(1.f, fmaf(fabsf(z0), 0.45f * 0.70710678f, 1.f)), t1 = __fdividef(1.f, fmaf(fabsf(z1), 0.45f * 0.70710678f, 1.f));
  e0 = exp2_fast(z0 * z0 * -0.72134752f), e1 = exp2_fast(z1 * z1 * -0.72134752f);
  float q0 = Q[9], q1 = Q[9];
#pragma unroll
  for (int i = 8; i >= 0; --i) {
    fma2(q0, q1, q0, q1, t0, t1, Q[i], Q[i]);
  }
  c0 = 0.5f * t0 * q0 * e0, c1 = 0.5f * t1 * q1 * e1;
  c0 = z0 > 0.f ? 1.f - c0 : c0, c1 = z1 > 0.f ? 1.f - c1 : c1;
}

// act of each element.
template <int N>
__device__ __forceinline__ void act_all(float (&z)[N], int act) {
  if (act == DSP_ACT_RELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) z[i] = z[i] < 0.f ? 0.f : z[i];  // NaN stays NaN
  } else if (act == DSP_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < N; ++i) z[i] = __fdividef(z[i], 1.f + exp2_fast(z[i] * -1.44269504f));
  } else if (act == DSP_ACT_GELU) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      constexpr int last = N - 1;
      const int j = i < last ? i + 1 : i;
      float c0, c1, e0, e1;
      normal2(z[i], z[j], c0, c1, e0, e1);
      const float y0 = z[i] * c0, y1 = z[j] * c1;
      z[i] = y0;
      if (j != i) z[j] = y1;
    }
  }
}

// x *= act'(z) of each element.
template <int N>
__device__ __forceinline__ void act_slopes(float (&x)[N], const float (&z)[N], int act) {
  if (act == DSP_ACT_RELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = z[i] <= 0.f ? 0.f : x[i];  // where z <= 0 nothing flows, an infinity neither; NaN lets all through
  } else if (act == DSP_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float e = __fdividef(1.f, 1.f + exp2_fast(z[i] * -1.44269504f));
      x[i] *= e * fmaf(z[i], 1.f - e, 1.f);
    }
  } else if (act == DSP_ACT_GELU) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      constexpr int last = N - 1;
      const int j = i < last ? i + 1 : i;
      float c0, c1, e0, e1;
      normal2(z[i], z[j], c0, c1, e0, e1);
      x[i] *= fmaf(z[i] * 0.39894228f, e0, c0);
      if (j != i) x[j] *= fmaf(z[j] * 0.39894228f, e1, c1);
    }
  }
}

// The epilogue of VE columns of one row: sum -> z -> pre, out. r: the residual's vector (zero where there is none).
template <class T, int VE>
__device__ __forceinline__ void finish(const ActArgs &a, int64_t row, int col, float (&z)[VE], const float (&bias)[VE],
                                       typename RowVec<T, VE>::Raw res) {
  using V = RowVec<T, VE>;
#pragma unroll
  for (int i = 0; i < VE; ++i) z[i] += bias[i];
  if (a.pre) st_f32<VE>(a.pre + row * a.ldp + col, z);
  act_all(z, a.act);
  if (a.residual) {
    float r[VE];
    V::widen(res, r);
#pragma unroll
    for (int i = 0; i < VE; ++i) z[i] += r[i];
  }
  V::st_stream((T *)a.out + row * a.ldo + col, z);
}

// Lanes of a warp: LPR of them span a row (VE elements each, VPL vectors), so G = 32 / LPR entries are gathered side by side, and
// each lane has the sums of its columns over its group's entries. scatter_sums adds the groups' sums and leaves FE = VE / G
// elements, number part() * FE on, with each lane: the epilogue's work is spread over all lanes.
template <int VE, int LPR>
struct Spread {
  static constexpr int G = 32 / LPR, FE = VE / G;
  static_assert(G <= VE, "an element for every group");
  static __device__ __forceinline__ int part() { return (threadIdx.x & 31) / LPR; }
  static __device__ __forceinline__ void scatter_sums(const float (&x)[VE], float (&out)[FE]) {
    float s[VE];
#pragma unroll
    for (int i = 0; i < VE; ++i) s[i] = x[i];
    int h = VE;
#pragma unroll
    for (int o = 16; o >= LPR; o >>= 1) {
      h >>= 1;
      const bool up = threadIdx.x & o;
#pragma unroll
      for (int i = 0; i < VE / 2; ++i)
        if (i < h) {
          const float keep = up ? s[i + h] : s[i], give = up ? s[i] : s[i + h];
          s[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
    }
#pragma unroll
    for (int i = 0; i < FE; ++i) out[i] = s[i];
  }
  // the inverse: every lane gets all VE elements
  static __device__ __forceinline__ void gather(const float (&in)[FE], float (&x)[VE]) {
#pragma unroll
    for (int i = 0; i < FE; ++i) x[i] = in[i];
    int h = FE;
#pragma unroll
    for (int o = LPR; o < 32; o <<= 1) {
      const bool up = threadIdx.x & o;
#pragma unroll
      for (int i = 0; i < VE / 2; ++i)
        if (i < h) {
          const float mine = x[i], other = __shfl_xor_sync(0xffffffffu, mine, o);
          x[i] = up ? other : mine;
          x[i + h] = up ? mine : other;
        }
      h <<= 1;
    }
  }
};

// A warp's chunk in shared memory: its entries (column, value) and row pointers. One coalesced read per list brings them in, so
// that a step waits for rows of B only, not for ids first (ids read step by step: 352 us instead of 275 on R-MAT 18, bf16,
// N = 128).
struct ChunkLists {
  int2 entry[kMaxUnits];
  int32_t ptr[kMaxUnits / kRowUnits + 4];
};
struct Chunk {
  int32_t r0, r1, p0, p1;
};
// value(p): the value of entry p.
template <class F>
__device__ __forceinline__ Chunk load_chunk(const DirView &d, int64_t chunk, ChunkLists &s, F &&value) {
  const int lane = threadIdx.x & 31;
  const Chunk c = {__ldg(d.row0 + chunk), __ldg(d.row0 + chunk + 1), __ldg(d.nz0 + chunk), __ldg(d.nz0 + chunk + 1)};
  __syncwarp();  // the last chunk's lists are read
  for (int i = lane; i <= c.r1 - c.r0 + 1; i += 32)
    if (c.r0 + i <= d.n) s.ptr[i] = __ldg(d.ptr + c.r0 + i);
#pragma unroll 4
  for (int i = lane; i < c.p1 - c.p0; i += 32) s.entry[i] = make_int2(__ldg(d.cols + c.p0 + i), __float_as_int(value(c.p0 + i)));
  __syncwarp();
  return c;
}

// One chunk per warp (TB: type of the gathered rows), row by row in steps of G U entries: a row's last step is partly masked. A finished row goes through the
// epilogue, a cut one to its slot. The residual of the running row is requested when the row begins, so that its end does not
// wait; rows without entries need no more than act(bias), worked out once.
template <class T, class TB, int VE, int LPR, int VPL, int U, int MINB, bool PERM>
__global__ void __launch_bounds__(kThreads, MINB) act_product_kernel(const DirView d, const ActArgs a) {
  using V = RowVec<TB, VE>;
  using S = Spread<VE, LPR>;
  constexpr int G = S::G, FE = S::FE;
  using F = RowVec<T, FE>;
  __shared__ ChunkLists lists[kThreads / 32];
  const int64_t chunk = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> 5;
  if (chunk >= d.n_chunks) return;
  ChunkLists &list = lists[threadIdx.x >> 5];
  const Chunk k = load_chunk(d, chunk, list, [&](int32_t p) { return __ldg(a.values + (PERM ? __ldg(d.perm + p) : p)); });
  const int g = S::part();
  const int col0 = blockIdx.y * (LPR * VE * VPL) + (threadIdx.x % LPR) * VE;  // gathered columns
  const int end0 = col0 + g * FE;                                            // columns finished here
  const bool head_cut = k.p0 > list.ptr[0];
  float acc[VPL][VE], bias[VPL][FE], idle[VPL][FE];
  typename F::Raw res[VPL];
  const char *src[VPL];  // lanes behind the last column read column 0 and store nothing
#pragma unroll
  for (int w = 0; w < VPL; ++w) {
    src[w] = (const char *)((const TB *)a.B + (col0 + w * LPR * VE < a.N ? col0 + w * LPR * VE : 0));
    res[w] = F::zero();
#pragma unroll
    for (int i = 0; i < FE; ++i) {
      const int col = end0 + w * LPR * VE + i;
      bias[w][i] = idle[w][i] = a.bias && col < a.N ? __ldg(a.bias + col) : 0.f;
    }
    act_all(idle[w], a.act);
  }
  int32_t row = k.r0;
  auto request = [&](int32_t r) {  // the residual of a row that ends here
#pragma unroll
    for (int w = 0; w < VPL; ++w) {
      const int col = end0 + w * LPR * VE;
      if (a.residual && r < k.r1 && col < a.N) res[w] = F::ld((const T *)a.residual + (int64_t)r * a.ldr + col);
    }
  };
  auto store_slot = [&](int64_t slot) {
#pragma unroll
    for (int w = 0; w < VPL; ++w) {
      const int col = end0 + w * LPR * VE;
      float z[FE];
      S::scatter_sums(acc[w], z);
      if (col < a.N) st_f32<FE>(a.slots + slot * a.N + col, z);
    }
  };
  auto fetch = [&](int32_t c, int w) { return V::ldg((const TB *)(src[w] + (uint64_t)(uint32_t)c * a.ldb_bytes)); };
  const int2 *entry = list.entry - k.p0;
  request(row);
  int32_t p = k.p0;
#pragma unroll 1
  for (; row <= k.r1; ++row) {
    const int32_t pe = row < k.r1 ? list.ptr[row - k.r0 + 1] : k.p1;
    const bool cut_head = row == k.r0 && head_cut;
    if (row == k.r1 && p >= pe) break;
    if (p >= pe && !cut_head) {  // no entries
      typename F::Raw now[VPL];
#pragma unroll
      for (int w = 0; w < VPL; ++w) now[w] = res[w];
      request(row + 1);
#pragma unroll
      for (int w = 0; w < VPL; ++w) {
        const int col = end0 + w * LPR * VE;
        if (col >= a.N) continue;
        if (a.pre) st_f32<FE>(a.pre + (int64_t)row * a.ldp + col, bias[w]);
        float y[FE], r[FE];
        F::widen(now[w], r);
#pragma unroll
        for (int i = 0; i < FE; ++i) y[i] = a.residual ? idle[w][i] + r[i] : idle[w][i];
        F::st_stream((T *)a.out + (int64_t)row * a.ldo + col, y);
      }
      continue;
    }
#pragma unroll
    for (int w = 0; w < VPL; ++w)
#pragma unroll
      for (int i = 0; i < VE; ++i) acc[w][i] = 0.f;
#pragma unroll 1
    for (; p + G * U <= pe; p += G * U) {
      typename V::Raw b[U][VPL];
      float v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int2 e = entry[p + u * G + g];
        v[u] = __int_as_float(e.y);
#pragma unroll
        for (int w = 0; w < VPL; ++w) b[u][w] = fetch(e.x, w);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int w = 0; w < VPL; ++w) fma_row<TB, VE>(acc[w], v[u], b[u][w]);
    }
    if (p < pe) {  // the last step: entries behind the row's end are read as its last one, and not added
      typename V::Raw b[U][VPL];
      float v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int2 e = entry[min(p + u * G + g, pe - 1)];
        v[u] = __int_as_float(e.y);
        if (u == 0 || p + u * G < pe) {
#pragma unroll
          for (int w = 0; w < VPL; ++w) b[u][w] = fetch(e.x, w);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (p + u * G + g < pe) {
#pragma unroll
          for (int w = 0; w < VPL; ++w) fma_row<TB, VE>(acc[w], v[u], b[u][w]);
        }
      p = pe;
    }
    if (cut_head || row == k.r1) {
      store_slot(cut_head ? 2 * chunk : 2 * chunk + 1);
      request(row + 1);
      continue;
    }
    typename F::Raw now[VPL];
    float z[VPL][FE];
#pragma unroll
    for (int w = 0; w < VPL; ++w) {
      now[w] = res[w];
      S::scatter_sums(acc[w], z[w]);
    }
    request(row + 1);
#pragma unroll
    for (int w = 0; w < VPL; ++w) {
      const int col = end0 + w * LPR * VE;
      if (col < a.N) finish<T, FE>(a, row, col, z[w], bias[w], now[w]);
    }
  }
}

// Rows cut across chunks: their partials go through the epilogue, added in chunk order: by one warp where there are few, in
// eight interleaved sums and then those eight in order where there are many (the first n_long of the list, a block each).
template <class T>
__global__ void __launch_bounds__(kThreads) act_join_kernel(const DirView d, const ActArgs a) {
  __shared__ float part[8][128];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool wide = (int)blockIdx.x < d.n_long;
  const int32_t at = wide ? (int)blockIdx.x : d.n_long + ((int)blockIdx.x - d.n_long) * 8 + warp;
  if (at >= d.n_split) return;  // whole warps of a narrow block: no barrier there
  const int32_t r = __ldg(d.split_row + at);
  const int64_t c0 = row_start(r, __ldg(d.ptr + r)) / d.L, c1 = row_start(r, __ldg(d.ptr + r + 1)) / d.L;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  typename RowVec<T, 1>::Raw res[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int col = blockIdx.y * 128 + lane + 32 * k;
    res[k] = RowVec<T, 1>::zero();
    if (a.residual && col < a.N) res[k] = RowVec<T, 1>::ld((const T *)a.residual + (int64_t)r * a.ldr + col);
  }
#pragma unroll 4
  for (int64_t c = c0 + (wide ? warp : 0); c <= c1; c += wide ? 8 : 1) {
    const float *src = a.slots + (c == c0 ? 2 * c + 1 : 2 * c) * a.N;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int col = blockIdx.y * 128 + lane + 32 * k;
      if (col < a.N) s[k] += src[col];
    }
  }
  if (wide) {
#pragma unroll
    for (int k = 0; k < 4; ++k) part[warp][lane + 32 * k] = s[k];
    __syncthreads();
    if (warp > 0) return;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      s[k] = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) s[k] += part[w][lane + 32 * k];
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int col = blockIdx.y * 128 + lane + 32 * k;
    if (col < a.N) {
      float z[1] = {s[k]}, b[1] = {a.bias ? __ldg(a.bias + col) : 0.f};
      finish<T, 1>(a, r, col, z, b, res[k]);
    }
  }
}

// ------------------------------------------------------------------------------------------------ gradients

struct GradArgs {
  int act, N;
  const void *B;
  uint32_t ldb_bytes;
  const float *pre;
  int64_t ldp;
  const void *dout;
  int64_t lddo;
  float *dz;         // [rows][N], or nullptr
  float *dvalues;    // [column blocks][nnz] (one block: the result itself), or nullptr
  float *dbias;      // [gridDim.x][N] partial sums, or nullptr
  int64_t nnz;
};

// Sum U values of each lane over the LPR lanes of a group. On return the lanes whose low bits (below LPR / U) are zero
// hold value number (lane within the group) / (LPR / U). Halving the values while crossing lanes takes U - 1 exchanges
// plus log2(LPR / U), instead of U log2(LPR).
template <int U, int LPR>
__device__ __forceinline__ float group_sums(float (&s)[U], int lane, uint32_t mask) {
  int h = U;
#pragma unroll
  for (int o = LPR / 2; o >= LPR / U && o > 0; o >>= 1) {
    h >>= 1;
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < U / 2; ++i)
      if (i < h) {
        const float keep = up ? s[i + h] : s[i], give = up ? s[i] : s[i + h];
        s[i] = keep + __shfl_xor_sync(mask, give, o);
      }
  }
  float x = s[0];
#pragma unroll
  for (int o = LPR / U / 2; o > 0; o >>= 1) x += __shfl_xor_sync(mask, x, o);
  return x;
}

// One pass over A's rows: dz (fp32, in registers for dvalues and dbias, and written for the product with A transposed: in 16 bits it
// added an error of the size of dB's own rounding, and in fp16 small gradients were lost; R-MAT 18, N = 128, bf16, silu, training step:
// 739 us with 16 bits, 794 with fp32, 850 with 24 bits in two planes), dvalues, and the block's share of dbias. The walk is the product
// kernel's; dout and z of the next row are requested when a row begins.
template <class T, int VE, int LPR, int VPL, int U, int MINB>
__global__ void __launch_bounds__(kThreads, MINB) act_grad_rows_kernel(const DirView d, const GradArgs a) {
  using V = RowVec<T, VE>;
  using S = Spread<VE, LPR>;
  constexpr int G = S::G, FE = S::FE;
  using F = RowVec<T, FE>;
  static_assert(LPR >= U, "a group holds a step's sums");
  constexpr int cols = LPR * VE * VPL;
  __shared__ union {
    ChunkLists lists[kThreads / 32];
    float sums[kThreads / 32][cols];
  } sm;
  ChunkLists &list = sm.lists[threadIdx.x >> 5];
  const int lane = threadIdx.x % LPR, g = S::part();
  const int col0 = blockIdx.y * cols + lane * VE;
  const int end0 = col0 + g * FE;  // columns whose dz this lane works out
  const char *src[VPL];  // lanes behind the last column read column 0 and drop it
#pragma unroll
  for (int w = 0; w < VPL; ++w) src[w] = (const char *)((const T *)a.B + (col0 + w * LPR * VE < a.N ? col0 + w * LPR * VE : 0));
  float *dv = a.dvalues ? a.dvalues + (int64_t)blockIdx.y * a.nnz : nullptr;
  float bsum[VPL][FE], z[VPL][FE];
  typename F::Raw dout[VPL];
#pragma unroll
  for (int w = 0; w < VPL; ++w)
#pragma unroll
    for (int i = 0; i < FE; ++i) bsum[w][i] = z[w][i] = 0.f;
  const int64_t warps = (int64_t)gridDim.x * (kThreads / 32);
#pragma unroll 1
  for (int64_t chunk = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> 5; chunk < d.n_chunks; chunk += warps) {
    const Chunk k = load_chunk(d, chunk, list, [](int32_t) { return 0.f; });
    const int2 *entry = list.entry - k.p0;
    auto request = [&](int32_t row) {  // dout and z of a row
#pragma unroll
      for (int w = 0; w < VPL; ++w) {
        const int col = end0 + w * LPR * VE;
        dout[w] = F::zero();
        if (row <= k.r1 && row < d.n && col < a.N) {
          dout[w] = F::ldg((const T *)a.dout + (int64_t)row * a.lddo + col);
          if (a.act != DSP_ACT_NONE) ld_f32<FE>(a.pre + (int64_t)row * a.ldp + col, z[w]);
        }
      }
    };
    request(k.r0);
    int32_t p = k.p0;
#pragma unroll 1
    for (int32_t row = k.r0; row <= k.r1; ++row) {
      const int32_t pe = row < k.r1 ? list.ptr[row - k.r0 + 1] : k.p1;
      if (row == k.r1 && p >= pe) break;
      float dz[VPL][VE];
      {
        float own[VPL][FE];
#pragma unroll
        for (int w = 0; w < VPL; ++w) {
          F::widen(dout[w], own[w]);
          act_slopes(own[w], z[w], a.act);
        }
        request(row + 1);
#pragma unroll
        for (int w = 0; w < VPL; ++w) {
          const int col = end0 + w * LPR * VE;
          if (row < k.r1) {  // the row ends here: counted and written once
#pragma unroll
            for (int i = 0; i < FE; ++i) bsum[w][i] += own[w][i];
            if (a.dz && col < a.N) st_f32<FE>(a.dz + (int64_t)row * a.N + col, own[w]);
          }
          if (p < pe) S::gather(own[w], dz[w]);
        }
      }
      if (!dv) p = pe;
#pragma unroll 1
      for (; p < pe; p += G * U) {
        typename V::Raw b[U][VPL];
        float s[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int2 e = entry[min(p + u * G + g, pe - 1)];
#pragma unroll
          for (int w = 0; w < VPL; ++w) b[u][w] = V::ldg((const T *)(src[w] + (uint64_t)(uint32_t)e.x * a.ldb_bytes));
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float x[2] = {0.f, 0.f};
#pragma unroll
          for (int w = 0; w < VPL; ++w)
            if (col0 + w * LPR * VE < a.N) dot_row<T, VE>(x, dz[w], b[u][w]);
          s[u] = x[0] + x[1];
        }
        const float x = group_sums<U, LPR>(s, lane, 0xffffffffu);
        constexpr int per = LPR / U;
        const int32_t at = p + (lane / per) * G + g;
        if (lane % per == 0 && at < pe) dv[at] = x;
      }
      p = pe;
    }
  }
  if (!a.dbias) return;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < VPL; ++w)
#pragma unroll
    for (int i = 0; i < FE; ++i) sm.sums[threadIdx.x >> 5][w * LPR * VE + lane * VE + g * FE + i] = bsum[w][i];
  __syncthreads();
  for (int c = threadIdx.x; c < cols; c += kThreads) {
    const int col = blockIdx.y * cols + c;
    if (col >= a.N) continue;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) s += sm.sums[w][c];
    a.dbias[(int64_t)blockIdx.x * a.N + col] = s;
  }
}

// out[c] = sum over the n rows of part, in an order that depends on n alone: 32 columns per block, 32 interleaved sums.
__global__ void __launch_bounds__(1024) column_sums_kernel(const float *part, int n, int N, float *out) {
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
  float x = 0.f;
  if (col < N) {
#pragma unroll 8
    for (int r = warp; r < n; r += 32) x += part[(int64_t)r * N + col];
  }
  s[warp][lane] = x;
  __syncthreads();
  if (warp == 0 && col < N) {
    x = 0.f;
#pragma unroll
    for (int w = 0; w < 32; ++w) x += s[w][lane];
    out[col] = x;
  }
}

// dvalues of a product wider than one column block: the blocks' shares, in order.
__global__ void __launch_bounds__(kThreads) add_blocks_kernel(const float *part, int blocks, int64_t nnz, float *out) {
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= nnz) return;
  float x = 0.f;
  for (int b = 0; b < blocks; ++b) x += part[b * nnz + i];
  out[i] = x;
}

// ------------------------------------------------------------------------------------------------ shapes and launches

struct Shape {
  int VE, LPR, VPL;
  int cols() const { return VE * LPR * VPL; }
};

bool aligned(const void *p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

// ve: the widest vector that every operand's address and leading dimension allow (8, 4 or 1). Lanes that span a row are the
// next power of two, at least 32 / VE; wider rows take two vectors a lane, then more column blocks.
Shape shape_of(int N, int ve, int size) {
  if (ve == 1) return {1, 32, N > 32 ? 4 : 1};
  int lpr = 32 / ve;
  while (lpr < 32 && lpr * ve < N) lpr *= 2;
  return {ve, lpr, lpr == 32 && N > 32 * ve ? 2 : 1};
}

// Entries a step and blocks an SM: 4 and 4 measured best (R-MAT 18 forward / R-MAT 16 fp32 training / R-MAT 18 training, us: 4, 4:
// 275 / 296 / 830; 4, 3: 276 / 377 / 895; 8, 3: 326 / 388 / 1007; 4, 5: 328 / 330 / 1044, spilling).
constexpr int kSteps = 4, kBlocks = 4;
template <class T, class TB, int VE, int LPR, int VPL, bool PERM>
void run_product(const DirView &d, const ActArgs &a, cudaStream_t s) {
  constexpr int U = kSteps, minb = VE * VPL >= 16 ? 2 : kBlocks;  // two vectors a lane take the registers of four blocks
  const dim3 grid((unsigned)((d.n_chunks + kThreads / 32 - 1) / (kThreads / 32)),
                  (unsigned)((a.N + VE * LPR * VPL - 1) / (VE * LPR * VPL)));
  act_product_kernel<T, TB, VE, LPR, VPL, U, minb, PERM><<<grid, kThreads, 0, s>>>(d, a);
}

template <class T, int VE, int LPR, int VPL>
void run_rows(const DirView &d, const GradArgs &a, int blocks, cudaStream_t s) {
  constexpr int U = kSteps, minb = VE * VPL >= 16 ? 2 : kBlocks;
  act_grad_rows_kernel<T, VE, LPR, VPL, U, minb>
      <<<dim3((unsigned)blocks, (unsigned)((a.N + VE * LPR * VPL - 1) / (VE * LPR * VPL))), kThreads, 0, s>>>(d, a);
}

// f.template operator()<VE, LPR, VPL>() of a shape.
template <class T, class F>
void with_shape(const Shape &h, F &&f) {
  if constexpr (sizeof(T) == 2) {
    if (h.VE == 8) {
      if (h.LPR == 4) return f.template operator()<8, 4, 1>();
      if (h.LPR == 8) return f.template operator()<8, 8, 1>();
      if (h.LPR == 16) return f.template operator()<8, 16, 1>();
      return h.VPL == 2 ? f.template operator()<8, 32, 2>() : f.template operator()<8, 32, 1>();
    }
  }
  if (h.VE == 4) {
    if (h.LPR == 8) return f.template operator()<4, 8, 1>();
    if (h.LPR == 16) return f.template operator()<4, 16, 1>();
    return h.VPL == 2 ? f.template operator()<4, 32, 2>() : f.template operator()<4, 32, 1>();
  }
  return h.VPL == 4 ? f.template operator()<1, 32, 4>() : f.template operator()<1, 32, 1>();
}

// TB: T, or float (dz of 16-bit operands; vectors of 4 at most).
template <class T, class TB>
struct Product {
  const DirView &d;
  const ActArgs &a;
  bool transposed;
  cudaStream_t s;
  template <int VE, int LPR, int VPL>
  void operator()() const {
    if constexpr (std::is_same<T, TB>::value) {
      if (transposed) run_product<T, TB, VE, LPR, VPL, true>(d, a, s);
      else run_product<T, TB, VE, LPR, VPL, false>(d, a, s);
    } else if constexpr (VE <= 4) {
      run_product<T, TB, VE, LPR, VPL, true>(d, a, s);
    }
  }
};

template <class T>
struct GradRows {
  const DirView &d;
  const GradArgs &a;
  int blocks;
  cudaStream_t s;
  template <int VE, int LPR, int VPL>
  void operator()() const {
    run_rows<T, VE, LPR, VPL>(d, a, blocks, s);
  }
};

template <class T, class TB>
int product(const DirView &d, const ActArgs &a, bool transposed, int ve, cudaStream_t s) {
  if (d.n_chunks > 0) with_shape<T>(shape_of(a.N, ve, (int)sizeof(T)), Product<T, TB>{d, a, transposed, s});
  if (d.n_split > 0)
    act_join_kernel<T><<<dim3((unsigned)join_blocks(d), (unsigned)((a.N + 127) / 128)), kThreads, 0, s>>>(d, a);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? DSP_OK : fail(DSP_ERR_CUDA, "dsp_spmm_act: %s", cudaGetErrorString(e));
}

int64_t up256(int64_t x) { return (x + 255) / 256 * 256; }

int64_t slot_bytes(const PatternDir &d, int N) { return d.n_split > 0 ? up256(8ll * d.n_chunks * N) : 0; }

// The widest vector (8, 4, 1 elements) for which each operand that is present is aligned.
struct Align {
  int size, N, ve;
  Align(int size_, int N_) : size(size_), N(N_), ve(size_ == 2 ? 8 : 4) {}
  void row(const void *p, int64_t ld) {
    if (!p) return;
    while (ve > 1 && (N % ve || ld % ve || !aligned(p, (size_t)ve * size))) ve = ve == 8 ? 4 : 1;
  }
  void row_f32(const void *p, int64_t ld) {  // fp32 beside rows of T: float4s
    if (p && ve > 1 && (ld % 4 || !aligned(p, 16))) ve = 1;
  }
};

int check_type(const char *who, int dtype, int act, int N) {
  DSP_TRY_ARG(dtype >= DSP_F32 && dtype <= DSP_F16, "%s: dtype %d", who, dtype);
  DSP_TRY_ARG(act >= DSP_ACT_NONE && act <= DSP_ACT_GELU, "%s: act %d", who, act);
  DSP_TRY_ARG(N >= 0, "%s: N = %d", who, N);
  if (N > (1 << 22)) return fail(DSP_ERR_UNSUPPORTED, "%s: N = %d: up to 2^22 is wanted", who, N);
  return DSP_OK;
}

int esize(int dtype) { return dtype == DSP_F32 ? 4 : 2; }

// Row strides of gathered operands are 32-bit byte counts in the kernels.
int check_stride(const char *who, const char *name, int64_t ld) {
  if (ld >= (1ll << 30)) return fail(DSP_ERR_UNSUPPORTED, "%s: %s = %lld: less than 2^30 is wanted", who, name, (long long)ld);
  return DSP_OK;
}

int check_workspace(const char *who, const void *ws, int64_t have, int64_t need) {
  if (need == 0) return DSP_OK;
  DSP_TRY_ARG(ws && have >= need, "%s: workspace of %lld bytes, %lld needed", who, (long long)(ws ? have : 0),
              (long long)need);
  DSP_TRY_ARG(aligned(ws, 256), "%s: the workspace must be 256-byte aligned", who);
  return DSP_OK;
}

struct GradPlan {
  Shape shape;
  int blocks, col_blocks;
  int64_t dz, slots, dbias, dvalues, total;  // workspace offsets
};

GradPlan grad_plan(const dsp_pattern *p, const dsp_act_grad_desc *d) {
  GradPlan g = {};
  Align al(esize(d->dtype), d->N);
  al.row(d->B, d->ldb);
  al.row(d->dout, d->lddo);
  al.row(d->dB, d->lddb);
  if (d->act != DSP_ACT_NONE) al.row_f32(d->pre, d->ldp);
  g.shape = shape_of(d->N, al.ve, esize(d->dtype));
  g.col_blocks = (d->N + g.shape.cols() - 1) / g.shape.cols();
  g.blocks = (int)std::max<int64_t>(
      1, std::min<int64_t>((int64_t)kBlocks * p->sms, (p->a.n_chunks + kThreads / 32 - 1) / (kThreads / 32)));
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at += up256(bytes);
    return o;
  };
  g.dz = take(d->dB && d->act != DSP_ACT_NONE ? 4 * p->rows * d->N : 0);
  g.slots = take(d->dB ? slot_bytes(p->t, d->N) : 0);
  g.dbias = take(d->dbias ? 4ll * g.blocks * d->N : 0);
  g.dvalues = take(d->dvalues && g.col_blocks > 1 ? 4ll * g.col_blocks * p->nnz : 0);
  g.total = at;
  return g;
}

template <class T>
int grad(const dsp_pattern *p, const dsp_act_grad_desc *d, char *ws, cudaStream_t s) {
  const GradPlan g = grad_plan(p, d);
  const bool needs_dz = d->dB && d->act != DSP_ACT_NONE;
  if (needs_dz || d->dvalues || d->dbias) {
    GradArgs a = {};
    a.act = d->act, a.N = d->N, a.B = d->B, a.ldb_bytes = (uint32_t)(d->ldb * sizeof(T)), a.pre = d->pre, a.ldp = d->ldp, a.dout = d->dout;
    a.lddo = d->lddo, a.nnz = p->nnz;
    a.dz = needs_dz ? (float *)(ws + g.dz) : nullptr;
    a.dvalues = !d->dvalues || p->nnz == 0 ? nullptr : g.col_blocks > 1 ? (float *)(ws + g.dvalues) : d->dvalues;
    a.dbias = d->dbias ? (float *)(ws + g.dbias) : nullptr;
    const DirView rows = view(p->a);
    with_shape<T>(g.shape, GradRows<T>{rows, a, g.blocks, s});
    if (d->dbias)
      column_sums_kernel<<<(d->N + 31) / 32, 1024, 0, s>>>((float *)(ws + g.dbias), g.blocks, d->N, d->dbias);
    if (a.dvalues && g.col_blocks > 1)
      add_blocks_kernel<<<(unsigned)((p->nnz + kThreads - 1) / kThreads), kThreads, 0, s>>>(a.dvalues, g.col_blocks, p->nnz,
                                                                                           d->dvalues);
  }
  if (d->dB) {
    ActArgs a = {};
    a.act = DSP_ACT_NONE, a.N = d->N, a.values = d->values, a.out = d->dB, a.ldo = d->lddb;
    a.slots = (float *)(ws + g.slots);
    Align al((int)sizeof(T), d->N);
    al.row(a.out, a.ldo);
    if (needs_dz) {
      a.B = ws + g.dz;
      a.ldb_bytes = 4u * (uint32_t)d->N;
      return product<T, float>(view(p->t), a, true, std::min(al.ve, 4), s);
    }
    a.B = d->dout;
    a.ldb_bytes = (uint32_t)(d->lddo * sizeof(T));
    al.row(a.B, d->lddo);
    return product<T, T>(view(p->t), a, true, al.ve, s);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? DSP_OK : fail(DSP_ERR_CUDA, "dsp_spmm_act_grad: %s", cudaGetErrorString(e));
}

}  // namespace
}  // namespace dsp

using namespace dsp;

extern "C" int64_t dsp_spmm_act_workspace(const dsp_pattern *p, int N) {
  return p && N > 0 ? slot_bytes(p->a, N) : 0;
}

extern "C" int dsp_spmm_act(const dsp_pattern *p, const dsp_act_desc *d, void *workspace, int64_t workspace_bytes,
                            void *stream) {
  const char *who = "dsp_spmm_act";
  DSP_TRY_ARG(p && d, "%s: null argument", who);
  int rc = check_type(who, d->dtype, d->act, d->N);
  if (rc) return rc;
  if (d->N == 0 || p->rows == 0) return DSP_OK;
  DSP_TRY_ARG(d->out && d->ldo >= d->N, "%s: out, ldo = %lld", who, (long long)d->ldo);
  DSP_TRY_ARG(p->nnz == 0 || (d->B && d->values && d->ldb >= d->N), "%s: B, values, ldb = %lld", who, (long long)d->ldb);
  DSP_TRY_ARG(!d->residual || d->ldr >= d->N, "%s: ldr = %lld", who, (long long)d->ldr);
  DSP_TRY_ARG(!d->pre || d->ldp >= d->N, "%s: ldp = %lld", who, (long long)d->ldp);
  DSP_TRY_ARG(d->residual != d->out || d->ldr == d->ldo, "%s: a residual in place needs ldr = ldo", who);
  if ((rc = check_stride(who, "ldb", d->ldb))) return rc;
  rc = check_workspace(who, workspace, workspace_bytes, dsp_spmm_act_workspace(p, d->N));
  if (rc) return rc;
  DeviceGuard g(p->device);
  if (g.err != cudaSuccess) return fail(DSP_ERR_CUDA, "%s: %s", who, cudaGetErrorString(g.err));
  Align al(esize(d->dtype), d->N);
  if (p->nnz) al.row(d->B, d->ldb);
  al.row(d->residual, d->ldr);
  al.row(d->out, d->ldo);
  al.row_f32(d->pre, d->ldp);
  ActArgs a = {d->act, d->N,   d->values, d->B,   (uint32_t)(d->ldb * esize(d->dtype)), d->bias, d->residual,
               d->ldr, d->out, d->ldo,    d->pre, d->ldp, (float *)workspace};
  cudaStream_t s = (cudaStream_t)stream;
  if (d->dtype == DSP_F32) return product<float, float>(view(p->a), a, false, al.ve, s);
  if (d->dtype == DSP_BF16) return product<__nv_bfloat16, __nv_bfloat16>(view(p->a), a, false, al.ve, s);
  return product<__half, __half>(view(p->a), a, false, al.ve, s);
}

extern "C" int64_t dsp_spmm_act_grad_workspace(const dsp_pattern *p, const dsp_act_grad_desc *d) {
  if (!p || !d || d->N <= 0 || d->dtype < DSP_F32 || d->dtype > DSP_F16) return 0;
  return grad_plan(p, d).total;
}

extern "C" int dsp_spmm_act_grad(const dsp_pattern *p, const dsp_act_grad_desc *d, void *workspace,
                                 int64_t workspace_bytes, void *stream) {
  const char *who = "dsp_spmm_act_grad";
  DSP_TRY_ARG(p && d, "%s: null argument", who);
  int rc = check_type(who, d->dtype, d->act, d->N);
  if (rc) return rc;
  if (d->dB && !(p->flags & DSP_PATTERN_GRAD))
    return fail(DSP_ERR_STATE, "%s: dB needs a pattern with DSP_PATTERN_GRAD", who);
  DSP_TRY_ARG(!d->dB || d->lddb >= d->N, "%s: lddb = %lld", who, (long long)d->lddb);
  DSP_TRY_ARG(d->act == DSP_ACT_NONE || p->rows == 0 || d->N == 0 || (d->pre && d->ldp >= d->N),
              "%s: the activation's gradient needs pre", who);
  DSP_TRY_ARG(p->rows == 0 || d->N == 0 || (d->dout && d->lddo >= d->N), "%s: dout, lddo = %lld", who, (long long)d->lddo);
  DSP_TRY_ARG(p->nnz == 0 || d->N == 0 || !d->dvalues || (d->B && d->ldb >= d->N), "%s: B, ldb = %lld", who,
              (long long)d->ldb);
  DSP_TRY_ARG(p->nnz == 0 || d->N == 0 || !d->dB || d->values, "%s: null values", who);
  DeviceGuard g(p->device);
  if (g.err != cudaSuccess) return fail(DSP_ERR_CUDA, "%s: %s", who, cudaGetErrorString(g.err));
  cudaStream_t s = (cudaStream_t)stream;
  if (d->N == 0) {  // an empty sum for every entry
    if (d->dvalues && p->nnz) {
      const cudaError_t e = cudaMemsetAsync(d->dvalues, 0, sizeof(float) * (size_t)p->nnz, s);
      if (e != cudaSuccess) return fail(DSP_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
    }
    return DSP_OK;
  }
  if ((rc = check_stride(who, "ldb", d->ldb)) || (rc = check_stride(who, "lddo", d->lddo))) return rc;
  rc = check_workspace(who, workspace, workspace_bytes, dsp_spmm_act_grad_workspace(p, d));
  if (rc) return rc;
  char *ws = (char *)workspace;
  if (d->dtype == DSP_F32) return grad<float>(p, d, ws, s);
  if (d->dtype == DSP_BF16) return grad<__nv_bfloat16>(p, d, ws, s);
  return grad<__half>(p, d, ws, s);
}
