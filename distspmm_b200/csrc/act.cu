// act.cu — out = act(A.B + bias) + residual and its gradients.
//
//   z_i = sum over the entries p of row i of a_p B[c_p] + bias,   out_i = act(z_i) + residual_i
//   dz_i = dout_i act'(z_i),   dB = A^T dz,   da_p = dz_{r_p} . B[c_p],   dbias = sum_i dz_i
//
// The work is a gather of one row of B (or dz) per entry; the arithmetic is two operations per element read, so the kernels
// are bound by how fast rows come out of L2 (or HBM, once B is larger than the 126 MB L2). What the design does about it:
// 16-bit rows stay 16-bit until they are in registers, the epilogue adds no pass over the result, and work is cut into
// chunks of equal entries + row ends, so that hub rows and runs of empty rows are spread evenly. A group of LPR lanes owns a
// chunk, each lane VPL vectors of VE columns; no lane talks to another in the product kernel.
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
  int64_t ldb;
  const float *bias;
  const void *residual;
  int64_t ldr;
  void *out;
  int64_t ldo;
  float *pre;
  int64_t ldp;
  float *slots;  // [2 n_chunks][N] partial rows
};

__device__ __forceinline__ float act_of(float z, int act) {
  if (act == DSP_ACT_RELU) return z > 0.f ? z : (z == z ? 0.f : z);  // NaN stays NaN
  if (act == DSP_ACT_SILU) return z / (1.f + expf(-z));
  if (act == DSP_ACT_GELU) return 0.5f * z * erfcf(-0.70710678118654752f * z);
  return z;
}

__device__ __forceinline__ float act_slope(float z, int act) {
  if (act == DSP_ACT_RELU) return z > 0.f ? 1.f : 0.f;
  if (act == DSP_ACT_SILU) {
    const float e = 1.f / (1.f + expf(-z));
    return e * (1.f + z * (1.f - e));
  }
  if (act == DSP_ACT_GELU)
    return 0.5f * erfcf(-0.70710678118654752f * z) + z * 0.39894228040143268f * expf(-0.5f * z * z);
  return 1.f;
}

// The epilogue of VE columns of one row: sum -> z -> pre, out. r: the residual's vector (zero where there is none).
template <class T, int VE>
__device__ __forceinline__ void finish(const ActArgs &a, int64_t row, int col, float (&z)[VE], const float (&bias)[VE],
                                       typename RowVec<T, VE>::Raw res) {
  using V = RowVec<T, VE>;
#pragma unroll
  for (int i = 0; i < VE; ++i) z[i] += bias[i];
  if (a.pre) st_f32<VE>(a.pre + row * a.ldp + col, z);
  if (a.act != DSP_ACT_NONE) {
#pragma unroll
    for (int i = 0; i < VE; ++i) z[i] = act_of(z[i], a.act);
  }
  if (a.residual) {
    float r[VE];
    V::widen(res, r);
#pragma unroll
    for (int i = 0; i < VE; ++i) z[i] += r[i];
  }
  V::st_stream((T *)a.out + row * a.ldo + col, z);
}

// One chunk per group of LPR lanes, walked in steps of U entries: the U rows of B are requested together, whatever rows of A
// they belong to, then added to the running row; a finished row goes through the epilogue, a cut one to its slot. The
// residual of the running row is requested when the row begins, so that a row's end does not wait for it.
template <class T, int VE, int LPR, int VPL, int U, int MINB, bool PERM>
__global__ void __launch_bounds__(kThreads, MINB) act_product_kernel(const DirView d, const ActArgs a) {
  using V = RowVec<T, VE>;
  const int64_t chunk = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / LPR;
  if (chunk >= d.n_chunks) return;
  const int col0 = blockIdx.y * (LPR * VE * VPL) + (threadIdx.x % LPR) * VE;
  const int32_t r0 = __ldg(d.row0 + chunk), r1 = __ldg(d.row0 + chunk + 1);
  const int32_t p0 = __ldg(d.nz0 + chunk), p1 = __ldg(d.nz0 + chunk + 1);
  const bool head_cut = p0 > __ldg(d.ptr + r0);
  float acc[VPL][VE], bias[VPL][VE];
  typename V::Raw res[VPL];
  int32_t row = r0;
  auto begin_row = [&]() {
#pragma unroll
    for (int w = 0; w < VPL; ++w) {
#pragma unroll
      for (int i = 0; i < VE; ++i) acc[w][i] = 0.f;
      const int col = col0 + w * LPR * VE;
      if (a.residual && row < r1 && col < a.N) res[w] = V::ld((const T *)a.residual + (int64_t)row * a.ldr + col);
    }
  };
#pragma unroll
  for (int w = 0; w < VPL; ++w) {
    res[w] = V::zero();
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      const int col = col0 + w * LPR * VE + i;
      bias[w][i] = a.bias && col < a.N ? __ldg(a.bias + col) : 0.f;
    }
  }
  begin_row();
  auto store_slot = [&](int64_t slot) {
#pragma unroll
    for (int w = 0; w < VPL; ++w) {
      const int col = col0 + w * LPR * VE;
      if (col < a.N) st_f32<VE>(a.slots + slot * a.N + col, acc[w]);
    }
  };
  auto end_rows = [&](int32_t to) {  // rows row .. to - 1 end in this chunk
#pragma unroll 1
    while (row < to) {
      if (row == r0 && head_cut) {
        store_slot(2 * chunk);
        ++row;
        begin_row();
        continue;
      }
      typename V::Raw now[VPL];
      float z[VPL][VE];
#pragma unroll
      for (int w = 0; w < VPL; ++w) {
        now[w] = res[w];
#pragma unroll
        for (int i = 0; i < VE; ++i) z[w][i] = acc[w][i];
      }
      const int64_t at = row++;
      begin_row();
#pragma unroll
      for (int w = 0; w < VPL; ++w) {
        const int col = col0 + w * LPR * VE;
        if (col < a.N) finish<T, VE>(a, at, col, z[w], bias[w], now[w]);
      }
    }
  };
  const T *B = (const T *)a.B + col0;
  // entries come in aligned groups of 4 (the id lists are padded); those outside [p0, p1) are masked
#pragma unroll 1
  for (int32_t p = p0 & ~3; p < p1; p += U) {
    int32_t c[U];
    float v[U];
#pragma unroll
    for (int q = 0; q < U / 4; ++q) {
      const int4 c4 = __ldg(reinterpret_cast<const int4 *>(d.cols + p) + q);
      c[4 * q] = c4.x, c[4 * q + 1] = c4.y, c[4 * q + 2] = c4.z, c[4 * q + 3] = c4.w;
    }
    const bool whole = p >= p0 && p + U <= p1;
    const int32_t last = __ldg(d.row_of + (p + U <= p1 ? p + U : p1) - 1);
    if (PERM) {
#pragma unroll
      for (int q = 0; q < U / 4; ++q) {
        const int4 x = __ldg(reinterpret_cast<const int4 *>(d.perm + p) + q);
        const int32_t at = p + 4 * q;
        v[4 * q] = at >= p0 && at < p1 ? __ldg(a.values + x.x) : 0.f;
        v[4 * q + 1] = at + 1 >= p0 && at + 1 < p1 ? __ldg(a.values + x.y) : 0.f;
        v[4 * q + 2] = at + 2 >= p0 && at + 2 < p1 ? __ldg(a.values + x.z) : 0.f;
        v[4 * q + 3] = at + 3 >= p0 && at + 3 < p1 ? __ldg(a.values + x.w) : 0.f;
      }
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = p + u >= p0 && p + u < p1 ? __ldg(a.values + p + u) : 0.f;
    }
    typename V::Raw b[U][VPL];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = whole || (p + u >= p0 && p + u < p1);
      const T *src = B + (int64_t)c[u] * a.ldb;
#pragma unroll
      for (int w = 0; w < VPL; ++w) b[u][w] = in && col0 + w * LPR * VE < a.N ? V::ldg(src + w * LPR * VE) : V::zero();
    }
    auto add = [&](int u) {
#pragma unroll
      for (int w = 0; w < VPL; ++w) {
        float f[VE];
        V::widen(b[u][w], f);
#pragma unroll
        for (int i = 0; i < VE; ++i) acc[w][i] = fmaf(v[u], f[i], acc[w][i]);
      }
    };
    if (whole && last == row) {  // rows are in order: the whole step belongs to the running row
#pragma unroll
      for (int u = 0; u < U; ++u) add(u);
    } else {
      int32_t r[U];
#pragma unroll
      for (int u = 0; u < U; ++u) r[u] = p + u < p0 ? -1 : p + u < p1 ? __ldg(d.row_of + p + u) : INT32_MAX;
#pragma unroll 1
      while (true) {
        int32_t next = last;  // the first listed row after the running one
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (r[u] == row) add(u);
          if (r[u] > row) next = min(next, r[u]);
        }
        if (row >= last) break;
        end_rows(next);
      }
    }
  }
  end_rows(r1);
  if (p1 > max(p0, __ldg(d.ptr + r1))) store_slot(r1 == r0 && head_cut ? 2 * chunk : 2 * chunk + 1);
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
  int64_t ldb;
  const float *pre;
  int64_t ldp;
  const void *dout;
  int64_t lddo;
  void *dz;          // [rows][N] T, or nullptr
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

// One pass over A's rows: dz (kept in registers in fp32, so that dvalues and dbias see it unrounded; written in T for the
// product with A transposed, whose sums over many rows are rounded to T anyway), dvalues, and the block's share of dbias.
template <class T, int VE, int LPR, int VPL>
__global__ void __launch_bounds__(kThreads) act_grad_rows_kernel(const DirView d, const GradArgs a) {
  using V = RowVec<T, VE>;
  constexpr int U = 8;
  static_assert(LPR >= U, "a group holds a step's sums");
  __shared__ float sums[kThreads * VE * VPL];
  const int lane = threadIdx.x % LPR;
  const uint32_t mask = LPR == 32 ? 0xffffffffu : ((1u << (LPR & 31)) - 1u) << ((threadIdx.x & 31) / LPR * LPR);
  const int col0 = blockIdx.y * (LPR * VE * VPL) + lane * VE;
  const T *B = (const T *)a.B + col0;
  float bsum[VPL][VE];
#pragma unroll
  for (int w = 0; w < VPL; ++w)
#pragma unroll
    for (int i = 0; i < VE; ++i) bsum[w][i] = 0.f;
  const int64_t groups = (int64_t)gridDim.x * (kThreads / LPR);
  for (int64_t chunk = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / LPR; chunk < d.n_chunks; chunk += groups) {
    const int32_t r0 = __ldg(d.row0 + chunk), r1 = __ldg(d.row0 + chunk + 1);
    const int32_t p0 = __ldg(d.nz0 + chunk), p1 = __ldg(d.nz0 + chunk + 1);
    int32_t p = p0;
    for (int32_t row = r0; row <= r1; ++row) {
      const int32_t pe = row < r1 ? __ldg(d.ptr + row + 1) : p1;
      if (row == r1 && p >= pe) break;
      float dz[VPL][VE];
#pragma unroll
      for (int w = 0; w < VPL; ++w) {
        const int col = col0 + w * LPR * VE;
        const bool in = col < a.N;
        V::widen(in ? V::ldg((const T *)a.dout + (int64_t)row * a.lddo + col) : V::zero(), dz[w]);
        if (a.act != DSP_ACT_NONE && in) {
          float z[VE];
          ld_f32<VE>(a.pre + (int64_t)row * a.ldp + col, z);
#pragma unroll
          for (int i = 0; i < VE; ++i) dz[w][i] *= act_slope(z[i], a.act);
        }
        if (row < r1) {  // the row ends here: it is counted and written once
#pragma unroll
          for (int i = 0; i < VE; ++i) bsum[w][i] += dz[w][i];
          if (a.dz && in) V::st((T *)a.dz + (int64_t)row * a.N + col, dz[w]);
        }
      }
      if (!a.dvalues) {
        p = pe;
        continue;
      }
      float *dv = a.dvalues + (int64_t)blockIdx.y * a.nnz;
      for (; p < pe; p += U) {
        const int n = min(U, pe - p);
        typename V::Raw b[U][VPL];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const T *src = B + (u < n ? (int64_t)__ldg(d.cols + p + u) * a.ldb : 0);
#pragma unroll
          for (int w = 0; w < VPL; ++w)
            b[u][w] = u < n && col0 + w * LPR * VE < a.N ? V::ldg(src + w * LPR * VE) : V::zero();
        }
        float s[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          s[u] = 0.f;
#pragma unroll
          for (int w = 0; w < VPL; ++w) {
            float f[VE];
            V::widen(b[u][w], f);
#pragma unroll
            for (int i = 0; i < VE; ++i) s[u] = fmaf(dz[w][i], f[i], s[u]);
          }
        }
        const float x = group_sums<U, LPR>(s, lane, mask);
        constexpr int per = LPR / U;
        if (lane % per == 0 && lane / per < n) dv[p + lane / per] = x;
      }
      p = pe;
    }
  }
  if (!a.dbias) return;
#pragma unroll
  for (int w = 0; w < VPL; ++w)
#pragma unroll
    for (int i = 0; i < VE; ++i) sums[(threadIdx.x / LPR) * (LPR * VE * VPL) + w * LPR * VE + lane * VE + i] = bsum[w][i];
  __syncthreads();
  constexpr int cols = LPR * VE * VPL;
  for (int c = threadIdx.x; c < cols; c += kThreads) {
    const int col = blockIdx.y * cols + c;
    if (col >= a.N) continue;
    float s = 0.f;
    for (int g = 0; g < kThreads / LPR; ++g) s += sums[g * cols + c];
    a.dbias[(int64_t)blockIdx.x * a.N + col] = s;
  }
}

// out[c] = sum over the n rows of part, in an order that depends on n alone: 32 columns per block, 8 interleaved sums.
__global__ void __launch_bounds__(kThreads) column_sums_kernel(const float *part, int n, int N, float *out) {
  __shared__ float s[8][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
  float x = 0.f;
  if (col < N)
    for (int r = warp; r < n; r += 8) x += part[(int64_t)r * N + col];
  s[warp][lane] = x;
  __syncthreads();
  if (warp == 0 && col < N) {
    x = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) x += s[w][lane];
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

// ve: the widest vector that every operand's address and leading dimension allow (8, 4 or 1). A whole warp spans a row where
// the row fills it; narrower rows give each chunk a part of the warp.
Shape shape_of(int N, int ve, int size) {
  if (ve == 8 && size == 2 && N >= 256) return {8, 32, N > 256 ? 2 : 1};
  if (ve >= 4) {
    if (N > 64) return {4, 32, N > 128 ? 2 : 1};
    return {4, N > 32 ? 16 : 8, 1};
  }
  return {1, 32, N > 32 ? 4 : 1};
}

template <class T, int VE, int LPR, int VPL, bool PERM>
void run_product(const DirView &d, const ActArgs &a, cudaStream_t s) {
#ifndef ACT_U
#define ACT_U 4
#define ACT_B 4
#endif
  constexpr int U = VE * VPL >= 8 ? 4 : ACT_U;
  const dim3 grid((unsigned)(((int64_t)d.n_chunks * LPR + kThreads - 1) / kThreads),
                  (unsigned)((a.N + VE * LPR * VPL - 1) / (VE * LPR * VPL)));
  constexpr int minb = VE * VPL >= 16 ? 2 : VE * VPL == 8 ? ACT_B - 1 : ACT_B;
  act_product_kernel<T, VE, LPR, VPL, U, minb, PERM><<<grid, kThreads, 0, s>>>(d, a);
}

template <class T, bool PERM>
void pick_product(const Shape &h, const DirView &d, const ActArgs &a, cudaStream_t s) {
  if constexpr (sizeof(T) == 2) {
    if (h.VE == 8) return h.VPL == 2 ? run_product<T, 8, 32, 2, PERM>(d, a, s) : run_product<T, 8, 32, 1, PERM>(d, a, s);
  }
  if (h.VE == 4) {
    if (h.LPR == 32) return h.VPL == 2 ? run_product<T, 4, 32, 2, PERM>(d, a, s) : run_product<T, 4, 32, 1, PERM>(d, a, s);
    return h.LPR == 16 ? run_product<T, 4, 16, 1, PERM>(d, a, s) : run_product<T, 4, 8, 1, PERM>(d, a, s);
  }
  return h.VPL == 4 ? run_product<T, 1, 32, 4, PERM>(d, a, s) : run_product<T, 1, 32, 1, PERM>(d, a, s);
}

template <class T>
int product(const DirView &d, const ActArgs &a, bool transposed, int ve, cudaStream_t s) {
  const Shape h = shape_of(a.N, ve, (int)sizeof(T));
  if (d.n_chunks > 0) {
    if (transposed) pick_product<T, true>(h, d, a, s);
    else pick_product<T, false>(h, d, a, s);
  }
  if (d.n_split > 0)
    act_join_kernel<T><<<dim3((unsigned)join_blocks(d), (unsigned)((a.N + 127) / 128)), kThreads, 0, s>>>(d, a);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? DSP_OK : fail(DSP_ERR_CUDA, "dsp_spmm_act: %s", cudaGetErrorString(e));
}

template <class T, int VE, int LPR, int VPL>
void run_rows(const DirView &d, const GradArgs &a, int blocks, cudaStream_t s) {
  act_grad_rows_kernel<T, VE, LPR, VPL>
      <<<dim3((unsigned)blocks, (unsigned)((a.N + VE * LPR * VPL - 1) / (VE * LPR * VPL))), kThreads, 0, s>>>(d, a);
}

template <class T>
void pick_rows(const Shape &h, const DirView &d, const GradArgs &a, int blocks, cudaStream_t s) {
  if constexpr (sizeof(T) == 2) {
    if (h.VE == 8) return h.VPL == 2 ? run_rows<T, 8, 32, 2>(d, a, blocks, s) : run_rows<T, 8, 32, 1>(d, a, blocks, s);
  }
  if (h.VE == 4) {
    if (h.LPR == 32) return h.VPL == 2 ? run_rows<T, 4, 32, 2>(d, a, blocks, s) : run_rows<T, 4, 32, 1>(d, a, blocks, s);
    return h.LPR == 16 ? run_rows<T, 4, 16, 1>(d, a, blocks, s) : run_rows<T, 4, 8, 1>(d, a, blocks, s);
  }
  return h.VPL == 4 ? run_rows<T, 1, 32, 4>(d, a, blocks, s) : run_rows<T, 1, 32, 1>(d, a, blocks, s);
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
  return DSP_OK;
}

int esize(int dtype) { return dtype == DSP_F32 ? 4 : 2; }

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
      1, std::min<int64_t>(8ll * p->sms, ((int64_t)p->a.n_chunks * g.shape.LPR + kThreads - 1) / kThreads));
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at += up256(bytes);
    return o;
  };
  g.dz = take(d->dB && d->act != DSP_ACT_NONE ? p->rows * d->N * esize(d->dtype) : 0);
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
    a.act = d->act, a.N = d->N, a.B = d->B, a.ldb = d->ldb, a.pre = d->pre, a.ldp = d->ldp, a.dout = d->dout;
    a.lddo = d->lddo, a.nnz = p->nnz;
    a.dz = needs_dz ? ws + g.dz : nullptr;
    a.dvalues = !d->dvalues || p->nnz == 0 ? nullptr : g.col_blocks > 1 ? (float *)(ws + g.dvalues) : d->dvalues;
    a.dbias = d->dbias ? (float *)(ws + g.dbias) : nullptr;
    pick_rows<T>(g.shape, view(p->a), a, g.blocks, s);
    if (d->dbias)
      column_sums_kernel<<<(d->N + 31) / 32, kThreads, 0, s>>>((float *)(ws + g.dbias), g.blocks, d->N, d->dbias);
    if (a.dvalues && g.col_blocks > 1)
      add_blocks_kernel<<<(unsigned)((p->nnz + kThreads - 1) / kThreads), kThreads, 0, s>>>(a.dvalues, g.col_blocks, p->nnz,
                                                                                           d->dvalues);
  }
  if (d->dB) {
    ActArgs a = {};
    a.act = DSP_ACT_NONE, a.N = d->N, a.values = d->values, a.out = d->dB, a.ldo = d->lddb;
    a.B = needs_dz ? ws + g.dz : d->dout;
    a.ldb = needs_dz ? d->N : d->lddo;
    a.slots = (float *)(ws + g.slots);
    Align al((int)sizeof(T), d->N);
    al.row(a.B, a.ldb);
    al.row(a.out, a.ldo);
    return product<T>(view(p->t), a, true, al.ve, s);
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
  rc = check_workspace(who, workspace, workspace_bytes, dsp_spmm_act_workspace(p, d->N));
  if (rc) return rc;
  DeviceGuard g(p->device);
  if (g.err != cudaSuccess) return fail(DSP_ERR_CUDA, "%s: %s", who, cudaGetErrorString(g.err));
  Align al(esize(d->dtype), d->N);
  if (p->nnz) al.row(d->B, d->ldb);
  al.row(d->residual, d->ldr);
  al.row(d->out, d->ldo);
  al.row_f32(d->pre, d->ldp);
  ActArgs a = {d->act, d->N,      d->values, d->B,   d->ldb, d->bias, d->residual,
               d->ldr, d->out,    d->ldo,    d->pre, d->ldp, (float *)workspace};
  cudaStream_t s = (cudaStream_t)stream;
  if (d->dtype == DSP_F32) return product<float>(view(p->a), a, false, al.ve, s);
  if (d->dtype == DSP_BF16) return product<__nv_bfloat16>(view(p->a), a, false, al.ve, s);
  return product<__half>(view(p->a), a, false, al.ve, s);
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
  rc = check_workspace(who, workspace, workspace_bytes, dsp_spmm_act_grad_workspace(p, d));
  if (rc) return rc;
  char *ws = (char *)workspace;
  if (d->dtype == DSP_F32) return grad<float>(p, d, ws, s);
  if (d->dtype == DSP_BF16) return grad<__nv_bfloat16>(p, d, ws, s);
  return grad<__half>(p, d, ws, s);
}
