// attn_decode.cu — single query tokens over listed cache rows, 16-bit caches of dim 64 or 128.
//
// Every listed key and value row is read once for all query heads of its group, so the cache's bytes bound the kernel (16
// query heads on one row of 256 bytes are 32 operations a byte, far below the tensor cores' rate). A warp owns a chunk of the
// list and one key/value head; its query heads (8 at a time) are the n = 8 side of m16n8k16 products:
//
//   S^T [16 keys x 8 heads] = K Q^T        A = 16 key rows, straight from global memory to the lanes that need them
//   O^T [dim x 8 heads]    += V^T P^T      A = V^T, B = P^T: S^T's lanes hold 8 x 8 blocks, movmatrix turns them
//
// Rows go from global memory to fragments without a stop (frag.cuh). The next 16 keys are requested as soon as the products
// have read the present ones, so each warp keeps about 8 KB in flight. Weights are split in two 16-bit parts, p = hi + lo, with a product
// for each: the tensor cores are idle anyway, and no more than 2^-16 of a weight (fp16: 2^-22) is lost. An infinity that is listed
// would meet lo parts of 0 or of the other sign: rows whose result is not finite, though their weights are, are done again by
// attn_row.cuh's gather.
#include <algorithm>
#include <type_traits>

#include "attn_decode.h"
#include "attn_row.cuh"
#include "frag.cuh"

namespace dsp {
namespace {

constexpr int kThreads = 128;
constexpr int kMaxList = 1024, kBadRows = kMaxList / kRowUnits + 4;  // units of a chunk; its rows

// A row is read once: past L1, and as DRAM delivers it (240 -> 231 us on 64 x ~4800 tokens, 8 heads of 128, against plain loads).
__device__ __forceinline__ uint4 ld_row(const void *p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}

// 16 keys of the list: K rows lane / 4 and lane / 4 + 8, of each the 16-byte vectors lane % 4 + 4 i; V rows (keys) 2 t, 2 t + 1,
// 2 t + 8, 2 t + 9 for t = lane % 4, of each the vectors lane / 4 + 8 i.
template <class T, int D>
struct Tile {
  uint4 k[2][D / 32];
  uint4 v[4][D / 64];

  // ids: entry e of the 16 in lanes e and e + 16; -1: behind the end, -2: no such key
  __device__ __forceinline__ void load_k(const AttnArgs &a, int hk, int ids) {
    const int lane = threadIdx.x & 31, t = lane & 3;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int id = __shfl_sync(0xffffffffu, ids, (lane >> 2) + 8 * j);
      const T *src = (const T *)a.k.p + (int64_t)id * a.k.row + (int64_t)hk * a.k.head + t * 8;
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
        k[j][i] = id >= 0 ? ld_row(src + 32 * i) : make_uint4(0, 0, 0, 0);
    }
  }
  __device__ __forceinline__ void load_v(const AttnArgs &a, int hk, int ids) {
    const int lane = threadIdx.x & 31, t = lane & 3;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int id = __shfl_sync(0xffffffffu, ids, 2 * t + (j & 1) + 8 * (j >> 1));
      const T *src = (const T *)a.v.p + (int64_t)id * a.v.row + (int64_t)hk * a.v.head + (lane >> 2) * 8;
#pragma unroll
      for (int i = 0; i < D / 64; ++i)
        v[j][i] = id >= 0 ? ld_row(src + 64 * i) : make_uint4(0, 0, 0, 0);
    }
  }
};

template <class T, int D>
__global__ void __launch_bounds__(kThreads, 3) attn_decode_kernel(const __grid_constant__ ListRows d, const __grid_constant__ AttnArgs a, int head_tiles) {
  const int lane = threadIdx.x & 31, t = lane & 3, n8 = lane >> 2;
  const int kv_heads = a.heads / a.group, per_chunk = kv_heads * head_tiles;
  const int64_t item = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> 5;
  const int64_t chunk = item / per_chunk;
  if (chunk >= d.n_chunks) return;
  const int hk = (int)(item - chunk * per_chunk) / head_tiles, tile = (int)(item % head_tiles);
  const int h0 = hk * a.group + tile * 8, live = min(8, a.group - tile * 8);  // query heads h0 .. h0 + live - 1
  const float inv_cap2 = a.cap > 0.f ? 2.f * kLog2e / a.cap : 0.f, scale2 = a.scale * kLog2e;
  // of S^T this lane holds keys n8 and n8 + 8 of heads 2 t and 2 t + 1
  float slope2[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) slope2[j] = a.slopes && 2 * t + j < live ? __ldg(a.slopes + h0 + 2 * t + j) * kLog2e : 0.f;
  int64_t r0, r1, p, p1;
  d.chunk(chunk, r0, r1, p, p1);
  // heads of the chunk's rows to be done again (lists that are no CSR may give a chunk more rows than kBadRows)
  __shared__ uint8_t all_bad[kThreads / 32][kBadRows];
  for (int i = lane; i < kBadRows; i += 32) all_bad[threadIdx.x >> 5][i] = 0;
  __syncwarp();
  const bool head_cut = p > d.ptr(r0);
  for (int64_t row = r0; row <= r1; ++row) {
    if (row == r1 && (p >= p1 || row >= d.n())) break;
    const int64_t end = d.ptr(row + 1), pe = row < r1 ? end : p1;
    auto ids_at = [&](int64_t b) {
      const int64_t at = b + (lane & 15);
      if (at >= pe) return -1;
      const int64_t c = d.col(at);
      return d.in_range(c) ? (int)c : -2;
    };
    int ids = ids_at(p), next = ids_at(p + 16);
    Tile<T, D> x;
    x.load_k(a, hk, ids);
    x.load_v(a, hk, ids);
    // Q^T as B fragments: k steps of 16 in the order of K's vectors (step 2 i + j: words 2 j, 2 j + 1 of vector i)
    uint32_t q[D / 16][2];
    load_column<T, D>(q, (const T *)a.q.p + row * a.q.row + (int64_t)(h0 + n8) * a.q.head, n8 < live);
    float acc[D / 16][4];
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};  // of heads 2 t, 2 t + 1; l: this lane's keys only
#pragma unroll 1
    for (int64_t b = p; b < pe; b += 16) {
      float s[4] = {0.f, 0.f, 0.f, 0.f};
      rows_times<T, D>(s, x.k, q);
      const int now = ids;
      ids = next;
      x.load_k(a, hk, ids);  // the next 16, while these are weighed
      next = ids_at(b + 32);
      // scores, base 2, of keys n8 (s[0], s[1]) and n8 + 8 (s[2], s[3])
      float top[2] = {m[0], m[1]};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = n8 + 8 * (j >> 1), id = __shfl_sync(0xffffffffu, now, key);
        float th, u = s[j];
        if (a.cap > 0.f) u = capped(u * a.scale, a.cap, inv_cap2, th) * kLog2e;
        else u *= scale2;
        u = fmaf(-slope2[j & 1], (float)(end - 1 - b - key), u);
        if (id == -1) u = -INFINITY;
        if (id == -2) u = NAN;
        s[j] = u;
        top[j & 1] = fmaxf(top[j & 1], u);
      }
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], o));
        top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], o));
      }
      float base[2], keep[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        base[j] = top[j] == -INFINITY ? 0.f : top[j];
        keep[j] = exp2_approx(m[j] - base[j]);
        m[j] = top[j];
        l[j] *= keep[j];
      }
      if (__any_sync(0xffffffffu, keep[0] != 1.f || keep[1] != 1.f)) {
        // acc's columns are heads 2 t, 2 t + 1 too (rows: places of dim)
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] *= keep[j & 1];
      }
      uint32_t parts[2][2];  // weights of keys n8 + 8 j as hi and lo parts, turned
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float p0 = exp2_approx(s[2 * j] - base[0]), p1w = exp2_approx(s[2 * j + 1] - base[1]);
        l[0] += p0;
        l[1] += p1w;
        uint32_t hi, lo;
        split2<T>(p0, p1w, hi, lo);
        parts[0][j] = transpose8x8(hi);
        parts[1][j] = transpose8x8(lo);
      }
      turned_times<T, D, 2>(acc, x.v, parts);
      x.load_v(a, hk, ids);
    }
    // the sum over all keys, then the rows' results
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      l[0] += __shfl_xor_sync(0xffffffffu, l[0], o);
      l[1] += __shfl_xor_sync(0xffffffffu, l[1], o);
    }
    const bool cut_head = row == r0 && head_cut, cut = cut_head || row == r1;
    const int64_t slot = (cut_head ? 2 * chunk : 2 * chunk + 1) * a.heads;
    uint32_t bad = 0;  // heads with a result that is not finite, though the weights are
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int h = h0 + 2 * t + j;
      if (2 * t + j >= live) continue;
      const float inv = l[j] == 0.f ? 0.f : 1.f / l[j];
      float zero = 0.f;
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        // elements 2 c (acc[.][j]) and 2 c + 1 (acc[.][2 + j]) of vector n8 + 8 i
        float f[8];
#pragma unroll
        for (int c = 0; c < 4; ++c) f[2 * c] = acc[4 * i + c][j], f[2 * c + 1] = acc[4 * i + c][2 + j];
        const int col = (n8 + 8 * i) * 8;
        if (cut) {
          st_f32<8>(a.slots + (slot + h) * D + col, f);
        } else {
#pragma unroll
          for (int c = 0; c < 8; ++c) f[c] *= inv, zero = fmaf(f[c], 0.f, zero);
          RowVec<T, 8>::st((T *)a.out.p + row * a.out.row + (int64_t)h * a.out.head + col, f);
        }
      }
      if (n8 == 0) {
        if (cut) a.slot_ml[2 * (slot + h)] = m[j], a.slot_ml[2 * (slot + h) + 1] = l[j];
        else if (a.lse) a.lse[row * a.heads + h] = l[j] == 0.f ? -INFINITY : (m[j] + log2f(l[j])) * kLn2;
      }
      if (zero != 0.f && l[j] == l[j]) bad |= 1u << (2 * t + j);
    }
    if (__any_sync(0xffffffffu, bad != 0) && row - r0 < kBadRows)
      all_bad[threadIdx.x >> 5][row - r0] = (uint8_t)__reduce_or_sync(0xffffffffu, bad);
    p = pe;
  }
  __syncwarp();
  const uint8_t *bad_rows = all_bad[threadIdx.x >> 5];
  uint32_t any = 0;
  for (int i = lane; i < kBadRows; i += 32) any |= bad_rows[i];
  if (!__any_sync(0xffffffffu, any != 0)) return;
#pragma unroll 1
  for (int i = 0; i < kBadRows; ++i)  // after the loop: a call within it would cost its registers
#pragma unroll 1
    for (uint32_t bad = bad_rows[i]; bad; bad &= bad - 1) attend_again<T, D>(d, a, r0 + i, h0 + __ffs(bad) - 1);
}

// Rows cut across chunks: a block per row and head. The partials' weights 2^(m - max) first, each by a thread, then the
// weighted sums: groups of dim threads, a thread per column, take every groups-th partial, and their sums are added in order.
constexpr int kJoin = 512;
template <class T>
__global__ void __launch_bounds__(kJoin, 2) attn_decode_join_kernel(const __grid_constant__ ListRows d, const __grid_constant__ AttnArgs a) {
  __shared__ float weight[kJoin], red[kJoin / 32], part[kJoin];
  const int64_t r = blockIdx.x;
  const int h = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t c0 = row_start(r, d.ptr(r)) / d.L, c1 = min(row_start(r, d.ptr(r + 1)) / d.L, (int64_t)d.n_chunks - 1);
  if (c0 >= c1) return;  // not cut
  auto slot = [&](int64_t c) { return (c == c0 ? 2 * c + 1 : 2 * c) * a.heads + h; };
  float m = -INFINITY;
  for (int64_t c = c0 + tid; c <= c1; c += kJoin) m = fmaxf(m, a.slot_ml[2 * slot(c)]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) red[warp] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kJoin / 32; ++w) m = fmaxf(m, red[w]);
  const float base = m == -INFINITY ? 0.f : m;
  const int groups = kJoin / a.dim, g = tid / a.dim, col = tid - g * a.dim;  // dim <= 256
  float l = 0.f, acc = 0.f;
  for (int64_t b = c0; b <= c1; b += kJoin) {
    const int n = (int)min((int64_t)kJoin, c1 - b + 1);
    float w = 0.f;
    if (tid < n) {
      const int64_t s = slot(b + tid);
      w = exp2_approx(a.slot_ml[2 * s] - base);
      l += w * a.slot_ml[2 * s + 1];
    }
    __syncthreads();
    weight[tid] = w;
    __syncthreads();
    if (g < groups) {
#pragma unroll 8
      for (int i = g; i < n; i += groups) acc = fmaf(weight[i], a.slots[slot(b + i) * a.dim + col], acc);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  __syncthreads();
  if (lane == 0) red[warp] = l;
  part[tid] = acc;
  __syncthreads();
  l = 0.f;
#pragma unroll
  for (int w = 0; w < kJoin / 32; ++w) l += red[w];
  bool bad = false;
  if (tid < a.dim) {
    for (int k = 1; k < groups; ++k) acc += part[k * a.dim + tid];
    acc = l == 0.f ? 0.f : acc / l;
    bad = !isfinite(acc);
    ((T *)a.out.p)[r * a.out.row + h * a.out.head + tid] = T(acc);
  }
  if (a.lse && tid == 0) a.lse[r * a.heads + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
  if constexpr (sizeof(T) == 2) {
    if (__syncthreads_or(bad && l == l) && warp == 0) {  // the barrier: other warps' results are written
      if (a.dim == 64) attend_again<T, 64>(d, a, r, h);
      else if (a.dim == 128) attend_again<T, 128>(d, a, r, h);
    }
  }
}

template <class T>
int run(const ListRows &d, const AttnArgs &a, cudaStream_t s) {
  const int kv_heads = a.heads / a.group, head_tiles = (a.group + 7) / 8;
  const unsigned blocks = (unsigned)(((int64_t)d.n_chunks * kv_heads * head_tiles + kThreads / 32 - 1) / (kThreads / 32));
  if (a.dim == 64) attn_decode_kernel<T, 64><<<blocks, kThreads, 0, s>>>(d, a, head_tiles);
  else attn_decode_kernel<T, 128><<<blocks, kThreads, 0, s>>>(d, a, head_tiles);
  return decode_join(d, a, std::is_same<T, __nv_bfloat16>::value ? DSP_BF16 : DSP_F16, s);
}

}  // namespace

bool decode_on_tensor_cores(int dtype, int dim) { return dtype != DSP_F32 && (dim == 64 || dim == 128); }

int32_t decode_units(int64_t rows, int64_t nnz, int heads, int kv_heads, bool tensor) {
  // Warps to fill the 12 places of every SM three times over (tensor cores: a warp has a key/value head and 8 query heads), 32
  // to 1024 units each. Fewer leave the last round uneven, more write more partials: 64 x ~4800 tokens, 8 heads of 128, with
  // 24 / 36 / 48 warps an SM: 250 / 231 / 240 us.
  const int64_t width = tensor ? (int64_t)kv_heads * ((heads / kv_heads + 7) / 8) : heads;
  const int64_t l = (row_start(rows, nnz) * width + 148 * 36 - 1) / (148 * 36);
  return (int32_t)std::min<int64_t>(kMaxList, std::max<int64_t>(32, (l + 15) / 16 * 16));
}

int decode_join(const ListRows &d, const AttnArgs &a, int dtype, cudaStream_t s) {
  if (d.n_chunks > 1) {
    const dim3 grid((unsigned)d.rows, (unsigned)a.heads);
    if (dtype == DSP_F32) attn_decode_join_kernel<float><<<grid, kJoin, 0, s>>>(d, a);
    else if (dtype == DSP_BF16) attn_decode_join_kernel<__nv_bfloat16><<<grid, kJoin, 0, s>>>(d, a);
    else attn_decode_join_kernel<__half><<<grid, kJoin, 0, s>>>(d, a);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? DSP_OK : fail(DSP_ERR_CUDA, "dsp_attn_decode: %s", cudaGetErrorString(e));
}

int decode_tensor(const ListRows &d, const AttnArgs &a, int dtype, cudaStream_t s) {
  return dtype == DSP_BF16 ? run<__nv_bfloat16>(d, a, s) : run<__half>(d, a, s);
}

}  // namespace dsp
