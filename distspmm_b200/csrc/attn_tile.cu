// attn_tile.cu — attention over the tile form of a pattern, on the 5th-generation tensor cores (bf16, fp16; dim 64 or 128).
//
// One kernel in three roles, each a stationary tile of 128 rows against a stream of tiles of 64 rows (the tiles the pattern
// lists), with products of 128 x 64 x dim and 128 x dim x 64 per tile:
//
//             stationary   stream    first products            weights (16-bit, in tensor memory)   second products
//   forward   Q            K, V      S = Q K^T                 P = exp(u - m)                       O += P V
//   dq        Q, dO        K, V      S = Q K^T, R = dO V^T     dS = P (R - delta0) c, P c           dQ += dS K, Y += P c K
//   dk, dv    K, V         Q, dO     S^T = K Q^T, R^T = V dO^T P^T, dS^T                            dV += P^T dO, dK += dS^T Q
//
// All weights but P c are in two parts.
//
// A CTA: four warps of weights (a thread owns one of the 128 rows: the running maximum, sum and all masks are its own
// registers, no shuffles), one warp of TMA loads, one that issues the products. Scores arrive in tensor memory, weights go
// back into the same columns as the A operand of the second product, so neither passes through shared memory; the stream's
// tiles serve both products from one swizzled image (K-major in the first, N-major in the second). The sums over keys stay in
// tensor memory; the forward pass rescales its own only when a row's maximum grew by more than 2^8 (kSlack), which leaves
// the result the same (weights and their sum share the stale maximum). It takes the tiles from the last to the first: under a
// causal mask with a distance bias scores fall along that way, and the maximum stands after one tile.
//
// Rounding: weights enter the second products as hi + lo, two parts of the operands' 16-bit type, and so do the score gradients
// (2^-16 of a value is lost at most). One part alone put a second rounding of the result's size into out and dv (window case below:
// 218 instead of 260 us forward; documents: 115 instead of 126 us dk and dv). The first delta0 = dout . out has a rounded out in it; so
// dq = scale (sum p c (dp - delta0) k - g sum p c k) with g = sum p (dp - delta0) = delta - delta0. The weights p c of the last sum may be
// rounded once, since g is of a rounding's size itself. dk and dv read delta0 + g.
//
// fp16 has few exponents: weights are carried 2^6 above (forward) or 2^12 above (backward) their value, and dS is scaled by a power of
// two that brings the largest |dout| (of the row for dq, of the streamed rows for dk and dv) near 16; both come off in the epilogue.
// Rows whose largest dS still leaves fp16's range, or comes so low that its parts lose bits, are computed again as below.
//
// Masks and values that are not finite: an entry that is not listed has weight 0, but 0 x NaN in the product is NaN. So a row
// whose result is not finite is computed again by attn_row.cuh's gather, which reads listed entries only. A NaN that belongs
// there stays, one that leaked in does not.
//
// Bounds: on the tensor cores a tile of dim 128 takes 256 cycles for each product (the forward's second: twice, for two parts), the
// first 384 since 128 x 64 x 16 steps read shared memory 1.5 times as fast as it delivers; its exponentials take 512 on the special
// function units. The forward takes some 1900 cycles a tile and SM: neither of the two bounds it, but the chain of waits from scores
// to weights to products, which two CTAs on an SM (tensor memory and registers allow no third) overlap only in part. Measured: 8192
// rows, window 1024 with 64 first keys, 32 query heads over 8 of 128, distance bias: 260 us, 525 TFLOP/s of listed entries; documents,
// 6001 rows, 16 heads of 64, cap: 67 us forward, 106 dq, 126 dk and dv.
#include <algorithm>
#include <type_traits>

#include "attn_row.cuh"
#include "attn_tile.h"
#include "frag.cuh"
#include "tcgen05.cuh"

namespace dsp {
namespace {

enum Mode { kFwd, kDq, kDkv };
constexpr int kThreads = 192, kWeightThreads = 128;
constexpr float kSlack = 8.f;

struct TileView {
  const int32_t *ptr, *col, *mask, *order;
  const uint64_t *words;
};

struct TileArgs {
  TileView t;
  AttnArgs a;
  PlanRows rows;        // the gather form of the same orientation
  int n_heads;          // heads of the grid (query heads, or key/value heads for dk, dv)
  int splits;           // pieces of a row tile's list (forward)
  float *part, *part_ml;  // their partial results: [splits][rows][heads][dim], [splits][rows][heads][2]
  int *err;
  long long wait_cycles;  // limit of a wait; 0: no copies are started, so that waits run out (tests)
};

template <int D, Mode M>
struct Cfg {
  static constexpr int kStatic = M == kFwd ? 1 : 2;            // stationary operands
  static constexpr int kScores = M == kFwd ? 1 : 2;            // score tiles of 64 columns
  static constexpr int NB = M == kFwd || D == 128 ? 2 : 1;  // score buffers
  static constexpr int ST = 2;                                 // stages of each streamed operand
  static constexpr int kAcc = kScores * NB * 64;               // first accumulator column
  static constexpr int kUsed = kAcc + (M == kFwd ? 1 : 2) * D;
  static constexpr int kCols = kUsed <= 128 ? 128 : kUsed <= 256 ? 256 : 512;
  static constexpr int kStaticBytes = 128 * D * 2, kStreamBytes = 64 * D * 2;
  static constexpr int kSmemUsed = kStatic * kStaticBytes + 2 * ST * kStreamBytes + 1024;
  // no more CTAs of a launch on an SM than tensor memory has room for: their allocations do not wait for one another. CTAs of
  // different launches (another stream's forward of 256 columns beside a backward of 512) may still meet on an SM: the later one's
  // allocation then waits until the earlier one ends, as it will, since all its own waits have limits.
  static constexpr int kCtas = 512 / kCols;
  static constexpr int kSmemLeast = 232448 / (kCtas + 1) + 1024;
  static constexpr int kSmem = kSmemUsed > kSmemLeast ? kSmemUsed : kSmemLeast;
};

// Bounded wait; gives up at once where another thread of the CTA has.
__device__ __noinline__ bool wait_slow(uint32_t bar, uint32_t parity, volatile int *dead, const TileArgs &x, int code) {
  const long long t0 = clock64();
  while (true) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    if (done) return true;
    if (*dead) return false;
    if (clock64() - t0 > x.wait_cycles) {
      *dead = 1;
      atomicExch(x.err, code);
      return false;
    }
  }
}
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile int *dead, const TileArgs &x, int code) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done ? true : wait_slow(bar, parity, dead, x, code);
}

// The same by a whole warp, which leaves it together.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int *dead, const TileArgs &x, int code) {
  return __all_sync(0xffffffffu, wait(bar, parity, dead, x, code));
}

// The second products of iterations 0, 1, ... complete on kAccBars barriers in turn. A thread waits for some of them only, and a
// wait tells two phases of a barrier apart by their parity alone: with one barrier, a late thread would take phase n for phase
// n - 2. On these, the phase before the awaited one is four iterations old and the one after it four ahead.
constexpr int kAccBars = 4;
__device__ __forceinline__ bool wait_acc(uint32_t bars, int it, volatile int *dead, const TileArgs &x, int code) {
  return warp_wait(bars + 8 * (it % kAccBars), (it / kAccBars) & 1, dead, x, code);
}

// s -> cap tanh(k s), k = scale / cap, of N columns of this thread's row. Where no score of the warp's rows is above half the cap, as
// is usual, tanh x = x P(x^2) (degree 9, through Chebyshev nodes, within 1.2e-7) leaves the special function units to the
// softmax, with k and the cap in the coefficients: 6 operations an element; else through the exponential (capped).
struct CapPoly {
  float limit, c[5];  // of s^2; s (c0 + c1 s^2 + ...)
  __device__ __forceinline__ CapPoly(float scale, float cap) {
    const float k = cap > 0.f ? scale / cap : 0.f, k2 = k * k;
    limit = k2 < 1e20f ? 0.25f / fmaxf(k2, 1e-20f) : -1.f;  // beyond, the coefficients overflow
    float f = k * cap;
    c[0] = kTanh0 * f;
    c[1] = kTanh1 * (f *= k2);
    c[2] = kTanh2 * (f *= k2);
    c[3] = kTanh3 * (f *= k2);
    c[4] = kTanh4 * (f *= k2);
  }
};
template <int N>
__device__ __forceinline__ void cap_row(float (&s)[N], const CapPoly &p, float cap, float scale, float inv_cap2) {
  float y[N], top = 0.f;
#pragma unroll
  for (int c = 0; c < N; c += 2) {
    mul2(y[c], y[c + 1], s[c], s[c + 1], s[c], s[c + 1]);
    top = max3(top, y[c], y[c + 1]);
  }
  if (__all_sync(0xffffffffu, top <= p.limit)) {
#pragma unroll
    for (int c = 0; c < N; c += 2) {
      float q0, q1;
      fma2(q0, q1, p.c[4], p.c[4], y[c], y[c + 1], p.c[3], p.c[3]);
      fma2(q0, q1, q0, q1, y[c], y[c + 1], p.c[2], p.c[2]);
      fma2(q0, q1, q0, q1, y[c], y[c + 1], p.c[1], p.c[1]);
      fma2(q0, q1, q0, q1, y[c], y[c + 1], p.c[0], p.c[0]);
      mul2(s[c], s[c + 1], s[c], s[c + 1], q0, q1);
    }
  } else {
#pragma unroll
    for (int c = 0; c < N; ++c) {
      float th;
      s[c] = capped(s[c] * scale, cap, inv_cap2, th);
    }
  }
}

// Tiles of the list as a thread of the weights sees them, in the order first, first + step, ...: place and mask two iterations
// ahead, the row's presence bits one ahead, so that no load is waited for.
struct TileWalk {
  const TileView &t;
  int r, at, left, step, wrap;  // wrap: tiles until the list starts again
  int mask, col, mask2 = 0, col2 = 0;
  uint64_t bits;
  int seen = 0;
  // full tiles read their words too: a choice between loaded and constant bits would wait for the load
  __device__ __forceinline__ uint64_t words(int m) const { return __ldg(t.words + (int64_t)m * kTileRows + r); }
  __device__ __forceinline__ TileWalk(const TileView &t_, int first, int step_, int n, int total, int r_)
      : t(t_), r(r_), at(first), left(total), step(step_), wrap(n) {
    mask = col = 0, bits = 0;
    if (left > 0) {
      mask = __ldg(t.mask + at), col = __ldg(t.col + at);
      next2();
      bits = words(mask);
    }
  }
  __device__ __forceinline__ void next2() {  // place and mask of the tile after the present one
    if (--left <= 0) return;
    at += step;
    if (++seen == wrap) seen = 0, at -= step * wrap;
    mask2 = __ldg(t.mask + at), col2 = __ldg(t.col + at);
  }
  __device__ __forceinline__ void advance() {
    mask = mask2, col = col2;
    bits = words(mask);
    next2();
  }
};

// Rows of a warp whose result is not finite (bits of `bad`), again by gather.
template <class T, int D, Mode M>
__device__ __noinline__ void redo(const TileArgs &x, int64_t row0, int head, uint32_t bad) {
  using H = HeadRow<T, 8, D / 8, 1>;
  const int lane = threadIdx.x % (D / 8), g = (threadIdx.x & 31) / (D / 8);
  __syncwarp();  // the rows' first results were written by other lanes than will write them now
  while (bad) {
    const int64_t row = row0 + __ffs(bad) - 1;
    bad &= bad - 1;
    const int64_t p = x.rows.ptr(row), pe = x.rows.ptr(row + 1);
    float y[1][8], z[1][8], m, l;  // dq: m is delta - delta0, l is delta0
    if constexpr (M == kFwd) {
      attend<H, D / 8>(x.rows, x.a, row, head, p, pe, pe, m, l, y);
      put_row<H, D / 8>(x.a, row, head, m, l, y);
    } else if constexpr (M == kDq) {
      attend_dq<H, D / 8>(x.rows, x.a, row, head, p, pe, m, l, y, z);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[0][i] = (y[0][i] - m * z[0][i]) * x.a.scale;
      if (g == 0) H::store(x.a.dq, row, head, lane, D, y);
      if ((threadIdx.x & 31) == 0) x.a.delta[row * x.a.heads + head] = l + m;
    } else {
      attend_dkv<H, D / 8>(x.rows, x.a, row, head, p, pe, y, z);
      if (g == 0) {
        H::store(x.a.dk, row, head, lane, D, y);
        H::store(x.a.dv, row, head, lane, D, z);
      }
    }
  }
}

// A row of NaN: what a wait that gave up leaves.
template <class T, int D>
__device__ __forceinline__ void put_nan(const HeadsOut &o, int64_t row, int head) {
  T *dst = (T *)o.p + row * o.row + (int64_t)head * o.head;
#pragma unroll 1
  for (int c = 0; c < D; c += 8) *reinterpret_cast<uint4 *>(dst + c) = make_uint4(0x7fff7fff, 0x7fff7fff, 0x7fff7fff, 0x7fff7fff);
}

// D columns of this thread's row at `addr`, times f (TWO: plus those at `addr2` times f2), to the row's place in global memory; whether
// all were finite.
template <class T, int D, bool TWO = false>
__device__ __forceinline__ bool put_acc(uint32_t addr, float f, const HeadsOut &o, int64_t row, int head, bool store, uint32_t addr2 = 0,
                                        float f2 = 0.f) {
  bool fine = true;
  T *dst = (T *)o.p + row * o.row + (int64_t)head * o.head;
#pragma unroll 1
  for (int c = 0; c < D; c += 32) {
    uint32_t r[32], r2[TWO ? 32 : 1];
    tmem_ld32(addr + c, r);
    if constexpr (TWO) tmem_ld32(addr2 + c, r2);
    tmem_wait_ld();
    auto value = [&](int i) {
      const float x = __uint_as_float(r[i]) * f;
      if constexpr (TWO) return fmaf(__uint_as_float(r2[i]), f2, x);
      else return x;
    };
#pragma unroll
    for (int i = 0; i < 32; i += 8) {
      uint4 w;
      uint32_t *w4 = &w.x;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float lo = value(i + 2 * j), hi = value(i + 2 * j + 1);
        fine &= isfinite(lo) && isfinite(hi);
        w4[j] = pack2<T>(lo, hi);
      }
      if (store) *reinterpret_cast<uint4 *>(dst + c + i) = w;
    }
  }
  return fine;
}

template <class T, int D, Mode M>
__global__ void __launch_bounds__(kThreads, Cfg<D, M>::kCtas > 2 ? 2 : Cfg<D, M>::kCtas)
    attn_tile_kernel(const __grid_constant__ CUtensorMap map_a0, const __grid_constant__ CUtensorMap map_a1,
                     const __grid_constant__ CUtensorMap map_x0, const __grid_constant__ CUtensorMap map_x1,
                     const __grid_constant__ TileArgs x) {
  using C = Cfg<D, M>;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr int NB = C::NB, ST = C::ST;
  extern __shared__ uint8_t raw_smem[];
  __shared__ uint64_t bars[1 + 4 * ST + 2 * NB + kAccBars + 1];
  __shared__ uint32_t tmem_result;
  __shared__ int dead_flag;
  __shared__ uint32_t tops[4];
  __shared__ __align__(16) float row_lse[2][64], row_delta[2][64];  // dk, dv: -lse (base 2) and -delta of the streamed rows
  volatile int *dead = &dead_flag;

  const int warp = threadIdx.x >> 5;
  const int head = blockIdx.x % x.n_heads, rt = __ldg(x.t.order + blockIdx.x / x.n_heads);
  int t0 = __ldg(x.t.ptr + rt), t1 = __ldg(x.t.ptr + rt + 1);
  if (M == kFwd && x.splits > 1) {
    const int n = t1 - t0, z = blockIdx.y;
    t1 = t0 + (int)((int64_t)n * (z + 1) / x.splits);
    t0 = t0 + (int)((int64_t)n * z / x.splits);
  }
  const int nt = t1 - t0, iters = M == kDkv ? nt * x.a.group : nt;
  const int64_t row0 = (int64_t)rt * kTileRows;

  const uint32_t sm = (smem_addr(raw_smem) + 1023u) & ~1023u;
  const uint32_t sm_a0 = sm, sm_a1 = sm + C::kStaticBytes * (C::kStatic - 1);
  const uint32_t sm_x0 = sm + C::kStatic * C::kStaticBytes, sm_x1 = sm_x0 + ST * C::kStreamBytes;
  const uint32_t b0 = smem_addr(bars);
  const uint32_t bar_static = b0, bar_x0_full = b0 + 8, bar_x0_free = bar_x0_full + 8 * ST, bar_x1_full = bar_x0_free + 8 * ST,
                 bar_x1_free = bar_x1_full + 8 * ST, bar_scores = bar_x1_free + 8 * ST, bar_weights = bar_scores + 8 * NB,
                 bar_acc = bar_weights + 8 * NB, bar_stats = bar_acc + 8 * kAccBars;

  if (iters > 0 && warp == 5) tmem_alloc(smem_addr(&tmem_result), C::kCols);
  if (threadIdx.x == 0) {
    dead_flag = 0;
    mbar_init(bar_static, 1);
    for (int i = 0; i < ST; ++i) {
      mbar_init(bar_x0_full + 8 * i, 1);
      mbar_init(bar_x0_free + 8 * i, 1);
      mbar_init(bar_x1_full + 8 * i, 1);
      mbar_init(bar_x1_free + 8 * i, 1);
    }
    for (int i = 0; i < NB; ++i) {
      mbar_init(bar_scores + 8 * i, 1);
      mbar_init(bar_weights + 8 * i, kWeightThreads);
    }
    for (int i = 0; i < kAccBars; ++i) mbar_init(bar_acc + 8 * i, 1);
    mbar_init(bar_stats, kWeightThreads);
    mbar_fence_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm = iters > 0 ? tmem_result : 0;
  const uint32_t tm_s = tm, tm_r = tm + NB * 64, tm_acc0 = tm + C::kAcc, tm_acc1 = tm_acc0 + D;

  if (warp == 4) {  // ------------------------------------------------------------------ loads
    if ((threadIdx.x & 31) == 0 && iters > 0 && x.wait_cycles > 0) {
      mbar_arrive_expect_tx(bar_static, C::kStatic * C::kStaticBytes);
      for (int c = 0; c < D / 64; ++c) {
        tma_load3(sm_a0 + c * 16384, &map_a0, c * 64, head, (int)row0, bar_static);
        if (C::kStatic == 2) tma_load3(sm_a1 + c * 16384, &map_a1, c * 64, head, (int)row0, bar_static);
      }
      for (int it = 0; it < iters; ++it) {
        const int s = it % ST, col = __ldg(x.t.col + (M == kFwd ? t1 - 1 - it : t0 + it % nt)) * kTileCols;
        const uint32_t parity = ((it / ST) & 1) ^ 1;
        const int hx = M == kDkv ? head * x.a.group + it / nt : head / x.a.group;
        if (!wait(bar_x0_free + 8 * s, parity, dead, x, 1)) break;
        mbar_arrive_expect_tx(bar_x0_full + 8 * s, C::kStreamBytes);
        for (int c = 0; c < D / 64; ++c)
          tma_load3(sm_x0 + s * C::kStreamBytes + c * 8192, &map_x0, c * 64, hx, col, bar_x0_full + 8 * s);
        if (!wait(bar_x1_free + 8 * s, parity, dead, x, 2)) break;
        mbar_arrive_expect_tx(bar_x1_full + 8 * s, C::kStreamBytes);
        for (int c = 0; c < D / 64; ++c)
          tma_load3(sm_x1 + s * C::kStreamBytes + c * 8192, &map_x1, c * 64, hx, col, bar_x1_full + 8 * s);
      }
    }
    __syncwarp();
  } else if (warp == 5) {  // ----------------------------------------------------------- products
    if ((threadIdx.x & 31) == 0 && iters > 0) {
      constexpr uint32_t id_first = mma_desc(kBf16, 128, 64, false), id_second = mma_desc(kBf16, 128, D, true);
      // scores of iteration it
      auto first = [&](int it) {
        const int s = it % ST, b = it % NB;
        const uint32_t parity = (it / ST) & 1;
        if (!wait(bar_x0_full + 8 * s, parity, dead, x, 3)) return false;
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t half = k / 4, off = (k % 4) * 32;
          mma_ss(tm_s + b * 64, desc_k_major(sm_a0 + half * 16384 + off),
                 desc_k_major(sm_x0 + s * C::kStreamBytes + half * 8192 + off), id_first, k > 0);
        }
        if (M == kFwd) mma_commit(bar_x0_free + 8 * s);  // K is not needed again
        if (M != kFwd) {
          if (!wait(bar_x1_full + 8 * s, parity, dead, x, 4)) return false;
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t half = k / 4, off = (k % 4) * 32;
            mma_ss(tm_r + b * 64, desc_k_major(sm_a1 + half * 16384 + off),
                   desc_k_major(sm_x1 + s * C::kStreamBytes + half * 8192 + off), id_first, k > 0);
          }
          if (M == kDq) mma_commit(bar_x1_free + 8 * s);  // nor is V
        }
        mma_commit(bar_scores + 8 * b);
        return true;
      };
      auto second = [&](int it) {
        const int s = it % ST, b = it % NB;
        if (!wait(bar_weights + 8 * b, (it / NB) & 1, dead, x, 5)) return false;
        if (M == kFwd && !wait(bar_x1_full + 8 * s, (it / ST) & 1, dead, x, 6)) return false;
        tc_fence_after();
        const uint32_t x0 = sm_x0 + s * C::kStreamBytes, x1 = sm_x1 + s * C::kStreamBytes;
        // 16 streamed rows each: 8 columns of weights, 2048 bytes of the stream's image
        if (M == kFwd) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {  // high parts in the first 32 columns, low parts in the others
            const uint64_t v = desc_mn_major(x1 + k * 2048, 8192);
            mma_ts(tm_acc0, tm_s + b * 64 + k * 8, v, id_second, it > 0 || k > 0);
            mma_ts(tm_acc0, tm_s + b * 64 + 32 + k * 8, v, id_second, true);
          }
        } else {
          // each half of a score tile (32 columns) holds: of S the weights (dq: p c) and the score gradients' low parts, of R the score
          // gradients and the weights' low parts (dk, dv)
          const uint32_t grads = M == kDq ? tm_acc0 : tm_acc1;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t at = b * 64 + (k / 2) * 32 + (k % 2) * 8;
            const uint64_t d0 = desc_mn_major(x0 + k * 2048, 8192);
            if (M == kDkv) {
              const uint64_t d1 = desc_mn_major(x1 + k * 2048, 8192);
              mma_ts(tm_acc0, tm_s + at, d1, id_second, it > 0 || k > 0);
              mma_ts(tm_acc0, tm_r + at + 16, d1, id_second, true);
            } else {
              mma_ts(tm_acc1, tm_s + at, d0, id_second, it > 0 || k > 0);
            }
            mma_ts(grads, tm_r + at, d0, id_second, it > 0 || k > 0);
            mma_ts(grads, tm_s + at + 16, d0, id_second, true);
          }
        }
        if (M != kFwd) mma_commit(bar_x0_free + 8 * s);
        if (M != kDq) mma_commit(bar_x1_free + 8 * s);
        mma_commit(bar_acc + 8 * (it % kAccBars));
        return true;
      };
      bool ok = wait(bar_static, 0, dead, x, 7);
      tc_fence_after();
      ok = ok && first(0);
      for (int it = 0; ok && it < iters; ++it) {
        // with two score buffers the next scores are computed while this iteration's weights are
        if (NB == 2 && it + 1 < iters) ok = first(it + 1);
        ok = ok && second(it);
        if (NB == 1 && ok && it + 1 < iters) ok = first(it + 1);
      }
    }
    __syncwarp();
  } else {  // -------------------------------------------------------------------------- weights
    const int r = threadIdx.x;  // row of the tile
    const int64_t row = row0 + r;
    const int64_t n_rows = x.rows.d.n;
    const uint32_t lanes = (uint32_t)warp << 21;  // lane 32 * warp
    const float cap = x.a.cap, inv_cap2 = cap > 0.f ? 2.f * kLog2e / cap : 0.f;
    const float scale2 = x.a.scale * kLog2e;
    bool ok = true;
    const CapPoly cap_poly(x.a.scale, cap);
    // scores of base 2 are f s - slope2 |distance|, s: as the product left them, or capped
    const float f = cap > 0.f ? kLog2e : scale2;
    TileWalk walk(x.t, M == kFwd ? t1 - 1 : t0, M == kFwd ? -1 : 1, nt, iters, r);
    if constexpr (M == kFwd) {
      constexpr float kUp = kBf16 ? 0.f : 6.f;
      const float slope2 = x.a.slopes ? __ldg(x.a.slopes + head) * kLog2e : 0.f;
      float m = -INFINITY, l = 0.f;  // weights are exp2(u - m); m lies kUp below a maximum of the row
      for (int it = 0; it < iters; ++it) {
        const int b = it % NB;
        const int now_mask = walk.mask, now_col = walk.col;
        const uint64_t now_bits = walk.bits;
        if (!(ok = warp_wait(bar_scores + 8 * b, (it / NB) & 1, dead, x, 8))) break;
        tc_fence_after();
        float u[64];
        {
          uint32_t raw[2][32];
          tmem_ld32(tm_s + lanes + b * 64, raw[0]);
          tmem_ld32(tm_s + lanes + b * 64 + 32, raw[1]);
          walk.advance();  // while they come
          tmem_wait_ld();
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            float part[32];
#pragma unroll
            for (int c = 0; c < 32; ++c) part[c] = __uint_as_float(raw[half][c]);
            if (cap > 0.f) cap_row(part, cap_poly, cap, x.a.scale, inv_cap2);
#pragma unroll
            for (int c = 0; c < 32; ++c) u[half * 32 + c] = part[c];
          }
        }
        float fu = f;  // what is left to multiply with; a factor of 0 would make NaN of a masked -infinity below
        if (slope2 != 0.f || f <= 0.f) {
          // -slope2 |d0 - c| = -+ |slope2 c - slope2 d0|
          const float k0 = -slope2 * (float)(row + x.a.row_offset - (int64_t)now_col * kTileCols), sign = slope2 < 0.f ? 1.f : -1.f;
#pragma unroll
          for (int c = 0; c < 64; c += 2) {
            float x0, x1;
            fma2(x0, x1, (float)c, (float)(c + 1), slope2, slope2, k0, k0);
            x0 = sign * fabsf(x0), x1 = sign * fabsf(x1);
            fma2(x0, x1, u[c], u[c + 1], f, f);
            u[c] = x0, u[c + 1] = x1;
          }
          fu = 1.f;
        }
        if (now_mask != 0) {
          const uint32_t lo = (uint32_t)now_bits, hi = (uint32_t)(now_bits >> 32);
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            u[c] = lo & (1u << c) ? u[c] : -INFINITY;
            u[c + 32] = hi & (1u << c) ? u[c + 32] : -INFINITY;
          }
        }
        float top[4] = {u[0], u[1], u[2], u[3]};
#pragma unroll
        for (int c = 4; c < 60; c += 8)
#pragma unroll
          for (int k = 0; k < 4; ++k) top[k] = max3(top[k], u[c + k], u[c + 4 + k]);
#pragma unroll
        for (int k = 0; k < 4; ++k) top[k] = fmaxf(top[k], u[60 + k]);
        const float best = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        const float mt = best == -INFINITY ? best : fmaf(best, fu, -kUp);
        const bool grow = mt > m + kSlack || (m == -INFINITY && mt > m);
        if (__any_sync(0xffffffffu, grow)) {
          const float m2 = grow ? mt : m, less = grow ? exp2_approx(m - m2) : 1.f;
          m = m2;
          l *= less;
          if (it > 0) {  // the sum so far, once the previous product has been added to it
            if (!(ok = wait_acc(bar_acc, it - 1, dead, x, 9))) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              uint32_t w[32];
              tmem_ld32(tm_acc0 + lanes + c, w);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) w[i] = __float_as_uint(__uint_as_float(w[i]) * less);
              tmem_st32(tm_acc0 + lanes + c, w);
            }
          }
        }
        const float base = m == -INFINITY ? 0.f : -m;
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t hi[16], lo[16];
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            const int at = half * 32 + 2 * c, k = 2 * (c & 1);
            float p0, p1;
            fma2(p0, p1, u[at], u[at + 1], fu, fu, base, base);
            p0 = exp2_approx(p0), p1 = exp2_approx(p1);
            add2(sum[k], sum[k + 1], sum[k], sum[k + 1], p0, p1);
            split2<T>(p0, p1, hi[c], lo[c]);
          }
          tmem_st16(tm_s + lanes + b * 64 + half * 16, hi);
          tmem_st16(tm_s + lanes + b * 64 + 32 + half * 16, lo);
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(bar_weights + 8 * b);
      }
      if (ok && iters > 0) ok = wait_acc(bar_acc, iters - 1, dead, x, 10);
      tc_fence_after();
      const bool live = row < n_rows;
      if (ok && x.splits > 1) {
        const int64_t at = ((int64_t)blockIdx.y * n_rows + row) * x.a.heads + head;
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t w[32];
          if (iters > 0) {
            tmem_ld32(tm_acc0 + lanes + c, w);
            tmem_wait_ld();
          }
          if (live) {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              *reinterpret_cast<uint4 *>(x.part + at * D + c + i) =
                  iters > 0 ? make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]) : make_uint4(0, 0, 0, 0);
          }
        }
        if (live) x.part_ml[2 * at] = m, x.part_ml[2 * at + 1] = l;
      } else if (ok && iters > 0) {
        const bool fine = put_acc<T, D>(tm_acc0 + lanes, l == 0.f ? 0.f : 1.f / l, x.a.out, row, head, live);
        if (live && x.a.lse) x.a.lse[row * x.a.heads + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
        const uint32_t bad = __ballot_sync(0xffffffffu, live && !(fine && l == l));
        if (bad) redo<T, D, M>(x, row0 + 32 * warp, head, bad);
      } else if (ok && live) {  // no tile: no entry
        T *dst = (T *)x.a.out.p + row * x.a.out.row + (int64_t)head * x.a.out.head;
        for (int c = 0; c < D; c += 8) *reinterpret_cast<uint4 *>(dst + c) = make_uint4(0, 0, 0, 0);
        if (x.a.lse) x.a.lse[row * x.a.heads + head] = -INFINITY;
      } else if (!ok && live) {  // a wait gave up
        if (x.splits > 1) {
          x.part_ml[2 * (((int64_t)blockIdx.y * n_rows + row) * x.a.heads + head)] = NAN;
        } else {
          put_nan<T, D>(x.a.out, row, head);
          if (x.a.lse) x.a.lse[row * x.a.heads + head] = NAN;
        }
      }
    } else {
      const bool live = row < n_rows;
      float up = 1.f, dout_top = 0.f;
      if (!kBf16) {  // the largest |dout|: dq: of this thread's row, dk, dv: of the rows that are streamed
        uint32_t bits = 0;
        if (M == kDq) {
          if (live) bits = __ldg(x.a.dout_max + (int64_t)head * n_rows + row);
        } else {
          for (int i = r; i < iters * kTileCols; i += kWeightThreads) {
            const int it = i / kTileCols;
            const int64_t q = (int64_t)__ldg(x.t.col + t0 + it % nt) * kTileCols + i % kTileCols;
            if (q < x.a.n_queries) bits = max(bits, __ldg(x.a.dout_max + (int64_t)(head * x.a.group + it / nt) * x.a.n_queries + q));
          }
          bits = __reduce_max_sync(0xffffffffu, bits);
          if ((threadIdx.x & 31) == 0) tops[warp] = bits;
          asm volatile("bar.sync 1, 128;" ::: "memory");  // the weights' warps
          bits = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
        }
        dout_top = __uint_as_float(bits);
        up = dout_scale(bits);
      }
      const float down = x.a.scale / up;
      if (M == kDkv && !kBf16) up *= 0x1p-12f;  // the weights of dk, dv are 2^12 up themselves
      constexpr float kUp = kBf16 ? 0.f : 12.f;
      float most = 0.f, most_p = 0.f;  // fp16: the largest score gradient and weight as they are carried
      float lse2 = INFINITY, delta = 0.f, gap[2] = {0.f, 0.f};  // gap: sum of p (dp - delta), times up
      if (M == kDq && live) {
        lse2 = x.a.lse[row * x.a.heads + head] * kLog2e;
        if (lse2 == -INFINITY) lse2 = INFINITY;  // a row without entries: weights of 0
        delta = x.a.delta[row * x.a.heads + head];
      }
      // dk, dv: lse and delta of streamed row r of the tile (threads below 64), requested one iteration ahead
      float next_lse = 0.f, next_delta = 0.f;
      auto request_stats = [&](int col, int h) {
        const int64_t q = (int64_t)col * kTileCols + r;
        next_lse = -INFINITY, next_delta = 0.f;
        if (r < 64 && q < x.a.n_queries) {
          next_lse = x.a.lse[q * x.a.heads + h];
          next_delta = x.a.delta[q * x.a.heads + h];
        }
      };
      if (M == kDkv && iters > 0) request_stats(walk.col, head * x.a.group);
      for (int it = 0; it < iters; ++it) {
        const int b = it % NB;
        const int now_mask = walk.mask, now_col = walk.col;
        const uint64_t now_bits = walk.bits;
        walk.advance();
        const int h = M == kDkv ? head * x.a.group + it / nt : head;
        if (M == kDkv) {
          if (r < 64) {  // a row without entries (lse = -infinity): weights of 0
            row_lse[it & 1][r] = next_lse == -INFINITY ? -INFINITY : fmaf(next_lse, -kLog2e, kUp);
            row_delta[it & 1][r] = -next_delta;
          }
          mbar_arrive(bar_stats);
        }
        if (M == kDkv && it + 1 < iters) request_stats(walk.col, head * x.a.group + (it + 1) / nt);
        const float slope2 = x.a.slopes ? __ldg(x.a.slopes + h) * kLog2e : 0.f;
        // -slope2 |distance| = sign |slope2 c + k0|, c the column
        const int64_t col = (int64_t)now_col * kTileCols;
        const float k0 = slope2 * (M == kDq ? -(float)(row + x.a.row_offset - col) : (float)(col + x.a.row_offset - row));
        const float sign = slope2 < 0.f ? 1.f : -1.f;
        if (M == kDkv && !(ok = warp_wait(bar_stats, it & 1, dead, x, 13))) break;
        if (!(ok = warp_wait(bar_scores + 8 * b, (it / NB) & 1, dead, x, 11))) break;
        tc_fence_after();
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          float s[32], e[32], p[32];
          {
            uint32_t s_raw[32], e_raw[32];
            tmem_ld32(tm_s + lanes + b * 64 + half * 32, s_raw);
            tmem_ld32(tm_r + lanes + b * 64 + half * 32, e_raw);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 32; ++c) s[c] = __uint_as_float(s_raw[c]), e[c] = __uint_as_float(e_raw[c]);
          }
          if (cap > 0.f) cap_row(s, cap_poly, cap, x.a.scale, inv_cap2);
          const float *stat_lse = row_lse[it & 1] + half * 32, *stat_delta = row_delta[it & 1] + half * 32;
          // weights
          if (slope2 != 0.f) {
            const float kh = fmaf(slope2, (float)(half * 32), k0);
#pragma unroll
            for (int c = 0; c < 32; c += 2) {
              fma2(p[c], p[c + 1], (float)c, (float)(c + 1), slope2, slope2, kh, kh);
              p[c] = sign * fabsf(p[c]), p[c + 1] = sign * fabsf(p[c + 1]);
              fma2(p[c], p[c + 1], s[c], s[c + 1], f, f);
              if (M == kDkv) {
                const float2 l = *reinterpret_cast<const float2 *>(stat_lse + c);
                add2(p[c], p[c + 1], p[c], p[c + 1], l.x, l.y);
              } else {
                add2(p[c], p[c + 1], p[c], p[c + 1], -lse2, -lse2);
              }
              p[c] = exp2_approx(p[c]), p[c + 1] = exp2_approx(p[c + 1]);
            }
          } else {
#pragma unroll
            for (int c = 0; c < 32; c += 2) {
              float2 l = make_float2(-lse2, -lse2);
              if (M == kDkv) l = *reinterpret_cast<const float2 *>(stat_lse + c);
              fma2(p[c], p[c + 1], s[c], s[c + 1], f, f, l.x, l.y);
              p[c] = exp2_approx(p[c]), p[c + 1] = exp2_approx(p[c + 1]);
            }
          }
          if (now_mask != 0) {
            const uint32_t bit = half ? (uint32_t)(now_bits >> 32) : (uint32_t)now_bits;
#pragma unroll
            for (int c = 0; c < 32; ++c) p[c] = bit & (1u << c) ? p[c] : 0.f;
          }
          if (M == kDkv) {
            uint32_t w[16], lo[16];
#pragma unroll
            for (int c = 0; c < 32; c += 2) {
              if (!kBf16) most_p = max3(most_p, p[c], p[c + 1]);
              split2<T>(p[c], p[c + 1], w[c / 2], lo[c / 2]);
            }
            tmem_st16(tm_s + lanes + b * 64 + half * 32, w);
            tmem_st16(tm_r + lanes + b * 64 + half * 32 + 16, lo);
          }
          // score gradients: p (dp - delta) (1 - tanh^2), up to the scale
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            float d0 = -delta, d1 = -delta;
            if (M == kDkv) {
              const float2 l = *reinterpret_cast<const float2 *>(stat_delta + c);
              d0 = l.x, d1 = l.y;
            }
            add2(e[c], e[c + 1], e[c], e[c + 1], d0, d1);
            if (!kBf16) mul2(e[c], e[c + 1], e[c], e[c + 1], up, up);
            mul2(e[c], e[c + 1], e[c], e[c + 1], p[c], p[c + 1]);
            if (M == kDq) add2(gap[0], gap[1], gap[0], gap[1], e[c], e[c + 1]);
          }
          if (cap > 0.f) {
            const float inv = -1.f / (cap * cap);
#pragma unroll
            for (int c = 0; c < 32; c += 2) {
              float y0, y1, z0, z1;
              mul2(y0, y1, s[c], s[c + 1], s[c], s[c + 1]);
              fma2(z0, z1, y0, y1, inv, inv, 1.f, 1.f);
              mul2(e[c], e[c + 1], e[c], e[c + 1], z0, z1);
              if (M == kDq) mul2(p[c], p[c + 1], p[c], p[c + 1], z0, z1);
            }
          }
          if (M == kDq) {  // p c, for the correction of delta
            uint32_t w[16];
#pragma unroll
            for (int c = 0; c < 32; c += 2) {
              if (!kBf16) mul2(p[c], p[c + 1], p[c], p[c + 1], 4096.f, 4096.f);
              w[c / 2] = pack2<T>(p[c], p[c + 1]);
            }
            tmem_st16(tm_s + lanes + b * 64 + half * 32, w);
          }
          uint32_t v[16], lo[16];
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            if (!kBf16) most = max3(most, fabsf(e[c]), fabsf(e[c + 1]));
            split2<T>(e[c], e[c + 1], v[c / 2], lo[c / 2]);
          }
          tmem_st16(tm_r + lanes + b * 64 + half * 32, v);
          tmem_st16(tm_s + lanes + b * 64 + half * 32 + 16, lo);
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(bar_weights + 8 * b);
      }
      if (ok && iters > 0) ok = wait_acc(bar_acc, iters - 1, dead, x, 12);
      tc_fence_after();
      if (ok && iters > 0) {
        bool fine;
        if constexpr (M == kDq) {
          const float g = gap[0] + gap[1];
          fine = put_acc<T, D, true>(tm_acc0 + lanes, down, x.a.dq, row, head, live, tm_acc1 + lanes, -g * down * (kBf16 ? 1.f : 0x1p-12f));
          if (live) x.a.delta[row * x.a.heads + head] = delta + g / up;
        } else {
          fine = put_acc<T, D>(tm_acc0 + lanes, kBf16 ? 1.f : 0x1p-12f, x.a.dv, row, head, live);
          fine = put_acc<T, D>(tm_acc1 + lanes, down, x.a.dk, row, head, live) && fine;
        }
        // fp16 parts are within 2^-25, 2^-13 of the largest at kLeast; below, the row is done again (dv: where 2^-37 of dout, from each of
        // the streamed rows, could be seen in it)
        constexpr float kLeast = 0x1p-12f;
        if (most > 0.f && most < kLeast) fine = false;
        if (most_p > 0.f && most_p < kLeast && dout_top * ((float)iters * kTileCols) > 2048.f) fine = false;
        const uint32_t bad = __ballot_sync(0xffffffffu, live && !fine);
        if (bad) redo<T, D, M>(x, row0 + 32 * warp, head, bad);
      } else if (ok && live) {
        for (int c = 0; c < D; c += 8) {
          const uint4 zero = make_uint4(0, 0, 0, 0);
          if (M == kDq) {
            *reinterpret_cast<uint4 *>((T *)x.a.dq.p + row * x.a.dq.row + (int64_t)head * x.a.dq.head + c) = zero;
          } else {
            *reinterpret_cast<uint4 *>((T *)x.a.dk.p + row * x.a.dk.row + (int64_t)head * x.a.dk.head + c) = zero;
            *reinterpret_cast<uint4 *>((T *)x.a.dv.p + row * x.a.dv.row + (int64_t)head * x.a.dv.head + c) = zero;
          }
        }
      } else if (!ok && live) {  // a wait gave up
        put_nan<T, D>(M == kDq ? x.a.dq : x.a.dk, row, head);
        if (M == kDkv) put_nan<T, D>(x.a.dv, row, head);
        if (M == kDq) x.a.delta[row * x.a.heads + head] = NAN;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*dead)  // a wait gave up: copies and products in flight land before memory is given back
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
  tc_fence_after();
  if (iters > 0 && warp == 5) tmem_free(tm, C::kCols);
}

// Splits of the forward pass, joined: a warp per row and head.
template <class T, int D>
__global__ void __launch_bounds__(256) attn_tile_join_kernel(const __grid_constant__ TileArgs x) {
  const int64_t item = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 5, n = x.rows.d.n * (int64_t)x.a.heads;
  if (item >= n) return;
  const int64_t row = item / x.a.heads;
  const int h = (int)(item - row * x.a.heads), lane = threadIdx.x & 31;
  float m = -INFINITY, l = 0.f, acc[D / 32];
  bool lost = false;  // a piece's wait gave up
#pragma unroll
  for (int i = 0; i < D / 32; ++i) acc[i] = 0.f;
  for (int z = 0; z < x.splits; ++z) {
    const int64_t at = z * n + item;
    const float m2 = x.part_ml[2 * at], l2 = x.part_ml[2 * at + 1];
    if (m2 != m2) {
      lost = true;
      break;
    }
    const float top = fmaxf(m, m2), base = top == -INFINITY ? 0.f : top;
    const float f1 = exp2_approx(m - base), f2 = exp2_approx(m2 - base);
    l = l * f1 + l2 * f2;
    m = top;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] = acc[i] * f1 + x.part[at * D + lane + 32 * i] * f2;
  }
  const float inv = lost ? NAN : l == 0.f ? 0.f : 1.f / l;
  bool fine = l == l;
  T *dst = (T *)x.a.out.p + row * x.a.out.row + (int64_t)h * x.a.out.head;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    const float o = acc[i] * inv;
    fine &= isfinite(o);
    dst[lane + 32 * i] = T(o);
  }
  if (x.a.lse && lane == 0) x.a.lse[item] = lost ? NAN : l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
  if (!lost && __any_sync(0xffffffffu, !fine)) redo<T, D, kFwd>(x, row, h, 1u);
}

// delta0_i = dout_i . out_i of each row and head, a warp each (fp16: and the largest finite |dout|, [heads][rows]).
template <class T, int D>
__global__ void __launch_bounds__(256) attn_delta_kernel(int64_t rows, const AttnArgs a, uint32_t *dout_max) {
  const int64_t item = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 5;
  const int64_t row = item / a.heads;
  const int h = (int)(item - row * a.heads), lane = threadIdx.x & 31;
  if (row >= rows) return;
  const T *p = (const T *)a.dout.p + row * a.dout.row + h * a.dout.head, *y = (const T *)a.o.p + row * a.o.row + h * a.o.head;
  float s = 0.f, top = 0.f;
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
    float f[2], g[2];
    RowVec<T, 2>::widen(RowVec<T, 2>::ldg(p + 2 * (lane + 32 * i)), f);
    RowVec<T, 2>::widen(RowVec<T, 2>::ldg(y + 2 * (lane + 32 * i)), g);
    s = fmaf(f[0], g[0], fmaf(f[1], g[1], s));
    if (isfinite(f[0])) top = fmaxf(top, fabsf(f[0]));
    if (isfinite(f[1])) top = fmaxf(top, fabsf(f[1]));
  }
  s = group_sum<32>(s);
  if (lane == 0) a.delta[item] = s;
  if (std::is_same<T, __half>::value) {
    const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
    if (lane == 0) dout_max[h * rows + row] = bits;
  }
}

// ------------------------------------------------------------------------------------------------ launches

using EncodeTiledFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                   const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_tiled() {
  static EncodeTiledFn fn = [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      return (EncodeTiledFn) nullptr;
    }
    return (EncodeTiledFn)p;
  }();
  return fn;
}

// rows x heads x dim of a 16-bit type; boxes of 64 elements of one head, `box_rows` rows.
bool encode(CUtensorMap *map, const Heads &x, int64_t rows, int heads, int dim, bool bf16, int box_rows) {
  EncodeTiledFn fn = encode_tiled();
  if (!fn) return false;
  const cuuint64_t size[3] = {(cuuint64_t)dim, (cuuint64_t)heads, (cuuint64_t)rows};
  // the stride of an axis of length one is free
  const cuuint64_t stride[2] = {(cuuint64_t)(heads > 1 ? x.head : dim) * 2, (cuuint64_t)(rows > 1 ? x.row : (int64_t)dim * heads) * 2};
  const cuuint32_t box[3] = {64, 1, (cuuint32_t)box_rows}, step[3] = {1, 1, 1};
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, (void *)x.p, size, stride, box, step,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

TileView view(const PatternTiles &t) { return {t.ptr, t.col, t.mask, t.order, t.words}; }

int64_t up256(int64_t x) { return (x + 255) / 256 * 256; }

template <class T, int D, Mode M>
int launch(const dsp_pattern *p, TileArgs x, cudaStream_t s) {
  using C = Cfg<D, M>;
  constexpr bool bf16 = std::is_same<T, __nv_bfloat16>::value;
  const PatternTiles &t = M == kDkv ? p->tt : p->at;
  if (t.n == 0) return DSP_OK;
  const int kv_heads = x.a.heads / x.a.group;
  x.t = view(t);
  x.rows = {view(M == kDkv ? p->t : p->a)};
  x.n_heads = M == kDkv ? kv_heads : x.a.heads;
  x.err = p->d_err;
  x.wait_cycles = p->wait_cycles;
  const Heads q = x.a.q, k = x.a.k, v = x.a.v, o = M == kFwd ? q : x.a.dout;  // the forward has no second stationary operand
  const int64_t nq = p->rows, nk = p->cols;
  CUtensorMap a0, a1, x0, x1;
  bool ok;
  if (M == kDkv)
    ok = encode(&a0, k, nk, kv_heads, D, bf16, kTileRows) && encode(&a1, v, nk, kv_heads, D, bf16, kTileRows) &&
         encode(&x0, q, nq, x.a.heads, D, bf16, kTileCols) && encode(&x1, o, nq, x.a.heads, D, bf16, kTileCols);
  else
    ok = encode(&a0, q, nq, x.a.heads, D, bf16, kTileRows) && encode(&a1, o, nq, x.a.heads, D, bf16, kTileRows) &&
         encode(&x0, k, nk, kv_heads, D, bf16, kTileCols) && encode(&x1, v, nk, kv_heads, D, bf16, kTileCols);
  if (!ok) return fail(DSP_ERR_CUDA, "dsp_attn: a tensor map was refused");
  const cudaError_t e = cudaFuncSetAttribute((const void *)attn_tile_kernel<T, D, M>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  if (e != cudaSuccess) return fail(DSP_ERR_CUDA, "dsp_attn: %s", cudaGetErrorString(e));
  attn_tile_kernel<T, D, M><<<dim3((unsigned)((int64_t)t.n * x.n_heads), (unsigned)std::max(1, x.splits)), kThreads, C::kSmem, s>>>(
      a0, a1, x0, x1, x);
  const cudaError_t l = cudaGetLastError();
  return l == cudaSuccess ? DSP_OK : fail(DSP_ERR_CUDA, "dsp_attn: %s", cudaGetErrorString(l));
}

template <class T, int D>
int forward(const dsp_pattern *p, TileArgs x, cudaStream_t s) {
  int rc = launch<T, D, kFwd>(p, x, s);
  if (rc || x.splits == 1) return rc;
  x.rows = {view(p->a)};
  attn_tile_join_kernel<T, D><<<(unsigned)((p->rows * x.a.heads + 7) / 8), 256, 0, s>>>(x);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? DSP_OK : fail(DSP_ERR_CUDA, "dsp_attn: %s", cudaGetErrorString(e));
}

template <class T, int D>
int gradients(const dsp_pattern *p, TileArgs x, uint32_t *dout_max, cudaStream_t s) {
  attn_delta_kernel<T, D><<<(unsigned)((p->rows * x.a.heads + 7) / 8), 256, 0, s>>>(p->rows, x.a, dout_max);
  x.a.dout_max = dout_max;
  const int rc = launch<T, D, kDq>(p, x, s);
  return rc ? rc : launch<T, D, kDkv>(p, x, s);
}

// Pieces that a row tile's list is cut into: enough CTAs for two on every SM where there are few row tiles and heads, each
// with four tiles at least.
int splits_of(const dsp_pattern *p, int heads) {
  const int64_t ctas = (int64_t)p->at.n * heads;
  return (int)std::max<int64_t>(1, std::min<int64_t>({2ll * p->sms / std::max<int64_t>(ctas, 1), p->at.max_tiles / 4, 64}));
}

}  // namespace

bool tile_form(const dsp_pattern *p, const dsp_attn_desc *d) {
  return p->tiled && p->rows > 0 && p->cols > 0 && (d->dtype == DSP_BF16 || d->dtype == DSP_F16) && (d->dim == 64 || d->dim == 128) &&
         (p->rows == 1 || d->q_row > 0) && (d->heads == 1 || d->q_head > 0) &&
         (p->cols == 1 || (d->k_row > 0 && d->v_row > 0)) && (d->kv_heads == 1 || (d->k_head > 0 && d->v_head > 0));
}

int64_t tile_forward_bytes(const dsp_pattern *p, const dsp_attn_desc *d) {
  const int s = splits_of(p, d->heads);
  return s == 1 ? 0 : up256(4 * s * p->rows * d->heads * d->dim) + up256(8 * s * p->rows * d->heads);
}

int tile_forward(const dsp_pattern *p, const AttnArgs &a, int dtype, void *ws, cudaStream_t s) {
  TileArgs x = {};
  x.a = a;
  x.splits = splits_of(p, a.heads);
  x.part = (float *)ws;
  x.part_ml = (float *)((char *)ws + up256(4 * x.splits * p->rows * a.heads * a.dim));
  if (dtype == DSP_BF16) return a.dim == 64 ? forward<__nv_bfloat16, 64>(p, x, s) : forward<__nv_bfloat16, 128>(p, x, s);
  return a.dim == 64 ? forward<__half, 64>(p, x, s) : forward<__half, 128>(p, x, s);
}

int64_t tile_grad_bytes(const dsp_pattern *p, const dsp_attn_desc *d) {
  return up256(4 * p->rows * d->heads) * (d->dtype == DSP_F16 ? 2 : 1);  // delta, and the largest |dout| of each row
}

int tile_gradients(const dsp_pattern *p, const AttnArgs &a, int dtype, void *ws, cudaStream_t s) {
  TileArgs x = {};
  x.a = a;
  x.a.delta = (float *)ws;
  x.a.n_queries = p->rows;
  x.splits = 1;
  uint32_t *dout_max = (uint32_t *)((char *)ws + up256(4 * p->rows * a.heads));
  if (dtype == DSP_BF16) return a.dim == 64 ? gradients<__nv_bfloat16, 64>(p, x, dout_max, s) : gradients<__nv_bfloat16, 128>(p, x, dout_max, s);
  return a.dim == 64 ? gradients<__half, 64>(p, x, dout_max, s) : gradients<__half, 128>(p, x, dout_max, s);
}

}  // namespace dsp
