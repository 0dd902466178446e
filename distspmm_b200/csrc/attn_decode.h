// attn_decode.h — single query tokens over listed cache rows (attn_decode.cu), and the view of such lists.
#pragma once
#include "attn.h"

namespace dsp {

// Rows listed by a CSR in device memory that nothing has validated: every value read from it is bounded before it is used,
// so that no list can make the kernel leave its operands.
struct ListRows {
  using Index = int64_t;
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
};

// Whether attn_decode.cu's kernel takes a call (else the gather kernel of attn.cu).
bool decode_on_tensor_cores(int dtype, int dim);
// Units of a chunk for a list of nnz entries.
int32_t decode_units(int64_t rows, int64_t nnz, int heads, int kv_heads, bool tensor);
int decode_tensor(const ListRows &d, const AttnArgs &a, int dtype, cudaStream_t s);
// Rows cut across chunks, after either kernel.
int decode_join(const ListRows &d, const AttnArgs &a, int dtype, cudaStream_t s);

}  // namespace dsp
