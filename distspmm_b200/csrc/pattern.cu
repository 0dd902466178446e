// pattern.cu — dsp_pattern: a CSR matrix prepared once for the fused product (act.cu) and for attention (attn.cu).
#include <stdlib.h>
#include <string.h>

#include <algorithm>
#include <new>

#include "mbar.cuh"
#include "pattern.h"

namespace dsp {

// Units of a chunk: enough chunks for some 32 warps on every SM, 64 to 512 units each.
static int32_t chunk_units(int64_t units) {
  int64_t l = (units + 148 * 32 - 1) / (148 * 32);
  l = (l + 31) / 32 * 32;
  return (int32_t)std::min<int64_t>(kMaxUnits, std::max<int64_t>(64, l));
}

void pattern_chunks(int32_t n, HostDir *d) {
  const int64_t nnz = d->ptr[n], units = row_start(n, nnz);
  d->L = chunk_units(units);
  d->n_chunks = (int32_t)((units + d->L - 1) / d->L);
  d->row_of.resize(nnz);
  d->row0.resize(d->n_chunks + 1);
  d->nz0.resize(d->n_chunks + 1);
  parallel_for(n, [&](int64_t b, int64_t e) {
    for (int64_t r = b; r < e; ++r)
      for (int32_t p = d->ptr[r]; p < d->ptr[r + 1]; ++p) d->row_of[p] = (int32_t)r;
  });
  parallel_for(d->n_chunks + 1, [&](int64_t b, int64_t e) {
    for (int64_t c = b; c < e; ++c) {
      const int64_t x = std::min<int64_t>(c * d->L, units);
      int64_t lo = 0, hi = n;  // the first row whose end is at x or behind
      while (lo < hi) {
        const int64_t m = (lo + hi) / 2;
        if (row_start(m, d->ptr[m + 1]) < x) lo = m + 1;
        else hi = m;
      }
      d->row0[c] = (int32_t)lo;
      d->nz0[c] = (int32_t)std::max<int64_t>(x - row_start(lo, 0), d->ptr[lo]);  // x may lie inside the end of row lo - 1
    }
  });
  d->split_row.clear();
  std::vector<int32_t> few;
  for (int32_t r = 0; r < n; ++r) {
    const int64_t cuts = row_start(r, d->ptr[r + 1]) / d->L - row_start(r, d->ptr[r]) / d->L;
    if (cuts > kLongSlots) d->split_row.push_back(r);
    else if (cuts > 0) few.push_back(r);
  }
  d->n_long = (int32_t)d->split_row.size();
  d->split_row.insert(d->split_row.end(), few.begin(), few.end());
}

bool build_tiles(int32_t n, int32_t n_cols, const HostDir &d, bool always, HostTiles *out) {
  const int32_t nt = (n + kTileRows - 1) / kTileRows, nc = (n_cols + kTileCols - 1) / kTileCols;
  std::vector<int32_t> ptr(nt + 1, 0);
  std::atomic<bool> no_memory{false};
  // tiles of each row tile: stamp[c] = the last row tile that touched column tile c
  parallel_for(nt, [&](int64_t b, int64_t e) {
    try {
      std::vector<int32_t> stamp(nc, -1);
      for (int64_t t = b; t < e; ++t) {
        int32_t k = 0;
        const int32_t hi = d.ptr[std::min<int64_t>(n, (t + 1) * kTileRows)];
        for (int32_t p = d.ptr[t * kTileRows]; p < hi; ++p) {
          int32_t &s = stamp[d.cols[p] / kTileCols];
          k += s != (int32_t)t;
          s = (int32_t)t;
        }
        ptr[t + 1] = k;
      }
    } catch (const std::bad_alloc &) {
      no_memory.store(true);
    }
  }, 8);
  if (no_memory.load()) throw std::bad_alloc();
  int64_t count = 0;
  for (int32_t t = 0; t < nt; ++t) count += ptr[t + 1];
  if (!always && (d.ptr[n] == 0 || (int64_t)d.ptr[n] < count * kTileFill)) return false;
  HostTiles &o = *out;
  for (int32_t t = 0; t < nt; ++t) {
    o.max_tiles = std::max(o.max_tiles, ptr[t + 1]);
    ptr[t + 1] += ptr[t];
  }
  o.ptr = std::move(ptr);
  o.col.resize(count);
  o.mask.resize(count);
  std::vector<uint64_t> words((size_t)count * kTileRows, 0);
  parallel_for(nt, [&](int64_t b, int64_t e) {
    try {
      std::vector<int32_t> at(nc, -1);
      for (int64_t t = b; t < e; ++t) {
        const int32_t r0 = (int32_t)(t * kTileRows), r1 = std::min(n, r0 + kTileRows), first = o.ptr[t], last = o.ptr[t + 1];
        int32_t k = first;
        for (int32_t p = d.ptr[r0]; p < d.ptr[r1]; ++p) {
          const int32_t c = d.cols[p] / kTileCols;
          if (at[c] < 0) at[c] = 0, o.col[k++] = c;
        }
        std::sort(o.col.begin() + first, o.col.begin() + last);
        for (k = first; k < last; ++k) at[o.col[k]] = k;
        for (int32_t r = r0; r < r1; ++r)
          for (int32_t p = d.ptr[r]; p < d.ptr[r + 1]; ++p)
            words[(size_t)at[d.cols[p] / kTileCols] * kTileRows + (r - r0)] |= 1ull << (d.cols[p] % kTileCols);
        for (k = first; k < last; ++k) at[o.col[k]] = -1;
      }
    } catch (const std::bad_alloc &) {
      no_memory.store(true);
    }
  }, 8);
  if (no_memory.load()) throw std::bad_alloc();
  int32_t masks = 0;  // words of tile k < masks hold a kept mask
  for (int64_t k = 0; k < count; ++k) {
    const uint64_t *w = &words[(size_t)k * kTileRows];
    bool full = true;
    for (int r = 0; r < kTileRows; ++r) full &= w[r] == ~0ull;
    o.mask[k] = full ? 0 : masks + 1;
    if (!full) {
      if (masks != k) std::copy(w, w + kTileRows, &words[(size_t)masks * kTileRows]);
      ++masks;
    }
  }
  words.resize((size_t)masks * kTileRows);
  o.words.assign(kTileRows, ~0ull);  // number 0: the full tile
  o.words.insert(o.words.end(), words.begin(), words.end());
  o.order.resize(nt);
  for (int32_t t = 0; t < nt; ++t) o.order[t] = t;
  std::stable_sort(o.order.begin(), o.order.end(),
                   [&](int32_t x, int32_t y) { return o.ptr[x + 1] - o.ptr[x] > o.ptr[y + 1] - o.ptr[y]; });
  return true;
}

namespace {

template <class V>
int put(dsp_pattern *p, const std::vector<V> &h, V **out) {
  *out = nullptr;
  const size_t bytes = std::max<size_t>(h.size(), 1) * sizeof(V);
  void *d = nullptr;
  cudaError_t e = cudaMalloc(&d, bytes);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(DSP_ERR_NOMEM, "dsp_pattern_create: %zu bytes: %s", bytes, cudaGetErrorString(e));
  }
  p->allocs.push_back(d);
  p->device_bytes += (int64_t)bytes;
  if (!h.empty() && (e = cudaMemcpy(d, h.data(), h.size() * sizeof(V), cudaMemcpyHostToDevice)) != cudaSuccess)
    return fail(DSP_ERR_CUDA, "dsp_pattern_create: %s", cudaGetErrorString(e));
  *out = (V *)d;
  return DSP_OK;
}

int put_dir(dsp_pattern *p, int32_t n, const HostDir &h, PatternDir *d) {
  d->n = n;
  d->L = h.L;
  d->n_chunks = h.n_chunks;
  d->n_split = (int32_t)h.split_row.size();
  d->n_long = h.n_long;
  int rc;
  if ((rc = put(p, h.ptr, &d->ptr)) || (rc = put(p, h.cols, &d->cols)) ||
      (rc = put(p, h.row0, &d->row0)) || (rc = put(p, h.nz0, &d->nz0)) || (rc = put(p, h.split_row, &d->split_row)))
    return rc;
  if (!h.perm.empty() && (rc = put(p, h.perm, &d->perm))) return rc;
  return DSP_OK;
}

int put_tiles(dsp_pattern *p, const HostTiles &h, PatternTiles *t) {
  t->n = (int32_t)h.order.size();
  t->max_tiles = h.max_tiles;
  t->count = (int64_t)h.col.size();
  int rc;
  if ((rc = put(p, h.ptr, &t->ptr)) || (rc = put(p, h.col, &t->col)) || (rc = put(p, h.mask, &t->mask)) ||
      (rc = put(p, h.order, &t->order)) || (rc = put(p, h.words, &t->words)))
    return rc;
  return DSP_OK;
}

// A row that lists a column twice, or -1.
int64_t repeated_column(const dsp_csr *a) {
  std::atomic<int64_t> bad{-1};
  std::atomic<bool> no_memory{false};
  parallel_for(a->num_rows, [&](int64_t b, int64_t e) {
    for (int64_t r = b; r < e && bad.load() < 0; ++r) {
      const int64_t *x = a->indices + a->indptr[r], *y = a->indices + a->indptr[r + 1];
      bool rising = true;
      for (const int64_t *q = x; q + 1 < y; ++q) rising &= q[0] < q[1];
      if (rising) continue;
      try {  // an exception must not leave the worker thread
        std::vector<int64_t> s(x, y);
        std::sort(s.begin(), s.end());
        if (std::adjacent_find(s.begin(), s.end()) != s.end()) bad.store(r);
      } catch (const std::bad_alloc &) {
        no_memory.store(true);
      }
    }
  }, 1024);
  if (no_memory.load()) throw std::bad_alloc();
  return bad.load();
}

int create(int device, const dsp_csr *a, int flags, dsp_pattern *p) {
  const int32_t M = (int32_t)a->num_rows, K = (int32_t)a->num_cols;
  p->device = device;
  p->flags = flags;
  p->rows = M;
  p->cols = K;
  p->nnz = a->nnz;
  p->wait_cycles = kMbarWaitCycles;
  if (const char *limit = getenv("DSP_ATTN_WAIT_CYCLES")) {  // of the tile kernels' waits; 0: they start no copies and so run out at once (tests)
    char *end = nullptr;
    const long long n = strtoll(limit, &end, 10);
    if (end != limit && *end == 0 && n >= 0) p->wait_cycles = n;
  }
  HostDir h;
  h.ptr.resize(M + 1);
  h.cols.resize(a->nnz);
  for (int32_t r = 0; r <= M; ++r) h.ptr[r] = (int32_t)a->indptr[r];
  for (int32_t r = 0; r < M; ++r) p->max_row_len = std::max<int64_t>(p->max_row_len, h.ptr[r + 1] - h.ptr[r]);
  parallel_for(a->nnz, [&](int64_t b, int64_t e) {
    for (int64_t i = b; i < e; ++i) h.cols[i] = (int32_t)a->indices[i];
  });
  pattern_chunks(M, &h);
  HostDir t;
  if (flags & DSP_PATTERN_GRAD) {  // counting sort by column: entries of a column in row order
    t.ptr.assign(K + 1, 0);
    t.cols.resize(a->nnz);
    t.perm.resize(a->nnz);
    for (int64_t i = 0; i < a->nnz; ++i) ++t.ptr[h.cols[i] + 1];
    for (int32_t c = 0; c < K; ++c) t.ptr[c + 1] += t.ptr[c];
    std::vector<int32_t> at(t.ptr.begin(), t.ptr.end() - 1);
    for (int64_t i = 0; i < a->nnz; ++i) {
      const int32_t q = at[h.cols[i]]++;
      t.cols[q] = h.row_of[i];
      t.perm[q] = (int32_t)i;
    }
    pattern_chunks(K, &t);
  }
  HostTiles ta, tt;
  if ((flags & DSP_PATTERN_ATTENTION) && !(flags & DSP_PATTERN_ROWS)) {
    p->tiled = build_tiles(M, K, h, flags & DSP_PATTERN_TILES, &ta);
    if (p->tiled && (flags & DSP_PATTERN_GRAD)) build_tiles(K, M, t, true, &tt);
  }
  DeviceGuard g(device);
  if (g.err != cudaSuccess) return fail(DSP_ERR_CUDA, "cudaSetDevice(%d): %s", device, cudaGetErrorString(g.err));
  cudaError_t e = cudaDeviceGetAttribute(&p->sms, cudaDevAttrMultiProcessorCount, device);
  if (e != cudaSuccess) return fail(DSP_ERR_CUDA, "dsp_pattern_create: %s", cudaGetErrorString(e));
  int rc = put_dir(p, M, h, &p->a);
  if (!rc && (flags & DSP_PATTERN_GRAD)) rc = put_dir(p, K, t, &p->t);
  if (!rc && p->tiled) rc = put_tiles(p, ta, &p->at);
  if (!rc && p->tiled && (flags & DSP_PATTERN_GRAD)) rc = put_tiles(p, tt, &p->tt);
  if (!rc) rc = put(p, std::vector<int>(1, 0), &p->d_err);
  return rc;
}

}  // namespace
}  // namespace dsp

using namespace dsp;

extern "C" int dsp_pattern_create(int device, const dsp_csr *a, int flags, dsp_pattern **out) {
  DSP_TRY_ARG(a && out && a->indptr, "dsp_pattern_create: null argument");
  *out = nullptr;
  const int forms = DSP_PATTERN_TILES | DSP_PATTERN_ROWS;
  DSP_TRY_ARG((flags & ~(DSP_PATTERN_GRAD | DSP_PATTERN_ATTENTION | forms)) == 0 && (flags & forms) != forms,
              "dsp_pattern_create: flags %d", flags);
  DSP_TRY_ARG(a->num_rows >= 0 && a->num_cols >= 0 && a->nnz >= 0, "dsp_pattern_create: negative size");
  DSP_TRY_ARG(a->nnz == 0 || a->indices, "dsp_pattern_create: null indices");
  // kernels step past an entry's place by up to 32 in 32 bits
  if (a->num_rows >= INT32_MAX || a->num_cols >= INT32_MAX || a->nnz > INT32_MAX - 64)
    return fail(DSP_ERR_UNSUPPORTED, "dsp_pattern_create: %lld x %lld with %lld entries: ids are 32-bit",
                (long long)a->num_rows, (long long)a->num_cols, (long long)a->nnz);
  dsp_pattern *p = nullptr;
  try {
    int rc = dsp_csr_validate(a);
    if (rc) return rc;
    if (flags & DSP_PATTERN_ATTENTION) {
      const int64_t r = repeated_column(a);
      if (r >= 0)
        return fail(DSP_ERR_FORMAT, "dsp_pattern_create: row %lld lists a column twice (attention needs distinct keys)",
                    (long long)r);
    }
    p = new dsp_pattern();
    rc = create(device, a, flags, p);
    if (rc) {
      dsp_pattern_destroy(p);
      return rc;
    }
  } catch (const std::bad_alloc &) {
    dsp_pattern_destroy(p);
    return fail(DSP_ERR_NOMEM, "dsp_pattern_create: out of host memory");
  } catch (const std::exception &e) {
    dsp_pattern_destroy(p);
    return fail(DSP_ERR_STATE, "dsp_pattern_create: %s", e.what());
  }
  *out = p;
  return DSP_OK;
}

extern "C" void dsp_pattern_destroy(dsp_pattern *p) {
  if (!p) return;
  {
    DeviceGuard g(p->device);
    for (void *d : p->allocs) cudaFree(d);
  }
  delete p;
}

extern "C" int dsp_pattern_check_error(dsp_pattern *p) {
  DSP_TRY_ARG(p, "dsp_pattern_check_error: null pattern");
  DeviceGuard g(p->device);
  int flag = 0;
  cudaError_t e = g.err;
  if (e == cudaSuccess) e = cudaMemcpy(&flag, p->d_err, sizeof flag, cudaMemcpyDeviceToHost);
  if (e == cudaSuccess && flag != 0) e = cudaMemset(p->d_err, 0, sizeof(int));
  if (e != cudaSuccess) return fail(DSP_ERR_CUDA, "dsp_pattern_check_error: %s", cudaGetErrorString(e));
  if (flag == 0) return DSP_OK;
  return fail(DSP_ERR_TIMEOUT, "attention: a bounded wait gave up (code %d); results are incomplete", flag);
}

extern "C" int dsp_pattern_info_get(const dsp_pattern *p, dsp_pattern_info *info) {
  DSP_TRY_ARG(p && info, "dsp_pattern_info_get: null argument");
  memset(info, 0, sizeof *info);
  info->rows = p->rows;
  info->cols = p->cols;
  info->nnz = p->nnz;
  info->flags = p->flags;
  info->chunk_units = p->a.L;
  info->chunks = p->a.n_chunks;
  info->split_rows = p->a.n_split;
  info->max_row_len = p->max_row_len;
  info->tiles = p->tiled ? p->at.count : 0;
  info->device_bytes = p->device_bytes;
  return DSP_OK;
}
