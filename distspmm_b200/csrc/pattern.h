// pattern.h — the device-resident CSR pattern shared by the fused product and the attention kernels.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <vector>

#include "internal.h"

namespace dsp {

// One orientation of the pattern (A, or A transposed), with its balanced work chunks.
//
// The work of one orientation is a path of units: the entries of row 0 (a unit each), the end of row 0 (kRowUnits units: it
// costs an epilogue, not a gathered row), the entries of row 1, its end, ... (merge path). Chunk c holds what begins in the
// units [c L, (c + 1) L): the row ends row0[c] .. row0[c+1] - 1 and the entries nz0[c] .. nz0[c+1] - 1, so rows of any length
// and runs of rows without entries are spread evenly. Row r begins at row_start(r, ptr[r]) and its end is at
// row_start(r, ptr[r+1]); it is cut when these lie in different chunks, and then leaves one partial in each of them: in slot
// 2c + 1 of the chunk it starts in, in slot 2c of every later one. split_row lists the cut rows, those of more than
// kLongSlots partials first (n_long of them).
constexpr int kRowUnits = 8;
constexpr int kLongSlots = 12;
constexpr int kMaxUnits = 512;  // of a chunk
DSP_HD int64_t row_start(int64_t r, int64_t p) { return r * kRowUnits + p; }

struct PatternDir {
  int32_t n = 0;          // rows of this orientation
  int32_t n_chunks = 0;
  int32_t L = 0;          // units of a chunk
  int32_t n_split = 0, n_long = 0;
  int32_t *ptr = nullptr;        // [n + 1]
  int32_t *cols = nullptr;       // [nnz]
  int32_t *perm = nullptr;       // [nnz] place of the entry in A's own order (transposed orientation only)
  int32_t *row0 = nullptr;       // [n_chunks + 1]
  int32_t *nz0 = nullptr;        // [n_chunks + 1]
  int32_t *split_row = nullptr;  // [n_split]
};

// Kernel-side view (passed by value).
struct DirView {
  int32_t n, n_chunks, L, n_split, n_long;
  const int32_t *ptr, *cols, *perm, *row0, *nz0, *split_row;
};

inline DirView view(const PatternDir &d) {
  return {d.n, d.n_chunks, d.L, d.n_split, d.n_long, d.ptr, d.cols, d.perm, d.row0, d.nz0, d.split_row};
}

// Blocks of 8 warps that join the cut rows: a block for each long one, a warp for each other.
inline int64_t join_blocks(const DirView &d) { return d.n_long + (d.n_split - d.n_long + 7) / 8; }

// Host form of one orientation.
struct HostDir {
  std::vector<int32_t> ptr, row_of, cols, perm, row0, nz0, split_row;
  int32_t L = 0, n_chunks = 0, n_long = 0;
};

// Fill row_of (which stays on the host), chunks and cut rows from ptr.
void pattern_chunks(int32_t n, HostDir *d);

// The tile form: tiles of kTileRows x kTileCols entries that hold at least one entry, by row tiles, columns rising. A tile
// with gaps has a 64-bit word of presence bits for each of its rows; the full ones share mask 0, all ones.
constexpr int kTileRows = 128, kTileCols = 64;
struct PatternTiles {
  int32_t n = 0, max_tiles = 0;  // row tiles; tiles of the longest one
  int64_t count = 0;
  int32_t *ptr = nullptr;     // [n + 1]
  int32_t *col = nullptr;     // [count] column tile
  int32_t *mask = nullptr;    // [count] its words at 128 * mask; 0: full
  int32_t *order = nullptr;   // [n] row tiles, longest first
  uint64_t *words = nullptr;
};
struct HostTiles {
  std::vector<int32_t> ptr, col, mask, order;
  std::vector<uint64_t> words;
  int32_t max_tiles = 0;
};
// Entries per tile, on average over the matrix, from which the tile form is built and used. A tile costs the same however many entries it
// has, a row's entry by itself. Measured with 8 heads of 64, bf16, training step (forward), tiles / rows in us, by entries a tile:
//   uniform rows     120: 448 / 488 (103 / 125)   160: 201 / 183 (47 / 49)   200: 448 / 670 (102 / 163)   240: 201 / 253 (47 / 68)
//   R-MAT 11, 10, 9   92: 203 / 146 (47 / 43)     165: 111 / 93 (27 / 27)    300: 66 / 58 (17 / 19)
//   a window of 8    345: 47 / 119 (12 / 35)
// One threshold cannot be right for all: skewed graphs leave many thin tiles beside full ones. 180 costs the two it misses (uniform 120,
// R-MAT 9) 9 and 14 %.
constexpr int64_t kTileFill = 180;
// False (and out untouched) where tiles would hold fewer than kTileFill entries on average.
bool build_tiles(int32_t n, int32_t n_cols, const HostDir &d, bool always, HostTiles *out);

// Makes `device` current where it is not, and restores the caller's on scope exit.
struct DeviceGuard {
  int before = -1;
  cudaError_t err;
  explicit DeviceGuard(int device) {
    int now = -1;
    err = cudaGetDevice(&now);
    if (err == cudaSuccess && now != device && (err = cudaSetDevice(device)) == cudaSuccess) before = now;
  }
  ~DeviceGuard() {
    if (before >= 0) cudaSetDevice(before);
  }
};

}  // namespace dsp

struct dsp_pattern {
  int device = 0;
  int sms = 0;
  int flags = 0;
  int64_t rows = 0, cols = 0, nnz = 0, max_row_len = 0;
  dsp::PatternDir a;  // A
  dsp::PatternDir t;  // A transposed (DSP_PATTERN_GRAD)
  bool tiled = false;  // the tile form of a (and of t) exists
  dsp::PatternTiles at, tt;
  int *d_err = nullptr;  // set by a kernel whose bounded wait gave up
  long long wait_cycles = 0;  // their limit
  int64_t device_bytes = 0;
  std::vector<void *> allocs;
};
