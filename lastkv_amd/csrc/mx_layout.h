// MX4 weight layout: 16 rows (output features) x 512 columns form one 4352-byte unit, units ordered
// [row tile][column unit]; in a unit, 4 tiles of 128 columns of 1024 bytes each, lane l = (row r = l & 15, g = l >> 4)
// holding 16 bytes at l * 16: the 32 codes of columns 32 g .. 32 g + 31 of the tile (the even one low), one scale
// block; then 64 words, word l byte t the scale of lane l's block of tile t.  So a wave's operand of a 16 x 128 tile
// is one contiguous 1 KiB load, both for the scaled 8-bit matrix instruction (lane (r, g) takes columns 32 g ..)
// and for bf16 ones (step j takes column 32 g + 8 j + i of every g: any order serves that both operands share).
// Rows and columns past the matrix hold zeros.
// (Plain arithmetic: also compiled for the host alone.)
#pragma once
#include <stdint.h>

#ifdef __HIPCC__
#define LKV_ANY __host__ __device__
#else
#define LKV_ANY
#endif

namespace lkv {

constexpr int kMxUnitCols = 512;
constexpr int kMxTileBytes = 1024;
constexpr int kMxUnitBytes = 4 * kMxTileBytes + 256;

LKV_ANY inline int mx4_units(int32_t cols) { return (cols + kMxUnitCols - 1) / kMxUnitCols; }

// Bytes from one row tile to the next: an odd number of 256-byte pieces.
LKV_ANY inline int mx4_tile_stride(int units) { return ((units * (kMxUnitBytes / 256)) | 1) * 256; }

// Where the i-th of a workgroup's row tiles starts, of which the weight holds `tiles` (at least one): those past the
// last repeat it (a buffer's bounds are checked against the lane's offset, not the scalar one that this goes into).
LKV_ANY inline int mx4_tile_start(int i, int tiles, int tile_stride) { return (i < tiles ? i : tiles - 1) * tile_stride; }

// Codes of column tile kt and scale words of unit u, from a row tile's start.
LKV_ANY inline int mx4_codes_at(int kt) { return (kt >> 2) * kMxUnitBytes + (kt & 3) * kMxTileBytes; }
LKV_ANY inline int mx4_scales_at(int u) { return u * kMxUnitBytes + 4 * kMxTileBytes; }

}  // namespace lkv
