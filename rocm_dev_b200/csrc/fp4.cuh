// Microscaled 4-bit floating point: the held form shared by the quantisers and the products.
//
// Elements are e2m1 codes, two to a byte (even index in the low half), rows of ceil(K / 32) * 16 bytes.  A block of
// consecutive elements along K shares one scale byte: 32 elements and a power of two (e8m0) in MXFP4, 16 elements and an
// e4m3 number in NVFP4.  Scale bytes lie in tiles of 128 rows x 4 blocks, 512 bytes: row r, block b of a tile at
// (r % 32) * 16 + (r / 32) * 4 + b - the 32 lanes x 16 bytes that one tcgen05.cp.32x128b.warpx4 moves into TMEM.  Tiles
// run along K first; K is filled up to a multiple of 256 with zero scales, so that a pipeline stage of 256 elements (one
// 128-byte swizzle row) always finds whole tiles: two in MXFP4, four in NVFP4.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "../../include/rocm_dev_b200.h"

namespace rdb {
namespace fp4 {

constexpr int STAGE_K = 256;             // elements of K per pipeline stage and granularity of the scale tiles
constexpr int TILE_BYTES = 512;          // 128 rows x 4 scale bytes
// Most rows and columns of a tensor: indices rounded up to whole tiles and read-ahead within them stay below 2^31.
constexpr int MAX_EXTENT = 2147483647 - 1024;

template <int FMT>
struct Format {
    static constexpr int BLOCK = FMT == RDB_FP4_NVFP4 ? 16 : 32;
    static constexpr int TILES = STAGE_K / BLOCK / 4;     // scale tiles per stage: 4 or 2
};

__host__ __device__ inline size_t row_bytes(int K) { return static_cast<size_t>((static_cast<long long>(K) + 31) / 32) * 16; }
__host__ __device__ inline int scale_tiles_per_row(int format, int K) {
    return static_cast<int>((static_cast<long long>(K) + STAGE_K - 1) / STAGE_K) * (format == RDB_FP4_NVFP4 ? 4 : 2);
}
__host__ __device__ inline size_t scale_bytes(int format, int rows, int K) {
    return static_cast<size_t>((static_cast<long long>(rows) + 127) / 128) * scale_tiles_per_row(format, K) * TILE_BYTES;
}
// First byte of the four scales of row r in tile column `col`.
__device__ __forceinline__ size_t scale_word(size_t r, int col, int tiles_per_row) {
    return ((r >> 7) * tiles_per_row + col) * TILE_BYTES + (r & 31) * 16 + ((r >> 5) & 3) * 4;
}

}  // namespace fp4
}  // namespace rdb
