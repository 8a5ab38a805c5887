// mx4.cuh — the packed form of a microscaled 4-bit matrix, shared by the cast
// and the product.
//
// Element codes: e2m1, two a byte (the even element in the low nibble), each
// row padded with zero codes to whole blocks of 32: `row_bytes` a row.
//
// Scale bytes: the shared exponent + 127 of each (row, block), in tiles of 128
// rows x 4 blocks of 512 bytes, the layout in which the tensor cores take
// scales: row r, block b of a tile is byte (r % 32) * 16 + (r / 32) * 4 + b.
// A row of tiles holds a whole number of pairs (256 elements of the
// contraction), and every padding byte is 127 (2^0), so that a kernel may load
// whole tiles and multiply the padding's zero codes.
#pragma once

#include <cstdint>

namespace drift {

constexpr int kMxBlock = 32;
constexpr int kMxTileRows = 128;
constexpr int kMxTileBytes = 512;

__host__ __device__ inline int64_t mx4_blocks(int64_t cols) { return (cols + 31) / 32; }
__host__ __device__ inline int64_t mx4_row_bytes(int64_t cols) { return mx4_blocks(cols) * 16; }
// Tiles in one row of tiles: an even number.
__host__ __device__ inline int64_t mx4_k_tiles(int64_t cols) { return (cols + 255) / 256 * 2; }
__host__ __device__ inline int64_t mx4_row_tiles(int64_t rows) { return (rows + 127) / 128; }
__host__ __device__ inline int64_t mx4_scale_offset(int64_t row, int64_t block, int64_t k_tiles) {
    return ((row / 128) * k_tiles + block / 4) * kMxTileBytes + (row % 32) * 16 +
           (row % 128 / 32) * 4 + block % 4;
}

}  // namespace drift
