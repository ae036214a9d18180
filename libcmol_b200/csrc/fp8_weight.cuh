// fp8_weight.cuh — e4m3 weights with a scale for each block of 128 x 128, as
// the matrix product reads them.
//
// The matrix is cut into its 128 x 128 blocks; block (rb, kb) is the
// contiguous 16 KB at tiles + (rb * kblocks + kb) * 16384, so the rows that a
// CTA owns are one contiguous stream along k.  Inside a block, row r is the
// 128 bytes at 128 r, with its 16-byte chunks permuted (chunk c at c ^ (r %
// 8)): the K-major 128-byte-swizzle layout in which the tensor core reads an
// operand from shared memory, so one bulk copy brings a block in place.  Rows
// and columns past the matrix are zero.
#pragma once
#include "fp8.cuh"

#define FP8_TILE_BYTES (FP8_BLOCK * FP8_BLOCK)

struct Fp8W {
    const uint8_t *tiles;
    const float   *scales;      // [row block][k block]
    int            rows, k;
    int            rblocks, kblocks;
};

struct cmolcu_fp8_weight {
    Fp8W  w;
    int   device;
    void *base;                 // one allocation: tiles, then scales
};

// Byte of value (r, c) of a block.
__host__ __device__ __forceinline__ int fp8_tile_byte(int r, int c) {
    return r * 128 + ((((c >> 4) ^ (r & 7)) << 4) | (c & 15));
}
