// Microscaled 4-bit rows (micro.cu, linear4.cu).
//
// value = R s c: c in e2m1 (0, 1/2, 1, 3/2, 2, 3, 4, 6 and a sign), s one scale per block of 16 or 32 values, R one
// fp32 power of two per row.
//
//   block 16   R = the least 2^k with |row| <= 2688 R = 6 * 448 R, k >= -126 (1 for a row of zeros);
//              s = e4m3(max |block| / (6 R)), c = e2m1(x / (R s))
//   block 32   R = 1; s = the least 2^e with |block| <= 6 s, e >= -127 (e8m0); c = e2m1(x / s)
//
// rounded once each, to nearest even, saturating; a block whose s is 0 holds zeros.  R is NaN for a row that holds an
// infinity or a NaN, its codes are zero.  A row's own R (rather than one for all rows) makes a row's result
// independent of the rows beside it; a power of two costs no bit of x.
//
// codes: rows of pitch bytes, two values to a byte, the even one low, zeros behind the last.
// scales: tiles of 128 rows x 4 blocks, 512 bytes, as tcgen05.cp takes them: row 32 q + l, block b at byte 16 l + 4 q + b;
// a group's rows are cut into tiles from its first row on: [tiles][column tiles][512].
#pragma once
#include "activation.cuh"
#include <cuda_fp8.h>

namespace odie {

constexpr int MICRO_ROWS = 128, MICRO_TILE = 512;
inline int64_t micro_pitch(int64_t width) { return (width + 31) / 32 * 16; }
inline int64_t micro_columns(int64_t width, int block) { return (width + 4 * block - 1) / (4 * block); }

// The byte of a row's first scale in a tile.
__host__ __device__ __forceinline__ int micro_byte(int row) { return (row & 31) * 16 + (row >> 5) * 4; }

struct MicroArgs {
    const void* x;
    long long rows;
    int width;
    long long group_rows;  // without offsets: rows of each group
    int groups;
    const int* offsets;    // null: groups of group_rows
    uint8_t* codes;
    uint8_t* scales;
    float* row_scales;
    long long pitch, columns;  // of codes in bytes, of scales in tiles
    int first_blocks;          // blocks of threads per tile of rows
};
// Tiles of rows that `rows` rows in `groups` groups may need: those of no group (behind the last offset) have some too.
inline int64_t micro_tiles(int64_t rows, int64_t groups) { return (rows + MICRO_ROWS - 1) / MICRO_ROWS + groups + 1; }

// rows of x (dtype, contiguous) with the pieces above; offsets on the device as for odie_linear.
void launch_quantize(MicroArgs a, int dtype, int block, cudaStream_t stream);

}  // namespace odie
