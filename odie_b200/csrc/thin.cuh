// Thin linear layers (thin.cu): up to 64 inputs and outputs, multiples of 8, the sizes of this library's own heads.
#pragma once
#include "activation.cuh"
#include <algorithm>

namespace odie {

struct ThinArgs {
    long long rows;
    int inputs, outputs, groups;
    const int* offsets;     // null: one group of all rows
    int chunk;              // rows per block, a multiple of 64
    const void* x;
    const void* weight;
    // forward
    const void* bias;
    const void* residual;
    void* y;
    void* slope;            // null: not kept
    int activation;
    // backward
    const void* d_y;
    const void* kept;       // the slope that forward kept; null: 1
    void* d_x;              // each null where not wanted
    void* d_weight;
    void* d_bias;
    void* d_residual;
    float* partial;         // [unit][outputs * inputs + outputs] sums of several units per group; null: one unit each
};

inline bool thin_sizes(int inputs, int outputs) { return inputs <= 64 && outputs <= 64 && inputs % 8 == 0 && outputs % 8 == 0; }
// Blocks that share an SM: as many as their registers allow without spilling (a ReLU's corner takes some: 2^20 rows of
// 32 -> 64, 64 -> 64 and 32 -> 32 fp16 take 61, 80 and 39 us at a block more, 47, 70 and 37 so) and, backward, the rows on their way in shared memory.  Backward with
// codes: two, with more stages each.
constexpr int thin_blocks(int inputs, int outputs, int activation, bool backward) {
    const int wide = (inputs > 32) + (outputs > 32);
    if (backward) return activation == ACT_SILU || activation == ACT_GELU ? 2 : 4 - wide;
    return activation == ACT_RELU ? 4 - wide : wide == 2 ? 3 : 4;
}
// Rows per block: as many blocks as fit the SMs at once, so that W is read and sums are written as seldom as that allows.
inline int thin_chunk(int64_t rows, int inputs, int outputs, int activation, bool backward) {
    const int64_t blocks = 148 * thin_blocks(inputs, outputs, activation, backward), share = (rows + blocks - 1) / blocks;
    return int(std::max<int64_t>(64, (share + 63) / 64 * 64));
}
// Units of work (blocks) at most: every group has at least one, and rows of no group their own.
inline int64_t thin_units(int64_t rows, int groups, int chunk) { return (rows + chunk - 1) / chunk + groups + 1; }

template <typename T>
void launch_thin_forward(const ThinArgs& a, cudaStream_t stream);
template <typename T>
void launch_thin_backward(const ThinArgs& a, cudaStream_t stream);

}  // namespace odie
