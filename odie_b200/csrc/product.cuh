// What the tensor-core products of rows share (linear.cu, linear4.cu): tiles walked without divisions, windows of the
// result moved between registers and global memory, the epilogue's arithmetic, bounded waits and their error word.
#pragma once
#include "activation.cuh"
#include "tc.cuh"
#include <cuda.h>
#include <cudaTypedefs.h>

namespace odie {

// Polls of a wait, up to 4 us each: some ten seconds.  Waits of the products have GemmArgs::limit, what gives up waits for
// its own copies and products with this one.
constexpr uint32_t WAIT_LIMIT = 1u << 22;
constexpr int STAGING = 2048;  // bytes per epilogue warp: 32 rows x 32 columns of 16 bits

// n / d for 0 <= n < 2^31 by a multiplication: m = ceil(2^64 / d).
struct Divide {
    unsigned long long m;
    uint32_t d;
    static Divide by(int64_t d) { return {d > 1 ? ~0ull / uint64_t(d) + 1 : 0, uint32_t(d)}; }
    __device__ __forceinline__ int operator()(int n) const { return d == 1 ? n : int(__umul64hi((unsigned long long)n, m)); }
};

constexpr int BAND = 16;  // row tiles walked together, so that a W tile serves them from L2

// The same value in every lane, as the compiler sees too.
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

// The staging tile of an epilogue warp: 32 rows of 64 bytes, the 16-byte units of a row permuted so that both a
// thread per row and four threads per row meet no bank twice.
__device__ __forceinline__ uint4* staged(char* base, int row, int unit) {
    return reinterpret_cast<uint4*>(base + row * 64 + ((unit ^ ((row >> 1) & 3)) << 4));
}

// 32 rows x 32 columns of a row-major 16-bit matrix, moved between global memory and the staging tile.  Where every
// row starts on a 16-byte boundary, thread (lane) moves the 16-byte unit lane % 4 of rows lane / 4 + 8 i, else the
// element `lane` of every row.
struct Window {
    int ld;
    int rows, columns;  // inside the matrix
    bool wide;          // 16-byte accesses
};
__device__ __forceinline__ void window_load(const uint16_t* at, const Window& w, int lane, uint4 (&v)[4]) {
    const int r = lane / 4, c = (lane & 3) * 8;
    const uint16_t* from = at + (long long)r * w.ld + c;
    const long long step = 8ll * w.ld;
    if (w.rows == 32 && w.columns >= 32) {
#pragma unroll
        for (int i = 0; i < 4; ++i, from += step) v[i] = __ldg(reinterpret_cast<const uint4*>(from));
    } else if (c + 8 <= w.columns) {  // wide rows: columns are a multiple of 8
#pragma unroll
        for (int i = 0; i < 4; ++i, from += step)
            v[i] = r + 8 * i < w.rows ? __ldg(reinterpret_cast<const uint4*>(from)) : make_uint4(0, 0, 0, 0);
    }
}
__device__ __forceinline__ uint16_t* staged_element(char* base, int row, int c) {
    return reinterpret_cast<uint16_t*>(staged(base, row, c >> 3)) + (c & 7);
}
__device__ __forceinline__ void window_fetch(const uint16_t* at, const Window& w, int lane, char* staging) {
    if (lane < w.columns) {
#pragma unroll 8
        for (int r = 0; r < w.rows; ++r) *staged_element(staging, r, lane) = at[(long long)r * w.ld + lane];
    }
}
__device__ __forceinline__ void window_store(uint16_t* at, const Window& w, int lane, char* staging) {
    if (w.wide) {
        const int r = lane / 4, c = (lane & 3) * 8;
        uint16_t* to = at + (long long)r * w.ld + c;
        const long long step = 8ll * w.ld;
        // rows r + 8 i share the permutation of row r: 512 bytes apart
        const uint4* from = staged(staging, r, lane & 3);
        if (w.rows == 32 && w.columns >= 32) {
#pragma unroll
            for (int i = 0; i < 4; ++i, to += step) *reinterpret_cast<uint4*>(to) = from[i * 32];
        } else if (c + 8 <= w.columns) {
#pragma unroll
            for (int i = 0; i < 4; ++i, to += step)
                if (r + 8 * i < w.rows) *reinterpret_cast<uint4*>(to) = from[i * 32];
        }
    } else if (lane < w.columns) {
#pragma unroll 8
        for (int r = 0; r < w.rows; ++r) at[(long long)r * w.ld + lane] = *staged_element(staging, r, lane);
    }
}

template <int ACT>
__device__ __forceinline__ void finish(float (&v)[32], uint32_t (&codes)[16], const float* bias) {
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
        const float4 b = *reinterpret_cast<const float4*>(bias + i);
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
            Pair slope;
            const float2 y = both(activate<ACT>(add2(pair(v[i + j], v[i + j + 1]), j ? pair(b.z, b.w) : pair(b.x, b.y)), slope));
            v[i + j] = y.x;
            v[i + j + 1] = y.y;
            codes[(i + j) / 2] = slope_codes(slope);
        }
    }
}
// ReLU: gives a mask, a bit where it is on.
__device__ __forceinline__ uint32_t finish_relu(float (&v)[32], const float* bias) {
    uint32_t off = 0;
#pragma unroll
    for (int i = 30; i >= 0; i -= 2) {
        const float2 z = both(add2(pair(v[i], v[i + 1]), pair(bias[i], bias[i + 1])));
        off = off_bits(off, z.x, z.y);
        v[i] = max_nan(z.x, 0.0f);
        v[i + 1] = max_nan(z.y, 0.0f);
    }
    return ~off;
}

// linear.cu: the device's error word, on the host (refused once after a wait has run out), the limit of the waits of
// kernels that are launched from now on, and the driver's encoder of tensor maps.
int* checked_error_word();
uint32_t product_wait_limit();
PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder();

}  // namespace odie
