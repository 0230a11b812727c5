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
// A kernel may start while the one before it on its stream ends, if that says so and the launch of the other allows it; it
// then waits for all of it, and for what it wrote, before it reads that.
__device__ __forceinline__ void dependents_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void dependencies_done() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// Tiles of rows that `rows` rows in `groups` groups may need: those of no group (behind the last offset) have some too.
inline int64_t micro_tiles(int64_t rows, int64_t groups) { return (rows + MICRO_ROWS - 1) / MICRO_ROWS + groups + 1; }

// ---- rounding (see micro.cu)
// a / b, a >= 0, b > 0, cut to 24 bits with the last one set where the quotient is not exact.
__device__ __forceinline__ float divide_odd(float a, float b) {
    const float q = __fdiv_rn(a, b), r = fmaf(-q, b, a);
    uint32_t bits = __float_as_uint(q);
    if (r < 0.0f) --bits;
    return __uint_as_float(r != 0.0f ? bits | 1u : bits);
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(uint32_t(e + 127) << 23); }  // -126 <= e <= 127
// The least e >= least with v <= most 2^e; most = mantissa(of 1.m) 2^shift, v >= 0 as its bits.
__device__ __forceinline__ int least_power(uint32_t bits, uint32_t most_mantissa, int shift, int least) {
    const int e = int(bits >> 23) - 127 - shift + ((bits & 0x7fffffu) > most_mantissa);
    return max(least, e);  // (a subnormal v: far below any `least`)
}
// Eight values as codes, the first in the lowest four bits.
__device__ __forceinline__ uint32_t codes_of(const float2 (&q)[4]) {
    uint32_t r;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(r)
        : "f"(q[0].x), "f"(q[0].y), "f"(q[1].x), "f"(q[1].y), "f"(q[2].x), "f"(q[2].y), "f"(q[3].x), "f"(q[3].y));
    return r;
}
__device__ __forceinline__ float e4m3_value(uint32_t byte) { return __half2float(__half(__nv_cvt_fp8_to_halfraw(uint8_t(byte), __NV_E4M3))); }

// Two codes, in the lowest byte, as a pair of fp16; eight as four pairs.  (Not for words whose upper half the compiler knows to
// be zero: nvcc 12.9 made all four pairs zero then.)
__device__ __forceinline__ __half2 halves_of(uint32_t codes) {
    uint32_t r;
    asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\t}" : "=r"(r) : "r"(codes));
    return *reinterpret_cast<const __half2*>(&r);
}
__device__ __forceinline__ void halves_of(uint32_t codes, __half2* h) {
    uint32_t r[4];
    asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\tcvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
        : "r"(codes));
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = *reinterpret_cast<const __half2*>(&r[i]);
}
template <int BLOCK>
__device__ __forceinline__ float scale_value(uint32_t byte) {
    return BLOCK == 16 ? e4m3_value(byte) : byte ? __uint_as_float(byte << 23) : 0x1p-127f;
}

// Where N values of each thread of a row are exchanged, one word per row of N beyond them: no two in one bank.  value(i): the
// thread's i-th of its N neighbours' in a row; strided(i): the one that is i x lanes behind its lane's (lanes a multiple of N).
template <int N>
struct Exchange {
    uint32_t *row, *at;
    int step;
    __device__ __forceinline__ Exchange(uint32_t* words, int lanes, int lane) {
        words += (threadIdx.x - lane) * (N + 1);
        row = words + lane * (N + 1);
        at = words + lane + lane / N;
        step = lanes + lanes / N;
    }
    __device__ __forceinline__ uint32_t& value(int i) const { return row[i]; }
    __device__ __forceinline__ uint32_t& strided(int i) const { return at[i * step]; }
};
__device__ __forceinline__ void sync_row(int lanes) {  // the threads of a row
    if (lanes > 32) __syncthreads();
    else __syncwarp();
}

// 16 consecutive values of a row from column c on, zeros behind its end.
template <typename T>
struct Run {
    static constexpr int WORDS = 16 * sizeof(T) / 4;
    uint32_t w[WORDS];
    __device__ __forceinline__ void load_wide(const T* row, long long c, int width) {  // width a multiple of PER
        constexpr int PER = 16 / int(sizeof(T));
#pragma unroll
        for (int i = 0; i < int(sizeof(T)); ++i) {
            const uint4 v = c + i * PER < width ? __ldg(reinterpret_cast<const uint4*>(row + c + i * PER)) : make_uint4(0, 0, 0, 0);
            w[4 * i] = v.x;
            w[4 * i + 1] = v.y;
            w[4 * i + 2] = v.z;
            w[4 * i + 3] = v.w;
        }
    }
    // The row's `lanes` threads take its 16 lanes values from `from` on, `left` of them inside.
    __device__ __forceinline__ void load(const T* from, int left, int lanes, int lane, const Exchange<16>& x) {
        from += lane;
        left -= lane;
        uint32_t v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if constexpr (sizeof(T) == 4) v[i] = i * lanes < left ? __float_as_uint(from[i * lanes]) : 0u;
            else v[i] = i * lanes < left ? reinterpret_cast<const uint16_t*>(from)[i * lanes] : 0u;
        }
        sync_row(lanes);
#pragma unroll
        for (int i = 0; i < 16; ++i) x.strided(i) = v[i];
        sync_row(lanes);
#pragma unroll
        for (int i = 0; i < WORDS; ++i) {
            if constexpr (sizeof(T) == 4) w[i] = x.value(i);
            else w[i] = x.value(2 * i) | x.value(2 * i + 1) << 16;
        }
    }
    __device__ __forceinline__ float2 pair_at(int i) const {  // values 2 i and 2 i + 1
        if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
        else return unpack_pair<T>(w[i]);
    }
    // The bits of the largest magnitude as fp32: those of infinities and NaNs are the largest.
    __device__ __forceinline__ uint32_t largest() const {
        uint32_t m = 0;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 16; ++i) m = max(m, w[i] & 0x7fffffffu);
            return m;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
            m = max(m & 0xffffu, m >> 16);
            if constexpr (std::is_same<T, __nv_bfloat16>::value) return m << 16;
            else return __float_as_uint(__half2float(__ushort_as_half(uint16_t(m))));
        }
    }
};

// Sixteen codes and their scale's byte; largest: of the block.
template <typename T, int BLOCK>
__device__ __forceinline__ uint2 round_run(const Run<T>& x, uint32_t largest, float inverse_row, uint32_t& scale) {
    float2 q[8];
    if constexpr (BLOCK == 32) {
        const int e = least_power(largest, 0x400000u, 2, -127);
        scale = uint32_t(e + 127);
        const Pair factor = same(power_of_two(-e));
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = both(mul2(pair(x.pair_at(i).x, x.pair_at(i).y), factor));
    } else if constexpr (sizeof(T) == 2) {
        const float t = __uint_as_float(largest) * inverse_row * (1.0f / 6.0f), wide = t * 257.0f;
        scale = __nv_cvt_float_to_fp8(__fsub_rn(wide, __fsub_rn(wide, t)), __NV_SATFINITE, __NV_E4M3);
        const float factor = scale ? inverse_approx(e4m3_value(scale)) : 0.0f;
        const Pair up = same(96.0f), down = same(-96.0f);
        if (std::is_same<T, __half>::value || inverse_row < 0x1p100f) {
            const Pair by = same(inverse_row * factor);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float2 v = x.pair_at(i);
                q[i] = both(add2(fma2(pair(v.x, v.y), by, up), down));
            }
        } else {  // the factors' product may be infinite
            const Pair first = same(inverse_row), second = same(factor);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float2 v = x.pair_at(i);
                q[i] = both(add2(fma2(mul2(pair(v.x, v.y), first), second, up), down));
            }
        }
    } else {
        scale = __nv_cvt_float_to_fp8(divide_odd(__uint_as_float(largest) * inverse_row, 6.0f), __NV_SATFINITE, __NV_E4M3);
        const float divisor = e4m3_value(scale);
        const Pair by = same(scale ? inverse_approx(divisor) : 0.0f), first = same(inverse_row), up = same(96.0f), down = same(-96.0f);
        auto side = [](float rest) { return fminf(fmaxf(rest * 0x1p100f, -0x1p-18f), 0x1p-18f); };
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 v = x.pair_at(i);
            const Pair y = mul2(pair(v.x, v.y), first), near = add2(fma2(y, by, up), down);
            const float2 rest = both(fma2(mul2(near, same(-1.0f)), same(divisor), y));
            q[i] = both(add2(near, pair(side(rest.x), side(rest.y))));
        }
    }
    const float2 low[4] = {q[0], q[1], q[2], q[3]}, high[4] = {q[4], q[5], q[6], q[7]};
    return make_uint2(codes_of(low), codes_of(high));
}

// rows of x (dtype, contiguous) with the pieces above; offsets on the device as for odie_linear.
void launch_quantize(MicroArgs a, int dtype, int block, cudaStream_t stream);

}  // namespace odie
