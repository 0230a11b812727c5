// Rows as microscaled 4-bit floats and back (micro.cuh has the format).
//
// Bound by HBM.  A thread takes 16 values at a time, a row is 8 to 256 threads of a block, whose values stay in
// registers between the row's maximum and the rounding (up to 64 per thread; longer rows are read again from L2).
//
// Roundings are exact: a quotient next to a border between two codes decides by a whole step.  x / R is exact.  For
// 16-bit x, q = x / (R s) is x times the rounded inverse of s, within 2^-22 of the quotient; a quotient of an 11-bit x
// that is not itself on a border (a number of three bits, times the four of s) is at least 2^-13 away from it, so that q
// rounded to a multiple of 2^-17 is on the border where the quotient is, and on the quotient's side of it else.  fp32 x
// and the scales take a division whose remainder, where it is not zero, goes into the last bit (rounding to odd:
// Boldo and Melquiond, "Emulation of FMA and correctly rounded sums", 2008), which makes the second rounding right.
#include "micro.cuh"
#include "odie_b200.h"
#include <algorithm>

namespace odie {
namespace {

constexpr int MICRO_THREADS = 256;
constexpr int HELD = 4;  // runs of 16 values per thread that stay in registers

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
__device__ __forceinline__ uint32_t codes_of(const float (&q)[8]) {
    uint32_t r;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(r)
        : "f"(q[0]), "f"(q[1]), "f"(q[2]), "f"(q[3]), "f"(q[4]), "f"(q[5]), "f"(q[6]), "f"(q[7]));
    return r;
}

// 16 consecutive values of a row from column c on, zeros behind its end.
template <typename T>
struct Run {
    uint32_t w[16 * sizeof(T) / 4];
    template <bool WIDE>
    __device__ __forceinline__ void load(const T* row, long long c, int width) {
        constexpr int PER = 16 / int(sizeof(T));
        if (WIDE) {  // width a multiple of PER
#pragma unroll
            for (int i = 0; i < int(sizeof(T)); ++i) {
                const uint4 v = c + i * PER < width ? __ldg(reinterpret_cast<const uint4*>(row + c + i * PER)) : make_uint4(0, 0, 0, 0);
                w[4 * i] = v.x;
                w[4 * i + 1] = v.y;
                w[4 * i + 2] = v.z;
                w[4 * i + 3] = v.w;
            }
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = c + i < width ? __float_as_uint(row[c + i]) : 0u;
        } else {
            const uint16_t* at = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                w[i] = (c + 2 * i < width ? at[c + 2 * i] : 0u) | uint32_t(c + 2 * i + 1 < width ? at[c + 2 * i + 1] : 0u) << 16;
        }
    }
    __device__ __forceinline__ float value(int i) const {
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(w[i]);
        } else {
            const float2 f = unpack_pair<T>(w[i / 2]);
            return i % 2 ? f.y : f.x;
        }
    }
    // The bits of the largest magnitude as fp32: those of infinities and NaNs are the largest.
    __device__ __forceinline__ uint32_t largest() const {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) m = max(m, __float_as_uint(value(i)) & 0x7fffffffu);
        return m;
    }
};

// Sixteen codes and their scale's byte; largest: of the block.
template <typename T, int BLOCK>
__device__ __forceinline__ uint2 round_run(const Run<T>& x, uint32_t largest, float inverse_row, uint32_t& scale) {
    float factor, divisor = 1.0f;
    if (BLOCK == 16) {
        scale = __nv_cvt_float_to_fp8(divide_odd(__uint_as_float(largest) * inverse_row, 6.0f), __NV_SATFINITE, __NV_E4M3);
        divisor = __half2float(__half(__nv_cvt_fp8_to_halfraw(uint8_t(scale), __NV_E4M3)));
        factor = scale ? __frcp_rn(divisor) : 0.0f;
    } else {
        const int e = least_power(largest, 0x400000u, 2, -127);
        scale = uint32_t(e + 127);
        factor = power_of_two(-e);
    }
    uint32_t out[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float q[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float v = x.value(h * 8 + i);
            if (BLOCK == 32) {
                q[i] = v * factor;
            } else if (sizeof(T) == 2) {
                q[i] = __fsub_rn(__fadd_rn(v * inverse_row * factor, 96.0f), 96.0f);
            } else {
                q[i] = scale ? copysignf(divide_odd(fabsf(v) * inverse_row, divisor), v) : 0.0f;
            }
        }
        out[h] = codes_of(q);
    }
    return make_uint2(out[0], out[1]);
}

template <typename T, int BLOCK, bool WIDE>
__global__ void __launch_bounds__(MICRO_THREADS) quantize_kernel(MicroArgs a, int lanes_log2) {
    __shared__ uint32_t tops[MICRO_THREADS / 32];
    const int lanes = 1 << lanes_log2, lane = threadIdx.x & (lanes - 1), line = threadIdx.x >> lanes_log2;
    // the tile of rows
    const int tile = blockIdx.x / a.first_blocks, part = blockIdx.x - tile * a.first_blocks;
    long long from, to;
    if (a.offsets) {
        const Unit u = unit_at<false>(a.offsets, a.groups, a.rows, MICRO_ROWS, tile);
        if (u.g < 0) return;
        from = u.from;
        to = u.to;
    } else {
        const int tiles = int((a.group_rows + MICRO_ROWS - 1) / MICRO_ROWS), g = tile / tiles;
        from = g * a.group_rows + (long long)(tile - g * tiles) * MICRO_ROWS;
        to = min((g + 1) * a.group_rows, from + MICRO_ROWS);
    }
    const int inside = part * (MICRO_THREADS >> lanes_log2) + line;
    const long long row = from + inside;
    const bool live = row < to;
    const T* x = static_cast<const T*>(a.x) + row * a.width;
    const int steps = int((a.columns * (4 * BLOCK) + 16 * lanes - 1) / (16 * lanes));

    Run<T> held[HELD];
    uint32_t top = 0;
#pragma unroll
    for (int s = 0; s < HELD; ++s) {
        const long long c = ((long long)s * lanes + lane) * 16;
        held[s] = Run<T>{};
        if (live && c < a.width) held[s].template load<WIDE>(x, c, a.width);
    }
#pragma unroll
    for (int s = 0; s < HELD; ++s) top = max(top, held[s].largest());
    for (int s = HELD; s < steps; ++s) {
        const long long c = ((long long)s * lanes + lane) * 16;
        if (!live || c >= a.width) continue;
        Run<T> run;
        run.template load<WIDE>(x, c, a.width);
        top = max(top, run.largest());
    }
    for (int d = 1; d < min(32, lanes); d *= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
    if (lanes > 32) {
        if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
        __syncthreads();
        const int first = (threadIdx.x >> lanes_log2) << (lanes_log2 - 5);
        for (int w = 0; w < lanes / 32; ++w) top = max(top, tops[first + w]);
    }
    const bool finite = top < 0x7f800000u;
    const int k = BLOCK == 16 && top ? least_power(top, 0x280000u, 11, -126) : 0;
    const float inverse_row = power_of_two(-k);
    if (live && lane == 0) a.row_scales[row] = finite ? power_of_two(k) : __int_as_float(0x7fffffff);

    auto finish = [&](const Run<T>& run, int s) {
        const long long unit = (long long)s * lanes + lane, c = unit * 16;
        uint32_t largest = run.largest(), scale = 0;
        if (BLOCK == 32) largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
        uint2 codes = round_run<T, BLOCK>(run, finite ? largest : 0u, inverse_row, scale);
        if (!finite || !live) {
            codes = make_uint2(0, 0);
            scale = 0;
        }
        // four scales to a word
        if (BLOCK == 16) {
            scale |= __shfl_xor_sync(0xffffffffu, scale, 1) << 8;
            scale |= __shfl_xor_sync(0xffffffffu, scale, 2) << 16;
        } else {
            scale |= __shfl_xor_sync(0xffffffffu, scale, 2) << 8;
            scale |= __shfl_xor_sync(0xffffffffu, scale, 4) << 16;
        }
        const int per = BLOCK / 4;  // threads of a word
        if (lane % per == 0 && unit / per < a.columns)
            *reinterpret_cast<uint32_t*>(a.scales + ((long long)tile * a.columns + unit / per) * MICRO_TILE + micro_byte(inside)) = scale;
        if (live && c / 2 < a.pitch) *reinterpret_cast<uint2*>(a.codes + row * a.pitch + c / 2) = codes;
    };
#pragma unroll
    for (int s = 0; s < HELD; ++s)
        if (s < steps) finish(held[s], s);
    for (int s = HELD; s < steps; ++s) {
        const long long c = ((long long)s * lanes + lane) * 16;
        Run<T> run{};
        if (live && c < a.width) run.template load<WIDE>(x, c, a.width);
        finish(run, s);
    }
}

struct ValuesArgs {
    const uint8_t* codes;
    const uint8_t* scales;
    const float* row_scales;
    long long rows;
    int width;
    long long group_rows;
    long long pitch, columns;
    void* out;
    long long units;  // of 16 values, per row
};

template <typename T, int BLOCK, bool WIDE>
__global__ void __launch_bounds__(256) values_kernel(ValuesArgs a) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long row = i / a.units;
    if (row >= a.rows) return;
    const int c = int(i - row * a.units) * 16;
    const long long g = row / a.group_rows, inside = row - g * a.group_rows, tiles = (a.group_rows + MICRO_ROWS - 1) / MICRO_ROWS;
    const long long tile = g * tiles + inside / MICRO_ROWS;
    const int block = c / BLOCK;
    const uint32_t scale = a.scales[(tile * a.columns + block / 4) * MICRO_TILE + micro_byte(int(inside % MICRO_ROWS)) + block % 4];
    const uint2 codes = *reinterpret_cast<const uint2*>(a.codes + row * a.pitch + c / 2);
    const float s = BLOCK == 16 ? __half2float(__half(__nv_cvt_fp8_to_halfraw(uint8_t(scale), __NV_E4M3)))
                                : scale ? __uint_as_float(scale << 23) : 0x1p-127f;
    const float r = a.row_scales[row];
    float v[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        // e2m1 as fp16, its exponent's bias 14 too small: exact, subnormals too
        const uint32_t code = (e < 8 ? codes.x : codes.y) >> (e % 8 * 4);
        const float m = __half2float(__ushort_as_half(uint16_t((code & 8) << 12 | (code & 7) << 9))) * 16384.0f;
        v[e] = m * s * r;
    }
    T* out = static_cast<T*>(a.out) + row * a.width + c;
    if (WIDE) {
        constexpr int PER = 16 / int(sizeof(T));
#pragma unroll
        for (int p = 0; p < 16 / PER; ++p) {
            Pack<T, 16> pack;
#pragma unroll
            for (int e = 0; e < PER; ++e) pack.v[e] = from_float<T>(v[p * PER + e]);
            if (c + p * PER < a.width) pack.store(out + p * PER);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 16; ++e)
            if (c + e < a.width) out[e] = from_float<T>(v[e]);
    }
}

bool wide_rows(const void* p, int64_t width, int dtype) { return (uintptr_t(p) | uintptr_t(width * row_type_size(dtype))) % 16 == 0; }

template <typename F>
void with_micro(int dtype, int block, bool wide, F&& f) {
    auto typed = [&](auto type) {
        using std::integral_constant;
        if (block == 16) wide ? f(type, integral_constant<int, 16>{}, std::true_type{}) : f(type, integral_constant<int, 16>{}, std::false_type{});
        else wide ? f(type, integral_constant<int, 32>{}, std::true_type{}) : f(type, integral_constant<int, 32>{}, std::false_type{});
    };
    if (dtype == ROW_F32) typed(float{});
    else if (dtype == ROW_BF16) typed(__nv_bfloat16{});
    else typed(__half{});
}

void check_micro(int64_t groups, int64_t rows, int64_t width, int dtype, int block) {
    ODIE_REQUIRE(groups >= 1 && rows >= 0 && rows < (int64_t(1) << 31) && groups < (int64_t(1) << 31) &&
                     groups * rows < (int64_t(1) << 31) - 256 && groups * ((rows + 127) / 128) < (int64_t(1) << 24),
                 "0 to 2^31 - 257 rows, and fewer than 2^24 tiles of 128 of them");
    ODIE_REQUIRE(width >= 1 && width <= (1 << 20), "1 to 2^20 columns");
    check_row_type(dtype);
    ODIE_REQUIRE(block == 16 || block == 32, "block must be 16 or 32");
}

}  // namespace

void launch_quantize(MicroArgs a, int dtype, int block, cudaStream_t stream) {
    // as few threads to a row as hold it: more rows at a time
    int log2 = 3;
    while (log2 < 8 && (16 * HELD << log2) < a.width) ++log2;
    a.first_blocks = MICRO_ROWS / (MICRO_THREADS >> log2);
    const int64_t tiles = a.offsets ? micro_tiles(a.rows, a.groups) : a.groups * ((a.group_rows + MICRO_ROWS - 1) / MICRO_ROWS);
    ODIE_REQUIRE(tiles * a.first_blocks < (int64_t(1) << 31), "too many rows for one launch");
    with_micro(dtype, block, wide_rows(a.x, a.width, dtype), [&](auto type, auto b, auto wide) {
        quantize_kernel<decltype(type), decltype(b)::value, decltype(wide)::value>
            <<<unsigned(tiles * a.first_blocks), MICRO_THREADS, 0, stream>>>(a, log2);
    });
    ODIE_CUDA(cudaGetLastError());
    note_launch();
}

}  // namespace odie

using namespace odie;

extern "C" int odie_quantize(const void* x, int64_t groups, int64_t rows, int64_t width, int dtype, int block, uint8_t* codes,
                             uint8_t* scales, float* row_scales, uint64_t stream) {
    return guarded([&] {
        check_micro(groups, rows, width, dtype, block);
        if (rows == 0) return;
        ODIE_REQUIRE(x && codes && scales && row_scales, "x, codes, scales and row_scales are required");
        ODIE_REQUIRE((uintptr_t(codes) | uintptr_t(scales)) % 16 == 0, "codes and scales must start on 16-byte boundaries");
        MicroArgs a{};
        a.x = x;
        a.rows = groups * rows;
        a.width = int(width);
        a.group_rows = rows;
        a.groups = int(groups);
        a.codes = codes;
        a.scales = scales;
        a.row_scales = row_scales;
        a.pitch = micro_pitch(width);
        a.columns = micro_columns(width, block);
        launch_quantize(a, dtype, block, reinterpret_cast<cudaStream_t>(stream));
    });
}

extern "C" int odie_dequantize(const uint8_t* codes, const uint8_t* scales, const float* row_scales, int64_t groups, int64_t rows,
                               int64_t width, int block, int dtype, void* out, uint64_t stream) {
    return guarded([&] {
        check_micro(groups, rows, width, dtype, block);
        if (rows == 0) return;
        ODIE_REQUIRE(codes && scales && row_scales && out, "codes, scales, row_scales and out are required");
        ODIE_REQUIRE((uintptr_t(codes) | uintptr_t(scales)) % 16 == 0, "codes and scales must start on 16-byte boundaries");
        const ValuesArgs a{codes, scales, row_scales, groups * rows, int(width), rows, micro_pitch(width), micro_columns(width, block), out, (width + 15) / 16};
        const int64_t blocks = (a.rows * a.units + 255) / 256;
        ODIE_REQUIRE(blocks < (int64_t(1) << 31), "too many rows and columns for one launch");
        with_micro(dtype, block, wide_rows(out, width, dtype), [&](auto type, auto b, auto wide) {
            values_kernel<decltype(type), decltype(b)::value, decltype(wide)::value>
                <<<unsigned(blocks), 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(a);
        });
        ODIE_CUDA(cudaGetLastError());
        note_launch();
    });
}
