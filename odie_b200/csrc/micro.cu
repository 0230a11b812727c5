// Rows as microscaled 4-bit floats and back (micro.cuh has the format).
//
// Bound by its instructions, 9 to 12 to a value, next to HBM (16384 x 2048 bf16: 18.5 us to 4 bits, 4.6 TB/s, and 16.5 back,
// 5.1 TB/s).  A thread takes 16 values at a time, a row is 4 to 256 threads of a block, whose values stay in registers
// between the row's maximum and the rounding (up to 64 per thread; longer rows are read again from L2).  Rows that do not
// start on 16-byte boundaries are moved element by element, neighbours by neighbouring threads, through shared memory.
//
// Roundings are exact: a quotient next to a border between two codes decides by a whole step.  x / R is exact.  For
// 16-bit x, q = x / (R s) is x times an approximate inverse of s, within 2^-22 of the quotient, rounded to a multiple of
// 2^-17 (by adding 96 in the same fused step): a quotient of an 11-bit x that is not itself on a border (a number of
// three bits, times the four of s) is at least 2^-13 away from it, so that the rounded q is on the border where the
// quotient is, and on the quotient's side of it else.  Their scales likewise, rounded to 16 bits: a border of e4m3 is a
// number of five bits, times 6.  fp32 x may be closer to a border: q is as above, and 2^-18 to the side that the sign of
// x / R - q s, one fused step, says, so that it is on the border for a quotient that is.  The scales of fp32 rows take a division
// whose remainder, where it is not zero, goes into the last bit (rounding to odd: Boldo and Melquiond, "Emulation of FMA and
// correctly rounded sums", 2008), which makes the second rounding right.
#include "micro.cuh"
#include "odie_b200.h"
#include <algorithm>

namespace odie {
namespace {

constexpr int MICRO_THREADS = 256;
constexpr int HELD = 4;  // runs of 16 values per thread that stay in registers

// unit_at<false> by a whole block, for tiles of rows: a few groups to a thread, one wait for their offsets.  Sums in 64 bits:
// offsets out of order may hold more tiles than 32 bits count, and one thread alone has the tile.
// From how many groups on: unit_at waits once for 32 groups, this once in all, but it stops the block twice.  A product of
// 2048 rows with unit_at | with this: 8 groups 12.9 | 14.6 us, 64: 22.9 | 26.4, 128: 27.6 | 28.9, 256: 51.3 | 48.3,
// 512: 79.1 | 65.2, 1024: 198 | 123; of 8 rows 8 groups 8.3 | 9.3, 128: 21.3 | 19.9, 256: 44.8 | 31.4, 1024: 234 | 90.
constexpr int MANY_GROUPS = 256;
struct Tile {
    long long from, to;  // rows; from < 0: no such tile
};
__device__ __forceinline__ Tile tile_at(const int* offsets, int groups, long long rows, int tile) {
    constexpr int EACH = 5;  // 256 x 5 hold 1024 groups and the rows of none
    __shared__ long long totals[MICRO_THREADS / 32];
    __shared__ Tile found;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, first = threadIdx.x * EACH;
    int from[EACH], to[EACH];
    uint32_t count[EACH];
    long long before = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        long long begin = 0, end = 0;
        if (first + i < groups) {
            group_rows(offsets, first + i, rows, begin, end);
        } else if (first + i == groups) {
            long long b;
            group_rows(offsets, groups - 1, rows, b, begin);
            end = rows;
        }
        from[i] = int(begin);
        to[i] = int(end);
        count[i] = (uint32_t(to[i] - from[i]) + (MICRO_ROWS - 1)) / MICRO_ROWS;
        before += count[i];
    }
    const long long own = before;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const long long other = __shfl_up_sync(0xffffffffu, before, d);
        if (lane >= d) before += other;
    }
    if (lane == 31) totals[warp] = before;
    if (threadIdx.x == 0) found = {-1, -1};
    __syncthreads();
    before -= own;
    for (int w = 0; w < warp; ++w) before += totals[w];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        if (tile >= before && tile < before + count[i]) {
            const long long begin = from[i] + (tile - before) * MICRO_ROWS;
            found = {begin, min((long long)to[i], begin + MICRO_ROWS)};
        }
        before += count[i];
    }
    __syncthreads();
    return found;
}

template <typename T, int BLOCK, bool WIDE>
__global__ void __launch_bounds__(MICRO_THREADS, sizeof(T) == 2 ? 4 : 2) quantize_kernel(MicroArgs a, int lanes_log2) {
    __shared__ uint32_t tops[MICRO_THREADS / 32];
    __shared__ uint32_t words[WIDE ? 1 : MICRO_THREADS * 17];
    const int lanes = 1 << lanes_log2, lane = threadIdx.x & (lanes - 1), line = threadIdx.x >> lanes_log2;
    const Exchange<16> exchange(words, lanes, lane);
    dependents_may_start();
    // the tile of rows
    const int tile = blockIdx.x / a.first_blocks, part = blockIdx.x - tile * a.first_blocks;
    long long from, to;
    if (a.offsets) {
        if (a.groups >= MANY_GROUPS) {
            const Tile t = tile_at(a.offsets, a.groups, a.rows, tile);
            from = t.from;
            to = t.to;
        } else {
            const Unit u = unit_at<false>(a.offsets, a.groups, a.rows, MICRO_ROWS, tile);
            from = u.g < 0 ? -1 : u.from;
            to = u.to;
        }
        if (from < 0) return;
    } else {
        const int tiles = int((a.group_rows + MICRO_ROWS - 1) / MICRO_ROWS), g = tile / tiles;
        from = g * a.group_rows + (long long)(tile - g * tiles) * MICRO_ROWS;
        to = min((g + 1) * a.group_rows, from + MICRO_ROWS);
    }
    const int inside = part * (MICRO_THREADS >> lanes_log2) + line;
    const long long row = from + inside;
    const bool live = row < to;
    const T* x = static_cast<const T*>(a.x) + row * a.width;
    const int steps = int((uint32_t(a.columns) * (4 * BLOCK) + 16 * lanes - 1) >> (lanes_log2 + 4));
    auto load = [&](Run<T>& run, int s) {
        const int first = s * lanes * 16;
        if constexpr (WIDE) {
            if (live && first + lane * 16 < a.width) run.load_wide(x, first + lane * 16, a.width);
        } else {
            run.load(x + first, live ? a.width - first : 0, lanes, lane, exchange);
        }
    };

    Run<T> held[HELD];
    uint32_t largest[HELD], top = 0;
#pragma unroll
    for (int s = 0; s < HELD; ++s) {
        held[s] = Run<T>{};
        if (s < steps) load(held[s], s);
    }
#pragma unroll
    for (int s = 0; s < HELD; ++s) {
        largest[s] = held[s].largest();
        top = max(top, largest[s]);
    }
    for (int s = HELD; s < steps; ++s) {
        Run<T> run{};
        load(run, s);
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
    const int k = BLOCK == 16 && top && finite ? least_power(top, 0x280000u, 11, -126) : 0;
    const float inverse_row = power_of_two(-k);
    if (live && lane == 0) a.row_scales[row] = finite ? power_of_two(k) : __int_as_float(0x7fffffff);

    constexpr uint32_t PER = BLOCK / 4;  // threads of four scales
    const uint32_t columns = uint32_t(a.columns), pitch = uint32_t(a.pitch);
    uint8_t* codes_at = a.codes + row * a.pitch + lane * 8;
    uint8_t* scales_at = a.scales + ((long long)tile * a.columns + uint32_t(lane) / PER) * MICRO_TILE + micro_byte(inside);
    auto finish = [&](const Run<T>& run, uint32_t most, int s) {
        const uint32_t unit = uint32_t(s) * lanes + lane;
        uint32_t scale = 0;
        if (BLOCK == 32) most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
        uint2 codes = round_run<T, BLOCK>(run, finite ? most : 0u, inverse_row, scale);
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
        if (lane % PER == 0 && unit / PER < columns) *reinterpret_cast<uint32_t*>(scales_at + uint32_t(s) * (uint32_t(lanes) / PER) * MICRO_TILE) = scale;
        if (live && unit * 8 < pitch) *reinterpret_cast<uint2*>(codes_at + uint32_t(s) * lanes * 8) = codes;
    };
#pragma unroll
    for (int s = 0; s < HELD; ++s)
        if (s < steps) finish(held[s], largest[s], s);
    for (int s = HELD; s < steps; ++s) {
        Run<T> run{};
        load(run, s);
        finish(run, run.largest(), s);
    }
}

struct ValuesArgs {
    const uint8_t* codes;
    const uint8_t* scales;
    const float* row_scales;
    long long rows;
    int width;
    uint32_t group_rows;
    long long pitch, columns;
    void* out;
};
constexpr int VALUES_RUNS = 4;  // of a thread, that finding its row's place is worth it

// A row by 2^lanes_log2 threads, N values (16 bytes, or 8 values that leave one by one) of each at a time.
template <typename T, int BLOCK, bool WIDE>
__global__ void __launch_bounds__(MICRO_THREADS) values_kernel(ValuesArgs a, int lanes_log2) {
    constexpr int N = WIDE ? 16 / int(sizeof(T)) : 8;
    __shared__ uint32_t shared_words[WIDE ? 1 : MICRO_THREADS * (N + 1)];
    const int lanes = 1 << lanes_log2, lane = threadIdx.x & (lanes - 1);
    const Exchange<N> exchange(shared_words, lanes, lane);
    const long long row = (long long)blockIdx.x * (MICRO_THREADS >> lanes_log2) + (threadIdx.x >> lanes_log2);
    const bool live = row < a.rows;
    const uint32_t g = live ? uint32_t(row) / a.group_rows : 0, inside = uint32_t(row) - g * a.group_rows;
    const long long tile = (long long)g * ((a.group_rows + MICRO_ROWS - 1) / MICRO_ROWS) + inside / MICRO_ROWS;
    const uint8_t* scales = a.scales + tile * a.columns * MICRO_TILE + micro_byte(inside % MICRO_ROWS);
    const uint8_t* codes_at = a.codes + row * a.pitch;
    T* out = static_cast<T*>(a.out) + row * a.width;
    const float row_scale = live ? __ldg(a.row_scales + row) : 0.0f;
    const uint32_t width = a.width;
    const uint32_t steps = (width + N * lanes - 1) >> (lanes_log2 + (N == 8 ? 3 : 2));
#pragma unroll VALUES_RUNS
    for (uint32_t s = 0; s < steps; ++s) {
        const uint32_t first = s * lanes * N, c = first + lane * N;
        uint32_t words[N * sizeof(T) / 4];
        if (live && c < width) {
            const uint32_t block = c / BLOCK;
            const uint32_t scale = __ldg(scales + block / 4 * MICRO_TILE + block % 4);  // (at most 2^16 x 512 bytes)
            const uint32_t codes = N == 8 ? __ldg(reinterpret_cast<const uint32_t*>(codes_at + c / 2)) : uint32_t(__ldg(reinterpret_cast<const uint16_t*>(codes_at + c / 2)));
            const Pair by = same(scale_value<BLOCK>(scale) * row_scale);  // exact, and so are the values: six bits
            __half2 halves[4];
            if constexpr (N == 8) {
                halves_of(codes, halves);
            } else {
                halves[0] = halves_of(codes);
                halves[1] = halves_of(codes >> 8);
            }
#pragma unroll
            for (int e = 0; e < N / 2; ++e) {
                const float2 m = __half22float2(halves[e]), v = both(mul2(pair(m.x, m.y), by));
                if constexpr (sizeof(T) == 4) {
                    words[2 * e] = __float_as_uint(v.x);
                    words[2 * e + 1] = __float_as_uint(v.y);
                } else {
                    words[e] = pack_pair<T>(v.x, v.y);
                }
            }
        }
        if constexpr (WIDE) {
            if (live && c < width) *reinterpret_cast<uint4*>(out + c) = make_uint4(words[0], words[1], words[2], words[3]);
        } else {
            sync_row(lanes);
#pragma unroll
            for (int e = 0; e < N; ++e) exchange.value(e) = sizeof(T) == 4 ? words[e * sizeof(T) / 4] : words[e * sizeof(T) / 4] >> (e % 2 * 16);
            sync_row(lanes);
            const int left = live ? int(width - first) - lane : 0;
            T* to = out + first + lane;
#pragma unroll
            for (int e = 0; e < N; ++e) {
                if (e * lanes >= left) continue;
                if constexpr (sizeof(T) == 4) to[e * lanes] = __uint_as_float(exchange.strided(e));
                else reinterpret_cast<uint16_t*>(to)[e * lanes] = uint16_t(exchange.strided(e));
            }
        }
    }
}

// The threads of a row, as a power of two of at least 2^least: as few as take it in `runs` runs of n values each; more, up
// to one run each, where the rows leave threads idle (four blocks to an SM; 64 x 4096 bf16 to 4 bits:
// 2.5 us, with the fewest threads 3.2).
int row_lanes(int64_t rows, int64_t width, int n, int runs, int least) {
    int log2 = least;
    while (log2 < 8 && (int64_t(n) * runs << log2) < width) ++log2;
    while (log2 < 8 && (int64_t(n) << log2) < width && (rows << log2) < 148 * 4 * MICRO_THREADS) ++log2;
    return log2;
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
    const bool whole = wide_rows(a.x, a.width, dtype);
    const int log2 = row_lanes(a.rows, a.width, 16, HELD, whole ? (block == 16 ? 2 : 3) : 4);  // (at least the threads of four scales)
    a.first_blocks = MICRO_ROWS / (MICRO_THREADS >> log2);
    const int64_t tiles = a.offsets ? micro_tiles(a.rows, a.groups) : a.groups * ((a.group_rows + MICRO_ROWS - 1) / MICRO_ROWS);
    ODIE_REQUIRE(tiles * a.first_blocks < (int64_t(1) << 31), "too many rows for one launch");
    with_micro(dtype, block, whole, [&](auto type, auto b, auto wide) {
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
        const ValuesArgs a{codes, scales, row_scales, groups * rows, int(width), uint32_t(rows), micro_pitch(width), micro_columns(width, block), out};
        const bool whole = wide_rows(out, width, dtype);
        const int n = whole ? 16 / row_type_size(dtype) : 8;  // values_kernel's N
        const int log2 = row_lanes(a.rows, width, n, VALUES_RUNS, whole ? 0 : 3);
        const int64_t blocks = (a.rows + (MICRO_THREADS >> log2) - 1) / (MICRO_THREADS >> log2);
        with_micro(dtype, block, whole, [&](auto type, auto b, auto wide) {
            values_kernel<decltype(type), decltype(b)::value, decltype(wide)::value>
                <<<unsigned(blocks), MICRO_THREADS, 0, reinterpret_cast<cudaStream_t>(stream)>>>(a, log2);
        });
        ODIE_CUDA(cudaGetLastError());
        note_launch();
    });
}
