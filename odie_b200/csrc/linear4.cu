// y = residual + act(q(x) W_g^T + b_g): rows and weights as microscaled 4-bit floats (micro.cuh), one weight matrix or
// one per group of consecutive rows; fp32 sums, one rounding.  x is quantised first, in a kernel of its own, its scales
// cut into tiles from each group's first row on, so that the products load them as they need them.
//
// Rows of no group (behind the last offset) give zero rows of y.
#include "micro.cuh"
#include "odie_b200.h"
#include "product.cuh"
#include <algorithm>
#include <type_traits>

namespace odie {
namespace {

// ---------------------------------------------------------------- the tensor-core product
//
// C = A B^T over tiles of 128 CG x BN, K in blocks of 256 values (128 bytes), by CG CTAs of an SM pair (CG = 2: 256 x
// 256 tiles, each CTA holding its 128 rows of A and half of B's) or one (CG = 1: 128 x 128).
// One warp loads codes (128-byte swizzle) and scales by TMA, STAGES blocks in flight; one thread copies the block's
// scales to TMEM and multiplies (tcgen05 kind::mxf4nvf4, a K-step of 64) into one of two accumulators; sixteen warps
// take the other one to global memory, with the rows' own scales, bias, activation and residual.  A CTA of a pair needs
// the scales of its own rows of A and of all of B's.
//
// TMEM has 512 columns.  A pair's two accumulators of 256 overlap by half ([0, 256) and [128, 384)), which leaves 128
// for two blocks' scales; the epilogue reads the shared half first, and the next tile's products wait for that alone.
constexpr int BK = 256;
constexpr int EPILOGUE_WARP = 4;  // the first one
constexpr int MAX_SHARED = 227 * 1024;
constexpr int AHEAD = 64;         // columns of the residual that are brought to L2 at a time

struct Gemm4Args {
    int groups;
    const int* offsets;  // null: one group of all rows
    long long rows;
    int n;               // outputs
    int k;               // inputs
    int a_rows;          // rows of A's boxes: 128 or, for fewer rows in all, those (rounded up to 8)
    int a_tiles;         // tiles of A's scales that there are
    int most_tiles;      // of the result, with offsets in order: less than 2^30
    int chunk, splits;   // without offsets: the sum over K cut among the CTAs of a cluster, `chunk` blocks each
    Divide by_bands;     // tiles of a full band
    const float* row_scales;     // [rows]
    const float* column_scales;  // [groups][n]
    const void* bias;
    const void* residual;
    void* out;
    int activation;
    bool boxes;          // TMA takes rows of out (every one starts on a 16-byte boundary); boxes_in: of the residual
    bool boxes_in;
    int stages;          // blocks in flight
    int* error;          // on the host: 2 once a wait has run out
    uint32_t limit;      // polls of a wait
};

template <int CG, int BN, int BLOCK>
struct Shape4 {
    static constexpr int TM = 128 * CG;
    static constexpr int B_ROWS = BN / CG;  // per CTA
    static constexpr int COLUMN_TILES = BK / (4 * BLOCK);  // tiles of scales in a block of K: 4 or 2
    static constexpr int A_BYTES = 128 * 128, B_BYTES = B_ROWS * 128;
    static constexpr int SA_BYTES = COLUMN_TILES * MICRO_TILE, SB_BYTES = BN / 128 * SA_BYTES;
    static constexpr int STAGE = A_BYTES + B_BYTES + SA_BYTES + SB_BYTES;
    static constexpr int STAGE_PITCH = (STAGE + 1023) / 1024 * 1024;
    static constexpr int STAGES = CG == 2 ? 4 : 5;  // at most: as many as there is room for beside the groups
    static constexpr int EPILOGUE_WARPS = 16, THREADS = (EPILOGUE_WARP + EPILOGUE_WARPS) * 32;
    static constexpr int COLS = BN / (EPILOGUE_WARPS / 4);  // columns of an epilogue warp's 32 rows: 64 or 32
    static constexpr int BOX = 32 * COLS * 2;               // its rows in shared memory, in bytes, as TMA swizzles them
    static constexpr bool OVERLAP = BN == 256;
    static constexpr int SCALES_AT = OVERLAP ? 384 : 256;  // TMEM column of the scales, 64 per block
    static constexpr int SB_AT = COLUMN_TILES * 4;         // B's behind A's
    static constexpr int COLUMNS = 512;
    // What the epilogue needs to know of a tile, written ahead by a warp of its own: the tile, whether it is one of zeros and
    // whether a scale is far from 1, its rows' scales, its columns' scales (1 if one is far) and bias (of two columns side by
    // side).
    static constexpr int SLOTS = 3, SLOT = 32 + 128 * 4 + BN * 8;
    static constexpr int HEAD = 512;  // barriers, TMEM address
    static int rest(int groups) { return 1024 + EPILOGUE_WARPS * BOX + SLOTS * SLOT + HEAD + 3 * (groups + 2) * 4; }
    static int stages(int groups) { return std::min(STAGES, (MAX_SHARED - rest(groups)) / STAGE_PITCH); }
    static int bytes(int groups) { return rest(groups) + stages(groups) * STAGE_PITCH; }
};

struct Tile4 {
    int g;
    int m0, n0;    // first row and column
    int m_end;     // rows from here on are not stored
    int k0;        // first block of K
    int k_blocks;
    int scales;    // tile of A's scales of row m0
    bool zero;     // nothing to sum: zeros are stored
};

// A role's walk over the tiles, in ascending order (as in linear.cu).
template <int CG, int BN, bool PARTIAL>
struct Walk4 {
    const Gemm4Args& p;
    const int* begin;
    const int* first;
    const int* scales;
    int split;  // PARTIAL: the part of K
    int g = 0;
    __device__ __forceinline__ Walk4(const Gemm4Args& args, const int* b, const int* f, const int* s, int part)
        : p(args), begin(b), first(f), scales(s), split(part) {}
    __device__ __forceinline__ Tile4 at(int t) {
        constexpr int TM = 128 * CG;
        Tile4 tile;
        while (g < p.groups && uniform(first[g + 1]) <= t) ++g;
        tile.g = g;
        const int from = uniform(begin[g]), to = g < p.groups ? uniform(begin[g + 1]) : int(p.rows);
        int local = t - uniform(first[g]);
        const int band = p.by_bands(local), left = (to - from + TM - 1) / TM - band * BAND;
        local -= band * int(p.by_bands.d);
        int n = local / BAND, m = local % BAND;
        if (left < BAND) {  // local < 2^18: the quotient is off by one at most
            n = int((float(local) + 0.5f) * inverse_approx(float(left)));
            m = local - n * left;
            if (m < 0) {
                --n;
                m += left;
            } else if (m >= left) {
                ++n;
                m -= left;
            }
        }
        tile.m0 = from + (band * BAND + m) * TM;
        tile.n0 = n * BN;
        tile.m_end = to;
        tile.k0 = PARTIAL ? split * p.chunk : 0;
        tile.k_blocks = (p.k + BK - 1) / BK;
        if (PARTIAL) tile.k_blocks = min(tile.k_blocks - tile.k0, p.chunk);
        tile.scales = uniform(scales[g]) + (band * BAND + m) * CG;
        tile.zero = g == p.groups;
        return tile;
    }
};

// The 16-byte unit `unit` of a row of a box, as TMA's swizzle of its rows' length (128 or 64 bytes) places it.
template <int COLS>
__device__ __forceinline__ uint4* boxed(char* box, int row, int unit) {
    return reinterpret_cast<uint4*>(box + row * (COLS * 2) + ((COLS == 64 ? unit ^ (row & 7) : unit ^ ((row >> 1) & 3)) << 4));
}
// The same rows moved by the warp itself: where some are outside the matrix, or do not start on 16-byte boundaries.
template <int COLS, bool STORE>
__device__ __forceinline__ void move_box(uint16_t* at, char* box, int ld, int rows, int columns, int lane) {
    constexpr int UNITS = COLS / 8;
    columns = min(columns, COLS);
    if (ld % 8 == 0 && reinterpret_cast<uintptr_t>(at) % 16 == 0) {  // (columns are a multiple of 8 then)
        for (int i = lane; i < rows * UNITS; i += 32) {
            const int r = i / UNITS, u = i % UNITS;
            if (u * 8 >= columns) continue;
            uint4* out = reinterpret_cast<uint4*>(at + (long long)r * ld + u * 8);
            if (STORE) *out = *boxed<COLS>(box, r, u);
            else *boxed<COLS>(box, r, u) = *out;
        }
    } else {
#pragma unroll
        for (int c = lane; c < COLS; c += 32) {
            if (c >= columns) continue;
#pragma unroll 16
            for (int r = 0; r < 32; ++r) {
                if (r >= rows) continue;
                uint16_t* in = reinterpret_cast<uint16_t*>(boxed<COLS>(box, r, c / 8)) + c % 8;
                uint16_t* out = at + (long long)r * ld + c;
                if (STORE) *out = *in;
                else *in = *out;
            }
        }
    }
}

// Of a row's or column's scale (a power of two, or NaN): first second = scale, both near its root.  v r c is taken as
// v (r1 c1) (r2 c2): sums are 0 or between 2^-20 (the least product of codes and e4m3 scales) and 2^42 (2^20 inputs), so that
// no step leaves fp32's range but where the result does.  (v r and r c do: rows of 2^118 by weights of 2^-118, both of 2^-66.)
struct Halves {
    float first, second;
};
__device__ __forceinline__ Halves halves_of_scale(float scale) {
    const int half = (int(__float_as_uint(scale) >> 23 & 255) - 127) >> 1;
    return {power_of_two(half), scale * power_of_two(-half)};
}
__device__ __forceinline__ float scaled(float v, float r, float c) {
    const Halves row = halves_of_scale(r), column = halves_of_scale(c);
    return v * (row.first * column.first) * (row.second * column.second);
}
// Within 2^-63 .. 2^63, or NaN.  Tiles of such rows and columns, all but strange ones, take v r c as (v r) c, which is in range
// then, in the fused step of the bias.
__device__ __forceinline__ bool is_near(float scale) {
    const uint32_t e = __float_as_uint(scale) >> 23 & 255;
    return e - 64u <= 126u || e == 255u;
}

// y = act(v r c + b) (+ residual, in the box), rounded into the box.  A thread has the columns 8 u + 2 (lane % 4) + 0, 1 of
// rows 8 j + lane / 4, as tcgen05.ld 16x256b and the 8 x 8 matrices of ldmatrix and stmatrix have them: c and b are read
// once for four rows.  (With a row to a thread, every thread read every column's: the shared memory was busy with that for
// longer than with the products.)  columns: c and b of two columns side by side.
template <typename T, int ACT, int COLS, bool ADD>
__device__ __forceinline__ void finish_box(const float (&v)[2][COLS / 2], const float (&row_scale)[4], const float* columns, char* box, int lane) {
#pragma unroll
    for (int u = 0; u < COLS / 8; ++u) {
        const float4 cb = *reinterpret_cast<const float4*>(columns + (u * 4 + (lane & 3)) * 4);
        const Pair c = pair(cb.x, cb.y), b = pair(cb.z, cb.w);
        const uint32_t at = tc::smem_u32(boxed<COLS>(box, lane, u));
        uint32_t out[4], in[4];
        if (ADD) tc::load_matrices(at, in);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int e = u * 4 + j % 2 * 2;
            const Pair z = fma2(mul2(pair(v[j / 2][e], v[j / 2][e + 1]), same(row_scale[j])), c, b);
            Pair slope, added{};
            if (ADD) {
                const float2 f = unpack_pair<T>(in[j]);
                added = pair(f.x, f.y);
            }
            const float2 y = both(activate<ACT, ADD>(z, slope, added));
            out[j] = pack_pair<T>(y.x, y.y);
        }
        tc::store_matrices(at, out);
    }
}

__device__ __forceinline__ float activated(int activation, float z, Pair added) {
    Pair slope, y;
    if (activation == ACT_RELU) y = activate<ACT_RELU, true>(same(z), slope, added);
    else if (activation == ACT_SILU) y = activate<ACT_SILU, true>(same(z), slope, added);
    else if (activation == ACT_GELU) y = activate<ACT_GELU, true>(same(z), slope, added);
    else y = activate<ACT_NONE, true>(same(z), slope, added);
    return both(y).x;
}

// A part's sums in shared memory, where its blocks of K were: rows of BN + 4.
template <int BN>
__device__ __forceinline__ float* part_at(char* base, int row, int column) {
    return reinterpret_cast<float*>(base) + row * (BN + 4) + column;
}
// The cluster's parts of a tile to y: a CTA takes every splits-th row.
template <typename T, int BN>
__device__ __forceinline__ void join_parts(const Gemm4Args& p, const Tile4& tile, char* base) {
    const int rank = int(tc::cluster_rank()), rows = min(128, tile.m_end - tile.m0), columns = min(BN, p.n - tile.n0);
    for (int i = threadIdx.x; i < (rows - rank + p.splits - 1) / p.splits * (BN / 4); i += blockDim.x) {
        const int r = rank + i / (BN / 4) * p.splits, c = i % (BN / 4) * 4;
        if (c >= columns) continue;
        float4 z = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        const uint32_t from = tc::smem_u32(part_at<BN>(base, r, c));
#pragma unroll 8
        for (int part = 0; part < p.splits; ++part) {
            const float4 v = tc::load_cluster(from, part);
            z.x += v.x;
            z.y += v.y;
            z.z += v.z;
            z.w += v.w;
        }
        const float by = __ldg(p.row_scales + tile.m0 + r), zs[4] = {z.x, z.y, z.z, z.w};
        const long long at = (long long)(tile.m0 + r) * p.n + tile.n0 + c;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (c + e >= columns) continue;
            const int n = tile.n0 + c + e;
            float y = scaled(zs[e], by, __ldg(p.column_scales + n));
            if (p.bias) y += to_float(static_cast<const T*>(p.bias)[n]);
            const Pair added = same(p.residual ? to_float(static_cast<const T*>(p.residual)[at + e]) : 0.0f);
            static_cast<T*>(p.out)[at + e] = from_float<T>(activated(p.activation, y, added));
        }
    }
}

// PARTIAL: one tile for each cluster, whose CTAs have a part of K each; they lay their sums into shared memory, and each
// finishes a share of the rows from all parts, in their order.
template <typename T, int CG, int BN, int BLOCK, bool PARTIAL>
__global__ void __launch_bounds__(Shape4<CG, BN, BLOCK>::THREADS, 1)
    gemm4_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                 const __grid_constant__ CUtensorMap map_sa, const __grid_constant__ CUtensorMap map_sb,
                 const __grid_constant__ CUtensorMap map_out, const __grid_constant__ CUtensorMap map_residual,
                 const __grid_constant__ CUtensorMap map_ahead, const Gemm4Args p) {
    using S = Shape4<CG, BN, BLOCK>;
    const int stage_count = p.stages;
    extern __shared__ char raw[];
    char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(raw) + 1023) / 1024 * 1024);
    char* stages = smem;
    char* boxes = stages + stage_count * S::STAGE_PITCH;
    char* slots = boxes + S::EPILOGUE_WARPS * S::BOX;
    uint64_t* full = reinterpret_cast<uint64_t*>(slots + S::SLOTS * S::SLOT);
    uint64_t* empty = full + S::STAGES;
    uint64_t* done = empty + S::STAGES; // per accumulator: summed
    uint64_t* drained = done + 2;       // per accumulator: read out (OVERLAP: what it shares with the other one)
    uint64_t* drain = drained + 2;
    uint64_t* arrived = drain + 1;      // per epilogue warp: its rows of the residual
    uint64_t* told = arrived + S::EPILOGUE_WARPS;  // per slot: written
    uint64_t* heard = told + S::SLOTS;             // per slot: read
    uint32_t* tmem_at = reinterpret_cast<uint32_t*>(heard + S::SLOTS);
    uint32_t* gave_up = tmem_at + 1;    // a wait of either CTA has run out
    uint32_t* issued_by = gave_up + 1;  // [2], the leader's: blocks that each CTA has loaded
    int* begin = reinterpret_cast<int*>(reinterpret_cast<char*>(full) + S::HEAD);  // [groups + 2] first row of each group
    int* first = begin + p.groups + 2;                                            // [groups + 2] first tile
    int* scales = first + p.groups + 2;                                           // [groups + 2] first tile of A's scales

    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int rank = CG == 2 ? uniform(tc::cluster_rank()) : 0;
    const int nt = (p.n + BN - 1) / BN;

    if (warp == 0 && lane == 0) {
        for (int s = 0; s < stage_count; ++s) {
            tc::bar_init(full + s, 1);
            tc::bar_init(empty + s, 1);
        }
        for (int a = 0; a < 2; ++a) {
            tc::bar_init(done + a, 1);
            tc::bar_init(drained + a, (S::OVERLAP ? S::EPILOGUE_WARPS / 2 : S::EPILOGUE_WARPS) * CG);
        }
        for (int w = 0; w < S::EPILOGUE_WARPS; ++w) tc::bar_init(arrived + w, 1);
        for (int i = 0; i < S::SLOTS; ++i) {
            tc::bar_init(told + i, 1);
            tc::bar_init(heard + i, S::EPILOGUE_WARPS);
        }
        tc::bar_init(drain, 1);
        tc::fence_bar_init();
        *gave_up = issued_by[0] = issued_by[1] = 0;
    }
    if (warp == 2) tc::tmem_alloc_group<CG>(tmem_at, S::COLUMNS);
    if (warp == 3) {  // the groups' rows, tiles and tiles of scales
        // The sums stop at what offsets in order can come to: others (overlapping groups) have more, up to what passes 32 bits.
        int tiles = 0, units = 0;
        const int most_units = p.a_tiles;
        for (int g0 = 0; g0 <= p.groups; g0 += 32) {
            const int g = g0 + lane;
            int sum = 0, unit_sum = 0;
            if (g <= p.groups) {
                long long from = 0, to = 0;
                if (g < p.groups) {
                    group_rows(p.offsets, g, p.rows, from, to);
                } else {  // the rows of no group
                    long long b;
                    group_rows(p.offsets, p.groups - 1, p.rows, b, from);
                    to = p.rows;
                }
                begin[g] = int(from);
                sum = int((to - from + S::TM - 1) / S::TM) * nt;
                unit_sum = int((to - from + MICRO_ROWS - 1) / MICRO_ROWS);
            }
#pragma unroll
            for (int d = 1; d < 32; d *= 2) {
                const int other = __shfl_up_sync(0xffffffffu, sum, d), other_unit = __shfl_up_sync(0xffffffffu, unit_sum, d);
                if (lane >= d) {
                    sum = min(sum + other, p.most_tiles);
                    unit_sum = min(unit_sum + other_unit, most_units);
                }
            }
            int before = __shfl_up_sync(0xffffffffu, sum, 1), unit_before = __shfl_up_sync(0xffffffffu, unit_sum, 1);
            if (lane == 0) before = unit_before = 0;
            if (g <= p.groups) {
                first[g] = min(tiles + before, p.most_tiles);
                scales[g] = min(units + unit_before, most_units);
            }
            tiles = min(tiles + __shfl_sync(0xffffffffu, sum, 31), p.most_tiles);
            units = min(units + __shfl_sync(0xffffffffu, unit_sum, 31), most_units);
        }
        if (lane == 0) first[p.groups + 1] = tiles;
    }
    tc::fence_before_sync();
    __syncthreads();
    if (CG == 2) tc::cluster_sync();
    tc::fence_after_sync();
    const uint32_t tmem = uniform(*tmem_at);
    const uint32_t full_leader = CG == 2 ? uniform(tc::leader_address(full)) : 0;
    const int units = uniform(first[p.groups + 1]);
    const int tiles = units;
    const int start = PARTIAL ? int(blockIdx.x) / p.splits : int(blockIdx.x) / CG, step = PARTIAL ? units : int(gridDim.x) / CG;
    bool fine = true;
    Walk4<CG, BN, PARTIAL> walk(p, begin, first, scales, PARTIAL ? uniform(tc::cluster_rank()) : 0);

    dependencies_done();  // (all of the above runs beside the end of the kernel that quantises x)
    // The loading and the multiplying warp walk their loops with all lanes, and one lane issues (see linear.cu).
    if (warp == 0) {
        const bool issuer = tc::elect_one();
        const uint32_t stage_bytes = uint32_t(p.a_rows * 128 + S::B_BYTES + S::SA_BYTES + S::SB_BYTES) * CG;
        int s = 0, phase = 1, issued = 0;
        for (int t = start; t < tiles && fine; t += step) {
            const Tile4 tile = walk.at(t);
            if (tile.zero) continue;
            const int m = tile.m0 + rank * 128, n = tile.n0 + rank * S::B_ROWS;
            const int sa = min(tile.scales + rank, p.a_tiles - 1);  // (a pair's second half may have no rows)
            for (int kb = 0; kb < tile.k_blocks; ++kb) {
                fine = __all_sync(0xffffffffu, tc::bar_wait(empty + s, phase, p.limit));
                if (!fine) break;
                if (issuer) {
                    const uint32_t bar = CG == 2 ? full_leader + s * 8 : tc::smem_u32(full + s);
                    if (rank == 0) tc::bar_expect(full + s, stage_bytes);
                    char* a = stages + s * S::STAGE_PITCH;
                    char* b = a + S::A_BYTES;
                    const int k = tile.k0 + kb;
                    tc::tma_load_2d<CG>(a, &map_a, k * 128, m, bar);
                    tc::tma_load_3d<CG>(b, &map_b, k * 128, n, tile.g, bar);
                    tc::tma_load_3d<CG>(b + S::B_BYTES, &map_sa, 0, k * S::COLUMN_TILES, sa, bar);
                    tc::tma_load_4d<CG>(b + S::B_BYTES + S::SA_BYTES, &map_sb, 0, k * S::COLUMN_TILES, tile.n0 / 128, tile.g, bar);
                }
                __syncwarp();
                ++issued;
                if (++s == stage_count) {
                    s = 0;
                    phase ^= 1;
                }
            }
        }
        // every stage read out: no arrival is on its way when the CTA ends, and no copy
        for (int i = 0; i < stage_count && i < issued && fine; ++i) {
            const int last = issued - 1 - i;
            fine = __all_sync(0xffffffffu, tc::bar_wait(empty + last % stage_count, (last / stage_count) & 1, p.limit));
        }
        if (lane == 0) tc::store_leader<CG>(issued_by + rank, issued);
    } else if (warp == 1) {
        if (rank == 0) {
            const bool issuer = tc::elect_one();
            const uint32_t a0 = tc::smem_u32(stages);
            const uint64_t da = tc::sdesc_swizzled(a0, 16), db = tc::sdesc_swizzled(a0 + S::A_BYTES, 16);
            int s = 0, phase = 0, half = 0;  // half: of the TMEM columns for scales
            uint32_t summed = 0;
            for (int t = start; t < tiles && fine; t += step, ++summed) {
                const Tile4 tile = walk.at(t);
                const int blocks = tile.zero ? 0 : tile.k_blocks, acc = summed & 1;
                // the accumulator is free, read out two tiles ago; with OVERLAP its half that the last tile had, too
                if (S::OVERLAP) fine = summed == 0 || __all_sync(0xffffffffu, tc::bar_wait(drained + (acc ^ 1), ((summed - 1) >> 1) & 1, p.limit));
                else fine = __all_sync(0xffffffffu, tc::bar_wait(drained + acc, ((summed >> 1) & 1) ^ 1, p.limit));
                if (!fine) break;
                tc::fence_after_sync();
                const uint32_t to = tmem + acc * 128;
                for (int kb = 0; kb < blocks; ++kb) {
                    fine = __all_sync(0xffffffffu, tc::bar_wait(full + s, phase, p.limit));
                    if (!fine) break;
                    tc::fence_after_sync();
                    if (issuer) {
                        const uint32_t at = s * S::STAGE_PITCH, sa = a0 + at + S::A_BYTES + S::B_BYTES, sb = sa + S::SA_BYTES;
                        const uint32_t scale = tmem + S::SCALES_AT + half * 64;
                        const int left = p.k - (tile.k0 + kb) * BK, steps = min(BK / 64, (left + 63) / 64);
#pragma unroll
                        for (int i = 0; i < S::COLUMN_TILES; ++i) {
                            tc::copy_scales<CG>(scale + i * 4, sa + i * MICRO_TILE);
#pragma unroll
                            for (int j = 0; j < BN / 128; ++j)
                                tc::copy_scales<CG>(scale + S::SB_AT + i * (BN / 32) + j * 4, sb + (j * S::COLUMN_TILES + i) * MICRO_TILE);
                        }
#pragma unroll
                        for (int i = 0; i < BK / 64; ++i) {
                            constexpr int PER = 4 / S::COLUMN_TILES;  // K-steps of a tile of scales
                            if (i < steps)
                                tc::mma_scaled<CG, BLOCK>(to, da + uint64_t(at >> 4) + i * 2, db + uint64_t(at >> 4) + i * 2,
                                                          tc::idesc_scaled<BLOCK>(S::TM, BN, i % PER), scale + i / PER * 4,
                                                          scale + S::SB_AT + i / PER * (BN / 32), kb > 0 || i > 0);
                        }
                        tc::commit_group<CG>(empty + s);
                    }
                    __syncwarp();
                    half ^= 1;
                    if (++s == stage_count) {
                        s = 0;
                        phase ^= 1;
                    }
                }
                if (!fine) break;
                if (issuer) tc::commit_group<CG>(done + acc);
                __syncwarp();
            }
        }
    } else if (warp == 3) {
        // Ahead of the epilogue, whose warps would each wait for these loads, and walk, between two tiles (a third of its
        // time).  The residual is on its way from HBM to L2 meanwhile.
        int q = 0, phase = 1;
        for (int t = start; t < tiles && fine; t += step) {
            const Tile4 tile = walk.at(t);
            float rows[4], columns[BN / 32], bias[BN / 32];
            bool far = false;
            if (!PARTIAL && !tile.zero) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = tile.m0 + rank * 128 + i * 32 + lane;
                    rows[i] = row < tile.m_end ? __ldg(p.row_scales + row) : 1.0f;
                    far |= !is_near(rows[i]);
                }
                const long long at = (long long)tile.g * p.n + tile.n0 + lane;
#pragma unroll
                for (int i = 0; i < BN / 32; ++i) {
                    columns[i] = tile.n0 + lane + i * 32 < p.n ? __ldg(p.column_scales + at + i * 32) : 1.0f;
                    far |= !is_near(columns[i]);
                }
#pragma unroll
                for (int i = 0; i < BN / 32; ++i)
                    bias[i] = p.bias && tile.n0 + lane + i * 32 < p.n ? to_float(static_cast<const T*>(p.bias)[at + i * 32]) : 0.0f;
            }
            far = BLOCK == 16 && __any_sync(0xffffffffu, far);  // (blocks of 32: rows and columns have 1)
            fine = __all_sync(0xffffffffu, tc::bar_wait(heard + q, phase, p.limit));
            if (!fine) break;
            if (!PARTIAL && p.boxes_in && !tile.zero && lane < BN / AHEAD && tile.n0 + lane * AHEAD < p.n)
                tc::tma_prefetch_2d(&map_ahead, tile.n0 + lane * AHEAD, tile.m0 + rank * 128);
            int* slot = reinterpret_cast<int*>(slots + q * S::SLOT);
            if (lane == 0) {
                *reinterpret_cast<int4*>(slot) = make_int4(tile.g, tile.m0, tile.n0, tile.m_end);
                *reinterpret_cast<int4*>(slot + 4) = make_int4(tile.zero, far, 0, 0);
            }
            if (!PARTIAL && !tile.zero) {
                float* to = reinterpret_cast<float*>(slot + 8);
#pragma unroll
                for (int i = 0; i < 4; ++i) to[i * 32 + lane] = rows[i];
                to += 128 + lane / 2 * 4 + lane % 2;
#pragma unroll
                for (int i = 0; i < BN / 32; ++i) {
                    to[i * 64] = far ? 1.0f : columns[i];
                    to[i * 64 + 2] = bias[i];
                }
            }
            __syncwarp();
            if (lane == 0) tc::bar_arrive(told + q);
            if (++q == S::SLOTS) {
                q = 0;
                phase ^= 1;
            }
        }
    } else if (warp >= EPILOGUE_WARP) {
        // Warp (group, quadrant) has rows 32 quadrant + lane and columns COLS group + 0 .. of a tile.  The residual is asked
        // for as soon as the box is free; the box goes out by TMA.
        constexpr int COLS = S::COLS;
        const int index = warp - EPILOGUE_WARP, quadrant = warp & 3, group = index >> 2;
        char* box = boxes + index * S::BOX;
        const uint32_t lanes = tmem + (uint32_t(quadrant * 32) << 16) + group * COLS;
        int q = 0, q_phase = 0;
        uint32_t summed = 0, phase = 0;
        bool asked = false;  // for rows of the residual that have not been awaited
        for (int t = start; t < tiles; t += step, ++summed) {
            fine = __all_sync(0xffffffffu, tc::bar_wait(told + q, q_phase, p.limit));
            if (!fine) break;
            const int* slot = reinterpret_cast<const int*>(slots + q * S::SLOT);
            const int4 first_word = *reinterpret_cast<const int4*>(slot), second_word = *reinterpret_cast<const int4*>(slot + 4);
            Tile4 tile;
            tile.g = uniform(first_word.x);
            tile.m0 = uniform(first_word.y);
            tile.n0 = uniform(first_word.z);
            tile.m_end = uniform(first_word.w);
            tile.zero = uniform(second_word.x);
            const float* column = reinterpret_cast<const float*>(slot + 8) + 128 + group * COLS * 2;
            const int acc = summed & 1;
            const int row = tile.m0 + rank * 128 + quadrant * 32, column0 = tile.n0 + group * COLS;
            const int rows = min(32, tile.m_end - row), columns = p.n - column0;  // inside the matrix
            const bool inside = rows > 0 && columns > 0, whole = rows == 32 && columns > 0;
            const long long at = (long long)row * p.n + column0;
            const bool residual = p.residual && !tile.zero && inside;
            float row_scale[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) row_scale[j] = reinterpret_cast<const float*>(slot + 8)[quadrant * 32 + j * 8 + lane / 4];
            auto ask = [&] {  // for the residual, into the box
                if (lane == 0) tc::stores_read();  // it is free
                __syncwarp();
                if (!residual) return;
                if (whole && p.boxes_in) {
                    if (lane == 0) {
                        tc::fence_async_smem();
                        tc::bar_expect(arrived + index, S::BOX);
                        tc::tma_load_2d<1>(box, &map_residual, column0, row, tc::smem_u32(arrived + index));
                    }
                    asked = true;
                } else {
                    move_box<COLS, false>(static_cast<uint16_t*>(const_cast<void*>(p.residual)) + at, box, p.n, rows, columns, lane);
                }
                __syncwarp();
            };
            if (!PARTIAL) ask();
            fine = __all_sync(0xffffffffu, tc::bar_wait(done + acc, (summed >> 1) & 1, p.limit));
            if (!fine) break;
            tc::fence_after_sync();
            float v[2][COLS / 2];  // (of a tile of nothing: of no use)
            tc::tmem_ld_rows<COLS>(lanes + acc * 128, v[0], v[1]);
            if (!S::OVERLAP || (group >> 1) != acc) {  // with OVERLAP: the half that both accumulators have
                tc::fence_before_sync();
                __syncwarp();
                if (lane == 0) tc::bar_arrive_cluster(CG == 2 ? tc::leader_address(drained + acc) : tc::smem_u32(drained + acc));
            }
            if (PARTIAL) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int u = 0; u < COLS / 8; ++u)
                        *reinterpret_cast<float2*>(part_at<BN>(stages, quadrant * 32 + j * 8 + lane / 4, group * COLS + u * 8 + (lane & 3) * 2)) =
                            make_float2(v[j / 2][u * 4 + j % 2 * 2], v[j / 2][u * 4 + j % 2 * 2 + 1]);
            } else {
                if (asked) {
                    fine = __all_sync(0xffffffffu, tc::bar_wait(arrived + index, phase, p.limit));
                    if (!fine) break;
                    phase ^= 1;
                    asked = false;
                }
                if (BLOCK == 16 && uniform(second_word.y)) {  // far scales: the slot's columns have 1; a lane holds that of every 32nd
                    float by[COLS / 32];
#pragma unroll
                    for (int i = 0; i < COLS / 32; ++i)
                        by[i] = i * 32 + lane < columns ? __ldg(p.column_scales + (long long)tile.g * p.n + column0 + i * 32 + lane) : 1.0f;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const Halves r = halves_of_scale(row_scale[j]);
#pragma unroll
                        for (int i = 0; i < COLS / 4; ++i) {
                            const Halves c = halves_of_scale(__shfl_sync(0xffffffffu, by[i / 8], i / 2 % 4 * 8 + (lane & 3) * 2 + i % 2));
                            float& z = v[j / 2][i / 2 * 4 + j % 2 * 2 + i % 2];
                            z = z * (r.first * c.first) * (r.second * c.second);
                        }
                        row_scale[j] = 1.0f;
                    }
                }
                auto go = [&](auto act) {
                    constexpr int ACT = decltype(act)::value;
                    if (residual) finish_box<T, ACT, COLS, true>(v, row_scale, column, box, lane);
                    else finish_box<T, ACT, COLS, false>(v, row_scale, column, box, lane);
                };
                if (!inside) {
                    // (a tile's rows behind its group, or columns behind the last)
                } else if (tile.zero) {
#pragma unroll
                    for (int u = 0; u < COLS / 8; ++u) *boxed<COLS>(box, lane, u) = make_uint4(0, 0, 0, 0);
                } else if (p.activation == ACT_RELU) go(std::integral_constant<int, ACT_RELU>{});
                else if (p.activation == ACT_SILU) go(std::integral_constant<int, ACT_SILU>{});
                else if (p.activation == ACT_GELU) go(std::integral_constant<int, ACT_GELU>{});
                else go(std::integral_constant<int, ACT_NONE>{});
                if (whole && p.boxes) {
                    tc::fence_async_smem();
                    __syncwarp();
                    if (lane == 0) tc::tma_store_2d(&map_out, column0, row, box);
                } else {
                    __syncwarp();
                    if (inside) move_box<COLS, true>(static_cast<uint16_t*>(p.out) + at, box, p.n, rows, columns, lane);
                    __syncwarp();
                }
            }
            __syncwarp();
            if (lane == 0) tc::bar_arrive(heard + q);
            if (++q == S::SLOTS) {
                q = 0;
                q_phase ^= 1;
            }
        }
        if (asked) tc::bar_wait(arrived + index, phase, WAIT_LIMIT);  // (a wait has run out: no copy is left behind)
        if (lane == 0) tc::stores_done();
        __syncwarp();
    }
    if (!fine && lane == 0) {
        *static_cast<volatile int*>(p.error) = 2;
        __threadfence_system();
        tc::store_both<CG>(gave_up, 1);
    }
    __syncwarp();
    tc::fence_before_sync();
    __syncthreads();
    if (CG == 2) tc::cluster_sync();
    tc::fence_after_sync();
    // Nothing is issued any more.  Had a wait run out, copies and products may still be on their way: they are awaited
    // before the shared memory and the TMEM go.
    if (tc::load_shared(gave_up)) {
        if (warp == 0 && rank == 0) {
            const int mine = int(tc::load_shared(issued_by)), other = CG == 2 ? int(tc::load_shared(issued_by + 1)) : mine;
            const uint32_t share = uint32_t(p.a_rows * 128 + S::B_BYTES + S::SA_BYTES + S::SB_BYTES);  // of one CTA in a block
            for (int b = max(0, max(mine, other) - stage_count); b < max(mine, other); ++b) {
                uint64_t* bar = full + b % stage_count;
                if (lane == 0 && b >= mine) tc::bar_expect(bar, share);
                if (lane == 0 && b >= other) tc::bar_unexpect(bar, share);
                __syncwarp();
                tc::bar_wait(bar, (b / stage_count) & 1, WAIT_LIMIT);
            }
        }
        if (warp == 1) {
            if (rank == 0 && tc::elect_one()) tc::commit_group<CG>(drain);
            __syncwarp();
            tc::bar_wait(drain, 0, WAIT_LIMIT);
        }
        tc::fence_before_sync();
        __syncthreads();
        if (CG == 2) tc::cluster_sync();
        tc::fence_after_sync();
    }
    if constexpr (PARTIAL) {
        tc::cluster_sync();  // all parts are there
        const Tile4 tile = walk.at(start);
        join_parts<T, BN>(p, tile, stages);
        tc::cluster_sync();  // and are not read any more
    }
    if (warp == 2) tc::tmem_dealloc_group<CG>(tmem, S::COLUMNS);
}

// ---------------------------------------------------------------- a few rows
// One kernel for one or two rows (four rows of 4096 -> 4096 took it 14.5 us, the tiles 9.8; two 8.5): bound by the bytes of W
// and by what one launch takes.  A warp has the rows n, n + 32, n + 64 and n + 96 of a tile of W, whose scales lie side by
// side, and every `splits`-th 1024 values of K; the first of them are on their way while the block quantises x into shared
// memory.  Products of codes are multiples of 1/4 of at most 36, and eight of them add up exactly in fp16: a block of 16 takes
// eight packed products and one fp32 step with its scales.  The scales of blocks of 32 may leave fp32's range multiplied, where
// a sum times them does not: their exponents are added and cut into halves, half an exponent a step (kept one bit below its
// place in a float, the sum's upper bits are the half's).
struct Few4Args {
    const void* x;
    const uint8_t* codes;
    const uint8_t* scales;
    const float* row_scales;
    const void* bias;
    const void* residual;
    void* y;
    int rows, inputs, outputs, activation;
    uint32_t pitch, columns;  // of W's codes and scales
    int splits, quads;        // warps that share a sum, and sums (of four rows of W) of a block
    int wide;                 // x starts on a 16-byte boundary, and so do its rows
};

constexpr int FEW4_ROWS = 2, FEW4_VALUES = 1024, FEW4_SHARED = 96 * 1024;
constexpr int FEW4_THREADS = 1024;

template <typename T, int M, int BLOCK>
__global__ void __launch_bounds__(FEW4_THREADS) few4_kernel(Few4Args a) {
    constexpr int WARPS = FEW4_THREADS / 32;
    extern __shared__ char raw[];
    uint8_t* const shared = reinterpret_cast<uint8_t*>(raw);
    __shared__ uint32_t tops[WARPS][M];
    __shared__ float parts[WARPS][4 * M];
    uint8_t* x_codes = shared;                                         // [M][pitch]
    float* x_scales = reinterpret_cast<float*>(shared + M * a.pitch);  // [M][runs], one per block
    const uint32_t runs = a.pitch / 8, per_row = BLOCK == 16 ? runs : runs / 2;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int split = warp % a.splits, quad = blockIdx.x * a.quads + warp / a.splits;
    const int n0 = quad / 32 * MICRO_ROWS + quad % 32;  // the first of the four rows of W
    const bool live = warp / a.splits < a.quads && n0 < a.outputs;
    const uint32_t chunks = (runs * 16 + FEW4_VALUES - 1) / FEW4_VALUES;

    uint4 w[4], s;
    auto fetch = [&](uint32_t chunk) {
        const uint32_t c = chunk * FEW4_VALUES + lane * 32;
        if (!live || chunk >= chunks || c >= runs * 16) return;
#pragma unroll
        for (int q = 0; q < 4; ++q)
            w[q] = n0 + q * 32 < a.outputs ? __ldg(reinterpret_cast<const uint4*>(a.codes + (long long)(n0 + q * 32) * a.pitch + c / 2)) : make_uint4(0, 0, 0, 0);
        s = __ldg(reinterpret_cast<const uint4*>(a.scales + ((long long)(quad / 32) * a.columns + c / (4 * BLOCK)) * MICRO_TILE + quad % 32 * 16));
    };
    fetch(split);

    // q(x)
    Run<T> first[M];
    uint32_t most[M];
    auto load = [&](Run<T>& run, int m, uint32_t u) {
        run = Run<T>{};
        if (m >= a.rows || u >= runs) return;
        const T* row = static_cast<const T*>(a.x) + (long long)m * a.inputs;
        if (a.wide) {
            run.load_wide(row, u * 16, a.inputs);
        } else {
            const uint16_t* at = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int c = int(u) * 16 + 2 * i;
                run.w[i] = (c < a.inputs ? at[c] : 0u) | uint32_t(c + 1 < a.inputs ? at[c + 1] : 0u) << 16;
            }
        }
    };
#pragma unroll
    for (int m = 0; m < M; ++m) {
        load(first[m], m, threadIdx.x);
        most[m] = first[m].largest();
        uint32_t top = most[m];
        for (uint32_t u = threadIdx.x + blockDim.x; u < runs; u += blockDim.x) {
            Run<T> run;
            load(run, m, u);
            top = max(top, run.largest());
        }
        top = __reduce_max_sync(0xffffffffu, top);
        if (lane == 0) tops[warp][m] = top;
    }
    __syncthreads();
    float row_scale[M];
#pragma unroll
    for (int m = 0; m < M; ++m) {
        const uint32_t top = __reduce_max_sync(0xffffffffu, lane < int(blockDim.x >> 5) ? tops[lane][m] : 0u);
        const bool finite = top < 0x7f800000u;
        const int k = BLOCK == 16 && top && finite ? least_power(top, 0x280000u, 11, -126) : 0;
        row_scale[m] = finite ? power_of_two(k) : __int_as_float(0x7fffffff);
        for (uint32_t u0 = 0; u0 < runs; u0 += blockDim.x) {
            const uint32_t u = u0 + threadIdx.x;
            if (u0 + warp * 32 >= runs) break;  // nothing for the whole warp
            if (u0) {
                load(first[m], m, u);
                most[m] = first[m].largest();
            }
            uint32_t largest = most[m], scale = 0;
            if (BLOCK == 32) largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
            uint2 codes = round_run<T, BLOCK>(first[m], finite ? largest : 0u, power_of_two(-k), scale);
            if (!finite) codes = make_uint2(0, 0);
            if (u >= runs) continue;
            *reinterpret_cast<uint2*>(x_codes + m * a.pitch + u * 8) = codes;
            if (BLOCK == 16) x_scales[m * per_row + u] = scale_value<BLOCK>(scale);
            else if (u % 2 == 0) x_scales[m * per_row + u / 2] = __uint_as_float(scale << 22);
        }
    }
    __syncthreads();

    float sum[4][M];
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int m = 0; m < M; ++m) sum[q][m] = 0.0f;
    for (uint32_t chunk = split; chunk < chunks; chunk += a.splits) {
        const uint32_t c = chunk * FEW4_VALUES + lane * 32;
        const uint4 now[4] = {w[0], w[1], w[2], w[3]}, scales = s;
        if (int(chunk + a.splits) < int(chunks)) fetch(chunk + a.splits);
        if (!live || c >= runs * 16) continue;
        const uint32_t words[4][4] = {{now[0].x, now[0].y, now[0].z, now[0].w},
                                      {now[1].x, now[1].y, now[1].z, now[1].w},
                                      {now[2].x, now[2].y, now[2].z, now[2].w},
                                      {now[3].x, now[3].y, now[3].z, now[3].w}};
        const uint32_t bytes[4] = {scales.x, scales.y, scales.z, scales.w};
#pragma unroll
        for (int b = 0; b < 2; ++b) {  // 16 values each
            __half2 x[M][8];
            float by[M];
#pragma unroll
            for (int m = 0; m < M; ++m) {
                const uint2 codes = *reinterpret_cast<const uint2*>(x_codes + m * a.pitch + c / 2 + b * 8);
                halves_of(codes.x, x[m]);
                halves_of(codes.y, x[m] + 4);
                by[m] = x_scales[m * per_row + (BLOCK == 16 ? c / 16 + b : c / 32)];
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                __half2 h[8];
                halves_of(words[q][2 * b], h);
                halves_of(words[q][2 * b + 1], h + 4);
                const uint32_t at = BLOCK == 16 ? (c / 16 + b) % 4 : c / 32 % 4;
                const uint32_t byte = bytes[q] >> (at * 8) & 0xffu;
                const float scale = BLOCK == 16 ? scale_value<BLOCK>(byte) : 0.0f;
#pragma unroll
                for (int m = 0; m < M; ++m) {
                    __half2 dot = __hmul2(h[0], x[m][0]);
#pragma unroll
                    for (int i = 1; i < 8; ++i) dot = __hfma2(h[i], x[m][i], dot);
                    const float2 d = __half22float2(dot);
                    if constexpr (BLOCK == 16) {
                        sum[q][m] = fmaf(d.x + d.y, scale * by[m], sum[q][m]);
                    } else {
                        const uint32_t both_scales = (byte << 22) + __float_as_uint(by[m]);
                        const float half = __uint_as_float(both_scales & 0x7f800000u), other = __uint_as_float((both_scales + 0x400000u) & 0x7f800000u);
                        sum[q][m] = fmaf((d.x + d.y) * half, other, sum[q][m]);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int m = 0; m < M; ++m) {
#pragma unroll
            for (int d = 16; d > 0; d /= 2) sum[q][m] += __shfl_xor_sync(0xffffffffu, sum[q][m], d);
            if (lane == 0) parts[warp][q * M + m] = sum[q][m];
        }
    __syncthreads();
    for (int i = threadIdx.x; i < a.quads * 4 * M; i += blockDim.x) {
        const int part = i / (4 * M), q = i / M % 4, m = i % M, of = blockIdx.x * a.quads + part;
        const int n = of / 32 * MICRO_ROWS + of % 32 + q * 32;
        if (n >= a.outputs || m >= a.rows) continue;
        float z = 0.0f;
        for (int t = 0; t < a.splits; ++t) z += parts[part * a.splits + t][q * M + m];
        float scale = 0.0f;
#pragma unroll
        for (int r = 0; r < M; ++r)
            if (r == m) scale = row_scale[r];
        z = scaled(z, scale, __ldg(a.row_scales + n));
        if (a.bias) z += to_float(static_cast<const T*>(a.bias)[n]);
        const long long at = (long long)m * a.outputs + n;
        const Pair added = same(a.residual ? to_float(static_cast<const T*>(a.residual)[at]) : 0.0f);
        static_cast<T*>(a.y)[at] = from_float<T>(activated(a.activation, z, added));
    }
}

// ---------------------------------------------------------------- host
constexpr int SMS = 148;  // of a B200: the sizes of scratch must not depend on the device that asks

int64_t aligned(int64_t bytes) { return (bytes + 255) / 256 * 256; }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// 256 x 256 tiles by pairs, or 128 x 128 by one CTA where those leave SMs idle: by the waves either takes, in columns, a
// column of the smaller ones for 1.35.  (8192 rows of 4096 -> 4096: 74 us by pairs, 91 by ones; 1024 of 1024 -> 1024: 9.6 and
// 7.9.  Over 128 to 8192 rows, 512 to 8192 outputs, 1024 and 4096 inputs the choice is within 8 % of the better one.  512 rows
// in 32 groups, 1024 -> 2048: 20 us by pairs, 17 by ones.)
bool pair_tiles(int64_t rows, int n, int groups) {
    if (n <= 128 || (groups > 1 && rows < groups * int64_t(128))) return false;
    const int64_t pairs = (groups > 1 ? rows / 256 + (groups + 1) / 2 : ceil_div(rows, 256)) * ceil_div(n, 256);
    const int64_t ones = (groups > 1 ? rows / 128 + (groups + 1) / 2 : ceil_div(rows, 128)) * ceil_div(n, 128);
    return double(ceil_div(std::max<int64_t>(1, pairs), SMS / 2)) * 256 <= double(ceil_div(std::max<int64_t>(1, ones), SMS)) * 128 * 1.35;
}

// Without offsets, where 128 x 128 tiles leave SMs idle: the sum over K is cut into up to 2, 4 or 8 parts, for which it has four
// blocks each; all but the last are of the same, rounded up, number (17 blocks in four: 5, 5, 5, 2; 33 in eight: six of 5, one of 3).
// (512 rows of 1024 -> 2048 in two parts of two blocks: 11.7 us, whole 7.7.  256 rows of 8192 -> 1024 in eight parts, for all
// of whose clusters there is not room at a time: 20.5 us, in four 13.5.  64 rows of 4096 -> 4096: 10.6 us in four parts.)
struct Splits4 {
    int parts, blocks;  // blocks of K per part
    Splits4(int64_t rows, int n, int k, int groups, bool offsets) : parts(1), blocks(int(ceil_div(k, BK))) {
        if (rows == 0 || offsets || pair_tiles(rows, n, groups)) return;
        const int64_t tiles = ceil_div(rows, 128) * ceil_div(n, 128), most = std::min<int64_t>(tiles <= 8 ? 8 : tiles <= 32 ? 4 : tiles <= 64 ? 2 : 1, blocks / 4);
        if (most < 2) return;
        parts = most >= 8 ? 8 : most >= 4 ? 4 : 2;
        blocks = int(ceil_div(blocks, parts));
        parts = int(ceil_div(ceil_div(k, BK), blocks));
    }
};

struct Scratch4 {
    uint8_t *codes, *scales;
    float* row_scales;
    int64_t tiles, bytes = 0;
    Scratch4(void* base, int64_t rows, int inputs, int groups, bool offsets, int block) {
        char* at = static_cast<char*>(base);
        auto take = [&](int64_t size) {
            char* p = at ? at + bytes : nullptr;
            bytes += aligned(size);
            return p;
        };
        tiles = offsets ? micro_tiles(rows, groups) : ceil_div(rows, MICRO_ROWS);
        codes = reinterpret_cast<uint8_t*>(take(rows * micro_pitch(inputs)));
        scales = reinterpret_cast<uint8_t*>(take(tiles * micro_columns(inputs, block) * MICRO_TILE));
        row_scales = reinterpret_cast<float*>(take(rows * 4));
    }
};

// A row-major array, the fastest dimension first, strides in bytes.
CUtensorMap tensor_map(const void* base, CUtensorMapDataType type, CUtensorMapSwizzle swizzle, int rank, const int64_t* dims, const int64_t* strides,
                       const int* box) {
    CUtensorMap map;
    cuuint64_t d[4], s[3];
    cuuint32_t b[4], unit[4] = {1, 1, 1, 1};
    for (int i = 0; i < rank; ++i) {
        d[i] = cuuint64_t(dims[i]);
        b[i] = cuuint32_t(box[i]);
        if (i > 0) s[i - 1] = cuuint64_t(strides[i - 1]);
    }
    ODIE_REQUIRE(uintptr_t(base) % 16 == 0, "codes, scales and scratch must start on 16-byte boundaries");
    const CUresult status = tensor_map_encoder()(&map, type, cuuint32_t(rank), const_cast<void*>(base), d, s, b, unit, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                                                 CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    ODIE_REQUIRE(status == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed with " + std::to_string(int(status)));
    return map;
}

struct Product4 {
    const uint8_t *a, *sa, *b, *sb;
};

template <typename T, int CG, int BN, int BLOCK, bool PARTIAL>
void launch_gemm4(const Product4& x, Gemm4Args p, int64_t tiles, cudaStream_t stream) {
    using S = Shape4<CG, BN, BLOCK>;
    ODIE_REQUIRE(tiles < (int64_t(1) << 30), "too many rows and columns for one launch");
    const int64_t nt = ceil_div(p.n, BN), pitch = micro_pitch(p.k), columns = micro_columns(p.k, BLOCK), row_tiles = ceil_div(p.n, MICRO_ROWS);
    p.by_bands = Divide::by(BAND * nt);
    const int64_t da[] = {pitch, p.rows}, ta[] = {pitch};
    const int xa[] = {128, p.a_rows};
    const CUtensorMap map_a = tensor_map(x.a, CU_TENSOR_MAP_DATA_TYPE_UINT8, CU_TENSOR_MAP_SWIZZLE_128B, 2, da, ta, xa);
    const int64_t db[] = {pitch, p.n, p.groups}, tb[] = {pitch, pitch * p.n};
    const int xb[] = {128, S::B_ROWS, 1};
    const CUtensorMap map_b = tensor_map(x.b, CU_TENSOR_MAP_DATA_TYPE_UINT8, CU_TENSOR_MAP_SWIZZLE_128B, 3, db, tb, xb);
    const int64_t dsa[] = {128, columns, p.a_tiles}, tsa[] = {MICRO_TILE, MICRO_TILE * columns};
    const int xsa[] = {128, S::COLUMN_TILES, 1};
    const CUtensorMap map_sa = tensor_map(x.sa, CU_TENSOR_MAP_DATA_TYPE_UINT32, CU_TENSOR_MAP_SWIZZLE_NONE, 3, dsa, tsa, xsa);
    const int64_t dsb[] = {128, columns, row_tiles, p.groups}, tsb[] = {MICRO_TILE, MICRO_TILE * columns, MICRO_TILE * columns * row_tiles};
    const int xsb[] = {128, S::COLUMN_TILES, BN / 128, 1};
    const CUtensorMap map_sb = tensor_map(x.sb, CU_TENSOR_MAP_DATA_TYPE_UINT32, CU_TENSOR_MAP_SWIZZLE_NONE, 4, dsb, tsb, xsb);

    p.stages = S::stages(p.groups);
    p.most_tiles = int(tiles);
    p.boxes = p.n % 8 == 0 && uintptr_t(p.out) % 16 == 0;
    p.boxes_in = p.residual && p.n % 8 == 0 && uintptr_t(p.residual) % 16 == 0;
    const int64_t dy[] = {p.n, p.rows}, ty[] = {int64_t(p.n) * 2};
    const int xy[] = {S::COLS, 32};
    const auto y_map = [&](bool on, const void* base) {
        return on ? tensor_map(base, CU_TENSOR_MAP_DATA_TYPE_UINT16, S::COLS == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, 2, dy, ty, xy) : CUtensorMap{};
    };
    const CUtensorMap map_out = y_map(p.boxes, p.out), map_residual = y_map(p.boxes_in, p.residual);
    const int xahead[] = {AHEAD, 128};
    const CUtensorMap map_ahead = p.boxes_in ? tensor_map(p.residual, CU_TENSOR_MAP_DATA_TYPE_UINT16, CU_TENSOR_MAP_SWIZZLE_NONE, 2, dy, ty, xahead) : CUtensorMap{};

    const auto kernel = gemm4_kernel<T, CG, BN, BLOCK, PARTIAL>;
    ODIE_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_SHARED));
    cudaLaunchConfig_t config{};
    const unsigned cluster = PARTIAL ? unsigned(p.splits) : CG;
    config.gridDim = dim3(unsigned(PARTIAL ? tiles : std::min<int64_t>(tiles, sm_count() / CG)) * cluster);
    config.blockDim = dim3(S::THREADS);
    config.dynamicSmemBytes = size_t(S::bytes(p.groups));
    config.stream = stream;
    cudaLaunchAttribute attributes[2]{};
    attributes[0].id = cudaLaunchAttributeClusterDimension;
    attributes[0].val.clusterDim.x = cluster;
    attributes[0].val.clusterDim.y = attributes[0].val.clusterDim.z = 1;
    attributes[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[1].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attributes;
    config.numAttrs = 2;
    ODIE_CUDA(cudaLaunchKernelEx(&config, kernel, map_a, map_b, map_sa, map_sb, map_out, map_residual, map_ahead, p));
    note_launch();
}

template <typename T, int BLOCK>
void launch_product4(const Product4& x, Gemm4Args p, const Splits4& split, cudaStream_t stream) {
    const bool pairs = pair_tiles(p.rows, p.n, p.groups);
    p.a_rows = int(std::min<int64_t>(128, (p.rows + 7) / 8 * 8));
    p.splits = 1;
    const int64_t side = pairs ? 256 : 128, tiles = (ceil_div(p.rows, side) + (p.offsets ? p.groups + 1 : 0)) * ceil_div(p.n, side);  // at most
    if (pairs) {
        launch_gemm4<T, 2, 256, BLOCK, false>(x, p, tiles, stream);
    } else if (split.parts == 1) {
        launch_gemm4<T, 1, 128, BLOCK, false>(x, p, tiles, stream);
    } else {
        p.splits = split.parts;
        p.chunk = split.blocks;
        launch_gemm4<T, 1, 128, BLOCK, true>(x, p, tiles, stream);
    }
}

// Whether few4_kernel takes the call: its rows of x have to fit the shared memory.
int64_t few4_shared(int64_t rows, int64_t inputs, int block) {
    const int64_t pitch = micro_pitch(inputs);
    return std::max<int64_t>(1, rows) * (pitch + pitch / 8 * (block == 16 ? 4 : 2));
}
bool few4(int64_t rows, int64_t inputs, bool offsets, int block) {
    return rows <= FEW4_ROWS && !offsets && few4_shared(rows, inputs, block) <= FEW4_SHARED;
}

template <typename T, int BLOCK>
void launch_few4(Few4Args a, cudaStream_t stream) {
    a.pitch = uint32_t(micro_pitch(a.inputs));
    a.columns = uint32_t(micro_columns(a.inputs, BLOCK));
    a.wide = (uintptr_t(a.x) | uintptr_t(a.inputs * 2)) % 16 == 0;
    const int shared = int(few4_shared(a.rows, a.inputs, BLOCK));
    auto go = [&](auto rows) {
        constexpr int M = decltype(rows)::value, WARPS = FEW4_THREADS / 32;
        const int64_t quads = ceil_div(a.outputs, MICRO_ROWS) * 32, chunks = ceil_div(a.inputs, FEW4_VALUES);
        // as many warps to a sum as it has chunks, up to eight, and as many sums to a block as fill the SMs once
        a.splits = int(std::min<int64_t>(chunks, 8));
        a.quads = int(std::min<int64_t>(std::max<int64_t>(1, ceil_div(quads, SMS)), WARPS / a.splits));
        const int threads = std::max(256, a.quads * a.splits * 32);
        const auto kernel = few4_kernel<T, M, BLOCK>;
        ODIE_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, FEW4_SHARED));
        kernel<<<unsigned(ceil_div(quads, a.quads)), threads, shared, stream>>>(a);
        ODIE_CUDA(cudaGetLastError());
        note_launch();
    };
    if (a.rows == 1) go(std::integral_constant<int, 1>{});
    else go(std::integral_constant<int, 2>{});
}

bool sizes4_fit(int64_t rows, int64_t inputs, int64_t outputs, int64_t groups, int block) {
    return rows >= 0 && rows < (int64_t(1) << 31) - 256 && inputs >= 1 && outputs >= 1 && inputs <= (1 << 20) && outputs <= (1 << 20) &&
           groups >= 1 && groups <= 1024 && (block == 16 || block == 32);
}

}  // namespace
}  // namespace odie

using namespace odie;

extern "C" int64_t odie_linear4_scratch(int64_t rows, int inputs, int outputs, int groups, int offsets, int block) {
    if (!sizes4_fit(rows, inputs, outputs, groups, block)) return 0;
    return few4(rows, inputs, offsets, block) ? 0 : Scratch4(nullptr, rows, inputs, groups, offsets, block).bytes;
}

extern "C" int odie_linear4(const void* x, const uint8_t* codes, const uint8_t* scales, const float* row_scales, int block, const void* bias,
                            const void* residual, int64_t rows, int inputs, int outputs, int groups, const int32_t* offsets, int dtype,
                            int activation, void* y, void* scratch, uint64_t stream_handle) {
    return guarded([&] {
        ODIE_REQUIRE(dtype == ROW_F16 || dtype == ROW_BF16, "linear4 takes fp16 (0) or bf16 (1)");
        ODIE_REQUIRE(sizes4_fit(rows, inputs, outputs, groups, block),
                     "0 to 2^31 - 257 rows, 1 to 2^20 inputs and outputs, 1 to 1024 groups, and blocks of 16 or 32");
        ODIE_REQUIRE(offsets || groups == 1, "more than one group needs offsets");
        ODIE_REQUIRE(activation >= ACT_NONE && activation <= ACT_GELU, "activation must be 0 (none), 1 (ReLU), 2 (SiLU) or 3 (GELU)");
        if (rows == 0) return;
        ODIE_REQUIRE(x && codes && scales && row_scales && y, "x, codes, scales, row_scales and y are required");
        ODIE_REQUIRE((uintptr_t(codes) | uintptr_t(scales)) % 16 == 0, "codes and scales must start on 16-byte boundaries");
        const bool few = few4(rows, inputs, offsets, block);
        ODIE_REQUIRE(few || (scratch && uintptr_t(scratch) % 256 == 0), "scratch is required, on a 256-byte boundary");
        int* const error = checked_error_word();
        const cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_handle);
        if (few) {
            const Few4Args f{x, codes, scales, row_scales, bias, residual, y, int(rows), inputs, outputs, activation};
            if (dtype == ROW_BF16) block == 16 ? launch_few4<__nv_bfloat16, 16>(f, stream) : launch_few4<__nv_bfloat16, 32>(f, stream);
            else block == 16 ? launch_few4<__half, 16>(f, stream) : launch_few4<__half, 32>(f, stream);
            return;
        }
        const Scratch4 s(scratch, rows, inputs, groups, offsets, block);
        MicroArgs q{};
        q.x = x;
        q.rows = q.group_rows = rows;
        q.width = inputs;
        q.groups = groups;
        q.offsets = offsets;
        q.codes = s.codes;
        q.scales = s.scales;
        q.row_scales = s.row_scales;
        q.pitch = micro_pitch(inputs);
        q.columns = micro_columns(inputs, block);
        launch_quantize(q, dtype, block, stream);
        Gemm4Args p{};
        p.groups = groups;
        p.offsets = offsets;
        p.rows = rows;
        p.n = outputs;
        p.k = inputs;
        p.a_tiles = int(s.tiles);
        p.row_scales = s.row_scales;
        p.column_scales = row_scales;
        p.bias = bias;
        p.residual = residual;
        p.out = y;
        p.activation = activation;
        p.error = error;
        p.limit = product_wait_limit();
        const Product4 operands{s.codes, s.scales, codes, scales};
        const Splits4 split(rows, outputs, inputs, groups, offsets);
        auto go = [&](auto type) {
            if (block == 16) launch_product4<decltype(type), 16>(operands, p, split, stream);
            else launch_product4<decltype(type), 32>(operands, p, split, stream);
        };
        if (dtype == ROW_BF16) go(__nv_bfloat16{});
        else go(__half{});
    });
}
