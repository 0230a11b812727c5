// y = residual + act(x W^T + b) for one weight matrix, or for one per group of consecutive rows, and its gradient.
//
//   forward    z = x W_g^T + b_g, y = residual + act(z); fp32 sums, one rounding
//   backward   dz = d y act'(z); d x = dz W_g, d W_g = dz^T x over the group's rows, d b_g = sum dz
//
// Rows of no group (behind the last offset) give zero rows of y and d x and add to no gradient.  Training keeps
// act'(z) as a 16-bit fixed-point code (15 fraction bits above -1/4): act' lies in (-0.13, 1.13) for every
// activation here, so the code is within 2^-16 of it absolutely.  (A 16-bit float of it is closer where it is small, fp16
// below 2^-5, bf16 below 2^-8: far in the negative tail a slope keeps few bits, and below 2^-16 none.)  A ReLU keeps
// one bit.
//
// The three products are one tensor-core kernel (gemm_kernel) with another operand order each; see there.  dz is
// rounded to the rows' type, because the tensor cores take 16-bit operands; the bias gradient sums it unrounded.  The
// rounding of dz is as large as that of d x and d W themselves: their error against 64 bits is 1.41 times what it would be
// without (a ReLU's dz is exact).
#include "thin.cuh"
#include "odie_b200.h"
#include "tc.cuh"
#include <cuda.h>
#include <cudaTypedefs.h>
#include <algorithm>
#include <atomic>
#include <initializer_list>
#include <type_traits>

namespace odie {
namespace {

// ---------------------------------------------------------------- the tensor-core product
//
// C = A B^T over tiles of 128 CG x BN, K in blocks of 64, by CG CTAs of an SM pair (CG = 2: tcgen05 cta_group::2,
// each CTA holding its 128 rows of A and half of B's rows; 256 x 256 tiles, twice the arithmetic per byte of
// shared memory) or one (CG = 1: 128 x 128 and 128 x 64 tiles for fewer rows or columns).
//
//   FWD  A = x [rows][inputs] (K-major), B = W_g [outputs][inputs] (K-major), K = inputs
//   DX   A = dz [rows][outputs] (K-major), B = W_g read along its columns (MN-major), K = outputs
//   DW   A = dz, B = x read along their columns (both MN-major), K = the group's rows; C = d W_g
//
// One warp loads (TMA, 128-byte swizzle, STAGES blocks in flight), one thread multiplies into one of two TMEM
// accumulators, sixteen warps take the other one to global memory with bias, activation, residual and slope, so
// that the epilogue of one tile runs beside the products of the next.  Persistent: CTA (pair) i takes tiles i,
// i + grid, ...  Rows of other groups that a tile loads are never stored (FWD, DX); for DW, whose sum runs over
// the rows, each group has its own tensor maps that end at the group's last row, and the hardware reads zeros
// behind it.
enum Mode : int { FWD = 0, DX = 1, DW = 2 };

constexpr int BK = 64;
constexpr int EPILOGUE_WARP = 4;  // the first one
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

struct GemmArgs {
    int groups;
    const int* offsets;  // null: one group of all rows
    long long rows;
    int m;               // DW: outputs (rows of d W)
    int n;               // columns of C
    int k;               // FWD, DX: length of the sum
    int a_rows;          // FWD, DX: rows of A's boxes, 128 or, for fewer rows in all, those (rounded up to 8)
    int chunk;           // DW: rows per unit of work (a multiple of BK); FWD, DX: blocks of K per split
    int units;           // DW: partial sums there is room for (offsets that run backwards would make more)
    int splits;          // FWD, DX without offsets: the sum over K cut among this many tiles, joined by finish_kernel
    Divide by_bands;     // FWD, DX: tiles of a full band
    Divide by_tiles, by_columns;  // tiles of d W (DW) or of C (splits), and of one row of them
    void* out;
    const void* bias;
    const void* residual;
    void* slope;         // null: not kept
    int activation;
    float* partial;      // with several units per tile: [unit][m][n] sums, joined by join_kernel or finish_kernel (m: rows)
    const CUtensorMap* group_maps;  // DW with offsets: [groups][2]
    int* error;          // on the host: 2 once a wait has run out
    uint32_t limit;      // polls of a wait
};

template <int CG, int BN>
struct Shape {
    static constexpr int TM = 128 * CG;
    static constexpr int B_ROWS = BN / CG;  // per CTA
    static constexpr int A_BYTES = 128 * 128, B_BYTES = B_ROWS * 128, STAGE = A_BYTES + B_BYTES;
    static constexpr int STAGES = STAGE < 32768 ? 6 : 5;
    // Sixteen epilogue warps, four per set of 32 TMEM columns (GROUPS) of a tile; tiles of 64 columns are handed out to
    // two such sets in turn (SETS), each with an accumulator of its own.
    static constexpr int EPILOGUE_WARPS = 16, THREADS = (EPILOGUE_WARP + EPILOGUE_WARPS) * 32;
    static constexpr int SETS = BN == 64 ? 2 : 1, GROUPS = EPILOGUE_WARPS / 4 / SETS;
    static constexpr int WINDOWS = BN / 32 / GROUPS;            // per warp and tile: columns 32 (group + GROUPS j)
    static constexpr int ACCUMULATORS = 2;
    static constexpr int WARP_BYTES = STAGING + WINDOWS * 128;  // staging tile and bias of an epilogue warp
    static constexpr int COLUMNS = ACCUMULATORS * BN;  // of TMEM
    static constexpr int HEAD = 1024;       // barriers, TMEM address
    static int bytes(int groups) {
        return 1024 + STAGES * STAGE + EPILOGUE_WARPS * WARP_BYTES + HEAD + (2 * (groups + 2)) * 4;
    }
};

struct Tile {
    int g;
    int m0, n0;          // first row (FWD, DX: global row; DW: output) of the tile and first column
    int m_end;           // rows from here on are not stored
    int k0, k_blocks;    // first value of K of the sum (DW: row); blocks of 64
    int unit;            // index of the partial sum
    bool zero;           // nothing to sum: zeros are stored
};

constexpr int BAND = 16;  // row tiles walked together, so that a W tile serves them from L2

// The same value in every lane, as the compiler sees too.
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

// A role's walk over the tiles, in ascending order: the group is found by stepping on from the last one, and no integer
// division is left (each of twenty warps walks; dividing, they spent four instructions per output element on it).
template <int MODE, int CG, int BN, bool PARTIAL>
struct Walk {
    const GemmArgs& p;
    const int* begin;
    const int* first;
    int g = 0;
    __device__ __forceinline__ Walk(const GemmArgs& args, const int* b, const int* f) : p(args), begin(b), first(f) {}
    __device__ __forceinline__ Tile at(int t) {
        constexpr int TM = 128 * CG;
        Tile tile;
        int key = t, inside = 0, split = 0;
        if (MODE == DW || PARTIAL) {
            key = p.by_tiles(t);
            inside = t - key * int(p.by_tiles.d);
            if (MODE != DW) {
                split = key;
                key = inside;
            }
        }
        while (g < p.groups && uniform(first[g + 1]) <= key) ++g;
        tile.g = g;
        const int from = uniform(begin[g]), to = g < p.groups ? uniform(begin[g + 1]) : int(p.rows);
        int local = key - uniform(first[g]);
        tile.unit = MODE == DW ? key : split;
        if (MODE == DW) {
            tile.k0 = from + local * p.chunk;
            const int rows = max(0, min(to - tile.k0, p.chunk));
            tile.k_blocks = (rows + BK - 1) / BK;
            tile.zero = rows == 0;
            const int m = p.by_columns(inside);
            tile.n0 = (inside - m * int(p.by_columns.d)) * BN;
            tile.m0 = m * TM;
            tile.m_end = p.m;
        } else {
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
            tile.k0 = PARTIAL ? split * p.chunk * BK : 0;
            tile.k_blocks = (p.k + BK - 1) / BK;
            if (PARTIAL) tile.k_blocks = min(tile.k_blocks - split * p.chunk, p.chunk);
            tile.zero = g == p.groups;
        }
        return tile;
    }
};

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

// A row's bits of 32 columns, per lane (rows: of the window inside the matrix, columns: from `column` on).
__device__ __forceinline__ void mask_store(const GemmArgs& p, int row, int column, int rows, int columns, int lane, uint32_t mask) {
    uint8_t* to = static_cast<uint8_t*>(p.slope) + (long long)(row + lane) * ((p.n + 7) / 8) + column / 8;
    if (lane >= rows) return;
    if (columns >= 32 && reinterpret_cast<uintptr_t>(to) % 4 == 0) {
        *reinterpret_cast<uint32_t*>(to) = mask;
    } else {
#pragma unroll
        for (int i = 0; i < 32; i += 8)
            if (i < columns) to[i / 8] = uint8_t(mask >> i & (columns - i < 8 ? (1u << (columns - i)) - 1 : 0xffu));
    }
}

// PARTIAL: the sums go to p.partial as they are, joined by another kernel.
template <typename T, int MODE, int CG, int BN, bool PARTIAL>
__global__ void __launch_bounds__(Shape<CG, BN>::THREADS, 1)
    gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const GemmArgs p) {
    using S = Shape<CG, BN>;
    constexpr int STAGES = S::STAGES;
    extern __shared__ char raw[];
    char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(raw) + 1023) / 1024 * 1024);
    char* stages = smem;
    char* staging = stages + STAGES * S::STAGE;
    uint64_t* full = reinterpret_cast<uint64_t*>(staging + S::EPILOGUE_WARPS * S::WARP_BYTES);
    uint64_t* empty = full + STAGES;
    uint64_t* done = empty + STAGES;                  // per accumulator: summed
    uint64_t* drained = done + S::ACCUMULATORS;       // per accumulator: read out
    uint64_t* drain = drained + S::ACCUMULATORS;
    uint32_t* tmem_at = reinterpret_cast<uint32_t*>(drain + 1);
    uint32_t* gave_up = tmem_at + 1;                  // a wait of either CTA has run out
    uint32_t* issued_by = gave_up + 1;                // [2], the leader's: blocks that each CTA has loaded
    int* begin = reinterpret_cast<int*>(reinterpret_cast<char*>(full) + S::HEAD);  // [groups + 2] first row of each group
    int* first = begin + p.groups + 2;                                            // [groups + 2] first unit

    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int rank = CG == 2 ? uniform(tc::cluster_rank()) : 0;
    const int nt = (p.n + BN - 1) / BN;

    if (warp == 0 && lane == 0) {
        for (int s = 0; s < STAGES; ++s) {
            tc::bar_init(full + s, 1);
            tc::bar_init(empty + s, 1);
        }
        for (int a = 0; a < S::ACCUMULATORS; ++a) {
            tc::bar_init(done + a, 1);
            tc::bar_init(drained + a, S::EPILOGUE_WARPS / S::SETS * CG);
        }
        tc::bar_init(drain, 1);
        tc::fence_bar_init();
        *gave_up = issued_by[0] = issued_by[1] = 0;
    }
    if (warp == 2) tc::tmem_alloc_group<CG>(tmem_at, S::COLUMNS);
    if (warp == 3) {  // the groups' rows and units
        int units = 0;
        for (int g0 = 0; g0 <= p.groups; g0 += 32) {
            const int g = g0 + lane;
            int count = 0;
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
                if (MODE == DW) count = g == p.groups ? 0 : max(1, int((to - from + p.chunk - 1) / p.chunk));
                else count = int((to - from + S::TM - 1) / S::TM) * nt;
            }
            int sum = count;
#pragma unroll
            for (int d = 1; d < 32; d *= 2) {
                const int other = __shfl_up_sync(0xffffffffu, sum, d);
                if (lane >= d) sum += other;
            }
            if (g <= p.groups) first[g] = units + sum - count;
            units += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (lane == 0) first[p.groups + 1] = units;
    }
    tc::fence_before_sync();
    __syncthreads();
    if (CG == 2) tc::cluster_sync();
    tc::fence_after_sync();
    const uint32_t tmem = uniform(*tmem_at);
    const uint32_t full_leader = CG == 2 ? uniform(tc::leader_address(full)) : 0;
    const int units = uniform(first[p.groups + 1]);
    const int tiles = MODE == DW ? units * nt * ((p.m + S::TM - 1) / S::TM) : PARTIAL ? units * p.splits : units;
    const int start = int(blockIdx.x) / CG, step = int(gridDim.x) / CG;
    bool fine = true;
    Walk<MODE, CG, BN, PARTIAL> walk(p, begin, first);

    // The loading and the multiplying warp walk their loops with all lanes and values that are the same in every lane,
    // and one lane issues: the operands of these instructions live in uniform registers.  (With one lane in the loops,
    // each of them was moved there first: 575 cycles a block, more than the products take.)
    if (warp == 0) {
        const bool issuer = tc::elect_one();
        const uint32_t stage_bytes = (MODE == DW ? S::STAGE : p.a_rows * 128 + S::B_BYTES) * CG;
        int s = 0, phase = 1, issued = 0;
        for (int t = start; t < tiles && fine; t += step) {
            const Tile tile = walk.at(t);
            if (tile.zero) continue;
            const void* ma = &map_a;
            const void* mb = &map_b;
            if (MODE == DW && p.group_maps) {
                ma = p.group_maps + 2 * tile.g;
                mb = p.group_maps + 2 * tile.g + 1;
                asm volatile("fence.proxy.tensormap::generic.acquire.gpu [%0], 128;" ::"l"(ma) : "memory");
                asm volatile("fence.proxy.tensormap::generic.acquire.gpu [%0], 128;" ::"l"(mb) : "memory");
            }
            const int m = tile.m0 + rank * 128, n = tile.n0 + rank * S::B_ROWS;
            for (int kb = 0; kb < tile.k_blocks; ++kb) {
                fine = __all_sync(0xffffffffu, tc::bar_wait(empty + s, phase, p.limit));
                if (!fine) break;
                if (issuer) {
                    const uint32_t bar = CG == 2 ? full_leader + s * 8 : tc::smem_u32(full + s);
                    if (rank == 0) tc::bar_expect(full + s, stage_bytes);
                    char* a = stages + s * S::STAGE;
                    char* b = a + S::A_BYTES;
                    const int k = tile.k0 + kb * BK;
                    if (MODE == DW) {
#pragma unroll
                        for (int i = 0; i < 2; ++i) tc::tma_load_2d<CG>(a + i * 8192, ma, m + 64 * i, k, bar);
#pragma unroll
                        for (int i = 0; i < S::B_ROWS / 64; ++i)
                            tc::tma_load_2d<CG>(b + i * 8192, mb, n + 64 * i, k, bar);
                    } else {
                        tc::tma_load_2d<CG>(a, ma, k, m, bar);
                        if (MODE == FWD) {
                            tc::tma_load_3d<CG>(b, mb, k, n, tile.g, bar);
                        } else {
#pragma unroll
                            for (int i = 0; i < S::B_ROWS / 64; ++i)
                                tc::tma_load_3d<CG>(b + i * 8192, mb, n + 64 * i, k, tile.g, bar);
                        }
                    }
                }
                __syncwarp();
                ++issued;
                if (++s == STAGES) {
                    s = 0;
                    phase ^= 1;
                }
            }
        }
        // every stage read out: no arrival is on its way when the CTA ends, and no copy
        for (int i = 0; i < STAGES && i < issued && fine; ++i) {
            const int last = issued - 1 - i;
            fine = __all_sync(0xffffffffu, tc::bar_wait(empty + last % STAGES, (last / STAGES) & 1, p.limit));
        }
        if (lane == 0) tc::store_leader<CG>(issued_by + rank, issued);
    } else if (warp == 1) {
        if (rank == 0) {
            constexpr int A_MN = MODE == DW, B_MN = MODE != FWD;
            constexpr uint32_t ID = std::is_same<T, __half>::value ? tc::idesc(S::TM, BN, A_MN, B_MN) : tc::idesc_bf16(S::TM, BN, A_MN, B_MN);
            constexpr uint64_t A_STEP = (A_MN ? 2048 : 32) >> 4, B_STEP = (B_MN ? 2048 : 32) >> 4;
            const bool issuer = tc::elect_one();
            const uint32_t a0 = tc::smem_u32(stages);
            const uint64_t da = tc::sdesc_swizzled(a0, A_MN ? 8192 : 16), db = tc::sdesc_swizzled(a0 + S::A_BYTES, B_MN ? 8192 : 16);
            int s = 0, phase = 0, acc = 0, acc_phase = 1;
            for (int t = start; t < tiles && fine; t += step) {
                const Tile tile = walk.at(t);
                const int blocks = tile.zero ? 0 : tile.k_blocks;
                fine = __all_sync(0xffffffffu, tc::bar_wait(drained + acc, acc_phase, p.limit));
                if (!fine) break;
                tc::fence_after_sync();
                for (int kb = 0; kb < blocks; ++kb) {
                    fine = __all_sync(0xffffffffu, tc::bar_wait(full + s, phase, p.limit));
                    if (!fine) break;
                    tc::fence_after_sync();
                    if (issuer) {
                        const uint64_t at = uint64_t(s * (S::STAGE >> 4));
#pragma unroll
                        for (int i = 0; i < BK / 16; ++i)
                            tc::mma_group<CG>(tmem + acc * BN, da + at + i * A_STEP, db + at + i * B_STEP, ID, kb > 0 || i > 0);
                        tc::commit_group<CG>(empty + s);
                    }
                    __syncwarp();
                    if (++s == STAGES) {
                        s = 0;
                        phase ^= 1;
                    }
                }
                if (!fine) break;
                if (issuer) tc::commit_group<CG>(done + acc);
                __syncwarp();
                if (++acc == S::ACCUMULATORS) {
                    acc = 0;
                    acc_phase ^= 1;
                }
            }
        }
    } else if (warp >= EPILOGUE_WARP) {
        constexpr int WINDOWS = S::WINDOWS, STRIDE = 32 * S::GROUPS;
        const int quadrant = warp & 3, group = ((warp - EPILOGUE_WARP) >> 2) % S::GROUPS;
        const int set = ((warp - EPILOGUE_WARP) >> 2) / S::GROUPS;
        char* stage = staging + (warp - EPILOGUE_WARP) * STAGING;
        float* bias = reinterpret_cast<float*>(staging + S::EPILOGUE_WARPS * STAGING) + (warp - EPILOGUE_WARP) * WINDOWS * 32;
        const uint32_t lanes = tmem + (uint32_t(quadrant * 32) << 16);
        const bool wide = p.n % 8 == 0 && (reinterpret_cast<uintptr_t>(p.out) | (p.activation == ACT_RELU ? 0 : reinterpret_cast<uintptr_t>(p.slope))) % 16 == 0;
        const bool wide_residual = p.n % 8 == 0 && reinterpret_cast<uintptr_t>(p.residual) % 16 == 0;
        int bias_g = -1, bias_n0 = -1;  // whose bias is held
        uint32_t summed = set;
        for (int t = start + set * step; t < tiles && fine; t += S::SETS * step, summed += S::SETS) {
            const Tile tile = walk.at(t);
            const int acc = summed % S::ACCUMULATORS;
            const int row = tile.m0 + rank * 128 + quadrant * 32, column0 = tile.n0 + group * 32;
            const long long at = (MODE == DW ? (long long)tile.g * p.m * p.n : 0) + (long long)row * p.n + column0;
            const uint16_t* residual = MODE == FWD && !PARTIAL && p.residual && !tile.zero ? static_cast<const uint16_t*>(p.residual) + at : nullptr;
            Window w{p.n, min(32, tile.m_end - row), p.n - column0, wide};
            Window wr{p.n, w.rows, w.columns, wide_residual};
            uint4 r[4];
            if (MODE == FWD && !PARTIAL && !tile.zero) {  // what does not need the sum is read while it is awaited
                if (residual) {
                    if (wr.wide) window_load(residual, wr, lane, r);
                    else window_fetch(residual, wr, lane, stage);
                }
                if (tile.g != bias_g || tile.n0 != bias_n0) {
                    bias_g = tile.g;
                    bias_n0 = tile.n0;
#pragma unroll
                    for (int j = 0; j < WINDOWS; ++j)
                        bias[j * 32 + lane] = p.bias && j * STRIDE + lane < w.columns
                                              ? to_float(static_cast<const T*>(p.bias)[(long long)tile.g * p.n + column0 + j * STRIDE + lane])
                                              : 0.0f;
                    __syncwarp();
                }
            }
            fine = __all_sync(0xffffffffu, tc::bar_wait(done + acc, (summed / S::ACCUMULATORS) & 1, p.limit));
            if (!fine) break;
            tc::fence_after_sync();
#pragma unroll 1
            for (int j = 0; j < WINDOWS; ++j) {
                const bool last = j + 1 == WINDOWS || w.columns <= STRIDE;  // of this warp's windows inside the matrix
                if (w.columns <= 0 && j > 0) break;
                float v[32];
                uint32_t codes[16];
                if (tile.zero) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = 0.0f;
#pragma unroll
                    for (int i = 0; i < 16; ++i) codes[i] = 0;
                } else {
                    tc::tmem_ld32(lanes + acc * BN + group * 32 + j * STRIDE, v);
                }
                if (last) {  // the accumulator is free as soon as it is in registers
                    tc::fence_before_sync();
                    __syncwarp();
                    if (lane == 0) tc::bar_arrive_cluster(CG == 2 ? tc::leader_address(drained + acc) : tc::smem_u32(drained + acc));
                }
                if (PARTIAL) {
                    if (lane < w.rows && (MODE != DW || tile.unit < p.units)) {
                        float* to = p.partial + ((long long)tile.unit * p.m + row + lane) * p.n + column0 + j * STRIDE;
                        if (p.n % 4 == 0) {
#pragma unroll
                            for (int i = 0; i < 32; i += 4)
                                if (i < w.columns) *reinterpret_cast<float4*>(to + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                if (i < w.columns) to[i] = v[i];
                        }
                    }
                    w.columns -= STRIDE;
                    continue;
                }
                if (MODE == FWD && tile.zero && p.slope && p.activation == ACT_RELU) mask_store(p, row, column0 + j * STRIDE, w.rows, w.columns, lane, 0);
                if (MODE == FWD && !tile.zero) {
                    if (residual) {
                        if (wr.wide) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) *staged(stage, lane / 4 + 8 * i, lane & 3) = r[i];
                            wr.columns -= STRIDE;
                            if (j + 1 < WINDOWS && wr.columns > 0) window_load(residual + (j + 1) * STRIDE, wr, lane, r);
                        } else {
                            if (j > 0) window_fetch(residual + j * STRIDE, wr, lane, stage);
                            wr.columns -= STRIDE;
                        }
                        __syncwarp();
                    }
                    if (p.activation == ACT_RELU) {
                        const uint32_t mask = finish_relu(v, bias + j * 32);
                        if (p.slope) mask_store(p, row, column0 + j * STRIDE, w.rows, w.columns, lane, mask);
                    } else if (p.activation == ACT_SILU) finish<ACT_SILU>(v, codes, bias + j * 32);
                    else if (p.activation == ACT_GELU) finish<ACT_GELU>(v, codes, bias + j * 32);
                    else finish<ACT_NONE>(v, codes, bias + j * 32);
                    if (residual) {
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            const uint4 q = *staged(stage, lane, u);
                            const uint32_t e[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const float2 f = unpack_pair<T>(e[i]);
                                v[u * 8 + i * 2] += f.x;
                                v[u * 8 + i * 2 + 1] += f.y;
                            }
                        }
                        __syncwarp();
                    }
                }
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    *staged(stage, lane, u) = make_uint4(pack_pair<T>(v[u * 8], v[u * 8 + 1]), pack_pair<T>(v[u * 8 + 2], v[u * 8 + 3]),
                                                         pack_pair<T>(v[u * 8 + 4], v[u * 8 + 5]), pack_pair<T>(v[u * 8 + 6], v[u * 8 + 7]));
                __syncwarp();
                window_store(static_cast<uint16_t*>(p.out) + at + j * STRIDE, w, lane, stage);
                __syncwarp();
                if (MODE == FWD && p.slope && p.activation != ACT_RELU) {
#pragma unroll
                    for (int u = 0; u < 4; ++u)
                        *staged(stage, lane, u) = make_uint4(codes[u * 4], codes[u * 4 + 1], codes[u * 4 + 2], codes[u * 4 + 3]);
                    __syncwarp();
                    window_store(static_cast<uint16_t*>(p.slope) + at + j * STRIDE, w, lane, stage);
                    __syncwarp();
                }
                w.columns -= STRIDE;
            }
        }
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
            const uint32_t share = MODE == DW ? S::STAGE : p.a_rows * 128 + S::B_BYTES;  // of one CTA in a block
            for (int b = max(0, max(mine, other) - STAGES); b < max(mine, other); ++b) {
                uint64_t* bar = full + b % STAGES;
                if (lane == 0 && b >= mine) tc::bar_expect(bar, share);
                if (lane == 0 && b >= other) tc::bar_unexpect(bar, share);
                __syncwarp();
                tc::bar_wait(bar, (b / STAGES) & 1, WAIT_LIMIT);
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
    if (warp == 2) tc::tmem_dealloc_group<CG>(tmem, S::COLUMNS);
}

// Tensor maps of dz and x that end at each group's last row.
__global__ void __launch_bounds__(32) group_maps_kernel(const __grid_constant__ CUtensorMap a, const __grid_constant__ CUtensorMap b,
                                                        const int* offsets, long long rows, CUtensorMap* maps) {
    __shared__ alignas(128) uint32_t map[32];
    const int g = blockIdx.x >> 1;
    const CUtensorMap& from = blockIdx.x & 1 ? b : a;
    map[threadIdx.x] = reinterpret_cast<const uint32_t*>(&from)[threadIdx.x];
    __syncwarp();
    if (threadIdx.x == 0) {
        long long begin, end;
        group_rows(offsets, g, rows, begin, end);
        asm volatile("tensormap.replace.tile.global_dim.shared::cta.b1024.b32 [%0], 1, %1;" ::"r"(tc::smem_u32(map)),
                     "r"(int(max(1ll, end)))
                     : "memory");
    }
    __syncwarp();
    asm volatile("tensormap.cp_fenceproxy.global.shared::cta.tensormap::generic.release.gpu.sync.aligned [%0], [%1], 128;" ::"l"(
                     maps + blockIdx.x),
                 "r"(tc::smem_u32(map))
                 : "memory");
}

// d W from the units' sums: a block per 32 x WIDTH elements (WIDTH 4 where sizes and pointers allow), each warp over its
// share of the units, the shares in order.  A unit holds `size` sums of d W and `bias` sums of d b (either may be
// unwanted: null).
template <typename T, int WIDTH>
__global__ void __launch_bounds__(256) join_kernel(const float* partial, T* d_weight, T* d_bias, const int* offsets, long long rows,
                                                   int chunk, long long units, long long size, int bias) {
    __shared__ float part[8][32 * WIDTH + 1];
    const int g = blockIdx.y, lane = threadIdx.x & 31, line = threadIdx.x >> 5;
    long long begin, end;
    int before = 0;  // units of earlier groups
    for (int i = lane; i < g; i += 32) {
        group_rows(offsets, i, rows, begin, end);
        before += int(max(1ll, (end - begin + chunk - 1) / chunk));
    }
    const long long unit = __reduce_add_sync(0xffffffffu, before);
    group_rows(offsets, g, rows, begin, end);
    // no more than were written: offsets that run backwards would make more
    const int count = int(max(0ll, min(units - unit, max(1ll, (end - begin + chunk - 1) / chunk)))), share = (count + 7) / 8;
    const int from = min(count, line * share), last = min(count, from + share);
    const long long all = size + bias;
    for (long long i0 = (long long)blockIdx.x * (32 * WIDTH); i0 < all; i0 += (long long)gridDim.x * (32 * WIDTH)) {
        const long long i = i0 + lane * WIDTH;
        T* to = i < size ? (d_weight ? d_weight + g * size + i : nullptr) : i < all && d_bias ? d_bias + (long long)g * bias + (i - size) : nullptr;
        float sum[WIDTH];
#pragma unroll
        for (int e = 0; e < WIDTH; ++e) sum[e] = 0.0f;
        if (to) {
            const float* at = partial + (unit + from) * all + i;
#pragma unroll 8
            for (int u = from; u < last; ++u, at += all) {
                if constexpr (WIDTH == 4) {
                    const float4 v = __ldg(reinterpret_cast<const float4*>(at));
                    sum[0] += v.x;
                    sum[1] += v.y;
                    sum[2] += v.z;
                    sum[3] += v.w;
                } else {
                    sum[0] += __ldg(at);
                }
            }
        }
#pragma unroll
        for (int e = 0; e < WIDTH; ++e) part[line][lane * WIDTH + e] = sum[e];
        __syncthreads();
        if (line == 0 && to) {
#pragma unroll
            for (int w = 1; w < 8; ++w)
#pragma unroll
                for (int e = 0; e < WIDTH; ++e) sum[e] += part[w][lane * WIDTH + e];
            if constexpr (WIDTH == 4) *reinterpret_cast<uint2*>(to) = make_uint2(pack_pair<T>(sum[0], sum[1]), pack_pair<T>(sum[2], sum[3]));
            else *to = from_float<T>(sum[0]);
        }
        __syncthreads();
    }
}

// The sums over parts of K, in order, with the epilogue of the products (DX: neither bias, residual nor activation).
// Rows of threads are padded to eight columns.
struct FinishArgs {
    const float* partial;  // [splits][rows][n]
    int splits;
    long long rows;
    int n;
    const void* bias;
    const void* residual;
    void* out;
    void* slope;
    int activation;
};
template <typename T>
__global__ void __launch_bounds__(256) finish_kernel(FinishArgs a) {
    const int pitch = (a.n + 7) / 8;
    // (K is cut only where there are fewer tiles than SMs, so that 32 bits hold the padded count)
    const unsigned unit = blockIdx.x * 256 + threadIdx.x, line = unit / unsigned(pitch * 8);
    const int column = int(unit - line * unsigned(pitch * 8));
    const long long row = line;
    const bool inside = row < a.rows && column < a.n;
    const long long at = row * a.n + column;
    float z = 0.0f;
    if (inside) {
#pragma unroll 8
        for (int s = 0; s < a.splits; ++s) z += __ldg(a.partial + s * a.rows * a.n + at);
        if (a.bias) z += to_float(static_cast<const T*>(a.bias)[column]);
        const Pair added = same(a.residual ? to_float(static_cast<const T*>(a.residual)[at]) : 0.0f);
        Pair slope, y;
        if (a.activation == ACT_RELU) y = activate<ACT_RELU, true>(same(z), slope, added);
        else if (a.activation == ACT_SILU) y = activate<ACT_SILU, true>(same(z), slope, added);
        else if (a.activation == ACT_GELU) y = activate<ACT_GELU, true>(same(z), slope, added);
        else y = activate<ACT_NONE, true>(same(z), slope, added);
        static_cast<T*>(a.out)[at] = from_float<T>(both(y).x);
        if (a.slope && a.activation != ACT_RELU) static_cast<uint16_t*>(a.slope)[at] = uint16_t(slope_codes(slope));
    }
    if (a.slope && a.activation == ACT_RELU) {  // eight lanes have a byte
        const uint32_t on = __ballot_sync(0xffffffffu, inside && !(z <= 0.0f));
        if (inside && column % 8 == 0) static_cast<uint8_t*>(a.slope)[row * pitch + column / 8] = uint8_t(on >> (threadIdx.x & 24));
    }
}

// ---------------------------------------------------------------- dz and the bias gradient
struct DzArgs {
    const void* d_y;
    const void* kept;       // the slope that forward kept
    void* dz;               // null: not wanted
    void* d_residual;       // null: not wanted
    void* d_bias;           // null: not wanted
    float* partial;         // [unit][n] sums of dz, joined by join_kernel; null: one unit, which writes d_bias itself
    long long rows;
    int n;
    long long ld;           // of dz
    int chunk;              // rows per unit
    int groups;
    const int* offsets;
};

// A block: one unit of rows (of one group, or of none) x COLUMNS columns per thread of `lanes` threads: eight, or one
// where rows do not start on 16-byte boundaries.  Column sums: each thread over its rows, the lanes of a warp in a
// tree, the warps in order.
template <typename T, int COLUMNS, int THREADS, int KIND>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? 5 : 1) dz_kernel(DzArgs a, int lanes_log2) {
    constexpr int WARPS = THREADS / 32;
    __shared__ float sums[WARPS][32 * COLUMNS];
    const Unit u = unit_at<true>(a.offsets, a.groups, a.rows, a.chunk, blockIdx.x);
    if (u.g < 0) return;
    const int lanes = 1 << lanes_log2, lane = threadIdx.x & (lanes - 1), line = threadIdx.x >> lanes_log2, lines = THREADS >> lanes_log2;
    const int column = (blockIdx.y * lanes + lane) * COLUMNS;
    const bool live = u.g < a.groups;
    const int mask_pitch = (a.n + 7) / 8;
    float sum[COLUMNS];
#pragma unroll
    for (int i = 0; i < COLUMNS; ++i) sum[i] = 0.0f;
    if (column < a.n) {
#pragma unroll COLUMNS == 8 ? 4 : 8
        for (long long row = u.from + line; row < u.to; row += lines) {
            const long long at = row * a.n + column;
            if constexpr (COLUMNS == 8) {
                const uint4 d = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.d_y) + at));
                uint4 k = make_uint4(0, 0, 0, 0);
                if (KIND == SLOPE_CODES) k = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.kept) + at));
                if (KIND == SLOPE_MASK) k.x = __ldg(static_cast<const uint8_t*>(a.kept) + row * mask_pitch + column / 8);
                const uint32_t ds[4] = {d.x, d.y, d.z, d.w}, ks[4] = {k.x, k.y, k.z, k.w};
                uint32_t z[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float2 f = unpack_pair<T>(ds[i]);
                    if (KIND == SLOPE_CODES) {
                        f.x *= slope_value(ks[i] & 0xffffu);
                        f.y *= slope_value(ks[i] >> 16);
                    } else if (KIND == SLOPE_MASK) {
                        f.x = k.x >> (2 * i) & 1 ? f.x : 0.0f;
                        f.y = k.x >> (2 * i + 1) & 1 ? f.y : 0.0f;
                    }
                    z[i] = pack_pair<T>(f.x, f.y);
                    sum[2 * i] += f.x;
                    sum[2 * i + 1] += f.y;
                }
                if (a.dz) *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.dz) + row * a.ld + column) = make_uint4(z[0], z[1], z[2], z[3]);
                if (a.d_residual)
                    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.d_residual) + at) = live ? d : make_uint4(0, 0, 0, 0);
            } else {
                const uint16_t d = static_cast<const uint16_t*>(a.d_y)[at];
                float f = unpack_pair<T>(d).x;
                if (KIND == SLOPE_CODES) f *= slope_value(static_cast<const uint16_t*>(a.kept)[at]);
                if (KIND == SLOPE_MASK) f = static_cast<const uint8_t*>(a.kept)[row * mask_pitch + column / 8] >> (column & 7) & 1 ? f : 0.0f;
                if (a.dz) static_cast<T*>(a.dz)[row * a.ld + column] = from_float<T>(f);
                if (a.d_residual) static_cast<uint16_t*>(a.d_residual)[at] = live ? d : uint16_t(0);
                sum[0] += f;
            }
        }
    }
    if (!a.d_bias || !live) return;
#pragma unroll
    for (int i = 0; i < COLUMNS; ++i) {
#pragma unroll
        for (int d = 16; d > 0; d /= 2) {
            const float other = __shfl_xor_sync(0xffffffffu, sum[i], d);
            if (d >= lanes) sum[i] += other;
        }
    }
    if ((threadIdx.x & 31) < lanes) {
#pragma unroll
        for (int i = 0; i < COLUMNS; ++i) sums[threadIdx.x >> 5][(threadIdx.x & 31) * COLUMNS + i] = sum[i];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < lanes * COLUMNS; i += THREADS) {
        const int at = blockIdx.y * lanes * COLUMNS + i;
        if (at >= a.n) continue;
        float total = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) total += sums[w][i];
        if (a.partial) a.partial[(long long)u.index * a.n + at] = total;
        else static_cast<T*>(a.d_bias)[(long long)u.g * a.n + at] = from_float<T>(total);
    }
}

// Rows whose length is no multiple of 16 bytes, copied to ones that are, zeros behind: TMA reads no others.  Two
// matrices of one width in one launch.
__global__ void __launch_bounds__(256) pad_kernel(const uint16_t* from0, uint16_t* to0, long long rows0, const uint16_t* from1,
                                                  uint16_t* to1, long long rows1, int width, int ld) {
    const int units = ld / 8;
    const long long count = (rows0 + rows1) * units;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < count; i += (long long)gridDim.x * 256) {
        long long row = i / units;
        const int c = int(i % units) * 8;
        const uint16_t* from = row < rows0 ? from0 : from1;
        uint16_t* to = row < rows0 ? to0 : to1;
        if (row >= rows0) row -= rows0;
        uint16_t e[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = c + j < width ? from[row * width + c + j] : uint16_t(0);
        *reinterpret_cast<uint4*>(to + row * ld + c) = make_uint4(e[0] | uint32_t(e[1]) << 16, e[2] | uint32_t(e[3]) << 16,
                                                                  e[4] | uint32_t(e[5]) << 16, e[6] | uint32_t(e[7]) << 16);
    }
}

// ---------------------------------------------------------------- a few rows
// One or two rows: y is bound by the bytes of W, which every warp reads straight into registers, 16 vectors in flight
// per lane: one row of W (one output) of up to 16 x 32 vectors, or four short ones.  x comes through shared memory
// meanwhile.  (The tensor-core tiles, 128 rows each, take 11.5 us for 4096 x 4096 bf16 however few the rows, this 6.7
// for one and 9.3 for two.  Widening x to fp32 first, or cutting K among a block's warps, left fewer vectors in flight
// and took 10 to 12 us.)
struct FewArgs {
    const void* x;
    const void* weight;
    const void* bias;
    const void* residual;
    void* y;
    void* slope;
    int rows, inputs, outputs;  // rows: M
    int activation;
};

constexpr int FEW_ROWS = 2, FEW_VECTORS = 16;

// M: rows; V: vectors per lane of one row of W at a time; MASK: a ReLU's bits are kept (the block has whole bytes).
template <typename T, int BYTES, int M, int V, int THREADS, bool MASK>
__global__ void __launch_bounds__(THREADS) few_rows_kernel(FewArgs a) {
    using P = Pack<T, BYTES>;
    constexpr int COLUMNS = FEW_VECTORS / V, CHUNK = 32 * P::N * V;  // CHUNK: values of K at a time
    constexpr int BLOCK = THREADS / 32 * COLUMNS;  // columns of the block
    static_assert(!MASK || BLOCK % 8 == 0, "whole bytes");
    __shared__ alignas(16) T xs[M][CHUNK];
    __shared__ bool on[M][BLOCK];
    const int lane = threadIdx.x & 31, n0 = blockIdx.x * BLOCK + (threadIdx.x >> 5) * COLUMNS;
    const T* w = static_cast<const T*>(a.weight);
    const T* x = static_cast<const T*>(a.x);
    float sum[COLUMNS][M];
#pragma unroll
    for (int c = 0; c < COLUMNS; ++c)
#pragma unroll
        for (int m = 0; m < M; ++m) sum[c][m] = 0.0f;
    for (int k0 = 0; k0 < a.inputs; k0 += CHUNK) {
        P v[COLUMNS][V];
#pragma unroll
        for (int c = 0; c < COLUMNS; ++c)
#pragma unroll
            for (int u = 0; u < V; ++u) {
                const int k = k0 + (u * 32 + lane) * P::N;
                v[c][u] = k < a.inputs ? P::load_once(w + (long long)min(n0 + c, a.outputs - 1) * a.inputs + k) : P::zero();
            }
        const int count = min(CHUNK, a.inputs - k0) / P::N;
        if (k0 > 0) __syncthreads();
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll 4
            for (int i = threadIdx.x; i < CHUNK / P::N; i += THREADS) {
                const P q = i < count ? P::load(x + (long long)m * a.inputs + k0 + i * P::N) : P::zero();
                q.store(&xs[m][i * P::N]);
            }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < V; ++u)
#pragma unroll
            for (int m = 0; m < M; ++m) {
                P q;
                *reinterpret_cast<typename Raw<BYTES>::type*>(&q) = *reinterpret_cast<const typename Raw<BYTES>::type*>(&xs[m][(u * 32 + lane) * P::N]);
#pragma unroll
                for (int c = 0; c < COLUMNS; ++c)
#pragma unroll
                    for (int e = 0; e < P::N; ++e) sum[c][m] = fmaf(to_float(v[c][u].v[e]), to_float(q.v[e]), sum[c][m]);
            }
    }
#pragma unroll
    for (int c = 0; c < COLUMNS; ++c) {
        const int n = n0 + c;
        float mine = 0.0f;
#pragma unroll
        for (int m = 0; m < M; ++m) {
#pragma unroll
            for (int d = 16; d > 0; d /= 2) sum[c][m] += __shfl_xor_sync(0xffffffffu, sum[c][m], d);
            if (lane == m) mine = sum[c][m];
        }
        if (MASK && lane < M) on[lane][n - blockIdx.x * BLOCK] = false;
        if (lane >= M || n >= a.outputs) continue;
        const long long at = (long long)lane * a.outputs + n;
        if (a.bias) mine += to_float(static_cast<const T*>(a.bias)[n]);
        const Pair z = same(mine), added = same(a.residual ? to_float(static_cast<const T*>(a.residual)[at]) : 0.0f);
        Pair slope, y;
        if (a.activation == ACT_RELU) y = activate<ACT_RELU, true>(z, slope, added);
        else if (a.activation == ACT_SILU) y = activate<ACT_SILU, true>(z, slope, added);
        else if (a.activation == ACT_GELU) y = activate<ACT_GELU, true>(z, slope, added);
        else y = activate<ACT_NONE, true>(z, slope, added);
        static_cast<T*>(a.y)[at] = from_float<T>(both(y).x);
        if (MASK) on[lane][n - blockIdx.x * BLOCK] = !(mine <= 0.0f);
        else if (a.slope) static_cast<uint16_t*>(a.slope)[at] = uint16_t(slope_codes(slope));
    }
    if constexpr (MASK) {
        __syncthreads();
        const int pitch = (a.outputs + 7) / 8, m = threadIdx.x / (BLOCK / 8), b = threadIdx.x % (BLOCK / 8), at = blockIdx.x * (BLOCK / 8) + b;
        if (m < M && at < pitch) {
            uint32_t bits = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) bits |= on[m][b * 8 + e] ? 1u << e : 0u;
            static_cast<uint8_t*>(a.slope)[m * pitch + at] = uint8_t(bits);
        }
    }
}

// ---------------------------------------------------------------- host
std::atomic<uint32_t> wait_limit{WAIT_LIMIT};

// The word of the current device in which its kernels leave 2 when a wait has run out: pinned host memory, so that the
// next call can look at it without waiting for the device.
constexpr int MAX_DEVICES = 64;
int* error_word() {
    static int* const words = [] {
        void* p = nullptr;
        // (the first call may come while a graph is captured, which an allocation does not concern)
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
        ODIE_CUDA(cudaThreadExchangeStreamCaptureMode(&mode));
        const cudaError_t status = cudaHostAlloc(&p, MAX_DEVICES * sizeof(int), cudaHostAllocPortable | cudaHostAllocMapped);
        cudaThreadExchangeStreamCaptureMode(&mode);
        ODIE_CUDA(status);
        std::fill_n(static_cast<int*>(p), MAX_DEVICES, 0);
        return static_cast<int*>(p);
    }();
    int device = 0;
    ODIE_CUDA(cudaGetDevice(&device));
    ODIE_REQUIRE(device < MAX_DEVICES, "at most 64 devices");
    return words + device;
}

// Refuses once after a wait has run out.
int* checked_error_word() {
    int* word = error_word();
    if (__atomic_load_n(word, __ATOMIC_RELAXED) != 0 && __atomic_exchange_n(word, 0, __ATOMIC_RELAXED) != 0)
        throw std::runtime_error("a wait of an earlier linear call on this device ran out: that call's results are incomplete");
    return word;
}

PFN_cuTensorMapEncodeTiled_v12000 encoder() {
    static const PFN_cuTensorMapEncodeTiled_v12000 found = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult status;
        ODIE_CUDA(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &status));
        ODIE_REQUIRE(f && status == cudaDriverEntryPointSuccess, "the driver has no cuTensorMapEncodeTiled");
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
    }();
    return found;
}

// A row-major [depth][rows][width] matrix of 16-bit elements with rows of ld elements; boxes of 64 columns x box_rows.
CUtensorMap tensor_map(const void* base, bool bf16, int64_t width, int64_t rows, int64_t depth, int64_t ld, int box_rows) {
    CUtensorMap map;
    const cuuint64_t dims[3] = {cuuint64_t(width), cuuint64_t(rows), cuuint64_t(std::max<int64_t>(1, depth))};
    const cuuint64_t strides[2] = {cuuint64_t(ld * 2), cuuint64_t(rows * ld * 2)};
    const cuuint32_t box[3] = {64, cuuint32_t(box_rows), 1}, unit[3] = {1, 1, 1};
    ODIE_REQUIRE(uintptr_t(base) % 16 == 0, "x, weight, d_y and scratch must start on 16-byte boundaries");
    const CUresult status = encoder()(&map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, depth ? 3 : 2,
                                      const_cast<void*>(base), dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    ODIE_REQUIRE(status == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed with " + std::to_string(int(status)));
    return map;
}

int64_t aligned(int64_t bytes) { return (bytes + 255) / 256 * 256; }
int64_t round8(int64_t n) { return (n + 7) / 8 * 8; }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

void check_linear(int64_t rows, int inputs, int outputs, int groups, const int32_t* offsets, int dtype, int activation) {
    ODIE_REQUIRE(dtype == ROW_F16 || dtype == ROW_BF16, "linear takes fp16 (0) or bf16 (1)");
    ODIE_REQUIRE(rows >= 0 && rows < (int64_t(1) << 31) - 256, "0 to 2^31 - 257 rows");
    ODIE_REQUIRE(inputs >= 1 && outputs >= 1 && inputs <= (1 << 20) && outputs <= (1 << 20), "1 to 2^20 inputs and outputs");
    ODIE_REQUIRE(groups >= 1 && groups <= 1024, "1 to 1024 groups");
    ODIE_REQUIRE(offsets || groups == 1, "more than one group needs offsets");
    ODIE_REQUIRE(activation >= ACT_NONE && activation <= ACT_GELU, "activation must be 0 (none), 1 (ReLU), 2 (SiLU) or 3 (GELU)");
}

template <typename F>
void with_linear_type(int dtype, F&& f) {
    if (dtype == ROW_BF16) f(__nv_bfloat16{});
    else f(__half{});
}

constexpr int SMS = 148;  // of a B200: the sizes of scratch must not depend on the device that asks

// The tile shape: the one whose waves over the SMs (or SM pairs) take the least time, in columns of 128 rows per CTA.
// The factors are what narrower tiles cost more per column, with less arithmetic per byte from L2 (input gradient of
// 16384 x 2048 -> 8192 bf16: 256 x 256 by pairs 1491 TFLOP/s, 128 x 128 1082, 128 x 64 699; weight gradient 1335, 1105,
// 694; 256 x 128 by pairs took a fifth longer than 256 x 256 and saved no wave there).
struct Config {
    int cg, bn;
};
Config tile_config(int64_t m, int n, int64_t groups, bool groups_share_m) {
    if (n <= 64) return {1, 64};
    Config best{};
    double least = 0;
    for (const auto& [config, factor] : {std::pair<Config, double>{{2, 256}, 1.0}, {{1, 128}, 1.35}, {{1, 64}, 2.0}}) {
        const int rows = 128 * config.cg;
        // several groups in m rows: each leaves half a tile on average
        const int64_t row_tiles = groups_share_m && groups > 1 ? m / rows + (groups + 1) / 2 : ceil_div(m, rows) * (groups_share_m ? 1 : groups);
        const double cost = double(ceil_div(std::max<int64_t>(1, row_tiles) * ceil_div(n, config.bn), SMS / config.cg)) * config.bn * factor;
        if (!best.cg || cost < least) {
            best = config;
            least = cost;
        }
    }
    return best;
}
template <typename F>
void with_config(Config c, F&& f) {
    if (c.cg == 2) f(std::integral_constant<int, 2>{}, std::integral_constant<int, 256>{});
    else if (c.bn == 128) f(std::integral_constant<int, 1>{}, std::integral_constant<int, 128>{});
    else f(std::integral_constant<int, 1>{}, std::integral_constant<int, 64>{});
}

template <typename T, int MODE, int CG, int BN, bool PARTIAL>
void launch_gemm(const CUtensorMap& a, const CUtensorMap& b, GemmArgs p, int64_t tiles, cudaStream_t stream) {
    ODIE_REQUIRE(tiles < (int64_t(1) << 30), "too many rows and columns for one launch");
    const int64_t nt = ceil_div(p.n, BN);
    p.by_bands = Divide::by(BAND * nt);
    p.by_columns = Divide::by(nt);
    p.by_tiles = Divide::by(nt * ceil_div(MODE == DW ? p.m : p.rows, 128 * CG));

    using S = Shape<CG, BN>;
    const auto kernel = gemm_kernel<T, MODE, CG, BN, PARTIAL>;
    ODIE_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::bytes(1024)));
    const int pairs = int(std::min<int64_t>(tiles, sm_count() / CG));
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(unsigned(pairs * CG));
    config.blockDim = dim3(S::THREADS);
    config.dynamicSmemBytes = size_t(S::bytes(p.groups));
    config.stream = stream;
    cudaLaunchAttribute cluster{};
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = CG;
    cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    config.attrs = &cluster;
    config.numAttrs = 1;
    ODIE_CUDA(cudaLaunchKernelEx(&config, kernel, a, b, p));
    note_launch();
}

void launch_pad(const void* from0, void* to0, int64_t rows0, const void* from1, void* to1, int64_t rows1, int width, cudaStream_t stream) {
    const int ld = int(round8(width));
    const int64_t blocks = std::min<int64_t>(ceil_div((rows0 + rows1) * (ld / 8), 256), 32 * sm_count());
    pad_kernel<<<unsigned(blocks), 256, 0, stream>>>(static_cast<const uint16_t*>(from0), static_cast<uint16_t*>(to0), rows0,
                                                     static_cast<const uint16_t*>(from1), static_cast<uint16_t*>(to1), rows1, width, ld);
    ODIE_CUDA(cudaGetLastError());
    note_launch();
}

template <typename T>
void launch_few_rows(const FewArgs& a, cudaStream_t stream) {
    const int vector = row_vector(a.inputs, ROW_F16, a.x, a.weight);
    auto go = [&](auto bytes, auto rows) {
        constexpr int B = decltype(bytes)::value, M = decltype(rows)::value;
        constexpr int SHORT = 4 * 32 * (B / 2);  // values of four vectors per lane
        auto launch = [&](auto v, auto threads, auto mask) {
            constexpr int V = decltype(v)::value, THREADS = decltype(threads)::value, BLOCK = THREADS / 32 * (FEW_VECTORS / V);
            few_rows_kernel<T, B, M, V, THREADS, decltype(mask)::value><<<unsigned(ceil_div(a.outputs, BLOCK)), THREADS, 0, stream>>>(a);
        };
        using std::integral_constant;
        const bool mask = a.slope && a.activation == ACT_RELU;
        if (a.inputs <= SHORT && mask) launch(integral_constant<int, 4>{}, integral_constant<int, 128>{}, std::true_type{});
        else if (a.inputs <= SHORT) launch(integral_constant<int, 4>{}, integral_constant<int, 128>{}, std::false_type{});
        else if (mask) launch(integral_constant<int, FEW_VECTORS>{}, integral_constant<int, 256>{}, std::true_type{});
        else launch(integral_constant<int, FEW_VECTORS>{}, integral_constant<int, 128>{}, std::false_type{});
    };
    auto with_rows = [&](auto bytes) {
        if (a.rows == 1) go(bytes, std::integral_constant<int, 1>{});
        else go(bytes, std::integral_constant<int, 2>{});
    };
    if (vector == 16) with_rows(std::integral_constant<int, 16>{});
    else if (vector == 4) with_rows(std::integral_constant<int, 4>{});
    else with_rows(std::integral_constant<int, 2>{});
    ODIE_CUDA(cudaGetLastError());
    note_launch();
}

template <typename T>
void launch_join(const float* partial, void* d_weight, void* d_bias, const int* offsets, int groups, int64_t rows, int64_t chunk,
                 int64_t units, int64_t size, int bias, cudaStream_t stream) {
    const bool wide = size % 4 == 0 && bias % 4 == 0 && (uintptr_t(d_weight) | uintptr_t(d_bias)) % 8 == 0;
    const dim3 grid(unsigned(std::min<int64_t>(ceil_div(size + bias, wide ? 128 : 32), 16384)), unsigned(groups));
    auto go = [&](auto kernel) {
        kernel<<<grid, 256, 0, stream>>>(partial, static_cast<T*>(d_weight), static_cast<T*>(d_bias), offsets, rows, int(chunk), units, size, bias);
    };
    if (wide) go(join_kernel<T, 4>);
    else go(join_kernel<T, 1>);
    ODIE_CUDA(cudaGetLastError());
    note_launch();
}

// Caller-owned scratch, handed out in 256-byte steps.
struct Scratch {
    char* at;
    int64_t used = 0;
    void* take(int64_t bytes) {
        char* p = at ? at + used : nullptr;
        used += aligned(bytes);
        return p;
    }
};

bool on_16_bytes(std::initializer_list<const void*> pointers) {
    uintptr_t bits = 0;
    for (const void* p : pointers) bits |= uintptr_t(p);
    return bits % 16 == 0;
}

// FWD, DX of one group without offsets: where the tiles leave SMs idle, the sum over K is cut into as many parts as
// there are SMs for (64 rows of 4096 -> 4096 bf16: 24 us in 64 tiles).
struct Splits {
    int parts, blocks;  // blocks of K per part
    Splits(int64_t rows, int n, int k, int groups, bool offsets) : parts(1), blocks(int(ceil_div(k, BK))) {
        if (rows == 0 || offsets) return;
        const Config c = tile_config(rows, n, groups, true);
        if (c.cg != 1) return;
        const int64_t tiles = ceil_div(rows, 128) * ceil_div(n, c.bn), wanted = std::min<int64_t>(SMS / tiles, blocks / 8);
        if (wanted < 2) return;
        blocks = int(ceil_div(blocks, wanted));
        parts = int(ceil_div(ceil_div(k, BK), blocks));
    }
    int64_t bytes(int64_t rows, int n) const { return parts > 1 ? parts * rows * n * 4 : 0; }
};

template <typename T, int MODE>
void launch_product(const void* a, const void* b, int64_t ld_a, int64_t ld_b, int outputs, int inputs, GemmArgs p, const Splits& split,
                    float* partial, cudaStream_t stream) {
    const bool bf16 = std::is_same<T, __nv_bfloat16>::value;
    if (split.parts > 1) {
        p.splits = split.parts;
        p.chunk = split.blocks;
        p.partial = partial;
        p.m = int(p.rows);
    }
    // (boxes of 128 rows over a matrix of fewer than 16 were twice as slow: 16 us against 9 for 15 and 16 rows of
    // 4096 -> 4096; what the rest of the tile holds only reaches rows that are not stored)
    p.a_rows = int(std::min<int64_t>(128, round8(p.rows)));
    with_config(tile_config(p.rows, p.n, p.groups, true), [&](auto cg, auto bn) {
        constexpr int CG = decltype(cg)::value, BN = decltype(bn)::value;
        const CUtensorMap map_a = tensor_map(a, bf16, p.k, p.rows, 0, ld_a, p.a_rows);
        const CUtensorMap map_b = tensor_map(b, bf16, inputs, outputs, p.groups, ld_b, MODE == FWD ? BN / CG : 64);
        const int64_t tiles = (ceil_div(p.rows, 128 * CG) + p.groups + 1) * ceil_div(p.n, BN) * split.parts;
        if constexpr (CG == 1) {
            if (split.parts > 1) return launch_gemm<T, MODE, CG, BN, true>(map_a, map_b, p, tiles, stream);
        }
        launch_gemm<T, MODE, CG, BN, false>(map_a, map_b, p, tiles, stream);
    });
    if (split.parts > 1) {
        const FinishArgs f{partial, split.parts, p.rows, p.n, p.bias, p.residual, p.out, p.slope, p.activation};
        finish_kernel<T><<<unsigned(ceil_div(p.rows * ceil_div(p.n, 8) * 8, 256)), 256, 0, stream>>>(f);
        ODIE_CUDA(cudaGetLastError());
        note_launch();
    }
}

// ---- the pieces of scratch, in order; the size functions walk the same list
struct ForwardScratch {
    void *x, *weight;
    float* partial;
    int64_t bytes;
    ForwardScratch(void* base, int64_t rows, int inputs, int outputs, int groups) {
        Scratch s{static_cast<char*>(base)};
        const bool pad = inputs % 8 != 0;
        x = pad ? s.take(rows * round8(inputs) * 2) : nullptr;
        weight = pad ? s.take(int64_t(groups) * outputs * round8(inputs) * 2) : nullptr;
        partial = static_cast<float*>(s.take(Splits(rows, outputs, inputs, groups, groups > 1).bytes(rows, outputs)));
        bytes = s.used;
    }
};

// DW: the rows of a unit of work.  Where there are fewer tiles than SMs, the rows are cut so that about two units
// fall to each.
struct WeightUnits {
    Config config;
    int64_t tiles;  // of one group
    int64_t chunk, units;
    bool split;
    WeightUnits(int64_t rows, int inputs, int outputs, int groups) {
        config = tile_config(outputs, inputs, groups, false);
        tiles = ceil_div(outputs, 128 * config.cg) * ceil_div(inputs, config.bn);
        const int64_t wanted = 2 * SMS / config.cg, have = tiles * groups;
        chunk = std::max<int64_t>(BK, ceil_div(rows, BK) * BK);
        split = have < wanted / 2 && rows > 32 * BK;  // a second kernel joins the sums: 2048 rows are walked sooner
        if (split) chunk = std::max<int64_t>(8 * BK, ceil_div(ceil_div(rows * tiles, wanted), BK) * BK);
        // a unit is at most 2^20 rows: its sum (7 ms) ends well before the epilogue's wait for it would give up
        if (rows > (1 << 20)) {
            split = true;
            chunk = std::min<int64_t>(chunk, 1 << 20);
        }
        units = split ? ceil_div(rows, chunk) + groups : groups;  // at most
    }
};

// Rows per unit of dz.  One group of up to 4096 rows is one unit, in blocks of 1024 threads: no second kernel joins
// its sums.  Else 64 to 1024 rows, so that a group's sums are few and the blocks many.
bool dz_single(int64_t rows, int groups) { return rows <= 4096 && groups == 1; }
int64_t dz_chunk(int64_t rows, int groups) {
    if (dz_single(rows, groups)) return std::max<int64_t>(1, rows);
    return std::max<int64_t>(64, std::min<int64_t>(1024, ceil_div(ceil_div(rows, int64_t(16) * groups), 64) * 64));
}
int64_t dz_units(int64_t rows, int groups) { return ceil_div(rows, dz_chunk(rows, groups)) + groups + 1; }

template <typename T>
void launch_dz(const DzArgs& a, int kind, cudaStream_t stream) {
    const bool wide = a.n % 8 == 0 && (uintptr_t(a.d_y) | (kind == SLOPE_CODES ? uintptr_t(a.kept) : 0) | uintptr_t(a.d_residual)) % 16 == 0;
    const bool single = dz_single(a.rows, a.groups);
    const int columns = wide ? 8 : 1;
    int log2 = 0;
    while (log2 < (single && wide ? 1 : 5) && (columns << log2) < a.n) ++log2;
    while (ceil_div(a.n, columns << log2) > 65535) ++log2;  // one unit of 2^20 outputs: four threads a row, not two
    const dim3 grid(unsigned(dz_units(a.rows, a.groups)), unsigned(ceil_div(a.n, columns << log2)));
    auto go = [&](auto k) {
        constexpr int KIND = decltype(k)::value;
        if (single && wide) dz_kernel<T, 8, 1024, KIND><<<grid, 1024, 0, stream>>>(a, log2);
        else if (single) dz_kernel<T, 1, 1024, KIND><<<grid, 1024, 0, stream>>>(a, log2);
        else if (wide) dz_kernel<T, 8, 256, KIND><<<grid, 256, 0, stream>>>(a, log2);
        else dz_kernel<T, 1, 256, KIND><<<grid, 256, 0, stream>>>(a, log2);
    };
    if (kind == SLOPE_MASK) go(std::integral_constant<int, SLOPE_MASK>{});
    else if (kind == SLOPE_CODES) go(std::integral_constant<int, SLOPE_CODES>{});
    else go(std::integral_constant<int, SLOPE_ONE>{});
    ODIE_CUDA(cudaGetLastError());
    note_launch();
}

struct BackwardScratch {
    void *dz, *x, *weight, *maps;
    float *bias, *partial, *split, *thin;
    int64_t bytes;
    BackwardScratch(void* base, int64_t rows, int inputs, int outputs, int groups) {
        Scratch s{static_cast<char*>(base)};
        const bool pad = inputs % 8 != 0;
        dz = s.take(rows * round8(outputs) * 2);
        x = pad ? s.take(rows * round8(inputs) * 2) : nullptr;
        weight = pad ? s.take(int64_t(groups) * outputs * round8(inputs) * 2) : nullptr;
        maps = s.take(int64_t(groups) * 2 * sizeof(CUtensorMap));
        bias = static_cast<float*>(s.take(dz_units(rows, groups) * outputs * 4));
        const WeightUnits u(rows, inputs, outputs, groups);
        partial = static_cast<float*>(u.split ? s.take(u.units * outputs * int64_t(inputs) * 4) : nullptr);
        split = static_cast<float*>(s.take(Splits(rows, inputs, outputs, groups, groups > 1).bytes(rows, inputs)));
        bytes = s.used;
        thin = static_cast<float*>(base);  // thin layers need nothing else
    }
    // (the activation whose units are most)
    static int64_t thin_bytes(int64_t rows, int inputs, int outputs, int groups) {
        return aligned(thin_units(rows, groups, thin_chunk(rows, inputs, outputs, ACT_NONE, true)) * (int64_t(outputs) * inputs + outputs) * 4);
    }
};

// The kernels that serve a forward pass (thin.cu decides a ReLU's corner, so one or two thin rows with a ReLU go there);
// a backward pass takes THIN or TILES.
enum class Path { FEW, THIN, TILES };
Path forward_path(int64_t rows, int inputs, int outputs, bool offsets, int activation, bool on_16) {
    const bool thin = thin_sizes(inputs, outputs) && on_16;
    if (rows <= FEW_ROWS && !offsets && !(thin && activation == ACT_RELU)) return Path::FEW;
    return thin ? Path::THIN : Path::TILES;
}
Path backward_path(int inputs, int outputs, bool on_16) { return thin_sizes(inputs, outputs) && on_16 ? Path::THIN : Path::TILES; }

bool sizes_fit(int64_t rows, int inputs, int outputs, int groups) {
    return rows >= 0 && rows < (int64_t(1) << 31) && inputs >= 1 && outputs >= 1 && inputs <= (1 << 20) && outputs <= (1 << 20) &&
           groups >= 1 && groups <= 1024;
}

}  // namespace
}  // namespace odie

using namespace odie;

extern "C" int64_t odie_linear_scratch_for(int64_t rows, int inputs, int outputs, int groups, int offsets, int on_16) {
    if (!sizes_fit(rows, inputs, outputs, groups)) return 0;
    return forward_path(rows, inputs, outputs, offsets, ACT_NONE, on_16) == Path::TILES ? ForwardScratch(nullptr, rows, inputs, outputs, groups).bytes : 0;
}

extern "C" int64_t odie_linear_scratch(int64_t rows, int inputs, int outputs, int groups) {
    return odie_linear_scratch_for(rows, inputs, outputs, groups, 1, 0);
}

extern "C" int odie_linear(const void* x, const void* weight, const void* bias, const void* residual, int64_t rows, int inputs,
                           int outputs, int groups, const int32_t* offsets, int dtype, int activation, void* y,
                           void* slope, void* scratch, uint64_t stream_handle) {
    return guarded([&] {
        check_linear(rows, inputs, outputs, groups, offsets, dtype, activation);
        if (rows == 0) return;
        ODIE_REQUIRE(x && weight && y, "x, weight and y are required");
        int* const error = checked_error_word();
        if (activation == ACT_NONE) slope = nullptr;  // 1 everywhere
        const cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_handle);
        const Path path = forward_path(rows, inputs, outputs, offsets, activation,
                                       on_16_bytes({x, weight, residual, y, activation == ACT_RELU ? nullptr : slope}));
        if (path == Path::FEW) {
            const FewArgs a{x, weight, bias, residual, y, slope, int(rows), inputs, outputs, activation};
            with_linear_type(dtype, [&](auto type) { launch_few_rows<decltype(type)>(a, stream); });
            return;
        }
        if (path == Path::THIN) {
            ThinArgs a{};
            a.rows = rows;
            a.inputs = inputs;
            a.outputs = outputs;
            a.groups = groups;
            a.offsets = offsets;
            a.chunk = thin_chunk(rows, inputs, outputs, activation, false);
            a.x = x;
            a.weight = weight;
            a.bias = bias;
            a.residual = residual;
            a.y = y;
            a.slope = slope;
            a.activation = activation;
            with_linear_type(dtype, [&](auto type) { launch_thin_forward<decltype(type)>(a, stream); });
            return;
        }
        const ForwardScratch s(scratch, rows, inputs, outputs, groups);
        ODIE_REQUIRE(s.bytes == 0 || (scratch && uintptr_t(scratch) % 256 == 0), "scratch is required, on a 256-byte boundary");
        const int64_t ld = round8(inputs);
        if (s.x) {
            launch_pad(x, s.x, rows, weight, s.weight, int64_t(groups) * outputs, inputs, stream);
            x = s.x;
            weight = s.weight;
        }
        GemmArgs p{};
        p.groups = groups;
        p.offsets = offsets;
        p.rows = rows;
        p.n = outputs;
        p.k = inputs;
        p.out = y;
        p.bias = bias;
        p.residual = residual;
        p.slope = slope;
        p.activation = activation;
        p.error = error;
        p.limit = wait_limit;
        with_linear_type(dtype, [&](auto type) {
            launch_product<decltype(type), FWD>(x, weight, ld, ld, outputs, inputs, p, Splits(rows, outputs, inputs, groups, offsets), s.partial,
                                                stream);
        });
    });
}

extern "C" int64_t odie_linear_backward_scratch_for(int64_t rows, int inputs, int outputs, int groups, int on_16) {
    if (!sizes_fit(rows, inputs, outputs, groups)) return 0;
    if (backward_path(inputs, outputs, on_16) == Path::THIN) return BackwardScratch::thin_bytes(rows, inputs, outputs, groups);
    return BackwardScratch(nullptr, rows, inputs, outputs, groups).bytes;
}

extern "C" int64_t odie_linear_backward_scratch(int64_t rows, int inputs, int outputs, int groups) {
    return std::max(odie_linear_backward_scratch_for(rows, inputs, outputs, groups, 0), odie_linear_backward_scratch_for(rows, inputs, outputs, groups, 1));
}

extern "C" int odie_linear_backward(const void* d_y, const void* slope, int activation, const void* x, const void* weight, int64_t rows,
                                    int inputs, int outputs, int groups, const int32_t* offsets, int dtype, void* d_x,
                                    void* d_weight, void* d_bias, void* d_residual, void* scratch, uint64_t stream_handle) {
    return guarded([&] {
        check_linear(rows, inputs, outputs, groups, offsets, dtype, activation);
        const cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_handle);
        if (rows == 0) {
            if (d_weight) ODIE_CUDA(cudaMemsetAsync(d_weight, 0, size_t(groups) * outputs * inputs * 2, stream));
            if (d_bias) ODIE_CUDA(cudaMemsetAsync(d_bias, 0, size_t(groups) * outputs * 2, stream));
            return;
        }
        ODIE_REQUIRE(d_y && (x || !d_weight) && (weight || !d_x) && scratch, "d_y, x, weight and scratch are required");
        ODIE_REQUIRE(uintptr_t(scratch) % 256 == 0, "scratch must start on a 256-byte boundary");
        ODIE_REQUIRE(slope || activation == ACT_NONE, "slope is required with an activation");
        int* const error = checked_error_word();
        const int kind = slope_kind(activation, slope);
        const BackwardScratch s(scratch, rows, inputs, outputs, groups);
        if (backward_path(inputs, outputs, on_16_bytes({d_y, kind == SLOPE_CODES ? slope : nullptr, x, weight, d_x, d_residual})) == Path::THIN) {
            ThinArgs a{};
            a.rows = rows;
            a.inputs = inputs;
            a.outputs = outputs;
            a.groups = groups;
            a.offsets = offsets;
            a.chunk = thin_chunk(rows, inputs, outputs, kind == SLOPE_ONE ? ACT_NONE : activation, true);
            a.x = x;
            a.weight = weight;
            a.d_y = d_y;
            a.kept = slope;
            a.activation = activation;
            a.d_x = d_x;
            a.d_weight = d_weight;
            a.d_bias = d_bias;
            a.d_residual = d_residual;
            const bool join = rows > a.chunk && (d_weight || d_bias);
            a.partial = join ? s.thin : nullptr;
            with_linear_type(dtype, [&](auto type) {
                using T = decltype(type);
                launch_thin_backward<T>(a, stream);
                if (join)
                    launch_join<T>(s.thin, d_weight, d_bias, offsets, groups, rows, a.chunk, thin_units(rows, groups, a.chunk),
                                   int64_t(outputs) * inputs, outputs, stream);
            });
            return;
        }
        const bool bf16 = dtype == ROW_BF16;
        const int64_t ld_x = round8(inputs), ld_z = round8(outputs);
        const bool products = d_x || d_weight;
        const bool as_is = kind == SLOPE_ONE && outputs % 8 == 0;  // dz is d_y
        const void* dz = as_is ? d_y : s.dz;
        with_linear_type(dtype, [&](auto type) {
            using T = decltype(type);
            if ((products && !as_is) || d_bias || d_residual) {
                DzArgs a{};
                a.d_y = d_y;
                a.kept = slope;
                a.dz = products && !as_is ? s.dz : nullptr;
                a.d_residual = d_residual;
                const bool join = d_bias && rows > dz_chunk(rows, groups);
                a.partial = join ? s.bias : nullptr;
                a.d_bias = d_bias;
                a.rows = rows;
                a.n = outputs;
                a.ld = ld_z;
                a.chunk = int(dz_chunk(rows, groups));
                a.groups = groups;
                a.offsets = offsets;
                launch_dz<T>(a, kind, stream);
                if (join) launch_join<T>(s.bias, nullptr, d_bias, offsets, groups, rows, a.chunk, dz_units(rows, groups), 0, outputs, stream);
            }
            if (s.x && products)
                launch_pad(x, s.x, d_weight ? rows : 0, weight, s.weight, d_x ? int64_t(groups) * outputs : 0, inputs, stream);
            GemmArgs p{};
            p.groups = groups;
            p.offsets = offsets;
            p.rows = rows;
            p.n = inputs;
            p.error = error;
            p.limit = wait_limit;
            if (d_x) {
                p.k = outputs;
                p.out = d_x;
                launch_product<T, DX>(dz, s.weight ? s.weight : weight, ld_z, ld_x, outputs, inputs, p,
                                      Splits(rows, inputs, outputs, groups, offsets), s.split, stream);
            }
            if (d_weight) {
                const WeightUnits u(rows, inputs, outputs, groups);
                const CUtensorMap a = tensor_map(dz, bf16, outputs, rows, 0, ld_z, 64);
                const CUtensorMap b = tensor_map(s.x ? s.x : x, bf16, inputs, rows, 0, ld_x, 64);
                p.m = outputs;
                p.chunk = int(u.chunk);
                p.units = int(u.units);
                p.out = d_weight;
                p.partial = u.split ? s.partial : nullptr;
                if (offsets) {
                    group_maps_kernel<<<unsigned(2 * groups), 32, 0, stream>>>(a, b, offsets, rows, static_cast<CUtensorMap*>(s.maps));
                    ODIE_CUDA(cudaGetLastError());
                    note_launch();
                    p.group_maps = static_cast<const CUtensorMap*>(s.maps);
                }
                with_config(u.config, [&](auto cg, auto bn) {
                    constexpr int CG = decltype(cg)::value, BN = decltype(bn)::value;
                    if (u.split) launch_gemm<T, DW, CG, BN, true>(a, b, p, u.units * u.tiles, stream);
                    else launch_gemm<T, DW, CG, BN, false>(a, b, p, u.units * u.tiles, stream);
                });
                if (u.split) {
                    const int64_t size = int64_t(outputs) * inputs;
                    launch_join<T>(s.partial, d_weight, nullptr, offsets, groups, rows, u.chunk, u.units, int64_t(outputs) * inputs, 0, stream);
                }
            }
        });
    });
}

extern "C" int odie_linear_wait_limit(int64_t polls) {
    return guarded([&] {
        ODIE_REQUIRE(polls >= -1 && polls <= int64_t(WAIT_LIMIT), "polls must be 0 to 2^22, or -1");
        wait_limit = polls < 0 ? WAIT_LIMIT : uint32_t(polls);
    });
}

extern "C" int odie_linear_status(int32_t* status, uint64_t stream) {
    return guarded([&] {
        ODIE_REQUIRE(status, "status is required");
        ODIE_CUDA(cudaMemcpyAsync(status, error_word(), sizeof(int), cudaMemcpyHostToDevice, reinterpret_cast<cudaStream_t>(stream)));
    });
}

extern "C" int odie_linear_check(void) {
    return guarded([&] { checked_error_word(); });
}
