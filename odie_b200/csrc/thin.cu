// Linear layers of up to 64 inputs and outputs: forward, and the whole backward pass (dz, d x, d W, d b) in one kernel.
//
// Bound by the bytes of the rows (64 to 128 bytes each), not by arithmetic: 2^20 rows of 32 -> 64 fp16 are 192 MB
// forward against 4.3 GFLOP.  So a warp keeps its 16 rows in registers from the 16-byte loads to the 16-byte stores
// and multiplies them with mma.sync fragments.  (The tensor-core tiles of linear.cu, whose rows pass through shared
// memory, TMEM and a staging tile, took 102 us forward and 205 us in four kernels backward; these take 47 and 55 with
// ReLU, 4.2 and 4.7 TB/s.  What is left is the wait of an instruction for the one before: registers leave room for 12
// warps per SM, each issues every 4.9 cycles forward and every 6.7 backward, 1.2 and 2.3 of them such waits, backward 0.9
// for memory; issue slots are 56 and 44 % busy.)
//
// The fragments' order of columns is chosen so that no data is exchanged.  Lane (g, c) = (lane / 4, lane % 4) loads
// the 8 columns 8 c .. 8 c + 7 of rows g and g + 8 for each 32-column block: word i (columns 8 c + 2 i, + 1) is what
// m16n8k16 wants of row g for K-step i / 2, first (i even) or second (i odd) half, if K is counted in this order;
// W is read in the same order.  Column n' of output tile j stands for column 8 (n' / 2) + 2 j + n' % 2, so a lane
// ends with the 8 columns 8 c .. 8 c + 7 of the result.  d W = dz^T x needs dz and x by columns: movmatrix turns
// each 8 x 8 tile, in the same order of columns.
//
// A ReLU's corner: where the tensor cores' sum is within its own error of zero, the fp32 chain of fused multiply-adds
// in ascending order of the inputs decides (the convention of this library's router), since at these sizes one unit is a
// large part of a row's gradient.  (Its own error is an estimate: 2^-20 of inputs x the largest input x the largest weight.
// An fp32 sum in another order may still differ in sign from the chain.)  About one step of 16 rows in forty looks at one.
#include "thin.cuh"
#include "odie_b200.h"
#include <algorithm>

namespace odie {
namespace {

constexpr int THREADS = 128, WARPS = 4, STEP = WARPS * 16;
// Steps of 16 rows per warp, one in work, the others on their way.
constexpr int FORWARD_STAGES = 4;
template <int KB, int NB, int KIND>
constexpr int STAGES_BACK = KB * NB == 4 ? 3 : KIND == SLOPE_CODES ? 5 : 4;

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t turned(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
// Byte 0's sign over the lower half, byte 2's over the upper.
__device__ __forceinline__ uint32_t signs_of_bytes_0_2(uint32_t v) {
    uint32_t r;
    asm("prmt.b32 %0, %1, 0, 0xaa88;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// Copies ahead: a lane's own 16-byte words, in shared memory slots that only it reads, so that rows are on their way
// without holding registers.  A copy that is off writes zeros.
__device__ __forceinline__ void copy_ahead(uint4* slot, const uint16_t* from, bool on, const void* base) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(uint32_t(__cvta_generic_to_shared(slot))),
                 "l"(on ? static_cast<const void*>(from) : base), "r"(on ? 16 : 0)
                 : "memory");
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}

__device__ __forceinline__ uint4 load_row(const void* base, long long row, int width, int column, bool on) {
    return on ? __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + row * width + column)) : make_uint4(0, 0, 0, 0);
}

// The larger magnitudes, pairwise, of two pairs of 16-bit elements; the signs are off.
template <typename T>
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    return __vmaxu2(a & 0x7fff7fffu, b & 0x7fff7fffu);  // magnitudes order as their bits do
}
template <typename T>
__device__ __forceinline__ uint32_t larger(uint32_t a, const uint4& v) {
    return larger<T>(larger<T>(larger<T>(a, v.x), larger<T>(v.y, v.z)), v.w);
}
// The larger of two magnitudes; infinity where either is NaN.
template <typename T>
__device__ __forceinline__ float larger_of(uint32_t pair) {
    constexpr uint32_t INF = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
    return unpack_pair<T>(min(max(pair & 0xffffu, pair >> 16), INF)).x;
}
// Two magnitudes, 0 in place of those that are not finite.
template <typename T>
__device__ __forceinline__ uint32_t finite(uint32_t pair) {
    return pair & ~__vcmpgeu2(pair & 0x7fff7fffu, std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u);
}

// x . w as the chain in ascending order; count is a multiple of 8.
template <typename T>
__device__ __forceinline__ float chain(const void* x, const void* w, int count) {
    float sum = 0.0f;
#pragma unroll 4
    for (int k = 0; k < count / 8; ++k) {
        const uint4 a = __ldg(static_cast<const uint4*>(x) + k), b = __ldg(static_cast<const uint4*>(w) + k);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = unpack_pair<T>(word(a, i)), g = unpack_pair<T>(word(b, i));
            sum = fmaf(f.y, g.y, fmaf(f.x, g.x, sum));
        }
    }
    return sum;
}

// A ReLU's bits in memory: lane (g, c) holds a byte per (h, nb), columns 32 nb + 8 c .. of row g + 8 h, as byte h NB + nb
// of a word; turned among the row's four lanes, lane c has the four bytes of the c-th (h, nb), one word of the mask.
__device__ __forceinline__ uint32_t turned_bytes(uint32_t v, int c) {
    uint32_t other = __shfl_xor_sync(0xffffffffu, v, 1);
    v = c & 1 ? __byte_perm(other, v, 0x7351) : __byte_perm(v, other, 0x6240);  // bytes (mine, theirs) of even or odd places
    other = __shfl_xor_sync(0xffffffffu, v, 2);
    return c & 2 ? __byte_perm(other, v, 0x7632) : __byte_perm(v, other, 0x5410);
}

// max(v, 0) of two packed values, NaN for NaN, +0 for -0.
template <typename T>
__device__ __forceinline__ uint32_t above_zero(uint32_t v) {
    uint32_t r;
    if constexpr (std::is_same<T, __half>::value) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(0));
    else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(0));
    return r;
}
__device__ __forceinline__ float least_magnitude(float a, float b, float c) {
    float r;
    asm("min.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// KB, NB: blocks of 32 inputs and outputs.
template <typename T, int KB, int NB, int ACT>
__global__ void __launch_bounds__(THREADS, thin_blocks(KB * 32, NB * 32, ACT, false)) thin_forward_kernel(ThinArgs a) {
    constexpr int VECTORS = KB * 2 + NB * 2;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
    const Unit u = unit_at<false>(a.offsets, a.groups, a.rows, a.chunk, blockIdx.x);
    if (u.g < 0) return;
    if (u.g == a.groups) {  // rows of no group
        for (long long row = u.from + warp * 8 + g; row < u.to; row += WARPS * 8) {
            for (int nb = 0; nb < NB; ++nb) {
                const int column = nb * 32 + c * 8;
                if (column >= a.outputs) continue;
                *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.y) + row * a.outputs + column) = make_uint4(0, 0, 0, 0);
                if (ACT == ACT_RELU && a.slope) static_cast<uint8_t*>(a.slope)[(row * a.outputs + column) / 8] = 0;
                else if (a.slope) *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.slope) + row * a.outputs + column) = make_uint4(0, 0, 0, 0);
            }
        }
        return;
    }
    uint4 w[NB][4][KB];
    float bias[NB][8];
    const uint16_t* weight = static_cast<const uint16_t*>(a.weight) + (long long)u.g * a.outputs * a.inputs;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                const int n = nb * 32 + (g >> 1) * 8 + j * 2 + (g & 1), k = kb * 32 + c * 8;
                w[nb][j][kb] = load_row(weight, n, a.inputs, k, n < a.outputs && k < a.inputs);
            }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int n = nb * 32 + c * 8 + e;
            bias[nb][e] = a.bias && n < a.outputs ? to_float(static_cast<const T*>(a.bias)[(long long)u.g * a.outputs + n]) : 0.0f;
        }
    }
    // corner: times a row's largest input: what the tensor cores' sum may be off by.  Of the finite weights and biases: a
    // unit of others has no finite sum.
    float bias_corner = 0.0f, corner = 0.0f;
    if (ACT == ACT_RELU) {
        uint32_t largest = 0;
        float most_bias = 0.0f;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int i = 0; i < 4; ++i) largest = larger<T>(largest, finite<T>(word(w[nb][j][kb], i)));
#pragma unroll
            for (int e = 0; e < 8; ++e) most_bias = fmaxf(most_bias, isfinite(bias[nb][e]) ? fabsf(bias[nb][e]) : 0.0f);
        }
        float most = larger_of<T>(largest);
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
            most_bias = fmaxf(most_bias, __shfl_xor_sync(0xffffffffu, most_bias, d));
        }
        corner = most * float(a.inputs) * 0x1p-20f;
        bias_corner = most_bias * 0x1p-21f;
    }
    extern __shared__ uint4 slots[];
    uint4* mine = slots + warp * (FORWARD_STAGES * VECTORS * 32) + lane;
    const long long row0 = u.from + warp * 16 + g;
    int left = int(u.to - row0);     // rows from the lane's first row of this step on: row 8 h is there if left > 8 h
    int left_ahead = left, fill = 0;  // of the step that is fetched, its slot
    const uint16_t* x_ahead = static_cast<const uint16_t*>(a.x) + row0 * a.inputs + c * 8;
    uint16_t* y = static_cast<uint16_t*>(a.y) + row0 * a.outputs + c * 8;
    auto ahead = [&]() {
        uint4* to = mine + fill * (VECTORS * 32);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
                copy_ahead(to + (kb * 2 + h) * 32, x_ahead + 8 * h * a.inputs + kb * 32, left_ahead > 8 * h && kb * 32 + c * 8 < a.inputs, a.x);
            if (a.residual) {
                const uint16_t* residual_ahead = static_cast<const uint16_t*>(a.residual) + (u.to - left_ahead) * a.outputs + c * 8;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
                    copy_ahead(to + (KB * 2 + nb * 2 + h) * 32, residual_ahead + 8 * h * a.outputs + nb * 32,
                               left_ahead > 8 * h && nb * 32 + c * 8 < a.outputs, a.residual);
            }
        }
        copies_end();
        x_ahead += STEP * a.inputs;
        left_ahead -= STEP;
        fill = fill + 1 == FORWARD_STAGES ? 0 : fill + 1;
    };
    for (int s = 0; s < FORWARD_STAGES - 1; ++s) ahead();
    const bool words = reinterpret_cast<uintptr_t>(a.slope) % 4 == 0;
    int use = 0;
    for (int from = warp * 16; from < u.to - u.from; from += STEP, left -= STEP, y += STEP * a.outputs) {
        ahead();
        copies_wait<FORWARD_STAGES - 1>();
        const uint4* now = mine + use * (VECTORS * 32);
        use = use + 1 == FORWARD_STAGES ? 0 : use + 1;
        uint4 x[KB][2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) x[kb][h] = now[(kb * 2 + h) * 32];
        uint32_t on = 0;    // ReLU: a byte per (h, nb)
        float near = 0.0f;  // for both rows of the lane; infinite or NaN if either holds no numbers: every finite sum goes by its chain
        if (ACT == ACT_RELU) {
            uint32_t largest = larger<T>(larger<T>(0, x[0][0]), x[0][1]);
            if (KB == 2) largest = larger<T>(larger<T>(largest, x[KB - 1][0]), x[KB - 1][1]);
            largest = larger<T>(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
            largest = larger<T>(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
            near = larger_of<T>(largest) * corner + bias_corner;
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const int column = nb * 32 + c * 8;
            const bool inside = column < a.outputs;
            uint4 r[2];
            if (a.residual) {
#pragma unroll
                for (int h = 0; h < 2; ++h) r[h] = now[(KB * 2 + nb * 2 + h) * 32];
            }
            float d[4][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
#pragma unroll
                for (int i = 0; i < 4; ++i) d[j][i] = bias[nb][j * 2 + (i & 1)];
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int s = 0; s < 2; ++s)
                        mma16816<T>(d[j], word(x[kb][0], 2 * s), word(x[kb][1], 2 * s), word(x[kb][0], 2 * s + 1), word(x[kb][1], 2 * s + 1),
                                    word(w[nb][j][kb], 2 * s), word(w[nb][j][kb], 2 * s + 1));
            }
            if (ACT == ACT_RELU) {
                float least = fabsf(d[0][0]);
#pragma unroll
                for (int e = 2; e < 16; e += 2) least = least_magnitude(least, d[e / 4][e % 4], d[e / 4][e % 4 + 1]);
                least = fminf(least, fabsf(d[0][1]));
                if (!(least > near)) {
                    uint32_t which = 0;
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const float z = fabsf(d[e / 4][e % 4]);
                        which |= !(z >= near) && z < INFINITY && inside && left > (e % 4 / 2) * 8 ? 1u << e : 0u;
                    }
#pragma unroll 1
                    for (; which; which &= which - 1) {
                        const int at = __ffs(which) - 1, n = column + at / 4 * 2 + at % 2;
                        const long long row = u.from + from + g + (at % 4 / 2) * 8;
                        const float z = chain<T>(static_cast<const uint16_t*>(a.x) + row * a.inputs, weight + n * a.inputs, a.inputs) +
                                        (a.bias ? to_float(static_cast<const T*>(a.bias)[(long long)u.g * a.outputs + n]) : 0.0f);
#pragma unroll
                        for (int e = 0; e < 16; ++e) d[e / 4][e % 4] = at == e ? z : d[e / 4][e % 4];
                    }
#pragma unroll
                    for (int e = 0; e < 16; ++e) d[e / 4][e % 4] = d[e / 4][e % 4] == 0.0f ? -0x1p-149f : d[e / 4][e % 4];
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const bool there = left > 8 * h && inside;
                const int at = 8 * h * a.outputs + nb * 32;
                uint32_t out[4], codes[4], off = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (ACT == ACT_RELU) {  // the packed sums' signs say where it is off (a zero is negative by now)
                        const uint32_t z = pack_pair<T>(d[j][2 * h], d[j][2 * h + 1]);
                        off |= z >> (15 - 2 * j) & (0x10001u << (2 * j));
                        out[j] = above_zero<T>(z);
                    } else {
                        const float2 f = a.residual ? unpack_pair<T>(word(r[h], j)) : make_float2(0.0f, 0.0f);
                        Pair slope;
                        const float2 v = both(activate<ACT, true>(pair(d[j][2 * h], d[j][2 * h + 1]), slope, pair(f.x, f.y)));
                        out[j] = pack_pair<T>(v.x, v.y);
                        if (a.slope) codes[j] = slope_codes(slope);
                    }
                }
                if (ACT == ACT_RELU && a.residual) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 f = unpack_pair<T>(word(r[h], j));
                        out[j] = pack_pair<T>(max_nan(d[j][2 * h], 0.0f) + f.x, max_nan(d[j][2 * h + 1], 0.0f) + f.y);
                    }
                }
                if (ACT == ACT_RELU) on |= (~(off | off >> 15) & 0xffu) << ((h * NB + nb) * 8);
                if (there) {
                    *reinterpret_cast<uint4*>(y + at) = make_uint4(out[0], out[1], out[2], out[3]);
                    if (ACT != ACT_RELU && a.slope)
                        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.slope) + (y + at - static_cast<uint16_t*>(a.y))) =
                            make_uint4(codes[0], codes[1], codes[2], codes[3]);
                }
            }
        }
        if (ACT == ACT_RELU && a.slope) {
            on = turned_bytes(on, c);
            const int h = c / NB, nb = c % NB, pitch = a.outputs / 8;
            if (h < 2 && left > 8 * h) {
                uint8_t* to = static_cast<uint8_t*>(a.slope) + (u.to - left + 8 * h) * pitch + nb * 4;
                if (pitch % 4 == 0 && words) {
                    *reinterpret_cast<uint32_t*>(to) = on;
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (nb * 4 + i < pitch) to[i] = uint8_t(on >> (8 * i));
                }
            }
        }
    }
}

template <typename T, int KB, int NB, int KIND>
__global__ void __launch_bounds__(THREADS, thin_blocks(KB * 32, NB * 32, KIND == SLOPE_CODES ? ACT_GELU : ACT_NONE, true)) thin_backward_kernel(ThinArgs a) {
    constexpr int BACKWARD_STAGES = STAGES_BACK<KB, NB, KIND>;
    constexpr int AT_X = NB * (KIND == SLOPE_CODES ? 4 : 2), VECTORS = AT_X + KB * 2;
    extern __shared__ uint4 slots[];
    // W by its rows' order for d x: [K-step of 16 outputs][8-column tile of inputs][lane]
    __shared__ uint2 turned_w[NB * 2][KB * 4][32];
    __shared__ float sums[NB * 32][KB * 32 + 1];
    __shared__ float bias_sums[NB * 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
    const Unit u = unit_at<true>(a.offsets, a.groups, a.rows, a.chunk, blockIdx.x);
    if (u.g < 0) return;
    if (u.g == a.groups) {  // rows of no group
        for (long long row = u.from + warp * 8 + g; row < u.to; row += WARPS * 8) {
            for (int kb = 0; kb < KB; ++kb)
                if (a.d_x && kb * 32 + c * 8 < a.inputs)
                    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.d_x) + row * a.inputs + kb * 32 + c * 8) = make_uint4(0, 0, 0, 0);
            for (int nb = 0; nb < NB; ++nb)
                if (a.d_residual && nb * 32 + c * 8 < a.outputs)
                    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.d_residual) + row * a.outputs + nb * 32 + c * 8) = make_uint4(0, 0, 0, 0);
        }
        return;
    }
    const bool sum_weights = a.d_weight || a.d_bias;
    if (a.d_x) {
        const uint16_t* weight = static_cast<const uint16_t*>(a.weight) + (long long)u.g * a.outputs * a.inputs;
        for (int i = warp; i < NB * 2 * KB * 4; i += WARPS) {
            const int step = i / (KB * 4), tile = i % (KB * 4), nb = step / 2, s = step % 2, kb = tile / 4, j = tile % 4;
            const int n = nb * 32 + c * 8 + s * 4, k = kb * 32 + (g >> 1) * 8 + j * 2 + (g & 1);
            uint32_t e[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) e[q] = n + q < a.outputs && k < a.inputs ? weight[(n + q) * a.inputs + k] : 0;
            turned_w[step][tile][lane] = make_uint2(e[0] | e[1] << 16, e[2] | e[3] << 16);
        }
    }
    for (int i = threadIdx.x; i < NB * 32 * (KB * 32 + 1); i += THREADS) (&sums[0][0])[i] = 0.0f;
    for (int i = threadIdx.x; i < NB * 32; i += THREADS) bias_sums[i] = 0.0f;
    __syncthreads();
    // d b: with codes the lanes' sums of the unrounded dz (db); else dz is exact, and a product with ones sums it (ones)
    constexpr bool BY_ONES = KIND != SLOPE_CODES;
    constexpr uint32_t ONES = std::is_same<T, __half>::value ? 0x3c003c00u : 0x3f803f80u;
    float dw[NB * 2][KB * 4][4], ones[NB * 2][4], db[NB][8];
#pragma unroll
    for (int m = 0; m < NB * 2; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            ones[m][i] = 0.0f;
#pragma unroll
            for (int n = 0; n < KB * 4; ++n) dw[m][n][i] = 0.0f;
        }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < 8; ++e) db[nb][e] = 0.0f;
    uint4* mine = slots + warp * (BACKWARD_STAGES * VECTORS * 32) + lane;
    const long long row0 = u.from + warp * 16 + g;
    int left = int(u.to - row0);      // row 8 h of this step is there if left > 8 h
    int left_ahead = left, fill = 0;  // of the step that is fetched, its slot
    const uint16_t* d_y_ahead = static_cast<const uint16_t*>(a.d_y) + row0 * a.outputs + c * 8;
    const uint16_t* x_ahead = static_cast<const uint16_t*>(a.x) + row0 * a.inputs + c * 8;
    const long long codes_from_d_y = static_cast<const uint16_t*>(a.kept) - static_cast<const uint16_t*>(a.d_y);
    uint16_t* d_x = static_cast<uint16_t*>(a.d_x) + row0 * a.inputs + c * 8;
    uint16_t* d_residual = static_cast<uint16_t*>(a.d_residual) + row0 * a.outputs + c * 8;
    auto ahead = [&]() {
        uint4* to = mine + fill * (VECTORS * 32);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                const bool on = left_ahead > 8 * h && nb * 32 + c * 8 < a.outputs;
                const uint16_t* from = d_y_ahead + 8 * h * a.outputs + nb * 32;
                copy_ahead(to + (nb * 2 + h) * 32, from, on, a.d_y);
                if (KIND == SLOPE_CODES) copy_ahead(to + (NB * 2 + nb * 2 + h) * 32, from + codes_from_d_y, on, a.kept);
            }
            if (a.d_weight) {
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
                    copy_ahead(to + (AT_X + kb * 2 + h) * 32, x_ahead + 8 * h * a.inputs + kb * 32, left_ahead > 8 * h && kb * 32 + c * 8 < a.inputs, a.x);
            }
        }
        copies_end();
        d_y_ahead += STEP * a.outputs;
        x_ahead += STEP * a.inputs;
        left_ahead -= STEP;
        fill = fill + 1 == BACKWARD_STAGES ? 0 : fill + 1;
    };
    for (int s = 0; s < BACKWARD_STAGES - 1; ++s) ahead();
    // the mask's bytes, a step ahead
    uint32_t next = 0;
    const bool words = reinterpret_cast<uintptr_t>(a.kept) % 4 == 0;
    auto masks = [&](int left) {
        const int h = c / NB, nb = c % NB, pitch = a.outputs / 8;
        next = 0;
        if (h < 2 && left > 8 * h) {
            const uint8_t* from = static_cast<const uint8_t*>(a.kept) + (u.to - left + 8 * h) * pitch + nb * 4;
            if (pitch % 4 == 0 && words) {
                next = __ldg(reinterpret_cast<const uint32_t*>(from));
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (nb * 4 + i < pitch) next |= uint32_t(__ldg(from + i)) << (8 * i);
            }
        }
    };
    if (KIND == SLOPE_MASK) masks(left);
    int use = 0;
    for (int from = warp * 16; from < u.to - u.from; from += STEP, left -= STEP) {
        uint32_t bits[NB][2];
        if (KIND == SLOPE_MASK) {
            const uint32_t on = turned_bytes(next, c);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t byte = on >> ((h * NB + nb) * 8) & 0xffu;
                    bits[nb][h] = byte | byte << 15;
                }
            masks(left - STEP);
        }
        ahead();
        copies_wait<BACKWARD_STAGES - 1>();
        const uint4* now = mine + use * (VECTORS * 32);
        use = use + 1 == BACKWARD_STAGES ? 0 : use + 1;
        uint4 z[NB][2], x[KB][2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) x[kb][h] = a.d_weight ? now[(AT_X + kb * 2 + h) * 32] : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                z[nb][h] = now[(nb * 2 + h) * 32];
                if (a.d_residual && left > 8 * h && nb * 32 + c * 8 < a.outputs)
                    *reinterpret_cast<uint4*>(d_residual + 8 * h * a.outputs + nb * 32) = z[nb][h];
                uint32_t q[4];
                if (KIND == SLOPE_CODES) {
                    const uint4 s = now[(NB * 2 + nb * 2 + h) * 32];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float2 f = unpack_pair<T>(word(z[nb][h], i));
                        f.x *= slope_value(word(s, i) & 0xffffu);
                        f.y *= slope_value(word(s, i) >> 16);
                        db[nb][2 * i] += f.x;
                        db[nb][2 * i + 1] += f.y;
                        q[i] = pack_pair<T>(f.x, f.y);
                    }
                    z[nb][h] = make_uint4(q[0], q[1], q[2], q[3]);
                } else if (KIND == SLOPE_MASK) {
                    // bit 2 i to the sign of byte 0, bit 2 i + 1 (its copy 15 above) to that of byte 2, and over their halves
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        q[i] = word(z[nb][h], i) & signs_of_bytes_0_2(bits[nb][h] << (7 - 2 * i));
                    z[nb][h] = make_uint4(q[0], q[1], q[2], q[3]);
                }
            }
        d_residual += STEP * a.outputs;
        if (a.d_x) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                float d[4][4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) d[j][i] = 0.0f;
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int t = 0; t < 2; ++t) {
                            const uint2 b = turned_w[nb * 2 + t][kb * 4 + j][lane];
                            mma16816<T>(d[j], word(z[nb][0], 2 * t), word(z[nb][1], 2 * t), word(z[nb][0], 2 * t + 1), word(z[nb][1], 2 * t + 1),
                                        b.x, b.y);
                        }
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (left > 8 * h && kb * 32 + c * 8 < a.inputs)
                        *reinterpret_cast<uint4*>(d_x + 8 * h * a.inputs + kb * 32) =
                            make_uint4(pack_pair<T>(d[0][2 * h], d[0][2 * h + 1]), pack_pair<T>(d[1][2 * h], d[1][2 * h + 1]),
                                       pack_pair<T>(d[2][2 * h], d[2][2 * h + 1]), pack_pair<T>(d[3][2 * h], d[3][2 * h + 1]));
                }
            }
        }
        d_x += STEP * a.inputs;
        if (a.d_weight || (BY_ONES && a.d_bias)) {
            uint32_t xt[KB][4][2];
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int h = 0; h < 2; ++h) xt[kb][i][h] = turned(word(x[kb][h], i));
#pragma unroll
            for (int m = 0; m < NB * 2; ++m) {
                const int nb = m / 2, p = m % 2;
                const uint32_t a0 = turned(word(z[nb][0], 2 * p)), a1 = turned(word(z[nb][0], 2 * p + 1));
                const uint32_t a2 = turned(word(z[nb][1], 2 * p)), a3 = turned(word(z[nb][1], 2 * p + 1));
#pragma unroll
                for (int n = 0; n < KB * 4; ++n) mma16816<T>(dw[m][n], a0, a1, a2, a3, xt[n / 4][n % 4][0], xt[n / 4][n % 4][1]);
                if (BY_ONES) mma16816<T>(ones[m], a0, a1, a2, a3, ONES, ONES);
            }
        }
    }
    if (!sum_weights) return;
    // the block's sums: the warps' in order
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int d = 4; d < 32; d *= 2) db[nb][e] += __shfl_xor_sync(0xffffffffu, db[nb][e], d);
    for (int w = 0; w < WARPS; ++w) {
        if (warp == w) {
#pragma unroll
            for (int m = 0; m < NB * 2; ++m)
#pragma unroll
                for (int n = 0; n < KB * 4; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int out = (m / 2) * 32 + (g >> 1) * 8 + (2 * (m % 2) + (i >> 1)) * 2 + (g & 1);
                        sums[out][(n / 4) * 32 + c * 8 + (n % 4) * 2 + (i & 1)] += dw[m][n][i];
                    }
            if (BY_ONES && c == 0) {
#pragma unroll
                for (int m = 0; m < NB * 2; ++m)
#pragma unroll
                    for (int i = 0; i < 2; ++i) bias_sums[(m / 2) * 32 + (g >> 1) * 8 + (2 * (m % 2) + i) * 2 + (g & 1)] += ones[m][2 * i];
            }
            if (!BY_ONES && g == 0) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int e = 0; e < 8; ++e) bias_sums[nb * 32 + c * 8 + e] += db[nb][e];
            }
        }
        __syncthreads();
    }
    const int size = a.outputs * a.inputs;
    if (a.partial) {
        float* to = a.partial + (long long)u.index * (size + a.outputs);
        if (a.d_weight)
            for (int i = threadIdx.x; i < size; i += THREADS) to[i] = sums[i / a.inputs][i % a.inputs];
        for (int i = threadIdx.x; i < a.outputs; i += THREADS) to[size + i] = bias_sums[i];
    } else {
        if (a.d_weight)
            for (int i = threadIdx.x; i < size; i += THREADS)
                static_cast<T*>(a.d_weight)[(long long)u.g * size + i] = from_float<T>(sums[i / a.inputs][i % a.inputs]);
        if (a.d_bias)
            for (int i = threadIdx.x; i < a.outputs; i += THREADS)
                static_cast<T*>(a.d_bias)[(long long)u.g * a.outputs + i] = from_float<T>(bias_sums[i]);
    }
}

template <typename F>
void with_blocks(int inputs, int outputs, F&& f) {
    auto second = [&](auto kb) {
        if (outputs <= 32) f(kb, std::integral_constant<int, 1>{});
        else f(kb, std::integral_constant<int, 2>{});
    };
    if (inputs <= 32) second(std::integral_constant<int, 1>{});
    else second(std::integral_constant<int, 2>{});
}

}  // namespace

template <typename T>
void launch_thin_forward(const ThinArgs& a, cudaStream_t stream) {
    with_blocks(a.inputs, a.outputs, [&](auto kb, auto nb) {
        constexpr int KB = decltype(kb)::value, NB = decltype(nb)::value;
        constexpr int BYTES = WARPS * FORWARD_STAGES * (KB * 2 + NB * 2) * 512;
        const auto kernel = a.activation == ACT_RELU   ? thin_forward_kernel<T, KB, NB, ACT_RELU>
                            : a.activation == ACT_SILU ? thin_forward_kernel<T, KB, NB, ACT_SILU>
                            : a.activation == ACT_GELU ? thin_forward_kernel<T, KB, NB, ACT_GELU>
                                                       : thin_forward_kernel<T, KB, NB, ACT_NONE>;
        ODIE_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, BYTES));
        kernel<<<unsigned(thin_units(a.rows, a.groups, a.chunk)), THREADS, BYTES, stream>>>(a);
    });
    ODIE_CUDA(cudaGetLastError());
    note_launch();
}

template <typename T>
void launch_thin_backward(const ThinArgs& a, cudaStream_t stream) {
    with_blocks(a.inputs, a.outputs, [&](auto kb, auto nb) {
        constexpr int KB = decltype(kb)::value, NB = decltype(nb)::value;
        auto go = [&](auto kind) {
            constexpr int KIND = decltype(kind)::value;
            constexpr int BYTES = WARPS * STAGES_BACK<KB, NB, KIND> * (NB * (KIND == SLOPE_CODES ? 4 : 2) + KB * 2) * 512;
            const auto kernel = thin_backward_kernel<T, KB, NB, KIND>;
            ODIE_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, BYTES));
            kernel<<<unsigned(thin_units(a.rows, a.groups, a.chunk)), THREADS, BYTES, stream>>>(a);
        };
        const int kind = slope_kind(a.activation, a.kept);
        if (kind == SLOPE_MASK) go(std::integral_constant<int, SLOPE_MASK>{});
        else if (kind == SLOPE_CODES) go(std::integral_constant<int, SLOPE_CODES>{});
        else go(std::integral_constant<int, SLOPE_ONE>{});
    });
    ODIE_CUDA(cudaGetLastError());
    note_launch();
}

template void launch_thin_forward<__half>(const ThinArgs&, cudaStream_t);
template void launch_thin_forward<__nv_bfloat16>(const ThinArgs&, cudaStream_t);
template void launch_thin_backward<__half>(const ThinArgs&, cudaStream_t);
template void launch_thin_backward<__nv_bfloat16>(const ThinArgs&, cudaStream_t);

}  // namespace odie
