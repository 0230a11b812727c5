// Activations of the linear layers with their slopes, two values at a time (linear.cu, thin.cu).
#pragma once
#include "rows.cuh"
#include <type_traits>

namespace odie {

enum Activation : int { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3 };

// How training keeps act'(z): a ReLU's as one bit per output, rows of ceil(outputs / 8) bytes, bit c % 8 of byte c / 8
// for column c,
// set unless z <= 0; the smooth ones' as a 16-bit code per output.
enum SlopeKind : int { SLOPE_ONE = 0, SLOPE_CODES = 1, SLOPE_MASK = 2 };
inline int slope_kind(int activation, const void* kept) { return !kept || activation == ACT_NONE ? SLOPE_ONE : activation == ACT_RELU ? SLOPE_MASK : SLOPE_CODES; }

// Pairs of fp32 values: sm_100 multiplies and adds two per instruction.
struct Pair {
    unsigned long long v;
};
__device__ __forceinline__ Pair pair(float a, float b) {
    Pair r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 both(Pair p) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p.v));
    return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return d;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
    Pair d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
    return d;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
    Pair d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
    return d;
}
__device__ __forceinline__ Pair same(float a) { return pair(a, a); }
__device__ __forceinline__ float exp2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float inverse_approx(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// The slope's code, as the low bits of 2^23 + code (one fused multiply-add rounds to nearest; act' in (-1/4, 7/4)
// needs no clamp).  A NaN slope is the canonical NaN, whose low 16 bits are 0xffff.
__device__ __forceinline__ uint32_t slope_codes(Pair slope) {
    const float2 c = both(fma2(slope, same(32768.0f), same(8388608.0f + 8192.0f)));
    return __byte_perm(__float_as_uint(c.x), __float_as_uint(c.y), 0x5410);
}
__device__ __forceinline__ float slope_value(uint32_t c) {  // c: 16 bits
    const float d = fmaf(__uint_as_float(0x4b000000u | c), 1.0f / 32768.0f, -256.25f);  // exact
    return c == 0xffffu ? __int_as_float(0x7fffffff) : d;
}

// bits, with (first <= 0, second <= 0) below them: where a ReLU is off.  They are the signs of z - 2^-149, the least
// fp32, negative for z <= 0 alone (a NaN that arithmetic returns is positive: its gradient passes).
__device__ __forceinline__ uint32_t off_bits(uint32_t bits, float first, float second) {
    const float2 below = both(add2(pair(first, second), same(-0x1p-149f)));
    return __funnelshift_l(__float_as_uint(below.x), __funnelshift_l(__float_as_uint(below.y), bits, 1), 1);
}

// act(z) (with ADD: added + act(z), its last product and the sum one fused step, so that kernels that do and do not
// keep the slope give the same bits), with act'(z) in slope, of two values.
//   SiLU  p = 1 / (1 + e^-z): z p and p + z p (1 - p).
//   GELU  z P(z) and P(z) + z e^(-z^2/2) / sqrt(2 pi), P the normal distribution function: P(-u) = r = e^(-u^2/2)
//         (b1 t + .. + b6 t^6), t = 1 / (1 + 0.3 u), u = |z|, and P(u) = 1 - r.  The b are a fit by linear programming
//         of erfc's scaled form on 0 <= u <= 13.5, within 2.1e-7 absolutely and 4.3e-5 of r.  (The tail is r itself: as
//         a difference of halves it would have an absolute grain of 3e-8, 4 % of z P(z) at z = -5.)  The slope shares
//         the exponential.
// Written in pairs, and with one instruction each for exponential and inverse: the epilogue shares the SM with
// nothing else, but at 45 instructions per element it took twice the products' time for 1024 inputs.
template <int ACT, bool ADD = false>
__device__ __forceinline__ Pair activate(Pair z, Pair& slope, Pair added = Pair{}) {
    constexpr float LOG2E = 1.4426950408889634f;
    const float2 s = both(z);
    if (ACT == ACT_RELU) {
        const Pair r = pair(max_nan(s.x, 0.0f), max_nan(s.y, 0.0f));
        slope = pair(s.x > 0.0f ? 1.0f : both(r).x, s.y > 0.0f ? 1.0f : both(r).y);  // 0 or NaN where z is not positive
        return ADD ? add2(r, added) : r;
    }
    if (ACT == ACT_SILU) {
        const float2 x = both(mul2(z, same(-LOG2E)));
        const float2 d = both(add2(pair(exp2_approx(x.x), exp2_approx(x.y)), same(1.0f)));
        const Pair p = pair(inverse_approx(d.x), inverse_approx(d.y));
        const Pair a = mul2(z, p);
        slope = fma2(a, fma2(p, same(-1.0f), same(1.0f)), p);
        return ADD ? fma2(z, p, added) : a;
    }
    if (ACT == ACT_GELU) {
        const float2 x = both(mul2(mul2(z, z), same(-0.5f * LOG2E)));
        const Pair e = pair(exp2_approx(x.x), exp2_approx(x.y));
        const Pair t = pair(inverse_approx(fmaf(fabsf(s.x), 0.3f, 1.0f)), inverse_approx(fmaf(fabsf(s.y), 0.3f, 1.0f)));
        Pair q = fma2(t, same(-0.07833299689735844f), same(0.21848363561565745f));
        q = fma2(t, q, same(-0.017992417809206296f));
        q = fma2(t, q, same(0.14364340372227793f));
        q = fma2(t, q, same(0.1141936688535498f));
        q = fma2(t, q, same(0.12000449997269431f));
        const Pair tail = mul2(mul2(q, t), e);
        const float2 r = both(tail), above = both(fma2(tail, same(-1.0f), same(1.0f)));
        const Pair p = pair(s.x < 0.0f ? r.x : above.x, s.y < 0.0f ? r.y : above.y);
        slope = fma2(mul2(z, same(0.39894228040143268f)), e, p);
        return ADD ? fma2(z, p, added) : mul2(z, p);
    }
    slope = same(1.0f);
    return ADD ? add2(z, added) : z;
}

template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float a, float b) {
    uint32_t r;
    if constexpr (std::is_same<T, __half>::value) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
template <typename T>
__device__ __forceinline__ float2 unpack_pair(uint32_t v) {
    if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&v));
    else return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}

// Rows [begin, end) of group g: offsets clamped to [0, rows], so no offset reads or writes out of range.
__device__ __forceinline__ long long clamp_offset(long long offset, long long rows) { return min(rows, max(0ll, offset)); }
__device__ __forceinline__ void group_rows(const int* offsets, int g, long long rows, long long& begin, long long& end) {
    if (!offsets) {
        begin = 0;
        end = rows;
        return;
    }
    begin = g == 0 ? 0 : clamp_offset(offsets[g], rows);
    end = max(begin, clamp_offset(offsets[g + 1], rows));
}

// The rows of a unit of work: chunk rows of a group, or of the rows of no group (g = groups).  Found by one warp.
struct Unit {
    int g;
    int index;          // among all units
    long long from, to;
};
template <bool EVERY_GROUP>  // a group without rows has a unit too
__device__ __forceinline__ Unit unit_at(const int* offsets, int groups, long long rows, long long chunk, int unit) {
    const int lane = threadIdx.x & 31;
    Unit u{-1, unit, 0, 0};
    int before = 0;
    for (int g0 = 0; g0 <= groups && u.g < 0; g0 += 32) {
        const int g = g0 + lane;
        long long from = 0, to = 0;
        if (g < groups) {
            group_rows(offsets, g, rows, from, to);
        } else if (g == groups) {
            long long b;
            group_rows(offsets, groups - 1, rows, b, from);
            to = rows;
        }
        int count = int((to - from + chunk - 1) / chunk);
        if (EVERY_GROUP && g < groups) count = max(1, count);
        int sum = count;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int other = __shfl_up_sync(0xffffffffu, sum, d);
            if (lane >= d) sum += other;
        }
        const int first = before + sum - count;
        const uint32_t found = __ballot_sync(0xffffffffu, unit >= first && unit < first + count);
        if (found) {
            const int at = __ffs(found) - 1;
            u.g = g0 + at;
            from = __shfl_sync(0xffffffffu, from, at) + (long long)(unit - __shfl_sync(0xffffffffu, first, at)) * chunk;
            to = __shfl_sync(0xffffffffu, to, at);
            u.from = from;
            u.to = min(to, from + chunk);
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
    }
    return u;
}

}  // namespace odie
