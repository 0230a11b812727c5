// Rows of a router's logits, held by groups of lanes (gate.cu, balance.cu).
#pragma once
#include "activation.cuh"
#include <initializer_list>
#include <type_traits>

namespace odie {

constexpr int MAX_EXPERTS = 1024;
constexpr int LOGIT_THREADS = 256;

enum GateScore : int { SCORE_SOFTMAX = 0, SCORE_SIGMOID = 1 };

// What a row may take: mask[row * row_step + e * expert_step] != 0 (steps of 0 repeat one value); null: everything.
struct Mask {
    const uint8_t* at;
    long long row_step, expert_step;
};

// A row of E logits among LANES lanes of a warp, V per lane in runs of 8: lane l has experts (c * LANES + l) * 8 + i,
// c < V / 8, i < 8.  So neighbouring lanes read neighbouring 16 bytes.  The kernels are bound by their instructions, of
// which a good part is per lane and row: 16 values to a lane rather than 8 up to 128 experts (2^20 rows of 16 fp16, one choice
// by the softmax: 14.5 us, with 8 to a lane 19.2).
struct LogitShape {
    long long rows;
    int experts;
    int wide;       // every row starts on a 16-byte boundary
    int mask_wide;  // every row of the mask on an 8-byte one, its experts side by side
};
inline LogitShape logit_shape(int64_t rows, int experts, int dtype, std::initializer_list<const void*> pointers, const Mask& mask) {
    LogitShape s{rows, experts, 0, 0};
    uintptr_t bits = uintptr_t(experts) * row_type_size(dtype);
    for (const void* p : pointers) bits |= uintptr_t(p);
    s.wide = bits % 16 == 0 && experts % 8 == 0;
    s.mask_wide = mask.at && mask.expert_step == 1 && (uintptr_t(mask.at) | uintptr_t(mask.row_step) | uintptr_t(experts)) % 8 == 0;
    return s;
}
struct LogitLanes {
    int lanes, values;
};
inline LogitLanes logit_lanes(int experts) {
    if (experts <= 8) return {1, 8};
    if (experts <= 128) return {experts <= 16 ? 1 : experts <= 32 ? 2 : experts <= 64 ? 4 : 8, 16};
    return {32, experts <= 256 ? 8 : experts <= 512 ? 16 : 32};
}
inline int64_t logit_blocks(int64_t rows, int experts) {
    const int per_block = LOGIT_THREADS / logit_lanes(experts).lanes;
    return (rows + per_block - 1) / per_block;
}

// Calls f(T{}, integral_constant<int, V>{}, integral_constant<int, LANES>{}) for the type and number of experts.
template <typename F>
void with_logits(int dtype, int experts, F&& f) {
    auto typed = [&](auto v, auto lanes) {
        if (dtype == ROW_F32) f(float{}, v, lanes);
        else if (dtype == ROW_BF16) f(__nv_bfloat16{}, v, lanes);
        else f(__half{}, v, lanes);
    };
    using std::integral_constant;
    const LogitLanes l = logit_lanes(experts);
    const integral_constant<int, 8> v8{};
    const integral_constant<int, 16> v16{};
    if (l.values == 32) typed(integral_constant<int, 32>{}, integral_constant<int, 32>{});
    else if (l.values == 8) l.lanes == 1 ? typed(v8, integral_constant<int, 1>{}) : typed(v8, integral_constant<int, 32>{});
    else if (l.lanes == 1) typed(v16, integral_constant<int, 1>{});
    else if (l.lanes == 2) typed(v16, integral_constant<int, 2>{});
    else if (l.lanes == 4) typed(v16, integral_constant<int, 4>{});
    else if (l.lanes == 8) typed(v16, integral_constant<int, 8>{});
    else typed(v16, integral_constant<int, 32>{});
}

constexpr float NOTHING = -INFINITY;

// The first expert of a lane's c-th run.
template <int LANES>
__device__ __forceinline__ int run_at(int c, int lane) { return (c * LANES + lane) * 8; }

// The lane's logits of a row; NOTHING where the mask is off or no expert is, and everywhere for a row that is not (`inside`).
template <typename T, int V, int LANES>
__device__ __forceinline__ void load_logits(const T* logits, const LogitShape& s, const Mask& mask, long long row, bool inside, int lane,
                                            float (&v)[V]) {
    constexpr int PER = 16 / int(sizeof(T));
    const T* at = logits + row * s.experts;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = NOTHING;
#pragma unroll
    for (int c = 0; c < V / 8; ++c) {
        const int e0 = run_at<LANES>(c, lane);
        if (!inside || e0 >= s.experts) continue;
        if (s.wide) {
#pragma unroll
            for (int p = 0; p < 8 / PER; ++p) {
                const auto x = Pack<T, 16>::load(at + e0 + p * PER);
#pragma unroll
                for (int i = 0; i < PER; ++i) v[c * 8 + p * PER + i] = to_float(x.v[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (e0 + i < s.experts) v[c * 8 + i] = to_float(at[e0 + i]);
        }
        if (!mask.at) continue;
        const uint8_t* m = mask.at + row * mask.row_step;
        if (s.mask_wide) {
            const uint2 bytes = __ldg(reinterpret_cast<const uint2*>(m + e0));
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (((i < 4 ? bytes.x : bytes.y) >> (i % 4 * 8) & 0xff) == 0) v[c * 8 + i] = NOTHING;
        } else if (mask.expert_step == 0) {
            if (*m == 0) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[c * 8 + i] = NOTHING;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (e0 + i < s.experts && m[(e0 + i) * mask.expert_step] == 0) v[c * 8 + i] = NOTHING;
        }
    }
}

template <typename T, int V, int LANES>
__device__ __forceinline__ void store_logits(T* to, const LogitShape& s, long long row, int lane, const float (&v)[V]) {
    constexpr int PER = 16 / int(sizeof(T));
    T* at = to + row * s.experts;
#pragma unroll
    for (int c = 0; c < V / 8; ++c) {
        const int e0 = run_at<LANES>(c, lane);
        if (e0 >= s.experts) continue;
        if (s.wide) {
#pragma unroll
            for (int p = 0; p < 8 / PER; ++p) {
                Pack<T, 16> x;
                if constexpr (sizeof(T) == 4) {
#pragma unroll
                    for (int i = 0; i < PER; ++i) x.v[i] = v[c * 8 + p * PER + i];
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) reinterpret_cast<uint32_t*>(x.v)[i] = pack_pair<T>(v[c * 8 + 2 * i], v[c * 8 + 2 * i + 1]);
                }
                x.store(at + e0 + p * PER);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (e0 + i < s.experts) at[e0 + i] = from_float<T>(v[c * 8 + i]);
        }
    }
}

// Over the lanes of a row (all lanes of the warp take part).
template <int LANES>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int d = 1; d < LANES; d *= 2) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}
template <int LANES>
__device__ __forceinline__ float group_max(float v) {  // a NaN stays
#pragma unroll
    for (int d = 1; d < LANES; d *= 2) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, d));
    return v;
}
template <int V>
__device__ __forceinline__ float largest(const float (&v)[V]) {
    float top = v[0];
#pragma unroll
    for (int i = 1; i < V; ++i) top = max_nan(top, v[i]);
    return top;
}

constexpr float LOG2E = 1.4426950408889634f;
// e^(v - top), within 2^-22 of it and the rounding of its exponent.  (The difference first: a multiple of the lowest number
// is -inf.)
__device__ __forceinline__ float power(float v, float top) { return exp2_approx((v - top) * LOG2E); }
// In place, with the sum.
template <int V>
__device__ __forceinline__ float powers(float (&v)[V], float top) {
    Pair sum = same(0.0f);
#pragma unroll
    for (int i = 0; i < V; i += 2) {
        const float2 x = both(mul2(add2(pair(v[i], v[i + 1]), same(-top)), same(LOG2E)));
        v[i] = exp2_approx(x.x);
        v[i + 1] = exp2_approx(x.y);
        sum = add2(sum, pair(v[i], v[i + 1]));
    }
    const float2 s = both(sum);
    return s.x + s.y;
}

// sigmoid(v) from e^-|v|, which both sigmoid(v) and sigmoid(-v) come from without cancellation.
__device__ __forceinline__ float sigmoid_of(float v) {
    const float e = exp2_approx(-fabsf(v) * LOG2E);
    return (v >= 0.0f ? 1.0f : e) * inverse_approx(1.0f + e);  // (NaN: e is)
}
// sigmoid(v) / e^low, low <= 0 the least of 0 and the row's largest logit: not all of a row's underflow.
__device__ __forceinline__ float sigmoid_over(float v, float low) {
    const float r = power(fminf(v, 0.0f), low) * inverse_approx(1.0f + exp2_approx(-fabsf(v) * LOG2E));
    return v != v ? v : r;
}

void check_logits(int64_t rows, int experts, int dtype, int score);

}  // namespace odie
