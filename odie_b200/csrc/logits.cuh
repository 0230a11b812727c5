// Rows of a router's logits, held by groups of lanes (gate.cu, balance.cu).
#pragma once
#include "rows.cuh"
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

// A row of E logits among 2^lanes_log2 lanes of a warp, V per lane in runs of 8: lane l has experts
// (c * lanes + l) * 8 + i, c < V / 8, i < 8.  So neighbouring lanes read neighbouring 16 bytes, and up to 8 experts are
// one thread's.
struct LogitShape {
    long long rows;
    int experts;
    int lanes_log2;
    int wide;       // every row starts on a 16-byte boundary
    int mask_wide;  // every row of the mask on an 8-byte one, its experts side by side
};
inline LogitShape logit_shape(int64_t rows, int experts, int dtype, std::initializer_list<const void*> pointers, const Mask& mask) {
    LogitShape s{rows, experts, 0, 0, 0};
    while (s.lanes_log2 < 5 && (8 << s.lanes_log2) < experts) ++s.lanes_log2;
    uintptr_t bits = uintptr_t(experts) * row_type_size(dtype);
    for (const void* p : pointers) bits |= uintptr_t(p);
    s.wide = bits % 16 == 0 && experts % 8 == 0;
    s.mask_wide = mask.at && mask.expert_step == 1 && (uintptr_t(mask.at) | uintptr_t(mask.row_step) | uintptr_t(experts)) % 8 == 0;
    return s;
}
inline int64_t logit_blocks(const LogitShape& s) { return (s.rows + (LOGIT_THREADS >> s.lanes_log2) - 1) / (LOGIT_THREADS >> s.lanes_log2); }

// Calls f(T{}, std::integral_constant<int, V>{}) for the type and values per lane at run time.
template <typename F>
void with_logits(int dtype, int experts, F&& f) {
    auto typed = [&](auto v) {
        if (dtype == ROW_F32) f(float{}, v);
        else if (dtype == ROW_BF16) f(__nv_bfloat16{}, v);
        else f(__half{}, v);
    };
    if (experts <= 256) typed(std::integral_constant<int, 8>{});
    else if (experts <= 512) typed(std::integral_constant<int, 16>{});
    else typed(std::integral_constant<int, 32>{});
}

constexpr float NOTHING = -INFINITY;

// The lane's logits of a row; NOTHING where the mask is off or no expert is.
template <typename T, int V>
__device__ __forceinline__ void load_logits(const T* logits, const LogitShape& s, const Mask& mask, long long row, int lane, float (&v)[V]) {
    constexpr int PER = 16 / int(sizeof(T));
    const T* at = logits + row * s.experts;
#pragma unroll
    for (int c = 0; c < V / 8; ++c) {
        const int e0 = ((c << s.lanes_log2) + lane) * 8;
        if (s.wide) {
#pragma unroll
            for (int p = 0; p < 8 / PER; ++p) {
                Pack<T, 16> x;
                if (e0 < s.experts) x = Pack<T, 16>::load(at + e0 + p * PER);
#pragma unroll
                for (int i = 0; i < PER; ++i) v[c * 8 + p * PER + i] = e0 < s.experts ? to_float(x.v[i]) : NOTHING;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[c * 8 + i] = e0 + i < s.experts ? to_float(at[e0 + i]) : NOTHING;
        }
        if (!mask.at) continue;
        const uint8_t* m = mask.at + row * mask.row_step;
        if (s.mask_wide) {
            if (e0 >= s.experts) continue;
            const uint2 bytes = __ldg(reinterpret_cast<const uint2*>(m + e0));
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (((i < 4 ? bytes.x : bytes.y) >> (i % 4 * 8) & 0xff) == 0) v[c * 8 + i] = NOTHING;
        } else if (mask.expert_step == 0) {
            if (*m == 0)
#pragma unroll
                for (int i = 0; i < 8; ++i) v[c * 8 + i] = NOTHING;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (e0 + i < s.experts && m[(e0 + i) * mask.expert_step] == 0) v[c * 8 + i] = NOTHING;
        }
    }
}

template <typename T, int V>
__device__ __forceinline__ void store_logits(T* to, const LogitShape& s, long long row, int lane, const float (&v)[V]) {
    constexpr int PER = 16 / int(sizeof(T));
    T* at = to + row * s.experts;
#pragma unroll
    for (int c = 0; c < V / 8; ++c) {
        const int e0 = ((c << s.lanes_log2) + lane) * 8;
        if (s.wide) {
            if (e0 >= s.experts) continue;
#pragma unroll
            for (int p = 0; p < 8 / PER; ++p) {
                Pack<T, 16> x;
#pragma unroll
                for (int i = 0; i < PER; ++i) x.v[i] = from_float<T>(v[c * 8 + p * PER + i]);
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
__device__ __forceinline__ float group_sum(float v, int lanes_log2) {
    for (int d = 1; d < 1 << lanes_log2; d *= 2) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}
__device__ __forceinline__ float group_max(float v, int lanes_log2) {  // a NaN stays
    for (int d = 1; d < 1 << lanes_log2; d *= 2) {
        const float other = __shfl_xor_sync(0xffffffffu, v, d);
        v = other > v || other != other ? other : v;
    }
    return v;
}

// e^-|v|, from which both sigmoid(v) and sigmoid(-v) come without cancellation.
__device__ __forceinline__ float sigmoid_of(float v) {
    const float e = expf(-fabsf(v));
    return (v >= 0.0f ? 1.0f : e) / (1.0f + e);  // (NaN: e is)
}
__device__ __forceinline__ float log_sigmoid(float v) { return fminf(v, 0.0f) - log1pf(expf(-fabsf(v))) + (v != v ? v : 0.0f); }

void check_logits(int64_t rows, int experts, int dtype, int score);

}  // namespace odie
