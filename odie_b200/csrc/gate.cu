// The experts of each row and their weights from a router's logits, and the weights' gradient.
//
//   key_e    = fp32(logit_e) + bias_e, for experts whose mask is on and whose key is not -inf
//   choices  = the k highest keys, ties to the lowest expert; -1 where none is left
//   s_e      = softmax over the row (mask on), or sigmoid(logit_e)
//   weight_j = scale s_j, or scale s_j / (sum of the chosen s)
//
// The key has no transcendental function in it, so that which experts a row takes does not depend on how one is
// rounded; the bias shifts choices and not weights, and has no gradient.  A softmax over the chosen logits is the
// normalised softmax over all, so that nothing but the chosen is read for it; normalised sigmoids are taken by their
// logarithms, which do not underflow.
//
//   backward, with g = d weight, p = s (normalised: divided by the sum):
//     softmax, normalised   d l_j = w_j (g_j - sum w g / scale)              at the chosen, 0 elsewhere
//     softmax               d l_e = scale p_e ([e chosen] g_e - sum p_j g_j)
//     sigmoid, normalised   d l_j = w_j (1 - s_j) (g_j - sum w g / scale)
//     sigmoid               d l_j = w_j (1 - s_j) g_j
#include "logits.cuh"
#include "odie_b200.h"
#include <cmath>

namespace odie {

void check_logits(int64_t rows, int experts, int dtype, int score) {
    ODIE_REQUIRE(rows >= 0 && rows < (int64_t(1) << 31), "0 to 2^31 - 1 rows");
    ODIE_REQUIRE(experts >= 1 && experts <= MAX_EXPERTS, "1 to 1024 experts");
    check_row_type(dtype);
    ODIE_REQUIRE(score == SCORE_SOFTMAX || score == SCORE_SIGMOID, "score must be 0 (softmax) or 1 (sigmoid)");
}

namespace {

constexpr int MAX_CHOICES = 64;

struct GateArgs {
    const void* logits;
    const float* bias;  // null: none
    Mask mask;
    int choices;
    int score;
    int normalize;
    float scale;
    int* expert;
    float* weights;
    // backward
    const float* d_weights;
    void* d_logits;
};

// The order of keys as unsigned numbers: 0 for what is not there, a NaN above all; -0 and 0 are one key.
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t bits = __float_as_uint(v + 0.0f);
    const uint32_t key = bits ^ (bits >> 31 ? 0xffffffffu : 0x80000000u);
    return v != v ? 0xffffffffu : v == NOTHING ? 0u : key;
}

template <typename T, int V>
__global__ void __launch_bounds__(LOGIT_THREADS) gate_kernel(GateArgs a, LogitShape s) {
    // Choice j is kept by lane j % lanes, in slot j / lanes: lanes x 8 cover the experts, so 8 slots cover the choices.
    constexpr int SLOTS = 8;
    const int lanes = 1 << s.lanes_log2, lane = threadIdx.x & (lanes - 1);
    const long long row = (long long)blockIdx.x * (LOGIT_THREADS >> s.lanes_log2) + (threadIdx.x >> s.lanes_log2);
    const bool inside = row < s.rows;
    const T* logits = static_cast<const T*>(a.logits);
    float v[V];
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = NOTHING;
    if (inside) load_logits<T, V>(logits, s, a.mask, row, lane, v);

    uint32_t key[V];
#pragma unroll
    for (int c = 0; c < V / 8; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int e = ((c << s.lanes_log2) + lane) * 8 + i;
            const float z = v[c * 8 + i];
            key[c * 8 + i] = ordered(a.bias && e < s.experts && z != NOTHING ? z + __ldg(a.bias + e) : z);
        }
    int chosen[SLOTS];
#pragma unroll
    for (int q = 0; q < SLOTS; ++q) chosen[q] = -1;
#pragma unroll
    for (int q = 0; q < SLOTS; ++q) {
        for (int t = 0; t < lanes && q * lanes + t < a.choices; ++t) {
            uint32_t best = 0;
#pragma unroll
            for (int i = 0; i < V; ++i) best = max(best, key[i]);
            for (int d = 1; d < lanes; d *= 2) best = max(best, __shfl_xor_sync(0xffffffffu, best, d));
            int at = MAX_EXPERTS;
#pragma unroll
            for (int i = V - 1; i >= 0; --i)
                if (key[i] == best) at = (((i / 8) << s.lanes_log2) + lane) * 8 + i % 8;
            for (int d = 1; d < lanes; d *= 2) at = min(at, __shfl_xor_sync(0xffffffffu, at, d));
#pragma unroll
            for (int i = 0; i < V; ++i)
                if ((((i / 8) << s.lanes_log2) + lane) * 8 + i % 8 == at) key[i] = 0;
            if (t == lane && best) chosen[q] = at;
        }
    }

    float l[SLOTS], w[SLOTS];
#pragma unroll
    for (int q = 0; q < SLOTS; ++q) l[q] = chosen[q] >= 0 ? to_float(logits[row * s.experts + chosen[q]]) : NOTHING;
    if (a.score == SCORE_SOFTMAX || a.normalize) {
        // a softmax of the chosen logits, or of the logarithms of their sigmoids; without normalize of all logits
        if (a.score == SCORE_SIGMOID) {
#pragma unroll
            for (int q = 0; q < SLOTS; ++q) l[q] = chosen[q] >= 0 ? log_sigmoid(l[q]) : NOTHING;
        }
        float top = NOTHING, sum = 0.0f;
        if (a.normalize) {
#pragma unroll
            for (int q = 0; q < SLOTS; ++q) top = l[q] > top || l[q] != l[q] ? l[q] : top;
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) top = v[i] > top || v[i] != v[i] ? v[i] : top;
        }
        top = group_max(top, s.lanes_log2);
        if (top == NOTHING) top = 0.0f;
        if (a.normalize) {
#pragma unroll
            for (int q = 0; q < SLOTS; ++q) sum += chosen[q] >= 0 ? expf(l[q] - top) : 0.0f;
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) sum += expf(v[i] - top);
        }
        sum = group_sum(sum, s.lanes_log2);
#pragma unroll
        for (int q = 0; q < SLOTS; ++q) w[q] = a.scale * (expf(l[q] - top) / sum);
    } else {
#pragma unroll
        for (int q = 0; q < SLOTS; ++q) w[q] = a.scale * sigmoid_of(l[q]);
    }
    if (!inside) return;
#pragma unroll
    for (int q = 0; q < SLOTS; ++q) {
        const int j = q * lanes + lane;
        if (j >= a.choices) break;
        a.expert[row * a.choices + j] = chosen[q];
        a.weights[row * a.choices + j] = chosen[q] >= 0 ? w[q] : 0.0f;
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(LOGIT_THREADS) gate_backward_kernel(GateArgs a, LogitShape s) {
    constexpr int SLOTS = 8;
    const int lanes = 1 << s.lanes_log2, lane = threadIdx.x & (lanes - 1);
    const long long row = (long long)blockIdx.x * (LOGIT_THREADS >> s.lanes_log2) + (threadIdx.x >> s.lanes_log2);
    const bool inside = row < s.rows;
    const T* logits = static_cast<const T*>(a.logits);
    const bool dense = a.score == SCORE_SOFTMAX && !a.normalize;

    // d l at the chosen experts, but for what all experts share
    int chosen[SLOTS];
    float w[SLOTS], d[SLOTS], sum = 0.0f;
#pragma unroll
    for (int q = 0; q < SLOTS; ++q) {
        const int j = q * lanes + lane;
        chosen[q] = -1;
        w[q] = d[q] = 0.0f;
        if (!inside || j >= a.choices) continue;
        const long long at = row * a.choices + j;
        const int e = a.expert[at];
        if (unsigned(e) >= unsigned(s.experts)) continue;
        chosen[q] = e;
        w[q] = a.weights[at];
        d[q] = a.d_weights[at];
        sum += w[q] * d[q];
    }
    sum = group_sum(sum, s.lanes_log2);
    const float mean = a.normalize || dense ? sum / a.scale : 0.0f;
#pragma unroll
    for (int q = 0; q < SLOTS; ++q) {
        if (chosen[q] < 0) continue;
        d[q] = w[q] * (dense ? d[q] : d[q] - mean);
        if (a.score == SCORE_SIGMOID) d[q] *= sigmoid_of(-to_float(logits[row * s.experts + chosen[q]]));
    }

    float v[V];
    if (dense) {  // - scale p_e sum p g
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = NOTHING;
        if (inside) load_logits<T, V>(logits, s, a.mask, row, lane, v);
        float top = NOTHING, total = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) top = v[i] > top || v[i] != v[i] ? v[i] : top;
        top = group_max(top, s.lanes_log2);
        if (top == NOTHING) top = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            v[i] = expf(v[i] - top);
            total += v[i];
        }
        total = group_sum(total, s.lanes_log2);
        const float share = total > 0.0f || total != total ? sum / total : 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] *= -share;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = 0.0f;
    }
#pragma unroll
    for (int q = 0; q < SLOTS; ++q) {
        for (int t = 0; t < lanes && q * lanes + t < a.choices; ++t) {
            const int e = __shfl_sync(0xffffffffu, chosen[q], t, lanes);
            const float add = __shfl_sync(0xffffffffu, d[q], t, lanes);
#pragma unroll
            for (int i = 0; i < V; ++i)
                if ((((i / 8) << s.lanes_log2) + lane) * 8 + i % 8 == e) v[i] += add;
        }
    }
    if (inside) store_logits<T, V>(static_cast<T*>(a.d_logits), s, row, lane, v);
}

void check_gate(int64_t rows, int experts, int choices, int dtype, int score, float scale) {
    check_logits(rows, experts, dtype, score);
    ODIE_REQUIRE(choices >= 1 && choices <= experts && choices <= MAX_CHOICES, "1 to 64 choices, no more than experts");
    ODIE_REQUIRE(rows * choices < (int64_t(1) << 31), "too many (row, choice) pairs");
    ODIE_REQUIRE(std::isfinite(scale) && scale != 0.0f, "scale must be finite and not 0");
}

}  // namespace
}  // namespace odie

using namespace odie;

extern "C" int odie_gate(const void* logits, int64_t rows, int experts, int dtype, const float* bias, const uint8_t* mask,
                         int64_t mask_row_step, int64_t mask_expert_step, int choices, int score, int normalize, float scale,
                         int32_t* expert, float* weights, uint64_t stream) {
    return guarded([&] {
        check_gate(rows, experts, choices, dtype, score, scale);
        if (rows == 0) return;
        ODIE_REQUIRE(logits && expert && weights, "logits, expert and weights are required");
        GateArgs a{};
        a.logits = logits;
        a.bias = bias;
        a.mask = {mask, mask_row_step, mask_expert_step};
        a.choices = choices;
        a.score = score;
        a.normalize = normalize != 0;
        a.scale = scale;
        a.expert = expert;
        a.weights = weights;
        const LogitShape s = logit_shape(rows, experts, dtype, {logits}, a.mask);
        with_logits(dtype, experts, [&](auto type, auto v) {
            gate_kernel<decltype(type), decltype(v)::value>
                <<<unsigned(logit_blocks(s)), LOGIT_THREADS, 0, reinterpret_cast<cudaStream_t>(stream)>>>(a, s);
        });
        ODIE_CUDA(cudaGetLastError());
        note_launch();
    });
}

extern "C" int odie_gate_backward(const float* d_weights, const void* logits, int64_t rows, int experts, int dtype, const uint8_t* mask,
                                  int64_t mask_row_step, int64_t mask_expert_step, const int32_t* expert, const float* weights,
                                  int choices, int score, int normalize, float scale, void* d_logits, uint64_t stream) {
    return guarded([&] {
        check_gate(rows, experts, choices, dtype, score, scale);
        if (rows == 0) return;
        ODIE_REQUIRE(d_weights && expert && weights && d_logits, "d_weights, expert, weights and d_logits are required");
        ODIE_REQUIRE(logits || (score == SCORE_SOFTMAX && normalize), "logits are required but for a normalised softmax");
        GateArgs a{};
        a.logits = logits;
        a.mask = {mask, mask_row_step, mask_expert_step};
        a.choices = choices;
        a.score = score;
        a.normalize = normalize != 0;
        a.scale = scale;
        a.expert = const_cast<int32_t*>(expert);
        a.weights = const_cast<float*>(weights);
        a.d_weights = d_weights;
        a.d_logits = d_logits;
        const LogitShape s = logit_shape(rows, experts, dtype, {logits, d_logits}, a.mask);
        with_logits(dtype, experts, [&](auto type, auto v) {
            gate_backward_kernel<decltype(type), decltype(v)::value>
                <<<unsigned(logit_blocks(s)), LOGIT_THREADS, 0, reinterpret_cast<cudaStream_t>(stream)>>>(a, s);
        });
        ODIE_CUDA(cudaGetLastError());
        note_launch();
    });
}
