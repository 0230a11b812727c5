// The experts of each row and their weights from a router's logits, and the weights' gradient.
//
//   key_e    = fp32(logit_e) + bias_e, for experts whose mask is on and of which neither logit nor key is -inf
//   choices  = the k highest keys, ties to the lowest expert; -1 where none is left
//   s_e      = softmax over the row (mask on), or sigmoid(logit_e)
//   weight_j = scale s_j, or scale s_j / (sum of the chosen s)
//
// The key has no transcendental function in it, so that which experts a row takes does not depend on how one is
// rounded; the bias shifts choices and not weights, and has no gradient.  A softmax over the chosen logits is the
// normalised softmax over all, so that nothing but the chosen is read for it.
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
    int bias_wide;      // on a 16-byte boundary
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

// The order of keys as unsigned numbers: a NaN (which an addition makes positive) above all, -0 and 0 one key.
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t bits = __float_as_uint(v + 0.0f);
    return bits ^ (uint32_t(int(bits) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t key) { return __uint_as_float(key >> 31 ? key ^ 0x80000000u : ~key); }
constexpr uint32_t NO_KEY = 0x007fffffu;  // -inf, and what was taken (0)

template <int LANES>
__device__ __forceinline__ uint32_t group_highest(uint32_t v) {
    if constexpr (LANES == 32) {
        return __reduce_max_sync(0xffffffffu, v);
    } else {
#pragma unroll
        for (int d = 1; d < LANES; d *= 2) v = max(v, __shfl_xor_sync(0xffffffffu, v, d));
        return v;
    }
}
template <int LANES>
__device__ __forceinline__ int group_lowest(int v) {
    if constexpr (LANES == 32) {
        return __reduce_min_sync(0xffffffffu, v);
    } else {
#pragma unroll
        for (int d = 1; d < LANES; d *= 2) v = min(v, __shfl_xor_sync(0xffffffffu, v, d));
        return v;
    }
}

// The choices one after another: the highest key, the lowest expert that has it, which is taken out.  Choice j goes to lane
// j % LANES, slot j / LANES.
template <int V, int LANES, int SLOTS>
__device__ __forceinline__ void choose(uint32_t (&key)[V], int choices, int lane, int (&chosen)[SLOTS], uint32_t (&won)[SLOTS], uint32_t& most) {
#pragma unroll
    for (int q = 0; q < SLOTS; ++q) {
        chosen[q] = -1;
        won[q] = NO_KEY;
#pragma unroll 1
        for (int t = 0; t < LANES && q * LANES + t < choices; ++t) {
            uint32_t best = key[0];
#pragma unroll
            for (int i = 1; i < V; ++i) best = max(best, key[i]);
            best = group_highest<LANES>(best);
            if (q == 0 && t == 0) most = best;
            int at = MAX_EXPERTS;
#pragma unroll
            for (int i = V - 1; i >= 0; --i)
                if (key[i] == best) at = run_at<LANES>(i / 8, lane) + i % 8;
            at = group_lowest<LANES>(at);
            if (t == lane && best > NO_KEY) {
                chosen[q] = at;
                won[q] = best;
            }
            if (q * LANES + t + 1 < choices) {
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (run_at<LANES>(i / 8, lane) + i % 8 == at) key[i] = 0;
            }
        }
    }
}

// The same for a warp to a row and 8 keys to a lane, for many choices: each lane sorts its keys first, so that a choice is the
// highest of the lanes' first ones and the lane that had it moves up.  (65536 rows of 256 bf16 with a bias, in us: 17 choices
// one after another 101, sorted 60 to 66; 32 choices 175 and 87.)
// `at` is where a key was in its lane; the lower lane has the lower experts.
__device__ __forceinline__ void exchange(uint32_t& a, uint32_t& b, int& at_a, int& at_b) {
    const bool turn = b > a || (b == a && at_b < at_a);
    const uint32_t high = turn ? b : a, low = turn ? a : b;
    const int at_high = turn ? at_b : at_a, at_low = turn ? at_a : at_b;
    a = high;
    b = low;
    at_a = at_high;
    at_b = at_low;
}
template <int SLOTS>
__device__ __forceinline__ void choose_sorted(uint32_t (&key)[8], int choices, int lane, int (&chosen)[SLOTS], uint32_t (&won)[SLOTS], uint32_t& most) {
    int at[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) at[i] = i;
    // Batcher's odd-even merge sort of eight
    constexpr int PAIRS[19][2] = {{0, 1}, {2, 3}, {4, 5}, {6, 7}, {0, 2}, {1, 3}, {4, 6}, {5, 7}, {1, 2}, {5, 6},
                                  {0, 4}, {1, 5}, {2, 6}, {3, 7}, {2, 4}, {3, 5}, {1, 2}, {3, 4}, {5, 6}};
#pragma unroll
    for (int i = 0; i < 19; ++i) exchange(key[PAIRS[i][0]], key[PAIRS[i][1]], at[PAIRS[i][0]], at[PAIRS[i][1]]);
    uint32_t places = 0;  // four bits each, the first lowest
#pragma unroll
    for (int i = 0; i < 8; ++i) places |= uint32_t(at[i]) << (4 * i);
#pragma unroll
    for (int q = 0; q < SLOTS; ++q) {
        chosen[q] = -1;
        won[q] = NO_KEY;
#pragma unroll 1
        for (int t = 0; t < 32 && q * 32 + t < choices; ++t) {
            const uint32_t best = __reduce_max_sync(0xffffffffu, key[0]);
            if (q == 0 && t == 0) most = best;
            const int winner = __ffs(__ballot_sync(0xffffffffu, key[0] == best)) - 1;
            const int e = winner * 8 + int(__shfl_sync(0xffffffffu, places, winner) & 15);
            if (t == lane && best > NO_KEY) {
                chosen[q] = e;
                won[q] = best;
            }
            if (lane == winner) {
#pragma unroll
                for (int i = 0; i < 7; ++i) key[i] = key[i + 1];
                key[7] = 0;
                places >>= 4;
            }
        }
    }
}

// And for 4 to FILTERED choices: the k-th highest of the lanes' highest keys is a bound that at least k keys reach, and few
// more; these are gathered, and each counts those before it.  (4, 8 and 16 choices of the rows above: 31, 36 and 45 us;
// sorted 37, 46 and 64; one after another 35, 56 and 95; 3 choices one after another 31.)  false: more than 32 reach it (many
// ties), choose_sorted takes the row.  found: [64] of the warp.
constexpr int FILTERED = 16;
template <int SLOTS>
__device__ __forceinline__ bool choose_filtered(const uint32_t (&key)[8], int choices, int lane, int (&chosen)[SLOTS], uint32_t (&won)[SLOTS],
                                                uint32_t& most, uint2* found) {
    uint32_t high = key[0], bound = 0;
#pragma unroll
    for (int i = 1; i < 8; ++i) high = max(high, key[i]);
    for (int t = 0; t < choices; ++t) {  // lanes with one and the same key leave together: the bound is lower then
        bound = __reduce_max_sync(0xffffffffu, high);
        if (t == 0) most = bound;
        if (high == bound) high = 0;
    }
    bound = max(bound, NO_KEY + 1);
    const uint32_t before = (1u << lane) - 1;
    int count = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t reach = __ballot_sync(0xffffffffu, key[i] >= bound);
        const int at = count + __popc(reach & before);
        if (key[i] >= bound && at < 32) found[at] = make_uint2(key[i], lane * 8 + i);
        count += __popc(reach);
    }
    if (count > 32) return false;
    __syncwarp();
    const uint2 mine = lane < count ? found[lane] : make_uint2(0, 0);
    int rank = 0;
    for (int i = 0; i < count; ++i) {
        const uint2 other = found[i];
        rank += other.x > mine.x || (other.x == mine.x && other.y < mine.y);
    }
    if (lane < count && rank < choices) found[32 + rank] = mine;
    __syncwarp();
    chosen[0] = -1;
    won[0] = NO_KEY;
    if (lane < min(count, choices)) {
        const uint2 taken = found[32 + lane];
        chosen[0] = int(taken.y);
        won[0] = taken.x;
    }
    __syncwarp();  // found is free again
    return true;
}

// As few slots as hold the choices are compiled for: never more than V, nor than hold 64.
template <typename T, int V, int LANES, int SLOTS>
__global__ void __launch_bounds__(LOGIT_THREADS) gate_kernel(GateArgs a, LogitShape s) {
    const int lane = threadIdx.x & (LANES - 1);
    const long long row = (long long)blockIdx.x * (LOGIT_THREADS / LANES) + threadIdx.x / LANES;
    const bool inside = row < s.rows;
    const T* logits = static_cast<const T*>(a.logits);
    float v[V];
    load_logits<T, V, LANES>(logits, s, a.mask, row, inside, lane, v);

    uint32_t key[V], most = 0;  // most: the highest key of all
    if (a.bias) {
#pragma unroll
        for (int c = 0; c < V / 4; ++c) {
            const int e = run_at<LANES>(c / 2, lane) + c % 2 * 4;
            float4 b = make_float4(0, 0, 0, 0);
            if (e + 4 <= s.experts && a.bias_wide) {
                b = __ldg(reinterpret_cast<const float4*>(a.bias + e));
            } else {
                if (e < s.experts) b.x = __ldg(a.bias + e);
                if (e + 1 < s.experts) b.y = __ldg(a.bias + e + 1);
                if (e + 2 < s.experts) b.z = __ldg(a.bias + e + 2);
                if (e + 3 < s.experts) b.w = __ldg(a.bias + e + 3);
            }
            const float add[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) key[c * 4 + i] = v[c * 4 + i] == NOTHING ? NO_KEY : ordered(v[c * 4 + i] + add[i]);  // (the bias may be infinite)
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) key[i] = ordered(v[i]);
    }
    int chosen[SLOTS];
    uint32_t won[SLOTS];  // their keys
    if constexpr (LANES == 32 && V == 8) {
        __shared__ uint2 found[LOGIT_THREADS / 32][64];
        if (SLOTS == 1 && a.choices > 3 && a.choices <= FILTERED &&
            choose_filtered<SLOTS>(key, a.choices, lane, chosen, won, most, found[threadIdx.x / 32])) {
        } else if (a.choices > 3) choose_sorted<SLOTS>(key, a.choices, lane, chosen, won, most);
        else choose<V, LANES, SLOTS>(key, a.choices, lane, chosen, won, most);
    } else {
        choose<V, LANES, SLOTS>(key, a.choices, lane, chosen, won, most);
    }

    float l[SLOTS], w[SLOTS];
#pragma unroll
    for (int q = 0; q < SLOTS; ++q) l[q] = a.bias && chosen[q] >= 0 ? to_float(logits[row * s.experts + chosen[q]]) : unordered(won[q]);
    if (a.score == SCORE_SOFTMAX || a.normalize) {  // e^(l - top), or sigmoids over e^top, over their sum (without normalize: of all)
        float top, sum = 0.0f;
        if (a.normalize) top = group_max<LANES>(largest(l));
        else if (!a.bias) top = unordered(most);
        else top = group_max<LANES>(largest(v));
        if (top == NOTHING) top = 0.0f;
        if (a.score == SCORE_SIGMOID) top = fminf(top, 0.0f);
#pragma unroll
        for (int q = 0; q < SLOTS; ++q) {
            w[q] = a.score == SCORE_SIGMOID ? sigmoid_over(l[q], top) : power(l[q], top);
            if (chosen[q] < 0) w[q] = 0.0f;
        }
        if (a.normalize) {
#pragma unroll
            for (int q = 0; q < SLOTS; ++q) sum += w[q];
        } else {
            sum = powers(v, top);
        }
        const float scale = a.scale * inverse_approx(group_sum<LANES>(sum));
#pragma unroll
        for (int q = 0; q < SLOTS; ++q) w[q] *= scale;
    } else {
#pragma unroll
        for (int q = 0; q < SLOTS; ++q) w[q] = a.scale * sigmoid_of(l[q]);
    }
    if (!inside) return;
#pragma unroll
    for (int q = 0; q < SLOTS; ++q) {
        const int j = q * LANES + lane;
        if (j >= a.choices) break;
        a.expert[row * a.choices + j] = chosen[q];
        a.weights[row * a.choices + j] = chosen[q] >= 0 ? w[q] : 0.0f;
    }
}

// Word i of the rows in shared memory: their 16-byte units permuted so that lanes that read V words each meet no bank twice.
__device__ __forceinline__ int spread(int i) { return i ^ (i >> 3 & 12); }

template <typename T, int V, int LANES, int SLOTS>
__global__ void __launch_bounds__(LOGIT_THREADS) gate_backward_kernel(GateArgs a, LogitShape s) {
    // where the lanes that have a choice find the lane that has its expert
    __shared__ alignas(16) float rows[LOGIT_THREADS * V];
    const int lane = threadIdx.x & (LANES - 1);
    const long long row = (long long)blockIdx.x * (LOGIT_THREADS / LANES) + threadIdx.x / LANES;
    const bool inside = row < s.rows;
    const T* logits = static_cast<const T*>(a.logits);
    const bool dense = a.score == SCORE_SOFTMAX && !a.normalize;

    float v[V];
    if (dense) load_logits<T, V, LANES>(logits, s, a.mask, row, inside, lane, v);
    // d l at the chosen experts, but for what all experts share
    int chosen[SLOTS];
    float w[SLOTS], d[SLOTS], sum = 0.0f;
#pragma unroll
    for (int q = 0; q < SLOTS; ++q) {
        const int j = q * LANES + lane;
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
    const int mine = threadIdx.x / LANES * (LANES * V);
#pragma unroll
    for (int c = 0; c < V / 4; ++c) *reinterpret_cast<float4*>(rows + spread(mine + run_at<LANES>(c / 2, lane) + c % 2 * 4)) = make_float4(0, 0, 0, 0);
    if (a.normalize || dense) sum = group_sum<LANES>(sum);
    const float mean = a.normalize ? sum * (1.0f / a.scale) : 0.0f;
    __syncwarp();
#pragma unroll
    for (int q = 0; q < SLOTS; ++q) {
        if (chosen[q] < 0) continue;
        d[q] = w[q] * (d[q] - mean);
        if (a.score == SCORE_SIGMOID) d[q] *= sigmoid_of(-to_float(logits[row * s.experts + chosen[q]]));
        rows[spread(mine + chosen[q])] = d[q];
    }

    bool finite = true;
    if (dense) {  // - scale p_e sum p g
        float top = group_max<LANES>(largest(v));
        if (top == NOTHING) top = 0.0f;
        const float total = group_sum<LANES>(powers(v, top)), share = total > 0.0f || total != total ? -sum * inverse_approx(total) : 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] *= share;
        finite = fabsf(share) < INFINITY;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = 0.0f;
    }
    __syncwarp();
#pragma unroll
    for (int c = 0; c < V / 4; ++c) {
        const float4 add = *reinterpret_cast<const float4*>(rows + spread(mine + run_at<LANES>(c / 2, lane) + c % 2 * 4));
        v[c * 4] += add.x;
        v[c * 4 + 1] += add.y;
        v[c * 4 + 2] += add.z;
        v[c * 4 + 3] += add.w;
    }
    if (!inside) return;
    store_logits<T, V, LANES>(static_cast<T*>(a.d_logits), s, row, lane, v);
    if (finite) return;
    // A row with an open NaN or infinity, or such a gradient: experts that are closed to it have none all the same.  (Here, with
    // nothing in registers, it costs the other rows none of theirs.)
#pragma unroll 1
    for (int i = 0; i < V; ++i) {
        const int e = run_at<LANES>(i / 8, lane) + i % 8;
        if (e >= s.experts) continue;
        const long long at = row * s.experts + e;
        if (to_float(logits[at]) == NOTHING || (a.mask.at && a.mask.at[row * a.mask.row_step + e * a.mask.expert_step] == 0))
            static_cast<T*>(a.d_logits)[at] = from_float<T>(0.0f);
    }
}

template <typename F>
void with_gate(int dtype, int experts, int choices, F&& f) {
    with_logits(dtype, experts, [&](auto type, auto v, auto lanes) {
        constexpr int LANES = decltype(lanes)::value;
        constexpr int V = decltype(v)::value, MOST = V < MAX_CHOICES / LANES ? V : MAX_CHOICES / LANES;
        if (choices <= LANES) f(type, v, lanes, std::integral_constant<int, 1>{});
        else if (choices <= 2 * LANES) f(type, v, lanes, std::integral_constant<int, 2>{});
        else if constexpr (MOST > 2) f(type, v, lanes, std::integral_constant<int, MOST>{});
    });
}

void check_gate(int64_t rows, int experts, int choices, int dtype, int score, float scale) {
    check_logits(rows, experts, dtype, score);
    ODIE_REQUIRE(choices >= 1 && choices <= experts && choices <= MAX_CHOICES, "1 to 64 choices, no more than experts");
    ODIE_REQUIRE(rows * choices < (int64_t(1) << 31), "too many (row, choice) pairs");
    ODIE_REQUIRE(std::isnormal(scale), "scale must be finite and not 0");  // (nor below the least normal number: its inverse is used)
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
        a.bias_wide = uintptr_t(bias) % 16 == 0;
        a.mask = {mask, mask_row_step, mask_expert_step};
        a.choices = choices;
        a.score = score;
        a.normalize = normalize != 0;
        a.scale = scale;
        a.expert = expert;
        a.weights = weights;
        const LogitShape s = logit_shape(rows, experts, dtype, {logits}, a.mask);
        with_gate(dtype, experts, choices, [&](auto type, auto v, auto lanes, auto slots) {
            gate_kernel<decltype(type), decltype(v)::value, decltype(lanes)::value, decltype(slots)::value>
                <<<unsigned(logit_blocks(rows, experts)), LOGIT_THREADS, 0, reinterpret_cast<cudaStream_t>(stream)>>>(a, s);
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
        with_gate(dtype, experts, choices, [&](auto type, auto v, auto lanes, auto slots) {
            gate_backward_kernel<decltype(type), decltype(v)::value, decltype(lanes)::value, decltype(slots)::value>
                <<<unsigned(logit_blocks(rows, experts)), LOGIT_THREADS, 0, reinterpret_cast<cudaStream_t>(stream)>>>(a, s);
        });
        ODIE_CUDA(cudaGetLastError());
        note_launch();
    });
}
