// The balance loss of a router, the mean square of its log-sum-exp, and the rows of each expert, with the gradient.
//
//   T     live rows: with an expert whose mask is on and whose logit is not -inf
//   p     softmax of a live row, or its sigmoids divided by their sum; P_e = (sum over rows of p_e) / T
//   f_e   share of expert e among the choices in [0, E): n_e / N (0 where there are none)
//   loss  = E sum_e f_e P_e, 1 for an even load        z = mean over live rows of lse^2, lse = log sum_e e^logit_e
//   d logit_k = d_loss E/T p_k c_k (f_k - sum_e f_e p_e) + d_z 2/T lse softmax_k,  c = 1 (softmax), 1 - sigmoid
//
// f has no gradient.  Two kernels forward: blocks of rows sum p in fp32 registers, a cluster joins them in 64 bits, in
// the blocks' order; the counts are whole numbers, added by shared-memory atomics.  One kernel backward.
#include "logits.cuh"
#include "odie_b200.h"
#include <cooperative_groups.h>
#include <algorithm>

namespace odie {
namespace {

struct BalanceArgs {
    const void* logits;
    Mask mask;
    int score;
    const void* expert;
    int key_bytes;
    long long pairs;
    // per block of rows
    float* sums;    // [blocks][experts] of p
    int* counts;    // [blocks][experts]
    float* squares; // [blocks] of lse
    int* live;      // [blocks]
};

// p of a row (unscaled: times `inverse` of it), the softmax's numerators where they differ, and lse.
template <int V, int LANES, bool SIGMOID>
struct Shares {
    float p[V];
    float soft[SIGMOID ? V : 1];
    float inverse, soft_inverse, lse;
    bool live;
    __device__ __forceinline__ explicit Shares(const float (&v)[V]) {
        const float top = group_max<LANES>(largest(v));
        live = top != NOTHING;
        const float base = live ? top : 0.0f;
        float sum;
        if constexpr (SIGMOID) {
            const float low = fminf(base, 0.0f);
            float all = 0.0f;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                p[i] = sigmoid_over(v[i], low);
                all += p[i];
                soft[i] = v[i];
            }
            // (every lane of the warp takes part in both sums, live or not)
            sum = group_sum<LANES>(powers(soft, base));
            all = group_sum<LANES>(all);
            inverse = live ? inverse_approx(all) : 0.0f;
            soft_inverse = live ? inverse_approx(sum) : 0.0f;
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) p[i] = v[i];
            sum = group_sum<LANES>(powers(p, base));
            soft_inverse = inverse = live ? inverse_approx(sum) : 0.0f;
        }
        lse = live ? base + logf(sum) : 0.0f;
    }
};

template <typename T, int V, int LANES, bool SIGMOID>
__global__ void __launch_bounds__(LOGIT_THREADS) balance_kernel(BalanceArgs a, LogitShape s) {
    constexpr int WARPS = LOGIT_THREADS / 32, PER_BLOCK = LOGIT_THREADS / LANES;
    __shared__ int hist[MAX_EXPERTS];
    __shared__ float sums[WARPS][LANES * V];
    __shared__ float squares[WARPS];
    __shared__ int alive[WARPS];
    const int lane = threadIdx.x & (LANES - 1), warp = threadIdx.x >> 5;
    for (int e = threadIdx.x; e < s.experts; e += LOGIT_THREADS) hist[e] = 0;
    __syncthreads();

    // lanes of one expert find each other bit by bit, and the first adds for all
    const int bits = 32 - __clz(s.experts);
    const long long step = (long long)gridDim.x * LOGIT_THREADS;
    for (long long i0 = (long long)blockIdx.x * LOGIT_THREADS; i0 < a.pairs; i0 += step) {
        const long long i = i0 + threadIdx.x;
        long long e = s.experts;
        if (i < a.pairs) e = a.key_bytes == 8 ? static_cast<const long long*>(a.expert)[i] : static_cast<const int*>(a.expert)[i];
        const int key = e >= 0 && e < s.experts ? int(e) : s.experts;
        uint32_t peers = 0xffffffffu;
        for (int b = 0; b < bits; ++b) {
            const uint32_t on = __ballot_sync(0xffffffffu, key >> b & 1);
            peers &= key >> b & 1 ? on : ~on;
        }
        if (key < s.experts && (threadIdx.x & 31) == __ffs(peers) - 1) atomicAdd(hist + key, __popc(peers));
    }

    float sum[V], square = 0.0f;
    int live = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = 0.0f;
    for (long long row0 = (long long)blockIdx.x * PER_BLOCK; row0 < s.rows; row0 += (long long)gridDim.x * PER_BLOCK) {
        const long long row = row0 + threadIdx.x / LANES;
        float v[V];
        load_logits<T, V, LANES>(static_cast<const T*>(a.logits), s, a.mask, row, row < s.rows, lane, v);
        const Shares<V, LANES, SIGMOID> share(v);
#pragma unroll
        for (int i = 0; i < V; ++i) sum[i] = fmaf(share.p[i], share.inverse, sum[i]);
        if (lane == 0) {
            square += share.lse * share.lse;
            live += share.live;
        }
    }
#pragma unroll
    for (int d = LANES; d < 32; d *= 2) {
#pragma unroll
        for (int i = 0; i < V; ++i) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], d);
        square += __shfl_xor_sync(0xffffffffu, square, d);
        live += __shfl_xor_sync(0xffffffffu, live, d);
    }
    if ((threadIdx.x & 31) < LANES) {
#pragma unroll
        for (int i = 0; i < V; ++i) sums[warp][run_at<LANES>(i / 8, lane) + i % 8] = sum[i];
        if (lane == 0) {
            squares[warp] = square;
            alive[warp] = live;
        }
    }
    __syncthreads();
    const long long at = (long long)blockIdx.x * s.experts;
    for (int e = threadIdx.x; e < s.experts; e += LOGIT_THREADS) {
        float total = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) total += sums[w][e];
        a.sums[at + e] = total;
        a.counts[at + e] = hist[e];
    }
    if (threadIdx.x == 0) {
        float total = 0.0f;
        int rows = 0;
        for (int w = 0; w < WARPS; ++w) {
            total += squares[w];
            rows += alive[w];
        }
        a.squares[blockIdx.x] = total;
        a.live[blockIdx.x] = rows;
    }
}

struct BalanceJoin {
    const float* sums;
    const int* counts;
    const float* squares;
    const int* live;
    int blocks;
    int experts;
    const long long* total;  // null: the counts
    float* loss;
    float* z;
    int* out;                // counts
    float* stats;            // [experts] f, [experts] = 1 / T
};

constexpr int JOIN_THREADS = 1024, JOIN_BLOCKS = 8;

template <typename T>
__device__ __forceinline__ T block_sum(T v, T* at) {  // in a fixed order; at: [32]
#pragma unroll
    for (int d = 16; d > 0; d /= 2) v += __shfl_xor_sync(0xffffffffu, v, d);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) at[threadIdx.x >> 5] = v;
    __syncthreads();
    v = at[threadIdx.x & 31];
#pragma unroll
    for (int d = 16; d > 0; d /= 2) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}

// One cluster: each of its blocks sums a share of the partial sums, the first one joins them.
__global__ void __cluster_dims__(JOIN_BLOCKS, 1, 1) __launch_bounds__(JOIN_THREADS) balance_join_kernel(BalanceJoin a) {
    namespace cg = cooperative_groups;
    const cg::cluster_group cluster = cg::this_cluster();
    __shared__ double sums[JOIN_THREADS];
    __shared__ int counts[JOIN_THREADS];
    __shared__ double doubles[32];
    __shared__ long long longs[32];
    const int rank = int(cluster.block_rank());
    int columns = 1;
    while (columns < a.experts) columns *= 2;
    const int e = threadIdx.x & (columns - 1), line = threadIdx.x / columns, lines = JOIN_THREADS / columns;
    const int share = (a.blocks + JOIN_BLOCKS - 1) / JOIN_BLOCKS, from = min(a.blocks, rank * share), to = min(a.blocks, from + share);
    double sum = 0.0;
    int count = 0;
    if (e < a.experts) {
#pragma unroll 8
        for (int b = from + line; b < to; b += lines) {
            sum += double(__ldg(a.sums + (long long)b * a.experts + e));
            count += __ldg(a.counts + (long long)b * a.experts + e);
        }
    }
    sums[threadIdx.x] = sum;
    counts[threadIdx.x] = count;
    __syncthreads();
    if (int(threadIdx.x) < columns) {
        for (int l = 1; l < lines; ++l) {
            sum += sums[l * columns + e];
            count += counts[l * columns + e];
        }
        sums[e] = sum;
        counts[e] = count;
    }
    cluster.sync();
    if (rank == 0) {
        const bool mine = int(threadIdx.x) < a.experts;
        if (mine) {
            for (int r = 1; r < JOIN_BLOCKS; ++r) {
                sum += *cluster.map_shared_rank(sums + e, r);
                count += *cluster.map_shared_rank(counts + e, r);
            }
            a.out[e] = count;
        } else {
            sum = 0.0;
            count = 0;
        }
        const long long load = !mine ? 0 : a.total ? a.total[e] : count;
        double squares = 0.0;
        long long live = 0;
        for (int b = threadIdx.x; b < a.blocks; b += JOIN_THREADS) {
            squares += double(a.squares[b]);
            live += a.live[b];
        }
        const long long all = block_sum(load, longs);
        live = block_sum(live, longs);
        squares = block_sum(squares, doubles);
        const double f = all > 0 ? double(load) / double(all) : 0.0, per = live > 0 ? 1.0 / double(live) : 0.0;
        const double loss = block_sum(f * sum, doubles);
        if (mine) a.stats[e] = float(f);
        if (threadIdx.x == 0) {
            a.stats[a.experts] = float(per);
            *a.loss = float(loss * double(a.experts) * per);
            *a.z = float(squares * per);
        }
    }
    cluster.sync();  // the shared memory that the first block reads stays
}

struct BalanceBackward {
    const void* logits;
    Mask mask;
    const float* stats;
    const float* d_loss;  // null: 0
    const float* d_z;     // null: 0
    void* d_logits;
};

template <typename T, int V, int LANES, bool SIGMOID>
__global__ void __launch_bounds__(LOGIT_THREADS) balance_backward_kernel(BalanceBackward a, LogitShape s) {
    const int lane = threadIdx.x & (LANES - 1);
    const long long row = (long long)blockIdx.x * (LOGIT_THREADS / LANES) + threadIdx.x / LANES;
    const bool inside = row < s.rows;
    float v[V], f[V];
    load_logits<T, V, LANES>(static_cast<const T*>(a.logits), s, a.mask, row, inside, lane, v);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int e = run_at<LANES>(i / 8, lane) + i % 8;
        f[i] = e < s.experts ? __ldg(a.stats + e) : 0.0f;
    }
    const float per = __ldg(a.stats + s.experts);
    const float first = a.d_loss ? __ldg(a.d_loss) * float(s.experts) * per : 0.0f, second = a.d_z ? __ldg(a.d_z) * 2.0f * per : 0.0f;
    const Shares<V, LANES, SIGMOID> share(v);
    float mean = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) mean += f[i] * share.p[i];
    mean = group_sum<LANES>(mean) * share.inverse;
    const float scale = first * share.inverse, pull = second * share.lse * share.soft_inverse;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        float d = scale * share.p[i] * (f[i] - mean);
        if (SIGMOID) d = d * sigmoid_of(-v[i]) + pull * share.soft[i];
        else d += pull * share.p[i];
        v[i] = v[i] == NOTHING || !share.live ? 0.0f : d;
    }
    if (inside) store_logits<T, V, LANES>(static_cast<T*>(a.d_logits), s, row, lane, v);
}

constexpr int SMS = 148;  // of a B200: the sizes of scratch must not depend on the device that asks

// Four blocks to an SM, and no more than 256 rows to a thread: its fp32 sums stay within 2^-16 of themselves.
int64_t balance_blocks(int64_t rows, int experts) {
    const int64_t blocks = logit_blocks(rows, experts);
    return std::min(blocks, std::max<int64_t>(SMS * 4, (blocks + 255) / 256));
}

template <typename F>
void with_balance(int dtype, int experts, int score, F&& f) {
    with_logits(dtype, experts, [&](auto type, auto v, auto lanes) {
        if (score == SCORE_SIGMOID) f(type, v, lanes, std::true_type{});
        else f(type, v, lanes, std::false_type{});
    });
}

}  // namespace
}  // namespace odie

using namespace odie;

extern "C" int64_t odie_balance_scratch(int64_t rows, int experts) {
    if (rows < 0 || rows >= (int64_t(1) << 31) || experts < 1 || experts > MAX_EXPERTS) return 0;
    return balance_blocks(rows, experts) * (int64_t(experts) + 1) * 8;
}

extern "C" int odie_balance(const void* logits, int64_t rows, int experts, int dtype, const uint8_t* mask, int64_t mask_row_step,
                            int64_t mask_expert_step, int score, const void* expert, int key_bytes, int64_t pairs, const int64_t* total,
                            float* loss, float* z, int32_t* counts, float* stats, void* scratch, uint64_t stream_handle) {
    return guarded([&] {
        check_logits(rows, experts, dtype, score);
        ODIE_REQUIRE(key_bytes == 4 || key_bytes == 8, "experts must be int32 or int64 (key_bytes 4 or 8)");
        ODIE_REQUIRE(pairs >= 0 && pairs < (int64_t(1) << 31), "too many (row, choice) pairs");
        ODIE_REQUIRE((logits || rows == 0) && (expert || pairs == 0), "logits and expert are required");
        ODIE_REQUIRE(rows > 0 || pairs == 0, "choices without rows");
        ODIE_REQUIRE(loss && z && counts && stats, "loss, z, counts and stats are required");
        const cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_handle);
        const int64_t blocks = balance_blocks(rows, experts);
        ODIE_REQUIRE(blocks == 0 || (scratch && uintptr_t(scratch) % 256 == 0), "scratch is required, on a 256-byte boundary");
        BalanceArgs a{};
        a.logits = logits;
        a.mask = {mask, mask_row_step, mask_expert_step};
        a.score = score;
        a.expert = expert;
        a.key_bytes = key_bytes;
        a.pairs = pairs;
        a.sums = static_cast<float*>(scratch);
        a.counts = reinterpret_cast<int*>(a.sums + blocks * experts);
        a.squares = reinterpret_cast<float*>(a.counts + blocks * experts);
        a.live = reinterpret_cast<int*>(a.squares + blocks);
        if (blocks) {
            const LogitShape s = logit_shape(rows, experts, dtype, {logits}, a.mask);
            with_balance(dtype, experts, score, [&](auto type, auto v, auto lanes, auto sigmoid) {
                balance_kernel<decltype(type), decltype(v)::value, decltype(lanes)::value, decltype(sigmoid)::value><<<unsigned(blocks), LOGIT_THREADS, 0, stream>>>(a, s);
            });
            ODIE_CUDA(cudaGetLastError());
            note_launch();
        }
        const BalanceJoin j{a.sums, a.counts, a.squares, a.live, int(blocks), experts, reinterpret_cast<const long long*>(total), loss, z, counts, stats};
        balance_join_kernel<<<JOIN_BLOCKS, JOIN_THREADS, 0, stream>>>(j);
        ODIE_CUDA(cudaGetLastError());
        note_launch();
    });
}

extern "C" int odie_balance_backward(const float* d_loss, const float* d_z, const void* logits, int64_t rows, int experts, int dtype,
                                     const uint8_t* mask, int64_t mask_row_step, int64_t mask_expert_step, int score, const float* stats,
                                     void* d_logits, uint64_t stream) {
    return guarded([&] {
        check_logits(rows, experts, dtype, score);
        if (rows == 0) return;
        ODIE_REQUIRE(logits && stats && d_logits, "logits, stats and d_logits are required");
        const BalanceBackward a{logits, {mask, mask_row_step, mask_expert_step}, stats, d_loss, d_z, d_logits};
        const LogitShape s = logit_shape(rows, experts, dtype, {logits, d_logits}, a.mask);
        with_balance(dtype, experts, score, [&](auto type, auto v, auto lanes, auto sigmoid) {
            balance_backward_kernel<decltype(type), decltype(v)::value, decltype(lanes)::value, decltype(sigmoid)::value>
                <<<unsigned(logit_blocks(rows, experts)), LOGIT_THREADS, 0, reinterpret_cast<cudaStream_t>(stream)>>>(a, s);
        });
        ODIE_CUDA(cudaGetLastError());
        note_launch();
    });
}
