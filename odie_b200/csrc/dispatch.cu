// Rows to their experts' places and back (odie_dispatch, odie_combine and the gradient of both).
//
// With slot[t * k + j] the place of row t's j-th choice among the rows sorted by expert:
//   dispatch   sorted[slot] = w x[t]             (w = 1 without weights), zero rows for dropped choices
//   combine    out[t] = sum_j w[t, j] sorted[slot[t, j]], an fp32 chain in ascending j, rounded once
//   backward   d sorted[slot] = w d out[t], d w[t, j] = <sorted[slot], d out[t]> in fp32
// The gradient of dispatch is combine without weights.  All are bound by the bytes of the rows: every kernel
// walks the unsorted side in order, so that a row is read once however many choices it has, and moves whole
// rows of the sorted side in 16-byte vectors.
#include "rows.cuh"
#include "odie_b200.h"
#include <type_traits>

namespace odie {
namespace {

constexpr int THREADS = 256;

struct RowArgs {
    long long n;        // unsorted rows
    int choices;
    long long width;    // elements of a row
    int lanes_log2;     // threads per row
    const int* slot;    // [n][choices]; negative: dropped, ~slot is its place
    const float* weights;
};

template <typename T, int BYTES>
__global__ void __launch_bounds__(THREADS) dispatch_kernel(RowArgs a, const T* __restrict__ rows, T* __restrict__ sorted) {
    using P = Pack<T, BYTES>;
    const int lanes = 1 << a.lanes_log2, lane = threadIdx.x & (lanes - 1);
    const long long t = ((long long)blockIdx.x * THREADS + threadIdx.x) >> a.lanes_log2;
    if (t >= a.n) return;
    const long long vectors = a.width / P::N, places = a.n * a.choices;
    const T* from = rows + t * a.width;
    for (long long c = lane; c < vectors; c += lanes) {
        const P v = P::load(from + c * P::N);
        for (int j = 0; j < a.choices; ++j) {
            const int s = __ldg(a.slot + t * a.choices + j);
            const long long place = s < 0 ? ~s : s;
            if (place >= places) continue;
            P o = v;
            if (s < 0) {
                o = P::zero();
            } else if (a.weights) {
                const float w = __ldg(a.weights + t * a.choices + j);
#pragma unroll
                for (int i = 0; i < P::N; ++i) o.v[i] = from_float<T>(w * to_float(v.v[i]));
            }
            o.store(sorted + place * a.width + c * P::N);
        }
    }
}

template <typename T, int BYTES>
__global__ void __launch_bounds__(THREADS) combine_kernel(RowArgs a, const T* __restrict__ sorted, T* __restrict__ out) {
    using P = Pack<T, BYTES>;
    constexpr int BATCH = 4;  // choices whose rows are loaded together
    const int lanes = 1 << a.lanes_log2, lane = threadIdx.x & (lanes - 1);
    const long long t = ((long long)blockIdx.x * THREADS + threadIdx.x) >> a.lanes_log2;
    if (t >= a.n) return;
    const long long vectors = a.width / P::N, places = a.n * a.choices;
    for (long long c = lane; c < vectors; c += lanes) {
        float sum[P::N] = {};
        for (int j0 = 0; j0 < a.choices; j0 += BATCH) {
            P v[BATCH];
            float w[BATCH];
            bool on[BATCH];
#pragma unroll
            for (int b = 0; b < BATCH; ++b) {
                const int j = j0 + b;
                const int s = j < a.choices ? __ldg(a.slot + t * a.choices + j) : -1;
                on[b] = s >= 0 && s < places;
                if (on[b]) {
                    v[b] = P::load(sorted + s * a.width + c * P::N);
                    w[b] = a.weights ? __ldg(a.weights + t * a.choices + j) : 1.0f;
                }
            }
#pragma unroll
            for (int b = 0; b < BATCH; ++b)
                if (on[b]) {
#pragma unroll
                    for (int i = 0; i < P::N; ++i) sum[i] = fmaf(w[b], to_float(v[b].v[i]), sum[i]);
                }
        }
        P o;
#pragma unroll
        for (int i = 0; i < P::N; ++i) o.v[i] = from_float<T>(sum[i]);
        o.store(out + t * a.width + c * P::N);
    }
}

// A row's threads per (row, choice).  The dot product's partial sums are joined in a fixed tree.
template <typename T, int BYTES>
__global__ void __launch_bounds__(THREADS) combine_backward_kernel(RowArgs a, const T* __restrict__ d_out,
                                                                   const T* __restrict__ sorted, T* __restrict__ d_sorted,
                                                                   float* __restrict__ d_weights) {
    using P = Pack<T, BYTES>;
    __shared__ float partial[THREADS / 32];
    const int lanes = 1 << a.lanes_log2, lane = threadIdx.x & (lanes - 1);
    const long long pair = ((long long)blockIdx.x * THREADS + threadIdx.x) >> a.lanes_log2;
    const long long places = a.n * a.choices, vectors = a.width / P::N;
    const bool live = pair < places;
    const int s = live ? __ldg(a.slot + pair) : 0;
    const long long place = s < 0 ? ~s : s;
    const bool inside = live && place < places;
    float dot = 0.0f;
    if (inside) {
        const long long t = pair / a.choices;
        const float w = a.weights ? __ldg(a.weights + pair) : 1.0f;
        for (long long c = lane; c < vectors; c += lanes) {
            P o = P::zero();
            if (s >= 0) {
                const P g = P::load(d_out + t * a.width + c * P::N);
#pragma unroll
                for (int i = 0; i < P::N; ++i) o.v[i] = from_float<T>(w * to_float(g.v[i]));
                if (d_weights) {
                    const P y = P::load(sorted + place * a.width + c * P::N);
                    float part = 0.0f;
#pragma unroll
                    for (int i = 0; i < P::N; ++i) part = fmaf(to_float(y.v[i]), to_float(g.v[i]), part);
                    dot += part;
                }
            }
            if (d_sorted) o.store(d_sorted + place * a.width + c * P::N);
        }
    }
    if (!d_weights) return;
#pragma unroll
    for (int d = 16; d > 0; d /= 2)
        if (d < lanes) dot += __shfl_xor_sync(0xffffffffu, dot, d);
    if (lanes > 32) {
        if ((threadIdx.x & 31) == 0) partial[threadIdx.x >> 5] = dot;
        __syncthreads();
        if (lane == 0) {
            dot = 0.0f;
            for (int w = 0; w < lanes / 32; ++w) dot += partial[(threadIdx.x >> 5) + w];
        }
    }
    if (live && lane == 0) d_weights[pair] = inside && s >= 0 ? dot : 0.0f;
}

RowArgs row_args(int64_t n, int choices, int64_t width, int dtype, const int32_t* slot, const float* weights, int vector) {
    RowArgs a{n, choices, width, 0, slot, weights};
    const int lanes = row_lanes(width * row_type_size(dtype) / vector);
    while ((1 << a.lanes_log2) < lanes) ++a.lanes_log2;
    return a;
}

void check_rows(int64_t n, int choices, int64_t width, int dtype, const int32_t* slot) {
    check_row_type(dtype);
    ODIE_REQUIRE(n >= 0 && choices >= 1 && n < (int64_t(1) << 31) / choices, "0 to 2^31 - 1 (row, choice) pairs");
    ODIE_REQUIRE(width >= 1 && width <= (int64_t(1) << 31), "rows have 1 to 2^31 elements");
    ODIE_REQUIRE(n == 0 || slot, "slot is required");
}

unsigned row_blocks(int64_t rows, const RowArgs& a) {
    const int64_t blocks = ((rows << a.lanes_log2) + THREADS - 1) / THREADS;
    ODIE_REQUIRE(blocks < (int64_t(1) << 31), "too many rows for one launch");
    return unsigned(blocks);
}

}  // namespace
}  // namespace odie

using namespace odie;

extern "C" int odie_dispatch(const void* rows, int64_t n, int choices, int64_t width, int dtype, const int32_t* slot,
                             const float* weights, void* sorted, uint64_t stream) {
    return guarded([&] {
        check_rows(n, choices, width, dtype, slot);
        if (n == 0) return;
        ODIE_REQUIRE(rows && sorted, "rows and sorted are required");
        const int vector = row_vector(width, dtype, rows, sorted);
        const RowArgs a = row_args(n, choices, width, dtype, slot, weights, vector);
        with_row_type(dtype, vector, [&](auto type, auto bytes) {
            using T = decltype(type);
            dispatch_kernel<T, decltype(bytes)::value><<<row_blocks(n, a), THREADS, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
                a, static_cast<const T*>(rows), static_cast<T*>(sorted));
        });
        ODIE_CUDA(cudaGetLastError());
        note_launch();
    });
}

extern "C" int odie_combine(const void* sorted, int64_t n, int choices, int64_t width, int dtype, const int32_t* slot,
                            const float* weights, void* out, uint64_t stream) {
    return guarded([&] {
        check_rows(n, choices, width, dtype, slot);
        if (n == 0) return;
        ODIE_REQUIRE(sorted && out, "sorted and out are required");
        const int vector = row_vector(width, dtype, sorted, out);
        const RowArgs a = row_args(n, choices, width, dtype, slot, weights, vector);
        with_row_type(dtype, vector, [&](auto type, auto bytes) {
            using T = decltype(type);
            combine_kernel<T, decltype(bytes)::value><<<row_blocks(n, a), THREADS, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
                a, static_cast<const T*>(sorted), static_cast<T*>(out));
        });
        ODIE_CUDA(cudaGetLastError());
        note_launch();
    });
}

extern "C" int odie_combine_backward(const void* d_out, const void* sorted, int64_t n, int choices, int64_t width, int dtype,
                                     const int32_t* slot, const float* weights, void* d_sorted, float* d_weights,
                                     uint64_t stream) {
    return guarded([&] {
        check_rows(n, choices, width, dtype, slot);
        if (n == 0 || (!d_sorted && !d_weights)) return;
        ODIE_REQUIRE(d_out && (sorted || !d_weights), "d_out is required, and sorted for the weights' gradient");
        const int vector = row_vector(width, dtype, d_out, d_weights ? sorted : d_out, d_sorted);
        const RowArgs a = row_args(n, choices, width, dtype, slot, weights, vector);
        with_row_type(dtype, vector, [&](auto type, auto bytes) {
            using T = decltype(type);
            combine_backward_kernel<T, decltype(bytes)::value>
                <<<row_blocks(n * choices, a), THREADS, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
                    a, static_cast<const T*>(d_out), static_cast<const T*>(sorted), static_cast<T*>(d_sorted), d_weights);
        });
        ODIE_CUDA(cudaGetLastError());
        note_launch();
    });
}
