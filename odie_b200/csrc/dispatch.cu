// Rows to their experts' places and back (odie_dispatch, odie_combine and the gradient of both).
//
// With slot[t * k + j] the place of row t's j-th choice among the rows sorted by expert:
//   dispatch   sorted[slot] = w x[t]             (w = 1 without weights), zero rows for dropped choices
//   combine    out[t] = sum_j w[t, j] sorted[slot[t, j]], an fp32 chain in ascending j, rounded once
//   backward   d sorted[slot] = w d out[t], d w[t, j] = <sorted[slot], d out[t]> in fp32
// The gradient of dispatch is combine without weights.  All are bound by the bytes of the rows.  Kernels walk the
// side that they write, so that writes are whole lines in order and only reads are scattered (writes of 64-byte rows
// to their places took half as long again), but for wide rows with several
// choices, whose places are whole lines anyway.
#include "rows.cuh"
#include "odie_b200.h"
#include <type_traits>

namespace odie {
namespace {

struct RowArgs {
    RowShape shape;     // of the side that the kernel walks
    long long places;   // rows of the sorted side, and (row, choice) pairs
    int choices;
    long long width;    // elements of a row
    const int* order;   // [places] pair at each place; negative: dropped, ~order is the pair
    const int* slot;    // [rows][choices] place of each pair; negative: dropped, ~slot is its place
    const float* weights;
};

// Rows that a thread takes of narrow ones, or vectors of a wide one.  (2^20 rows of 32 fp16: 51 us with one row, 35 with
// two, 41 with four, whose registers leave half the blocks; 4-byte vectors, rows of 20 fp16: 84 with two, 72 with four; all
// with L2 cold, one call at a time, ten in a row 44, 29, 33 and 75, 62.)
template <int BYTES, bool NARROW>
constexpr int DISPATCH_ITEMS = NARROW && BYTES == 16 ? 2 : 4;

// Walks the sorted rows: they are written in order, and row order[p] / choices is fetched for each.
template <typename T, int BYTES, bool NARROW>
__global__ void __launch_bounds__(ROW_THREADS) dispatch_kernel(RowArgs a, const T* __restrict__ rows, T* __restrict__ sorted) {
    using P = Pack<T, BYTES>;
    constexpr int ITEMS = DISPATCH_ITEMS<BYTES, NARROW>;
    const RowWalk<NARROW, ITEMS> walk(a.shape);
    long long row[ITEMS];
    float w[ITEMS];
    bool kept[ITEMS];
#pragma unroll
    for (int q = 0; q < ITEMS; ++q) {
        const int i = walk.row_of(q) < walk.rows ? __ldg(a.order + walk.row_of(q)) : -1;
        kept[q] = i >= 0 && i < a.places;
        row[q] = kept[q] ? i / a.choices : 0;
        w[q] = kept[q] && a.weights ? __ldg(a.weights + i) : 1.0f;
    }
    for (long long c = walk.lane; c < walk.vectors; c += walk.stride()) {
        P v[ITEMS];
#pragma unroll
        for (int q = 0; q < ITEMS; ++q)
            v[q] = P::load(rows + row[q] * a.width + (walk.vector_of(c, q) < walk.vectors ? walk.vector_of(c, q) : 0) * P::N);
#pragma unroll
        for (int q = 0; q < ITEMS; ++q) {
            P o = kept[q] ? v[q] : P::zero();
            if (a.weights && kept[q]) {
#pragma unroll
                for (int i = 0; i < P::N; ++i) o.v[i] = from_float<T>(w[q] * to_float(v[q].v[i]));
            }
            if (walk.on(c, q)) o.store(sorted + walk.row_of(q) * a.width + walk.vector_of(c, q) * P::N);
        }
    }
}

// Vectors of a wide row that a thread takes together where they are 16 bytes (1) or fewer (4: as many bytes in flight).
template <int BYTES, bool NARROW = false>
constexpr int SCALE = NARROW || BYTES == 16 ? 1 : 4;

// Wide rows with several choices: walks the unsorted rows, so that each is read once however many choices it has.
// (Walking the sorted side, rows were evicted from L2 between their choices: 16384 rows of 4 KB, four choices each,
// took 82 us against 54.)
template <typename T, int BYTES>
__global__ void __launch_bounds__(ROW_THREADS) dispatch_rows_kernel(RowArgs a, const T* __restrict__ rows, T* __restrict__ sorted) {
    using P = Pack<T, BYTES>;
    constexpr int ITEMS = SCALE<BYTES>;
    const RowWalk<false, ITEMS> walk(a.shape);
    if (walk.row >= walk.rows) return;
    const long long pair = walk.row * a.choices;
    for (long long c = walk.lane; c < walk.vectors; c += walk.stride()) {
        P v[ITEMS];
#pragma unroll
        for (int q = 0; q < ITEMS; ++q) v[q] = P::load(rows + walk.row * a.width + (walk.on(c, q) ? walk.vector_of(c, q) : 0) * P::N);
#pragma unroll 4
        for (int j = 0; j < a.choices; ++j) {
            const int s = __ldg(a.slot + pair + j);
            const long long place = s < 0 ? ~s : s;
            const float w = s >= 0 && a.weights ? __ldg(a.weights + pair + j) : 1.0f;
#pragma unroll
            for (int q = 0; q < ITEMS; ++q) {
                P o = s < 0 ? P::zero() : v[q];
                if (s >= 0 && a.weights) {
#pragma unroll
                    for (int i = 0; i < P::N; ++i) o.v[i] = from_float<T>(w * to_float(v[q].v[i]));
                }
                if (place < a.places && walk.on(c, q)) o.store(sorted + place * a.width + walk.vector_of(c, q) * P::N);
            }
        }
    }
}

// BATCH choices of ITEMS vectors are loaded together (dropped ones as the first row, and left out of the sum): one
// choice takes four vectors, two take two, and more take four choices of one.
template <typename T, int BYTES, bool NARROW, int BATCH>
__global__ void __launch_bounds__(ROW_THREADS) combine_kernel(RowArgs a, const T* __restrict__ sorted, T* __restrict__ out) {
    using P = Pack<T, BYTES>;
    constexpr int ITEMS = 4 / BATCH * SCALE<BYTES, NARROW>, ROWS = NARROW ? ITEMS : 1;
    const RowWalk<NARROW, ITEMS> walk(a.shape);
    for (long long c = walk.lane; c < walk.vectors; c += walk.stride()) {
        float sum[ITEMS][P::N];
#pragma unroll
        for (int q = 0; q < ITEMS; ++q)
#pragma unroll
            for (int i = 0; i < P::N; ++i) sum[q][i] = 0.0f;
        for (int j0 = 0; j0 < a.choices; j0 += BATCH) {
            P v[ITEMS][BATCH];
            float w[ROWS][BATCH];
            bool on[ROWS][BATCH];
            long long place[ROWS][BATCH];
#pragma unroll
            for (int q = 0; q < ROWS; ++q)
#pragma unroll
                for (int b = 0; b < BATCH; ++b) {
                    const bool inside = walk.row_of(q) < walk.rows && j0 + b < a.choices;
                    const long long pair = inside ? walk.row_of(q) * a.choices + j0 + b : 0;
                    const int s = __ldg(a.slot + pair);
                    w[q][b] = a.weights ? __ldg(a.weights + pair) : 1.0f;
                    on[q][b] = inside && s >= 0 && s < a.places;
                    place[q][b] = on[q][b] ? s : 0;
                }
#pragma unroll
            for (int q = 0; q < ITEMS; ++q)
#pragma unroll
                for (int b = 0; b < BATCH; ++b) {
                    const long long at = walk.vector_of(c, q);
                    v[q][b] = P::load(sorted + place[NARROW ? q : 0][b] * a.width + (at < walk.vectors ? at : 0) * P::N);
                }
#pragma unroll
            for (int q = 0; q < ITEMS; ++q)
#pragma unroll
                for (int b = 0; b < BATCH; ++b)
#pragma unroll
                    for (int i = 0; i < P::N; ++i) {
                        const float next = fmaf(w[NARROW ? q : 0][b], to_float(v[q][b].v[i]), sum[q][i]);
                        sum[q][i] = on[NARROW ? q : 0][b] ? next : sum[q][i];
                    }
        }
#pragma unroll
        for (int q = 0; q < ITEMS; ++q) {
            P o;
#pragma unroll
            for (int i = 0; i < P::N; ++i) o.v[i] = from_float<T>(sum[q][i]);
            if (walk.on(c, q)) o.store(out + walk.row_of(q) * a.width + walk.vector_of(c, q) * P::N);
        }
    }
}

// Blocks per SM of the gradient kernels, more of them at the price of spilled registers.  Us at none asked for (as the
// compiler's registers leave), four, five and six, 2^20 rows of 32 and of 64:
//   fp16  59, 59, 55, 53;  98, 98, 92, 84       fp32  98, 100, 92, 86;  184, 186, 170, 158
//   bf16  72, 64, 66, 70;  127, 109, 111, 115   (its product takes more registers; at six it spills 56 bytes)
// Wide rows, several choices, at none, two, three and four: 16384 rows of 2048, four choices, fp16 107, 121, 104, 100; bf16
// 123, 123, 111, 115; fp32 188, 221, 193, 189; two choices of 4096, 139, 176, 139, 123; 180, 180, 150, 148; 229, 315, 258,
// 231; 4-byte vectors, four choices of 1026 fp16 102, 100, 82, 104; bf16 168, 168, 143, 145; of 1025 fp32 148, 180, 145, 184.
template <typename T, int BYTES, bool NARROW>
constexpr int GRADIENT_BLOCKS = NARROW && BYTES == 16 ? (std::is_same<T, __nv_bfloat16>::value ? 4 : 6) : 0;
template <typename T, int BYTES>
constexpr int GRADIENT_ROWS_BLOCKS = BYTES == 16 && !std::is_same<T, __nv_bfloat16>::value ? 4 : 3;

// Walks the sorted rows.  The dot product's partial sums are joined in a fixed tree.
template <typename T, int BYTES, bool NARROW>
__global__ void __launch_bounds__(ROW_THREADS, (GRADIENT_BLOCKS<T, BYTES, NARROW>)) combine_backward_kernel(RowArgs a, const T* __restrict__ d_out,
                                                                       const T* __restrict__ sorted, T* __restrict__ d_sorted,
                                                                       float* __restrict__ d_weights) {
    using P = Pack<T, BYTES>;
    constexpr int ITEMS = 2;
    __shared__ float partial[ROW_THREADS / 32];
    const RowWalk<NARROW, ITEMS> walk(a.shape);
    long long place[ITEMS], row[ITEMS], pair[ITEMS];
    float w[ITEMS], dot[ITEMS];
    bool kept[ITEMS];
#pragma unroll
    for (int q = 0; q < ITEMS; ++q) {
        place[q] = walk.row_of(q) < walk.rows ? walk.row_of(q) : 0;
        const int i = __ldg(a.order + place[q]);
        pair[q] = i < 0 ? ~i : i;
        kept[q] = i >= 0 && i < a.places;
        row[q] = kept[q] ? i / a.choices : 0;
        w[q] = kept[q] && a.weights ? __ldg(a.weights + i) : 1.0f;
        dot[q] = 0.0f;
    }
    for (long long c = walk.lane; c < walk.vectors; c += walk.stride()) {
        P g[ITEMS], y[ITEMS];
#pragma unroll
        for (int q = 0; q < ITEMS; ++q) {
            const long long at = (walk.vector_of(c, q) < walk.vectors ? walk.vector_of(c, q) : 0) * P::N;
            g[q] = P::load(d_out + row[q] * a.width + at);
            if (d_weights) y[q] = P::load(sorted + place[q] * a.width + at);
        }
#pragma unroll
        for (int q = 0; q < ITEMS; ++q) {
            const bool on = walk.on(c, q);
            if (d_weights) {
                float part = 0.0f;
#pragma unroll
                for (int i = 0; i < P::N; ++i) part = fmaf(to_float(y[q].v[i]), to_float(g[q].v[i]), part);
                const int to = NARROW ? q : 0;
                dot[to] = kept[q] && on ? dot[to] + part : dot[to];
            }
            if (d_sorted && on) {
                P o = P::zero();
                if (kept[q]) {
#pragma unroll
                    for (int i = 0; i < P::N; ++i) o.v[i] = from_float<T>(w[q] * to_float(g[q].v[i]));
                }
                o.store(d_sorted + place[q] * a.width + walk.vector_of(c, q) * P::N);
            }
        }
    }
    if (!d_weights) return;
#pragma unroll
    for (int q = 0; q < (NARROW ? ITEMS : 1); ++q) {
#pragma unroll
        for (int d = 16; d > 0; d /= 2) {
            const float other = __shfl_xor_sync(0xffffffffu, dot[q], d);
            if (d < walk.lanes) dot[q] += other;
        }
        if (!NARROW && walk.lanes > 32) {
            if ((threadIdx.x & 31) == 0) partial[threadIdx.x >> 5] = dot[q];
            __syncthreads();
            if (walk.lane == 0) {
                dot[q] = 0.0f;
                for (int i = 0; i < walk.lanes / 32; ++i) dot[q] += partial[(threadIdx.x >> 5) + i];
            }
        }
        if (walk.lane == 0 && walk.row_of(q) < walk.rows && pair[q] < a.places) d_weights[pair[q]] = kept[q] ? dot[q] : 0.0f;
    }
}

// The same for wide rows with several choices, walking the unsorted rows: d out is read once for up to four choices.
template <typename T, int BYTES>
__global__ void __launch_bounds__(ROW_THREADS, (GRADIENT_ROWS_BLOCKS<T, BYTES>)) combine_backward_rows_kernel(RowArgs a, const T* __restrict__ d_out,
                                                                            const T* __restrict__ sorted, T* __restrict__ d_sorted,
                                                                            float* __restrict__ d_weights) {
    using P = Pack<T, BYTES>;
    constexpr int BATCH = 4, ITEMS = SCALE<BYTES>;
    __shared__ float partial[BATCH][ROW_THREADS / 32];
    const RowWalk<false, ITEMS> walk(a.shape);
    const bool live = walk.row < walk.rows;
    const long long row = live ? walk.row : 0;
    for (int j0 = 0; j0 < a.choices; j0 += BATCH) {
        long long place[BATCH];
        float w[BATCH], dot[BATCH];
        bool kept[BATCH], on[BATCH];
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
            const bool inside = live && j0 + b < a.choices;
            const long long pair = row * a.choices + (inside ? j0 + b : 0);
            const int s = __ldg(a.slot + pair);
            place[b] = s < 0 ? ~s : s;
            on[b] = inside && place[b] < a.places;
            kept[b] = on[b] && s >= 0;
            if (!on[b]) place[b] = 0;
            w[b] = a.weights ? __ldg(a.weights + pair) : 1.0f;
            dot[b] = 0.0f;
        }
        for (long long c = walk.lane; c < walk.vectors; c += walk.stride()) {
            P g[ITEMS], y[ITEMS][BATCH];
#pragma unroll
            for (int q = 0; q < ITEMS; ++q) {
                const long long at = (walk.vector_of(c, q) < walk.vectors ? walk.vector_of(c, q) : 0) * P::N;
                g[q] = P::load(d_out + row * a.width + at);
#pragma unroll
                for (int b = 0; b < BATCH; ++b)
                    if (d_weights) y[q][b] = P::load(sorted + place[b] * a.width + at);
            }
#pragma unroll
            for (int q = 0; q < ITEMS; ++q) {
                if (walk.vector_of(c, q) >= walk.vectors) continue;
#pragma unroll
                for (int b = 0; b < BATCH; ++b) {
                    if (d_weights) {
                        float part = 0.0f;
#pragma unroll
                        for (int i = 0; i < P::N; ++i) part = fmaf(to_float(y[q][b].v[i]), to_float(g[q].v[i]), part);
                        dot[b] = kept[b] ? dot[b] + part : 0.0f;
                    }
                    if (d_sorted && on[b]) {
                        P o = P::zero();
                        if (kept[b]) {
#pragma unroll
                            for (int i = 0; i < P::N; ++i) o.v[i] = from_float<T>(w[b] * to_float(g[q].v[i]));
                        }
                        o.store(d_sorted + place[b] * a.width + walk.vector_of(c, q) * P::N);
                    }
                }
            }
        }
        if (!d_weights) continue;
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
#pragma unroll
            for (int d = 16; d > 0; d /= 2) dot[b] += __shfl_xor_sync(0xffffffffu, dot[b], d);
            if ((threadIdx.x & 31) == 0) partial[b][threadIdx.x >> 5] = dot[b];
        }
        __syncthreads();
        if (walk.lane < BATCH && live && j0 + walk.lane < a.choices) {
            float total = 0.0f;
            for (int i = 0; i < walk.lanes / 32; ++i) total += partial[walk.lane][(threadIdx.x >> 5) + i];
            d_weights[row * a.choices + j0 + walk.lane] = total;
        }
        __syncthreads();
    }
}

void check_rows(int64_t n, int choices, int64_t width, int dtype, const int32_t* order, const char* name) {
    check_row_type(dtype);
    ODIE_REQUIRE(n >= 0 && choices >= 1 && n < (int64_t(1) << 31) / choices, "0 to 2^31 - 1 (row, choice) pairs");
    ODIE_REQUIRE(width >= 1 && width <= (int64_t(1) << 31), "rows have 1 to 2^31 elements");
    ODIE_REQUIRE(n == 0 || order, std::string(name) + " is required");
}

// Which rows are narrow: up to 32 vectors always; more where there are many rows and few choices, whose rows one thread
// then reads side by side.  Measured at 2^26 halves in all, dispatch / combine / its gradient in us, narrow against wide:
//   16 bytes  one choice, 64 vectors 49 / 55 / 74 against 78 / 100 / 90, 256: 51 / 57 / 76 against 53 / 64 / 78, 512:
//             53 / 68 / 92 against 53 / 61 / 78; two, 64: 45 / 47 / 70 against 45 / 47 / 86; four, 64: 39 / 41 / 68
//             against 35 / 41 / 61
//   4 bytes   one choice, 150: 84 / 100 / 121 against 137 / 274 / 143, 501: 80 / 100 / 109 against 78 / 104 / 107; two,
//             115: 82 / 92 / 125 against 84 / 94 / 143, 150: 78 / 92 / 117 against 100 / 78 / 150; four, 50: 104 / 80 /
//             168 against 121 / 119 / 152, 115: 74 / 70 / 121 against 59 / 74 / 90
bool narrow_rows(int64_t n, int64_t vectors, int bytes, int choices) {
    int most = 32;
    if (n * choices >= MANY_ROWS) {
        if (bytes == 16) most = choices <= 2 ? 256 : 32;
        else most = choices == 1 ? 256 : choices == 2 ? 128 : 64;
    }
    return vectors <= most;
}

// The walk of a kernel that writes the sorted side: by rows (slot) for wide rows with several choices, by places
// (order) for the others.
RowArgs sorted_args(int64_t n, int choices, int64_t width, int dtype, int vector, const int32_t* order, const int32_t* slot,
                    const float* weights) {
    const int64_t vectors = width * row_type_size(dtype) / vector;
    const bool narrow = narrow_rows(n, vectors, vector, choices);
    RowArgs a{row_shape(n * choices, vectors, vector, narrow), n * choices, choices, width, order, nullptr, weights};
    if (!a.shape.narrow && choices > 1) {
        a.shape = row_shape(n, vectors, vector, narrow);
        a.order = nullptr;
        a.slot = slot;
    }
    return a;
}

// f(T{}, integral_constant<int, BYTES>, bool_constant<NARROW>)
template <typename F>
void with_rows(int dtype, int vector, bool narrow, F&& f) {
    with_row_type(dtype, vector, [&](auto type, auto bytes) {
        if (narrow) f(type, bytes, std::true_type{});
        else f(type, bytes, std::false_type{});
    });
}

}  // namespace
}  // namespace odie

using namespace odie;

extern "C" int odie_dispatch(const void* rows, int64_t n, int choices, int64_t width, int dtype, const int32_t* order,
                             const int32_t* slot, const float* weights, void* sorted, uint64_t stream) {
    return guarded([&] {
        check_rows(n, choices, width, dtype, order, "order");
        ODIE_REQUIRE(n == 0 || slot, "slot is required");
        if (n == 0) return;
        ODIE_REQUIRE(rows && sorted, "rows and sorted are required");
        const int vector = row_vector(width, dtype, rows, sorted);
        const RowArgs a = sorted_args(n, choices, width, dtype, vector, order, slot, weights);
        if (a.slot) {
            with_row_type(dtype, vector, [&](auto type, auto bytes) {
                using T = decltype(type);
                dispatch_rows_kernel<T, decltype(bytes)::value>
                    <<<row_blocks(a.shape, 1), ROW_THREADS, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
                        a, static_cast<const T*>(rows), static_cast<T*>(sorted));
            });
        } else with_rows(dtype, vector, a.shape.narrow, [&](auto type, auto bytes, auto narrow) {
            using T = decltype(type);
            dispatch_kernel<T, decltype(bytes)::value, decltype(narrow)::value>
                <<<row_blocks(a.shape, (DISPATCH_ITEMS<decltype(bytes)::value, decltype(narrow)::value>)), ROW_THREADS, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
                    a, static_cast<const T*>(rows), static_cast<T*>(sorted));
        });
        ODIE_CUDA(cudaGetLastError());
        note_launch();
    });
}

extern "C" int odie_combine(const void* sorted, int64_t n, int choices, int64_t width, int dtype, const int32_t* slot,
                            const float* weights, void* out, uint64_t stream) {
    return guarded([&] {
        check_rows(n, choices, width, dtype, slot, "slot");
        if (n == 0) return;
        ODIE_REQUIRE(sorted && out, "sorted and out are required");
        const int vector = row_vector(width, dtype, sorted, out);
        const int64_t vectors = width * row_type_size(dtype) / vector;
        const RowArgs a{row_shape(n, vectors, vector, narrow_rows(n, vectors, vector, choices)), n * choices, choices, width, nullptr, slot, weights};
        with_rows(dtype, vector, a.shape.narrow, [&](auto type, auto bytes, auto narrow) {
            using T = decltype(type);
            auto go = [&](auto batch) {
                combine_kernel<T, decltype(bytes)::value, decltype(narrow)::value, decltype(batch)::value>
                    <<<row_blocks(a.shape, 4 / decltype(batch)::value * SCALE<decltype(bytes)::value, decltype(narrow)::value>), ROW_THREADS, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
                        a, static_cast<const T*>(sorted), static_cast<T*>(out));
            };
            if (choices == 1) go(std::integral_constant<int, 1>{});
            else if (choices == 2) go(std::integral_constant<int, 2>{});
            else go(std::integral_constant<int, 4>{});
        });
        ODIE_CUDA(cudaGetLastError());
        note_launch();
    });
}

extern "C" int odie_combine_backward(const void* d_out, const void* sorted, int64_t n, int choices, int64_t width, int dtype,
                                     const int32_t* order, const int32_t* slot, const float* weights, void* d_sorted,
                                     float* d_weights, uint64_t stream) {
    return guarded([&] {
        check_rows(n, choices, width, dtype, order, "order");
        ODIE_REQUIRE(n == 0 || slot, "slot is required");
        if (n == 0 || (!d_sorted && !d_weights)) return;
        ODIE_REQUIRE(d_out && (sorted || !d_weights), "d_out is required, and sorted for the weights' gradient");
        const int vector = row_vector(width, dtype, d_out, d_weights ? sorted : d_out, d_sorted);
        const RowArgs a = sorted_args(n, choices, width, dtype, vector, order, slot, weights);
        if (a.slot) {
            with_row_type(dtype, vector, [&](auto type, auto bytes) {
                using T = decltype(type);
                combine_backward_rows_kernel<T, decltype(bytes)::value>
                    <<<row_blocks(a.shape, 1), ROW_THREADS, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
                        a, static_cast<const T*>(d_out), static_cast<const T*>(sorted), static_cast<T*>(d_sorted), d_weights);
            });
        } else with_rows(dtype, vector, a.shape.narrow, [&](auto type, auto bytes, auto narrow) {
            using T = decltype(type);
            combine_backward_kernel<T, decltype(bytes)::value, decltype(narrow)::value>
                <<<row_blocks(a.shape, 2), ROW_THREADS, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
                    a, static_cast<const T*>(d_out), static_cast<const T*>(sorted), static_cast<T*>(d_sorted), d_weights);
        });
        ODIE_CUDA(cudaGetLastError());
        note_launch();
    });
}
