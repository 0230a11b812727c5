// Lookup of table rows by integer id, times a scale, and the table's gradient by sorted ids.
//
//   out[i] = scale table[id_i];   d table[v] = scale sum over {i : id_i = v}, in ascending i, of d out[i]
//
// An id outside the table gives a zero row and takes no gradient.  The gradient sorts the ids (sort.cu), so that
// the rows of one id are consecutive, and sums each run in fp32 without atomics: the same bits in every run.  A
// run may be one row or the whole batch, so the sorted positions are cut into chunks of CHUNK; a chunk sums the
// runs that lie inside it and writes them as finished, and leaves at most two partial sums of runs that cross its
// ends, which a second pass over the table rows joins in chunk order (and writes the zero rows of absent ids).
// Bound by the bytes of d out and d table.
#include "rows.cuh"
#include "odie_b200.h"
#include <algorithm>
#include <type_traits>

namespace odie {
namespace {

constexpr int THREADS = ROW_THREADS;
constexpr int CHUNK = 64, BATCH = 4;  // BATCH rows are loaded together, the next ones' positions with them

struct EmbedArgs {
    RowShape shape;   // of the result
    const void* ids;
    int id_bytes;
    long long rows;   // of the table
    long long width;
    float scale;
};

template <typename T, int BYTES, bool NARROW>
__global__ void __launch_bounds__(THREADS) embed_kernel(EmbedArgs a, const T* __restrict__ table, T* __restrict__ out) {
    using P = Pack<T, BYTES>;
    constexpr int ITEMS = 4;
    const RowWalk<NARROW, ITEMS> walk(a.shape);
    long long id[ITEMS];
    bool inside[ITEMS];
#pragma unroll
    for (int q = 0; q < ITEMS; ++q) {
        const long long i = walk.row_of(q) < walk.rows ? walk.row_of(q) : 0;
        id[q] = a.id_bytes == 8 ? __ldg(static_cast<const long long*>(a.ids) + i) : (long long)__ldg(static_cast<const int*>(a.ids) + i);
        inside[q] = id[q] >= 0 && id[q] < a.rows;
        if (!inside[q]) id[q] = 0;
    }
    for (long long c = walk.lane; c < walk.vectors; c += walk.stride()) {
        P v[ITEMS];
#pragma unroll
        for (int q = 0; q < ITEMS; ++q)
            v[q] = P::load(table + id[q] * a.width + (walk.vector_of(c, q) < walk.vectors ? walk.vector_of(c, q) : 0) * P::N);
#pragma unroll
        for (int q = 0; q < ITEMS; ++q) {
            P o = P::zero();
            if (inside[q]) {
#pragma unroll
                for (int e = 0; e < P::N; ++e) o.v[e] = from_float<T>(a.scale * to_float(v[q].v[e]));
            }
            if (walk.on(c, q)) o.store(out + walk.row_of(q) * a.width + walk.vector_of(c, q) * P::N);
        }
    }
}

struct GradArgs {
    long long n, rows, width;
    int lanes_log2;
    long long column0;       // first vector of the launch: a grid has at most 65535 blocks of columns
    float scale;
    const uint32_t* sorted;  // [n] ids in order; the table's row count for ids outside it
    const int* order;        // [n] position in d out
    float* partial;          // [chunks][2][width]: sums of the runs that cross the chunk's begin, and its end
    int2* runs;              // [rows] first and past-the-last sorted position; zero for absent ids
};

// One unit: CHUNK sorted positions x one vector per thread of `lanes` columns.
template <typename T, int BYTES>
__global__ void __launch_bounds__(THREADS, 4) embed_chunk_kernel(GradArgs a, const T* __restrict__ d_out, T* __restrict__ d_table) {
    using P = Pack<T, BYTES>;
    const int lanes = 1 << a.lanes_log2, lane = threadIdx.x & (lanes - 1);
    const long long chunk = ((long long)blockIdx.x * THREADS + threadIdx.x) >> a.lanes_log2;
    const long long c = a.column0 + (long long)blockIdx.y * lanes + lane;
    const long long begin = chunk * CHUNK;
    if (begin >= a.n || c * P::N >= a.width) return;
    const int count = int(min((long long)CHUNK, a.n - begin));
    const uint32_t outside = uint32_t(a.rows);
    uint32_t current = a.sorted[begin];
    if (current >= outside) return;  // ids outside the table sort behind all others
    const uint32_t before = begin > 0 ? a.sorted[begin - 1] : 0xffffffffu;
    const uint32_t after = begin + count < a.n ? a.sorted[begin + count] : 0xffffffffu;
    bool open = before == current;  // the run began in an earlier chunk
    const bool marks = c == 0;
    if (marks && !open) a.runs[current].x = int(begin);
    float sum[P::N] = {};
    bool done = false;
    auto flush = [&](bool crosses_end) {
        if (open || crosses_end) {
            float* to = a.partial + (chunk * 2 + (open ? 0 : 1)) * a.width + c * P::N;
#pragma unroll
            for (int e = 0; e < P::N; ++e) to[e] = sum[e];
        } else {
            P o;
#pragma unroll
            for (int e = 0; e < P::N; ++e) o.v[e] = from_float<T>(a.scale * sum[e]);
            o.store(d_table + (long long)current * a.width + c * P::N);
        }
    };
    uint32_t key[BATCH];
    int at[BATCH];
    auto positions = [&](int b) {
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const long long p = min(begin + b + i, a.n - 1);
            key[i] = b + i < count ? __ldg(a.sorted + p) : outside;
            at[i] = __ldg(a.order + p);
        }
    };
    positions(0);
    for (int b = 0; b < count && !done; b += BATCH) {
        uint32_t now[BATCH];
        P v[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            now[i] = key[i];
            v[i] = P::load(d_out + (long long)(now[i] < outside ? at[i] : 0) * a.width + c * P::N);
        }
        positions(b + BATCH);
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            if (b + i >= count || done) continue;
            if (now[i] != current) {
                flush(false);
                if (marks) a.runs[current].y = int(begin + b + i);
                open = false;
                current = now[i];
                if (current >= outside) {
                    done = true;
                    continue;
                }
                if (marks) a.runs[current].x = int(begin + b + i);
#pragma unroll
                for (int e = 0; e < P::N; ++e) sum[e] = 0.0f;
            }
#pragma unroll
            for (int e = 0; e < P::N; ++e) sum[e] += to_float(v[i].v[e]);
        }
    }
    if (done) return;
    const bool crosses = after == current;
    flush(crosses);
    if (marks && !crosses) a.runs[current].y = int(begin + count);
}

// A block: `span` table rows, whose runs are read together, x one vector per thread.  (With a row per thread the wait
// for its run alone took 33 us for 65536 rows of 2 KB, most of them zero.)
constexpr int MAX_SPAN = 128;
template <typename T, int BYTES>
__global__ void __launch_bounds__(THREADS) embed_join_kernel(GradArgs a, T* __restrict__ d_table, int span) {
    using P = Pack<T, BYTES>;
    __shared__ int2 runs[MAX_SPAN];
    const long long v0 = (long long)blockIdx.x * span;
    const int count = int(min((long long)span, a.rows - v0));
    if (threadIdx.x < count) runs[threadIdx.x] = a.runs[v0 + threadIdx.x];
    __syncthreads();
    const int lanes = 1 << a.lanes_log2, lane = threadIdx.x & (lanes - 1), step = THREADS >> a.lanes_log2;
    const long long c = a.column0 + (long long)blockIdx.y * lanes + lane;
    if (c * P::N >= a.width) return;
    for (int q = threadIdx.x >> a.lanes_log2; q < count; q += step) {
        const int2 run = runs[q];
        P o = P::zero();
        if (run.y > run.x) {
            const long long first = run.x / CHUNK, last = (run.y - 1) / CHUNK;
            if (first == last) continue;  // written by its chunk
            float sum[P::N];
            const float* from = a.partial + (first * 2 + 1) * a.width + c * P::N;
#pragma unroll
            for (int e = 0; e < P::N; ++e) sum[e] = from[e];
#pragma unroll 4
            for (long long k = first + 1; k <= last; ++k) {
                const float* more = a.partial + k * 2 * a.width + c * P::N;
#pragma unroll
                for (int e = 0; e < P::N; ++e) sum[e] += more[e];
            }
#pragma unroll
            for (int e = 0; e < P::N; ++e) o.v[e] = from_float<T>(a.scale * sum[e]);
        }
        o.store(d_table + (v0 + q) * a.width + c * P::N);
    }
}

int log2_of(int lanes) {
    int l = 0;
    while ((1 << l) < lanes) ++l;
    return l;
}

void check_embed(int id_bytes, int64_t n, int64_t rows, int64_t width, int dtype) {
    check_row_type(dtype);
    ODIE_REQUIRE(id_bytes == 4 || id_bytes == 8, "ids are int32 or int64");
    ODIE_REQUIRE(n >= 0 && n < (int64_t(1) << 31) - 4096, "0 to 2^31 - 4097 ids");
    ODIE_REQUIRE(rows >= 1 && rows < (int64_t(1) << 30), "the table has 1 to 2^30 - 1 rows");
    ODIE_REQUIRE(width >= 1 && width <= (int64_t(1) << 31), "rows have 1 to 2^31 elements");
}

int64_t aligned(int64_t bytes) { return (bytes + 255) / 256 * 256; }

}  // namespace
}  // namespace odie

using namespace odie;

extern "C" int odie_embed(const void* ids, int id_bytes, int64_t n, const void* table, int64_t rows, int64_t width, int dtype,
                          float scale, void* out, uint64_t stream) {
    return guarded([&] {
        check_embed(id_bytes, n, rows, width, dtype);
        if (n == 0) return;
        ODIE_REQUIRE(ids && table && out, "ids, table and out are required");
        const int vector = row_vector(width, dtype, table, out);
        // (65536 rows of 64 vectors of 16 bytes: 25 us as narrow rows, 33 as wide ones; of 128: 45 and 43)
        const int64_t vectors = width * row_type_size(dtype) / vector;
        const EmbedArgs a{row_shape(n, vectors, vector, vectors <= (n < MANY_ROWS ? 32 : vector == 16 ? 64 : 128)), ids, id_bytes, rows, width, scale};
        with_row_type(dtype, vector, [&](auto type, auto bytes) {
            using T = decltype(type);
            constexpr int B = decltype(bytes)::value;
            const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
            const unsigned blocks = row_blocks(a.shape, 4);
            if (a.shape.narrow) embed_kernel<T, B, true><<<blocks, THREADS, 0, s>>>(a, static_cast<const T*>(table), static_cast<T*>(out));
            else embed_kernel<T, B, false><<<blocks, THREADS, 0, s>>>(a, static_cast<const T*>(table), static_cast<T*>(out));
        });
        ODIE_CUDA(cudaGetLastError());
        note_launch();
    });
}

extern "C" int64_t odie_embed_backward_scratch(int64_t n, int64_t rows, int64_t width) {
    if (n < 0 || rows < 1 || rows >= (int64_t(1) << 30) || width < 1) return 0;
    const int64_t chunks = (n + CHUNK - 1) / CHUNK;
    return aligned(sort_scratch_bytes(n, int(rows))) + 2 * aligned(4 * n) + aligned(8 * rows) + aligned(chunks * 2 * width * 4);
}

extern "C" int odie_embed_backward(const void* ids, int id_bytes, int64_t n, const void* d_out, int64_t rows, int64_t width,
                                   int dtype, float scale, void* d_table, void* scratch, uint64_t stream_handle) {
    return guarded([&] {
        check_embed(id_bytes, n, rows, width, dtype);
        ODIE_REQUIRE(d_table, "d_table is required");
        const cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_handle);
        if (n == 0) {
            ODIE_CUDA(cudaMemsetAsync(d_table, 0, size_t(rows * width) * row_type_size(dtype), stream));
            return;
        }
        ODIE_REQUIRE(ids && d_out && scratch, "ids, d_out and scratch are required");
        char* at = static_cast<char*>(scratch);
        auto take = [&](int64_t bytes) {
            char* p = at;
            at += aligned(bytes);
            return p;
        };
        const int64_t chunks = (n + CHUNK - 1) / CHUNK;
        SortArgs s;
        s.keys = ids;
        s.key_bytes = id_bytes;
        s.n = n;
        s.bins = int(rows);
        s.scratch = take(sort_scratch_bytes(n, int(rows)));
        s.order = reinterpret_cast<int*>(take(4 * n));
        s.sorted = reinterpret_cast<uint32_t*>(take(4 * n));
        GradArgs g{};
        g.n = n;
        g.rows = rows;
        g.width = width;
        g.scale = scale;
        g.sorted = s.sorted;
        g.order = s.order;
        g.runs = reinterpret_cast<int2*>(take(8 * rows));
        g.partial = reinterpret_cast<float*>(take(chunks * 2 * width * 4));
        ODIE_CUDA(cudaMemsetAsync(g.runs, 0, size_t(rows) * 8, stream));
        launch_sort(s, stream);
        const int vector = row_vector(width, dtype, d_out, d_table);
        const int64_t vectors = width * row_type_size(dtype) / vector;
        int lanes = 1;
        while (lanes < THREADS && lanes < vectors) lanes *= 2;
        g.lanes_log2 = log2_of(lanes);
        const int64_t columns = (vectors + lanes - 1) / lanes;
        const int64_t chunk_blocks = ((chunks << g.lanes_log2) + THREADS - 1) / THREADS;
        const int64_t step = THREADS >> g.lanes_log2;
        const int64_t span = std::max<int64_t>(1, std::min<int64_t>({MAX_SPAN, 16 * step, rows / (148 * 8)})), join_blocks = (rows + span - 1) / span;
        ODIE_REQUIRE(chunk_blocks < (int64_t(1) << 31) && join_blocks < (int64_t(1) << 31), "too many rows for one launch");
        with_row_type(dtype, vector, [&](auto type, auto bytes) {
            using T = decltype(type);
            constexpr int B = decltype(bytes)::value;
            for (int64_t first = 0; first < columns; first += 65535) {
                const unsigned count = unsigned(std::min<int64_t>(65535, columns - first));
                g.column0 = first * lanes;
                embed_chunk_kernel<T, B><<<dim3(unsigned(chunk_blocks), count), THREADS, 0, stream>>>(
                    g, static_cast<const T*>(d_out), static_cast<T*>(d_table));
                embed_join_kernel<T, B><<<dim3(unsigned(join_blocks), count), THREADS, 0, stream>>>(g, static_cast<T*>(d_table), int(span));
                ODIE_CUDA(cudaGetLastError());
                note_launch(2);
            }
        });
    });
}
