// Rows of any width and type, loaded and stored a vector at a time (dispatch.cu, embed.cu, linear.cu).
#pragma once
#include <cuda_bf16.h>
#include "common.cuh"

namespace odie {

// The element types of the row operators, as the C-ABI numbers them.
enum RowType : int { ROW_F16 = 0, ROW_BF16 = 1, ROW_F32 = 2 };
__host__ inline int row_type_size(int dtype) { return dtype == ROW_F32 ? 4 : 2; }

__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(float v) { return v; }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }

template <int BYTES>
struct Raw;
template <>
struct Raw<16> { using type = uint4; };
template <>
struct Raw<4> { using type = uint32_t; };
template <>
struct Raw<2> { using type = uint16_t; };

// BYTES / sizeof(T) consecutive elements, moved by one load or store.
template <typename T, int BYTES>
struct alignas(BYTES) Pack {
    static constexpr int N = BYTES / int(sizeof(T));
    T v[N];
    __device__ __forceinline__ static Pack load(const T* p) {
        Pack r;
        *reinterpret_cast<typename Raw<BYTES>::type*>(&r) = __ldg(reinterpret_cast<const typename Raw<BYTES>::type*>(p));
        return r;
    }
    // Read once: not kept in L1, whose lines are for what is read again.
    __device__ __forceinline__ static Pack load_once(const T* p) {
        Pack r;
        if constexpr (BYTES == 16) {
            uint4& v = *reinterpret_cast<uint4*>(&r);
            asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
            return r;
        } else {
            return load(p);
        }
    }
    __device__ __forceinline__ static Pack zero() {
        Pack r;
        *reinterpret_cast<typename Raw<BYTES>::type*>(&r) = typename Raw<BYTES>::type{};
        return r;
    }
    __device__ __forceinline__ void store(T* p) const {
        *reinterpret_cast<typename Raw<BYTES>::type*>(p) = *reinterpret_cast<const typename Raw<BYTES>::type*>(this);
    }
};

// The widest vector that every row of these buffers starts on: 16 bytes, 4 bytes or one element.
inline int row_vector(int64_t width, int dtype, const void* a, const void* b = nullptr, const void* c = nullptr) {
    const int size = row_type_size(dtype);
    const uintptr_t bits = uintptr_t(a) | uintptr_t(b) | uintptr_t(c) | uintptr_t(width * size);
    return bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : size;
}

// Calls f(T{}, std::integral_constant<int, BYTES>) for the type and vector width at run time.
template <typename F>
void with_row_type(int dtype, int vector, F&& f) {
    if (dtype == ROW_F32) {
        if (vector == 16) f(float{}, std::integral_constant<int, 16>{});
        else f(float{}, std::integral_constant<int, 4>{});
    } else if (dtype == ROW_BF16) {
        if (vector == 16) f(__nv_bfloat16{}, std::integral_constant<int, 16>{});
        else if (vector == 4) f(__nv_bfloat16{}, std::integral_constant<int, 4>{});
        else f(__nv_bfloat16{}, std::integral_constant<int, 2>{});
    } else {
        if (vector == 16) f(__half{}, std::integral_constant<int, 16>{});
        else if (vector == 4) f(__half{}, std::integral_constant<int, 4>{});
        else f(__half{}, std::integral_constant<int, 2>{});
    }
}

// How the 256 threads of a block share rows of `vectors` vectors, so that each has several independent loads in
// flight and neighbours read neighbouring vectors.  Narrow rows (as the caller says): 2^lanes_log2 threads, 32 at most,
// take one vector each of a row at a time, and each of them ITEMS rows.  Wide rows: 32 to 256 threads walk a row
// together, ITEMS vectors at a time.  item<ITEMS>(q, ..) is the thread's q-th (row, vector) of a step.
constexpr int ROW_THREADS = 256;
// Rows from which a warp or less for several of them fills the SMs.
constexpr int64_t MANY_ROWS = 1 << 14;
struct RowShape {
    long long rows;
    long long vectors;
    int lanes_log2;
    bool narrow;
};
inline RowShape row_shape(int64_t rows, int64_t vectors, int bytes, bool narrow) {
    const int most = bytes == 16 ? 4 : 16;  // vectors per thread of a wide row: 64 bytes
    RowShape s{rows, vectors, 0, narrow};
    if (s.narrow) {
        while (s.lanes_log2 < 5 && (1 << s.lanes_log2) < vectors) ++s.lanes_log2;
    } else {
        s.lanes_log2 = 5;
        while (s.lanes_log2 < 8 && (int64_t(most) << s.lanes_log2) < vectors) ++s.lanes_log2;
    }
    return s;
}
inline unsigned row_blocks(const RowShape& s, int items) {
    const int64_t per = (ROW_THREADS >> s.lanes_log2) * int64_t(s.narrow ? items : 1);
    const int64_t blocks = (s.rows + per - 1) / per;
    ODIE_REQUIRE(blocks < (int64_t(1) << 31), "too many rows for one launch");
    return unsigned(blocks);
}
template <bool NARROW, int ITEMS>
struct RowWalk {
    long long row, vectors, rows;
    int lane, lanes, step;
    __device__ __forceinline__ explicit RowWalk(const RowShape& s) : vectors(s.vectors), rows(s.rows) {
        lanes = 1 << s.lanes_log2;
        lane = threadIdx.x & (lanes - 1);
        step = ROW_THREADS >> s.lanes_log2;
        row = (long long)blockIdx.x * (step * (NARROW ? ITEMS : 1)) + (threadIdx.x >> s.lanes_log2);
    }
    __device__ __forceinline__ long long row_of(int q) const { return NARROW ? row + q * step : row; }
    __device__ __forceinline__ long long vector_of(long long c, int q) const { return NARROW ? c : c + q * lanes; }
    __device__ __forceinline__ bool on(long long c, int q) const { return row_of(q) < rows && vector_of(c, q) < vectors; }
    __device__ __forceinline__ int stride() const { return NARROW ? lanes : lanes * ITEMS; }
};

// Sorted (key, index) pairs: sort_pairs (sort.cu).  keys: int32 or int64 (key_bytes 4 or 8), anything outside
// [0, bins) counts as `bins`.  Writes order[p] = index of the p-th pair by (key, index), and where non-null
// sorted[p] = its key and slot[i] = its place; for keys outside the range order is ~index and
// slot ~place.
// offsets (may be null): i32[bins + 1], the number of pairs with a smaller key.
struct SortArgs {
    const void* keys = nullptr;
    int key_bytes = 4;
    int64_t n = 0;
    int bins = 0;
    int* order = nullptr;
    uint32_t* sorted = nullptr;
    int* slot = nullptr;
    int* offsets = nullptr;
    void* scratch = nullptr;
};
int64_t sort_scratch_bytes(int64_t n, int bins);
void launch_sort(const SortArgs& a, cudaStream_t stream);

inline void check_row_type(int dtype) { ODIE_REQUIRE(dtype >= 0 && dtype <= 2, "element type must be 0 (fp16), 1 (bf16) or 2 (fp32)"); }

}  // namespace odie
