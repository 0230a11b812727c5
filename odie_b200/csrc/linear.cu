// y = residual + act(x W^T + b) for one weight matrix, or for one per group of consecutive rows, and its gradient.
//
//   forward    z = x W_g^T + b_g, y = residual + act(z); fp32 sums, one rounding
//   backward   dz = d y act'(z); d x = dz W_g, d W_g = dz^T x over the group's rows, d b_g = sum dz
//
// Rows of no group (behind the last offset) give zero rows of y and d x and add to no gradient.  Training keeps
// act'(z) as a 16-bit fixed-point code (15 fraction bits above -1/4): act' lies in (-0.13, 1.13) for every
// activation here, so the code is within 2^-16 of it, closer than a 16-bit float of it or of z would be.
#include "rows.cuh"
#include "odie_b200.h"
#include <type_traits>

namespace odie {
namespace {

enum Activation : int { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3 };

// 0xffff is kept for NaN.
__device__ __forceinline__ uint16_t slope_code(float d) {
    return d == d ? uint16_t(min(65534.0f, max(0.0f, rintf(fmaf(d, 32768.0f, 8192.0f))))) : uint16_t(0xffff);
}
__device__ __forceinline__ float slope_value(uint16_t c) {
    return c == 0xffff ? __int_as_float(0x7fffffff) : fmaf(float(c), 1.0f / 32768.0f, -0.25f);
}

template <int ACT>
__device__ __forceinline__ float activate(float z, float& slope) {
    if (ACT == ACT_RELU) {
        slope = z > 0.0f ? 1.0f : z != z ? z : 0.0f;
        return z > 0.0f || z != z ? z : 0.0f;
    }
    if (ACT == ACT_SILU) {
        const float p = 1.0f / (1.0f + __expf(-z));
        slope = p * (1.0f + z * (1.0f - p));
        return z * p;
    }
    if (ACT == ACT_GELU) {
        const float p = 0.5f * (1.0f + erff(z * 0.70710678118654752f));
        slope = p + z * __expf(-0.5f * z * z) * 0.39894228040143268f;
        return z * p;
    }
    slope = 1.0f;
    return z;
}

// Rows [begin, end) of group g: offsets clamped to [0, rows], so no offset reads or writes out of range.
__device__ __forceinline__ void group_rows(const int* offsets, int g, long long rows, long long& begin, long long& end) {
    if (!offsets) {
        begin = 0;
        end = rows;
        return;
    }
    begin = g == 0 ? 0 : min(rows, max(0ll, (long long)offsets[g]));
    end = max(begin, min(rows, max(0ll, (long long)offsets[g + 1])));
}

// C[m][n] = sum_k A(m, k) B(n, k) with element strides.
struct Product {
    const void* a;
    const void* b;
    long long a_m, a_k, b_n, b_k, b_group, c_group;
    long long rows;     // of all groups
    int m, n, k;        // of dW: m = outputs, n = inputs; of y, dX: m unused
    int groups;
    const int* offsets;
    bool reduce_rows;   // k runs over the group's rows (dW)
};

template <typename T, typename Out>
__global__ void __launch_bounds__(256) product_kernel(Product p, Out out) {
    __shared__ float as[16][65], bs[16][65];
    const T* a = static_cast<const T*>(p.a);
    const T* b = static_cast<const T*>(p.b);
    const int g = blockIdx.z, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    long long begin, end;
    if (g < p.groups) group_rows(p.offsets, g, p.rows, begin, end);
    else {  // the rows of no group
        long long from;
        group_rows(p.offsets, p.groups - 1, p.rows, from, begin);
        end = p.rows;
    }
    const bool nothing = g >= p.groups;
    const long long m_count = p.reduce_rows ? p.m : end - begin, k_count = nothing ? 0 : p.reduce_rows ? end - begin : p.k;
    const long long m_base = p.reduce_rows ? 0 : begin, k_base = p.reduce_rows ? begin : 0;
    const int n0 = blockIdx.x * 64;
    if (!nothing) b += p.reduce_rows ? 0 : g * p.b_group;
    for (long long m0 = (long long)blockIdx.y * 64; m0 < m_count; m0 += (long long)gridDim.y * 64) {
        float acc[4][4] = {};
        for (long long k0 = 0; k0 < k_count; k0 += 16) {
            for (int i = threadIdx.x; i < 1024; i += 256) {
                const int kk = i & 15, r = i >> 4;
                as[kk][r] = m0 + r < m_count && k0 + kk < k_count
                                ? to_float(a[(m_base + m0 + r) * p.a_m + (k_base + k0 + kk) * p.a_k]) : 0.0f;
                bs[kk][r] = n0 + r < p.n && k0 + kk < k_count
                                ? to_float(b[(long long)(n0 + r) * p.b_n + (k_base + k0 + kk) * p.b_k]) : 0.0f;
            }
            __syncthreads();
#pragma unroll
            for (int kk = 0; kk < 16; ++kk)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(as[kk][ty * 4 + i], bs[kk][tx * 4 + j], acc[i][j]);
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (m0 + ty * 4 + i < m_count && n0 + tx * 4 + j < p.n)
                    out(g, m_base + m0 + ty * 4 + i, n0 + tx * 4 + j, acc[i][j], nothing);
    }
}

template <typename T, int ACT>
struct ForwardOut {
    const T* bias;
    const T* residual;
    T* y;
    uint16_t* slope;
    long long n;
    __device__ void operator()(int g, long long m, int c, float acc, bool nothing) const {
        float s = 0.0f, v = 0.0f;
        if (!nothing) {
            v = activate<ACT>(acc + (bias ? to_float(bias[g * n + c]) : 0.0f), s);
            if (residual) v += to_float(residual[m * n + c]);
        }
        y[m * n + c] = from_float<T>(v);
        if (slope) slope[m * n + c] = slope_code(s);
    }
};
template <typename T>
struct PlainOut {
    T* c;
    long long ld, group;
    __device__ void operator()(int g, long long m, int n, float acc, bool) const { c[g * group + m * ld + n] = from_float<T>(acc); }
};

template <typename T>
__global__ void __launch_bounds__(256) dz_kernel(const T* d_y, const uint16_t* slope, T* dz, T* d_residual, long long rows, int n,
                                                 const int* offsets, int groups) {
    long long from, live;
    group_rows(offsets, groups - 1, rows, from, live);
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < rows * n; i += (long long)gridDim.x * 256) {
        dz[i] = from_float<T>(to_float(d_y[i]) * (slope ? slope_value(slope[i]) : 1.0f));
        if (d_residual) d_residual[i] = i < live * n ? d_y[i] : from_float<T>(0.0f);
    }
}

template <typename T>
__global__ void __launch_bounds__(256) bias_kernel(const T* d_y, const uint16_t* slope, T* d_bias, long long rows, int n,
                                                   const int* offsets) {
    const int g = blockIdx.y, c = blockIdx.x * 32 + (threadIdx.x & 31);
    __shared__ float part[8][32];
    long long begin, end;
    group_rows(offsets, g, rows, begin, end);
    float sum = 0.0f;
    if (c < n)
        for (long long r = begin + (threadIdx.x >> 5); r < end; r += 8)
            sum += to_float(d_y[r * n + c]) * (slope ? slope_value(slope[r * n + c]) : 1.0f);
    part[threadIdx.x >> 5][threadIdx.x & 31] = sum;
    __syncthreads();
    if (threadIdx.x < 32 && c < n) {
        sum = 0.0f;
        for (int i = 0; i < 8; ++i) sum += part[i][threadIdx.x];
        d_bias[(long long)g * n + c] = from_float<T>(sum);
    }
}

void check_linear(int64_t rows, int inputs, int outputs, int groups, const int32_t* offsets, int dtype, int activation) {
    ODIE_REQUIRE(dtype == ROW_F16 || dtype == ROW_BF16, "linear takes fp16 (0) or bf16 (1)");
    ODIE_REQUIRE(rows >= 0 && rows < (int64_t(1) << 31), "0 to 2^31 - 1 rows");
    ODIE_REQUIRE(inputs >= 1 && outputs >= 1 && inputs <= (1 << 20) && outputs <= (1 << 20), "1 to 2^20 inputs and outputs");
    ODIE_REQUIRE(groups >= 1 && groups <= 1024, "1 to 1024 groups");
    ODIE_REQUIRE(offsets || groups == 1, "more than one group needs offsets");
    ODIE_REQUIRE(activation >= ACT_NONE && activation <= ACT_GELU, "activation must be 0 (none), 1 (ReLU), 2 (SiLU) or 3 (GELU)");
}

template <typename F>
void with_linear_type(int dtype, F&& f) {
    if (dtype == ROW_BF16) f(__nv_bfloat16{});
    else f(__half{});
}

dim3 product_grid(int64_t m, int64_t n, int groups) {
    return dim3(unsigned((n + 63) / 64), unsigned(std::min<int64_t>(65535, (m + 63) / 64)), unsigned(groups));
}

}  // namespace
}  // namespace odie

using namespace odie;

extern "C" int64_t odie_linear_scratch(int64_t rows, int inputs, int outputs, int groups) { return 0; }

extern "C" int odie_linear(const void* x, const void* weight, const void* bias, const void* residual, int64_t rows, int inputs,
                           int outputs, int groups, const int32_t* offsets, int dtype, int activation, void* y,
                           uint16_t* slope, void* scratch, uint64_t stream_handle) {
    return guarded([&] {
        check_linear(rows, inputs, outputs, groups, offsets, dtype, activation);
        if (rows == 0) return;
        ODIE_REQUIRE(x && weight && y, "x, weight and y are required");
        const cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_handle);
        Product p{x, weight, inputs, 1, inputs, 1, int64_t(outputs) * inputs, 0, rows, 0, outputs, inputs, groups, offsets, false};
        with_linear_type(dtype, [&](auto type) {
            using T = decltype(type);
            auto go = [&](auto act) {
                ForwardOut<T, decltype(act)::value> out{static_cast<const T*>(bias), static_cast<const T*>(residual),
                                                       static_cast<T*>(y), slope, outputs};
                product_kernel<T><<<product_grid(rows, outputs, groups + (offsets ? 1 : 0)), 256, 0, stream>>>(p, out);
            };
            if (activation == ACT_RELU) go(std::integral_constant<int, ACT_RELU>{});
            else if (activation == ACT_SILU) go(std::integral_constant<int, ACT_SILU>{});
            else if (activation == ACT_GELU) go(std::integral_constant<int, ACT_GELU>{});
            else go(std::integral_constant<int, ACT_NONE>{});
        });
        ODIE_CUDA(cudaGetLastError());
        note_launch();
    });
}

extern "C" int64_t odie_linear_backward_scratch(int64_t rows, int inputs, int outputs, int groups) {
    return rows * outputs * 2;
}

extern "C" int odie_linear_backward(const void* d_y, const uint16_t* slope, const void* x, const void* weight, int64_t rows,
                                    int inputs, int outputs, int groups, const int32_t* offsets, int dtype, void* d_x,
                                    void* d_weight, void* d_bias, void* d_residual, void* scratch, uint64_t stream_handle) {
    return guarded([&] {
        check_linear(rows, inputs, outputs, groups, offsets, dtype, ACT_NONE);
        const cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_handle);
        const int64_t weights = int64_t(groups) * outputs * inputs;
        if (rows == 0) {
            if (d_weight) ODIE_CUDA(cudaMemsetAsync(d_weight, 0, size_t(weights) * 2, stream));
            if (d_bias) ODIE_CUDA(cudaMemsetAsync(d_bias, 0, size_t(groups) * outputs * 2, stream));
            return;
        }
        ODIE_REQUIRE(d_y && (x || !d_weight) && (weight || !d_x) && scratch, "d_y, x, weight and scratch are required");
        with_linear_type(dtype, [&](auto type) {
            using T = decltype(type);
            T* dz = static_cast<T*>(scratch);
            dz_kernel<T><<<1184, 256, 0, stream>>>(static_cast<const T*>(d_y), slope, dz, static_cast<T*>(d_residual), rows, outputs,
                                                   offsets, groups);
            if (d_bias)
                bias_kernel<T><<<dim3((outputs + 31) / 32, groups), 256, 0, stream>>>(static_cast<const T*>(d_y), slope,
                                                                                     static_cast<T*>(d_bias), rows, outputs, offsets);
            if (d_x) {
                Product p{dz, weight, outputs, 1, 1, inputs, int64_t(outputs) * inputs, 0, rows, 0, inputs, outputs, groups, offsets, false};
                product_kernel<T><<<product_grid(rows, inputs, groups + (offsets ? 1 : 0)), 256, 0, stream>>>(
                    p, PlainOut<T>{static_cast<T*>(d_x), inputs, 0});
            }
            if (d_weight) {
                Product p{dz, x, 1, outputs, 1, inputs, 0, int64_t(outputs) * inputs, rows, outputs, inputs, 0, groups, offsets, true};
                product_kernel<T><<<product_grid(outputs, inputs, groups), 256, 0, stream>>>(
                    p, PlainOut<T>{static_cast<T*>(d_weight), inputs, int64_t(outputs) * inputs});
            }
        });
        ODIE_CUDA(cudaGetLastError());
        note_launch(1 + (d_bias ? 1 : 0) + (d_x ? 1 : 0) + (d_weight ? 1 : 0));
    });
}
