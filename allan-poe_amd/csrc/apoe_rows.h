// Rows of a matrix held in registers by groups of threads, shared by the operators that work on one row after the other (residual.hip, norm.hip,
// embed.hip): a group of G threads holds a row of up to 16 G values, 16 a thread.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

namespace apoe {

constexpr int ROW_E = 16; // values of a row that a thread holds

// Values (c G + t) V .. of a row, c = 0, 1, ..: 16 bytes a load with V > 1. WHOLE: rows begin at multiples of 16 bytes and have a multiple of V values;
// otherwise they begin at any value, and a row's last few are read and written one by one.
template <typename T, int V, int G, bool WHOLE = true> struct RowOf {
    typedef T tv __attribute__((ext_vector_type(V)));
    typedef tv tu __attribute__((aligned(WHOLE ? sizeof(tv) : sizeof(T))));
    static constexpr int C = ROW_E / V;
    // as it comes, and as numbers
    __device__ static void fetch(tv* raw, const void* p, uint64_t row, uint64_t stride, uint32_t dim, int t) {
        const T* at = (const T*)p + row * stride;
#pragma unroll
        for (int c = 0; c < C; c++) {
            const uint32_t d = (c * G + t) * V;
            raw[c] = tv{};
            if constexpr (V == 1) {
                if (d < dim) raw[c][0] = at[d];
            } else if constexpr (WHOLE) {
                if (d < dim) raw[c] = *reinterpret_cast<const tv*>(at + d);
            } else {
                if (d + V <= dim) {
                    raw[c] = *reinterpret_cast<const tu*>(at + d);
                } else if (d < dim) {
#pragma unroll
                    for (int k = 0; k < V - 1; k++)
                        if (d + k < dim) raw[c][k] = at[d + k];
                }
            }
        }
    }
    __device__ static void widen(float* v, const tv* raw) {
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int k = 0; k < V; k++) v[c * V + k] = (float)raw[c][k];
    }
    __device__ static void load(float* v, const void* p, uint64_t row, uint64_t stride, uint32_t dim, int t) {
        tv raw[C];
        fetch(raw, p, row, stride, dim, t);
        widen(v, raw);
    }
    __device__ static void store(void* p, uint64_t row, uint64_t stride, uint32_t dim, int t, const float* v) {
        T* at = (T*)p + row * stride;
#pragma unroll
        for (int c = 0; c < C; c++) {
            const uint32_t d = (c * G + t) * V;
            if (d >= dim) continue;
            if constexpr (V == 1) {
                at[d] = (T)v[c];
            } else {
                tv x;
#pragma unroll
                for (int k = 0; k < V; k++) x[k] = (T)v[c * V + k];
                if constexpr (WHOLE) {
                    *reinterpret_cast<tv*>(at + d) = x;
                } else if (d + V <= dim) {
                    *reinterpret_cast<tu*>(at + d) = x;
                } else {
#pragma unroll
                    for (int k = 0; k < V - 1; k++)
                        if (d + k < dim) at[d + k] = x[k];
                }
            }
        }
    }
    // a vector of floats (ones without one)
    __device__ static void vec(float* v, const float* p, uint32_t dim, int t, bool aligned) {
        if constexpr (V > 1 && WHOLE) {
            if (p && aligned) {
                typedef float f4 __attribute__((ext_vector_type(4)));
#pragma unroll
                for (int c = 0; c < C; c++) {
                    const uint32_t d = (c * G + t) * V;
#pragma unroll
                    for (int q = 0; q < V / 4; q++) {
                        const f4 x = d < dim ? *reinterpret_cast<const f4*>(p + d + 4 * q) : f4{};
#pragma unroll
                        for (int k = 0; k < 4; k++) v[c * V + 4 * q + k] = x[k];
                    }
                }
                return;
            }
        }
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int k = 0; k < V; k++) {
                const uint32_t d = (c * G + t) * V + k;
                v[c * V + k] = d < dim ? (p ? p[d] : 1.f) : 0.f;
            }
    }
};

// N sums over the threads of a group, the same for all of them.
template <int G, int N> __device__ inline void group_sum(float* v, float (*buf)[8]) {
#pragma unroll
    for (int d = G < 64 ? G / 2 : 32; d; d >>= 1)
#pragma unroll
        for (int n = 0; n < N; n++) v[n] += __shfl_xor(v[n], d);
    if constexpr (G > 64) { // one row a workgroup
        const int w = threadIdx.x >> 6;
        __syncthreads();
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int n = 0; n < N; n++) buf[n][w] = v[n];
        __syncthreads();
#pragma unroll
        for (int n = 0; n < N; n++) {
            float s = buf[n][0];
#pragma unroll
            for (int k = 1; k < G / 64; k++) s += buf[n][k];
            v[n] = s;
        }
    }
}

// The group that holds a row of `dim` columns, as a constant: calls go(std::integral_constant<int, G>).
template <typename F> inline int with_group(uint32_t dim, F&& go) {
    if (dim <= 16 * ROW_E) return go(std::integral_constant<int, 16>{});
    if (dim <= 64 * ROW_E) return go(std::integral_constant<int, 64>{});
    if (dim <= 256 * ROW_E) return go(std::integral_constant<int, 256>{});
    return go(std::integral_constant<int, 512>{});
}

} // namespace apoe
