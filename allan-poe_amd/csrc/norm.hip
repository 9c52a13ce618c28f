// Layer norm of rows, and its gradient:
//   y = w n + b, n = r (x - mean x), r = 1 / sqrt(mean (x - mean x)^2 + eps);
//   gx = r (g - mean g - n mean(g n)) with g = w gy (and what x's gradient has by another way), gw = sum gy n, gb = sum gy over the rows.
//
// Bound by memory. A row is held in registers from its one read to its writes (a group of G threads, 16 values each), so the variance is
// that of the values about their mean, in a second pass over registers: no difference of squares. A float's mean of values far from zero is off by as much as their differences may be: what
// is left of it in the differences is taken off them and out of the variance (a row of 1024 values of 10 000 gave 0.3 for 0 without). The gradient forms the statistics again
// from x, which it reads anyway. Groups walk over rows in strides of the grid, w and b stay in registers, and a row is asked for before the
// one in front of it is worked on. The vectors' gradients: each group adds up its rows, a workgroup its groups, a second kernel the workgroups, in
// a fixed order.
// Measured (a copy of 2 GiB runs at 4.9 TB/s): 65 536 bf16 rows of 1024, forward 51 us for 268 MB (5.3 TB/s), gradient with grad_skip 106 us for 537 MB (5.1), the vectors'
// sums 5 to 6; 10 007 float rows 16 and 24 us (5 TB/s); 262 144 bf16 rows of 256 49 and 125 us; rows of 1001 fp16 values, which begin anywhere and end in a value by itself: 60 000 of
// them 77 and 126 us (3.1 and 2.9 TB/s); 64 rows 4 us.
#include <algorithm>

#include "apoe_internal.h"
#include "apoe_rows.h"

namespace apoe {

constexpr uint32_t NORM_BLOCKS = 512; // workgroups of the gradient, at most: rows of the partial sums

struct NormArgs {
    apoe_layer_norm_args p;
    float* part; // [blocks][2][dim]
    uint32_t blocks;
    bool aligned; // the vectors begin at multiples of 16 bytes
};

// v less its mean (zeros beyond the row), and one over its deviation.
template <typename R, int V, int G, bool WHOLE> __device__ inline float normalise(float* v, uint32_t dim, float inv, float eps, int t, float (*buf)[8]) {
    float s[1] = {0.f};
#pragma unroll
    for (int k = 0; k < ROW_E; k++) s[0] += v[k];
    group_sum<G, 1>(s, buf);
    const float mean = s[0] * inv;
    float q[2] = {0.f, 0.f};
#pragma unroll
    for (int c = 0; c < R::C; c++) {
        const uint32_t d = (c * G + t) * V;
#pragma unroll
        for (int k = 0; k < V; k++) {
            float& x = v[c * V + k];
            x = d + (WHOLE ? 0 : k) < dim ? x - mean : 0.f;
            q[0] += x;
            q[1] = __builtin_fmaf(x, x, q[1]);
        }
    }
    group_sum<G, 2>(q, buf);
    const float rest = q[0] * inv;
#pragma unroll
    for (int c = 0; c < R::C; c++) {
        const uint32_t d = (c * G + t) * V;
#pragma unroll
        for (int k = 0; k < V; k++) v[c * V + k] -= d + (WHOLE ? 0 : k) < dim ? rest : 0.f;
    }
    return 1.f / sqrtf(fmaxf(__builtin_fmaf(-rest, rest, q[1] * inv), 0.f) + eps);
}

template <typename T, int V, int G, bool WHOLE> __global__ __launch_bounds__(G > 256 ? G : 256) void norm_forward(NormArgs a) {
    using R = RowOf<T, V, G, WHOLE>;
    constexpr int GROUPS = (G > 256 ? G : 256) / G;
    __shared__ float buf[2][8];
    const apoe_layer_norm_args& p = a.p;
    const int t = threadIdx.x % G;
    const float inv = 1.f / (float)p.dim;
    typename R::tv xr[R::C];
    const uint64_t step = (uint64_t)gridDim.x * GROUPS;
    uint64_t row = (uint64_t)blockIdx.x * GROUPS + threadIdx.x / G;
    if (row < p.rows) R::fetch(xr, p.x, row, p.x_stride, p.dim, t);
    float w[ROW_E], b[ROW_E];
    R::vec(w, p.w, p.dim, t, a.aligned);
    if (p.b) {
        R::vec(b, p.b, p.dim, t, a.aligned);
    } else {
#pragma unroll
        for (int k = 0; k < ROW_E; k++) b[k] = 0.f;
    }
    for (; row < p.rows; row += step) {
        float v[ROW_E];
        R::widen(v, xr);
        if (row + step < p.rows) R::fetch(xr, p.x, row + step, p.x_stride, p.dim, t);
        const float r = normalise<R, V, G, WHOLE>(v, p.dim, inv, p.eps, t, buf);
#pragma unroll
        for (int k = 0; k < ROW_E; k++) v[k] = __builtin_fmaf(v[k] * r, w[k], b[k]);
        R::store(p.y, row, p.y_stride, p.dim, t, v);
    }
}

template <typename T, int V, int G, bool WHOLE> __global__ __launch_bounds__(G > 256 ? G : 256) void norm_backward(NormArgs a) {
    using R = RowOf<T, V, G, WHOLE>;
    constexpr int THREADS = G > 256 ? G : 256, GROUPS = THREADS / G;
    __shared__ float buf[2][8];
    __shared__ float sums[GROUPS > 1 ? THREADS * ROW_E : 1];
    const apoe_layer_norm_args& p = a.p;
    const int t = threadIdx.x % G, group = threadIdx.x / G;
    const float inv = 1.f / (float)p.dim;
    typename R::tv xr[R::C], gr[R::C], sr[R::C];
    auto ask = [&](uint64_t row) {
        if (row >= p.rows) return;
        R::fetch(xr, p.x, row, p.x_stride, p.dim, t);
        R::fetch(gr, p.grad_y, row, p.grad_y_stride, p.dim, t);
        if (p.grad_skip) R::fetch(sr, p.grad_skip, row, p.grad_skip_stride, p.dim, t);
    };
    const uint64_t step = (uint64_t)gridDim.x * GROUPS;
    uint64_t row = (uint64_t)blockIdx.x * GROUPS + group;
    ask(row);
    float w[ROW_E], gw[ROW_E] = {}, gb[ROW_E] = {};
    R::vec(w, p.w, p.dim, t, a.aligned);
    for (; row < p.rows; row += step) {
        float v[ROW_E], g[ROW_E];
        R::widen(v, xr);
        R::widen(g, gr);
        typename R::tv skip[R::C];
#pragma unroll
        for (int c = 0; c < R::C; c++) skip[c] = sr[c];
        ask(row + step);
        const float r = normalise<R, V, G, WHOLE>(v, p.dim, inv, p.eps, t, buf);
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < ROW_E; k++) {
            v[k] *= r;
            gb[k] += g[k];
            gw[k] = __builtin_fmaf(g[k], v[k], gw[k]);
            g[k] *= w[k];
            s[0] += g[k];
            s[1] = __builtin_fmaf(g[k], v[k], s[1]);
        }
        if (!p.grad_x) continue;
        group_sum<G, 2>(s, buf);
        const float mean = s[0] * inv, along = s[1] * inv;
#pragma unroll
        for (int k = 0; k < ROW_E; k++) g[k] = r * (g[k] - mean - v[k] * along);
        if (p.grad_skip) {
            R::widen(v, skip);
#pragma unroll
            for (int k = 0; k < ROW_E; k++) g[k] += v[k];
        }
        R::store(p.grad_x, row, p.grad_x_stride, p.dim, t, g);
    }
    if (!a.part) return;
    float* out = a.part + (size_t)blockIdx.x * 2 * p.dim;
#pragma unroll
    for (int which = 0; which < 2; which++) {
        float* v = which ? gb : gw;
        if constexpr (GROUPS > 1) {
            __syncthreads();
#pragma unroll
            for (int k = 0; k < ROW_E; k++) sums[k * THREADS + threadIdx.x] = v[k];
            __syncthreads();
            if (group == 0)
#pragma unroll
                for (int k = 0; k < ROW_E; k++) {
                    float s = v[k];
                    for (int g = 1; g < GROUPS; g++) s += sums[k * THREADS + g * G + t];
                    v[k] = s;
                }
        }
        if (group == 0)
#pragma unroll
            for (int c = 0; c < R::C; c++)
#pragma unroll
                for (int k = 0; k < V; k++) {
                    const uint32_t d = (c * G + t) * V + k;
                    if (d < p.dim) out[(size_t)which * p.dim + d] = v[c * V + k];
                }
    }
}

// Columns' sums over the workgroups: 16 columns a workgroup, 64 threads each, one vector for each blockIdx.y.
__global__ __launch_bounds__(1024) void norm_vectors(NormArgs a) {
    __shared__ float q[64][17];
    const uint32_t c = threadIdx.x & 15, l = threadIdx.x >> 4, d = blockIdx.x * 16 + c, dim = a.p.dim;
    float* out = blockIdx.y ? a.p.grad_b : a.p.grad_w;
    if (!out) return;
    float s = 0.f;
    if (d < dim)
        for (uint32_t b0 = l; b0 < a.blocks; b0 += 512) { // eight loads at once, beyond the last row that one again
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; u++) v[u] = a.part[((size_t)min(b0 + u * 64, a.blocks - 1) * 2 + blockIdx.y) * dim + d];
#pragma unroll
            for (int u = 0; u < 8; u++) s += b0 + u * 64 < a.blocks ? v[u] : 0.f;
        }
    q[l][c] = s;
    for (uint32_t n = 32; n; n >>= 1) {
        __syncthreads();
        if (l < n) q[l][c] += q[l + n][c];
    }
    if (l == 0 && d < dim) out[d] = q[0][c];
}

template <typename T, int V, bool WHOLE> static int run_norm(apoe_ctx* ctx, const apoe_layer_norm_args* p, bool grad) {
    NormArgs a{*p, nullptr, 0, (((uintptr_t)p->w | (uintptr_t)p->b) & 15) == 0};
    hipStream_t s = ctx->stream;
    const uint32_t cus = (uint32_t)ctx->num_cus;
    APOE_TRY(with_group(p->dim, [&](auto size) -> int {
        constexpr int G = decltype(size)::value, THREADS = G > 256 ? G : 256;
        const uint32_t need = (uint32_t)(((uint64_t)p->rows + THREADS / G - 1) / (THREADS / G));
        if (!grad) {
            norm_forward<T, V, G, WHOLE><<<std::min(need, cus * 8), THREADS, 0, s>>>(a);
            return APOE_OK;
        }
        a.blocks = std::min(need, NORM_BLOCKS);
        const bool vectors = p->grad_w || p->grad_b;
        if (vectors) {
            char* ws = nullptr;
            APOE_TRY(ctx->adapt_workspace((size_t)a.blocks * 2 * p->dim * 4, &ws));
            a.part = (float*)ws;
        }
        if (a.blocks) norm_backward<T, V, G, WHOLE><<<a.blocks, THREADS, 0, s>>>(a); // no rows: the vectors' gradients alone, which are zeros
        if (vectors) norm_vectors<<<dim3((p->dim + 15) / 16, 2), 1024, 0, s>>>(a);
        return APOE_OK;
    }));
    APOE_HIP(hipGetLastError());
    return APOE_OK;
}

template <typename T> static int run_aligned(apoe_ctx* ctx, const apoe_layer_norm_args* p, bool grad) {
    constexpr int V = 16 / (int)sizeof(T);
    bool whole = p->dim % V == 0;
    for (const void* q : {p->x, (const void*)p->y, p->grad_y, p->grad_skip, (const void*)p->grad_x}) whole &= ((uintptr_t)q & 15) == 0;
    for (uint64_t q : {p->x_stride, p->y_stride, p->grad_y_stride, p->grad_skip_stride, p->grad_x_stride}) whole &= q % V == 0;
    return whole ? run_norm<T, V, true>(ctx, p, grad) : run_norm<T, V, false>(ctx, p, grad);
}

int launch_layer_norm(apoe_ctx* ctx, const apoe_layer_norm_args* p, bool grad) {
    switch (p->dtype) {
    case APOE_F32: return run_aligned<float>(ctx, p, grad);
    case APOE_F16: return run_aligned<_Float16>(ctx, p, grad);
    default: return run_aligned<__bf16>(ctx, p, grad);
    }
}

} // namespace apoe
