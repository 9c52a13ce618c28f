// A block's way back into the stream of rows, with the norm in front of the next one, and its gradient:
//   y = x + s sigmoid(g) w h / rms(h),  u = w' y / rms(y).
//
// Bound by memory: forward reads x, h (and g) and writes y and u; the gradient reads those and what comes in, and writes one
// gradient an input. A row is held in registers by a group of G threads (16 values each) from its one read to its writes;
// statistics and everything between are 32 bits, y is rounded once and u comes from the y that is not rounded. The groups walk
// over rows in strides of the grid, so that the vectors s, w, w' stay in registers. The gradients of s, w and a channel gate
// are all multiples of one sum over rows, Q = sum gy sigmoid(g) h / rms(h), and that of w' is R = sum gu y / rms(y): each group
// adds up its rows, a workgroup its groups, a second kernel the workgroups, in a fixed order.
// Measured: 65 536 bf16 rows of 1024 with an element gate, forward 129 us for 671 MB (5.2 TB/s; 152 when a row was asked for only once the one
// in front of it was done), gradient 205 us for 1.07 GB (5.2 TB/s; a copy of 2 GiB runs at 4.86); 10 007 float rows, channel gate: 33 and
// 39 us (164 and 205 MB); the vectors' sums 5 us; 64 rows 5 us. Rows of up to 256 columns are held by 16 threads, in more registers: the gradient runs
// one wave a SIMD, with no loads on their way meanwhile (262 144 bf16 rows of 256: forward 126 us, 5.3 TB/s; gradient 324 us, 3.3 TB/s; of 128
// columns, which leave half of a thread's values empty, 374 us for both, 1.8 TB/s).
#include "apoe_internal.h"
#include "apoe_rows.h"

namespace apoe {

constexpr int RES_E = ROW_E;         // values of a row that a thread holds
constexpr uint32_t RES_BLOCKS = 512; // workgroups of the gradient, at most: rows of the partial sums

struct ResArgs {
    apoe_gated_residual_args p;
    float* part;     // [blocks][2][dim]
    uint32_t blocks;
    bool aligned; // the vectors begin at multiples of 16 bytes
};

__device__ inline float sigmoid(float g) { return 1.f / (1.f + expf(-g)); }

// A gate as the gradient holds it: sigmoid(g) or 1 - sigmoid(g), whichever is smaller, the latter with its sign bit set. Both come from it with
// full accuracy (1 - sigmoid(g) as a difference of floats has 13 bits left at g = 8 and none from 17 on), in one register a value.
constexpr float GATE_OPEN = -0.f;
__device__ inline float gate_of(float g) {
    const float t = expf(-fabsf(g)), least = t * __builtin_amdgcn_rcpf(1.f + t); // a reciprocal of 1 .. 2, right to a unit of the last place
    return g >= 0.f ? -least : least;
}
__device__ inline float gate_open(float v) { return __builtin_signbit(v) ? 1.f + v : v; }
__device__ inline float gate_rest(float v) { return __builtin_signbit(v) ? -v : 1.f - v; }

// GATE: what multiplies the block, in `open` (ones, sigmoid of the row's gate, or of the channel's, which the caller holds).
template <typename T, int V, int G> __global__ __launch_bounds__(G > 256 ? G : 256) void residual_forward(ResArgs a) {
    using R = RowOf<T, V, G>;
    constexpr int GROUPS = (G > 256 ? G : 256) / G;
    __shared__ float buf[2][8];
    const apoe_gated_residual_args& p = a.p;
    const int t = threadIdx.x % G;
    const float inv = 1.f / (float)p.dim;
    const bool element = p.gate_kind == APOE_GATE_ELEMENT;
    // a row is asked for before the one in front of it is worked on, the first before the vectors
    typename R::tv xr[R::C], hr[R::C], gr[R::C];
    auto ask = [&](uint64_t row) {
        if (row >= p.rows) return;
        R::fetch(xr, p.x, row, p.x_stride, p.dim, t);
        if (!p.h) return;
        R::fetch(hr, p.h, row, p.h_stride, p.dim, t);
        if (element) R::fetch(gr, p.gate, row, p.gate_stride, p.dim, t);
    };
    const uint64_t step = (uint64_t)gridDim.x * GROUPS;
    uint64_t row = (uint64_t)blockIdx.x * GROUPS + threadIdx.x / G;
    ask(row);
    float sw[RES_E], wn[RES_E];
    R::vec(sw, p.scale, p.dim, t, a.aligned);
    R::vec(wn, p.w_next, p.dim, t, a.aligned);
    {
        float w[RES_E];
        R::vec(w, p.w_post, p.dim, t, a.aligned);
#pragma unroll
        for (int k = 0; k < RES_E; k++) sw[k] *= w[k];
        if (p.gate_kind == APOE_GATE_CHANNEL) {
            R::load(w, p.gate, 0, 0, p.dim, t);
#pragma unroll
            for (int k = 0; k < RES_E; k++) sw[k] *= sigmoid(w[k]);
        }
    }
    for (; row < p.rows; row += step) {
        float y[RES_E], h[RES_E], g[RES_E];
        R::widen(y, xr);
        if (p.h) {
            R::widen(h, hr);
            if (element) R::widen(g, gr);
        }
        ask(row + step);
        if (p.h) {
            float s[1] = {0.f};
#pragma unroll
            for (int k = 0; k < RES_E; k++) s[0] = __builtin_fmaf(h[k], h[k], s[0]);
            group_sum<G, 1>(s, buf);
            const float rh = rsqrtf(__builtin_fmaf(s[0], inv, p.eps));
#pragma unroll
            for (int k = 0; k < RES_E; k++) {
                float b = h[k] * rh * sw[k];
                if (element) b *= sigmoid(g[k]);
                y[k] += b;
            }
            if (p.y) R::store(p.y, row, p.y_stride, p.dim, t, y);
        }
        if (p.u) {
            float s[1] = {0.f};
#pragma unroll
            for (int k = 0; k < RES_E; k++) s[0] = __builtin_fmaf(y[k], y[k], s[0]);
            group_sum<G, 1>(s, buf);
            const float ry = rsqrtf(__builtin_fmaf(s[0], inv, p.eps));
#pragma unroll
            for (int k = 0; k < RES_E; k++) y[k] = y[k] * ry * wn[k];
            R::store(p.u, row, p.u_stride, p.dim, t, y);
        }
    }
}

template <typename T, int V, int G> __global__ __launch_bounds__(G > 256 ? G : 256) void residual_backward(ResArgs a) {
    using R = RowOf<T, V, G>;
    constexpr int THREADS = G > 256 ? G : 256, GROUPS = THREADS / G;
    __shared__ float buf[2][8];
    __shared__ float sums[GROUPS > 1 ? THREADS * RES_E : 1];
    const apoe_gated_residual_args& p = a.p;
    const int t = threadIdx.x % G, group = threadIdx.x / G;
    const float inv = 1.f / (float)p.dim;
    const bool channel = p.gate_kind == APOE_GATE_CHANNEL, element = p.gate_kind == APOE_GATE_ELEMENT;
    float sw[RES_E], wn[RES_E], oc[RES_E], Q[RES_E] = {}, Rn[RES_E] = {};
    R::vec(sw, p.scale, p.dim, t, a.aligned);
    R::vec(wn, p.w_next, p.dim, t, a.aligned);
    {
        float w[RES_E];
        R::vec(w, p.w_post, p.dim, t, a.aligned);
        if (channel) R::load(oc, p.gate, 0, 0, p.dim, t);
#pragma unroll
        for (int k = 0; k < RES_E; k++) {
            sw[k] *= w[k];
            oc[k] = channel ? gate_of(oc[k]) : GATE_OPEN;
        }
    }
    for (uint64_t row = (uint64_t)blockIdx.x * GROUPS + group; row < p.rows; row += (uint64_t)gridDim.x * GROUPS) {
        float y[RES_E], h[RES_E], o[RES_E], gy[RES_E], rh = 0.f;
        R::load(y, p.x, row, p.x_stride, p.dim, t);
        if (p.h) {
            R::load(h, p.h, row, p.h_stride, p.dim, t);
            if (element) R::load(o, p.gate, row, p.gate_stride, p.dim, t);
            float s[1] = {0.f};
#pragma unroll
            for (int k = 0; k < RES_E; k++) s[0] = __builtin_fmaf(h[k], h[k], s[0]);
            group_sum<G, 1>(s, buf);
            rh = rsqrtf(__builtin_fmaf(s[0], inv, p.eps));
#pragma unroll
            for (int k = 0; k < RES_E; k++) {
                o[k] = element ? gate_of(o[k]) : oc[k];
                h[k] *= rh;
                y[k] = __builtin_fmaf(h[k] * sw[k], gate_open(o[k]), y[k]);
            }
        }
        if (p.grad_u) {
            float gu[RES_E], s[2] = {0.f, 0.f};
            R::load(gu, p.grad_u, row, p.grad_u_stride, p.dim, t);
            if (p.grad_y) R::load(gy, p.grad_y, row, p.grad_y_stride, p.dim, t);
#pragma unroll
            for (int k = 0; k < RES_E; k++) {
                s[0] = __builtin_fmaf(y[k], y[k], s[0]);
                s[1] = __builtin_fmaf(gu[k] * wn[k], y[k], s[1]);
            }
            group_sum<G, 2>(s, buf);
            const float ry = rsqrtf(__builtin_fmaf(s[0], inv, p.eps)), mean = s[1] * ry * inv;
#pragma unroll
            for (int k = 0; k < RES_E; k++) {
                const float yn = y[k] * ry;
                Rn[k] = __builtin_fmaf(gu[k], yn, Rn[k]);
                const float g = ry * (gu[k] * wn[k] - yn * mean);
                gy[k] = p.grad_y ? gy[k] + g : g;
            }
        } else {
            R::load(gy, p.grad_y, row, p.grad_y_stride, p.dim, t);
        }
        if (p.grad_x) R::store(p.grad_x, row, p.grad_x_stride, p.dim, t, gy);
        if (p.h) {
            float s[1] = {0.f};
#pragma unroll
            for (int k = 0; k < RES_E; k++) {
                gy[k] *= gate_open(o[k]); // from here on with the gate
                Q[k] = __builtin_fmaf(gy[k], h[k], Q[k]);
                s[0] = __builtin_fmaf(gy[k] * sw[k], h[k], s[0]);
            }
            if (element && p.grad_gate) {
                float gg[RES_E];
#pragma unroll
                for (int k = 0; k < RES_E; k++) gg[k] = gy[k] * sw[k] * h[k] * gate_rest(o[k]);
                R::store(p.grad_gate, row, p.grad_gate_stride, p.dim, t, gg);
            }
            if (p.grad_h) {
                group_sum<G, 1>(s, buf);
                const float mean = s[0] * inv;
#pragma unroll
                for (int k = 0; k < RES_E; k++) gy[k] = rh * (gy[k] * sw[k] - h[k] * mean);
                R::store(p.grad_h, row, p.grad_h_stride, p.dim, t, gy);
            }
        }
    }
    if (!a.part) return;
    float* out = a.part + (size_t)blockIdx.x * 2 * p.dim;
#pragma unroll
    for (int which = 0; which < 2; which++) {
        float* v = which ? Rn : Q;
        if constexpr (GROUPS > 1) {
            __syncthreads();
#pragma unroll
            for (int k = 0; k < RES_E; k++) sums[k * THREADS + threadIdx.x] = v[k];
            __syncthreads();
            if (group == 0)
#pragma unroll
                for (int k = 0; k < RES_E; k++) {
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

// Columns' sums over the workgroups, and from them the vectors' gradients: 16 columns a workgroup, 64 threads each (512 rows of
// partial sums are eight loads a thread; four threads a column took 42 us at 1024 columns, these 6).
template <typename T> __global__ __launch_bounds__(1024) void residual_vectors(ResArgs a) {
    __shared__ float q[64][17], r[64][17];
    const apoe_gated_residual_args& p = a.p;
    const uint32_t c = threadIdx.x & 15, l = threadIdx.x >> 4, d = blockIdx.x * 16 + c;
    float Q = 0.f, R = 0.f;
    if (d < p.dim)
#pragma unroll 4
        for (uint32_t b = l; b < a.blocks; b += 64) {
            Q += a.part[(size_t)b * 2 * p.dim + d];
            R += a.part[((size_t)b * 2 + 1) * p.dim + d];
        }
    q[l][c] = Q;
    r[l][c] = R;
    for (uint32_t n = 32; n; n >>= 1) {
        __syncthreads();
        if (l < n) {
            q[l][c] += q[l + n][c];
            r[l][c] += r[l + n][c];
        }
    }
    if (l || d >= p.dim) return;
    Q = q[0][c];
    R = r[0][c];
    const float s = p.scale ? p.scale[d] : 1.f, w = p.w_post ? p.w_post[d] : 1.f;
    if (p.grad_scale) p.grad_scale[d] = Q * w;
    if (p.grad_w_post) p.grad_w_post[d] = Q * s;
    if (p.grad_w_next) p.grad_w_next[d] = R;
    if (p.gate_kind == APOE_GATE_CHANNEL && p.grad_gate) ((T*)p.grad_gate)[d] = (T)(Q * s * w * sigmoid(-(float)((const T*)p.gate)[d]));
}

template <typename T, int V> static int run_residual(apoe_ctx* ctx, const apoe_gated_residual_args* p, bool grad) {
    ResArgs a{*p, nullptr, 0, (((uintptr_t)p->scale | (uintptr_t)p->w_post | (uintptr_t)p->w_next) & 15) == 0};
    hipStream_t s = ctx->stream;
    const uint32_t cus = (uint32_t)ctx->num_cus;
    auto go = [&](auto size) -> int {
        constexpr int G = decltype(size)::value, THREADS = G > 256 ? G : 256;
        const uint32_t need = (uint32_t)(((uint64_t)p->rows + THREADS / G - 1) / (THREADS / G));
        if (!grad) {
            residual_forward<T, V, G><<<std::min(need, cus * 8), THREADS, 0, s>>>(a);
            return APOE_OK;
        }
        a.blocks = std::min(need, RES_BLOCKS);
        const bool vectors = p->grad_scale || p->grad_w_post || p->grad_w_next || (p->gate_kind == APOE_GATE_CHANNEL && p->grad_gate);
        if (vectors) {
            char* ws = nullptr;
            APOE_TRY(ctx->adapt_workspace((size_t)a.blocks * 2 * p->dim * 4, &ws));
            a.part = (float*)ws;
        }
        if (a.blocks) residual_backward<T, V, G><<<a.blocks, THREADS, 0, s>>>(a); // no rows: the vectors' gradients alone, which are zeros
        if (vectors) residual_vectors<T><<<(p->dim + 15) / 16, 1024, 0, s>>>(a);
        return APOE_OK;
    };
    APOE_TRY(with_group(p->dim, go));
    APOE_HIP(hipGetLastError());
    return APOE_OK;
}

template <typename T> static int run_aligned(apoe_ctx* ctx, const apoe_gated_residual_args* p, bool grad) {
    constexpr int V = 16 / (int)sizeof(T);
    // 16 bytes a load where every row begins at a multiple of that
    bool whole = p->dim % V == 0;
    const void* ptrs[] = {p->x, p->h, p->gate, p->y, p->u, p->grad_y, p->grad_u, p->grad_x, p->grad_h, p->gate_kind == APOE_GATE_ELEMENT ? p->grad_gate : nullptr};
    for (const void* q : ptrs) whole &= ((uintptr_t)q & 15) == 0;
    const uint64_t strides[] = {p->x_stride, p->h_stride, p->gate_stride, p->y_stride, p->u_stride, p->grad_y_stride, p->grad_u_stride, p->grad_x_stride, p->grad_h_stride, p->grad_gate_stride};
    for (uint64_t q : strides) whole &= q % V == 0;
    return whole ? run_residual<T, V>(ctx, p, grad) : run_residual<T, 1>(ctx, p, grad);
}

int launch_gated_residual(apoe_ctx* ctx, const apoe_gated_residual_args* p, bool grad) {
    switch (p->dtype) {
    case APOE_F32: return run_aligned<float>(ctx, p, grad);
    case APOE_F16: return run_aligned<_Float16>(ctx, p, grad);
    default: return run_aligned<__bf16>(ctx, p, grad);
    }
}

} // namespace apoe
