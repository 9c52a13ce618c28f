// One AdamW step over many parameters, moments in 32 bits or in 8:
//   m' = m + (1 - b1)(g - m), v' = v + (1 - b2)(g g - v), p' = p - lr (decay p + (m' / (1 - b1^t)) / (sqrt(v' / (1 - b2^t)) + eps)).
//
// Bound by memory: p, m, v read and written, g read, a 16-bit copy written: 28 to 30 bytes a value, in 8 bits 14 to 16. The list of parameters
// travels in the kernel's arguments, so that there is nothing to copy to the GPU and a call can be captured; a workgroup finds its parameter
// by the number of its piece. A wave works on 256 values at a time, a block of the 8-bit moments.
// 8 bits: m = s c |c| / 127^2, v = s c^4 / 255^4, s the block's largest. Squares and fourth powers put the codes close together where values are
// small: the smallest v is 4e9 times below the largest (a root that steps divide by: 65 025 times). An average that moves by a
// thousandth a step would stand still if it were rounded to the nearest code, so it goes up or down by chance, with the probability that keeps
// its mean in m and in v. What is above a code is a difference of two close numbers, and the comparison with the chance decides a
// code: both in 64 bits, at the same rate as 32 on this GPU's vector units.
// Measured: 132 M values in twelve layers and a table, 32 bits 711 us for 3.7 GB (5.2 TB/s); 8 bits 571 us for 2.1 GB (3.7 TB/s): 140 vector instructions a value, which
// keep the units busy in nine cycles of ten (guesses that may be off at a code's very end 536; deciding the codes in 32 bits with 64 as a fallback 719); reading
// the moments back 297 us for 1.3 GB. 8.4 M values in 32 bits 50 us (4.7 TB/s).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "apoe_internal.h"

namespace apoe {

constexpr uint32_t ADAM_LIST = 44;       // parameters of a launch: what the kernel's arguments have room for
constexpr uint32_t ADAM_PIECE = 4096;    // values of a workgroup
constexpr uint32_t BLOCK = APOE_ADAMW_BLOCK;

using f32x4a = float __attribute__((ext_vector_type(4)));
using u32x2a = uint32_t __attribute__((ext_vector_type(2)));
using u32x4a = uint32_t __attribute__((ext_vector_type(4)));

struct AdamTensor {
    float* p;
    const void* g;
    void *m, *v;
    float *ms, *vs;
    void* copy;
    uint64_t n;
    float decay;
    uint32_t index;       // in the caller's list
    uint32_t first;       // its first piece
    uint8_t g_type, copy_type, whole; // whole: four values a load
};

struct AdamArgs {
    AdamTensor t[ADAM_LIST];
    uint32_t count, pieces, seed, step;
    const uint32_t* step_dev;
    const float* lr_dev;
    uint32_t* taken;
    double b1, b2, grad_scale;
    float lr, eps, c1, c2; // c: one over 1 - b^t
};
static_assert(sizeof(AdamArgs) <= 4096, "the arguments of a kernel");

__device__ __host__ inline uint32_t mix(uint32_t h) { // the finishing rounds of a 32-bit hash (Appleby's fmix32): shifts and odd multipliers
    h = (h ^ (h >> 16)) * 0x85ebca6bu;
    h = (h ^ (h >> 13)) * 0xc2b2ae35u;
    return h ^ (h >> 16);
}

__device__ __host__ inline double power(double b, uint32_t t) {
    double r = 1.;
    for (; t; t >>= 1, b *= b)
        if (t & 1) r *= b;
    return r;
}

// A moment's step in 64 bits, every operation rounded by itself: a tenth of the way between two floats lies half way between two others often enough
// that the largest of a block, which is rounded to a float, must not hang on how the operations are joined.
__device__ inline double moved(double m, double target, double share) {
#pragma clang fp contract(off)
    const double way = target - m;
    const double part = share * way;
    return m + part;
}
__device__ inline double value_of_m(float scale, int c) {
#pragma clang fp contract(off)
    const double r = (double)(c * abs(c)) * (1. / (127. * 127.));
    return (double)scale * r;
}
__device__ inline double value_of_v(float scale, uint32_t c) {
#pragma clang fp contract(off)
    const double r = (double)(c * c * c * c) * (1. / (255. * 255. * 255. * 255.)); // below 2^32
    return (double)scale * r;
}

// Values k of a lane: four in a row, or (parameters that begin anywhere, a block's rest) 64 apart.
__device__ inline uint32_t place(bool whole, int lane, int k) { return whole ? (uint32_t)lane * 4 + k : (uint32_t)k * 64 + lane; }

template <typename T> __device__ inline void load4(T* x, const T* from, uint64_t at, bool whole, int lane, uint32_t left) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    if (whole) {
        const t4 v = *reinterpret_cast<const t4*>(from + at + lane * 4);
#pragma unroll
        for (int k = 0; k < 4; k++) x[k] = v[k];
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const uint32_t i = place(false, lane, k);
            x[k] = i < left ? from[at + i] : (T)0;
        }
    }
}

template <typename T> __device__ inline void store4(T* to, const T* x, uint64_t at, bool whole, int lane, uint32_t left) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    if (whole) {
        t4 v;
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = x[k];
        *reinterpret_cast<t4*>(to + at + lane * 4) = v;
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const uint32_t i = place(false, lane, k);
            if (i < left) to[at + i] = x[k];
        }
    }
}

// The largest of the wave's numbers by magnitude, the same for all lanes: as bits of floats without their signs, so that a NaN is larger than all. Rows of
// sixteen lanes by moves between lanes, the four rows in scalar registers.
__device__ inline float wave_largest(uint32_t b) {
    const auto with = [&](auto control) { b = max(b, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)b, decltype(control)::value, 0xf, 0xf, true)); };
    with(std::integral_constant<int, 0xB1>{});  // lane xor 1
    with(std::integral_constant<int, 0x4E>{});  // lane xor 2
    with(std::integral_constant<int, 0x141>{}); // mirrored in eight
    with(std::integral_constant<int, 0x140>{}); // mirrored in sixteen
    const uint32_t r0 = __builtin_amdgcn_readlane((int)b, 0), r1 = __builtin_amdgcn_readlane((int)b, 16), r2 = __builtin_amdgcn_readlane((int)b, 32), r3 = __builtin_amdgcn_readlane((int)b, 48);
    return __uint_as_float(max(max(r0, r1), max(r2, r3)));
}

// most / top, off by a unit of the last place at most; zero where top is zero or not finite.
__device__ inline double share_of(double most, float top) {
    if (!(top > 0.f && top < INFINITY)) return 0.;
    const double t = (double)top;
    double r = __builtin_amdgcn_rcp(t);
    r = __builtin_fma(__builtin_fma(-t, r, 1.), r, r);
    r = __builtin_fma(__builtin_fma(-t, r, 1.), r, r);
    return most * r;
}

// The code of w = STEPS^POWER x / top >= 0: k, the last one at or below w, or k + 1 where `chance` is below the share of the way between them that w has gone. k comes from
// a root in 32 bits that is taken a little too large: it is the right one or, seldom, the next, with w below it; whoever calls looks for that. The block's largest
// counts as on its way to the last code: rounded to a float it can be larger than it was. A top that is not finite gives zero: the block's values are its scale's.
template <int POWER, int STEPS> struct Code {
    float k;
    double above; // of w, above k
    __device__ double gap() const { // from k to the next: of numbers that floats hold, as k k is
        const double g = (double)__builtin_fmaf(2.f, k, 1.f);
        return POWER == 2 ? g : g * (double)__builtin_fmaf(2.f, __builtin_fmaf(k, k, k), 1.f);
    }
    __device__ void guess(double w) {
        float r = __builtin_amdgcn_sqrtf((float)w);
        if constexpr (POWER == 4) r = __builtin_amdgcn_sqrtf(r);
        k = floorf(__builtin_fmaf(r, 0x1p-21f, r));
        k = k >= (float)STEPS ? (float)(STEPS - 1) : k;
        const double square = (double)(k * k);
        above = POWER == 2 ? w - square : __builtin_fma(-square, square, w);
    }
    __device__ void correct() {
        if (above < 0.) {
            k -= 1.f;
            above += gap();
        }
    }
    __device__ uint32_t sign() const { return (uint32_t)(__builtin_bit_cast(uint64_t, above) >> 32); }
    __device__ int take(uint32_t chance) const {
        const double u = __builtin_fma((double)chance, 0x1p-32, 0x1p-33);
        return (int)k + (u * gap() < above ? 1 : 0);
    }
};

// What a lane needs of a block, as it comes: nothing here waits for a load.
template <int BITS> struct AdamRaw {
    f32x4a p, m, v;
    u32x4a g;        // floats, or two 16-bit values a word
    uint32_t cm, cv; // four codes
    float sm, sv;
    __device__ void fetch(const AdamTensor& t, uint64_t at, int lane) {
        const uint32_t left = (uint32_t)min((uint64_t)BLOCK, t.n - at);
        if (t.whole && left == BLOCK) {
            const uint64_t e = at + lane * 4;
            p = *reinterpret_cast<const f32x4a*>(t.p + e);
            if (t.g_type == APOE_F32) {
                g = *reinterpret_cast<const u32x4a*>((const float*)t.g + e);
            } else {
                const u32x2a x = *reinterpret_cast<const u32x2a*>((const uint16_t*)t.g + e);
                g[0] = x[0];
                g[1] = x[1];
            }
            if constexpr (BITS == 32) {
                m = *reinterpret_cast<const f32x4a*>((const float*)t.m + e);
                v = *reinterpret_cast<const f32x4a*>((const float*)t.v + e);
            } else {
                cm = *reinterpret_cast<const uint32_t*>((const int8_t*)t.m + e);
                cv = *reinterpret_cast<const uint32_t*>((const uint8_t*)t.v + e);
            }
        } else {
            g = u32x4a{};
            cm = cv = 0;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const uint32_t i = place(false, lane, k);
                const bool in = i < left;
                p[k] = in ? t.p[at + i] : 0.f;
                if (t.g_type == APOE_F32) g[k] = in ? ((const uint32_t*)t.g)[at + i] : 0u;
                else g[k >> 1] |= (in ? (uint32_t)((const uint16_t*)t.g)[at + i] : 0u) << (16 * (k & 1));
                if constexpr (BITS == 32) {
                    m[k] = in ? ((const float*)t.m)[at + i] : 0.f;
                    v[k] = in ? ((const float*)t.v)[at + i] : 0.f;
                } else {
                    cm |= (in ? (uint32_t)((const uint8_t*)t.m)[at + i] : 0u) << (8 * k);
                    cv |= (in ? (uint32_t)((const uint8_t*)t.v)[at + i] : 0u) << (8 * k);
                }
            }
        }
        if constexpr (BITS == 8) {
            sm = t.ms[at / BLOCK];
            sv = t.vs[at / BLOCK];
        }
    }
    __device__ float grad(int k, uint32_t type) const {
        if (type == APOE_F32) return __uint_as_float(g[k]);
        const uint16_t h = (uint16_t)(g[k >> 1] >> (16 * (k & 1)));
        return type == APOE_F16 ? (float)__builtin_bit_cast(_Float16, h) : __uint_as_float((uint32_t)h << 16);
    }
};

// NEAR: root and reciprocal to a unit of the last place. A block is asked for before the one in front of it is worked on.
template <int BITS, bool NEAR> __global__ __launch_bounds__(256) void adamw_step(AdamArgs a) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint32_t which = 0;
    for (uint32_t lo = 0, hi = a.count; hi - lo > 1;) { // the last parameter whose first piece is at or before this one
        const uint32_t mid = (lo + hi) / 2;
        if (a.t[mid].first <= blockIdx.x) lo = mid;
        else hi = mid;
        which = lo;
    }
    const AdamTensor& t = a.t[which];
    const uint64_t begin = (uint64_t)(blockIdx.x - t.first) * ADAM_PIECE, end = min(begin + ADAM_PIECE, t.n);
    uint64_t at = begin + wave * BLOCK;
    AdamRaw<BITS> next;
    if (at < end) next.fetch(t, at, lane);
    float c1 = a.c1, c2 = a.c2, lr = a.lr;
    uint32_t step = a.step;
    if (a.step_dev) {
        step = *a.step_dev;
        c1 = (float)(1. / (1. - power(a.b1, step)));
        c2 = (float)(1. / (1. - power(a.b2, step)));
    }
    if (a.lr_dev) lr = *a.lr_dev;
    if (a.taken && blockIdx.x == 0 && threadIdx.x == 0) *a.taken = step;
    const uint32_t key = mix(mix(mix(a.seed) ^ step) ^ t.index);
    const uint32_t g_type = t.g_type;
    for (; at < end; at += 4 * BLOCK) {
        const uint32_t left = (uint32_t)min((uint64_t)BLOCK, t.n - at);
        const bool whole = t.whole && left == BLOCK;
        const AdamRaw<BITS> now = next;
        if (at + 4 * BLOCK < end) next.fetch(t, at + 4 * BLOCK, lane);
        float p[4], m[4], v[4];
        if constexpr (BITS == 32) {
            const float d1 = (float)(1. - a.b1), d2 = (float)(1. - a.b2), gs = (float)a.grad_scale;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float x = now.grad(k, g_type) * gs;
                m[k] = __builtin_fmaf(d1, x - now.m[k], now.m[k]);
                v[k] = __builtin_fmaf(d2, __builtin_fmaf(x, x, -now.v[k]), now.v[k]);
            }
            store4((float*)t.m, m, at, whole, lane, left);
            store4((float*)t.v, v, at, whole, lane, left);
        } else {
            const uint64_t block = at / BLOCK;
            double md[4], vd[4];
            uint32_t mb = 0, vb = 0; // the largest, by magnitude; a value beyond the parameter's end is zero
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const bool in = whole || place(false, lane, k) < left;
                const double x = (double)now.grad(k, g_type) * a.grad_scale;
                md[k] = in ? moved(value_of_m(now.sm, (int8_t)(now.cm >> (8 * k))), x, 1. - a.b1) : 0.;
                vd[k] = in ? moved(value_of_v(now.sv, (uint8_t)(now.cv >> (8 * k))), x * x, 1. - a.b2) : 0.;
                m[k] = (float)md[k];
                v[k] = (float)vd[k];
                mb = max(mb, __float_as_uint(m[k]) & 0x7fffffffu);
                vb = max(vb, __float_as_uint(v[k]) & 0x7fffffffu);
            }
            const float mt = wave_largest(mb), vt = wave_largest(vb);
            const double im = share_of(127. * 127., mt), iv = share_of(255. * 255. * 255. * 255., vt);
            const uint32_t bk = mix(mix(key ^ (uint32_t)block) ^ (uint32_t)(block >> 32));
            int8_t cm[4];
            uint8_t cv[4];
            const auto codes = [&](auto code, const double* x, double inv, uint32_t which, auto&& put) { // the codes of four numbers without their signs
                decltype(code) c[4];
                uint32_t below = 0; // whether a guess is above its number: one in some 20 000, so that a wave seldom has any
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    c[k].guess(fabs(x[k]) * inv);
                    below |= c[k].sign();
                }
                if (__builtin_expect(__ballot((int32_t)below < 0) != 0, 0)) {
#pragma unroll
                    for (int k = 0; k < 4; k++) c[k].correct();
                }
#pragma unroll
                for (int k = 0; k < 4; k++) put(k, c[k].take(mix(bk + 2 * place(whole, lane, k) + which)));
            };
            codes(Code<2, 127>{}, md, im, 0, [&](int k, int c) { cm[k] = (int8_t)(md[k] < 0. ? -c : c); });
            codes(Code<4, 255>{}, vd, iv, 1, [&](int k, int c) { cv[k] = (uint8_t)(vd[k] > 0. ? max(c, 1) : 0); });
            store4((int8_t*)t.m, cm, at, whole, lane, left);
            store4((uint8_t*)t.v, cv, at, whole, lane, left);
            if (lane == 0) {
                t.ms[block] = mt;
                t.vs[block] = vt;
            }
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
            m[k] = NEAR ? m[k] * c1 * __builtin_amdgcn_rcpf(__builtin_amdgcn_sqrtf(v[k] * c2) + a.eps) : m[k] * c1 / (sqrtf(v[k] * c2) + a.eps);
            p[k] = __builtin_fmaf(-lr, __builtin_fmaf(t.decay, now.p[k], m[k]), now.p[k]);
        }
        store4(t.p, p, at, whole, lane, left);
        if (t.copy) {
            if (t.copy_type == APOE_F16) {
                _Float16 h[4];
#pragma unroll
                for (int k = 0; k < 4; k++) h[k] = (_Float16)p[k];
                store4((_Float16*)t.copy, h, at, whole, lane, left);
            } else {
                __bf16 h[4];
#pragma unroll
                for (int k = 0; k < 4; k++) h[k] = (__bf16)p[k];
                store4((__bf16*)t.copy, h, at, whole, lane, left);
            }
        }
    }
}

// A step of no parameter at all.
__global__ void adamw_count(AdamArgs a) { *a.taken = a.step_dev ? *a.step_dev : a.step; }

// Four values a thread from a block's beginning on.
__global__ __launch_bounds__(256) void adamw_read(uint64_t n, const int8_t* m, const float* ms, const uint8_t* v, const float* vs, float* m_out, float* v_out, bool whole) {
    const int lane = threadIdx.x & 63;
    for (uint64_t at = ((uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * BLOCK; at < n; at += (uint64_t)gridDim.x * 4 * BLOCK) {
        const uint32_t left = (uint32_t)min((uint64_t)BLOCK, n - at);
        const bool w = whole && left == BLOCK;
        int8_t cm[4];
        uint8_t cv[4];
        load4(cm, m, at, w, lane, left);
        load4(cv, v, at, w, lane, left);
        const float sm = ms[at / BLOCK], sv = vs[at / BLOCK];
        float x[4], y[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            x[k] = (float)value_of_m(sm, cm[k]);
            y[k] = (float)value_of_v(sv, cv[k]);
        }
        store4(m_out, x, at, w, lane, left);
        store4(v_out, y, at, w, lane, left);
    }
}

int launch_adamw(apoe_adamw* opt, const apoe_adamw_step_args* p) {
    AdamArgs a{};
    a.seed = opt->seed;
    a.step = p->step;
    a.step_dev = p->step_dev;
    a.lr_dev = p->lr_dev;
    a.taken = p->step_taken;
    a.b1 = p->beta1;
    a.b2 = p->beta2;
    a.grad_scale = p->grad_scale;
    a.lr = (float)p->lr;
    a.eps = (float)p->eps;
    if (!p->step_dev) {
        a.c1 = (float)(1. / (1. - power(a.b1, a.step)));
        a.c2 = (float)(1. / (1. - power(a.b2, a.step)));
    }
    auto go = [&]() -> int {
        if (a.pieces == 0) return APOE_OK;
        // In 8 bits the kernel's operations are what it waits for: root and reciprocal to a unit of the last place (132 M values then took 568 us, with a
        // rounded root and quotient 670). Their instructions take numbers below 2^-126 for zero: beside an eps of 2^-36 and more, such a root counts nothing.
        const bool near = p->eps >= 0x1p-36;
        const auto run = [&](auto kernel) { kernel<<<a.pieces, 256, 0, opt->ctx->stream>>>(a); };
        if (opt->bits == 32) run(near ? adamw_step<32, true> : adamw_step<32, false>);
        else run(near ? adamw_step<8, true> : adamw_step<8, false>);
        a.count = a.pieces = 0;
        a.taken = nullptr; // (the first launch tells)
        APOE_HIP(hipGetLastError());
        return APOE_OK;
    };
    for (size_t i = 0; i < opt->tensors.size(); i++) {
        const apoe_adamw_tensor& t = opt->tensors[i];
        if (!p->grads[i] || t.n == 0) continue;
        const uint32_t pieces = (uint32_t)((t.n + ADAM_PIECE - 1) / ADAM_PIECE);
        if (a.count == ADAM_LIST || a.pieces + (uint64_t)pieces > (1u << 23)) APOE_TRY(go());
        const uintptr_t g = (uintptr_t)p->grads[i], c = (uintptr_t)t.copy;
        const bool narrow = p->grad_dtypes[i] != APOE_F32;
        bool whole = ((uintptr_t)t.p & 15) == 0 && (g & (narrow ? 7 : 15)) == 0 && (c & 7) == 0;
        whole &= (((uintptr_t)t.m | (uintptr_t)t.v) & (opt->bits == 32 ? 15 : 3)) == 0;
        a.t[a.count++] = AdamTensor{t.p, p->grads[i], t.m, t.v, t.m_scale, t.v_scale, t.copy, t.n, (float)t.decay, (uint32_t)i, a.pieces, (uint8_t)p->grad_dtypes[i],
                                    (uint8_t)t.copy_dtype, (uint8_t)whole};
        a.pieces += pieces;
    }
    if (a.pieces == 0 && a.taken) {
        adamw_count<<<1, 1, 0, opt->ctx->stream>>>(a);
        APOE_HIP(hipGetLastError());
        return APOE_OK;
    }
    return go();
}

int launch_adamw_moments(apoe_ctx* ctx, uint64_t n, const int8_t* m, const float* m_scale, const uint8_t* v, const float* v_scale, float* m_out, float* v_out) {
    const bool whole = ((((uintptr_t)m | (uintptr_t)v) & 3) | (((uintptr_t)m_out | (uintptr_t)v_out) & 15)) == 0;
    adamw_read<<<(uint32_t)std::min<uint64_t>((n + 1023) / 1024, 1u << 16), 256, 0, ctx->stream>>>(n, m, m_scale, v, v_scale, m_out, v_out, whole);
    APOE_HIP(hipGetLastError());
    return APOE_OK;
}

} // namespace apoe
