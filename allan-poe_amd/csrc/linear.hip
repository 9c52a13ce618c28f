// A linear layer and its gradient:
//   z = x w^T + b, y = act(z) + residual;   gz = gy act'(z), gx = gz w, gw = gz^T x, gb = sum of gz's rows.
//
// Three products of one kernel: an operand's inner dimension goes along its rows (x, w, and gz for gx) or down them (w for gx, both for gw; read
// transposed from LDS). Float matrices go through the bfloat16 units: a wave takes each value of its operands apart into three parts of eight bits as it comes from LDS, and of
// the nine products the six that count are added up: as accurate value by value as float products, for values of any size from 2^-111 on (the
// last part of smaller ones ends at 2^-133), at a sixth of 1400 TFLOP/s where the float matrix units have 154. What is done to a result (bias, activation, residual, rounding) is done behind the last stage,
// through LDS, 16 bytes a thread. gz of 16-bit matrices with GELU or SiLU has more bits than their type: it is multiplied as two parts, which costs its two products
// twice their operations (rounded to one, gx and gw would be off by 1.4 times their own rounding). Where tiles are too few for the GPU the inner dimension is cut and a second launch adds the cuts up, in order.
// Up to 16 rows a kernel of its own streams w once (the serving form).
// Measured (a library product of 8192 x 8192 x 8192 in bf16 runs at 1470 TFLOP/s, of 8192 x 4096 x 1024 at 1160): 8192 x 4096 x 1024 bf16 73 us (940 TFLOP/s), with GELU and
// both outputs 99, whose operations cost what the products wait for; 8192 x 1024 x 4096 68 (1010), in two parts 131; 4096 x 1024 x 8192, both sides transposed, 76 (900), in two parts 138; 8192 x 4096 x
// 4096 fp16 237 to 243 (1140), with SiLU 258. The matrix units are busy in 55 % of the cycles at most; stages and ends of tiles are what the rest goes to. Float 4096 x
// 4096 x 1024 191 us (180 TFLOP/s; the library 153).
#include <algorithm>
#include <cmath>

#include "apoe_internal.h"
#include "apoe_tile.h"

namespace apoe {

struct LinOut { // what becomes of a product's sums
    void* out;
    const float* bias;      // by columns
    const void* residual;
    void* pre;
    uint64_t out_stride, residual_stride, pre_stride;
    uint32_t m, n, act;
};

struct LinBias { // the bias' gradient, which workgroups behind the tiles' add up from the strips' sums
    const float* part; // [strips][cols]
    float* out;
    uint32_t strips, cols;
};

struct LinTile {
    const void *a, *b;
    uint32_t a_pitch, b_pitch; // bytes
    uint32_t k, mt, nt;     // inner side, tiles down and along
    uint32_t band;          // rows of tiles that are walked through together, column by column
    uint32_t cuts, cut_stages;
    float* part;            // [cuts][m][np]
    uint32_t np;
    uint32_t groups;        // of the product; workgroups behind them: the bias' gradient
    LinOut o;
    LinBias bias;
    uint64_t second;        // bytes from a to its second part (0: it has one)
    bool a_down, b_down;    // the inner dimension goes down the rows
};

// gz of 16-bit matrices with GELU or SiLU, which its type does not hold, as two parts: its rounding, and the rounding of what that leaves. (What ReLU lets back is a value of grad_y.) float16
// holds halves, so that no slope above one makes an infinity, and the second part times 2^11, so that it does not fall below the smallest numbers.
template <typename T> struct Two {
    static constexpr float HALF = 1.f, DOWN = 1.f;
};
template <> struct Two<_Float16> {
    static constexpr float HALF = 0.5f, DOWN = 0x1p-11f;
};

// Phi(-u), the normal distribution's tail, for u >= 0, and its density there: exp(-u u / 2) times a polynomial in 1 / (1 + c u), fitted to
// erfc's scaled form: off by 1.4e-7 of itself up to u = 13, behind which the exponential is zero, with its coefficients as floats, by 4e-7 as operations of 32 bits form it; the exponent's
// rounding adds up to 1.3 u u 2^-24.
__device__ inline float normal_tail(float u, float& density) {
    const float e = __builtin_amdgcn_exp2f(-0.72134752f * (u * u)), t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.28284271f, u, 1.f));
    density = 0.39894228f * e;
    float s = 0.0201337803f;
    s = __builtin_fmaf(s, t, -0.0677357092f);
    s = __builtin_fmaf(s, t, 0.0369214416f);
    s = __builtin_fmaf(s, t, 0.0498643406f);
    s = __builtin_fmaf(s, t, 0.0357544832f);
    s = __builtin_fmaf(s, t, 0.0984813645f);
    s = __builtin_fmaf(s, t, 0.100479335f);
    s = __builtin_fmaf(s, t, 0.113287851f);
    s = __builtin_fmaf(s, t, 0.112813152f);
    return s * t * e;
}

__device__ inline float relu(float z) { return z < 0.f ? 0.f : z; }
__device__ inline float gelu(float z) {
    float d;
    const float q = normal_tail(fabsf(z), d);
    return z * (z > 0.f ? 1.f - q : q);
}
__device__ inline float silu(float z) { return z * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504f * z)); }

__device__ inline float activate1(float z, uint32_t act) { return act == APOE_ACT_RELU ? relu(z) : act == APOE_ACT_GELU ? gelu(z) : act == APOE_ACT_SILU ? silu(z) : z; }

// Eight values under one decision, so that the roots of one do not wait for another's.
__device__ inline void activate8(float* z, uint32_t act) {
    if (act == APOE_ACT_RELU) {
#pragma unroll
        for (int k = 0; k < 8; k++) z[k] = relu(z[k]);
    } else if (act == APOE_ACT_GELU) {
#pragma unroll
        for (int k = 0; k < 8; k++) z[k] = gelu(z[k]);
    } else if (act == APOE_ACT_SILU) {
#pragma unroll
        for (int k = 0; k < 8; k++) z[k] = silu(z[k]);
    }
}

// v times the activation's slope at z.
__device__ inline void slope8(float* v, const float* z, uint32_t act) {
    if (act == APOE_ACT_RELU) {
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = z[k] > 0.f ? v[k] : 0.f; // whatever comes in where nothing went out: an infinity too
    } else if (act == APOE_ACT_GELU) {
#pragma unroll
        for (int k = 0; k < 8; k++) {
            float d;
            const float q = normal_tail(fabsf(z[k]), d);
            v[k] *= __builtin_fmaf(z[k], d, z[k] > 0.f ? 1.f - q : q);
        }
    } else if (act == APOE_ACT_SILU) { // o (1 + z (1 - o))
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const float e = __builtin_amdgcn_exp2f(-1.44269504f * z[k]), o = __builtin_amdgcn_rcpf(1.f + e), rest = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(1.44269504f * z[k]));
            v[k] *= o * __builtin_fmaf(z[k], rest, 1.f);
        }
    }
}

// Eight values of a row as numbers, `left` of them there. They begin at any value: the vector loads and stores ask for no more alignment than its type's.
template <typename T> __device__ inline void take8(float* v, const void* p, uint64_t at, uint32_t left) {
    const T* from = (const T*)p + at;
    if (left >= 8) {
        typedef T tv __attribute__((ext_vector_type(16 / sizeof(T))));
        typedef tv tu __attribute__((aligned(sizeof(T))));
        constexpr int E = 16 / sizeof(T);
#pragma unroll
        for (int c = 0; c < 8 / E; c++) {
            const tv x = *reinterpret_cast<const tu*>(from + c * E);
#pragma unroll
            for (int k = 0; k < E; k++) v[c * E + k] = (float)x[k];
        }
        return;
    }
#pragma unroll
    for (int k = 0; k < 8; k++) v[k] = (uint32_t)k < left ? (float)from[k] : 0.f;
}
template <typename T> __device__ inline void give8(void* p, uint64_t at, const float* v, uint32_t left) {
    T* to = (T*)p + at;
    if (left >= 8) {
        typedef T tv __attribute__((ext_vector_type(16 / sizeof(T))));
        typedef tv tu __attribute__((aligned(sizeof(T))));
        constexpr int E = 16 / sizeof(T);
#pragma unroll
        for (int c = 0; c < 8 / E; c++) {
            tv x;
#pragma unroll
            for (int k = 0; k < E; k++) x[k] = (T)v[c * E + k];
            *reinterpret_cast<tu*>(to + c * E) = x;
        }
        return;
    }
#pragma unroll
    for (int k = 0; k < 8; k++)
        if ((uint32_t)k < left) to[k] = (T)v[k];
}

// Eight sums of row i from column j on. T: the type of the results.
template <typename T> __device__ inline void finish8(const LinOut& o, uint32_t i, uint32_t j, float* v) {
    const uint32_t left = o.n - j;
    if (o.bias) {
        float b[8];
        take8<float>(b, o.bias, j, left);
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] += b[k];
    }
    if (o.pre) give8<T>(o.pre, i * o.pre_stride + j, v, left);
    activate8(v, o.act);
    if (o.residual) {
        float r[8];
        take8<T>(r, o.residual, i * o.residual_stride + j, left);
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] += r[k];
    }
    give8<T>(o.out, i * o.out_stride + j, v, left);
}

// One.
template <typename T> __device__ inline void finish1(const LinOut& o, uint32_t i, uint32_t j, float z) {
    if (o.bias) z += o.bias[j];
    if (o.pre) ((T*)o.pre)[i * o.pre_stride + j] = (T)z;
    z = activate1(z, o.act);
    if (o.residual) z += (float)((const T*)o.residual)[i * o.residual_stride + j];
    ((T*)o.out)[i * o.out_stride + j] = (T)z;
}

__device__ inline bool is_finite(float v) { return fabsf(v) < INFINITY; }

// Those of row i's sums v from column j on that are NaN, once more, one product after the other, until they are: a part that is zero makes NaN of the other side's infinity, floats' parts of
// an infinity leave NaN, and parts of either sign do where a product is beyond the largest float. (Infinities are right: the first part's, whose sign is the value's.) Float 4096 x 4096 x 1024 with an
// infinity in one row 0.4 ms, in every row 29, all NaN 0.7.
template <typename T> __device__ inline void make_sums_again(const LinTile& a, uint32_t i, uint32_t j, float* v) {
    uint32_t bad = 0;
#pragma unroll
    for (int c = 0; c < 8; c++) bad |= v[c] == v[c] || j + c >= a.o.n ? 0 : 1u << c;
    if (__builtin_expect(bad == 0, 1)) return;
    const char* pa = (const char*)a.a + (a.a_down ? i * sizeof(T) : (uint64_t)i * a.a_pitch);
    const char* pb = (const char*)a.b + (a.b_down ? j * sizeof(T) : (uint64_t)j * a.b_pitch);
    const uint64_t sa = a.a_down ? a.a_pitch : sizeof(T), sb = a.b_down ? a.b_pitch : sizeof(T), across = a.b_down ? sizeof(T) : a.b_pitch;
    const uint32_t last = a.o.n - 1 - j;
    float s[8] = {};
    for (uint32_t k0 = 0; k0 < a.k && bad; k0 += 16) {
        const uint32_t end = min(k0 + 16, a.k);
#pragma unroll 2
        for (uint32_t k = k0; k < end; k++) {
            float x = (float)*(const T*)(pa + k * sa);
            if (a.second) x = __builtin_fmaf((float)*(const T*)(pa + k * sa + a.second), Two<T>::DOWN, x) * (1.f / Two<T>::HALF);
#pragma unroll
            for (uint32_t c = 0; c < 8; c++) s[c] = __builtin_fmaf(x, (float)*(const T*)(pb + k * sb + min(c, last) * across), s[c]);
        }
#pragma unroll
        for (int c = 0; c < 8; c++) {
            if (s[c] != s[c]) bad &= ~(1u << c); // as it was
        }
    }
#pragma unroll
    for (int c = 0; c < 8; c++) v[c] = bad >> c & 1 ? s[c] : v[c];
}

// (ADD: groups of waves hold parts of every sum; otherwise each group has whole ones of its share of the blocks.)
// What the waves hold goes out: one block of 32 rows a wave at a time through LDS, then a thread has eight values of a row. Waits between are for LDS alone: the
// stores of the block before are on their way meanwhile.
template <typename T, int MT, int NT, int WM, int WN, int KG, int BYTES, bool ADD = false, bool TWO = false>
__device__ inline void tile_out(const LinTile& a, f32x16 (&acc)[MT][NT], char* lds, uint32_t row, uint32_t col, uint32_t cut, int kg, int wm, int wn, int lane) {
    constexpr int NW = WM * WN * KG, BN = WN * NT * 32, PITCH = BN + 4, ROWS = WM * 32, ITEMS = (ROWS * BN / 8 + 64 * NW - 1) / (64 * NW);
    static_assert(ROWS * PITCH * 4 <= BYTES, "the sums fit the stages");
    const uint32_t m = a.o.m, n = a.o.n;
    float* sum = reinterpret_cast<float*>(lds);
    const int half = lane >> 5;
#pragma unroll
    for (int i = 0; i < MT; i++) {
        const auto each = [&](auto&& use) {
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int k = 0; k < 16; k++) use(sum[(wm * 32 + result_row(k, half)) * PITCH + (wn * NT + t) * 32 + (lane & 31)], acc[i][t][k]);
        };
        if constexpr (ADD) {
#pragma unroll
            for (int g = KG - 1; g > 0; g--) {
                if (kg == g) each([&](float& at, float v) { at = g == KG - 1 ? v : at + v; });
                tile_wait<63>();
            }
            if (kg == 0) each([](float& at, float v) { at += v; });
        } else if (KG == 1 || i / (MT / KG) == kg) {
            each([](float& at, float v) { at = v; });
        }
        tile_wait<63>();
#pragma unroll 1
        for (int item = 0; item < ITEMS; item++) {
            const uint32_t at = item * 64 * NW + threadIdx.x, r = at / (BN / 8), c = at % (BN / 8) * 8;
            const uint32_t gi = row + (r / 32 * MT + i) * 32 + r % 32, gj = col + c;
            if (r >= ROWS || gi >= m || gj >= n) continue;
            const f32x4 v0 = *reinterpret_cast<const f32x4*>(sum + r * PITCH + c), v1 = *reinterpret_cast<const f32x4*>(sum + r * PITCH + c + 4);
            if (a.cuts > 1) {
                float* to = a.part + ((uint64_t)cut * m + gi) * a.np + gj;
                *reinterpret_cast<f32x4*>(to) = v0;
                *reinterpret_cast<f32x4*>(to + 4) = v1;
            } else {
                float v[8] = {v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
                if constexpr (TWO || sizeof(T) == 4) make_sums_again<T>(a, gi, gj, v);
                finish8<T>(a.o, gi, gj, v);
            }
        }
        if (i + 1 < MT) tile_wait<63>();
    }
}

// Columns' sums over the strips: THREADS / 16 columns a workgroup, sixteen threads each, the same order whatever THREADS is.
template <int THREADS> __device__ inline void bias_sums(const LinBias& a, uint32_t group, float* lds) {
    constexpr uint32_t WIDE = THREADS / 16;
    const uint32_t c = threadIdx.x % WIDE, l = threadIdx.x / WIDE, d = group * WIDE + c;
    float s = 0.f;
    if (d < a.cols)
        for (uint32_t b0 = l; b0 < a.strips; b0 += 128) { // eight loads at once, beyond the last strip that one again
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; u++) v[u] = a.part[(uint64_t)min(b0 + u * 16, a.strips - 1) * a.cols + d];
#pragma unroll
            for (int u = 0; u < 8; u++) s += b0 + u * 16 < a.strips ? v[u] : 0.f;
        }
    float* q = lds + l * (WIDE + 1) + c;
    *q = s;
    for (uint32_t k = 8; k; k >>= 1) {
        __syncthreads();
        if (l < k) *q += q[k * (WIDE + 1)];
    }
    if (l == 0 && d < a.cols) a.out[d] = *q;
}

// 16-bit matrices. ACOL, BCOL: the inner dimension goes down the rows. TWO: a has two parts; all of the second's products are added up in front of the first's.
template <typename T, bool ACOL, bool BCOL, bool TWO, int MT, int NT, int WM, int WN, int KG, int SF, int ST>
__device__ inline void one_tile(const LinTile& a, uint32_t block, char* lds) {
    constexpr int NW = WM * WN * KG, FS = SF / KG, BM = WM * MT * 32, BN = WN * NT * 32;
    using ATile = std::conditional_t<ACOL, ColTile<T, BM, SF, NW, ORDER_ROWS>, RowTile<T, BM, SF, NW>>;
    using BTile = std::conditional_t<BCOL, ColTile<T, BN, SF, NW, ORDER_ROWS>, RowTile<T, BN, SF, NW>>;
    constexpr int STAGE = ATile::BYTES + BTile::BYTES, PER = ATile::LOADS + BTile::LOADS, KE = ATile::KE;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), kg = wave / (WM * WN), wm = wave % (WM * WN) / WN, wn = wave % WN;
    const uint32_t m = a.o.m, n = a.o.n;
    if (block >= a.groups) {
        bias_sums<64 * NW>(a.bias, block - a.groups, reinterpret_cast<float*>(lds));
        return;
    }
    const uint32_t id = xcd_run(block, a.groups), tile = id / a.cuts, cut = id % a.cuts;
    // an XCD's run of tiles is about as high as it is wide: it reads the fewest rows of both sides into its L2
    const uint32_t band = tile / (a.band * a.nt), in_band = tile % (a.band * a.nt), high = min(a.band, a.mt - band * a.band);
    const uint32_t row = (band * a.band + in_band % high) * BM, col = in_band / high * BN;
    const uint32_t s0 = cut * a.cut_stages, stages = min(a.cut_stages, (a.k + KE - 1) / KE - s0);
    const int mrows = (int)min((uint32_t)BM, m - row), ncols = (int)min((uint32_t)BN, n - col);
    ATile ta;
    BTile tb;
    const char *pa = (const char*)a.a, *pb = (const char*)a.b;
    if constexpr (TWO) pa += a.second;
    if constexpr (ACOL) ta.init((const T*)(pa + (uint64_t)s0 * KE * a.a_pitch) + row, a.a_pitch, (mrows + 7) / 8 * 8, wave, lane);
    else ta.init((const T*)(pa + (uint64_t)row * a.a_pitch) + (uint64_t)s0 * KE, a.a_pitch, mrows, wave, lane);
    if constexpr (BCOL) tb.init((const T*)(pb + (uint64_t)s0 * KE * a.b_pitch) + col, a.b_pitch, (ncols + 7) / 8 * 8, wave, lane);
    else tb.init((const T*)(pb + (uint64_t)col * a.b_pitch) + (uint64_t)s0 * KE, a.b_pitch, ncols, wave, lane);
    const uint32_t base = lds_address(lds);
    const int inner = (int)min(stages * KE, a.k - s0 * KE); // a row's values are followed by zeros up to a multiple of eight
    int left = inner;
    uint32_t into = 0;
    [[maybe_unused]] uint64_t first_a = 0, first_b = 0;
    if constexpr (TWO) {
        first_a = uniform64(ta.base - a.second);
        first_b = tb.base;
    }
    [[maybe_unused]] int more = 1;
    auto issue = [&]() {
        const auto one = [&](auto& t, uint32_t at, auto down) {
            if constexpr (decltype(down)::value) {
                using Mask = typename std::remove_reference_t<decltype(t)>::Mask;
                t.load(at, left >= KE ? t.ALL : left > 0 ? (Mask)(((Mask)1 << left) - 1) : (Mask)0, wave, lane);
            } else {
                t.load(at, (left + 7) / 8 * 16, wave);
            }
            t.next();
        };
        one(ta, base + into, std::integral_constant<bool, ACOL>{});
        one(tb, base + into + ATile::BYTES, std::integral_constant<bool, BCOL>{});
        left -= KE;
        if constexpr (TWO) { // (selections: a branch would end the block whose order is given below)
            const bool turn = left < more; // more: 1, then a number that left never is below
            ta.base = turn ? first_a : ta.base;
            tb.base = turn ? first_b : tb.base;
            left = turn ? inner : left;
            more = turn ? INT32_MIN : more;
        }
        into = into + STAGE == ST * STAGE ? 0 : into + STAGE;
    };
#pragma unroll
    for (int s = 0; s < ST - 1; s++) issue();
    f32x16 acc[MT][NT] = {};
    uint32_t from = 0;
    const auto scale = [&](float by) {
        if constexpr (Two<T>::HALF != 1.f)
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int t = 0; t < NT; t++) acc[i][t] *= by;
    };
#pragma unroll 1
    for (int part = 0; part < (TWO ? 2 : 1); part++) {
        if (part) scale(Two<T>::DOWN);
        for (uint32_t s = 0; s < stages; s++) {
            tile_wait<(ST - 2) * PER>();
            const char* A = lds + from;
            const char* B = A + ATile::BYTES;
            i32x4 x[2][MT], y[2][NT];
            auto read = [&](int f) {
#pragma unroll
                for (int i = 0; i < MT; i++) x[f & 1][i] = ATile::read(A, wm * MT + i, kg * FS + f, lane);
#pragma unroll
                for (int t = 0; t < NT; t++) y[f & 1][t] = BTile::read(B, wn * NT + t, kg * FS + f, lane);
            };
            read(0);
            issue();
#pragma unroll
            for (int f = 0; f < FS; f++) {
                if (f + 1 < FS) read(f + 1);
#pragma unroll
                for (int i = 0; i < MT; i++)
#pragma unroll
                    for (int t = 0; t < NT; t++) acc[i][t] = mfma_step<T>(x[f & 1][i], y[f & 1][t], acc[i][t]);
            }
            interleave<(ACOL ? 2 : 1) * MT + (BCOL ? 2 : 1) * NT, MT * NT, FS>();
            from = from + STAGE == ST * STAGE ? 0 : from + STAGE;
        }
    }
    if constexpr (TWO) scale(1.f / Two<T>::HALF);
    tile_wait<0>();
    if constexpr (KG == 2) {
        static_assert(BM * BN * 4 <= ST * STAGE, "the sums fit the stages");
        exchange_halves<MT, NT, WM * WN>(acc, lds, kg, wave % (WM * WN), lane);
        __syncthreads();
    }
    tile_out<T, MT, NT, WM, WN, KG, ST * STAGE, false, TWO>(a, acc, lds, row, col, cut, kg, wm, wn, lane);
}

template <typename T, bool ACOL, bool BCOL, bool TWO, int MT, int NT, int WM, int WN, int KG, int SF, int ST> __global__ __launch_bounds__(64 * WM * WN * KG, 2) void linear_tile(LinTile a) {
    __shared__ __align__(1024) char lds[ST * (WM * MT + WN * NT) * 32 * SF * 32];
    one_tile<T, ACOL, BCOL, TWO, MT, NT, WM, WN, KG, SF, ST>(a, blockIdx.x, lds);
}

// gx = gz w and gw = gz^T x in one launch (gx may have no workgroups): neither waits for the other's last tiles.
template <typename T, bool TWO, int MT, int NT, int WM, int WN, int KG, int SF, int ST> __global__ __launch_bounds__(64 * WM * WN * KG, 2) void linear_grads(LinTile x, LinTile w) {
    __shared__ __align__(1024) char lds[ST * (WM * MT + WN * NT) * 32 * SF * 32];
    if (blockIdx.x < x.groups) one_tile<T, false, true, TWO, MT, NT, WM, WN, KG, SF, ST>(x, blockIdx.x, lds);
    else one_tile<T, true, true, TWO, MT, NT, WM, WN, KG, SF, ST>(w, blockIdx.x - x.groups, lds);
}

// ---- float matrices ----

// Eight floats as three parts of eight bits that add up to them exactly: the leading bits as they are, then what each part leaves, rounded to the next.
struct Parts {
    bf16x8 p[3];
};
__device__ inline Parts split8(f32x4 lo, f32x4 hi) {
    Parts s;
    i32x4 top;
    float rest[8];
#pragma unroll
    for (int k = 0; k < 8; k++) {
        const float v = k < 4 ? lo[k] : hi[k - 4];
        rest[k] = v - __uint_as_float(__float_as_uint(v) & 0xffff0000u);
    }
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const uint32_t a = __float_as_uint(k < 2 ? lo[2 * k] : hi[2 * k - 4]), b = __float_as_uint(k < 2 ? lo[2 * k + 1] : hi[2 * k - 3]);
        top[k] = (int)__builtin_amdgcn_perm(b, a, 0x07060302u); // the upper halves
    }
    s.p[0] = __builtin_bit_cast(bf16x8, top);
#pragma unroll
    for (int k = 0; k < 8; k++) s.p[1][k] = (__bf16)rest[k];
#pragma unroll
    for (int k = 0; k < 8; k++) s.p[2][k] = (__bf16)(rest[k] - (float)s.p[1][k]);
    return s;
}

// What a lane gets of sixteen inner indices is 4 h + 0..3 and 8 + 4 h + 0..3 for its half h: the same on both sides. Rows begin at multiples of 16 bytes, and a row's
// values are followed by zeros up to one.
template <int ROWS, int NW, int KE> struct RowTile32 { // inner index along the rows; a row's 16-byte pieces lie at places that its number turns
    static constexpr int BYTES = ROWS * KE * 4, LOADS = BYTES / (1024 * NW);
    static_assert(BYTES % (1024 * NW) == 0, "whole loads");
    uint32_t offset[LOADS], at[LOADS]; // at: byte in a row's stage
    uint64_t base;
    __device__ static int turn(int row) { return KE == 64 ? row & 15 : (row >> 1) & 7; }
    __device__ void init(const float* row0, uint32_t pitch_bytes, int rows, int wave, int lane) {
        base = uniform64((uint64_t)row0);
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            const int l = ((i * NW + wave) * 64 + lane) * 4, row = l / KE, k = l % KE;
            at[i] = (uint32_t)(((k / 4) ^ turn(row)) * 16);
            offset[i] = row < rows ? (uint32_t)row * pitch_bytes + at[i] : TILE_MASKED;
        }
    }
    __device__ void load(uint32_t lds, int left, int wave, int) const { // left: inner indices from here on
        const i32x4 buffer = buffer_of(base);
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            const uint32_t from = left >= KE || (int)at[i] < left * 4 ? offset[i] : TILE_MASKED;
            load_to_lds16(buffer, from, lds + (i * NW + wave) * 1024);
        }
    }
    __device__ void next() { base += KE * 4; }
    __device__ static f32x4 read(const char* lds, int rb, int e, int lane) { // eight inner indices, four a half
        const int row = lane & 31;
        return *reinterpret_cast<const f32x4*>(lds + (rb * 32 + row) * KE * 4 + (((2 * e + (lane >> 5)) ^ turn(row)) * 16));
    }
};
// The same for rows that begin at any value: a float a load. What a lane asks for in load i follows from load 0.
template <int ROWS, int NW, int KE> struct RowTile32One : RowTile32<ROWS, NW, KE> {
    using Whole = RowTile32<ROWS, NW, KE>;
    static constexpr int LOADS = Whole::BYTES / (256 * NW), STEP = 64 * NW / KE; // STEP: rows from one load to the next
    static_assert(NW == 8 && (KE == 32 || KE == 64), "a row's turn is that of load 0, with 64 inner indices turned by 8 more in every second load");
    uint32_t first, place, step; // bytes: of the lane's row, in a row's stage, from one load to the next
    int rows;                    // that are there, from load 0's on
    __device__ void init(const float* row0, uint32_t pitch_bytes, int count, int wave, int lane) {
        this->base = uniform64((uint64_t)row0);
        const int l = wave * 64 + lane, row = l / KE, k = l % KE;
        place = (uint32_t)(((k / 4) ^ Whole::turn(row)) * 16 + k % 4 * 4);
        first = (uint32_t)row * pitch_bytes;
        step = STEP * pitch_bytes;
        rows = count - row;
    }
    __device__ void load(uint32_t lds, int left, int wave, int) const {
        const i32x4 buffer = buffer_of(this->base);
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            const uint32_t to = place ^ (KE == 64 && i & 1 ? 8 * 16 : 0);
            load_to_lds4(buffer, i * STEP < rows && (int)to < left * 4 ? first + i * step + to : TILE_MASKED, lds + (i * NW + wave) * 256);
        }
    }
};
template <int COLS, int NW, int KE> struct ColTile32 { // inner index down the rows
    static constexpr int BYTES = COLS * KE * 4, LOADS = BYTES / (1024 * NW);
    static_assert(BYTES % (1024 * NW) == 0, "whole loads");
    uint32_t offset[LOADS];
    uint64_t base, step;
    __device__ static int row_of(int i, int wave, int lane) { return ((i * NW + wave) * 64 + lane) * 4 / COLS; }
    __device__ void init(const float* at, uint32_t pitch_bytes, int cols, int wave, int lane) {
        base = uniform64((uint64_t)at);
        step = (uint64_t)KE * pitch_bytes;
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            const int col = ((i * NW + wave) * 64 + lane) * 4 % COLS;
            offset[i] = col < cols ? (uint32_t)row_of(i, wave, lane) * pitch_bytes + col * 4 : TILE_MASKED;
        }
    }
    __device__ void load(uint32_t lds, int left, int wave, int lane) const {
        const i32x4 buffer = buffer_of(base);
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            const uint32_t from = left >= KE || row_of(i, wave, lane) < left ? offset[i] : TILE_MASKED;
            load_to_lds16(buffer, from, lds + (i * NW + wave) * 1024);
        }
    }
    __device__ void next() { base += step; }
    __device__ static f32x4 read(const char* lds, int cb, int e, int lane) {
        const float* p = reinterpret_cast<const float*>(lds) + (8 * e + 4 * (lane >> 5)) * COLS + cb * 32 + (lane & 31);
        return f32x4{p[0], p[COLS], p[2 * COLS], p[3 * COLS]};
    }
};

// ONE: rows that begin at any value, on both sides.
template <bool ACOL, bool BCOL, bool ONE, int MT, int NT, int WM, int WN, int KG, int KE, int ST>
__device__ inline void one_tile32(const LinTile& a, uint32_t block, char* lds) {
    constexpr int NW = WM * WN * KG, BM = WM * MT * 32, BN = WN * NT * 32, FS = KE / 16 / KG;
    using ATile = std::conditional_t<ACOL, ColTile32<BM, NW, KE>, std::conditional_t<ONE, RowTile32One<BM, NW, KE>, RowTile32<BM, NW, KE>>>;
    using BTile = std::conditional_t<BCOL, ColTile32<BN, NW, KE>, std::conditional_t<ONE, RowTile32One<BN, NW, KE>, RowTile32<BN, NW, KE>>>;
    constexpr int STAGE = ATile::BYTES + BTile::BYTES, PER = ATile::LOADS + BTile::LOADS;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), kg = wave / (WM * WN), wm = wave % (WM * WN) / WN, wn = wave % WN;
    const uint32_t m = a.o.m, n = a.o.n;
    if (block >= a.groups) {
        bias_sums<64 * NW>(a.bias, block - a.groups, reinterpret_cast<float*>(lds));
        return;
    }
    const uint32_t id = xcd_run(block, a.groups), tile = id / a.cuts, cut = id % a.cuts;
    const uint32_t band = tile / (a.band * a.nt), in_band = tile % (a.band * a.nt), high = min(a.band, a.mt - band * a.band);
    const uint32_t row = (band * a.band + in_band % high) * BM, col = in_band / high * BN;
    const uint32_t s0 = cut * a.cut_stages, stages = min(a.cut_stages, (a.k + KE - 1) / KE - s0);
    const int mrows = (int)min((uint32_t)BM, m - row), ncols = (int)min((uint32_t)BN, n - col);
    ATile ta;
    BTile tb;
    if constexpr (ACOL) ta.init((const float*)((const char*)a.a + (uint64_t)s0 * KE * a.a_pitch) + row, a.a_pitch, (mrows + 3) / 4 * 4, wave, lane);
    else ta.init((const float*)((const char*)a.a + (uint64_t)row * a.a_pitch) + (uint64_t)s0 * KE, a.a_pitch, mrows, wave, lane);
    if constexpr (BCOL) tb.init((const float*)((const char*)a.b + (uint64_t)s0 * KE * a.b_pitch) + col, a.b_pitch, (ncols + 3) / 4 * 4, wave, lane);
    else tb.init((const float*)((const char*)a.b + (uint64_t)col * a.b_pitch) + (uint64_t)s0 * KE, a.b_pitch, ncols, wave, lane);
    const uint32_t base = lds_address(lds);
    int left = (int)min(stages * KE, a.k - s0 * KE);
    uint32_t into = 0;
    auto issue = [&]() {
        ta.load(base + into, left, wave, lane);
        tb.load(base + into + ATile::BYTES, left, wave, lane);
        ta.next();
        tb.next();
        left -= KE;
        into = into + STAGE == ST * STAGE ? 0 : into + STAGE;
    };
#pragma unroll
    for (int s = 0; s < ST - 1; s++) issue();
    f32x16 acc[MT][NT] = {};
    uint32_t from = 0;
    for (uint32_t s = 0; s < stages; s++) {
        tile_wait<(ST - 2) * PER>();
        const char* A = lds + from;
        const char* B = A + ATile::BYTES;
        f32x4 x[FS][MT][2], y[FS][NT][2];
#pragma unroll
        for (int f = 0; f < FS; f++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
#pragma unroll
                for (int i = 0; i < MT; i++) x[f][i][e] = ATile::read(A, wm * MT + i, 2 * (kg * FS + f) + e, lane);
#pragma unroll
                for (int t = 0; t < NT; t++) y[f][t][e] = BTile::read(B, wn * NT + t, 2 * (kg * FS + f) + e, lane);
            }
        issue();
#pragma unroll
        for (int f = 0; f < FS; f++) {
            Parts sx[MT], sy[NT];
#pragma unroll
            for (int i = 0; i < MT; i++) sx[i] = split8(x[f][i][0], x[f][i][1]);
#pragma unroll
            for (int t = 0; t < NT; t++) sy[t] = split8(y[f][t][0], y[f][t][1]);
#pragma unroll
            for (int total = 2; total >= 0; total--) // the smaller products first
#pragma unroll
                for (int p = 0; p <= total; p++)
#pragma unroll
                    for (int i = 0; i < MT; i++)
#pragma unroll
                        for (int t = 0; t < NT; t++) acc[i][t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(sx[i].p[p], sy[t].p[total - p], acc[i][t], 0, 0, 0);
        }
        from = from + STAGE == ST * STAGE ? 0 : from + STAGE;
    }
    tile_wait<0>();
    tile_out<float, MT, NT, WM, WN, KG, ST * STAGE, (KG > 1)>(a, acc, lds, row, col, cut, kg, wm, wn, lane);
}

template <bool ACOL, bool BCOL, bool ONE, int MT, int NT, int WM, int WN, int KG, int KE, int ST> __global__ __launch_bounds__(64 * WM * WN * KG, 2) void linear_tile32(LinTile a) {
    __shared__ __align__(1024) char lds[ST * (WM * MT + WN * NT) * 32 * KE * 4];
    one_tile32<ACOL, BCOL, ONE, MT, NT, WM, WN, KG, KE, ST>(a, blockIdx.x, lds);
}

template <int MT, int NT, int WM, int WN, int KG, int KE, int ST> __global__ __launch_bounds__(64 * WM * WN * KG, 2) void linear_grads32(LinTile x, LinTile w) {
    __shared__ __align__(1024) char lds[ST * (WM * MT + WN * NT) * 32 * KE * 4];
    if (blockIdx.x < x.groups) one_tile32<false, true, false, MT, NT, WM, WN, KG, KE, ST>(x, blockIdx.x, lds);
    else one_tile32<true, true, false, MT, NT, WM, WN, KG, KE, ST>(w, blockIdx.x - x.groups, lds);
}

// The cuts' sums, eight columns a thread. PARTS: of parts.
template <typename T, bool PARTS> __global__ __launch_bounds__(256) void linear_join(LinTile a) {
    const uint32_t per = a.np / 8;
    const uint64_t total = (uint64_t)a.o.m * per;
    for (uint64_t at = (uint64_t)blockIdx.x * 256 + threadIdx.x; at < total; at += (uint64_t)gridDim.x * 256) {
        const uint32_t i = (uint32_t)(at / per), j = (uint32_t)(at % per) * 8;
        f32x4 s0 = {}, s1 = {};
#pragma unroll 4
        for (uint32_t c = 0; c < a.cuts; c++) {
            const float* from = a.part + ((uint64_t)c * a.o.m + i) * a.np + j;
            s0 += *reinterpret_cast<const f32x4*>(from);
            s1 += *reinterpret_cast<const f32x4*>(from + 4);
        }
        float v[8] = {s0[0], s0[1], s0[2], s0[3], s1[0], s1[1], s1[2], s1[3]};
        if constexpr (PARTS) make_sums_again<T>(a, i, j, v);
        finish8<T>(a.o, i, j, v);
    }
}

// ---- up to 16 rows ----

struct LinFew {
    const void *x, *w;
    uint64_t x_stride, w_stride;
    uint32_t k;
    LinOut o;
};

// Bound by the one reading of w (and for small layers by its latency): a workgroup has 16 of w's rows, its NW waves share the inner side, 128 indices at a time, all of
// whose loads are on their way at once; x comes from the L2. 16 x 16 matrix instructions, float matrices on the float ones. The waves' sums meet in LDS, one
// result a thread. 16 x 1024 -> 4096 fp16: 4.5 us (64 x 64 tiles in two cuts and their sum 9).
template <typename T, int NW> __global__ __launch_bounds__(64 * NW) void linear_few(LinFew a) {
    constexpr int E = 16 / sizeof(T), STEP = 4 * E, U = 128 / STEP; // values a lane loads; inner indices of a load; loads of a turn
    typedef T tv __attribute__((ext_vector_type(E)));
    __shared__ float sums[NW][256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4, r = lane & 15;
    const uint32_t m = a.o.m, n = a.o.n, col = blockIdx.x * 16;
    const T* xr = (const T*)a.x + (uint64_t)min((uint32_t)r, m - 1) * a.x_stride; // rows beyond the end: the last one again, whose results go nowhere
    const T* wr = (const T*)a.w + (uint64_t)min(col + r, n - 1) * a.w_stride;
    f32x4 acc = {};
    for (uint32_t k0 = wave * 128; k0 < a.k; k0 += NW * 128) {
        tv xv[U], wv[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t k = k0 + u * STEP + q * E;
            xv[u] = k < a.k ? *reinterpret_cast<const tv*>(xr + k) : tv{};
            wv[u] = k < a.k ? *reinterpret_cast<const tv*>(wr + k) : tv{};
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if constexpr (std::is_same_v<T, float>) {
#pragma unroll
                for (int j = 0; j < 4; j++) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(xv[u][j], wv[u][j], acc, 0, 0, 0);
            } else if constexpr (std::is_same_v<T, _Float16>) {
                acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(xv[u], wv[u], acc, 0, 0, 0);
            } else {
                acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xv[u], wv[u], acc, 0, 0, 0);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) sums[wave][(4 * q + i) * 16 + r] = acc[i];
    __syncthreads();
    const uint32_t i = threadIdx.x / 16, j = col + threadIdx.x % 16;
    if (i >= m || j >= n) return;
    float z = 0.f;
#pragma unroll
    for (int w = 0; w < NW; w++) z += sums[w][threadIdx.x];
    finish1<T>(a.o, i, j, z);
}

// ---- operands in the products' form, gz, and the columns' sums ----

struct LinPack {
    const void *src, *pre;  // pre: multiply by the activation's slope there
    uint64_t src_stride, pre_stride;
    void *dst, *second;     // [rows][pitch], zeros behind a row's end; NULL: sums alone. second: the second part, or NULL
    uint32_t rows, cols, pitch, act;
    float* part;            // [strips][cols] sums of columns, or NULL
    uint32_t across, strips, first; // workgroups: 512 columns each, strips of rows; the first one's number
};
struct LinPacks {
    LinPack one[3];
    uint32_t count, groups;
};

// A thread has eight columns and every fourth row of a strip; one launch for all matrices that a call needs in another form. (TWO: one of them in two parts, which takes registers for a wave
// less a SIMD; without it the rest goes 4 % slower.)
template <typename T, bool TWO> __global__ __launch_bounds__(256) void linear_pack(LinPacks all) {
    __shared__ float sums[4][512];
    const uint32_t which = all.count > 2 && blockIdx.x >= all.one[2].first ? 2 : all.count > 1 && blockIdx.x >= all.one[1].first ? 1 : 0;
    const LinPack& a = all.one[which];
    const uint32_t group = blockIdx.x - a.first, strip = group / a.across, bx = group % a.across;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = bx * 512 + lane * 8;
    float s[8] = {};
    if (j < a.pitch) {
        const uint32_t left = a.cols - j;
#pragma unroll 2
        for (uint64_t i = (uint64_t)strip * 4 + wave; i < a.rows; i += a.strips * 4ull) {
            float v[8];
            take8<T>(v, a.src, i * a.src_stride + j, left);
            if (a.pre) {
                float z[8];
                take8<T>(z, a.pre, i * a.pre_stride + j, left);
                slope8(v, z, a.act);
            }
#pragma unroll
            for (int k = 0; k < 8; k++) s[k] += v[k];
            if (!a.dst) continue;
            if constexpr (TWO) {
                if (a.second) {
                    float rest[8];
#pragma unroll
                    for (int k = 0; k < 8; k++) {
                        v[k] *= Two<T>::HALF;
                        const float r = v[k] - (float)(T)v[k];
                        rest[k] = is_finite(r) ? r * (1.f / Two<T>::DOWN) : 0.f; // (an infinity is all in its first part)
                    }
                    give8<T>(a.second, i * a.pitch + j, rest, 8);
                }
            }
            give8<T>(a.dst, i * a.pitch + j, v, 8);
        }
    }
    if (!a.part) return;
#pragma unroll
    for (int k = 0; k < 8; k++) sums[wave][lane * 8 + k] = s[k];
    __syncthreads();
    for (uint32_t c = threadIdx.x; c < 512; c += 256)
        if (bx * 512 + c < a.cols) a.part[(uint64_t)strip * a.cols + bx * 512 + c] = (sums[0][c] + sums[1][c]) + (sums[2][c] + sums[3][c]);
}

__global__ __launch_bounds__(512) void linear_bias(LinBias a) {
    __shared__ float lds[16 * 33];
    bias_sums<512>(a, blockIdx.x, lds);
}

// ---- host ----

struct LinOperand { // as the products take it
    const void* p;
    uint32_t pitch; // bytes
};

constexpr uint32_t LIN_STRIPS = 256; // of rows under one partial sum of the bias' gradient, at most

// Whether a matrix can be taken where it lies: offsets of 256 rows in 31 bits, and 16 bytes a load.
template <typename T> static bool near_rows(uint64_t stride) { return stride * sizeof(T) <= (1u << 22); }
template <typename T> static bool as_it_is(const void* p, uint64_t stride, uint32_t cols) {
    constexpr uint32_t E = 16 / sizeof(T);
    return cols % E == 0 && stride % E == 0 && near_rows<T>(stride) && ((uintptr_t)p & 15) == 0;
}

struct LinPlan {
    uint64_t bytes = 0;
    uint64_t take(uint64_t b) {
        const uint64_t at = bytes;
        bytes += (b + 1023) / 1024 * 1024;
        return at;
    }
};

static uint32_t pitch_of(uint32_t cols) { return (cols + 7) / 8 * 8; }

template <typename T> static uint64_t packed_bytes(uint64_t rows, uint32_t cols) { return rows * pitch_of(cols) * sizeof(T); }

template <typename T>
static LinPack& add_pack(apoe_ctx* ctx, LinPacks& all, const void* src, uint64_t stride, uint32_t rows, uint32_t cols, void* dst) {
    LinPack& a = all.one[all.count++];
    a = LinPack{src, nullptr, stride, 0, dst, nullptr, rows, cols, pitch_of(cols), 0, nullptr, 0, 0, 0};
    a.across = (a.pitch + 511) / 512;
    a.strips = std::max(1u, std::min({(rows + 3) / 4, LIN_STRIPS, std::max(1u, (uint32_t)ctx->num_cus * 8 / a.across)}));
    return a;
}

template <typename T> static void pack(apoe_ctx* ctx, LinPacks& all) {
    for (uint32_t i = 0; i < all.count; i++) {
        all.one[i].first = all.groups;
        all.groups += all.one[i].across * all.one[i].strips;
    }
    if (!all.groups) return;
    if constexpr (sizeof(T) == 2) {
        if (all.one[0].second) { // gz is the first
            linear_pack<T, true><<<all.groups, 256, 0, ctx->stream>>>(all);
            return;
        }
    }
    linear_pack<T, false><<<all.groups, 256, 0, ctx->stream>>>(all);
}

struct LinShape {
    uint32_t bm, bn, kind, cuts, cut_stages;
    float us;
};

// Tiles and cuts, by what a product of each kind takes (us, fitted to fp16 and bf16 products of 256 to 8192 a side: a fixed part and one for each
// inner index, for every round of tiles over the CUs; `two`: pairs of workgroups share a CU, and a CU with one alone takes `alone`). Where few large tiles
// would leave CUs idle, smaller ones or parts of the inner side win, for which a launch adds the parts up:
//   256 x 256 8192 x 4096 x 1024 74 (256 x 128: 89); 256 x 128 8192 x 1024 x 4096 69 (256 x 256 in two cuts 84, 128 x 128 76); 128 x 128 with two groups
//   of waves 4096 x 1024 x 8192 75 (one group, in two cuts 82, 256 x 256 in four 82); 64 x 64 2048 x 1024 x 1024 9.4 (128 x 128 13), 512 x 512 x 4096
//   17.5, in four cuts 12.
struct LinKind {
    uint32_t bm, bn, ke;
    bool two;
    float fixed, inner, alone_fixed, alone_inner;
};
constexpr LinKind LIN_KINDS[] = {{256, 256, 64, false, 9.f, .0243f, 0.f, 0.f}, {256, 128, 64, false, 6.5f, .0142f, 0.f, 0.f}, {128, 128, 64, true, 5.4f, .0165f, 2.5f, .0103f},
                                 {128, 128, 64, false, 3.f, .0082f, 0.f, 0.f}, {64, 64, 64, true, 1.f, .0055f, 1.f, .0033f}};
constexpr LinKind LIN_KINDS_FLOAT[] = {{256, 256, 32, false, 12.f, .157f, 0.f, 0.f}, {128, 128, 32, false, 6.5f, .044f, 0.f, 0.f}, {64, 64, 64, false, 2.f, .0155f, 0.f, 0.f}};

template <typename T> static LinShape choose(apoe_ctx* ctx, uint32_t m, uint32_t n, uint32_t k, uint32_t parts = 1) {
    const uint64_t cus = (uint64_t)ctx->num_cus;
    LinShape best{};
    float least = INFINITY;
    const auto look = [&](const LinKind& kind, uint32_t number) {
        const uint64_t tiles = (uint64_t)((m + kind.bm - 1) / kind.bm) * ((n + kind.bn - 1) / kind.bn);
        const uint32_t stages = (k + kind.ke - 1) / kind.ke;
        if (number && tiles > (1u << 22)) return; // more than a launch takes
        for (uint32_t cuts = 1; cuts <= 16 && (cuts == 1 || (stages / cuts >= 4 && tiles * cuts <= 2 * cus)); cuts++) {
            const uint32_t each = std::max(1u, (stages + cuts - 1) / cuts);
            const uint64_t groups = tiles * cuts, at_once = kind.two ? 2 * cus : cus;
            const bool alone = kind.two && groups <= cus;
            const float inner = (float)(each * kind.ke * parts);
            float t = 3.f + (float)((groups + at_once - 1) / at_once) * (alone ? kind.alone_fixed + kind.alone_inner * inner : kind.fixed + kind.inner * inner);
            if (cuts > 1) t += 3.f + (float)(cuts + 1) * (float)m * (float)n * 1e-6f; // 4 bytes at 4 TB/s
            if (t < least) {
                least = t;
                best = LinShape{kind.bm, kind.bn, number, std::max(1u, (stages + each - 1) / each), each, t};
            }
        }
    };
    uint32_t number = 0;
    if constexpr (sizeof(T) == 2) {
        for (const LinKind& kind : LIN_KINDS) look(kind, number++);
    } else {
        for (const LinKind& kind : LIN_KINDS_FLOAT) look(kind, number++);
    }
    return best;
}

static uint64_t cut_bytes(const LinShape& s, uint32_t m, uint32_t n) { return s.cuts > 1 ? (uint64_t)s.cuts * m * pitch_of(n) * 4 : 0; }

static LinTile tiles_of(const LinShape& s, LinOperand a, LinOperand b, uint32_t k, float* part, const LinOut& o, const LinBias& bias = {}, uint64_t second = 0, bool a_down = false,
                        bool b_down = false) {
    const uint32_t mt = (o.m + s.bm - 1) / s.bm, nt = (o.n + s.bn - 1) / s.bn;
    uint32_t band = 1; // a power of two, so that runs end where bands do (8192 x 8192 x 4096: 444 us, row by row 482; 8192 x 1024 x 4096 67, 75)
    while (band * 2 <= mt && (uint64_t)band * band * 32 <= (uint64_t)mt * nt) band *= 2;
    return LinTile{a.p, b.p, a.pitch, b.pitch, k, mt, nt, band, s.cuts, s.cut_stages, part, pitch_of(o.n), (uint32_t)((uint64_t)mt * nt * s.cuts), o, bias, second, a_down, b_down};
}

static uint32_t bias_groups(const LinBias& b, uint32_t threads) { return b.out ? (b.cols + threads / 16 - 1) / (threads / 16) : 0; }

template <typename T> static void join(apoe_ctx* ctx, const LinTile& t) {
    if (t.cuts <= 1) return;
    const uint32_t grid = (uint32_t)std::min<uint64_t>(((uint64_t)t.o.m * (t.np / 8) + 255) / 256, 1u << 16);
    if constexpr (sizeof(T) == 4) {
        linear_join<T, true><<<grid, 256, 0, ctx->stream>>>(t);
    } else {
        if (t.second) linear_join<T, true><<<grid, 256, 0, ctx->stream>>>(t);
        else linear_join<T, false><<<grid, 256, 0, ctx->stream>>>(t);
    }
}

// Calls go(threads of a workgroup, the kernel's numbers) for the tiles of a kind.
template <int... N> struct Numbers {};
template <typename T, typename F> static void with_kind(uint32_t kind, F&& go) {
    if constexpr (sizeof(T) == 2) {
        if (kind == 0) go(512, Numbers<4, 2, 2, 4, 1, 4, 2>{});
        else if (kind == 1) go(512, Numbers<2, 2, 4, 2, 1, 4, 3>{});
        else if (kind == 2) go(256, Numbers<2, 2, 2, 2, 1, 4, 2>{});
        else if (kind == 3) go(512, Numbers<2, 2, 2, 2, 2, 4, 4>{});
        else go(256, Numbers<1, 1, 2, 2, 1, 4, 4>{});
    } else {
        if (kind == 0) go(512, Numbers<4, 2, 2, 4, 1, 32, 2>{});
        else if (kind == 1) go(512, Numbers<2, 2, 2, 2, 2, 32, 4>{});
        else go(512, Numbers<2, 1, 1, 2, 4, 64, 4>{});
    }
}

template <typename T, bool BCOL, bool ONE, int... N> static void start(hipStream_t s, uint32_t threads, const LinTile& t, Numbers<N...>) {
    const uint32_t grid = t.groups + bias_groups(t.bias, threads);
    if constexpr (sizeof(T) == 4) {
        linear_tile32<false, BCOL, ONE, N...><<<grid, threads, 0, s>>>(t);
    } else if constexpr (BCOL) {
        if (t.second) linear_tile<T, false, true, true, N...><<<grid, threads, 0, s>>>(t);
        else linear_tile<T, false, true, false, N...><<<grid, threads, 0, s>>>(t);
    } else {
        linear_tile<T, false, false, false, N...><<<grid, threads, 0, s>>>(t);
    }
}
template <typename T, bool BCOL, bool ONE = false> static void product(apoe_ctx* ctx, uint32_t kind, const LinTile& t) {
    with_kind<T>(kind, [&](uint32_t threads, auto numbers) { start<T, BCOL, ONE>(ctx->stream, threads, t, numbers); });
    join<T>(ctx, t);
}

template <typename T, int... N> static void start_grads(hipStream_t s, uint32_t threads, const LinTile& x, const LinTile& w, Numbers<N...>) {
    const uint32_t grid = x.groups + w.groups + bias_groups(w.bias, threads);
    if constexpr (sizeof(T) == 4) {
        linear_grads32<N...><<<grid, threads, 0, s>>>(x, w);
    } else {
        if (w.second) linear_grads<T, true, N...><<<grid, threads, 0, s>>>(x, w);
        else linear_grads<T, false, N...><<<grid, threads, 0, s>>>(x, w);
    }
}
template <typename T> static void grad_products(apoe_ctx* ctx, uint32_t kind, const LinTile& x, const LinTile& w) {
    with_kind<T>(kind, [&](uint32_t threads, auto numbers) { start_grads<T>(ctx->stream, threads, x, w, numbers); });
    if (x.groups) join<T>(ctx, x);
    join<T>(ctx, w);
}

template <typename T> static bool whole_rows(const void* p, uint64_t stride) { return ((uintptr_t)p & 15) == 0 && stride % (16 / sizeof(T)) == 0; }

template <typename T> static int run_linear(apoe_ctx* ctx, const apoe_linear_args* p) {
    const uint32_t m = p->rows, n = p->cols_out, k = p->cols_in;
    constexpr uint32_t E = 16 / sizeof(T);
    // Few rows and a w that is soon read (us of a call, tiles of 64 x 64 in brackets: 16 rows of fp16, 1024 x 1024 6.8 (7.4), 4096 -> 1024 9.0 (9.9), 4096 x 4096 9.4 (11),
    // 4096 -> 16 384 39 (31), one row 26 (31); float, 1024 x 1024 6.5 (9.8), 2048 x 2048 10 (12), 4096 -> 1024 18 (12)); more rows: tiles (32 of 4096 x 4096 13.5 (11)).
    const bool soon = k <= (sizeof(T) == 2 ? 4096 : 2048) && ((uint64_t)n * k <= 1u << 25 || m <= 4);
    if (m <= 16 && soon && k % E == 0 && whole_rows<T>(p->x, p->x_stride) && whole_rows<T>(p->w, p->w_stride)) {
        const LinFew a{p->x, p->w, p->x_stride, p->w_stride, k, LinOut{p->y, p->bias, p->residual, p->pre, p->y_stride, p->residual_stride, p->pre_stride, m, n, p->act}};
        if (k >= 4096) linear_few<T, 16><<<(n + 15) / 16, 1024, 0, ctx->stream>>>(a); // two turns of the inner side for each wave
        else linear_few<T, 8><<<(n + 15) / 16, 512, 0, ctx->stream>>>(a);
        APOE_HIP(hipGetLastError());
        return APOE_OK;
    }
    bool x_is = as_it_is<T>(p->x, p->x_stride, k), w_is = as_it_is<T>(p->w, p->w_stride, k);
    const LinShape s = choose<T>(ctx, m, n, k);
    // Floats that begin anywhere: taken a float a load where that costs the product (a seventh more) less than laying them out anew costs, 5 us and the bytes
    // (777 x 1001 x 999 26 us, laid out anew 31; 8191 x 4095 x 1001 388, 424; 4096 x 4095 x 4097 is laid out, 950, a float a load 978).
    bool one = false;
    if constexpr (sizeof(T) == 4) {
        const float anew = 5.f + ((x_is ? 0.f : (float)m) + (w_is ? 0.f : (float)n)) * (float)k * 8.f / 4e6f;
        one = !(x_is && w_is) && near_rows<T>(p->x_stride) && near_rows<T>(p->w_stride) && .15f * s.us < anew;
        if (one) x_is = w_is = true;
    }
    LinPlan plan;
    const uint64_t o_x = plan.take(x_is ? 0 : packed_bytes<T>(m, k)), o_w = plan.take(w_is ? 0 : packed_bytes<T>(n, k)), o_part = plan.take(cut_bytes(s, m, n));
    char* ws = nullptr;
    if (plan.bytes) APOE_TRY(ctx->adapt_workspace(plan.bytes, &ws));
    LinOperand x{p->x, (uint32_t)(p->x_stride * sizeof(T))}, w{p->w, (uint32_t)(p->w_stride * sizeof(T))};
    LinPacks packs{};
    if (!x_is) {
        x = LinOperand{ws + o_x, pitch_of(k) * (uint32_t)sizeof(T)};
        add_pack<T>(ctx, packs, p->x, p->x_stride, m, k, ws + o_x);
    }
    if (!w_is) {
        w = LinOperand{ws + o_w, pitch_of(k) * (uint32_t)sizeof(T)};
        add_pack<T>(ctx, packs, p->w, p->w_stride, n, k, ws + o_w);
    }
    pack<T>(ctx, packs);
    LinOut o{p->y, p->bias, p->residual, p->pre, p->y_stride, p->residual_stride, p->pre_stride, m, n, p->act};
    const LinTile t = tiles_of(s, x, w, k, (float*)(ws + o_part), o);
    if constexpr (sizeof(T) == 4) {
        if (one) product<T, false, true>(ctx, s.kind, t);
    }
    if (!one) product<T, false>(ctx, s.kind, t);
    APOE_HIP(hipGetLastError());
    return APOE_OK;
}

template <typename T> static int run_linear_grad(apoe_ctx* ctx, const apoe_linear_args* p) {
    const uint32_t m = p->rows, n = p->cols_out, k = p->cols_in;
    const bool act = p->act != APOE_ACT_NONE, products = p->grad_x || p->grad_w;
    const bool g_is = !act && as_it_is<T>(p->grad_y, p->grad_y_stride, n), x_is = !p->grad_w || as_it_is<T>(p->x, p->x_stride, k), w_is = !p->grad_x || as_it_is<T>(p->w, p->w_stride, k);
    const bool pack_g = products && !g_is;
    const uint32_t parts = sizeof(T) == 2 && (p->act == APOE_ACT_GELU || p->act == APOE_ACT_SILU) ? 2 : 1;
    const uint64_t second = parts == 2 ? packed_bytes<T>(m, n) : 0;
    LinShape sx{}, sw{};
    if (p->grad_x) sx = choose<T>(ctx, m, k, n, parts);
    if (p->grad_w) sw = choose<T>(ctx, n, k, m, parts);
    LinPlan plan;
    const uint64_t o_g = plan.take(pack_g ? parts * packed_bytes<T>(m, n) : 0), o_x = plan.take(x_is ? 0 : packed_bytes<T>(m, k)), o_w = plan.take(w_is ? 0 : packed_bytes<T>(n, k));
    // Both products in one launch where they have tiles of one kind: none waits for the other's last tiles (bf16, the whole call: 512 rows of 1024 x 1024 21.4 -> 18.3 us, 2048
    // of them 25.8 -> 23.2, 8192 of 4096 x 4096 479 -> 477; float 4096 rows of 1024 x 1024 116 -> 114). Each has the tiles and cuts that it has alone: the same bits.
    const bool together = p->grad_x && p->grad_w && m && sx.kind == sw.kind;
    const uint64_t x_part = p->grad_x ? cut_bytes(sx, m, k) : 0, w_part = p->grad_w ? cut_bytes(sw, n, k) : 0;
    const uint64_t o_part = plan.take(together ? x_part : std::max(x_part, w_part)), o_more = together ? plan.take(w_part) : o_part;
    const uint64_t o_bias = plan.take(p->grad_bias ? (uint64_t)LIN_STRIPS * n * 4 : 0);
    char* ws = nullptr;
    if (plan.bytes) APOE_TRY(ctx->adapt_workspace(plan.bytes, &ws));
    LinOperand g{p->grad_y, (uint32_t)(p->grad_y_stride * sizeof(T))}, x{p->x, (uint32_t)(p->x_stride * sizeof(T))}, w{p->w, (uint32_t)(p->w_stride * sizeof(T))};
    LinPacks packs{};
    LinBias bias{};
    if (pack_g || p->grad_bias) {
        LinPack& a = add_pack<T>(ctx, packs, p->grad_y, p->grad_y_stride, m, n, pack_g ? ws + o_g : nullptr);
        if (act) {
            a.pre = p->pre;
            a.pre_stride = p->pre_stride;
            a.act = p->act;
            if (pack_g && second) a.second = ws + o_g + second;
        }
        if (p->grad_bias) {
            a.part = (float*)(ws + o_bias);
            bias = LinBias{a.part, p->grad_bias, a.strips, n};
        }
        if (pack_g) g = LinOperand{ws + o_g, pitch_of(n) * (uint32_t)sizeof(T)};
    }
    if (!x_is) {
        x = LinOperand{ws + o_x, pitch_of(k) * (uint32_t)sizeof(T)};
        add_pack<T>(ctx, packs, p->x, p->x_stride, m, k, ws + o_x);
    }
    if (!w_is) {
        w = LinOperand{ws + o_w, pitch_of(k) * (uint32_t)sizeof(T)};
        add_pack<T>(ctx, packs, p->w, p->w_stride, n, k, ws + o_w);
    }
    pack<T>(ctx, packs);
    LinTile tx{};
    if (p->grad_x && m) {
        const LinOut o{p->grad_x, nullptr, nullptr, nullptr, p->grad_x_stride, 0, 0, m, k, APOE_ACT_NONE};
        tx = tiles_of(sx, g, w, n, (float*)(ws + o_part), o, p->grad_w ? LinBias{} : bias, second, false, true);
        if (!together) product<T, true>(ctx, sx.kind, tx);
    }
    if (p->grad_w) {
        const LinOut o{p->grad_w, nullptr, nullptr, nullptr, p->grad_w_stride, 0, 0, n, k, APOE_ACT_NONE};
        grad_products<T>(ctx, sw.kind, together ? tx : LinTile{}, tiles_of(sw, g, x, m, (float*)(ws + o_more), o, bias, second, true, true));
    }
    if (p->grad_bias && !p->grad_w && !(p->grad_x && m)) linear_bias<<<(n + 31) / 32, 512, 0, ctx->stream>>>(bias);
    APOE_HIP(hipGetLastError());
    return APOE_OK;
}

int launch_linear(apoe_ctx* ctx, const apoe_linear_args* p, bool grad) {
    switch (p->dtype) {
    case APOE_F32: return grad ? run_linear_grad<float>(ctx, p) : run_linear<float>(ctx, p);
    case APOE_F16: return grad ? run_linear_grad<_Float16>(ctx, p) : run_linear<_Float16>(ctx, p);
    default: return grad ? run_linear_grad<__bf16>(ctx, p) : run_linear<__bf16>(ctx, p);
    }
}

} // namespace apoe
