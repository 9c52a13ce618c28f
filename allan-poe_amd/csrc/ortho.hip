// Newton-Schulz orthogonalisation of a matrix (or a batch): X = in / |in|, then a number of times X = a X + (b A + c A A) X with
// A = X X^T, on the short side (a tall matrix is worked on transposed).
//
// What rounding costs here: a gradient has a few strong directions over a floor that is hundreds of times lower, and the steps
// raise the floor by up to a^steps (485 for the usual five). Rounding X itself to 16 bits plants noise of the strong directions'
// size in the floor, which is raised with it (fp16: 1.6 % of the result at 1024 x 1024, bf16: 13 %). Rounding A and B = b A + c A A
// does not: they multiply X, so their errors are relative to what they multiply, and B is near zero on the floor. So X is kept
// in 32 bits and the products take fp16 copies of X, A and B (times 2^12: X and A are about one at most, their small values stay
// clear of the subnormal numbers); B's diagonal, which is its largest part when all singular values are alike, stays in 32
// bits and scales X's rows outside the product. That leaves 1e-4 to 6e-4 (fp16 rounds its result by 2e-4, bf16 by 17e-4), less the
// longer the sides are, over which the roundings average.
// SPLIT, for results in 32 bits, for fp16 ones and for short sides, where nothing averages: every operand is two fp16 matrices, its
// rounded value and what that left (22 bits together), and a product is three: high x high, high x low, low x high.
#include <type_traits>

#include "apoe_internal.h"
#include "apoe_tile.h"

namespace apoe {

constexpr int ORTHO_PARTS = 256; // partial sums of squares of a matrix, at most
constexpr uint32_t ORTHO_PAD = 64; // columns of the working matrices are rounded up to this, with zeros

struct OrthoArgs {
    const void* in;
    void* out;
    uint64_t in_stride, out_stride, in_batch, out_batch; // elements
    uint32_t in_dtype, out_dtype, m, n, mp, np, parts;   // m <= n: the sides; mp, np: rounded up
    bool tall;
    float a, b, c, alpha, beta;
    double* part;  // [batch][ORTHO_PARTS]
    float* x;      // [batch][m][np] the iterate
    _Float16 *h, *h2;      // [batch][m][np] operand of the products, now and next; SPLIT: the low parts lie h_low values behind
    _Float16 *gram, *poly; // [batch][m][mp]; SPLIT: g_low values behind
    uint64_t h_low, g_low;
    float* diag;   // [batch][mp]
};

constexpr float ORTHO_UP = 4096.f, ORTHO_DOWN = 1.f / 4096.f; // of the fp16 copies

// v times 2^12 as fp16, and what that leaves.
template <bool SPLIT> __device__ inline void put(_Float16* at, uint64_t low, float v) {
    v *= ORTHO_UP;
    const _Float16 hi = (_Float16)v;
    *at = hi;
    if constexpr (SPLIT) at[low] = (_Float16)(v - (float)hi);
}

__device__ inline float load_as_float(const void* p, uint64_t i, uint32_t dtype) {
    return dtype == APOE_F32 ? ((const float*)p)[i] : dtype == APOE_F16 ? (float)((const _Float16*)p)[i] : (float)((const __bf16*)p)[i];
}
__device__ inline void store_from_float(void* p, uint64_t i, uint32_t dtype, float v) {
    if (dtype == APOE_F32) ((float*)p)[i] = v;
    else if (dtype == APOE_F16) ((_Float16*)p)[i] = (_Float16)v;
    else ((__bf16*)p)[i] = (__bf16)v;
}

// Sums of squares, in 64 bits (no input over- or underflows): grid (parts, batch), a part takes every parts-th row.
__global__ __launch_bounds__(256) void ortho_squares(OrthoArgs a) {
    __shared__ double buf[4];
    const uint32_t rows = a.tall ? a.n : a.m, cols = a.tall ? a.m : a.n;
    double s = 0;
    for (uint32_t r = blockIdx.x; r < rows; r += gridDim.x)
        for (uint32_t c = threadIdx.x; c < cols; c += 256) {
            const double v = load_as_float(a.in, blockIdx.y * a.in_batch + r * a.in_stride + c, a.in_dtype);
            s += v * v;
        }
    for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
    if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) a.part[blockIdx.y * ORTHO_PARTS + blockIdx.x] = (buf[0] + buf[1]) + (buf[2] + buf[3]);
}

// X and its operand copy, 64 x 64 at a time (through LDS where the matrix is turned): grid (np / 64, m / 64 up, batch).
template <bool SPLIT> __global__ __launch_bounds__(256) void ortho_first(OrthoArgs a) {
    __shared__ double buf[4];
    __shared__ float tile[64][65];
    double s = threadIdx.x < a.parts ? a.part[blockIdx.z * ORTHO_PARTS + threadIdx.x] : 0.;
    for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
    if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = s;
    __syncthreads();
    const double norm = sqrt((buf[0] + buf[1]) + (buf[2] + buf[3])), inv = norm == 0. ? 0. : 1. / norm;
    const uint32_t i0 = blockIdx.y * 64, j0 = blockIdx.x * 64, tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
    const uint64_t in0 = blockIdx.z * a.in_batch;
    if (a.tall) {
        for (uint32_t r = ty; r < 64; r += 4)
            if (j0 + r < a.n && i0 + tx < a.m) tile[tx][r] = load_as_float(a.in, in0 + (uint64_t)(j0 + r) * a.in_stride + i0 + tx, a.in_dtype);
        __syncthreads();
    }
    const uint32_t j = j0 + tx;
    for (uint32_t r = ty; r < 64; r += 4) {
        const uint32_t i = i0 + r;
        if (i >= a.m) break;
        float v = 0.f;
        if (j < a.n) v = a.tall ? tile[r][tx] : load_as_float(a.in, in0 + (uint64_t)i * a.in_stride + j, a.in_dtype);
        v = (float)(v * inv);
        const uint64_t at = ((uint64_t)blockIdx.z * a.m + i) * a.np + j;
        a.x[at] = v;
        put<SPLIT>(a.h + at, a.h_low, v);
    }
}

enum { ORTHO_GRAM = 0, ORTHO_POLY = 1, ORTHO_STEP = 2, ORTHO_LAST = 3 };

// One product of a step. GRAM: A = X X^T; POLY: B = b A + c A A, whose diagonal goes to `diag`; both symmetric, so the tiles on and
// below the diagonal are computed and written twice. STEP: X = (a + diag) X + B X; LAST: the same into `out`.
template <bool SPLIT, int MT, int NT, int WM, int WN, int SF, int ST, int KIND>
__global__ __launch_bounds__(64 * WM * WN, 2) void ortho_tile(OrthoArgs a) {
    using T = _Float16;
    constexpr int NW = WM * WN, BM = WM * MT * 32, BN = WN * NT * 32, PLANES = SPLIT ? 2 : 1;
    constexpr bool SYM = KIND == ORTHO_GRAM || KIND == ORTHO_POLY;
    using ATile = RowTile<T, BM, SF, NW>;
    using BTile = std::conditional_t<SYM, RowTile<T, BN, SF, NW>, ColTile<T, BN, SF, NW, ORDER_ROWS>>;
    static_assert(!SYM || BM == BN, "square tiles");
    constexpr int PLANE = ATile::BYTES + BTile::BYTES, STAGE = PLANES * PLANE, PER = PLANES * (ATile::LOADS + BTile::LOADS), KE = ATile::KE;
    __shared__ __align__(1024) char lds[ST * STAGE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
    uint32_t ti, tj;
    if constexpr (SYM) {
        ti = (uint32_t)((sqrtf(8.f * blockIdx.x + 1.f) - 1.f) * 0.5f);
        while (ti * (ti + 1) / 2 > blockIdx.x) ti--;
        while ((ti + 1) * (ti + 2) / 2 <= blockIdx.x) ti++;
        tj = blockIdx.x - ti * (ti + 1) / 2;
        ti = __builtin_amdgcn_readfirstlane(ti);
        tj = __builtin_amdgcn_readfirstlane(tj);
    } else {
        const uint32_t nt = (a.n + BN - 1) / BN;
        ti = blockIdx.x / nt;
        tj = blockIdx.x % nt;
    }
    const uint32_t row = ti * BM, col = tj * BN, batch = blockIdx.y;
    const uint64_t xo = (uint64_t)batch * a.m * a.np, go = (uint64_t)batch * a.m * a.mp;
    const T* h = a.h + xo;
    const T* gram = a.gram + go;
    const T* poly = a.poly + go;
    ATile ta[PLANES];
    BTile tb[PLANES];
    const uint32_t xp = a.np * (uint32_t)sizeof(T), gp = a.mp * (uint32_t)sizeof(T);
    const int mrows = (int)min((uint32_t)BM, a.m - row);
#pragma unroll
    for (int p = 0; p < PLANES; p++) {
        const uint64_t hl = p * a.h_low, gl = p * a.g_low;
        if constexpr (KIND == ORTHO_GRAM) {
            ta[p].init(h + hl + (uint64_t)row * a.np, xp, mrows, wave, lane);
            tb[p].init(h + hl + (uint64_t)col * a.np, xp, (int)min((uint32_t)BN, a.m - col), wave, lane);
        } else if constexpr (KIND == ORTHO_POLY) {
            ta[p].init(gram + gl + (uint64_t)row * a.mp, gp, mrows, wave, lane);
            tb[p].init(gram + gl + (uint64_t)col * a.mp, gp, (int)min((uint32_t)BN, a.m - col), wave, lane);
        } else {
            ta[p].init(poly + gl + (uint64_t)row * a.mp, gp, mrows, wave, lane);
            tb[p].init(h + hl + col, xp, (int)min((uint32_t)BN, a.np - col), wave, lane);
        }
    }
    const int inner = (int)(KIND == ORTHO_GRAM ? a.np : a.mp); // pads are zeros (STEP: rows beyond m are masked)
    const int stages = (inner + KE - 1) / KE;
    const uint32_t base = lds_address(lds);
    int left = inner;
    uint32_t into = 0;
    auto issue = [&]() {
#pragma unroll
        for (int p = 0; p < PLANES; p++) {
            const uint32_t at = base + into + p * PLANE;
            ta[p].load(at, left * (int)sizeof(T), wave);
            if constexpr (SYM) {
                tb[p].load(at + ATile::BYTES, left * (int)sizeof(T), wave);
            } else {
                using Mask = typename BTile::Mask;
                const int rows = left - (int)(a.mp - a.m); // of X
                tb[p].load(at + ATile::BYTES, rows >= KE ? BTile::ALL : rows > 0 ? (Mask)(((Mask)1 << rows) - 1) : (Mask)0, wave, lane);
            }
            ta[p].next();
            tb[p].next();
        }
        left -= KE;
        into = into + STAGE == ST * STAGE ? 0 : into + STAGE;
    };
#pragma unroll
    for (int s = 0; s < ST - 1; s++) issue();
    f32x16 acc[MT][NT] = {};
    uint32_t from = 0;
    for (int s = 0; s < stages; s++) {
        tile_wait<(ST - 2) * PER>();
        issue();
        const char* A = lds + from;
        const char* B = A + ATile::BYTES;
        i32x4 x[2][PLANES][MT], y[2][PLANES][NT];
        auto read = [&](int f) {
#pragma unroll
            for (int p = 0; p < PLANES; p++) {
#pragma unroll
                for (int m = 0; m < MT; m++) x[f & 1][p][m] = ATile::read(A + p * PLANE, wm * MT + m, f, lane);
#pragma unroll
                for (int t = 0; t < NT; t++) y[f & 1][p][t] = BTile::read(B + p * PLANE, wn * NT + t, f, lane);
            }
        };
        read(0);
#pragma unroll
        for (int f = 0; f < SF; f++) {
            if (f + 1 < SF) read(f + 1);
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    if constexpr (SPLIT) {
                        acc[m][t] = mfma_step<T>(x[f & 1][1][m], y[f & 1][0][t], acc[m][t]);
                        acc[m][t] = mfma_step<T>(x[f & 1][0][m], y[f & 1][1][t], acc[m][t]);
                    }
                    acc[m][t] = mfma_step<T>(x[f & 1][0][m], y[f & 1][0][t], acc[m][t]);
                }
        }
        interleave<PLANES * (MT + (SYM ? 1 : 2) * NT), (SPLIT ? 3 : 1) * MT * NT, SF>();
        from = from + STAGE == ST * STAGE ? 0 : from + STAGE;
    }
    tile_wait<0>();
    const int half = lane >> 5;
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const uint32_t j = col + (wn * NT + t) * 32 + (lane & 31);
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const uint32_t i0 = row + (wm * MT + m) * 32 + 8 * g + 4 * half;
                float v[4];
#pragma unroll
                for (int k = 0; k < 4; k++) v[k] = acc[m][t][4 * g + k] * (ORTHO_DOWN * ORTHO_DOWN);
                if constexpr (SYM) {
                    if (j >= a.mp) continue;
                    T* to = (KIND == ORTHO_GRAM ? a.gram : a.poly) + go;
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const uint32_t i = i0 + k;
                        if (i >= a.m) continue;
                        const uint64_t at = (uint64_t)i * a.mp + j;
                        if constexpr (KIND == ORTHO_POLY) {
                            float own = (float)gram[at];
                            if constexpr (SPLIT) own += (float)gram[at + a.g_low];
                            v[k] = j < a.m ? __builtin_fmaf(a.c, v[k], a.b * ORTHO_DOWN * own) : 0.f;
                            if (i == j) {
                                a.diag[(uint64_t)batch * a.mp + i] = v[k];
                                v[k] = 0.f;
                            }
                        }
                        put<SPLIT>(to + at, a.g_low, v[k]);
                    }
                    if (ti != tj && j < a.m && i0 < a.mp) {
                        // four values of a row at once; beyond m they are the zeros that the pad holds
                        typedef T t4 __attribute__((ext_vector_type(4)));
                        t4 hi, lo;
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            hi[k] = (T)(v[k] * ORTHO_UP);
                            lo[k] = (T)(v[k] * ORTHO_UP - (float)hi[k]);
                        }
                        T* at = to + (uint64_t)j * a.mp + i0;
                        *reinterpret_cast<t4*>(at) = hi;
                        if constexpr (SPLIT) *reinterpret_cast<t4*>(at + a.g_low) = lo;
                    }
                } else {
                    if (j >= a.np) continue;
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const uint32_t i = i0 + k;
                        if (i >= a.m) continue;
                        const uint64_t at = xo + (uint64_t)i * a.np + j;
                        v[k] = __builtin_fmaf(a.a + a.diag[(uint64_t)batch * a.mp + i], a.x[at], v[k]);
                        if constexpr (KIND == ORTHO_STEP) {
                            a.x[at] = v[k];
                            put<SPLIT>(a.h2 + at, a.h_low, v[k]);
                        } else if (j < a.n) {
                            const uint64_t o = batch * a.out_batch + (a.tall ? (uint64_t)j * a.out_stride + i : (uint64_t)i * a.out_stride + j);
                            float r = a.alpha * v[k];
                            if (a.beta != 0.f) r = __builtin_fmaf(a.beta, load_as_float(a.out, o, a.out_dtype), r);
                            store_from_float(a.out, o, a.out_dtype, r);
                        }
                    }
                }
            }
        }
}

template <bool SPLIT> static int run_ortho(apoe_ctx* ctx, const apoe_orthogonalize_args* p) {
    OrthoArgs a{};
    a.in = p->in;
    a.out = p->out;
    a.in_stride = p->in_stride;
    a.out_stride = p->out_stride;
    a.in_batch = p->in_batch_stride;
    a.out_batch = p->out_batch_stride;
    a.in_dtype = p->in_dtype;
    a.out_dtype = p->out_dtype;
    a.tall = p->rows > p->cols;
    a.m = a.tall ? p->cols : p->rows;
    a.n = a.tall ? p->rows : p->cols;
    a.mp = (a.m + ORTHO_PAD - 1) / ORTHO_PAD * ORTHO_PAD;
    a.np = (a.n + ORTHO_PAD - 1) / ORTHO_PAD * ORTHO_PAD;
    a.a = p->a;
    a.b = p->b;
    a.c = p->c;
    a.alpha = p->alpha;
    a.beta = p->beta;
    a.parts = std::min<uint32_t>(ORTHO_PARTS, p->rows);
    const uint32_t batch = p->batch;
    size_t bytes = 0;
    auto take = [&](size_t b) {
        const size_t at = bytes;
        bytes += (b + 1023) / 1024 * 1024;
        return at;
    };
    const size_t xs = (size_t)batch * a.m * a.np, gs = (size_t)batch * a.m * a.mp;
    const size_t o_part = take((size_t)batch * ORTHO_PARTS * 8), o_diag = take((size_t)batch * a.mp * 4), o_x = take(xs * 4);
    constexpr int PLANES = SPLIT ? 2 : 1;
    a.h_low = (xs + 511) / 512 * 512;
    a.g_low = (gs + 511) / 512 * 512;
    const size_t o_h = take(PLANES * a.h_low * 2), o_h2 = take(PLANES * a.h_low * 2), o_gram = take(PLANES * a.g_low * 2), o_poly = take(PLANES * a.g_low * 2);
    char* ws = nullptr;
    APOE_TRY(ctx->adapt_workspace(bytes, &ws));
    a.part = (double*)(ws + o_part);
    a.diag = (float*)(ws + o_diag);
    a.x = (float*)(ws + o_x);
    a.h = (_Float16*)(ws + o_h);
    a.h2 = (_Float16*)(ws + o_h2);
    a.gram = (_Float16*)(ws + o_gram);
    a.poly = (_Float16*)(ws + o_poly);
    hipStream_t s = ctx->stream;
    ortho_squares<<<dim3(a.parts, batch), 256, 0, s>>>(a);
    ortho_first<SPLIT><<<dim3(a.np / 64, (a.m + 63) / 64, batch), 256, 0, s>>>(a);
    auto triangle = [](uint32_t t) { return t * (t + 1) / 2; };
    // tiles of 128 x 128 where they fill the GPU, else of 64 x 64
    const uint32_t t128 = (a.m + 127) / 128, t64 = (a.m + 63) / 64, n128 = (a.n + 127) / 128, n64 = (a.n + 63) / 64;
    const bool wide_sym = (uint64_t)triangle(t128) * batch >= (uint32_t)ctx->num_cus;
    const bool wide_step = (uint64_t)t128 * n128 * batch >= (uint32_t)ctx->num_cus;
    auto sym = [&](auto kind) {
        constexpr int K = decltype(kind)::value;
        if (wide_sym) ortho_tile<SPLIT, 2, 2, 2, 2, 2, SPLIT ? 2 : 3, K><<<dim3(triangle(t128), batch), 256, 0, s>>>(a);
        else ortho_tile<SPLIT, 1, 1, 2, 2, SPLIT ? 2 : 4, 3, K><<<dim3(triangle(t64), batch), 256, 0, s>>>(a);
    };
    auto step = [&](auto kind) {
        constexpr int K = decltype(kind)::value;
        if (wide_step) ortho_tile<SPLIT, 2, 2, 2, 2, 2, SPLIT ? 2 : 3, K><<<dim3(t128 * n128, batch), 256, 0, s>>>(a);
        else ortho_tile<SPLIT, 1, 1, 2, 2, SPLIT ? 2 : 4, 3, K><<<dim3(t64 * n64, batch), 256, 0, s>>>(a);
    };
    for (uint32_t i = 0; i < p->steps; i++) {
        sym(std::integral_constant<int, ORTHO_GRAM>{});
        sym(std::integral_constant<int, ORTHO_POLY>{});
        if (i + 1 < p->steps) step(std::integral_constant<int, ORTHO_STEP>{});
        else step(std::integral_constant<int, ORTHO_LAST>{});
        std::swap(a.h, a.h2);
    }
    APOE_HIP(hipGetLastError());
    return APOE_OK;
}

int launch_orthogonalize(apoe_ctx* ctx, const apoe_orthogonalize_args* p) {
    // a side of one tile: the roundings do not average (2 x 3: 0.8 % off in fp16 products); 87 us for 74 at 64 x 64, 143 for 97 at 64 x 1024
    const bool split = p->products == APOE_F32 || std::min(p->rows, p->cols) <= 64;
    return split ? run_ortho<true>(ctx, p) : run_ortho<false>(ctx, p);
}

} // namespace apoe
