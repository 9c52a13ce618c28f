// Newton-Schulz orthogonalisation of a matrix (or a batch): X = in / |in|, then a number of times X = a X + (b A + c A A) X with
// A = X X^T, on the short side (a tall matrix is worked on transposed).
//
// What rounding costs here: a gradient has a few strong directions over a floor that is hundreds of times lower, and the steps
// raise the floor by up to a^steps (485 for the usual five). Rounding X itself to 16 bits plants noise of the strong directions'
// size in the floor, which is raised with it (fp16: 1.6 % of the result at 1024 x 1024, bf16: 13 %). Rounding A and B = b A + c A A
// does not: they multiply X, so their errors are relative to what they multiply, and B is near zero on the floor. So X is kept
// as two fp16 matrices, its rounded value and what that left (22 bits together; kept in fp32 beside an fp16 copy, the errors below are
// the same in two digits, and the traffic of B X half as much again: 4 x 1024 x 4096 625 us for 595), and the products take fp16
// copies of X (the high part), A and B, all times 2^12: X and A are about one at most, their small values stay clear of the subnormal
// numbers (an entry of 16 would be infinite, in any of the three, and so would be the result); B's diagonal, which is its largest part when all singular values are alike, stays in 32 bits and scales X's rows outside
// the product. That leaves 1e-4 to 6e-4 (fp16 rounds its result by 2e-4, bf16 by 17e-4), less the longer the sides are, over which
// the roundings average.
// SPLIT, for results in 32 bits, for fp16 ones and (ortho_narrow) for short sides, where nothing averages: X in fp32, every operand two fp16 matrices,
// and a product is three: high x high, high x low, low x high.
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
    bool tall, whole_out; // worked on transposed; rows of `out` are multiples of 16 bytes
    float a, b, c, alpha, beta;
    double* part;  // [batch][ORTHO_PARTS]
    float* x;      // [batch][m][np] the iterate, SPLIT only
    _Float16 *h, *h2;      // [batch][m][np] the iterate, now and next: high parts, operand of the products; the low parts lie h_low values behind
    _Float16 *gram, *poly; // [batch][m][mp]; SPLIT: g_low values behind
    uint64_t h_low, g_low;
    float* diag;   // [batch][mp]
    float* cut;    // [batch][tiles][cuts][64 x 64]: X X^T of parts of the inner side
    uint32_t cuts, cut_stages; // 1: none
};

constexpr float ORTHO_UP = 4096.f, ORTHO_DOWN = 1.f / 4096.f; // of the fp16 copies

// v times 2^12 as fp16, and what that leaves.
__device__ inline void put(_Float16* at, uint64_t low, float v) {
    v *= ORTHO_UP;
    const _Float16 hi = (_Float16)v;
    *at = hi;
    at[low] = (_Float16)(v - (float)hi);
}

__device__ inline float load_as_float(const void* p, uint64_t i, uint32_t dtype) {
    return dtype == APOE_F32 ? ((const float*)p)[i] : dtype == APOE_F16 ? (float)((const _Float16*)p)[i] : (float)((const __bf16*)p)[i];
}
__device__ inline void store_from_float(void* p, uint64_t i, uint32_t dtype, float v) {
    if (dtype == APOE_F32) ((float*)p)[i] = v;
    else if (dtype == APOE_F16) ((_Float16*)p)[i] = (_Float16)v;
    else ((__bf16*)p)[i] = (__bf16)v;
}

// Sums of squares, in 64 bits (no input over- or underflows): grid (parts, batch), a wave a row. WHOLE: rows are multiples of 16 bytes.
template <bool WHOLE> __global__ __launch_bounds__(256) void ortho_squares(OrthoArgs a) {
    __shared__ double buf[4];
    const uint32_t rows = a.tall ? a.n : a.m, cols = a.tall ? a.m : a.n, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double s = 0;
    for (uint32_t r = blockIdx.x * 4 + wave; r < rows; r += gridDim.x * 4) {
        const uint64_t at = blockIdx.y * a.in_batch + r * a.in_stride;
        if constexpr (WHOLE) {
            const uint32_t v = a.in_dtype == APOE_F32 ? 4 : 8;
#pragma unroll 4
            for (uint32_t c = lane * v; c < cols; c += 64 * v) {
                if (a.in_dtype == APOE_F32) {
                    const f32x4 x = *reinterpret_cast<const f32x4*>((const float*)a.in + at + c);
                    for (int k = 0; k < 4; k++) s += (double)x[k] * (double)x[k];
                } else if (a.in_dtype == APOE_F16) {
                    const f16x8 x = *reinterpret_cast<const f16x8*>((const _Float16*)a.in + at + c);
                    for (int k = 0; k < 8; k++) s += (double)((float)x[k] * (float)x[k]); // a square of 11 bits is exact in fp32
                } else {
                    const bf16x8 x = *reinterpret_cast<const bf16x8*>((const __bf16*)a.in + at + c);
                    for (int k = 0; k < 8; k++) s += (double)(float)x[k] * (double)(float)x[k];
                }
            }
        } else {
            for (uint32_t c = lane; c < cols; c += 64) {
                const double v = load_as_float(a.in, at + c, a.in_dtype);
                s += v * v;
            }
        }
    }
    for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
    if (lane == 0) buf[wave] = s;
    __syncthreads();
    if (threadIdx.x == 0) a.part[blockIdx.y * ORTHO_PARTS + blockIdx.x] = (buf[0] + buf[1]) + (buf[2] + buf[3]);
}

// One over the norm, from the parts; the same for all 256 threads.
__device__ inline double ortho_inverse(const OrthoArgs& a, uint32_t batch, double* buf) {
    double s = threadIdx.x < a.parts ? a.part[batch * ORTHO_PARTS + threadIdx.x] : 0.;
    for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
    if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = s;
    __syncthreads();
    const double norm = sqrt((buf[0] + buf[1]) + (buf[2] + buf[3]));
    return norm == 0. ? 0. : 1. / norm;
}

// X and its operand copy from rows that are multiples of 16 bytes (and not turned), eight values a thread: grid (.., batch).
template <bool SPLIT> __global__ __launch_bounds__(256) void ortho_first_whole(OrthoArgs a) {
    __shared__ double buf[4];
    const double inv = ortho_inverse(a, blockIdx.y, buf);
    const uint32_t per = a.np / 8, rows_at_once = gridDim.x * 256 / per;
    const uint32_t at0 = blockIdx.x * 256 + threadIdx.x;
    if (at0 >= rows_at_once * per) return;
    const uint32_t j = at0 % per * 8;
    for (uint32_t i = at0 / per; i < a.m; i += rows_at_once) {
        const uint64_t from = blockIdx.y * a.in_batch + i * a.in_stride + j;
        float v[8] = {};
        if (j < a.n) {
            if (a.in_dtype == APOE_F32) {
#pragma unroll
                for (int k = 0; k < 8; k += 4)
                    if (j + k < a.n) {
                        const f32x4 x = *reinterpret_cast<const f32x4*>((const float*)a.in + from + k);
                        for (int l = 0; l < 4; l++) v[k + l] = x[l];
                    }
            } else if (a.in_dtype == APOE_F16) {
                const f16x8 x = *reinterpret_cast<const f16x8*>((const _Float16*)a.in + from);
                for (int k = 0; k < 8; k++) v[k] = (float)x[k];
            } else {
                const bf16x8 x = *reinterpret_cast<const bf16x8*>((const __bf16*)a.in + from);
                for (int k = 0; k < 8; k++) v[k] = (float)x[k];
            }
        }
        const uint64_t at = ((uint64_t)blockIdx.y * a.m + i) * a.np + j;
        f16x8 hi, lo;
#pragma unroll
        for (int k = 0; k < 8; k++) {
            v[k] = (float)(v[k] * inv);
            hi[k] = (_Float16)(v[k] * ORTHO_UP);
            lo[k] = (_Float16)(v[k] * ORTHO_UP - (float)hi[k]);
        }
        if constexpr (SPLIT) {
            *reinterpret_cast<f32x4*>(a.x + at) = f32x4{v[0], v[1], v[2], v[3]};
            *reinterpret_cast<f32x4*>(a.x + at + 4) = f32x4{v[4], v[5], v[6], v[7]};
        }
        *reinterpret_cast<f16x8*>(a.h + at) = hi;
        *reinterpret_cast<f16x8*>(a.h + a.h_low + at) = lo;
    }
}

// X and its operand copy, 64 x 64 at a time (through LDS where the matrix is turned): grid (np / 64, m / 64 up, batch).
template <bool SPLIT> __global__ __launch_bounds__(256) void ortho_first(OrthoArgs a) {
    __shared__ double buf[4];
    __shared__ float tile[64][65];
    const double inv = ortho_inverse(a, blockIdx.z, buf);
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
        if constexpr (SPLIT) a.x[at] = v;
        put(a.h + at, a.h_low, v);
    }
}

template <bool SPLIT> __device__ inline void put8(_Float16* at, uint64_t low, const float* v) {
    f16x8 hi, lo;
#pragma unroll
    for (int k = 0; k < 8; k++) {
        hi[k] = (_Float16)(v[k] * ORTHO_UP);
        lo[k] = (_Float16)(v[k] * ORTHO_UP - (float)hi[k]);
    }
    *reinterpret_cast<f16x8*>(at) = hi;
    if constexpr (SPLIT) *reinterpret_cast<f16x8*>(at + low) = lo;
}

// Eight values of the iterate, as they come (two times f32x4, or high and low parts), and as numbers.
template <bool SPLIT> struct Iterate8 {
    f32x4 x0 = {}, x1 = {};
    __device__ void load(const OrthoArgs& a, uint64_t at) {
        x0 = *reinterpret_cast<const f32x4*>(a.x + at);
        x1 = *reinterpret_cast<const f32x4*>(a.x + at + 4);
    }
    __device__ float operator[](int k) const { return k < 4 ? x0[k] : x1[k - 4]; }
};
template <> struct Iterate8<false> {
    f16x8 hi = {}, lo = {};
    __device__ void load(const OrthoArgs& a, uint64_t at) {
        hi = *reinterpret_cast<const f16x8*>(a.h + at);
        lo = *reinterpret_cast<const f16x8*>(a.h + a.h_low + at);
    }
    __device__ float operator[](int k) const { return ((float)hi[k] + (float)lo[k]) * ORTHO_DOWN; }
};
template <bool SPLIT> __device__ inline float iterate1(const OrthoArgs& a, uint64_t at) {
    if constexpr (SPLIT) return a.x[at];
    else return ((float)a.h[at] + (float)a.h[a.h_low + at]) * ORTHO_DOWN;
}
template <bool SPLIT> __device__ inline void put_iterate8(const OrthoArgs& a, uint64_t at, const float* v) {
    if constexpr (SPLIT) {
        *reinterpret_cast<f32x4*>(a.x + at) = f32x4{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4*>(a.x + at + 4) = f32x4{v[4], v[5], v[6], v[7]};
    }
    put8<true>(a.h2 + at, a.h_low, v);
}

// v = b A + c v, for eight values of A at `gram`.
template <bool SPLIT> __device__ inline void ortho_poly(const OrthoArgs& a, const _Float16* gram, float* v) {
    const f16x8 hi = *reinterpret_cast<const f16x8*>(gram);
    f16x8 lo = {};
    if constexpr (SPLIT) lo = *reinterpret_cast<const f16x8*>(gram + a.g_low);
#pragma unroll
    for (int k = 0; k < 8; k++) v[k] = __builtin_fmaf(a.c, v[k], a.b * ORTHO_DOWN * ((float)hi[k] + (float)lo[k]));
}

// Eight values from rows that are multiples of 16 bytes.
__device__ inline void load8(const void* p, uint64_t at, uint32_t dtype, float* v) {
    if (dtype == APOE_F32) {
        const f32x4 x0 = *reinterpret_cast<const f32x4*>((const float*)p + at), x1 = *reinterpret_cast<const f32x4*>((const float*)p + at + 4);
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = k < 4 ? x0[k] : x1[k - 4];
    } else if (dtype == APOE_F16) {
        const f16x8 x = *reinterpret_cast<const f16x8*>((const _Float16*)p + at);
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = (float)x[k];
    } else {
        const bf16x8 x = *reinterpret_cast<const bf16x8*>((const __bf16*)p + at);
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = (float)x[k];
    }
}

// Eight values into `out`, whose rows are multiples of 16 bytes (and of eight values).
__device__ inline void add_row8(const OrthoArgs& a, uint64_t at, float* v) {
    if (a.beta != 0.f) {
        float old[8];
        load8(a.out, at, a.out_dtype, old);
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = __builtin_fmaf(a.beta, old[k], v[k]);
    }
    if (a.out_dtype == APOE_F32) {
        *reinterpret_cast<f32x4*>((float*)a.out + at) = f32x4{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4*>((float*)a.out + at + 4) = f32x4{v[4], v[5], v[6], v[7]};
    } else if (a.out_dtype == APOE_F16) {
        f16x8 x;
#pragma unroll
        for (int k = 0; k < 8; k++) x[k] = (_Float16)v[k];
        *reinterpret_cast<f16x8*>((_Float16*)a.out + at) = x;
    } else {
        bf16x8 x;
#pragma unroll
        for (int k = 0; k < 8; k++) x[k] = (__bf16)v[k];
        *reinterpret_cast<bf16x8*>((__bf16*)a.out + at) = x;
    }
}

// The tiles on and below the diagonal, row by row.
__device__ inline void tile_of(uint32_t tile, uint32_t& ti, uint32_t& tj) {
    ti = (uint32_t)((sqrtf(8.f * tile + 1.f) - 1.f) * 0.5f);
    while (ti * (ti + 1) / 2 > tile) ti--;
    while ((ti + 1) * (ti + 2) / 2 <= tile) ti++;
    tj = tile - ti * (ti + 1) / 2;
    ti = __builtin_amdgcn_readfirstlane(ti);
    tj = __builtin_amdgcn_readfirstlane(tj);
}

enum { ORTHO_GRAM = 0, ORTHO_POLY = 1, ORTHO_STEP = 2, ORTHO_LAST = 3 };

// One product of a step. GRAM: A = X X^T; POLY: B = b A + c A A, whose diagonal goes to `diag`; both symmetric, so the tiles on and
// below the diagonal are computed and written twice. KG groups of waves share a stage's inner indices. STEP: X = (a + diag) X + B X; LAST: the same into `out`.
template <bool SPLIT, int MT, int NT, int WM, int WN, int KG, int SF, int ST, int KIND>
__global__ __launch_bounds__(64 * WM * WN * KG, 2) void ortho_tile(OrthoArgs a) {
    using T = _Float16;
    constexpr int NW = WM * WN * KG, FS = SF / KG, BM = WM * MT * 32, BN = WN * NT * 32, PLANES = SPLIT ? 2 : 1;
    constexpr bool SYM = KIND == ORTHO_GRAM || KIND == ORTHO_POLY;
    using ATile = RowTile<T, BM, SF, NW>;
    using BTile = std::conditional_t<SYM, RowTile<T, BN, SF, NW>, ColTile<T, BN, SF, NW, ORDER_ROWS>>;
    static_assert(!SYM || BM == BN, "square tiles");
    constexpr int PLANE = ATile::BYTES + BTile::BYTES, STAGE = PLANES * PLANE, PER = PLANES * (ATile::LOADS + BTile::LOADS), KE = ATile::KE;
    __shared__ __align__(1024) char lds[ST * STAGE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), kg = wave / (WM * WN), wm = wave % (WM * WN) / WN, wn = wave % WN;
    const uint32_t id = xcd_run(blockIdx.y * gridDim.x + blockIdx.x, gridDim.x * gridDim.y), tile = id % gridDim.x, batch = id / gridDim.x;
    uint32_t ti, tj;
    if constexpr (SYM) {
        tile_of(tile, ti, tj);
    } else {
        const uint32_t nt = (a.n + BN - 1) / BN;
        ti = tile / nt;
        tj = tile % nt;
    }
    const uint32_t row = ti * BM, col = tj * BN;
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
        const char* A = lds + from;
        const char* B = A + ATile::BYTES;
        i32x4 x[2][PLANES][MT], y[2][PLANES][NT];
        auto read = [&](int f) {
#pragma unroll
            for (int p = 0; p < PLANES; p++) {
#pragma unroll
                for (int m = 0; m < MT; m++) x[f & 1][p][m] = ATile::read(A + p * PLANE, wm * MT + m, kg * FS + f, lane);
#pragma unroll
                for (int t = 0; t < NT; t++) y[f & 1][p][t] = BTile::read(B + p * PLANE, wn * NT + t, kg * FS + f, lane);
            }
        };
        read(0);
        issue();
#pragma unroll
        for (int f = 0; f < FS; f++) {
            if (f + 1 < FS) read(f + 1);
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
        interleave<PLANES * (MT + (SYM ? 1 : 2) * NT), (SPLIT ? 3 : 1) * MT * NT, FS>();
        from = from + STAGE == ST * STAGE ? 0 : from + STAGE;
    }
    tile_wait<0>();
    if constexpr (KG == 2) {
        static_assert(BM * BN * 4 <= ST * STAGE, "the sums fit the stages");
        exchange_halves<MT, NT, WM * WN>(acc, lds, kg, wave % (WM * WN), lane);
        __syncthreads();
    }
    // 64 rows at a time through LDS: then a thread has eight values of a row, of the tile and of the mirrored one
    constexpr int PITCH = BN + 1, ITEMS = 64 * BN / 8 / (64 * NW), OWN = 64 / 32; // OWN: blocks of 32 rows of a wave in a chunk
    static_assert(64 * PITCH * 4 <= ST * STAGE && MT % OWN == 0, "the sum fits the stages");
    float* sum = reinterpret_cast<float*>(lds);
    const int half = lane >> 5;
#pragma unroll
    for (int chunk = 0; chunk < BM / 64; chunk++) {
        const uint32_t crow = row + chunk * 64;
        if (crow >= a.m) break;
        if (wm == chunk / (MT / OWN)) {
#pragma unroll
            for (int o = 0; o < OWN; o++) {
                if (KG == 2 && (chunk % (MT / OWN) * OWN + o) / (MT / 2) != kg) continue;
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int k = 0; k < 16; k++)
                        sum[(o * 32 + result_row(k, half)) * PITCH + (wn * NT + t) * 32 + (lane & 31)] = acc[chunk % (MT / OWN) * OWN + o][t][k] * (ORTHO_DOWN * ORTHO_DOWN);
            }
        }
        __syncthreads();
#pragma unroll(KIND == ORTHO_LAST && MT > 2 ? 1 : ITEMS) // the last kind's three ways out would not fit beside the largest sums
        for (int item = 0; item < ITEMS; item++) {
            const uint32_t at = item * 64 * NW + threadIdx.x;
            if constexpr (SYM || KIND == ORTHO_STEP) {
                const uint32_t r = at / (BN / 8), c = at % (BN / 8) * 8, i = crow + r, j = col + c;
                if (i < a.m && j < (SYM ? a.mp : a.np)) {
                    float v[8];
#pragma unroll
                    for (int k = 0; k < 8; k++) v[k] = sum[r * PITCH + c + k];
                    if constexpr (SYM) {
                        if constexpr (KIND == ORTHO_POLY) {
                            ortho_poly<SPLIT>(a, gram + (uint64_t)i * a.mp + j, v);
#pragma unroll
                            for (int k = 0; k < 8; k++)
                                if (i == j + k) {
                                    a.diag[(uint64_t)batch * a.mp + i] = v[k];
                                    v[k] = 0.f;
                                }
                        }
                        put8<SPLIT>((KIND == ORTHO_GRAM ? a.gram : a.poly) + go + (uint64_t)i * a.mp + j, a.g_low, v);
                    } else {
                        const uint64_t o = xo + (uint64_t)i * a.np + j;
                        const float d = a.a + a.diag[(uint64_t)batch * a.mp + i];
                        Iterate8<SPLIT> x;
                        x.load(a, o);
#pragma unroll
                        for (int k = 0; k < 8; k++) v[k] = __builtin_fmaf(d, x[k], v[k]);
                        put_iterate8<SPLIT>(a, o, v);
                    }
                }
                if constexpr (SYM) {
                    const uint32_t mr = at / 8, mc = at % 8 * 8, mj = col + mr, mi = crow + mc;
                    if (ti != tj && mj < a.m && mi < a.mp) {
                        float v[8];
#pragma unroll
                        for (int k = 0; k < 8; k++) v[k] = sum[(mc + k) * PITCH + mr];
                        if constexpr (KIND == ORTHO_POLY) ortho_poly<SPLIT>(a, gram + (uint64_t)mj * a.mp + mi, v);
                        put8<SPLIT>((KIND == ORTHO_GRAM ? a.gram : a.poly) + go + (uint64_t)mj * a.mp + mi, a.g_low, v);
                    }
                }
            } else if (a.whole_out) {
                const uint32_t r = at / (BN / 8), c = at % (BN / 8) * 8, i = crow + r, j = col + c;
                if (i < a.m && j < a.n) {
                    const uint64_t o = xo + (uint64_t)i * a.np + j, to = batch * a.out_batch + (uint64_t)i * a.out_stride + j;
                    const float d = a.a + a.diag[(uint64_t)batch * a.mp + i];
                    Iterate8<SPLIT> x;
                    x.load(a, o);
                    float v[8];
#pragma unroll
                    for (int k = 0; k < 8; k++) v[k] = a.alpha * __builtin_fmaf(d, x[k], sum[r * PITCH + c + k]);
                    add_row8(a, to, v);
                }
            } else {
                // consecutive threads along a row of `out`
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const uint32_t e = (item * 8 + k) * 64 * NW + threadIdx.x;
                    const uint32_t r = a.tall ? e % 64 : e / BN, c = a.tall ? e / 64 : e % BN, i = crow + r, j = col + c;
                    if (i >= a.m || j >= a.n) continue;
                    const uint64_t o = batch * a.out_batch + (a.tall ? (uint64_t)j * a.out_stride + i : (uint64_t)i * a.out_stride + j);
                    float v = a.alpha * __builtin_fmaf(a.a + a.diag[(uint64_t)batch * a.mp + i], iterate1<SPLIT>(a, xo + (uint64_t)i * a.np + j), sum[r * PITCH + c]);
                    if (a.beta != 0.f) v = __builtin_fmaf(a.beta, load_as_float(a.out, o, a.out_dtype), v);
                    store_from_float(a.out, o, a.out_dtype, v);
                }
            }
        }
        __syncthreads();
    }
}

// The same on tiles of 64 x 64 for matrices that larger tiles do not fill the GPU with. What counts then is the time of one tile:
// eight waves, of which four take the even and four the odd half of a stage's fragments; what the epilogue needs of memory is
// asked for before the first stage; and the sum goes through LDS, so that rows are written (and mirrored) 16 bytes a thread.
template <bool SPLIT, int KIND, bool DEEP> __global__ __launch_bounds__(512, 2) void ortho_small(OrthoArgs a) {
    using T = _Float16;
    constexpr int NW = 8, B = 64, SF = 4, AT_ONCE = DEEP ? 2 : 1, ST = DEEP ? 6 : 3, PLANES = SPLIT ? 2 : 1, PITCH = 65;
    constexpr bool SYM = KIND == ORTHO_GRAM || KIND == ORTHO_POLY;
    using ATile = RowTile<T, B, SF, NW>;
    using BTile = std::conditional_t<SYM, RowTile<T, B, SF, NW>, ColTile<T, B, SF, NW, ORDER_ROWS>>;
    constexpr int PLANE = ATile::BYTES + BTile::BYTES, STAGE = PLANES * PLANE, PER = PLANES * (ATile::LOADS + BTile::LOADS), KE = ATile::KE;
    static_assert(B * PITCH * 4 <= ST * STAGE, "the sum fits the stages");
    __shared__ __align__(1024) char lds[ST * STAGE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = wave >> 2, wm = (wave >> 1) & 1, wn = wave & 1;
    const uint32_t batch = blockIdx.y, tile = KIND == ORTHO_GRAM ? blockIdx.x / a.cuts : blockIdx.x, cut = KIND == ORTHO_GRAM ? blockIdx.x % a.cuts : 0;
    uint32_t ti, tj;
    if constexpr (SYM) {
        tile_of(tile, ti, tj);
    } else {
        const uint32_t nt = (a.n + B - 1) / B;
        ti = tile / nt;
        tj = tile % nt;
    }
    const uint32_t row = ti * B, col = tj * B;
    const uint64_t xo = (uint64_t)batch * a.m * a.np, go = (uint64_t)batch * a.m * a.mp;
    const T* h = a.h + xo;
    const T* gram = a.gram + go;
    const T* poly = a.poly + go;
    ATile ta[PLANES];
    BTile tb[PLANES];
    const uint32_t xp = a.np * (uint32_t)sizeof(T), gp = a.mp * (uint32_t)sizeof(T);
    const int mrows = (int)min((uint32_t)B, a.m - row);
#pragma unroll
    for (int p = 0; p < PLANES; p++) {
        const uint64_t hl = p * a.h_low, gl = p * a.g_low;
        if constexpr (KIND == ORTHO_GRAM) {
            ta[p].init(h + hl + (uint64_t)row * a.np + cut * a.cut_stages * KE, xp, mrows, wave, lane);
            tb[p].init(h + hl + (uint64_t)col * a.np + cut * a.cut_stages * KE, xp, (int)min((uint32_t)B, a.m - col), wave, lane);
        } else if constexpr (KIND == ORTHO_POLY) {
            ta[p].init(gram + gl + (uint64_t)row * a.mp, gp, mrows, wave, lane);
            tb[p].init(gram + gl + (uint64_t)col * a.mp, gp, (int)min((uint32_t)B, a.m - col), wave, lane);
        } else {
            ta[p].init(poly + gl + (uint64_t)row * a.mp, gp, mrows, wave, lane);
            tb[p].init(h + hl + col, xp, (int)min((uint32_t)B, a.np - col), wave, lane);
        }
    }
    // the epilogue's place: eight columns of a row (GRAM, POLY, STEP); eight values down a column or along a row (LAST)
    const uint32_t er = threadIdx.x >> 3, ec = (threadIdx.x & 7) * 8, i = row + er, j = col + ec;
    const uint32_t mi = row + ec, mj = col + er; // of the mirrored tile
    f16x8 own = {}, own_low = {}, mir = {}, mir_low = {};
    Iterate8<SPLIT> x_own;
    float diag = 0.f, xl[8] = {}, dl[8] = {};
    const bool turned = KIND == ORTHO_LAST && a.tall;
    const uint32_t lc = threadIdx.x & 63, lr = threadIdx.x >> 6; // LAST: lc along the row of `out`
    if constexpr (KIND == ORTHO_POLY) {
        if (i < a.m) {
            own = *reinterpret_cast<const f16x8*>(gram + (uint64_t)i * a.mp + j);
            if constexpr (SPLIT) own_low = *reinterpret_cast<const f16x8*>(gram + a.g_low + (uint64_t)i * a.mp + j);
        }
        if (ti != tj && mj < a.m) {
            mir = *reinterpret_cast<const f16x8*>(gram + (uint64_t)mj * a.mp + mi);
            if constexpr (SPLIT) mir_low = *reinterpret_cast<const f16x8*>(gram + a.g_low + (uint64_t)mj * a.mp + mi);
        }
    } else if constexpr (KIND == ORTHO_STEP) {
        if (i < a.m) {
            diag = a.diag[(uint64_t)batch * a.mp + i];
            x_own.load(a, xo + (uint64_t)i * a.np + j);
        }
    } else if constexpr (KIND == ORTHO_LAST) {
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const uint32_t r = row + (turned ? lc : lr + 8 * k), c = col + (turned ? lr + 8 * k : lc);
            if (r < a.m) {
                dl[k] = a.diag[(uint64_t)batch * a.mp + r];
                xl[k] = iterate1<SPLIT>(a, xo + (uint64_t)r * a.np + c);
            }
        }
    }
    const int inner = (int)(KIND == ORTHO_GRAM ? a.np : a.mp);
    const int all = (inner + KE - 1) / KE, stage0 = (int)(cut * a.cut_stages), stages = KIND == ORTHO_GRAM ? min(all - stage0, (int)a.cut_stages) : all;
    const uint32_t base = lds_address(lds);
    int left = min(inner - stage0 * KE, stages * KE); // of this part
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
    for (int s = 0; s < ST - AT_ONCE; s++) issue();
    f32x16 acc[2] = {}; // even and odd fragments: two chains
    uint32_t from = 0;
    for (int s = 0; s < stages; s += AT_ONCE) {
        tile_wait<(ST - 2 * AT_ONCE) * PER>();
        i32x4 x[AT_ONCE][2][PLANES], y[AT_ONCE][2][PLANES];
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++) {
            const char* A = lds + from + u * STAGE;
            const char* Bt = A + ATile::BYTES;
#pragma unroll
            for (int f = 0; f < 2; f++)
#pragma unroll
                for (int p = 0; p < PLANES; p++) {
                    x[u][f][p] = ATile::read(A + p * PLANE, wm, group * 2 + f, lane);
                    y[u][f][p] = BTile::read(Bt + p * PLANE, wn, group * 2 + f, lane);
                }
        }
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++) issue();
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++)
#pragma unroll
            for (int f = 0; f < 2; f++) {
                if constexpr (SPLIT) {
                    acc[f] = mfma_step<T>(x[u][f][1], y[u][f][0], acc[f]);
                    acc[f] = mfma_step<T>(x[u][f][0], y[u][f][1], acc[f]);
                }
                acc[f] = mfma_step<T>(x[u][f][0], y[u][f][0], acc[f]);
            }
        from = from + AT_ONCE * STAGE == ST * STAGE ? 0 : from + AT_ONCE * STAGE;
    }
    tile_wait<0>();
    float* sum = reinterpret_cast<float*>(lds);
    const int half = lane >> 5;
#pragma unroll
    for (int g = 1; g >= 0; g--) {
        if (group == g) {
#pragma unroll
            for (int k = 0; k < 16; k++) {
                float* at = sum + (wm * 32 + result_row(k, half)) * PITCH + wn * 32 + (lane & 31);
                const float v = acc[0][k] + acc[1][k];
                *at = g ? v : (*at + v) * (ORTHO_DOWN * ORTHO_DOWN);
            }
        }
        __syncthreads();
    }
    if constexpr (KIND == ORTHO_GRAM) {
        if (a.cuts > 1) {
            float* to = a.cut + (((uint64_t)batch * gridDim.x + blockIdx.x) * B + er) * B + ec;
            f32x4 v[2];
#pragma unroll
            for (int k = 0; k < 8; k++) v[k >> 2][k & 3] = sum[er * PITCH + ec + k];
            *reinterpret_cast<f32x4*>(to) = v[0];
            *reinterpret_cast<f32x4*>(to + 4) = v[1];
            return;
        }
    }
    if constexpr (SYM) {
        T* to = (KIND == ORTHO_GRAM ? a.gram : a.poly) + go;
        if (i < a.m) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                v[k] = sum[er * PITCH + ec + k];
                if constexpr (KIND == ORTHO_POLY) {
                    v[k] = __builtin_fmaf(a.c, v[k], a.b * ORTHO_DOWN * ((float)own[k] + (float)own_low[k]));
                    if (i == j + k) {
                        a.diag[(uint64_t)batch * a.mp + i] = v[k];
                        v[k] = 0.f;
                    }
                }
            }
            put8<SPLIT>(to + (uint64_t)i * a.mp + j, a.g_low, v);
        }
        if (ti != tj && mj < a.m) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                v[k] = sum[(ec + k) * PITCH + er];
                if constexpr (KIND == ORTHO_POLY) v[k] = __builtin_fmaf(a.c, v[k], a.b * ORTHO_DOWN * ((float)mir[k] + (float)mir_low[k]));
            }
            put8<SPLIT>(to + (uint64_t)mj * a.mp + mi, a.g_low, v);
        }
    } else if constexpr (KIND == ORTHO_STEP) {
        if (i < a.m) {
            float v[8];
            const float d = a.a + diag;
#pragma unroll
            for (int k = 0; k < 8; k++) v[k] = __builtin_fmaf(d, x_own[k], sum[er * PITCH + ec + k]);
            put_iterate8<SPLIT>(a, xo + (uint64_t)i * a.np + j, v);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const uint32_t r = turned ? lc : lr + 8 * k, c = turned ? lr + 8 * k : lc;
            if (row + r >= a.m || col + c >= a.n) continue;
            const uint64_t o = batch * a.out_batch + (turned ? (uint64_t)(col + c) * a.out_stride + row + r : (uint64_t)(row + r) * a.out_stride + col + c);
            float v = a.alpha * __builtin_fmaf(a.a + dl[k], xl[k], sum[r * PITCH + c]);
            if (a.beta != 0.f) v = __builtin_fmaf(a.beta, load_as_float(a.out, o, a.out_dtype), v);
            store_from_float(a.out, o, a.out_dtype, v);
        }
    }
}

// A from the parts that its inner side was cut into: grid (tiles, batch).
template <bool SPLIT> __global__ __launch_bounds__(512) void ortho_join(OrthoArgs a) {
    constexpr int B = 64, PITCH = 65;
    __shared__ float sum[B * PITCH];
    uint32_t ti, tj;
    tile_of(blockIdx.x, ti, tj);
    const uint32_t er = threadIdx.x >> 3, ec = (threadIdx.x & 7) * 8, row = ti * B, col = tj * B, i = row + er, mi = row + ec, mj = col + er;
    const float* from = a.cut + (((uint64_t)blockIdx.y * gridDim.x + blockIdx.x) * a.cuts * B + er) * B + ec;
    f32x4 lo = {}, hi = {};
#pragma unroll 4
    for (uint32_t c = 0; c < a.cuts; c++) {
        lo += *reinterpret_cast<const f32x4*>(from + (uint64_t)c * B * B);
        hi += *reinterpret_cast<const f32x4*>(from + (uint64_t)c * B * B + 4);
    }
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; k++) sum[er * PITCH + ec + k] = v[k] = k < 4 ? lo[k] : hi[k - 4];
    _Float16* to = a.gram + (uint64_t)blockIdx.y * a.m * a.mp;
    if (i < a.m) put8<SPLIT>(to + (uint64_t)i * a.mp + col + ec, a.g_low, v);
    __syncthreads();
    if (ti != tj && mj < a.m) {
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = sum[(ec + k) * PITCH + er];
        put8<SPLIT>(to + (uint64_t)mj * a.mp + mi, a.g_low, v);
    }
}

// ---- a side of at most 64 ----
// All of A fits a workgroup, so a step needs no kernel of its own for A and B: a workgroup has 256 columns of X in registers (a wave 32,
// as a 32x32 result lies in its lanes, which is a fragment of the next product too), every workgroup forms the same A from the sums of
// all of them, and B from it, then its columns of (a + diag) X + B X and what they add to the next A. 256 columns and less are one
// workgroup and one launch; otherwise a launch a step, X and the sums in memory between them.
// What it costs is launches and waiting, about 3.5 us a step where one workgroup has everything, 8 us a launch otherwise (five steps, by the
// kernels above and by these: 64 x 64 68 and 27 us, 64 x 1024 95 and 55, 64 x 4096 200 and 70, 64 x 65 536 2.27 and 0.14 ms, 512 of 16 x 64
// 121 and 53 us). More than NARROW_PARTS sums of 64 x 64 are joined by a launch of their own, fewer by each workgroup (64 x 4096, sixteen: 73 us).
constexpr uint32_t NARROW = 64, NARROW_COLS = 256, NARROW_PARTS = 8;

struct NarrowArgs {
    float* x;       // [batch][slabs][8 waves][32 values][64 lanes]
    float* sums[2]; // [batch][slabs][64 x 64], of the launch before and of this one
    float* joined;  // [batch][64 x 64]: those of the launch before added up, where there are more than NARROW_PARTS
    uint32_t slabs, steps;
};

// Planes of a 64 x 64 matrix that is symmetric, or of columns of X: 64 values of a column, and what keeps sixteen lanes in different banks.
constexpr int NARROW_PITCH = 72;
// Of values that a 32x32 result's lane holds (rows from `at` on): four at a time, times 2^12, as high and low part.
template <int SIZE> __device__ inline void narrow_put(_Float16 (*planes)[SIZE], int at, const float* v) {
#pragma unroll
    for (int q = 0; q < 4; q++) {
        f16x4 hi, lo;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float x = v[4 * q + k] * ORTHO_UP;
            hi[k] = (_Float16)x;
            lo[k] = (_Float16)(x - (float)hi[k]);
        }
        *reinterpret_cast<f16x4*>(planes[0] + at + 8 * q) = hi;
        *reinterpret_cast<f16x4*>(planes[1] + at + 8 * q) = lo;
    }
}
// Fragments. Of a symmetric matrix, a row: 8 values in order, or as ORDER_BLOCKS has them.
__device__ inline i32x4 narrow_row(const _Float16* plane, int row, int f, int half) { return *reinterpret_cast<const i32x4*>(plane + row * NARROW_PITCH + f * 16 + 8 * half); }
__device__ inline i32x4 narrow_row_blocks(const _Float16* plane, int row, int f, int half) {
    const i32x2 a = *reinterpret_cast<const i32x2*>(plane + row * NARROW_PITCH + f * 16 + 4 * half);
    const i32x2 b = *reinterpret_cast<const i32x2*>(plane + row * NARROW_PITCH + f * 16 + 8 + 4 * half);
    return i32x4{a[0], a[1], b[0], b[1]};
}
// Of X: 32 rows from `row` on, 16 columns, read transposed.
__device__ inline i32x4 narrow_columns(const _Float16* plane, int row, int f, int lane) {
    i32x2 part[2];
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const _Float16* p = plane + (f * 16 + 8 * (lane >> 5) + 4 * j + ((lane & 15) >> 2)) * NARROW_PITCH + row + ((lane >> 4) & 1) * 16 + 4 * (lane & 3);
        part[j] = __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p));
    }
    return i32x4{part[0][0], part[0][1], part[1][0], part[1][1]};
}

// A thread's 32 of the 64 x 256 values of `in` or `out` from column j0 on, consecutive threads along the rows as they lie in memory:
// every second row, or where the matrix lies the other way every eighth column.
struct NarrowPlaces {
    uint32_t row, j, first, by, end; // of the first value; `first` counts on by `by`, up to `end`, from one value to the next
    bool tall, any;
    __device__ NarrowPlaces(const OrthoArgs& a, uint32_t j0, uint32_t thread) {
        tall = a.tall;
        row = tall ? thread % NARROW : thread / NARROW_COLS;
        j = tall ? thread / NARROW : thread % NARROW_COLS;
        first = tall ? j0 + j : row;
        by = tall ? 512 / NARROW : 512 / NARROW_COLS;
        end = tall ? a.n : a.m;
        any = tall ? row < a.m : j0 + j < a.n;
    }
    __device__ uint64_t offset(uint32_t j0, uint64_t stride) const { return tall ? (uint64_t)(j0 + j) * stride + row : (uint64_t)row * stride + j0 + j; }
    __device__ bool in(int k) const { return any && first + k * by < end; }
};
template <typename F> __device__ inline void narrow_read(const NarrowPlaces& p, const F* from, uint64_t at, uint64_t stride, float (&v)[32]) {
    const uint64_t step = p.by * stride;
#pragma unroll
    for (int k = 0; k < 32; k++) {
        const float x = (float)from[p.in(k) ? at : 0]; // no branch, so that all are on their way together
        v[k] = p.in(k) ? x : 0.f;
        at += step;
    }
}
__device__ inline void narrow_read(const NarrowPlaces& p, const void* from, uint64_t first, uint64_t at, uint64_t stride, uint32_t dtype, float (&v)[32]) {
    if (dtype == APOE_F32) narrow_read(p, (const float*)from + first, at, stride, v);
    else if (dtype == APOE_F16) narrow_read(p, (const _Float16*)from + first, at, stride, v);
    else narrow_read(p, (const __bf16*)from + first, at, stride, v);
}
template <typename F> __device__ inline void narrow_write(const NarrowPlaces& p, F* to, uint64_t at, uint64_t stride, const float (&v)[32]) {
    const uint64_t step = p.by * stride;
#pragma unroll
    for (int k = 0; k < 32; k++) {
        if (p.in(k)) to[at] = (F)v[k];
        at += step;
    }
}

// FIRST: from `in`, else a step on X in memory. ONE: the only workgroup of its matrix, all steps. Grid (slabs, batch).
// The three products of a fragment have sums of their own, added at the end: a third of the chain.
template <bool FIRST, bool ONE> __global__ __launch_bounds__(512) void ortho_narrow(OrthoArgs a, NarrowArgs w, bool last) {
    constexpr int STP = NARROW_COLS + 1;
    __shared__ __align__(16) _Float16 ap[2][NARROW * NARROW_PITCH], bp[2][NARROW * NARROW_PITCH], xp[2][NARROW_COLS * NARROW_PITCH];
    __shared__ float other[4 * 16 * 64];
    __shared__ __align__(16) float diag[NARROW];
    __shared__ double buf[8];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const uint32_t batch = blockIdx.y, slab0 = blockIdx.x * NARROW_COLS;
    const uint64_t slab = (uint64_t)batch * w.slabs + blockIdx.x;
    float* kept = w.x + (slab * 8 + wave) * 32 * 64 + lane;
    float x[2][16];
    const int bi = (wave & 1) * 32, bj = ((wave >> 1) & 1) * 32; // a wave's block of the 64 x 64
    auto multiply = [&](f32x16 (&acc)[3], const i32x4* l, const i32x4* r) {
        acc[0] = mfma_step<_Float16>(l[1], r[0], acc[0]);
        acc[1] = mfma_step<_Float16>(l[0], r[1], acc[1]);
        acc[2] = mfma_step<_Float16>(l[0], r[0], acc[2]);
    };
    auto total = [&](const f32x16 (&acc)[3], int k) { return (acc[0][k] + acc[1][k]) + acc[2][k]; };
    // A = X X^T over this workgroup's columns: the first four waves have it, 32 x 32 each, in `mine`
    float mine[16];
    auto gram = [&]() {
#pragma unroll
        for (int b = 0; b < 2; b++) narrow_put(xp, (wave * 32 + (lane & 31)) * NARROW_PITCH + b * 32 + 4 * half, x[b]);
        __syncthreads();
        const int frags = (int)(min(NARROW_COLS, a.n - slab0) + 15) / 16, end = min(frags, (wave >> 2) * 8 + 8);
        f32x16 acc[3] = {};
#pragma unroll 2
        for (int f = (wave >> 2) * 8; f < end; f++) {
            const i32x4 l[2] = {narrow_columns(xp[0], bi, f, lane), narrow_columns(xp[1], bi, f, lane)};
            const i32x4 r[2] = {narrow_columns(xp[0], bj, f, lane), narrow_columns(xp[1], bj, f, lane)};
            multiply(acc, l, r);
        }
        float* at = other + (wave & 3) * 16 * 64 + lane;
        if (frags > 8) {
            if (wave >> 2)
#pragma unroll
                for (int k = 0; k < 16; k++) at[k * 64] = total(acc, k);
            __syncthreads();
        }
        if (wave < 4)
#pragma unroll
            for (int k = 0; k < 16; k++) mine[k] = (total(acc, k) + (frags > 8 ? at[k * 64] : 0.f)) * (ORTHO_DOWN * ORTHO_DOWN);
    };
    auto step = [&]() { // B from A, and X
        if (wave < 4) narrow_put(ap, (bj + (lane & 31)) * NARROW_PITCH + bi + 4 * half, mine);
        __syncthreads();
        if (wave < 4) {
            f32x16 acc[3] = {};
#pragma unroll
            for (int f = 0; f < 4; f++) {
                const i32x4 l[2] = {narrow_row(ap[0], bi + (lane & 31), f, half), narrow_row(ap[1], bi + (lane & 31), f, half)};
                const i32x4 r[2] = {narrow_row(ap[0], bj + (lane & 31), f, half), narrow_row(ap[1], bj + (lane & 31), f, half)};
                multiply(acc, l, r);
            }
#pragma unroll
            for (int k = 0; k < 16; k++) {
                mine[k] = __builtin_fmaf(a.c, total(acc, k) * (ORTHO_DOWN * ORTHO_DOWN), a.b * mine[k]);
                if (bi + result_row(k, half) == bj + (lane & 31)) {
                    diag[bj + (lane & 31)] = mine[k];
                    mine[k] = 0.f;
                }
            }
            narrow_put(bp, (bj + (lane & 31)) * NARROW_PITCH + bi + 4 * half, mine);
        }
        __syncthreads();
        f32x16 acc[2][3] = {};
#pragma unroll
        for (int f = 0; f < 4; f++) {
            f16x8 hi, lo; // X's fragment is eight of the lane's own values
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float v = x[f / 2][f % 2 * 8 + j] * ORTHO_UP;
                hi[j] = (_Float16)v;
                lo[j] = (_Float16)(v - (float)hi[j]);
            }
            const i32x4 r[2] = {__builtin_bit_cast(i32x4, hi), __builtin_bit_cast(i32x4, lo)};
#pragma unroll
            for (int b = 0; b < 2; b++) {
                const i32x4 l[2] = {narrow_row_blocks(bp[0], b * 32 + (lane & 31), f, half), narrow_row_blocks(bp[1], b * 32 + (lane & 31), f, half)};
                multiply(acc[b], l, r);
            }
        }
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int i = 0; i < 16; i++) x[b][i] = __builtin_fmaf(a.a + diag[b * 32 + result_row(i, half)], x[b][i], total(acc[b], i) * (ORTHO_DOWN * ORTHO_DOWN));
    };
    // 256 columns of `in` or `out` pass through LDS, so that consecutive threads are along their rows whichever way they lie
    float* stage = reinterpret_cast<float*>(&xp[0][0]);
    static_assert(NARROW * STP * 4 <= sizeof(xp), "fp32 in the planes' place");
    auto staged = [&](int b, int i) -> float& { return stage[(b * 32 + result_row(i, half)) * STP + wave * 32 + (lane & 31)]; };
    auto stage_at = [&](const NarrowPlaces& p, int k) -> float& { return stage[p.row * STP + p.j + k * (p.tall ? 512 / NARROW : 512 / NARROW_COLS * STP)]; };
    float v[32];
    if constexpr (FIRST) {
        const NarrowPlaces places(a, slab0, threadIdx.x);
        narrow_read(places, a.in, batch * a.in_batch, places.offset(slab0, a.in_stride), a.in_stride, a.in_dtype, v);
        double s = 0;
#pragma unroll
        for (int k = 0; k < 32; k++) {
            stage_at(places, k) = v[k];
            if constexpr (ONE) s += (double)v[k] * (double)v[k];
        }
        double inv;
        if constexpr (ONE) {
            for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
            if (lane == 0) buf[wave] = s;
            __syncthreads();
            const double norm = sqrt(((buf[0] + buf[1]) + (buf[2] + buf[3])) + ((buf[4] + buf[5]) + (buf[6] + buf[7])));
            inv = norm == 0. ? 0. : 1. / norm;
        } else {
            inv = ortho_inverse(a, batch, buf); // which waits for all threads
        }
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int i = 0; i < 16; i++) x[b][i] = (float)(staged(b, i) * inv);
        __syncthreads();
        if constexpr (ONE)
            for (uint32_t k = 0; k < w.steps; k++) {
                gram();
                step();
            }
    } else {
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int i = 0; i < 16; i++) x[b][i] = kept[(b * 16 + i) * 64];
        const uint32_t parts = w.slabs > NARROW_PARTS ? 1 : w.slabs;
        const float* from = (parts == 1 ? w.joined : w.sums[0]) + (uint64_t)batch * parts * NARROW * NARROW;
        if (wave < 4) {
#pragma unroll
            for (int k = 0; k < 16; k++) mine[k] = 0.f;
#pragma unroll 2
            for (uint32_t g = 0; g < parts; g++)
#pragma unroll
                for (int k = 0; k < 16; k++) mine[k] += from[(uint64_t)g * NARROW * NARROW + (bi + result_row(k, half)) * NARROW + bj + (lane & 31)];
        }
        step();
    }
    if constexpr (!ONE) {
        if (!last) {
#pragma unroll
            for (int b = 0; b < 2; b++)
#pragma unroll
                for (int i = 0; i < 16; i++) kept[(b * 16 + i) * 64] = x[b][i];
            gram();
            if (wave < 4)
#pragma unroll
                for (int k = 0; k < 16; k++) w.sums[1][slab * NARROW * NARROW + (bi + result_row(k, half)) * NARROW + bj + (lane & 31)] = mine[k];
            return;
        }
    }
    __syncthreads();
#pragma unroll
    for (int b = 0; b < 2; b++)
#pragma unroll
        for (int i = 0; i < 16; i++) staged(b, i) = a.alpha * x[b][i];
    __syncthreads();
    uint32_t thread = threadIdx.x;
    asm volatile("" : "+v"(thread)); // places are worked out anew: kept since the reading, they would not leave room for the steps
    const NarrowPlaces places(a, slab0, thread);
    const uint64_t first = batch * a.out_batch, to = places.offset(slab0, a.out_stride);
    if (a.beta != 0.f) narrow_read(places, a.out, first, to, a.out_stride, a.out_dtype, v);
#pragma unroll
    for (int k = 0; k < 32; k++) {
        const float own = stage_at(places, k);
        v[k] = a.beta != 0.f ? __builtin_fmaf(a.beta, v[k], own) : own;
    }
    if (a.out_dtype == APOE_F32) narrow_write(places, (float*)a.out + first, to, a.out_stride, v);
    else if (a.out_dtype == APOE_F16) narrow_write(places, (_Float16*)a.out + first, to, a.out_stride, v);
    else narrow_write(places, (__bf16*)a.out + first, to, a.out_stride, v);
}

// The sums of many workgroups, added up: grid (16, batch), four groups of waves that take every fourth of 256 values' sums.
__global__ __launch_bounds__(1024) void ortho_narrow_join(NarrowArgs w) {
    __shared__ float part[4][256];
    const uint32_t value = threadIdx.x & 255, group = threadIdx.x >> 8, at = blockIdx.x * 256 + value;
    const float* from = w.sums[0] + (uint64_t)blockIdx.y * w.slabs * NARROW * NARROW + at;
    float v = 0.f;
#pragma unroll 8
    for (uint32_t g = group; g < w.slabs; g += 4) v += from[(uint64_t)g * NARROW * NARROW];
    part[group][value] = v;
    __syncthreads();
    if (group == 0) w.joined[blockIdx.y * NARROW * NARROW + at] = (part[0][value] + part[1][value]) + (part[2][value] + part[3][value]);
}

static OrthoArgs ortho_args(const apoe_orthogonalize_args* p) {
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
    a.parts = std::min<uint32_t>(ORTHO_PARTS, (p->rows + 3) / 4);
    return a;
}

// Rows of `in` are multiples of 16 bytes.
static bool whole_rows(const apoe_orthogonalize_args* p, const OrthoArgs& a) {
    const uint32_t v = p->in_dtype == APOE_F32 ? 4 : 8;
    return p->cols % v == 0 && a.in_stride % v == 0 && (p->batch == 1 || a.in_batch % v == 0) && ((uintptr_t)a.in & 15) == 0;
}

// A short side of up to 64.
static int run_narrow(apoe_ctx* ctx, const apoe_orthogonalize_args* p) {
    OrthoArgs a = ortho_args(p);
    NarrowArgs w{};
    w.slabs = (a.n + NARROW_COLS - 1) / NARROW_COLS;
    w.steps = p->steps;
    const dim3 grid(w.slabs, p->batch);
    hipStream_t s = ctx->stream;
    if (w.slabs == 1) {
        ortho_narrow<true, true><<<grid, 512, 0, s>>>(a, w, true);
        APOE_HIP(hipGetLastError());
        return APOE_OK;
    }
    const size_t part = (size_t)p->batch * ORTHO_PARTS * 8, x = (size_t)p->batch * w.slabs * NARROW * NARROW_COLS * 4, sums = (size_t)p->batch * w.slabs * NARROW * NARROW * 4;
    char* ws = nullptr;
    APOE_TRY(ctx->adapt_workspace(part + x + 2 * sums + (size_t)p->batch * NARROW * NARROW * 4, &ws));
    a.part = (double*)ws;
    w.x = (float*)(ws + part);
    w.sums[0] = (float*)(ws + part + x + sums);
    w.sums[1] = (float*)(ws + part + x);
    w.joined = (float*)(ws + part + x + 2 * sums);
    if (whole_rows(p, a)) ortho_squares<true><<<dim3(a.parts, p->batch), 256, 0, s>>>(a);
    else ortho_squares<false><<<dim3(a.parts, p->batch), 256, 0, s>>>(a);
    ortho_narrow<true, false><<<grid, 512, 0, s>>>(a, w, false);
    for (uint32_t i = 0; i < p->steps; i++) {
        std::swap(w.sums[0], w.sums[1]);
        if (w.slabs > NARROW_PARTS) ortho_narrow_join<<<dim3(NARROW * NARROW / 256, p->batch), 1024, 0, s>>>(w);
        ortho_narrow<false, false><<<grid, 512, 0, s>>>(a, w, i + 1 == p->steps);
    }
    APOE_HIP(hipGetLastError());
    return APOE_OK;
}

template <bool SPLIT> static int run_ortho(apoe_ctx* ctx, const apoe_orthogonalize_args* p) {
    OrthoArgs a = ortho_args(p);
    const uint32_t batch = p->batch;
    size_t bytes = 0;
    auto take = [&](size_t b) {
        const size_t at = bytes;
        bytes += (b + 1023) / 1024 * 1024;
        return at;
    };
    const size_t xs = (size_t)batch * a.m * a.np, gs = (size_t)batch * a.m * a.mp;
    const size_t o_part = take((size_t)batch * ORTHO_PARTS * 8), o_diag = take((size_t)batch * a.mp * 4), o_x = take(SPLIT ? xs * 4 : 0);
    constexpr int PLANES = SPLIT ? 2 : 1;
    a.h_low = (xs + 511) / 512 * 512;
    a.g_low = (gs + 511) / 512 * 512;
    const uint32_t cus = (uint32_t)ctx->num_cus;
    auto tiles = [](uint32_t side, uint32_t t) { return (side + t - 1) / t; };
    auto triangle = [](uint32_t t) { return t * (t + 1) / 2; };
    // X X^T on tiles of 64 that leave CUs idle: its inner side is cut, and what the cuts give is joined by a launch of its own. 1024 values
    // a cut at least, no more workgroups than CUs (the whole, fp16: 128 x 4096 103 us for 141, 128 x 16 384 136 for 382, 512 x 4096 142 for
    // 173; twice the CUs: 4 x 512 x 4096 263 for 245).
    const uint64_t g64 = (uint64_t)triangle(tiles(a.m, 64)) * batch;
    const uint32_t stages = a.np / 64;
    a.cuts = std::max(1u, std::min((uint32_t)(cus / g64), stages / 16));
    a.cut_stages = (stages + a.cuts - 1) / a.cuts;
    a.cuts = (stages + a.cut_stages - 1) / a.cut_stages;
    const size_t o_cut = take(a.cuts > 1 ? g64 * a.cuts * 64 * 64 * 4 : 0);
    const size_t o_h = take(2 * a.h_low * 2), o_h2 = take(2 * a.h_low * 2), o_gram = take(PLANES * a.g_low * 2), o_poly = take(PLANES * a.g_low * 2);
    char* ws = nullptr;
    APOE_TRY(ctx->adapt_workspace(bytes, &ws));
    a.part = (double*)(ws + o_part);
    a.diag = (float*)(ws + o_diag);
    a.x = (float*)(ws + o_x);
    a.h = (_Float16*)(ws + o_h);
    a.h2 = (_Float16*)(ws + o_h2);
    a.gram = (_Float16*)(ws + o_gram);
    a.poly = (_Float16*)(ws + o_poly);
    a.cut = (float*)(ws + o_cut);
    hipStream_t s = ctx->stream;
    const bool whole = whole_rows(p, a);
    a.whole_out = !a.tall && p->cols % 8 == 0 && a.out_stride % 8 == 0 && (batch == 1 || a.out_batch % 8 == 0) && ((uintptr_t)a.out & 15) == 0;
    if (whole) ortho_squares<true><<<dim3(a.parts, batch), 256, 0, s>>>(a);
    else ortho_squares<false><<<dim3(a.parts, batch), 256, 0, s>>>(a);
    if (whole && !a.tall) {
        const uint32_t per = a.np / 8; // at least one row at once, at most all of them
        const uint32_t blocks = std::max((per + 255) / 256, std::min((uint32_t)(((uint64_t)a.m * per + 255) / 256), std::max(1u, 2048 / batch)));
        ortho_first_whole<SPLIT><<<dim3(blocks, batch), 256, 0, s>>>(a);
    } else {
        ortho_first<SPLIT><<<dim3(a.np / 64, (a.m + 63) / 64, batch), 256, 0, s>>>(a);
    }
    // Tiles, by how many there are for the CUs (times of one product or of the whole, 256 CUs, fp16):
    //  symmetric products from half as many tiles of 256 as CUs on: 256, or 192 on twelve waves where the rounds over the CUs times a
    //    tile's size (and a seventh, which the smaller one is slower by) are less (4096 x 4096: 253 tiles of 192 for 136 of 256, X X^T 84 us
    //    for 106, the whole 1.53 ms for 1.80; 4608: 300 for 171, 2.86 ms for 2.62)
    //  128: from as many tiles as CUs on; from half as many where the inner side is long enough, there with the waves in two groups that take
    //    half of a stage each: larger pieces a wave, fewer reads (X X^T of 4 x 1024 x 4096: 45 us in the run of the whole, 51 with one group, 53 on
    //    tiles of 64). From 512 on (the whole, with them and on tiles of 64: 25 x 300 x 400 165 us for 153, 14 x 500 x 600 192 for 206, 5 x 900 x 1300
    //    284 for 328, 2500 x 2500 546 for 714; SPLIT 281 for 268, 370 for 392, 590 for 649, 1282 for 1584)
    //  64: below (1024 x 1024: X X^T 9 us; 128: 12)
    //  B X: 256 where those fill the GPU and the inner side is long enough to hide the end of a tile, whose traffic the next one does not
    //    overlap (the whole: 4096 x 8192 2.62 ms for 2.98, 8192 x 8192 11.0 for 12.4; 4 x 1024 x 4096 0.575 for 0.541), 128, 64
    const uint64_t s256 = (uint64_t)triangle(tiles(a.m, 256)) * batch, s192 = (uint64_t)triangle(tiles(a.m, 192)) * batch, s128 = (uint64_t)triangle(tiles(a.m, 128)) * batch, x256 = (uint64_t)tiles(a.m, 256) * tiles(a.n, 256) * batch, x128 = (uint64_t)tiles(a.m, 128) * tiles(a.n, 128) * batch;
    auto rounds = [&](uint64_t t) { return (t + cus - 1) / cus; };
    // tiles of 64: where a workgroup has its CU to itself, six stages and two of them at a time (1024 x 1024: 120 us for 126; 768 x 3000, where two
    // share one, 204 for 184); not SPLIT, whose stages are twice the size (777 x 1001: 201 for 174)
    auto small = [&](auto kind, uint32_t grid) {
        constexpr int K = decltype(kind)::value;
        if constexpr (!SPLIT) {
            if ((uint64_t)grid * batch <= cus) {
                ortho_small<SPLIT, K, true><<<dim3(grid, batch), 512, 0, s>>>(a);
                return;
            }
        }
        ortho_small<SPLIT, K, false><<<dim3(grid, batch), 512, 0, s>>>(a);
    };
    auto sym = [&](auto kind) {
        constexpr int K = decltype(kind)::value;
        const uint32_t inner = K == ORTHO_GRAM ? a.n : a.m;
        if constexpr (!SPLIT) {
            if (s256 >= cus / 2) {
                if (rounds(s192) * 36864 * 23 / 20 < rounds(s256) * 65536) ortho_tile<SPLIT, 2, 3, 3, 2, 2, 4, 3, K><<<dim3(triangle(tiles(a.m, 192)), batch), 768, 0, s>>>(a);
                else ortho_tile<SPLIT, 4, 2, 2, 4, 1, 4, 2, K><<<dim3(triangle(tiles(a.m, 256)), batch), 512, 0, s>>>(a);
                return;
            }
        }
        if (s128 < cus && s128 >= cus / 2 && inner >= 512) ortho_tile<SPLIT, 2, 2, 2, 2, 2, SPLIT ? 2 : 4, 4, K><<<dim3(triangle(tiles(a.m, 128)), batch), 512, 0, s>>>(a);
        else if (s128 >= cus) ortho_tile<SPLIT, 2, 1, 2, 4, 1, 4, 2, K><<<dim3(triangle(tiles(a.m, 128)), batch), 512, 0, s>>>(a);
        else {
            small(kind, triangle(tiles(a.m, 64)) * (K == ORTHO_GRAM ? a.cuts : 1));
            if (K == ORTHO_GRAM && a.cuts > 1) ortho_join<SPLIT><<<dim3(triangle(tiles(a.m, 64)), batch), 512, 0, s>>>(a);
        }
    };
    auto step = [&](auto kind) {
        constexpr int K = decltype(kind)::value;
        if constexpr (!SPLIT) {
            if (x256 >= cus * 4 / 5 && a.m >= 2048) {
                ortho_tile<SPLIT, 4, 2, 2, 4, 1, 4, 2, K><<<dim3(tiles(a.m, 256) * tiles(a.n, 256), batch), 512, 0, s>>>(a);
                return;
            }
        }
        if (x128 >= cus) ortho_tile<SPLIT, 2, 1, 2, 4, 1, 4, 2, K><<<dim3(tiles(a.m, 128) * tiles(a.n, 128), batch), 512, 0, s>>>(a);
        else small(kind, tiles(a.m, 64) * tiles(a.n, 64));
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
    if (std::min(p->rows, p->cols) <= NARROW) return run_narrow(ctx, p); // in fp16 products the roundings would not average (2 x 3: 0.8 % off)
    const bool split = p->products == APOE_F32;
    return split ? run_ortho<true>(ctx, p) : run_ortho<false>(ctx, p);
}

} // namespace apoe
