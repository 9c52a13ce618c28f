// Softmax cross entropy of queries over the rows of a table (documents, passages, terms), without the logits, and its gradients.
//
//   s_ij = scale <q_i, x_j> over the live rows j,  lse_i = log sum_j exp(s_ij),  W_i = sum_t w_it over query i's live targets
//   loss_i = W_i lse_i - sum_t w_it s_it,   G_ij = weight_i scale (W_i exp(s_ij - lse_i) - w_ij),   grad q = G x,   grad x = G^T q
//
// The rows are taken in pieces. loss_tile multiplies rows with queries (rows on the M side, so that a lane holds one query and
// its maximum and sum are taken in registers), and each 128 rows x query give a reference exponent and a sum: base 2, and the
// reference is the maximum rounded up to a whole number, so that going over to another reference is exact. For gradients the
// tile's exponentials are rounded to the rows' type and written as 32x32 blocks in the order that a lane has them, which is a
// fragment of the next product; a piece of them is at most LOSS_PIECE_BYTES.
//   grad q (for 16 bits: alone): one pass. A piece's exponentials (relative to their own references) are multiplied with the piece's rows at
//     once; what the references lack to the common one goes into the exponents of the fragments on their way to the product.
//   grad x: the normalised G is needed. Where one piece holds everything its 16-bit exponentials are brought to G in place (a pass
//     over memory: 38 us for 2048 x 30 522, forming the logits again 130 us); otherwise the logits are formed again once lse is known.
// The targets' own terms are not left to the rounded blocks: their places are zeroed (or rewritten) and W p_t - w_t, which
// nearly cancels for a query that is served well, is formed in 32 bits.
// Exponentials (or G) in 16 bits are what the 16-bit products take; a second part of each would double the gradients' products. What it costs, against a
// gradient formed in 32 bits and rounded once: nothing in the queries' gradient (0.00166 and 0.00166 at 4096 x 4096 bf16), where the other rows' roundings
// average, the second one of G (its exponentials were rounded before) too, and what the targets' would do is added in 32 bits (loss_targets); in the
// rows' gradients, where a rounded target is most of a row, 1.25 times at 4096 x 4096 (0.00206 for 0.00166), 1.5 times for 100 queries of 4000 rows.
#include "apoe_internal.h"
#include "apoe_tile.h"

namespace apoe {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr uint32_t LOSS_GROUP = 128;               // rows that share a reference
// Of exponentials (or of G) that exist at a time. Each piece reads and writes the queries' partial sums once more: 1024 queries x 1 M
// rows take 5.17 ms with pieces of 256 MiB, 4.82 ms with 1 GiB.
constexpr size_t LOSS_PIECE_BYTES = 1u << 30;
constexpr uint32_t LOSS_MAX_COLUMNS = APOE_LOSS_MAX_DIM;
constexpr uint32_t LOSS_CHUNKS = 64;               // parts that the join of the sums is split into, at most

// What the tiles are made of: the type itself, or for float two fp16 planes, a value (times a power of two) rounded and what that
// left: 22 bits, and a product is three, high x high, high x low, low x high (fp32 products on the matrix cores are 16 times as long).
template <typename T> struct Tiles {
    using S = T;
    static constexpr int PLANES = 1;
};
template <> struct Tiles<float> {
    using S = _Float16;
    static constexpr int PLANES = 2;
};
// G and the queries that it is multiplied with for grad x. fp16 planes hold what is within 2^-38 of the largest of their group, which
// a sum over rows does not miss; a row of grad x has a sum of its own, however small, so float takes three bf16 planes: 24 bits at any
// size, and a product is six.
template <typename T> struct GradTiles : Tiles<T> {};
template <> struct GradTiles<float> {
    using S = __bf16;
    static constexpr int PLANES = 3;
};

// ---- blocks of 32 queries x 32 rows ----
// Part p (16 bytes a lane) holds values 8 p .. 8 p + 7 of a lane's 16; half 1 is turned by four lanes and odd parts by eight, so that
// the transposed read finds halves and parts in different banks.
constexpr int BLOCK_BYTES = 2048, BLOCK_PARTS = 2;
__device__ inline int block_slot(int query, int half, int part) { return half * 32 + (query ^ (half * 4) ^ (part * 8)); }
__device__ inline uint32_t block_place(int query, int row) { // byte offset of one value
    const int half = (row >> 2) & 1, i = ((row >> 3) << 2) | (row & 3);
    return (uint32_t)((i >> 3) * 1024 + block_slot(query, half, i >> 3) * 16 + (i & 7) * 2);
}

// Words that no kernel writes while one reads them, at a place that is the same in the wave: a scalar load, which does not wait
// for the loads into LDS as a vector load's result would.
using UniformWords = const __attribute__((address_space(4))) uint32_t*;

// Live rows among 32 from `row` on, the same row in the whole wave.
__device__ inline uint32_t live_word(const uint32_t* live, uint32_t row, uint32_t n) {
    if (row >= n) return 0;
    uint32_t w = live ? ((UniformWords)live)[row >> 5] : ~0u;
    if (n - row < 32) w &= (1u << (n - row)) - 1u;
    return w;
}

struct LossArgs {
    const void* q;
    const void* rows;
    uint32_t q_pitch, r_pitch; // bytes
    uint32_t nq, n, dim, qp;   // qp: queries rounded up to whole tiles
    const uint32_t *t_off, *t_idx;
    const float* t_val;
    const uint32_t* live;
    const float* weight;
    float scale;
    // one piece
    uint32_t row0, row_tiles, q_tiles, row_blocks; // first row, tiles of either side, blocks of 32 rows (the pitch of `blocks`)
    // workspace
    float *ref, *sum;           // [n / LOSS_GROUP][qp]
    float* block_ref;           // the same for the blocks: `ref` itself, or with planes of the exponentials times the rows' powers of two
    // the tiles' operands: rows and q themselves, or (float) planes of this piece's rows and of q, whose low parts lie *_low bytes behind
    const char *tile_rows, *tile_q;
    uint32_t tile_row0, tile_r_pitch, tile_q_pitch, tile_dim; // the first row at tile_rows; bytes; columns with the pad
    uint64_t tile_r_low, tile_q_low, block_low;
    const char* grad_tile_q;    // q as grad x takes it, over the queries' powers of two (fp16), or in planes tile_q_low bytes apart (float)
    uint32_t grad_tile_q_pitch; // bytes
    float *row_exp, *q_exp;     // planes: exponents of each row and of each query
    float *chunk_ref, *chunk_sum; // [LOSS_CHUNKS][qp]
    float2* lse_w;              // [qp]: lse in base 2, weight W (to be multiplied with exp(s - lse))
    float *coef, *total;        // [qp]: |weight| (|W| + sum |w|); W
    uint32_t *top_coef, *q_on;  // the largest of them, as bits; those that are not zero, as a bit mask
    float* q_size;              // [qp], for fp16: each query's largest value over its power of two (grad_scale)
    uint32_t* top_size;         // the largest of them, as bits
    float *peak, *part_of_two;  // [qp]: the largest |weight w| of a query's targets; what brings the largest of all to a power of two (grad_scale)
    char* blocks;
    float* part;                // [splits][qp][dim]
    float* fix;                 // [qp][dim], with G: the targets' terms that rounding took out of G; behind the last split
    float* part_ref[2];         // [splits][qp]
    float *loss, *lse;
    void *grad_q, *grad_x;
    uint32_t gq_pitch, gx_pitch;
    uint32_t groups, chunks, splits;
};

// fp16 holds 30 binades of normal numbers, half of them above one: the largest exponential of a group is brought up to 2^14, so
// that 28 binades stay below it. A query that is served well needs them: its target is the largest, and the gradient is what the
// others, far below, leave.
template <typename T> constexpr float HEADROOM = __is_same(T, __bf16) ? 0.f : 14.f;

enum { TILE_SUMS = 0, TILE_EXP = 1, TILE_GRAD = 2 };

// What a query's coefficients are taken times in G: near 2^13 at most. First a power of two: fp16, whose numbers would not reach from the largest of
// all queries to what a light one leaves at each row, takes one a query: it is taken out again where the query's own gradient is written, and for the
// rows' gradients put into the query, times a power of two that is the same for all (scale_of_sizes); the others take that of the largest of all. Then a
// factor of a half to one, the same for all, under which the heaviest target's weight is a power of two: with equal weights, the usual case, a
// rounded target loses what its row's probability is and not also the weight's own bits, which are the same for all targets and would not average.
template <typename T> constexpr bool OWN_SCALE = __is_same(T, _Float16);
template <typename T> __device__ inline float grad_power(const LossArgs& a, uint32_t qi) {
    const float t = OWN_SCALE<T> ? a.coef[qi] : __uint_as_float(*a.top_coef);
    return t > 0.f && t < 1e30f && t > 1e-30f ? exp2f(13.f - ceilf(log2f(t))) : 1.f;
}
template <typename T> __device__ inline float grad_scale(const LossArgs& a, uint32_t qi) { return grad_power<T>(a, qi) * *a.part_of_two; }
// Exponent that brings the largest of q_size to 2^13 .. 2^14.
__device__ inline int scale_of_sizes(const LossArgs& a) {
    const float t = __uint_as_float(*a.top_size);
    int e = 14;
    if (t > 0.f) (void)frexpf(t, &e);
    return 14 - e;
}

// A value as a sum of P values of type S.
template <typename S, int P> __device__ inline void split(float v, S* out) {
#pragma unroll
    for (int p = 0; p < P; p++) {
        out[p] = (S)v;
        v -= (float)out[p];
    }
}

// Eight values of a block (16 bytes of a lane's), and one; the planes lie `low` bytes apart. W: Tiles or GradTiles.
template <typename W> __device__ inline void put_block(char* at, uint64_t low, const float* v) {
    using S = typename W::S;
    typedef S s8 __attribute__((ext_vector_type(8)));
    s8 planes[W::PLANES];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        S x[W::PLANES];
        split<S, W::PLANES>(v[i], x);
#pragma unroll
        for (int p = 0; p < W::PLANES; p++) planes[p][i] = x[p];
    }
#pragma unroll
    for (int p = 0; p < W::PLANES; p++) *reinterpret_cast<s8*>(at + p * low) = planes[p];
}
template <typename W> __device__ inline void put_value(char* at, uint64_t low, float v) {
    typename W::S x[W::PLANES];
    split<typename W::S, W::PLANES>(v, x);
#pragma unroll
    for (int p = 0; p < W::PLANES; p++) *reinterpret_cast<typename W::S*>(at + p * low) = x[p];
}

// The product of two fragments of one, two or three planes: the terms that the planes' bits reach, small ones first.
template <typename W> __device__ inline f32x16 multiply(const i32x4* x, const i32x4* y, f32x16 c) {
    using S = typename W::S;
#pragma unroll
    for (int order = W::PLANES - 1; order >= 0; order--)
#pragma unroll
        for (int p = 0; p <= order; p++) c = mfma_step<S>(x[p], y[order - p], c);
    return c;
}
template <typename W> constexpr int PRODUCTS = W::PLANES * (W::PLANES + 1) / 2;

// ---- planes of float matrices ----
// The power of two that brings `top` to 2^14 .. 2^15.
__device__ inline int plane_exp(float top) {
    int e = 0;
    if (top > 0.f) (void)frexpf(top, &e);
    return top > 0.f ? 15 - e : 0;
}
__device__ inline float finite_abs(float v) {
    v = fabsf(v);
    return v <= 3.402823466e38f ? v : 0.f; // not a number: zero
}
template <typename S, int P> __device__ inline void put_planes(char* at, uint64_t low, f32x4 x, int k) {
    typedef S s4 __attribute__((ext_vector_type(4)));
    s4 planes[P];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        S v[P];
        split<S, P>(ldexpf(x[i], k), v);
#pragma unroll
        for (int p = 0; p < P; p++) planes[p][i] = v[p];
    }
#pragma unroll
    for (int p = 0; p < P; p++) *reinterpret_cast<s4*>(at + p * low) = planes[p];
}

// Rows of a matrix that a wave holds between their largest value and the planes, HELD times 256 columns at most.
template <int HELD> struct HeldRow {
    f32x4 x[HELD];
    __device__ void fetch(const void* row, uint32_t dim, bool on, int lane) {
#pragma unroll
        for (int i = 0; i < HELD; i++) {
            const uint32_t d = (i * 64 + lane) * 4;
            x[i] = on && d < dim ? *reinterpret_cast<const f32x4*>((const char*)row + d * 4) : f32x4{};
        }
    }
    __device__ float top() const { // the largest magnitude, the same for all lanes
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < HELD; i++) top = fmaxf(fmaxf(fmaxf(top, finite_abs(x[i][0])), fmaxf(finite_abs(x[i][1]), finite_abs(x[i][2]))), finite_abs(x[i][3]));
#pragma unroll
        for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
        return top;
    }
    template <typename S, int P> __device__ void put(char* row, uint64_t low, uint32_t tile_dim, int k, int lane) const {
#pragma unroll
        for (int i = 0; i < HELD; i++) {
            const uint32_t d = (i * 64 + lane) * 4;
            if (d < tile_dim) put_planes<S, P>(row + d * 2, low, x[i], k);
        }
    }
};

// float to planes, each row and each query with an exponent of its own, bound by memory: 99 991 rows of 1024, 0.7 of
// them live, in 116 us (697 MB, 6.0 TB/s).
// Workgroups from row_groups on: eight queries each, the others 32 rows, four a wave. A row of zeros, left out or live, has an exponent that no other
// has: with an ordinary one it would count as larger than the rows beside it (loss_tile).
constexpr int EMPTY_EXP = 1000;
template <int HELD> __global__ __launch_bounds__(512) void loss_split(LossArgs a, uint32_t row_groups) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (blockIdx.x >= row_groups) {
        const uint32_t qi = (blockIdx.x - row_groups) * 8 + wave;
        if (qi >= a.nq) return;
        HeldRow<HELD> q;
        q.fetch((const char*)a.q + (uint64_t)qi * a.q_pitch, a.dim, true, lane);
        const int k = plane_exp(q.top());
        if (lane == 0) a.q_exp[qi] = (float)k;
        const uint64_t at = (uint64_t)qi * a.tile_q_pitch;
        q.template put<_Float16, 2>((char*)a.tile_q + at, a.tile_q_low, a.tile_dim, k, lane);
        if (a.grad_x) q.template put<__bf16, 3>((char*)a.grad_tile_q + at, a.tile_q_low, a.tile_dim, 0, lane);
        return;
    }
    const uint32_t row0 = a.row0 + blockIdx.x * 32;
    uint32_t on = 0;
    if (row0 < a.n) {
        on = a.live ? a.live[row0 >> 5] : ~0u;
        if (a.n - row0 < 32) on &= (1u << (a.n - row0)) - 1u;
    }
    constexpr int AT_ONCE = HELD <= 4 ? 4 : 1; // rows that are on their way together
    HeldRow<HELD> x[AT_ONCE];
#pragma unroll
    for (int r0 = 0; r0 < 4; r0 += AT_ONCE) {
#pragma unroll
        for (int r = 0; r < AT_ONCE; r++) {
            const uint32_t row = wave * 4 + r0 + r;
            x[r].fetch((const char*)a.rows + (uint64_t)(row0 + row) * a.r_pitch, a.dim, (on >> row) & 1, lane);
        }
#pragma unroll
        for (int r = 0; r < AT_ONCE; r++) {
            const uint32_t row = wave * 4 + r0 + r;
            const float top = x[r].top();
            const int k = plane_exp(top);
            if (lane == 0) a.row_exp[row0 + row] = (float)(top > 0.f ? k : EMPTY_EXP);
            x[r].template put<_Float16, 2>((char*)a.tile_rows + (uint64_t)(row0 + row - a.tile_row0) * a.tile_r_pitch, a.tile_r_low, a.tile_dim, k, lane);
        }
    }
}

// Rows x queries, rows on the M side: 128 rows a wave (a group), so that a query's maximum and sum over them need one exchange between a
// lane and its other half. SUMS: references and sums. EXP: the exponentials too, as blocks. GRAD: with lse known, G as blocks.
// Bound by the matrix units and the clock that they leave: 256 x 256 tiles reach 1040 TFLOP/s at 1024 queries x 65 536 fp16 rows of 1024 (zeros
// in place of data 1240, a library product of 1024 x 131 072 x 1024 1005), float (three products each) 1190 at 1024 x 100 000; over a million rows 990,
// with the matrix units busy in 47 % of the cycles, the clock at 1.9 GHz of 2.4 and 2.5 TB/s of memory traffic. Eight waves of
// 128 x 64: two a SIMD (four waves of 128 x 128: 800); reads of the next fragment between the products of this one (974 without).
template <typename T, int NT, int WM, int WN, int SF, int ST, int MODE>
__global__ __launch_bounds__(64 * WM * WN, NT > 2 ? 1 : 2) void loss_tile(LossArgs a) {
    using S = typename Tiles<T>::S;
    constexpr int NW = WM * WN, BM = WM * 128, BN = WN * NT * 32, P = Tiles<T>::PLANES;
    using ATile = RowTile<S, BM, SF, NW>;
    using BTile = RowTile<S, BN, SF, NW>;
    constexpr int PLANE = ATile::BYTES + BTile::BYTES, STAGE = P * PLANE, PER = P * (ATile::LOADS + BTile::LOADS);
    constexpr bool SCALED = P == 2 && MODE == TILE_EXP; // the exponentials take the rows' exponents
    __shared__ __align__(1024) char lds[ST * STAGE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
    // consecutive workgroups go to the eight XCDs in turn: those of one XCD share a tile of rows, one after the other
    uint32_t rt = blockIdx.x / a.q_tiles, qt = blockIdx.x % a.q_tiles;
    const uint32_t whole = a.row_tiles / 8 * 8;
    if (blockIdx.x < whole * a.q_tiles) {
        const uint32_t i = blockIdx.x >> 3;
        rt = (i / a.q_tiles) * 8 + (blockIdx.x & 7);
        qt = i % a.q_tiles;
    }
    const uint32_t row = a.row0 + rt * BM, query = qt * BN;
    ATile ta[P];
    BTile tb[P];
#pragma unroll
    for (int p = 0; p < P; p++) {
        ta[p].init(reinterpret_cast<const S*>(a.tile_rows + p * a.tile_r_low + (uint64_t)(row - a.tile_row0) * a.tile_r_pitch), a.tile_r_pitch, (int)(row < a.n ? min((uint32_t)BM, a.n - row) : 0u), wave, lane);
        tb[p].init(reinterpret_cast<const S*>(a.tile_q + p * a.tile_q_low + (uint64_t)query * a.tile_q_pitch), a.tile_q_pitch, (int)min((uint32_t)BN, a.nq - query), wave, lane);
    }
    const int bytes = (int)(a.tile_dim * 2), stages = (bytes + SF * 32 - 1) / (SF * 32);
    const uint32_t base = lds_address(lds);
    int left = bytes;
    uint32_t into = 0;
    auto issue = [&]() {
#pragma unroll
        for (int p = 0; p < P; p++) {
            ta[p].load(base + into + p * PLANE, left, wave);
            tb[p].load(base + into + p * PLANE + ATile::BYTES, left, wave);
            ta[p].next();
            tb[p].next();
        }
        left -= SF * 32;
        into = into + STAGE == ST * STAGE ? 0 : into + STAGE;
    };
#pragma unroll
    for (int s = 0; s < ST - 1; s++) issue();
    f32x16 acc[4][NT] = {};
    uint32_t from = 0;
    for (int s = 0; s < stages; s++) {
        tile_wait<(ST - 2) * PER>();
        issue();
        const char* A = lds + from;
        const char* B = A + ATile::BYTES;
        i32x4 x[2][4][P], y[2][NT][P];
        auto read = [&](int f) {
#pragma unroll
            for (int p = 0; p < P; p++) {
#pragma unroll
                for (int m = 0; m < 4; m++) x[f & 1][m][p] = ATile::read(A + p * PLANE, wm * 4 + m, f, lane);
#pragma unroll
                for (int t = 0; t < NT; t++) y[f & 1][t][p] = BTile::read(B + p * PLANE, wn * NT + t, f, lane);
            }
        };
        read(0);
#pragma unroll
        for (int f = 0; f < SF; f++) {
            if (f + 1 < SF) read(f + 1);
#pragma unroll
            for (int m = 0; m < 4; m++)
#pragma unroll
                for (int t = 0; t < NT; t++) acc[m][t] = multiply<Tiles<T>>(x[f & 1][m], y[f & 1][t], acc[m][t]);
        }
        interleave<P * (4 + NT), PRODUCTS<Tiles<T>> * 4 * NT, SF>();
        from = from + STAGE == ST * STAGE ? 0 : from + STAGE;
    }
    // epilogue: one query a lane (and its other half), 128 rows a wave
    const int h = lane >> 5;
    const uint32_t wrow = row + wm * LOSS_GROUP;
    // planes: what brings a row's sums to the exponent of the largest of the group's rows, as a lane has the rows: a factor, or (SCALED) its logarithm
    f32x4 down[P == 2 ? 4 : 1][4];
    float least = 0.f; // that row's exponent
    if constexpr (P == 2) {
        least = INFINITY;
#pragma unroll
        for (int m = 0; m < 4; m++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
                down[m][k] = *reinterpret_cast<const f32x4*>(a.row_exp + wrow + m * 32 + 8 * k + 4 * h);
                least = fminf(fminf(fminf(least, down[m][k][0]), fminf(down[m][k][1], down[m][k][2])), down[m][k][3]);
            }
        least = fminf(least, __shfl_xor(least, 32));
#pragma unroll
        for (int m = 0; m < 4; m++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const float l = least - down[m][i >> 2][i & 3];
                down[m][i >> 2][i & 3] = SCALED ? l : __builtin_amdgcn_exp2f(l);
            }
    }
    uint32_t words[4];
#pragma unroll
    for (int m = 0; m < 4; m++) words[m] = live_word(a.live, wrow + m * 32, a.n);
    const bool all = (words[0] & words[1] & words[2] & words[3]) == ~0u;
#pragma unroll
    for (int t = 0; t < NT; t++) {
        const uint32_t qi = query + (wn * NT + t) * 32 + (lane & 31);
        float c = a.scale * LOG2E; // from sums to logits in base 2
        if constexpr (P == 2) {
            c = ldexpf(c, -(int)(least + (qi < a.nq ? a.q_exp[qi] : 0.f)));
#pragma unroll
            for (int m = 0; m < 4; m++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const float d = down[m][i >> 2][i & 3];
                    acc[m][t][i] = SCALED ? ldexpf(acc[m][t][i], (int)d) : acc[m][t][i] * d;
                }
        }
        if (!all) {
#pragma unroll
            for (int m = 0; m < 4; m++) {
                const uint32_t w = words[m] >> (4 * h);
#pragma unroll
                for (int i = 0; i < 16; i++)
                    if (!((w >> (8 * (i >> 2) + (i & 3))) & 1)) acc[m][t][i] = -INFINITY;
            }
        }
        float p[16];
        char* out = a.blocks + ((size_t)(qi >> 5) * a.row_blocks + ((wrow - a.row0) >> 5)) * BLOCK_BYTES;
        if constexpr (MODE == TILE_GRAD) {
            const float2 lw = a.lse_w[qi];
            const float g = lw.y * grad_scale<T>(a, qi);
#pragma unroll
            for (int m = 0; m < 4; m++) {
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const float z = acc[m][t][i];
                    // a query that counts nothing, and a row that is left out, give zero whatever the logit is
                    p[i] = g == 0.f || z == -INFINITY ? 0.f : g * __builtin_amdgcn_exp2f(__builtin_fmaf(z, c, -lw.x));
                }
#pragma unroll
                for (int k = 0; k < BLOCK_PARTS; k++) put_block<GradTiles<T>>(out + m * BLOCK_BYTES + k * 1024 + block_slot(lane & 31, h, k) * 16, a.block_low, p + k * 8);
            }
        } else {
            float top = -INFINITY, block_top = -INFINITY;
#pragma unroll
            for (int m = 0; m < 4; m++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    top = fmaxf(top, acc[m][t][i]);
                    if constexpr (SCALED) block_top = fmaxf(block_top, __builtin_fmaf(acc[m][t][i], c, down[m][i >> 2][i & 3]));
                }
            top = fmaxf(top, __shfl_xor(top, 32));
            if (top != -INFINITY) top *= c; // -inf: all left out (and c may be zero)
            const float ref = top == -INFINITY ? -INFINITY : ceilf(top) - HEADROOM<T>;
            const float less = top == -INFINITY ? 0.f : -ref;
            float block_ref = ref, block_less = less;
            if constexpr (SCALED) {
                block_top = fmaxf(block_top, __shfl_xor(block_top, 32));
                block_ref = top == -INFINITY ? -INFINITY : ceilf(block_top) - HEADROOM<T>;
                block_less = top == -INFINITY ? 0.f : -block_ref;
            }
            float sum = 0.f;
#pragma unroll
            for (int m = 0; m < 4; m++) {
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const float z = acc[m][t][i];
                    p[i] = z == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(__builtin_fmaf(z, c, less));
                    sum += p[i];
                    if constexpr (SCALED) p[i] = z == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(__builtin_fmaf(z, c, block_less + down[m][i >> 2][i & 3]));
                }
                if constexpr (MODE == TILE_EXP) {
#pragma unroll
                    for (int k = 0; k < BLOCK_PARTS; k++) put_block<Tiles<T>>(out + m * BLOCK_BYTES + k * 1024 + block_slot(lane & 31, h, k) * 16, a.block_low, p + k * 8);
                }
            }
            sum += __shfl_xor(sum, 32);
            if (h == 0) {
                const size_t at = (size_t)(wrow / LOSS_GROUP) * a.qp + qi;
                a.ref[at] = ref;
                a.sum[at] = sum;
                if constexpr (SCALED) a.block_ref[at] = block_ref - least;
            }
        }
    }
    tile_wait<0>(); // the stages beyond the last have landed before the LDS goes to another workgroup
}

// (reference, sum) of two parts joined.
__device__ inline void join_sums(float& ref, float& sum, float r, float s) {
    const float top = fmaxf(ref, r);
    if (top == -INFINITY) {
        sum += s; // zeros, or NaN
        return;
    }
    sum = sum * __builtin_amdgcn_exp2f(ref - top) + s * __builtin_amdgcn_exp2f(r - top);
    ref = top;
}

// The groups' sums of 32 queries joined, chunk by chunk: grid (qp / 32, chunks). ZERO: the targets' places in this piece's
// exponentials are zeroed as well, by chunk 0.
template <typename T, bool ZERO> __global__ __launch_bounds__(256) void loss_join(LossArgs a, uint32_t group0, uint32_t groups, uint32_t chunk0) {
    __shared__ float sr[8][32], ss[8][32];
    const uint32_t ql = threadIdx.x & 31, gl = threadIdx.x >> 5, qi = blockIdx.x * 32 + ql;
    const uint32_t per = (groups + gridDim.y - 1) / gridDim.y, g0 = blockIdx.y * per, g1 = min(g0 + per, groups);
    float ref = -INFINITY, sum = 0.f;
    for (uint32_t g = g0 + gl; g < g1; g += 8) {
        const size_t at = (size_t)(group0 + g) * a.qp + qi;
        join_sums(ref, sum, a.ref[at], a.sum[at]);
    }
    sr[gl][ql] = ref;
    ss[gl][ql] = sum;
    __syncthreads();
    if (gl == 0) {
        for (int k = 1; k < 8; k++) join_sums(ref, sum, sr[k][ql], ss[k][ql]);
        a.chunk_ref[(chunk0 + blockIdx.y) * (size_t)a.qp + qi] = ref;
        a.chunk_sum[(chunk0 + blockIdx.y) * (size_t)a.qp + qi] = sum;
    }
    if constexpr (ZERO) {
        if (blockIdx.y == 0 && qi < a.nq && a.t_off) {
            const uint32_t end = min(a.row0 + a.row_blocks * 32, a.n);
            for (uint32_t e = a.t_off[qi] + gl; e < a.t_off[qi + 1]; e += 8) {
                const uint32_t t = a.t_idx[e];
                if (t < a.row0 || t >= end) continue;
                char* block = a.blocks + ((size_t)(qi >> 5) * a.row_blocks + ((t - a.row0) >> 5)) * BLOCK_BYTES;
                put_value<Tiles<T>>(block + block_place(ql, (t - a.row0) & 31), a.block_low, 0.f);
            }
        }
    }
}

__device__ inline bool is_live(const LossArgs& a, uint32_t t) { return t < a.n && (!a.live || ((a.live[t >> 5] >> (t & 31)) & 1)); }
__device__ inline float target_weight(const LossArgs& a, uint32_t e, uint32_t e0, uint32_t e1) { return a.t_val ? a.t_val[e] : 1.f / (float)(e1 - e0); }

// lse (base 2) of a query from the chunks, by one wave.
__device__ inline float join_chunks(const LossArgs& a, uint32_t qi, int lane) {
    float ref = -INFINITY, sum = 0.f;
    for (uint32_t k = lane; k < a.chunks; k += 64) join_sums(ref, sum, a.chunk_ref[(size_t)k * a.qp + qi], a.chunk_sum[(size_t)k * a.qp + qi]);
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        const float r = __shfl_xor(ref, d), s = __shfl_xor(sum, d);
        join_sums(ref, sum, r, s);
    }
    if (ref == -INFINITY) return sum == 0.f ? -INFINITY : sum; // no live row (or NaN)
    return ref + log2f(sum);
}

// What the second pass needs of a query, one wave each: lse, and weight W.
template <typename T> __global__ __launch_bounds__(64) void loss_coefs(LossArgs a) {
    const uint32_t qi = blockIdx.x;
    const int lane = threadIdx.x;
    if (qi >= a.nq) {
        if (lane == 0) {
            a.lse_w[qi] = make_float2(0.f, 0.f);
            a.coef[qi] = 0.f;
        }
        return;
    }
    float size = 0.f;
    if constexpr (OWN_SCALE<T>) {
        for (uint32_t d = lane * 8; d < a.dim; d += 512) {
            const f16x8 x = *reinterpret_cast<const f16x8*>((const char*)a.q + (uint64_t)qi * a.q_pitch + d * 2);
#pragma unroll
            for (int k = 0; k < 8; k++) size = fmaxf(size, finite_abs((float)x[k]));
        }
#pragma unroll
        for (int d = 32; d; d >>= 1) size = fmaxf(size, __shfl_xor(size, d));
    }
    const float lse = join_chunks(a, qi, lane);
    const uint32_t e0 = a.t_off[qi], e1 = a.t_off[qi + 1];
    float W = 0.f, A = 0.f, M = 0.f;
    for (uint32_t e = e0 + lane; e < e1; e += 64) {
        const float w = is_live(a, a.t_idx[e]) ? target_weight(a, e, e0, e1) : 0.f;
        W += w;
        A += fabsf(w);
        M = fmaxf(M, fabsf(w));
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        W += __shfl_xor(W, d);
        A += __shfl_xor(A, d);
        M = fmaxf(M, __shfl_xor(M, d));
    }
    if (lane == 0) {
        const float c = a.weight ? a.weight[qi] : 1.f;
        a.lse_w[qi] = make_float2(lse, c * W);
        a.coef[qi] = fabsf(c) * (fabsf(W) + A);
        a.total[qi] = W;
        if constexpr (OWN_SCALE<T>) a.q_size[qi] = a.coef[qi] != 0.f ? size / grad_power<T>(a, qi) : 0.f;
        a.peak[qi] = fabsf(c) * M;
    }
}

// The largest coefficient, target and (fp16) size, and which queries count something (what the others hold is not multiplied), as bits: one workgroup.
template <typename T> __global__ __launch_bounds__(1024) void loss_queries(LossArgs a) {
    constexpr int N = OWN_SCALE<T> ? 3 : 2;
    __shared__ uint32_t top[N][16];
    uint32_t most[N] = {}; // of floats that are not negative, as bits
    for (uint32_t q0 = 0; q0 < a.qp; q0 += 1024) {
        const uint32_t qi = q0 + threadIdx.x;
        const uint32_t c = qi < a.nq ? __float_as_uint(a.coef[qi]) : 0;
        most[0] = max(most[0], c);
        most[1] = max(most[1], qi < a.nq ? __float_as_uint(a.peak[qi]) : 0);
        if constexpr (N == 3) most[2] = max(most[2], qi < a.nq ? __float_as_uint(a.q_size[qi]) : 0);
        const unsigned long long b = __ballot(c != 0);
        if ((threadIdx.x & 31) == 0 && qi < a.qp) a.q_on[qi >> 5] = (uint32_t)(b >> (threadIdx.x & 32));
    }
#pragma unroll
    for (int n = 0; n < N; n++) {
#pragma unroll
        for (int d = 32; d; d >>= 1) most[n] = max(most[n], (uint32_t)__shfl_xor((int)most[n], d));
        if ((threadIdx.x & 63) == 0) top[n][threadIdx.x >> 6] = most[n];
    }
    __syncthreads();
    if (threadIdx.x < N) {
        uint32_t all = 0;
        for (int k = 0; k < 16; k++) all = max(all, top[threadIdx.x][k]);
        if (threadIdx.x == 0) *a.top_coef = all;
        if (threadIdx.x == 1) {
            const float peak = __uint_as_float(all);
            int e;
            *a.part_of_two = peak > 0.f && peak < 1e30f ? 0.5f / frexpf(peak, &e) : 1.f;
        }
        if (threadIdx.x == 2) *a.top_size = all;
    }
}

// fp16: the queries as the rows' gradients take them, one wave each. Those that count nothing are not read there.
__global__ __launch_bounds__(256) void loss_scale_queries(LossArgs a) {
    const uint32_t qi = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (qi >= a.nq || a.coef[qi] == 0.f) return;
    int own;
    (void)frexpf(grad_power<_Float16>(a, qi), &own); // 2^(own - 1)
    const int k = scale_of_sizes(a) + 1 - own;
    for (uint32_t d = (threadIdx.x & 63) * 8; d < a.dim; d += 512) {
        f16x8 x = *reinterpret_cast<const f16x8*>((const char*)a.q + (uint64_t)qi * a.q_pitch + d * 2);
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = (_Float16)ldexpf((float)x[i], k);
        *reinterpret_cast<f16x8*>((char*)a.grad_tile_q + (uint64_t)qi * a.grad_tile_q_pitch + d * 2) = x;
    }
}

// Exponentials to G in place, one wave a group of rows and 32 queries.
template <typename T> __global__ __launch_bounds__(256) void loss_normalise(LossArgs a, uint32_t groups) {
    const uint32_t wave = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    const uint32_t g = wave % groups, qb = wave / groups;
    if (qb >= a.qp / 32) return;
    char* block = a.blocks + ((size_t)qb * a.row_blocks + g * (LOSS_GROUP / 32)) * BLOCK_BYTES + lane * 16;
    constexpr int LOADS = LOSS_GROUP / 32 * BLOCK_PARTS;
    float f[2]; // of odd parts another lane's query
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const uint32_t qi = qb * 32 + (uint32_t)((int)(lane & 31) ^ ((int)(lane >> 5) * 4) ^ (k * 8)); // a slot is its own inverse within a half
        const float ref = a.ref[(size_t)(a.row0 / LOSS_GROUP + g) * a.qp + qi];
        const float2 lw = a.lse_w[qi];
        const float c = lw.y * grad_scale<T>(a, qi);
        f[k] = c == 0.f || ref == -INFINITY ? 0.f : c * __builtin_amdgcn_exp2f(ref - lw.x);
    }
    typedef T t8 __attribute__((ext_vector_type(8)));
    t8 v[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; i++) v[i] = *reinterpret_cast<const t8*>(block + i * 1024);
#pragma unroll
    for (int i = 0; i < LOADS; i++) {
        float p[8];
        const float c = f[i & 1];
#pragma unroll
        for (int k = 0; k < 8; k++) p[k] = c == 0.f ? 0.f : (float)v[i][k] * c;
        put_block<Tiles<T>>(block + i * 1024, 0, p);
    }
}

// Second pass: the targets' places in this piece's G, formed in 32 bits; one wave a query. ALL: the piece holds all rows and no
// kernel behind this one adds anything, so it writes the loss. FIX: what the places' rounding leaves of a query's targets, which are most of its
// gradient, times their rows: the queries' gradient adds it up beside the product (4096 x 4096 bf16, off by 0.00166 for 0.00210; the result's
// own rounding is 0.00166). The rows' gradients would need it by row, and go without.
template <typename T, bool ALL, bool FIX, int COLUMNS> __global__ __launch_bounds__(64) void loss_targets(LossArgs a, int first_piece) {
    constexpr int V = 16 / (int)sizeof(T), C = COLUMNS / (64 * V);
    typedef T tv __attribute__((ext_vector_type(V)));
    const uint32_t qi = blockIdx.x, end = min(a.row0 + a.row_blocks * 32, a.n);
    const int lane = threadIdx.x;
    const uint32_t e0 = a.t_off[qi], e1 = a.t_off[qi + 1];
    const float2 lw = a.lse_w[qi];
    const float gs = grad_scale<T>(a, qi), cw = a.weight ? a.weight[qi] : 1.f;
    const char* q = (const char*)a.q + (uint64_t)qi * a.q_pitch;
    float at = 0.f, fix[FIX ? C : 1][V] = {};
    for (uint32_t e = e0; e < e1; e++) {
        const uint32_t t = a.t_idx[e];
        if (t < a.row0 || t >= end || !is_live(a, t)) continue;
        // a row that is named twice: its first entry takes the weights of all
        float w = 0.f;
        bool first = true;
        for (uint32_t k = e0 + lane; k < e1; k += 64) {
            if (a.t_idx[k] != t) continue;
            w += target_weight(a, k, e0, e1);
            if (k < e) first = false;
        }
        if (__any(!first)) continue;
        float dot = 0.f;
        const char* x = (const char*)a.rows + (uint64_t)t * a.r_pitch;
        tv held[C];
#pragma unroll
        for (int c = 0; c < C; c++) {
            const uint32_t d = (c * 64 + lane) * V;
            if (d >= a.dim) continue;
            held[c] = *reinterpret_cast<const tv*>(x + d * sizeof(T));
            const tv u = *reinterpret_cast<const tv*>(q + d * sizeof(T));
#pragma unroll
            for (int v = 0; v < V; v++) dot = __builtin_fmaf((float)u[v], (float)held[c][v], dot);
        }
#pragma unroll
        for (int d = 32; d; d >>= 1) {
            dot += __shfl_xor(dot, d);
            w += __shfl_xor(w, d);
        }
        if (w != 0.f) at = __builtin_fmaf(w, dot * a.scale, at);
        const float p = exp2f(__builtin_fmaf(dot, a.scale * LOG2E, -lw.x));
        const float g = cw == 0.f ? 0.f : gs * (lw.y * p - cw * w);
        if (lane == 0) {
            char* block = a.blocks + ((size_t)(qi >> 5) * a.row_blocks + ((t - a.row0) >> 5)) * BLOCK_BYTES;
            put_value<GradTiles<T>>(block + block_place(qi & 31, (t - a.row0) & 31), a.block_low, g);
        }
        if constexpr (FIX) {
            const float left = g - (float)(T)g;
#pragma unroll
            for (int c = 0; c < C; c++)
                if ((uint32_t)(c * 64 + lane) * V < a.dim) {
#pragma unroll
                    for (int v = 0; v < V; v++) fix[c][v] = __builtin_fmaf(left, (float)held[c][v], fix[c][v]);
                }
        }
    }
    if constexpr (FIX) {
#pragma unroll
        for (int c = 0; c < C; c++) {
            const uint32_t d = (c * 64 + lane) * V;
            if (d >= a.dim) continue;
            f32x4* to = reinterpret_cast<f32x4*>(a.fix + (size_t)qi * a.dim + d);
#pragma unroll
            for (int k = 0; k < V / 4; k++) {
                const f32x4 v = {fix[c][4 * k], fix[c][4 * k + 1], fix[c][4 * k + 2], fix[c][4 * k + 3]};
                to[k] = first_piece ? v : to[k] + v;
            }
        }
    }
    if (ALL && lane == 0) {
        const float W = a.total[qi], lse = lw.x * LN2;
        if (a.lse) a.lse[qi] = lse;
        if (a.loss) a.loss[qi] = W == 0.f ? 0.f - at : __builtin_fmaf(W, lse, -at);
    }
}

// A fragment's values times 2^-less, less >= 0. bf16 exponentials are not negative and need one saturating subtraction on the exponent of
// two at a time: what falls below the smallest normal number becomes zero or stays below it.
template <typename T> __device__ inline i32x4 scale_down(i32x4 v, float less) {
    if constexpr (__is_same(T, _Float16)) {
        // in two steps: a factor below 2^-24 is no fp16 number, but 2^14 times it may be
        const float some = fminf(less, 14.f);
        const _Float16 f = (_Float16)__builtin_amdgcn_exp2f(-some), g = (_Float16)__builtin_amdgcn_exp2f(some - less);
        const f16x8 x = __builtin_bit_cast(f16x8, v) * f * g;
        v = __builtin_bit_cast(i32x4, x);
    } else {
        const unsigned short k = (unsigned short)((int)fminf(less, 255.f) << 7);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int two = v[i]; // a bit cast of a vector's element takes the vector's first
            v[i] = __builtin_bit_cast(int, __builtin_elementwise_sub_sat(__builtin_bit_cast(u16x2, two), u16x2{k, k}));
        }
    }
    return v;
}

// grad q: a split's rows x its queries' blocks. M side: queries (blocks), N side: columns of the rows. EXP: fragments are brought
// to the largest reference of the split, and a split's sum to the largest so far.
// DIRECT: the only split of the only piece, whose sum is the gradient.
// 256 x 256 tiles, 1024 queries x 500 000 fp16 rows of 1024: 1.30 ms, 810 TFLOP/s (the exponents' sums beside the products); 2048 x 30 522 bf16, G: 115 us, 1115.
// KG: groups of waves that take every KG-th stage, where one workgroup has a CU to itself: two waves a SIMD, each with a whole wave's
// piece of the tile (4096 x 4096 x 1024, direct: 47 us; one group 53, the same on eight waves of half the piece 52; grad x 42, 48.6).
template <typename T, int MT, int NT, int WM, int WN, int ST, bool EXP, bool DIRECT = false, int KG = 1>
__global__ __launch_bounds__(64 * WM * WN * KG, 2) void loss_grad_q(LossArgs a, uint32_t n_tiles, uint32_t groups_per_split, uint32_t piece_groups, int turn, int first) {
    using S = typename Tiles<T>::S;
    constexpr int NW = WM * WN * KG, BM = WM * MT * 32, BN = WN * NT * 32, SF = 2, P = Tiles<T>::PLANES;
    using BTile = ColTile<S, BN, SF, NW, ORDER_BLOCKS>;
    static_assert(BTile::KE == 32, "a block a stage");
    constexpr int ABYTES = BM / 32 * BLOCK_BYTES, AINS = ABYTES / 1024, ALOADS = (AINS + NW - 1) / NW, PLANE = ABYTES + BTile::BYTES;
    constexpr int RBYTES = NW * 256; // references: 64 queries a wave
    static_assert(NW * 64 >= BM, "a reference a query");
    constexpr int STAGE = P * PLANE + (EXP ? RBYTES : 0), PER = P * (ALOADS + BTile::LOADS) + (EXP ? 1 : 0);
    __shared__ __align__(1024) char lds[ST * STAGE];
    __shared__ float factor[2][BM];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), kg = wave / (WM * WN), wm = wave % (WM * WN) / WN, wn = wave % WN;
    // the workgroups of one split, which read the same rows, on one XCD, and of those with one tile of queries the same blocks
    const uint32_t per_split = a.q_tiles * n_tiles, id = xcd_run(blockIdx.x, gridDim.x), split = id / per_split, rest = id % per_split;
    const uint32_t query = rest / n_tiles * BM, col = rest % n_tiles * BN;
    const uint32_t g0 = min(split * groups_per_split, piece_groups), g1 = min(g0 + groups_per_split, piece_groups);
    const uint32_t group0 = a.row0 / LOSS_GROUP;
    float top = -INFINITY; // of query `query + threadIdx.x` (the first BM threads)
    if constexpr (EXP) {
        if (threadIdx.x < BM) {
            const uint32_t qi = query + threadIdx.x;
            const bool real = qi < a.qp;
            for (uint32_t g = g0; g < g1; g++) top = fmaxf(top, real ? a.block_ref[(size_t)(group0 + g) * a.qp + qi] : -INFINITY);
            factor[0][threadIdx.x] = top;
        }
        __syncthreads();
    }
    float mine[MT]; // the split's reference of the query whose blocks' lane this is
#pragma unroll
    for (int m = 0; m < MT; m++) mine[m] = EXP ? factor[0][(wm * MT + m) * 32 + (lane & 31)] : 0.f;

    // queries: whole blocks, one 32 rows after the other
    uint32_t aoff[ALOADS], adst[ALOADS];
    const uint32_t q_blocks = a.qp / 32;
#pragma unroll
    for (int i = 0; i < ALOADS; i++) {
        const int ins = (i * NW + wave) % AINS, b = ins / BLOCK_PARTS, k = ins % BLOCK_PARTS; // a wave without one of its own repeats another's
        adst[i] = ins * 1024;
        aoff[i] = query / 32 + b < q_blocks ? (uint32_t)b * (a.row_blocks * (uint32_t)BLOCK_BYTES) + k * 1024 + lane * 16 : TILE_MASKED;
    }
    uint64_t abase = uniform64((uint64_t)a.blocks + ((uint64_t)(query / 32) * a.row_blocks + g0 * (LOSS_GROUP / 32)) * BLOCK_BYTES);
    uint64_t rbase = uniform64((uint64_t)(a.block_ref + (size_t)(group0 + g0) * a.qp + query));
    BTile tb[P];
    const uint32_t first_row = a.row0 + g0 * LOSS_GROUP;
#pragma unroll
    for (int p = 0; p < P; p++)
        tb[p].init(reinterpret_cast<const S*>(a.tile_rows + p * a.tile_r_low + (uint64_t)(first_row - a.tile_row0) * a.tile_r_pitch) + col, a.tile_r_pitch, (int)min((uint32_t)BN, a.tile_dim - col), wave, lane);
    const uint32_t roff = query + wave * 64 + lane < a.qp ? (wave * 64 + lane) * 4 : TILE_MASKED;

    const int stages = (int)(g1 - g0) * (LOSS_GROUP / 32);
    const uint32_t base = lds_address(lds);
    uint32_t into = 0, issued = 0;
    uint32_t word = stages ? live_word(a.live, first_row, a.n) : 0u;
    auto issue = [&]() {
        const bool in = (int)issued < stages;
#pragma unroll
        for (int p = 0; p < P; p++) {
            const i32x4 ab = buffer_of(abase + p * a.block_low);
#pragma unroll
            for (int i = 0; i < ALOADS; i++) load_to_lds16(ab, in ? aoff[i] : TILE_MASKED, base + into + p * PLANE + adst[i]);
            tb[p].load(base + into + p * PLANE + ABYTES, in ? word : 0u, wave, lane);
            tb[p].next();
        }
        if constexpr (EXP) load_to_lds4(buffer_of(uniform64(rbase)), in ? roff : TILE_MASKED, base + into + P * PLANE + wave * 256);
        abase += BLOCK_BYTES;
        issued++;
        if (issued % (LOSS_GROUP / 32) == 0) rbase += a.qp * 4;
        word = (int)issued < stages ? live_word(a.live, first_row + issued * 32, a.n) : 0u;
        into = into + STAGE == ST * STAGE ? 0 : into + STAGE;
    };
#pragma unroll
    for (int s = 0; s < ST - KG; s++) issue();
    f32x16 acc[MT][NT] = {};
    uint32_t from = 0;
    for (int s = 0; s < stages; s += KG) {
        tile_wait<(ST - 2 * KG) * PER>();
        const char* A = lds + from + kg * STAGE;
        const char* B = A + ABYTES;
        float less[MT];
        if constexpr (EXP) {
            const float* r = reinterpret_cast<const float*>(A + P * PLANE);
#pragma unroll
            for (int m = 0; m < MT; m++) {
                const float own = r[(wm * MT + m) * 32 + (lane & 31)];
                less[m] = own == -INFINITY ? 0.f : mine[m] - own; // a group without live rows holds zeros
            }
        }
        i32x4 x[2][MT][P], y[2][NT][P];
        auto read = [&](int f) {
#pragma unroll
            for (int p = 0; p < P; p++) {
#pragma unroll
                for (int m = 0; m < MT; m++)
                    x[f & 1][m][p] = *reinterpret_cast<const i32x4*>(A + p * PLANE + (wm * MT + m) * BLOCK_BYTES + f * 1024 + block_slot(lane & 31, lane >> 5, f) * 16);
#pragma unroll
                for (int t = 0; t < NT; t++) y[f & 1][t][p] = BTile::read(B + p * PLANE, wn * NT + t, f, lane);
            }
        };
        read(0);
#pragma unroll
        for (int k = 0; k < KG; k++) issue();
#pragma unroll
        for (int f = 0; f < SF; f++) {
            if (f + 1 < SF) read(f + 1);
            if constexpr (EXP) {
#pragma unroll
                for (int m = 0; m < MT; m++)
#pragma unroll
                    for (int p = 0; p < P; p++) x[f & 1][m][p] = scale_down<S>(x[f & 1][m][p], less[m]);
            }
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int t = 0; t < NT; t++) acc[m][t] = multiply<Tiles<T>>(x[f & 1][m], y[f & 1][t], acc[m][t]);
        }
        interleave<P * (MT + 2 * NT), PRODUCTS<Tiles<T>> * MT * NT, SF>();
        from = from + KG * STAGE == ST * STAGE ? 0 : from + KG * STAGE;
    }
    float fix[DIRECT ? MT / KG : 1][16][NT]; // asked for together, before the last loads are waited for (4096 x 4096: 51 us; one by one beside the stores 57, without it 50)
    if constexpr (DIRECT) {
#pragma unroll
        for (int m = 0; m < MT / KG; m++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const uint32_t qi = query + (wm * MT + kg * (MT / KG) + m) * 32 + result_row(i, lane >> 5);
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const uint32_t d = col + (wn * NT + t) * 32 + (lane & 31);
                    fix[m][i][t] = qi < a.nq && d < a.dim ? a.fix[(size_t)qi * a.dim + d] : 0.f;
                }
            }
    }
    tile_wait<0>();
    if constexpr (KG == 2) {
        static_assert(BM * BN * 4 <= ST * STAGE, "the sums fit the stages");
        exchange_halves<MT, NT, WM * WN>(acc, lds, kg, wave % (WM * WN), lane);
    }
    if constexpr (EXP) {
        if (threadIdx.x < BM) {
            const uint32_t qi = query + threadIdx.x;
            const size_t at = (size_t)split * a.qp + qi;
            const float old = first || qi >= a.qp ? -INFINITY : a.part_ref[turn ^ 1][at];
            const float both = fmaxf(old, top);
            factor[0][threadIdx.x] = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - both);
            factor[1][threadIdx.x] = old == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(old - both);
            if (col == 0 && qi < a.qp) a.part_ref[turn][at] = both;
        }
        __syncthreads();
    }
    const int h = lane >> 5;
    const float all_back = DIRECT && !OWN_SCALE<T> ? a.scale / grad_scale<T>(a, 0) : 1.f;
#pragma unroll
    for (int m = 0; m < MT; m++) {
        if (KG == 2 && m / (MT / 2) != kg) continue;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int r = (wm * MT + m) * 32 + result_row(i, h);
            if (query + r >= a.nq) continue;
            if constexpr (DIRECT) {
                const bool on = (a.q_on[(query + r) >> 5] >> (r & 31)) & 1;
                T* to = reinterpret_cast<T*>((char*)a.grad_q + (uint64_t)(query + r) * a.gq_pitch);
                const float back = OWN_SCALE<T> ? a.scale / grad_scale<T>(a, query + r) : all_back;
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const uint32_t d = col + (wn * NT + t) * 32 + (lane & 31);
                    if (d < a.dim) to[d] = (T)(on ? (acc[m][t][i] + fix[m % (MT / KG)][i][t]) * back : 0.f);
                }
                continue;
            }
            float* out = a.part + ((size_t)split * a.qp + query + r) * a.dim;
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const uint32_t d = col + (wn * NT + t) * 32 + (lane & 31);
                if (d >= a.dim) continue;
                float v = acc[m][t][i];
                if constexpr (EXP) v *= factor[0][r];
                if (!first) v += EXP ? out[d] * factor[1][r] : out[d];
                out[d] = v;
            }
        }
    }
}

// grad x of a piece: rows (blocks read transposed) x queries. Each row's gradient is whole here: all queries are in.
// 256 x 256 tiles, 2048 queries x 30 522 bf16 rows of 1024: 130 us, 990 TFLOP/s; 128 x 128, 4096 x 4096: 42 us (KG as above), 820.
template <typename T, int MT, int NT, int WM, int WN, int ST, int KG = 1>
__global__ __launch_bounds__(64 * WM * WN * KG, 2) void loss_grad_x(LossArgs a, uint32_t n_tiles) {
    using S = typename GradTiles<T>::S;
    constexpr int NW = WM * WN * KG, BM = WM * MT * 32, BN = WN * NT * 32, SF = 2, P = GradTiles<T>::PLANES;
    using BTile = ColTile<S, BN, SF, NW, ORDER_ROWS>;
    constexpr int ABYTES = BM / 32 * BLOCK_BYTES, ALOADS = ABYTES / (1024 * NW), PLANE = ABYTES + BTile::BYTES;
    constexpr int STAGE = P * PLANE, PER = P * (ALOADS + BTile::LOADS);
    __shared__ __align__(1024) char lds[ST * STAGE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), kg = wave / (WM * WN), wm = wave % (WM * WN) / WN, wn = wave % WN;
    uint32_t rt = blockIdx.x / n_tiles, col = blockIdx.x % n_tiles * BN;
    const uint32_t whole = gridDim.x / n_tiles / 8 * 8;
    if (blockIdx.x < whole * n_tiles) { // the column tiles of one tile of rows, which read the same blocks, on one XCD
        const uint32_t i = blockIdx.x >> 3;
        rt = (i / n_tiles) * 8 + (blockIdx.x & 7);
        col = i % n_tiles * BN;
    }
    const uint32_t block0 = rt * (BM / 32);
    uint32_t aoff[ALOADS];
#pragma unroll
    for (int i = 0; i < ALOADS; i++) {
        const int ins = i * NW + wave;
        aoff[i] = block0 + ins / BLOCK_PARTS < a.row_blocks ? ins * 1024 + lane * 16 : TILE_MASKED;
    }
    uint64_t abase = uniform64((uint64_t)a.blocks + (uint64_t)block0 * BLOCK_BYTES);
    const uint64_t astep = (uint64_t)a.row_blocks * BLOCK_BYTES;
    BTile tb[P];
#pragma unroll
    for (int p = 0; p < P; p++) tb[p].init(reinterpret_cast<const S*>(a.grad_tile_q + p * a.tile_q_low) + col, a.grad_tile_q_pitch, (int)min((uint32_t)BN, a.tile_dim - col), wave, lane);
    const UniformWords q_on = (UniformWords)a.q_on;
    const int stages = (int)((a.nq + 31) / 32);
    const uint32_t base = lds_address(lds);
    uint32_t into = 0, issued = 0;
    auto issue = [&]() {
        const bool in = (int)issued < stages;
        const uint32_t on = in ? q_on[issued] : 0u;
#pragma unroll
        for (int p = 0; p < P; p++) {
            const i32x4 ab = buffer_of(abase + p * a.block_low);
#pragma unroll
            for (int i = 0; i < ALOADS; i++) load_to_lds16(ab, in ? aoff[i] : TILE_MASKED, base + into + p * PLANE + (i * NW + wave) * 1024);
            tb[p].load(base + into + p * PLANE + ABYTES, on, wave, lane);
            tb[p].next();
        }
        abase += astep;
        issued++;
        into = into + STAGE == ST * STAGE ? 0 : into + STAGE;
    };
#pragma unroll
    for (int s = 0; s < ST - KG; s++) issue();
    f32x16 acc[MT][NT] = {};
    uint32_t from = 0;
    for (int s = 0; s < stages; s += KG) {
        tile_wait<(ST - 2 * KG) * PER>();
        const char* A = lds + from + kg * STAGE;
        const char* B = A + ABYTES;
        i32x4 x[2][MT][P], y[2][NT][P];
        auto read = [&](int f) {
            const int h = lane >> 5, i = lane & 15, g = (lane >> 4) & 1;
#pragma unroll
            for (int p = 0; p < P; p++) {
#pragma unroll
                for (int m = 0; m < MT; m++) {
                    const char* block = A + p * PLANE + (wm * MT + m) * BLOCK_BYTES;
                    i32x2 part[2];
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const int q = f * 16 + 8 * h + 4 * j + (i >> 2);
                        const char* at = block + g * 1024 + block_slot(q, i & 1, g) * 16 + ((i & 3) >> 1) * 8;
                        part[j] = __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at));
                    }
                    x[f & 1][m][p] = i32x4{part[0][0], part[0][1], part[1][0], part[1][1]};
                }
#pragma unroll
                for (int t = 0; t < NT; t++) y[f & 1][t][p] = BTile::read(B + p * PLANE, wn * NT + t, f, lane);
            }
        };
        read(0);
#pragma unroll
        for (int k = 0; k < KG; k++) issue();
#pragma unroll
        for (int f = 0; f < SF; f++) {
            if (f + 1 < SF) read(f + 1);
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int t = 0; t < NT; t++) acc[m][t] = multiply<GradTiles<T>>(x[f & 1][m], y[f & 1][t], acc[m][t]);
        }
        interleave<P * (2 * MT + 2 * NT), PRODUCTS<GradTiles<T>> * MT * NT, SF>();
        from = from + KG * STAGE == ST * STAGE ? 0 : from + KG * STAGE;
    }
    tile_wait<0>();
    if constexpr (KG == 2) {
        static_assert(BM * BN * 4 <= ST * STAGE, "the sums fit the stages");
        exchange_halves<MT, NT, WM * WN>(acc, lds, kg, wave % (WM * WN), lane);
    }
    const float back = OWN_SCALE<T> ? ldexpf(a.scale, -scale_of_sizes(a)) / *a.part_of_two : a.scale / grad_scale<T>(a, 0);
    const int h = lane >> 5;
#pragma unroll
    for (int m = 0; m < MT; m++) {
        if (KG == 2 && m / (MT / 2) != kg) continue;
        const uint32_t row = a.row0 + rt * BM + (wm * MT + m) * 32;
        const uint32_t word = live_word(a.live, row, a.n);
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const uint32_t r = row + result_row(i, h);
            if (r >= a.n) continue;
            const bool on = (word >> result_row(i, h)) & 1;
            T* out = reinterpret_cast<T*>((char*)a.grad_x + (uint64_t)r * a.gx_pitch);
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const uint32_t d = col + (wn * NT + t) * 32 + (lane & 31);
                if (d < a.dim) out[d] = (T)(on ? acc[m][t][i] * back : 0.f);
            }
        }
    }
}

template <int THREADS> __device__ inline float block_sum(float v, float* buf) { // the same for all threads
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < THREADS / 64; k++) s += buf[k];
    return s;
}

constexpr uint32_t LOSS_SPLITS = 512; // of the rows under one partial sum of grad q, at most

// One workgroup a query: lse, loss, and the query's gradient from its splits. EXP: the splits are sums of exponentials relative
// to their references without the targets, whose terms are added here; otherwise they are sums of scaled G. A thread holds four
// columns (and their next 4 THREADS); where a row has fewer than 4 THREADS columns the threads share the splits.
template <typename T, bool GRAD, bool EXP, int THREADS> __global__ __launch_bounds__(THREADS, THREADS == 1024 ? 8 : 4) void loss_finish(LossArgs a, int turn) {
    constexpr int C = APOE_LOSS_MAX_DIM / (THREADS * 4);
    typedef T t4 __attribute__((ext_vector_type(4)));
    __shared__ float buf[THREADS / 64], lse_of, factor[GRAD ? LOSS_SPLITS : 1];
    __shared__ f32x4 share[GRAD ? THREADS : 1];
    const uint32_t qi = blockIdx.x, tid = threadIdx.x;
    f32x4 acc[C] = {};
    uint32_t lanes = THREADS;
    while (lanes * 2 >= a.dim && lanes > 64) lanes /= 2; // threads along a row
    const uint32_t groups = THREADS / lanes, g = tid / lanes, d0 = tid % lanes * 4;
    constexpr int EARLY = GRAD && EXP ? 4 : 1; // sums of the splits that are asked for before their factors are known
    f32x4 early[EARLY];
    if constexpr (GRAD && EXP) {
#pragma unroll
        for (int i = 0; i < EARLY; i++) {
            const uint32_t s = g + i * groups;
            early[i] = s < a.splits && d0 < a.dim ? *reinterpret_cast<const f32x4*>(a.part + ((size_t)s * a.qp + qi) * a.dim + d0) : f32x4{};
        }
    }
    auto add_splits = [&]() {
#pragma unroll
        for (int k = 0; k < C; k++) {
            const uint32_t d = d0 + k * THREADS * 4;
            if (d >= a.dim || (k && groups > 1)) continue;
            const float* p = a.part + (size_t)qi * a.dim + d;
            if (EXP && k == 0) {
#pragma unroll
                for (int i = 0; i < EARLY; i++) {
                    const uint32_t s = g + i * groups;
                    if (s < a.splits) acc[0] += factor[s] * early[i];
                }
            }
#pragma unroll 4
            for (uint32_t s = g + (EXP && k == 0 ? EARLY * groups : 0); s < a.splits; s += groups) {
                const f32x4 x = *reinterpret_cast<const f32x4*>(p + (size_t)s * a.qp * a.dim);
                acc[k] += EXP ? factor[s] * x : x;
            }
        }
    };
    if constexpr (GRAD && !EXP) add_splits(); // on their way while the sums are joined
    if (tid < 64) {
        const float l = join_chunks(a, qi, tid);
        if (tid == 0) lse_of = l;
    }
    const uint32_t e0 = a.t_off ? a.t_off[qi] : 0, e1 = a.t_off ? a.t_off[qi + 1] : 0;
    float W = 0.f;
    bool any = false;
    for (uint32_t e = e0 + tid; e < e1; e += THREADS) {
        const float w = is_live(a, a.t_idx[e]) ? target_weight(a, e, e0, e1) : 0.f;
        W += w;
        any |= w != 0.f;
    }
    W = block_sum<THREADS>(W, buf);
    const bool on = __syncthreads_or(any);
    const float lse = lse_of, cw = a.weight ? a.weight[qi] : 1.f;
    const bool counts = on && cw != 0.f;
    if constexpr (GRAD) {
        if constexpr (EXP) {
            for (uint32_t s = tid; s < a.splits; s += THREADS) {
                const float r = a.part_ref[turn][(size_t)s * a.qp + qi];
                factor[s] = r == -INFINITY ? 0.f : W * __builtin_amdgcn_exp2f(r - lse);
            }
            __syncthreads();
            if (counts) add_splits();
        }
        if (groups > 1) {
            share[tid] = acc[0];
            __syncthreads();
            if (g == 0)
                for (uint32_t k = 1; k < groups; k++) acc[0] += share[k * lanes + tid];
            if (g) acc[0] = f32x4{};
        }
        if constexpr (!EXP) {
            const float gs = 1.f / grad_scale<T>(a, qi);
#pragma unroll
            for (int k = 0; k < C; k++) acc[k] *= gs;
        }
    }
    // targets: s_t in 32 bits, in the order of the list
    const char* q = (const char*)a.q + (uint64_t)qi * a.q_pitch;
    float at = 0.f;
    for (uint32_t e = e0; e < e1; e++) {
        const uint32_t t = a.t_idx[e];
        if (!is_live(a, t)) continue;
        const float w = target_weight(a, e, e0, e1);
        if (w == 0.f && !(GRAD && EXP)) continue;
        const char* x = (const char*)a.rows + (uint64_t)t * a.r_pitch;
        float dot = 0.f;
        t4 xs[C];
#pragma unroll
        for (int k = 0; k < C; k++) {
            const uint32_t d = (k * THREADS + tid) * 4;
            if (d >= a.dim) continue;
            xs[k] = *reinterpret_cast<const t4*>(x + d * sizeof(T));
            const t4 u = *reinterpret_cast<const t4*>(q + d * sizeof(T));
#pragma unroll
            for (int v = 0; v < 4; v++) dot = __builtin_fmaf((float)u[v], (float)xs[k][v], dot);
        }
        dot = block_sum<THREADS>(dot, buf);
        if (w != 0.f) at = __builtin_fmaf(w, dot * a.scale, at);
        if constexpr (GRAD && EXP) {
            bool again = false; // its exponential was taken out once
            for (uint32_t k = e0 + tid; k < e; k += THREADS) again |= a.t_idx[k] == t;
            again = __syncthreads_or(again);
            const float f = (again ? 0.f : W * exp2f(__builtin_fmaf(dot, a.scale * LOG2E, -lse))) - w;
            if (counts) {
#pragma unroll
                for (int k = 0; k < C; k++)
                    if ((k * THREADS + tid) * 4 < a.dim) {
#pragma unroll
                        for (int v = 0; v < 4; v++) acc[k][v] = __builtin_fmaf(f, (float)xs[k][v], acc[k][v]);
                    }
            }
        }
    }
    if (tid == 0) {
        if (a.lse) a.lse[qi] = lse * LN2;
        if (a.loss) a.loss[qi] = W == 0.f ? (on ? -at : 0.f) : __builtin_fmaf(W, lse * LN2, -at);
    }
    if constexpr (GRAD) {
        const float f = EXP ? cw * a.scale : a.scale;
        char* out = (char*)a.grad_q + (uint64_t)qi * a.gq_pitch;
#pragma unroll
        for (int k = 0; k < C; k++) {
            const uint32_t d = (k * THREADS + tid) * 4;
            if (d >= a.dim) continue;
            t4 o;
#pragma unroll
            for (int v = 0; v < 4; v++) o[v] = (T)(counts ? f * acc[k][v] : 0.f);
            *reinterpret_cast<t4*>(out + d * sizeof(T)) = o;
        }
    }
}

// ---- few queries ----
// Up to four queries (float: eight) of up to 1024 columns: every row is read once from memory, by one wave, which keeps the queries, its running sums and the
// rows on their way in registers (a tile of 32 queries would be mostly empty, and its rows would be read twice). A wave takes four
// rows at a time and asks for the next four before it works on these; four inner products are summed over the lanes together.
// Exponentials are relative to a whole exponent that moves only when a logit passes it by 2^60: sums in 32 bits bear that.
constexpr int FEW_E = 16; // values of a row that a lane holds
constexpr uint32_t FEW_MAX_DIM = 64 * FEW_E, FEW_BLOCKS = 512;
// What the registers hold beside the rows on their way, and up to how many queries: pairs of float queries are worked on side by side,
// by workgroups that read the same rows at the same time (8 queries x 1 M rows: 2.48 ms; by tiles, whose planes are written first: 3.34).
template <typename T> constexpr uint32_t FEW_HELD = sizeof(T) == 2 ? 4 : 2;
template <typename T> constexpr uint32_t FEW_QUERIES = sizeof(T) == 2 ? 4 : 8;

template <typename T, int NQ, bool GRAD> __global__ __launch_bounds__(256, 2) void loss_few(LossArgs a, uint32_t sets) {
    constexpr int V = 16 / (int)sizeof(T), C = FEW_E / V;
    typedef T tv __attribute__((ext_vector_type(V)));
    __shared__ float refs[NQ][4], sums[NQ][4];
    __shared__ float part[GRAD ? 4 : 1][GRAD ? NQ * FEW_MAX_DIM : 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t split = blockIdx.x / sets, q0 = blockIdx.x % sets * NQ; // the sets of one split side by side
    const uint32_t fours = (a.n + 3) / 4, step = gridDim.x / sets * 4;
    const float c = a.scale * LOG2E;
    float q[NQ][FEW_E], acc[NQ][FEW_E] = {}, ref[NQ], sum[NQ] = {};
#pragma unroll
    for (int n = 0; n < NQ; n++) {
        ref[n] = -INFINITY;
#pragma unroll
        for (int k = 0; k < C; k++) {
            const uint32_t d = (k * 64 + lane) * V;
            tv x = {};
            if (q0 + n < a.nq && d < a.dim) x = *reinterpret_cast<const tv*>((const char*)a.q + (uint64_t)(q0 + n) * a.q_pitch + d * sizeof(T));
#pragma unroll
            for (int v = 0; v < V; v++) q[n][k * V + v] = (float)x[v];
        }
    }
    auto live_four = [&](uint32_t four) { return four < fours ? (live_word(a.live, four * 4 & ~31u, a.n) >> (four * 4 & 31)) & 15u : 0u; };
    auto load = [&](tv (&x)[4][C], uint32_t four, uint32_t on) {
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int k = 0; k < C; k++) {
                const uint32_t d = (k * 64 + lane) * V;
                x[r][k] = tv{};
                if (((on >> r) & 1) && d < a.dim) x[r][k] = *reinterpret_cast<const tv*>((const char*)a.rows + (uint64_t)(four * 4 + r) * a.r_pitch + d * sizeof(T));
            }
    };
    uint32_t four = split * 4 + wave, on = live_four(four);
    tv next[4][C];
    load(next, four, on);
    while (four < fours) {
        tv raw[4][C];
        const uint32_t now = on;
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int k = 0; k < C; k++) raw[r][k] = next[r][k];
        four += step;
        on = live_four(four);
        load(next, four, on);
        if (!now) continue;
        float x[4][FEW_E];
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int k = 0; k < C; k++)
#pragma unroll
                for (int v = 0; v < V; v++) x[r][k * V + v] = (float)raw[r][k][v];
#pragma unroll
        for (int n = 0; n < NQ; n++) {
            float z[4];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                z[r] = 0.f;
#pragma unroll
                for (int e = 0; e < FEW_E; e++) z[r] = __builtin_fmaf(q[n][e], x[r][e], z[r]);
            }
            // four sums over 64 lanes in seven exchanges: each halves what a lane carries, or the lanes that differ
            const bool hi = lane & 32, mid = lane & 16;
            float u = (hi ? z[1] : z[0]) + __shfl_xor(hi ? z[0] : z[1], 32);
            float w = (hi ? z[3] : z[2]) + __shfl_xor(hi ? z[2] : z[3], 32);
            u = (mid ? w : u) + __shfl_xor(mid ? u : w, 16);
#pragma unroll
            for (int d = 8; d; d >>= 1) u += __shfl_xor(u, d);
#pragma unroll
            for (int r = 0; r < 4; r++) {
                if (!((now >> r) & 1)) continue;
                const float y = c * __int_as_float(__builtin_amdgcn_readlane(__float_as_int(u), (r & 1) * 32 + (r >> 1) * 16));
                if (y > ref[n] + 60.f) {
                    const float to = ceilf(y), f = __builtin_amdgcn_exp2f(ref[n] - to);
                    ref[n] = to;
                    sum[n] *= f;
                    if constexpr (GRAD) {
#pragma unroll
                        for (int e = 0; e < FEW_E; e++) acc[n][e] *= f;
                    }
                }
                const float p = y == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(y - ref[n]);
                sum[n] += p;
                if constexpr (GRAD) {
#pragma unroll
                    for (int e = 0; e < FEW_E; e++) acc[n][e] = __builtin_fmaf(p, x[r][e], acc[n][e]);
                }
            }
        }
    }
    // the four waves joined
    if (lane == 0)
#pragma unroll
        for (int n = 0; n < NQ; n++) {
            refs[n][wave] = ref[n];
            sums[n][wave] = sum[n];
        }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NQ; n++) {
        const float top = fmaxf(fmaxf(refs[n][0], refs[n][1]), fmaxf(refs[n][2], refs[n][3]));
        if (threadIdx.x == 0) {
            float t = 0.f, r = -INFINITY;
            for (int k = 0; k < 4; k++) join_sums(r, t, refs[n][k], sums[n][k]);
            const size_t at = (size_t)split * a.qp + q0 + n;
            a.chunk_ref[at] = r;
            a.chunk_sum[at] = t;
            if constexpr (GRAD) a.part_ref[0][at] = top;
        }
        if constexpr (GRAD) {
            const float f = top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ref[n] - top); // without live rows: zeros (or NaN)
#pragma unroll
            for (int k = 0; k < C; k++)
#pragma unroll
                for (int v = 0; v < V; v++) part[wave][n * FEW_MAX_DIM + (k * 64 + lane) * V + v] = acc[n][k * V + v] * f;
        }
    }
    if constexpr (GRAD) {
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NQ; n++)
            for (uint32_t d = threadIdx.x; d < a.dim; d += 256) {
                const uint32_t at = n * FEW_MAX_DIM + d;
                a.part[((size_t)split * a.qp + q0 + n) * a.dim + d] = (part[0][at] + part[1][at]) + (part[2][at] + part[3][at]);
            }
    }
}

// Grid (queries, parts of 256 columns): each of a query's workgroups forms lse and the targets' logits anew and adds up its columns of
// the splits' sums, the first of which are on their way before anything else is known (1 query x 4000 rows: 7.3 us, one workgroup for all columns 11).
template <typename T, bool GRAD> __global__ __launch_bounds__(1024) void loss_few_finish(LossArgs a) {
    __shared__ float lse_of, buf[16], scale_of[FEW_BLOCKS];
    __shared__ f32x4 sixteenth[GRAD ? 16 : 1][GRAD ? 64 : 1];
    const uint32_t qi = blockIdx.x, tid = threadIdx.x, c0 = blockIdx.y * 256, d4 = c0 + (tid & 63) * 4;
    const float* part = a.part + (size_t)qi * a.dim + d4;
    const size_t pitch = (size_t)a.qp * a.dim;
    constexpr int EARLY = 8;
    f32x4 early[EARLY];
    if constexpr (GRAD) {
#pragma unroll
        for (int k = 0; k < EARLY; k++) {
            const uint32_t s = (tid >> 6) + 16 * k;
            early[k] = s < a.splits && d4 < a.dim ? *reinterpret_cast<const f32x4*>(part + s * pitch) : f32x4{};
        }
    }
    const float qd = tid < a.dim ? (float)reinterpret_cast<const T*>((const char*)a.q + (uint64_t)qi * a.q_pitch)[tid] : 0.f;
    if (tid < 64) {
        const float l = join_chunks(a, qi, tid);
        if (tid == 0) lse_of = l;
    }
    auto all_sum = [&](float v) {
#pragma unroll
        for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
        __syncthreads();
        if ((tid & 63) == 0) buf[tid >> 6] = v;
        __syncthreads();
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < 16; k++) s += buf[k];
        return s;
    };
    const uint32_t e0 = a.t_off ? a.t_off[qi] : 0, e1 = a.t_off ? a.t_off[qi + 1] : 0;
    float W = 0.f;
    bool any = false;
    for (uint32_t e = e0 + tid; e < e1; e += 1024) {
        const float w = is_live(a, a.t_idx[e]) ? target_weight(a, e, e0, e1) : 0.f;
        W += w;
        any |= w != 0.f;
    }
    W = all_sum(W);
    const bool on = __syncthreads_or(any);
    const float lse = lse_of, cw = a.weight ? a.weight[qi] : 1.f;
    const bool counts = on && cw != 0.f;
    float g = 0.f;
    if constexpr (GRAD) {
        for (uint32_t s = tid; s < a.splits; s += 1024) {
            const float r = a.part_ref[0][(size_t)s * a.qp + qi];
            scale_of[s] = r == -INFINITY ? 0.f : W * __builtin_amdgcn_exp2f(r - lse);
        }
        __syncthreads();
        f32x4 v = {};
        if (counts && d4 < a.dim) {
#pragma unroll
            for (int k = 0; k < EARLY; k++) {
                const uint32_t s = (tid >> 6) + 16 * k;
                if (s < a.splits) v += scale_of[s] * early[k];
            }
#pragma unroll 8
            for (uint32_t s = (tid >> 6) + 16 * EARLY; s < a.splits; s += 16) v += scale_of[s] * *reinterpret_cast<const f32x4*>(part + s * pitch);
        }
        sixteenth[tid >> 6][tid & 63] = v;
        __syncthreads();
        if (tid < 256) {
            const float* p = reinterpret_cast<const float*>(sixteenth) + tid;
#pragma unroll
            for (int k = 0; k < 16; k++) g += p[k * 256];
        }
    }
    const uint32_t own = c0 + tid; // the first 256 threads' column
    const bool mine = GRAD && tid < 256 && own < a.dim;
    float at = 0.f;
    for (uint32_t e = e0; e < e1; e++) {
        const uint32_t t = a.t_idx[e];
        const float w = is_live(a, t) ? target_weight(a, e, e0, e1) : 0.f;
        if (w == 0.f) continue;
        const T* row = reinterpret_cast<const T*>((const char*)a.rows + (uint64_t)t * a.r_pitch);
        const float xd = tid < a.dim ? (float)row[tid] : 0.f, xo = mine ? (float)row[own] : 0.f;
        at = __builtin_fmaf(w, all_sum(qd * xd) * a.scale, at);
        if (GRAD && counts) g = __builtin_fmaf(-w, xo, g);
    }
    if (tid == 0 && c0 == 0) {
        if (a.lse) a.lse[qi] = lse * LN2;
        if (a.loss) a.loss[qi] = W == 0.f ? (on ? -at : 0.f) : __builtin_fmaf(W, lse * LN2, -at);
    }
    if (mine) reinterpret_cast<T*>((char*)a.grad_q + (uint64_t)qi * a.gq_pitch)[own] = (T)(counts ? cw * a.scale * g : 0.f);
}

// ---- launches ----

static uint32_t up(uint64_t v, uint64_t to) { return (uint32_t)((v + to - 1) / to * to); }

template <typename T> static int run_few(apoe_ctx* ctx, LossArgs& a, bool grad) {
    // a wave has two turns of four rows at least, a CU two workgroups at most
    const uint32_t held = std::min(FEW_HELD<T>, next_pow2(a.nq)), sets = (a.nq + held - 1) / held;
    const uint32_t blocks = std::max(1u, std::min((a.n + 31) / 32, std::min(FEW_BLOCKS, 2 * (uint32_t)ctx->num_cus) / sets));
    a.qp = sets * held;
    a.chunks = a.splits = blocks;
    const size_t sums = (size_t)blocks * a.qp * 4, up16 = (sums + 15) / 16 * 16;
    char* ws = nullptr;
    APOE_TRY(ctx->adapt_workspace(3 * up16 + (grad ? (size_t)blocks * a.qp * a.dim * 4 : 0), &ws));
    a.chunk_ref = (float*)ws;
    a.chunk_sum = (float*)(ws + up16);
    a.part_ref[0] = (float*)(ws + 2 * up16);
    a.part = (float*)(ws + 3 * up16);
    hipStream_t s = ctx->stream;
    auto go = [&](auto n) {
        constexpr int NQ = decltype(n)::value;
        if (grad) loss_few<T, NQ, true><<<blocks * sets, 256, 0, s>>>(a, sets);
        else loss_few<T, NQ, false><<<blocks * sets, 256, 0, s>>>(a, sets);
    };
    if (held == 1) go(std::integral_constant<int, 1>{});
    else if (held == 2) go(std::integral_constant<int, 2>{});
    else if constexpr (FEW_HELD<T> == 4) go(std::integral_constant<int, 4>{});
    if (grad) loss_few_finish<T, true><<<dim3(a.nq, (a.dim + 255) / 256), 1024, 0, s>>>(a);
    else loss_few_finish<T, false><<<a.nq, 1024, 0, s>>>(a);
    APOE_HIP(hipGetLastError());
    return APOE_OK;
}

template <typename T> static int run_loss(apoe_ctx* ctx, const apoe_softmax_loss_args* p) {
    LossArgs a{};
    const bool gq = p->grad_q != nullptr, gx = p->grad_rows != nullptr;
    a.q = p->q;
    a.rows = p->rows;
    a.q_pitch = (uint32_t)(p->q_stride * sizeof(T));
    a.r_pitch = (uint32_t)(p->rows_stride * sizeof(T));
    a.gq_pitch = (uint32_t)(p->grad_q_stride * sizeof(T));
    a.gx_pitch = (uint32_t)(p->grad_rows_stride * sizeof(T));
    a.nq = p->n_queries;
    a.n = p->n_rows;
    a.dim = p->dim;
    a.t_off = p->t_off;
    a.t_idx = p->t_idx;
    a.t_val = p->t_val;
    a.live = p->live;
    a.weight = p->weight;
    a.scale = p->scale;
    a.loss = p->loss;
    a.lse = p->lse;
    a.grad_q = p->grad_q;
    a.grad_x = p->grad_rows;
    if (a.nq <= FEW_QUERIES<T> && a.dim <= FEW_MAX_DIM && !gx) return run_few<T>(ctx, a, gq);
    // Tiles of rows x queries (times at 1024 columns, fp16, with the exponentials written):
    //   256 x 256  where they fill the GPU and the queries they pad beyond what 128 would cost less than they gain (1024 x 65 536: 130 us, 256 x 128:
    //              150), up to an eighth: 1100 x 100 000 without gradient 244 us for 259 with 1.11 times the queries, 777 205 for 199 with 1.14 times.
    //              float without gradient up to 1.3 times: 600 x 100 000 (1.2 times) 555 us for 578 on 128 x 128, 384 (1.33) 460 for 429; with one,
    //              whose product is padded alike, an eighth too: 1100 x 60 000 1.17 ms for 1.20, 896 x 50 000 (1.14) 822 us for 797, 600 650 for 589,
    //              with both 1310 for 1244
    //   256 x 128  where those fill it (128 x 131 072: 56 us; 128 x 128: 66)
    //   128 x 128  for fewer rows (1024 x 4000: 16.5 us; 256 x 128: 20)
    //   128 x 64   up to 64 queries (64 x 30 000: 15.5 us; 128 x 128: 17), 512 x 32 for up to 32 where those fill it (32 x 131 072: 44 us; 48)
    // For float, whose planes are twice the bytes, 256 x 256, 128 x 128 or 128 x 64.
    enum { T256, T256_128, T128, T128_64, T512_32 } form;
    constexpr int PLANES = Tiles<T>::PLANES;
    const uint32_t cus = (uint32_t)ctx->num_cus;
    auto count = [&](uint32_t rows, uint32_t queries) { return (uint64_t)((a.n + rows - 1) / rows) * ((a.nq + queries - 1) / queries); };
    if (PLANES == 1 && a.nq <= 32 && count(512, 32) >= cus) form = T512_32;
    else if (a.nq <= 64) form = T128_64;
    else if (count(256, 256) >= cus && up(a.nq, 256) * 40 < up(a.nq, 128) * (PLANES == 2 && !gq && !gx ? 52 : 45)) form = T256;
    else if (PLANES == 1 && count(256, 128) >= cus) form = T256_128;
    else form = T128;
    const uint32_t bm = form == T512_32 ? 512 : form == T128 || form == T128_64 ? 128 : 256;
    const uint32_t bn = form == T256 ? 256 : form == T128_64 ? 64 : form == T512_32 ? 32 : 128;
    a.qp = up(a.nq, bn);
    a.q_tiles = a.qp / bn;
    const uint32_t rows_up = up(a.n, bm);
    a.tile_dim = up(a.dim, 8);
    // rows of a piece, whole tiles: bounded by the exponentials, by the planes, and by what a launch may count
    uint64_t most = (uint64_t)bm * std::max<uint32_t>(1, (1u << 22) / a.q_tiles);
    if (gq || gx) most = std::min(most, LOSS_PIECE_BYTES / ((uint64_t)a.qp * 2 * (gx ? GradTiles<T>::PLANES : PLANES)) / bm * bm);
    if (PLANES == 2) most = std::min(most, LOSS_PIECE_BYTES / ((uint64_t)a.tile_dim * 4) / bm * bm);
    most = std::max<uint64_t>(bm, most);
    const uint64_t even = (rows_up + most - 1) / most;
    const uint64_t piece = up((rows_up + even - 1) / even, bm);
    const uint32_t pieces = (uint32_t)((rows_up + piece - 1) / piece);
    a.groups = rows_up / LOSS_GROUP;
    const uint32_t chunks_per_piece = std::min<uint32_t>(std::max<uint32_t>(1, LOSS_CHUNKS / pieces), (uint32_t)((piece / LOSS_GROUP + 31) / 32));
    a.chunks = chunks_per_piece * pieces;
    // grad q: tiles of 256 x 256, of 128 or 64 x 256 (float: 128 or 64 x 128); enough splits of the rows to give each CU one. The smaller
    // tiles with two groups of waves (16 bits, 1000 x 4000: 53 us in all; with one group, two workgroups a CU and twice the splits, whose
    // sums are written and read again, 60; 128 x 1 M 900 for 975; float 1024 x 20 000 357 for 368, but not up to 64 queries, which wait for
    // memory: 20 x 1 M 3.51 ms for 3.35)
    const uint32_t qm = a.nq <= 64 ? 64 : form == T256 && PLANES == 1 ? 256 : 128, qn = PLANES == 2 ? 128 : 256;
    const uint32_t gq_q_tiles = (a.qp + qm - 1) / qm, gq_n_tiles = (a.dim + qn - 1) / qn;
    const uint32_t piece_groups = (uint32_t)(piece / LOSS_GROUP);
    // With G whole in one piece, tiles of 128 x 128 that fill the GPU need no splits: 4096 x 4096 takes 15 us less.
    const bool direct = PLANES == 1 && gq && gx && pieces == 1 && (uint64_t)((a.qp + 127) / 128) * ((a.dim + 127) / 128) >= cus * 9 / 10;
    uint32_t splits = std::min(LOSS_SPLITS, std::max<uint32_t>(1, cus / (gq_q_tiles * gq_n_tiles)));
    splits = std::min(splits, piece_groups);
    const uint32_t per_split = (piece_groups + splits - 1) / splits;
    splits = (piece_groups + per_split - 1) / per_split;
    a.splits = splits;

    // workspace
    size_t bytes = 0;
    auto take = [&](size_t b) {
        const size_t at = bytes;
        bytes += (b + 1023) / 1024 * 1024;
        return at;
    };
    const size_t o_ref = take((size_t)a.groups * a.qp * 4), o_sum = take((size_t)a.groups * a.qp * 4);
    const size_t o_cr = take((size_t)a.chunks * a.qp * 4), o_cs = take((size_t)a.chunks * a.qp * 4);
    const size_t o_lw = take((size_t)a.qp * 8), o_top = take(12), o_peak = take((size_t)a.qp * 4), o_size = take(OWN_SCALE<T> ? (size_t)a.qp * 4 : 0), o_on = take(a.qp / 8), o_coef = take((size_t)a.qp * 4), o_total = take((size_t)a.qp * 4);
    a.block_low = (size_t)a.qp * piece * 2;
    const size_t o_blocks = take(gx ? GradTiles<T>::PLANES * a.block_low : gq ? PLANES * a.block_low : 0);
    a.tile_r_low = PLANES == 2 ? piece * a.tile_dim * 2 : 0;
    a.tile_q_low = PLANES == 2 ? (uint64_t)a.qp * a.tile_dim * 2 : 0;
    const size_t o_rows = take(2 * a.tile_r_low), o_q = take(2 * a.tile_q_low), o_gq = take(!gx ? 0 : PLANES == 2 ? 3 * a.tile_q_low : OWN_SCALE<T> ? (size_t)a.qp * a.dim * 2 : 0), o_bref = take(PLANES == 2 && gq ? (size_t)a.groups * a.qp * 4 : 0);
    const size_t o_rexp = take((size_t)a.groups * LOSS_GROUP * 4), o_qexp = take((size_t)a.qp * 4);
    const size_t part_bytes = gq && !direct ? (size_t)splits * a.qp * a.dim * 4 : 0;
    const size_t o_part = take(part_bytes + (PLANES == 1 && gq && gx ? (size_t)a.qp * a.dim * 4 : 0));
    const size_t o_pr0 = take((size_t)splits * a.qp * 4), o_pr1 = take((size_t)splits * a.qp * 4);
    char* ws = nullptr;
    APOE_TRY(ctx->adapt_workspace(bytes, &ws));
    a.ref = (float*)(ws + o_ref);
    a.sum = (float*)(ws + o_sum);
    a.chunk_ref = (float*)(ws + o_cr);
    a.chunk_sum = (float*)(ws + o_cs);
    a.lse_w = (float2*)(ws + o_lw);
    a.top_coef = (uint32_t*)(ws + o_top);
    a.top_size = a.top_coef + 1;
    a.part_of_two = (float*)(a.top_coef + 2);
    a.peak = (float*)(ws + o_peak);
    a.q_size = (float*)(ws + o_size);
    a.blocks = ws + o_blocks;
    a.part = (float*)(ws + o_part);
    a.fix = (float*)(ws + o_part + part_bytes);
    a.part_ref[0] = (float*)(ws + o_pr0);
    a.part_ref[1] = (float*)(ws + o_pr1);
    a.q_on = (uint32_t*)(ws + o_on);
    a.coef = (float*)(ws + o_coef);
    a.total = (float*)(ws + o_total);
    a.row_exp = (float*)(ws + o_rexp);
    a.q_exp = (float*)(ws + o_qexp);
    a.block_ref = PLANES == 2 ? (float*)(ws + o_bref) : a.ref;
    a.tile_rows = PLANES == 2 ? ws + o_rows : (const char*)a.rows;
    a.tile_q = PLANES == 2 ? ws + o_q : (const char*)a.q;
    a.grad_tile_q = PLANES == 2 || OWN_SCALE<T> ? ws + o_gq : a.tile_q;
    a.tile_r_pitch = PLANES == 2 ? a.tile_dim * 2 : a.r_pitch;
    a.tile_q_pitch = PLANES == 2 ? a.tile_dim * 2 : a.q_pitch;
    a.grad_tile_q_pitch = OWN_SCALE<T> ? a.dim * 2 : a.tile_q_pitch;
    hipStream_t s = ctx->stream;
    uint32_t split_piece = ~0u;
    auto set_piece = [&](uint32_t i) {
        a.row0 = (uint32_t)(i * piece);
        const uint32_t rows = (uint32_t)std::min<uint64_t>(piece, rows_up - a.row0);
        a.row_tiles = rows / bm;
        a.row_blocks = rows / 32;
        if constexpr (PLANES == 2) {
            a.tile_row0 = a.row0;
            // unless the planes are of this piece already; the queries' once
            if (i != split_piece) {
                const uint32_t grid = rows / 32 + (split_piece == ~0u ? (a.nq + 7) / 8 : 0);
                if (a.dim <= 1024) loss_split<4><<<grid, 512, 0, s>>>(a, rows / 32);
                else loss_split<LOSS_MAX_COLUMNS / 256><<<grid, 512, 0, s>>>(a, rows / 32);
            }
            split_piece = i;
        }
        return rows / LOSS_GROUP;
    };
    auto tiles = [&](auto mode) {
        constexpr int M = decltype(mode)::value;
        const dim3 grid(a.row_tiles * a.q_tiles);
        if constexpr (PLANES == 2) {
            if (form == T256) loss_tile<T, 2, 2, 4, 2, 2, M><<<grid, 512, 0, s>>>(a);
            else if (form == T128) loss_tile<T, 1, 1, 4, 4, 2, M><<<grid, 256, 0, s>>>(a);
            else loss_tile<T, 1, 1, 2, 4, 3, M><<<grid, 128, 0, s>>>(a);
        } else {
            if (form == T256) loss_tile<T, 2, 2, 4, 4, 2, M><<<grid, 512, 0, s>>>(a);
            else if (form == T256_128) loss_tile<T, 1, 2, 4, 4, 3, M><<<grid, 512, 0, s>>>(a);
            else if (form == T128) loss_tile<T, 1, 1, 4, 4, 2, M><<<grid, 256, 0, s>>>(a);
            else if (form == T128_64) loss_tile<T, 1, 1, 2, 4, 3, M><<<grid, 128, 0, s>>>(a);
            else loss_tile<T, 1, 4, 1, 4, 2, M><<<grid, 256, 0, s>>>(a);
        }
    };
    auto grad_q = [&](auto exp, uint32_t groups, int turn, int first) {
        constexpr bool E = decltype(exp)::value;
        const uint32_t keep = a.q_tiles;
        a.q_tiles = gq_q_tiles;
        const dim3 grid(gq_q_tiles * gq_n_tiles * splits);
        if constexpr (PLANES == 2) {
            if (qm == 64) loss_grad_q<T, 2, 1, 1, 4, 3, E><<<grid, 256, 0, s>>>(a, gq_n_tiles, per_split, groups, turn, first);
            else loss_grad_q<T, 2, 2, 2, 2, 4, E, false, 2><<<grid, 512, 0, s>>>(a, gq_n_tiles, per_split, groups, turn, first);
        } else {
            if (qm == 64) loss_grad_q<T, 2, 2, 1, 4, 6, E, false, 2><<<grid, 512, 0, s>>>(a, gq_n_tiles, per_split, groups, turn, first);
            else if (qm == 256) loss_grad_q<T, 4, 2, 2, 4, 4, E><<<grid, 512, 0, s>>>(a, gq_n_tiles, per_split, groups, turn, first);
            else loss_grad_q<T, 2, 4, 2, 2, 6, E, false, 2><<<grid, 512, 0, s>>>(a, gq_n_tiles, per_split, groups, turn, first);
        }
        a.q_tiles = keep;
    };
    using Sums = std::integral_constant<int, TILE_SUMS>;
    using Exp = std::integral_constant<int, TILE_EXP>;
    using Grad = std::integral_constant<int, TILE_GRAD>;
    const bool many = splits > 16; // of which one workgroup adds up a query's: with 16 waves
    const dim3 join(a.qp / 32, chunks_per_piece);
    auto join_piece = [&](uint32_t i, uint32_t groups, auto zero) {
        loss_join<T, decltype(zero)::value><<<join, 256, 0, s>>>(a, a.row0 / LOSS_GROUP, groups, i * chunks_per_piece);
    };
    auto finish = [&](auto grad, auto exp, int turn) {
        constexpr bool G = decltype(grad)::value, E = decltype(exp)::value;
        if (G && many) loss_finish<T, G, E, 1024><<<a.nq, 1024, 0, s>>>(a, turn);
        else loss_finish<T, G, E, 256><<<a.nq, 256, 0, s>>>(a, turn);
    };
    using Yes = std::true_type;
    using No = std::false_type;
    // One pass, for what needs no G: everything without grad x, and for float the loss and grad q beside it too.
    const bool one_pass = !gx || PLANES == 2;
    const bool unjoined = !(gq && one_pass) && a.groups <= LOSS_CHUNKS; // few enough for one wave as they are
    if (unjoined) {
        a.chunk_ref = a.ref;
        a.chunk_sum = a.sum;
        a.chunks = a.groups;
    }
    if (one_pass) {
        for (uint32_t i = 0; i < pieces; i++) {
            const uint32_t groups = set_piece(i);
            if (gq) {
                tiles(Exp{});
                join_piece(i, groups, Yes{});
                grad_q(Yes{}, groups, (int)(i & 1), i == 0);
            } else {
                tiles(Sums{});
                if (!unjoined) join_piece(i, groups, No{});
            }
        }
        if (gq) finish(Yes{}, Yes{}, (int)((pieces - 1) & 1));
        else finish(No{}, No{}, 0);
    } else {
        for (uint32_t i = 0; i < pieces; i++) {
            const uint32_t groups = set_piece(i);
            if (pieces == 1) tiles(Exp{});
            else tiles(Sums{});
            if (!unjoined) join_piece(i, groups, No{});
        }
    }
    if (gx) {
        loss_coefs<T><<<a.qp, 64, 0, s>>>(a);
        loss_queries<T><<<1, 1024, 0, s>>>(a);
        if constexpr (OWN_SCALE<T>) loss_scale_queries<<<(a.nq + 3) / 4, 256, 0, s>>>(a);
        // grad x: tiles of 256 rows x 256 columns, or of 128 x 128 where those do not fill the GPU, and for float
        const bool x_wide = PLANES == 1 && (uint64_t)((piece + 255) / 256) * ((a.dim + 255) / 256) >= cus;
        const uint32_t xm = x_wide ? 256 : 128, x_tiles = (a.dim + xm - 1) / xm;
        const bool whole = !one_pass && pieces == 1 && (!gq || direct); // nothing is left to a last kernel
        for (uint32_t i = 0; i < pieces; i++) {
            const uint32_t groups = set_piece(i);
            if constexpr (PLANES == 1) {
                if (pieces == 1) loss_normalise<T><<<(uint32_t)(((uint64_t)groups * (a.qp / 32) + 3) / 4), 256, 0, s>>>(a, groups);
                else tiles(Grad{});
            } else {
                tiles(Grad{});
            }
            const bool fix = PLANES == 1 && gq;
            auto targets = [&](auto columns) { // up to how many a wave holds
                constexpr int N = decltype(columns)::value;
                if (whole && fix) loss_targets<T, true, PLANES == 1, N><<<a.nq, 64, 0, s>>>(a, i == 0);
                else if (whole) loss_targets<T, true, false, N><<<a.nq, 64, 0, s>>>(a, i == 0);
                else if (fix) loss_targets<T, false, PLANES == 1, N><<<a.nq, 64, 0, s>>>(a, i == 0);
                else loss_targets<T, false, false, N><<<a.nq, 64, 0, s>>>(a, i == 0);
            };
            if (a.dim <= 1024) targets(std::integral_constant<int, 1024>{});
            else targets(std::integral_constant<int, (int)LOSS_MAX_COLUMNS>{});
            const dim3 grid((a.row_blocks * 32 + xm - 1) / xm * x_tiles);
            if constexpr (PLANES == 1) {
                if (direct) {
                    LossArgs d = a;
                    d.q_tiles = (a.qp + 127) / 128;
                    d.splits = 1;
                    const uint32_t nt = (a.dim + 127) / 128;
                    loss_grad_q<T, 2, 2, 2, 2, 6, false, true, 2><<<d.q_tiles * nt, 512, 0, s>>>(d, nt, groups, groups, 0, 1);
                } else if (gq) {
                    grad_q(No{}, groups, 0, i == 0);
                }
                if (x_wide) loss_grad_x<T, 4, 2, 2, 4, 4><<<grid, 512, 0, s>>>(a, x_tiles);
            }
            if (!x_wide) {
                if constexpr (PLANES == 1) loss_grad_x<T, 2, 2, 2, 2, 6, 2><<<grid, 512, 0, s>>>(a, x_tiles);
                else loss_grad_x<T, 2, 2, 2, 2, 3><<<grid, 256, 0, s>>>(a, x_tiles);
            }
        }
        if (!one_pass && !whole) {
            if (gq) {
                a.splits++; // and `fix`
                finish(Yes{}, No{}, 0);
            } else {
                finish(No{}, No{}, 0);
            }
        }
    }
    APOE_HIP(hipGetLastError());
    return APOE_OK;
}

int launch_softmax_loss(apoe_ctx* ctx, const apoe_softmax_loss_args* p) {
    switch (p->dtype) {
    case APOE_F32: return run_loss<float>(ctx, p);
    case APOE_F16: return run_loss<_Float16>(ctx, p);
    default: return run_loss<__bf16>(ctx, p);
    }
}

} // namespace apoe
