// Weighted sums of a table's rows, and the gradients of the table and of the weights:
//   out_i = base_i + s sum_e val_e T[idx_e] over the entries of row i,  gT[r] = s sum_{e: idx_e = r} val_e g[row e],  gval_e = s <T[idx_e], g[row e]>.
//
// Bound by memory: forward reads a row of the table for every entry (what is named often comes from the caches) and writes a row of out; the
// table's gradient reads g once an entry and writes the table. A row is held in registers by a group of G threads; four entries' rows are asked
// for at once. Few rows with many entries each: a workgroup's groups share a row's entries and join their sums.
// The table's gradient sorts the entries by the row that they name (a stable radix sort of up to 8 bits a pass: what two entries with the same name
// are added up in never changes), then walks over them in blocks of 32: a row whose entries lie in one block is written directly, of one that
// crosses blocks each block leaves its part, and a last launch adds the parts up in order. So a token that is a tenth of all entries costs what
// its rows' bytes cost, and no atomic changes a bit between two calls.
// Measured: 65 536 bf16 tokens of 1024 columns, table of 30 522 rows: forward 41 us (134 MB written, 62 read at least: 4.8 TB/s), gradient 90: sort 25 (four launches),
// walk 56 (212 MB: 3.8 TB/s; rows in order 47), join 8; every entry the same row: join 43. 777 float queries of 40 terms: forward 26, weights 22 (127 MB each
// through the L2 and what lies behind), sort 24, walk 31, join 10. 32 fp16 queries of 40 terms 7 us.
#include <algorithm>

#include "apoe_internal.h"
#include "apoe_rows.h"

namespace apoe {

constexpr uint32_t EMBED_BLOCK = 32;     // entries that one group adds up, at most (and the lanes that hold their names)
constexpr uint32_t SORT_TILE = 1024;     // entries that a workgroup of the sort ranks at a time
constexpr uint32_t SORT_ONE = 4096;      // entries that one workgroup sorts by itself
constexpr uint32_t SORT_TILES = 1024;    // workgroups of the sort, at most
constexpr uint32_t ROW_STARTS = 2048;    // places where rows begin that a workgroup of the sort keeps in LDS
constexpr uint32_t NO_ROW = 0xffffffffu;

using f32x4e = float __attribute__((ext_vector_type(4)));

struct Entry { // sorted: the row of the table, the row of g, and the weight
    uint32_t key, row;
    float val;
    uint32_t pad;
};

struct EmbedArgs {
    apoe_embed_args p;
    uint2 *pairs[2];   // key and entry, between passes
    Entry* sorted;
    uint32_t* counts;  // [tiles][256]
    uint32_t tile_entries, tiles;
    float* part;       // [blocks][2][part_pitch]: what a block's first and last row have in it, where they go on in other blocks
    uint32_t block, blocks, part_pitch; // block: entries of one
};

// S groups share a row's entries, in turn, and are the workgroup's threads; with S = 1 a workgroup has as many rows as groups.
template <typename T, int V, int G, bool WHOLE, int S> __global__ __launch_bounds__(S > 1 ? S * G : (G > 256 ? G : 256)) void embed_rows(apoe_embed_args p) {
    using R = RowOf<T, V, G, WHOLE>;
    constexpr int THREADS = S > 1 ? S * G : (G > 256 ? G : 256), GROUPS = S > 1 ? 1 : THREADS / G, U = 4;
    __shared__ float sums[S > 1 ? S * G * ROW_E : 1];
    const int t = threadIdx.x % G, group = threadIdx.x / G;
    for (uint64_t row = (uint64_t)blockIdx.x * GROUPS + (S > 1 ? 0 : group); row < p.n_rows; row += (uint64_t)gridDim.x * GROUPS) {
        uint32_t begin = (uint32_t)row, end = (uint32_t)row + 1;
        if (p.off) {
            end = min(p.off[row + 1], p.n_entries);
            begin = min(p.off[row], end);
        }
        float acc[ROW_E] = {};
        for (uint64_t e = (uint64_t)begin + (S > 1 ? group : 0); e < end; e += S * U) {
            typename R::tv raw[U][R::C];
            float w[U];
            uint32_t id[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const uint64_t at = e + u * S;
                id[u] = at < end ? p.idx[at] : NO_ROW;
                w[u] = at < end && p.val ? p.val[at] : 1.f;
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (id[u] < p.n_table) {
                    R::fetch(raw[u], p.table, id[u], p.table_stride, p.dim, t);
                } else {
                    w[u] = 0.f;
#pragma unroll
                    for (int c = 0; c < R::C; c++) raw[u][c] = typename R::tv{};
                }
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                float x[ROW_E];
                R::widen(x, raw[u]);
#pragma unroll
                for (int k = 0; k < ROW_E; k++) acc[k] = __builtin_fmaf(w[u], x[k], acc[k]);
            }
        }
        if constexpr (S > 1) {
            __syncthreads();
#pragma unroll
            for (int c = 0; c < R::C; c++)
#pragma unroll
                for (int k = 0; k < V; k++) sums[group * G * ROW_E + (c * G + t) * V + k] = acc[c * V + k];
            __syncthreads();
            for (uint32_t d = threadIdx.x; d < p.dim; d += THREADS) {
                float s = sums[d];
#pragma unroll
                for (int g = 1; g < S; g++) s += sums[g * G * ROW_E + d];
                s *= p.scale;
                if (p.base) s += (float)((const T*)p.base)[row * p.base_stride + d];
                ((T*)p.out)[row * p.out_stride + d] = (T)s;
            }
        } else {
            float b[ROW_E] = {};
            if (p.base) R::load(b, p.base, row, p.base_stride, p.dim, t);
#pragma unroll
            for (int k = 0; k < ROW_E; k++) acc[k] = __builtin_fmaf(p.scale, acc[k], b[k]);
            R::store(p.out, row, p.out_stride, p.dim, t, acc);
        }
    }
}

// One number an entry: the entries of a row in turn by blockIdx.y.
template <typename T, int V, int G, bool WHOLE> __global__ __launch_bounds__(G > 256 ? G : 256) void embed_weights(apoe_embed_args p) {
    using R = RowOf<T, V, G, WHOLE>;
    constexpr int GROUPS = (G > 256 ? G : 256) / G, U = 4;
    __shared__ float buf[U][8];
    const int t = threadIdx.x % G;
    for (uint64_t row = (uint64_t)blockIdx.x * GROUPS + threadIdx.x / G; row < p.n_rows; row += (uint64_t)gridDim.x * GROUPS) {
        uint32_t begin = (uint32_t)row, end = (uint32_t)row + 1;
        if (p.off) {
            end = min(p.off[row + 1], p.n_entries);
            begin = min(p.off[row], end);
        }
        float g[ROW_E];
        R::load(g, p.grad, row, p.grad_stride, p.dim, t);
        for (uint64_t e = (uint64_t)begin + (uint64_t)blockIdx.y * U; e < end; e += (uint64_t)gridDim.y * U) {
            typename R::tv raw[U][R::C];
            bool on[U];
            uint32_t id[U];
#pragma unroll
            for (int u = 0; u < U; u++) id[u] = e + u < end ? p.idx[e + u] : NO_ROW;
#pragma unroll
            for (int u = 0; u < U; u++) {
                on[u] = id[u] < p.n_table;
                if (on[u]) {
                    R::fetch(raw[u], p.table, id[u], p.table_stride, p.dim, t);
                } else {
#pragma unroll
                    for (int c = 0; c < R::C; c++) raw[u][c] = typename R::tv{};
                }
            }
            float s[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                float x[ROW_E];
                R::widen(x, raw[u]);
                s[u] = 0.f;
#pragma unroll
                for (int k = 0; k < ROW_E; k++) s[u] = __builtin_fmaf(x[k], g[k], s[u]);
            }
            group_sum<G, U>(s, buf);
#pragma unroll
            for (int u = 0; u < U; u++)
                if (t == u && e + u < end) p.grad_val[e + u] = on[u] ? s[u] * p.scale : 0.f;
        }
    }
    if (p.off) { // entries in front of the first row and behind the last one
        const uint32_t last = min(p.off[p.n_rows], p.n_entries), first = min(p.off[0], last);
        const uint64_t at = ((uint64_t)blockIdx.y * gridDim.x + blockIdx.x) * blockDim.x + threadIdx.x, step = (uint64_t)gridDim.x * gridDim.y * blockDim.x;
        for (uint64_t e = at; e < first; e += step) p.grad_val[e] = 0.f;
        for (uint64_t e = last + at; e < p.n_entries; e += step) p.grad_val[e] = 0.f;
    }
}

// ---- the sort ----

__device__ inline uint2 pair_of(const EmbedArgs& a, const uint2* from, uint64_t e) {
    if (from) return from[e];
    return uint2{min(a.p.idx[e], a.p.n_table), (uint32_t)e};
}

__global__ __launch_bounds__(256) void embed_count(EmbedArgs a, const uint2* from, uint32_t shift, uint32_t mask) {
    __shared__ uint32_t n[256];
    n[threadIdx.x] = 0;
    __syncthreads();
    const uint64_t begin = (uint64_t)blockIdx.x * a.tile_entries, end = min(begin + a.tile_entries, (uint64_t)a.p.n_entries);
    constexpr int U = SORT_TILE / 256;
    for (uint64_t e = begin + threadIdx.x; e < end + threadIdx.x; e += SORT_TILE) {
        uint32_t key[U];
#pragma unroll
        for (int u = 0; u < U; u++) key[u] = pair_of(a, from, min(e + u * 256, end - 1)).x;
#pragma unroll
        for (int u = 0; u < U; u++)
            if (e + u * 256 < end) atomicAdd(&n[(key[u] >> shift) & mask], 1u); // whole numbers: in any order
    }
    __syncthreads();
    a.counts[blockIdx.x * 256 + threadIdx.x] = n[threadIdx.x];
}

// Ranks of a wave's items among those of the same digit before them, round by round; `seen` counts the wave's items of each digit.
template <int ROUNDS> __device__ inline void rank_in_wave(const uint2* item, const bool* in, uint32_t* rank, volatile uint32_t* seen, uint32_t shift, uint32_t mask, int lane) {
    for (int k = lane; k < 256; k += 64) seen[k] = 0;
#pragma unroll
    for (int r = 0; r < ROUNDS; r++) {
        const uint32_t digit = (item[r].x >> shift) & mask;
        uint64_t same = __ballot(in[r]);
#pragma unroll
        for (int b = 0; b < 8; b++) {
            const uint64_t set = __ballot((digit >> b) & 1);
            same &= (digit >> b) & 1 ? set : ~set;
        }
        const uint64_t below = same & ((1ull << lane) - 1);
        rank[r] = in[r] ? seen[digit] + (uint32_t)__popcll(below) : 0;
        if (in[r] && below == 0) seen[digit] = rank[r] + (uint32_t)__popcll(same); // one lane a digit; a wave's LDS accesses keep their order
    }
}

// Sums of all smaller digits' counts, for 256 threads of a larger workgroup or all of them.
__device__ inline void scan256(uint32_t* total, int tid) {
    for (int d = 1; d < 256; d <<= 1) {
        const uint32_t v = tid < 256 && tid >= d ? total[tid - d] : 0;
        __syncthreads();
        if (tid < 256) total[tid] += v;
        __syncthreads();
    }
}

// Where rows begin, every 2^shift-th of them: what a search of them starts with. Searched in LDS, where a step waits for no memory (31 080
// entries of 777 rows, the whole launch: 13.0 us with every step in memory, 8.2 so).
__device__ inline uint32_t starts_shift(uint32_t n_rows) {
    uint32_t s = 0;
    while ((n_rows >> s) >= ROW_STARTS) s++;
    return s;
}
template <int THREADS> __device__ inline void fill_starts(const EmbedArgs& a, uint32_t* starts, int tid) {
    if (!a.p.off) return;
    const uint32_t shift = starts_shift(a.p.n_rows);
#pragma unroll
    for (uint32_t k = 0; k < ROW_STARTS / THREADS; k++) {
        const uint32_t i = k * THREADS + tid;
        starts[i] = a.p.off[min(i << shift, a.p.n_rows - 1)];
    }
}

// Each item's row, the last one that begins at or before it, and weight, to its place. The searches of all rounds go step by step together: a step waits for one
// load, not for ROUNDS.
template <int ROUNDS> __device__ inline void put_entries(const EmbedArgs& a, const uint2* item, const bool* in, const uint32_t* place, const uint32_t* starts) {
    uint32_t row[ROUNDS];
    float val[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; r++) {
        row[r] = item[r].y;
        val[r] = in[r] && a.p.val ? a.p.val[item[r].y] : 1.f;
    }
    if (a.p.off) {
        const uint32_t n = a.p.n_rows, shift = starts_shift(n), last = (n - 1) >> shift;
#pragma unroll
        for (int r = 0; r < ROUNDS; r++) row[r] = 0;
        for (uint32_t step = ROW_STARTS / 2; step; step >>= 1)
#pragma unroll
            for (int r = 0; r < ROUNDS; r++) {
                const uint32_t to = min(row[r] + step, last);
                if (starts[to] <= item[r].y) row[r] = to;
            }
#pragma unroll
        for (int r = 0; r < ROUNDS; r++) row[r] <<= shift;
        for (uint32_t step = (1u << shift) >> 1; step; step >>= 1)
#pragma unroll
            for (int r = 0; r < ROUNDS; r++) {
                const uint32_t to = min(row[r] + step, n - 1); // off[to] of the last row says where that begins
                if (a.p.off[to] <= item[r].y) row[r] = to;
            }
#pragma unroll
        for (int r = 0; r < ROUNDS; r++)
            if (!(a.p.off[row[r]] <= item[r].y && item[r].y < a.p.off[row[r] + 1])) row[r] = NO_ROW;
    }
#pragma unroll
    for (int r = 0; r < ROUNDS; r++)
        if (in[r]) a.sorted[place[r]] = Entry{item[r].x, row[r], val[r], 0};
}

// Every entry goes behind those with a smaller digit, and behind the earlier ones with the same. LAST: the last pass, which looks up rows and weights.
template <bool LAST> __global__ __launch_bounds__(256) void embed_place(EmbedArgs a, const uint2* from, uint2* to, uint32_t shift, uint32_t mask) {
    constexpr int WAVES = 4, ROUNDS = SORT_TILE / (64 * WAVES);
    __shared__ uint32_t next[256], total[256];
    __shared__ uint32_t seen[WAVES][256]; // per wave: entries of a digit so far, then where its first one goes
    __shared__ uint32_t starts[LAST ? ROW_STARTS : 1];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if constexpr (LAST) fill_starts<256>(a, starts, tid);
    uint32_t all = 0, before = 0;
    for (uint32_t t0 = 0; t0 < a.tiles; t0 += 16) { // sixteen loads at once, beyond the last tile that one again
        uint32_t n[16];
#pragma unroll
        for (uint32_t u = 0; u < 16; u++) n[u] = a.counts[min(t0 + u, a.tiles - 1) * 256 + tid];
#pragma unroll
        for (uint32_t u = 0; u < 16; u++) {
            const uint32_t c = t0 + u < a.tiles ? n[u] : 0;
            all += c;
            before += t0 + u < blockIdx.x ? c : 0;
        }
    }
    total[tid] = all;
    __syncthreads();
    scan256(total, tid);
    next[tid] = total[tid] - all + before;
    const uint64_t begin = (uint64_t)blockIdx.x * a.tile_entries, end = min(begin + a.tile_entries, (uint64_t)a.p.n_entries);
    for (uint64_t tile = begin; tile < end; tile += SORT_TILE) {
        uint2 item[ROUNDS];
        uint32_t rank[ROUNDS];
        bool in[ROUNDS];
#pragma unroll
        for (int r = 0; r < ROUNDS; r++) {
            const uint64_t e = tile + wave * (64 * ROUNDS) + r * 64 + lane;
            in[r] = e < end;
            item[r] = in[r] ? pair_of(a, from, e) : uint2{0, 0};
        }
        rank_in_wave<ROUNDS>(item, in, rank, seen[wave], shift, mask, lane);
        __syncthreads();
        uint32_t at = next[tid];
        for (int w = 0; w < WAVES; w++) {
            const uint32_t n = seen[w][tid];
            seen[w][tid] = at;
            at += n;
        }
        next[tid] = at;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < ROUNDS; r++) {
            rank[r] += seen[wave][(item[r].x >> shift) & mask];
            if constexpr (!LAST)
                if (in[r]) to[rank[r]] = item[r];
        }
        if constexpr (LAST) put_entries<ROUNDS>(a, item, in, rank, starts);
        __syncthreads(); // the next tile clears the counts
    }
}

// Few entries: every pass in one workgroup's LDS.
__global__ __launch_bounds__(1024) void embed_sort(EmbedArgs a, uint32_t passes, uint32_t width) {
    constexpr int WAVES = 16, ROUNDS = SORT_ONE / (64 * WAVES);
    __shared__ uint2 items[SORT_ONE];
    __shared__ uint32_t total[256];
    __shared__ uint32_t seen[WAVES][256];
    __shared__ uint32_t starts[ROW_STARTS];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t n = a.p.n_entries, mask = (1u << width) - 1;
    fill_starts<1024>(a, starts, tid); // (every pass has barriers between this and its use)
    uint2 item[ROUNDS];
    uint32_t rank[ROUNDS];
    bool in[ROUNDS];
    for (uint32_t pass = 0; pass < passes; pass++) {
        const uint32_t shift = pass * width;
#pragma unroll
        for (int r = 0; r < ROUNDS; r++) {
            const uint32_t e = wave * (64 * ROUNDS) + r * 64 + lane;
            in[r] = e < n;
            item[r] = in[r] ? (pass ? items[e] : pair_of(a, nullptr, e)) : uint2{0, 0};
        }
        rank_in_wave<ROUNDS>(item, in, rank, seen[wave], shift, mask, lane);
        __syncthreads();
        uint32_t all = 0;
        if (tid < 256) {
            for (int w = 0; w < WAVES; w++) all += seen[w][tid];
            total[tid] = all;
        }
        __syncthreads();
        scan256(total, tid);
        if (tid < 256) {
            uint32_t at = total[tid] - all;
            for (int w = 0; w < WAVES; w++) {
                const uint32_t k = seen[w][tid];
                seen[w][tid] = at;
                at += k;
            }
        }
        __syncthreads();
        const bool last = pass + 1 == passes;
#pragma unroll
        for (int r = 0; r < ROUNDS; r++) {
            rank[r] += seen[wave][(item[r].x >> shift) & mask];
            if (in[r] && !last) items[rank[r]] = item[r];
        }
        if (last) put_entries<ROUNDS>(a, item, in, rank, starts);
        __syncthreads();
    }
}

// ---- the table's gradient ----

// First sorted entry whose key is at least `key`.
__device__ inline uint32_t first_at_least(const Entry* sorted, uint32_t lo, uint32_t hi, uint32_t key) {
    while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (sorted[mid].key < key) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

template <typename T, int V, int G, bool WHOLE> __device__ inline void put_table_row(const apoe_embed_args& p, uint32_t key, int t, const float* sum) {
    using R = RowOf<T, V, G, WHOLE>;
    float v[ROW_E];
    if (p.accumulate) {
        R::load(v, p.grad_table, key, p.grad_table_stride, p.dim, t);
#pragma unroll
        for (int k = 0; k < ROW_E; k++) v[k] = __builtin_fmaf(p.scale, sum[k], v[k]);
    } else {
#pragma unroll
        for (int k = 0; k < ROW_E; k++) v[k] = p.scale * sum[k];
    }
    R::store(p.grad_table, key, p.grad_table_stride, p.dim, t, v);
}

// The first workgroups: a group a block of entries. The others: zeros for the rows that no entry names, 64 of the table a workgroup.
template <typename T, int V, int G, bool WHOLE> __global__ __launch_bounds__(G > 256 ? G : 256) void embed_table(EmbedArgs a, uint32_t entry_groups) {
    using R = RowOf<T, V, G, WHOLE>;
    constexpr int THREADS = G > 256 ? G : 256, GROUPS = THREADS / G, U = sizeof(T) == 4 ? 2 : 4;
    const apoe_embed_args& p = a.p;
    const int t = threadIdx.x % G, group = threadIdx.x / G;
    if (blockIdx.x >= entry_groups) {
        __shared__ uint32_t named[64];
        const float zero[ROW_E] = {};
        for (uint64_t row0 = (uint64_t)(blockIdx.x - entry_groups) * 64; row0 < p.n_table; row0 += (uint64_t)(gridDim.x - entry_groups) * 64) {
            __syncthreads();
            if (threadIdx.x < 64) {
                const uint64_t row = row0 + threadIdx.x;
                bool found = true;
                if (row < p.n_table) {
                    const uint32_t at = first_at_least(a.sorted, 0, p.n_entries, (uint32_t)row);
                    found = at < p.n_entries && a.sorted[at].key == row;
                }
                named[threadIdx.x] = found;
            }
            __syncthreads();
            for (int r = group; r < 64; r += GROUPS)
                if (!named[r]) R::store(p.grad_table, row0 + r, p.grad_table_stride, p.dim, t, zero);
        }
        return;
    }
    const uint32_t block = blockIdx.x * GROUPS + group;
    if (block >= a.blocks) return;
    const uint32_t begin = block * a.block, n = min(a.block, p.n_entries - begin);
    constexpr int WIDTH = G < 64 ? G : 64; // every lane holds one entry of the block
    const int l = threadIdx.x % WIDTH;
    const Entry mine = a.sorted[begin + min((uint32_t)l, n - 1)];
    const uint32_t in_front = begin ? a.sorted[begin - 1].key : NO_ROW, behind = begin + n < p.n_entries ? a.sorted[begin + n].key : NO_ROW;
    const auto key_of = [&](uint32_t e) { return (uint32_t)__shfl((int)mine.key, (int)e, WIDTH); };
    uint32_t key = key_of(0);
    bool goes_on = in_front == key; // the row began in an earlier block
    float acc[ROW_E] = {};
    auto leave = [&](bool last) {
        if (key >= p.n_table) return;
        if (!goes_on && !(last && behind == key)) {
            put_table_row<T, V, G, WHOLE>(p, key, t, acc);
            return;
        }
        float* out = a.part + ((size_t)block * 2 + (goes_on ? 0 : 1)) * a.part_pitch;
#pragma unroll
        for (int c = 0; c < R::C; c++)
#pragma unroll
            for (int k = 0; k < V; k++) {
                const uint32_t d = (c * G + t) * V + k;
                if (d < a.part_pitch) out[d] = acc[c * V + k]; // zeros behind the row's end
            }
    };
    typename R::tv raw[2][U][R::C]; // the next entries' rows are asked for before these are added up
    float w[2][U];
    auto ask = [&](uint32_t e, auto side) {
        constexpr int Q = decltype(side)::value;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int at = (int)min(e + u, n - 1);
            const uint32_t row = (uint32_t)__shfl((int)mine.row, at, WIDTH), k = key_of(at);
            w[Q][u] = __shfl(mine.val, at, WIDTH);
            if (e + u < n && row < p.n_rows && k < p.n_table) {
                R::fetch(raw[Q][u], p.grad, row, p.grad_stride, p.dim, t);
            } else {
                w[Q][u] = 0.f;
#pragma unroll
                for (int c = 0; c < R::C; c++) raw[Q][u][c] = typename R::tv{};
            }
        }
    };
    auto add = [&](uint32_t e, auto side) {
        constexpr int Q = decltype(side)::value;
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (e + u >= n) break;
            const uint32_t k0 = key_of(e + u);
            if (k0 != key) {
                leave(false);
                key = k0;
                goes_on = false;
#pragma unroll
                for (int k = 0; k < ROW_E; k++) acc[k] = 0.f;
            }
            float x[ROW_E];
            R::widen(x, raw[Q][u]);
#pragma unroll
            for (int k = 0; k < ROW_E; k++) acc[k] = __builtin_fmaf(w[Q][u], x[k], acc[k]);
        }
    };
    const std::integral_constant<int, 0> even;
    const std::integral_constant<int, 1> odd;
    ask(0, even);
    for (uint32_t e = 0; e < n; e += 2 * U) {
        if (e + U < n) ask(e + U, odd);
        add(e, even);
        if (e + 2 * U < n) ask(e + 2 * U, even);
        if (e + U < n) add(e + U, odd);
    }
    leave(true);
}

// Rows whose entries lie in more than one block: a wave takes one that begins in its block, 256 columns by blockIdx.y. Long ones (a token that is
// everywhere) are added up by the workgroup's waves together.
template <typename T> __global__ __launch_bounds__(1024) void embed_join(EmbedArgs a) {
    constexpr uint32_t WAVES = 16, LONG = 16;
    __shared__ uint32_t later[WAVES], later_key[WAVES];
    __shared__ __align__(16) float sums[WAVES][256];
    const apoe_embed_args& p = a.p;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t block = blockIdx.x * WAVES + wave, d0 = blockIdx.y * 256;
    uint32_t parts = 0, key = 0; // blocks after this one that have a part of the row
    auto look = [&](uint32_t b) {
        parts = 0;
        const uint64_t end = (uint64_t)(b + 1) * a.block;
        if (b >= a.blocks || end >= p.n_entries) return;
        const uint32_t begin = b * a.block;
        key = a.sorted[end - 1].key;
        const uint32_t next = a.sorted[end].key, first = a.sorted[begin].key, in_front = begin ? a.sorted[begin - 1].key : NO_ROW;
        if (key >= p.n_table || next != key) return;
        if (first == key && in_front == key) return; // it began earlier
        // the last block that has a part: the wave's lanes look at 64 places at once, in strides that grow until one is beyond, then shrink
        uint64_t has = b + 1, stride = 1;
        const auto reach = [&]() {
            const uint64_t c = has + stride * (lane + 1); // block c has a part where the row's name is its first one
            const uint64_t yes = __ballot(c < a.blocks && a.sorted[c * a.block].key == key);
            has += stride * __popcll(yes);
            return yes == ~0ull;
        };
        while (reach()) stride *= 64;
        while (stride > 1) {
            stride /= 64;
            reach();
        }
        parts = (uint32_t)(has - b);
    };
    // Parts `first`, `first` + step, .. of the row that begins in block b, four columns a lane: eight rows are asked for at once, beyond the last one
    // that one again, which is not counted (a load under a condition would be waited for before the next is sent).
    auto add = [&](uint32_t b, uint32_t first, uint32_t step) {
        const uint32_t last = __builtin_amdgcn_readfirstlane(parts);
        const float* column = a.part + min(d0 + lane * 4, a.part_pitch - 4);
        f32x4e s = {};
        for (uint32_t k = first; k <= last; k += 8 * step) {
            f32x4e x[8];
#pragma unroll
            for (int u = 0; u < 8; u++) {
                const uint32_t q = min(k + u * step, last);
                x[u] = *reinterpret_cast<const f32x4e*>(column + ((size_t)(b + q) * 2 + (q ? 0 : 1)) * a.part_pitch);
            }
#pragma unroll
            for (int u = 0; u < 8; u++) s += k + u * step <= last ? x[u] : f32x4e{};
        }
        return s;
    };
    auto put = [&](uint32_t d, float s) {
        if (d >= p.dim) return;
        T* at = (T*)p.grad_table + (uint64_t)key * p.grad_table_stride + d;
        s *= p.scale;
        *at = (T)(p.accumulate ? s + (float)*at : s);
    };
    look(block);
    if (lane == 0) {
        later[wave] = parts > LONG ? parts : 0;
        later_key[wave] = key;
    }
    if (parts && parts <= LONG) {
        const f32x4e s = add(block, 0, 1);
#pragma unroll
        for (int c = 0; c < 4; c++) put(d0 + lane * 4 + c, s[c]);
    }
    __syncthreads();
    for (uint32_t w = 0; w < WAVES; w++) {
        parts = later[w];
        if (!parts) continue;
        key = later_key[w];
        const f32x4e s = add(blockIdx.x * WAVES + w, wave, WAVES);
        __syncthreads();
        *reinterpret_cast<f32x4e*>(&sums[wave][lane * 4]) = s;
        __syncthreads();
        if (threadIdx.x < 256) {
            float v = 0.f;
            for (uint32_t k = 0; k < WAVES; k++) v += sums[k][threadIdx.x];
            put(d0 + threadIdx.x, v);
        }
    }
}

template <typename T, int V, bool WHOLE> static int run_embed(apoe_ctx* ctx, const apoe_embed_args* p) {
    hipStream_t s = ctx->stream;
    // Few rows with many entries each: groups share a row, so that the GPU has some 16 waves a CU to wait for memory with, and each at least two entries.
    return with_group(p->dim, [&](auto size) -> int {
        constexpr int G = decltype(size)::value, THREADS = G > 256 ? G : 256, MOST = 1024 / G < 16 ? 1024 / G : 16;
        const uint64_t waves = (uint64_t)p->n_rows * (G > 64 ? G / 64 : 1), room = (uint64_t)ctx->num_cus * 16;
        const auto shared_by = [&](uint64_t groups) { return p->n_entries >= (uint64_t)p->n_rows * groups * 2 && waves * groups <= room * 4; };
        if (shared_by(MOST)) {
            embed_rows<T, V, G, WHOLE, MOST><<<p->n_rows, MOST * G, 0, s>>>(*p);
            return APOE_OK;
        }
        if constexpr (MOST > 4) {
            if (shared_by(4)) {
                embed_rows<T, V, G, WHOLE, 4><<<p->n_rows, 4 * G, 0, s>>>(*p);
                return APOE_OK;
            }
        }
        const uint64_t need = ((uint64_t)p->n_rows + THREADS / G - 1) / (THREADS / G);
        embed_rows<T, V, G, WHOLE, 1><<<(uint32_t)std::min<uint64_t>(need, 1u << 20), THREADS, 0, s>>>(*p);
        return APOE_OK;
    });
}

template <typename T, int V, bool WHOLE> static int run_embed_grad(apoe_ctx* ctx, const apoe_embed_args* p) {
    hipStream_t s = ctx->stream;
    if (p->grad_val && p->n_rows && p->n_entries) {
        APOE_TRY(with_group(p->dim, [&](auto size) -> int {
            constexpr int G = decltype(size)::value, THREADS = G > 256 ? G : 256;
            const uint64_t need = ((uint64_t)p->n_rows + THREADS / G - 1) / (THREADS / G);
            // few rows: their entries in turn by up to 16 workgroups
            const uint32_t share = (uint32_t)std::min<uint64_t>(16, std::max<uint64_t>(1, std::min<uint64_t>((uint64_t)ctx->num_cus * 8 / need, p->n_entries / (p->n_rows * 4ull))));
            embed_weights<T, V, G, WHOLE><<<dim3((uint32_t)std::min<uint64_t>(need, 1u << 20), share), THREADS, 0, s>>>(*p);
            return APOE_OK;
        }));
    }
    if (!p->grad_table || p->n_table == 0) return APOE_OK;
    if (p->n_entries == 0 && p->accumulate) return APOE_OK;
    EmbedArgs a{};
    a.p = *p;
    const uint64_t n = p->n_entries;
    a.tile_entries = (uint32_t)(((n + SORT_TILES - 1) / SORT_TILES + SORT_TILE - 1) / SORT_TILE * SORT_TILE);
    a.tiles = n ? (uint32_t)((n + a.tile_entries - 1) / a.tile_entries) : 0;
    // Some 8 waves a CU, of 8 to 32 entries each (16: groups of 16 lanes): smaller blocks fill the GPU, larger ones cut fewer rows (launch that walks and
    // launch that joins, us: 31 080 float entries of 1024 columns, blocks of 8 30 + 37, 16 31 + 24, 32 45 + 23; 65 536 bf16 ones, 16 62 + 39, 32 57 + 25).
    const uint32_t most = p->dim <= 16 * ROW_E ? 16 : EMBED_BLOCK;
    a.block = (uint32_t)std::min<uint64_t>(most, std::max<uint64_t>(8, (n / ((uint64_t)ctx->num_cus * 8) + 2) / 4 * 4));
    a.blocks = (uint32_t)((n + a.block - 1) / a.block);
    a.part_pitch = (p->dim + 3) / 4 * 4;
    const size_t records = n * sizeof(Entry), pairs = n * sizeof(uint2), counts = (size_t)a.tiles * 256 * 4;
    char* ws = nullptr;
    APOE_TRY(ctx->adapt_workspace(records + 2 * pairs + counts + (size_t)a.blocks * 2 * a.part_pitch * 4 + 64, &ws));
    a.sorted = (Entry*)ws;
    a.pairs[0] = (uint2*)(ws + records);
    a.pairs[1] = a.pairs[0] + n;
    a.counts = (uint32_t*)(ws + records + 2 * pairs);
    a.part = (float*)(ws + (records + 2 * pairs + counts + 15) / 16 * 16);
    uint32_t bits = 1;
    while (bits < 32 && (p->n_table >> bits)) bits++; // keys go to n_table
    const uint32_t passes = (bits + 7) / 8, width = (bits + passes - 1) / passes;
    if (n && n <= SORT_ONE) {
        embed_sort<<<1, 1024, 0, s>>>(a, passes, width);
    } else if (n) {
        const uint2* from = nullptr;
        for (uint32_t pass = 0; pass < passes; pass++) {
            const uint32_t shift = pass * width, mask = (1u << width) - 1;
            embed_count<<<a.tiles, 256, 0, s>>>(a, from, shift, mask);
            if (pass + 1 < passes) embed_place<false><<<a.tiles, 256, 0, s>>>(a, from, a.pairs[pass & 1], shift, mask);
            else embed_place<true><<<a.tiles, 256, 0, s>>>(a, from, nullptr, shift, mask);
            from = a.pairs[pass & 1];
        }
    }
    APOE_TRY(with_group(p->dim, [&](auto size) -> int {
        constexpr int G = decltype(size)::value, THREADS = G > 256 ? G : 256;
        const uint32_t entry_groups = (a.blocks + THREADS / G - 1) / (THREADS / G), zero_groups = p->accumulate ? 0 : std::min((p->n_table + 63) / 64, 1u << 20);
        embed_table<T, V, G, WHOLE><<<entry_groups + zero_groups, THREADS, 0, s>>>(a, entry_groups);
        return APOE_OK;
    }));
    if (a.blocks > 1) embed_join<T><<<dim3((a.blocks + 15) / 16, (p->dim + 255) / 256), 1024, 0, s>>>(a);
    return APOE_OK;
}

template <typename T> static int run_aligned(apoe_ctx* ctx, const apoe_embed_args* p, bool grad) {
    constexpr int V = 16 / (int)sizeof(T);
    bool whole = p->dim % V == 0;
    for (const void* q : {p->table, p->base, (const void*)p->out, p->grad, (const void*)p->grad_table}) whole &= ((uintptr_t)q & 15) == 0;
    for (uint64_t q : {p->table_stride, p->base_stride, p->out_stride, p->grad_stride, p->grad_table_stride}) whole &= q % V == 0;
    if (grad) APOE_TRY(whole ? (run_embed_grad<T, V, true>(ctx, p)) : (run_embed_grad<T, V, false>(ctx, p)));
    else APOE_TRY(whole ? (run_embed<T, V, true>(ctx, p)) : (run_embed<T, V, false>(ctx, p)));
    APOE_HIP(hipGetLastError());
    return APOE_OK;
}

int launch_embed(apoe_ctx* ctx, const apoe_embed_args* p, bool grad) {
    switch (p->dtype) {
    case APOE_F32: return run_aligned<float>(ctx, p, grad);
    case APOE_F16: return run_aligned<_Float16>(ctx, p, grad);
    default: return run_aligned<__bf16>(ctx, p, grad);
    }
}

} // namespace apoe
