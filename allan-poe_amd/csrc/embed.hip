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
#include <algorithm>

#include "apoe_internal.h"
#include "apoe_rows.h"

namespace apoe {

constexpr uint32_t EMBED_BLOCK = 32;     // entries that one group adds up
constexpr uint32_t SORT_TILE = 4096;     // entries that a workgroup of the sort ranks at a time
constexpr uint32_t SORT_TILES = 1024;    // workgroups of the sort, at most
constexpr uint32_t NO_ROW = 0xffffffffu;

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
    uint32_t blocks, part_pitch;
};

// WIDE: a workgroup of 1024 threads a row, whose groups take its entries in turn; otherwise a group a row.
template <typename T, int V, int G, bool WIDE> __global__ __launch_bounds__(WIDE ? 1024 : (G > 256 ? G : 256)) void embed_rows(apoe_embed_args p) {
    using R = RowOf<T, V, G>;
    constexpr int THREADS = WIDE ? 1024 : (G > 256 ? G : 256), GROUPS = THREADS / G, S = WIDE ? GROUPS : 1, U = 4;
    __shared__ float sums[WIDE ? GROUPS * G * ROW_E : 1];
    const int t = threadIdx.x % G, group = threadIdx.x / G;
    for (uint64_t row = WIDE ? blockIdx.x : (uint64_t)blockIdx.x * GROUPS + group; row < p.n_rows; row += WIDE ? gridDim.x : (uint64_t)gridDim.x * GROUPS) {
        uint32_t begin = (uint32_t)row, end = (uint32_t)row + 1;
        if (p.off) {
            end = min(p.off[row + 1], p.n_entries);
            begin = min(p.off[row], end);
        }
        float acc[ROW_E] = {};
        for (uint64_t e = (uint64_t)begin + (WIDE ? group : 0); e < end; e += S * U) {
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
        if constexpr (WIDE) {
            __syncthreads();
#pragma unroll
            for (int c = 0; c < R::C; c++)
#pragma unroll
                for (int k = 0; k < V; k++) sums[group * G * ROW_E + (c * G + t) * V + k] = acc[c * V + k];
            __syncthreads();
            for (uint32_t d = threadIdx.x; d < p.dim; d += THREADS) {
                float s = sums[d];
#pragma unroll
                for (int g = 1; g < GROUPS; g++) s += sums[g * G * ROW_E + d];
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
template <typename T, int V, int G> __global__ __launch_bounds__(G > 256 ? G : 256) void embed_weights(apoe_embed_args p) {
    using R = RowOf<T, V, G>;
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
    for (uint64_t e = begin + threadIdx.x; e < end; e += 256) atomicAdd(&n[(pair_of(a, from, e).x >> shift) & mask], 1u); // whole numbers: in any order
    __syncthreads();
    a.counts[blockIdx.x * 256 + threadIdx.x] = n[threadIdx.x];
}

// Every entry goes behind those with a smaller digit, and behind the earlier ones with the same. TO: the last pass, which looks up rows and weights.
template <bool LAST> __global__ __launch_bounds__(256) void embed_place(EmbedArgs a, const uint2* from, uint2* to, uint32_t shift, uint32_t mask) {
    constexpr int WAVES = 4, ROUNDS = SORT_TILE / (64 * WAVES);
    __shared__ uint32_t next[256], total[256];
    __shared__ uint32_t seen[WAVES][256]; // per wave: entries of a digit so far, then where its first one goes
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint32_t all = 0, before = 0;
#pragma unroll 8
    for (uint32_t t = 0; t < a.tiles; t++) {
        const uint32_t n = a.counts[t * 256 + tid];
        all += n;
        before += t < blockIdx.x ? n : 0;
    }
    total[tid] = all;
    __syncthreads();
    for (int d = 1; d < 256; d <<= 1) {
        const uint32_t v = tid >= d ? total[tid - d] : 0;
        __syncthreads();
        total[tid] += v;
        __syncthreads();
    }
    next[tid] = total[tid] - all + before;
    const uint64_t begin = (uint64_t)blockIdx.x * a.tile_entries, end = min(begin + a.tile_entries, (uint64_t)a.p.n_entries);
    for (uint64_t tile = begin; tile < end; tile += SORT_TILE) {
        volatile uint32_t* mine = seen[wave];
        for (int k = lane; k < 256; k += 64) mine[k] = 0;
        uint2 item[ROUNDS];
        uint32_t rank[ROUNDS];
#pragma unroll
        for (int r = 0; r < ROUNDS; r++) {
            const uint64_t e = tile + wave * (64 * ROUNDS) + r * 64 + lane;
            item[r] = e < end ? pair_of(a, from, e) : uint2{0, 0};
        }
#pragma unroll
        for (int r = 0; r < ROUNDS; r++) {
            const bool in = tile + wave * (64 * ROUNDS) + r * 64 + lane < end;
            const uint32_t digit = (item[r].x >> shift) & mask;
            uint64_t same = __ballot(in);
#pragma unroll
            for (int b = 0; b < 8; b++) {
                const uint64_t set = __ballot((digit >> b) & 1);
                same &= (digit >> b) & 1 ? set : ~set;
            }
            const uint64_t below = same & ((1ull << lane) - 1);
            rank[r] = in ? mine[digit] + (uint32_t)__popcll(below) : 0;
            if (in && below == 0) mine[digit] = rank[r] + (uint32_t)__popcll(same); // one lane a digit; a wave's LDS accesses keep their order
        }
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
            if (tile + wave * (64 * ROUNDS) + r * 64 + lane >= end) continue;
            const uint32_t place = seen[wave][(item[r].x >> shift) & mask] + rank[r], e = item[r].y;
            if constexpr (LAST) {
                uint32_t row = e;
                if (a.p.off) { // the last row that begins at or before the entry
                    uint32_t lo = 0, hi = a.p.n_rows;
                    while (hi - lo > 1) {
                        const uint32_t mid = lo + (hi - lo) / 2;
                        if (a.p.off[mid] <= e) lo = mid;
                        else hi = mid;
                    }
                    row = a.p.n_rows && a.p.off[lo] <= e && e < a.p.off[lo + 1] ? lo : NO_ROW;
                }
                a.sorted[place] = Entry{item[r].x, row, a.p.val ? a.p.val[e] : 1.f, 0};
            } else {
                to[place] = item[r];
            }
        }
        __syncthreads(); // the next tile clears the counts
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

template <typename T, int V, int G> __device__ inline void put_table_row(const apoe_embed_args& p, uint32_t key, int t, const float* sum) {
    using R = RowOf<T, V, G>;
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
template <typename T, int V, int G> __global__ __launch_bounds__(G > 256 ? G : 256) void embed_table(EmbedArgs a, uint32_t entry_groups) {
    using R = RowOf<T, V, G>;
    constexpr int THREADS = G > 256 ? G : 256, GROUPS = THREADS / G, U = 4;
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
    const uint32_t begin = block * EMBED_BLOCK, end = min(begin + EMBED_BLOCK, p.n_entries);
    uint32_t key = a.sorted[begin].key;
    bool goes_on = begin > 0 && a.sorted[begin - 1].key == key; // the row began in an earlier block
    float acc[ROW_E] = {};
    auto leave = [&](bool last) {
        if (key >= p.n_table) return;
        const bool open = last && end < p.n_entries && a.sorted[end].key == key;
        if (!goes_on && !open) {
            put_table_row<T, V, G>(p, key, t, acc);
            return;
        }
        float* out = a.part + ((size_t)block * 2 + (goes_on ? 0 : 1)) * a.part_pitch;
#pragma unroll
        for (int c = 0; c < R::C; c++)
#pragma unroll
            for (int k = 0; k < V; k++) {
                const uint32_t d = (c * G + t) * V + k;
                if (d < p.dim) out[d] = acc[c * V + k];
            }
    };
    for (uint32_t e = begin; e < end; e += U) {
        Entry item[U];
        typename R::tv raw[U][R::C];
#pragma unroll
        for (int u = 0; u < U; u++) item[u] = a.sorted[min(e + u, end - 1)];
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (item[u].row < p.n_rows && item[u].key < p.n_table) {
                R::fetch(raw[u], p.grad, item[u].row, p.grad_stride, p.dim, t);
            } else {
                item[u].val = 0.f;
#pragma unroll
                for (int c = 0; c < R::C; c++) raw[u][c] = typename R::tv{};
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (e + u >= end) break;
            if (item[u].key != key) {
                leave(false);
                key = item[u].key;
                goes_on = false;
#pragma unroll
                for (int k = 0; k < ROW_E; k++) acc[k] = 0.f;
            }
            float x[ROW_E];
            R::widen(x, raw[u]);
#pragma unroll
            for (int k = 0; k < ROW_E; k++) acc[k] = __builtin_fmaf(item[u].val, x[k], acc[k]);
        }
    }
    leave(true);
}

// Rows whose entries lie in more than one block: a wave takes one that begins in its block, 256 columns by blockIdx.y. Long ones (a token that is
// everywhere) are added up by the workgroup's waves together.
template <typename T> __global__ __launch_bounds__(1024) void embed_join(EmbedArgs a) {
    constexpr uint32_t WAVES = 16, LONG = 16;
    __shared__ uint32_t later[WAVES];
    __shared__ float sums[WAVES][257];
    const apoe_embed_args& p = a.p;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t block = blockIdx.x * WAVES + wave, d0 = blockIdx.y * 256;
    uint32_t parts = 0, key = 0; // blocks after this one that have a part of the row
    auto look = [&](uint32_t b) {
        parts = 0;
        const uint64_t end = (uint64_t)(b + 1) * EMBED_BLOCK;
        if (b >= a.blocks || end >= p.n_entries) return;
        key = a.sorted[end - 1].key;
        const uint32_t begin = b * EMBED_BLOCK;
        if (key >= p.n_table || a.sorted[end].key != key) return;
        if (a.sorted[begin].key == key && begin > 0 && a.sorted[begin - 1].key == key) return; // it began earlier
        parts = (first_at_least(a.sorted, (uint32_t)end, p.n_entries, key + 1) - 1) / EMBED_BLOCK - b;
    };
    auto add = [&](uint32_t b, uint32_t first, uint32_t step, float* s) { // parts `first`, `first` + step, .. of the row that begins in block b
#pragma unroll 4
        for (uint32_t k = first; k <= parts; k += step) {
            const float* from = a.part + ((size_t)(b + k) * 2 + (k ? 0 : 1)) * a.part_pitch + d0;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const uint32_t d = c * 64 + lane;
                if (d0 + d < p.dim) s[c] += from[d];
            }
        }
    };
    auto put = [&](uint32_t d, float s) {
        if (d >= p.dim) return;
        T* at = (T*)p.grad_table + (uint64_t)key * p.grad_table_stride + d;
        s *= p.scale;
        *at = (T)(p.accumulate ? s + (float)*at : s);
    };
    look(block);
    if (lane == 0) later[wave] = parts > LONG;
    if (parts && parts <= LONG) {
        float s[4] = {};
        add(block, 0, 1, s);
#pragma unroll
        for (int c = 0; c < 4; c++) put(d0 + c * 64 + lane, s[c]);
    }
    __syncthreads();
    for (uint32_t w = 0; w < WAVES; w++) {
        if (!later[w]) continue;
        look(blockIdx.x * WAVES + w);
        float s[4] = {};
        add(blockIdx.x * WAVES + w, wave, WAVES, s);
        __syncthreads();
#pragma unroll
        for (int c = 0; c < 4; c++) sums[wave][c * 64 + lane] = s[c];
        __syncthreads();
        if (threadIdx.x < 256) {
            float v = 0.f;
            for (uint32_t k = 0; k < WAVES; k++) v += sums[k][threadIdx.x];
            put(d0 + threadIdx.x, v);
        }
    }
}

template <typename T, int V> static int run_embed(apoe_ctx* ctx, const apoe_embed_args* p) {
    hipStream_t s = ctx->stream;
    const uint32_t cus = (uint32_t)ctx->num_cus;
    // a workgroup a row where groups of a row each would leave most of the GPU idle and there are entries to share
    const bool wide = p->n_rows <= cus * 4 && (uint64_t)p->n_entries >= (uint64_t)p->n_rows * 8;
    return with_group(p->dim, [&](auto size) -> int {
        constexpr int G = decltype(size)::value, THREADS = G > 256 ? G : 256;
        if (wide) {
            embed_rows<T, V, G, true><<<p->n_rows, 1024, 0, s>>>(*p);
        } else {
            const uint64_t need = ((uint64_t)p->n_rows + THREADS / G - 1) / (THREADS / G);
            embed_rows<T, V, G, false><<<(uint32_t)std::min<uint64_t>(need, 1u << 20), THREADS, 0, s>>>(*p);
        }
        return APOE_OK;
    });
}

template <typename T, int V> static int run_embed_grad(apoe_ctx* ctx, const apoe_embed_args* p) {
    hipStream_t s = ctx->stream;
    if (p->grad_val && p->n_rows && p->n_entries) {
        APOE_TRY(with_group(p->dim, [&](auto size) -> int {
            constexpr int G = decltype(size)::value, THREADS = G > 256 ? G : 256;
            const uint64_t need = ((uint64_t)p->n_rows + THREADS / G - 1) / (THREADS / G);
            // few rows: their entries in turn by up to 16 workgroups
            const uint32_t share = (uint32_t)std::min<uint64_t>(16, std::max<uint64_t>(1, std::min<uint64_t>((uint64_t)ctx->num_cus * 8 / need, p->n_entries / (p->n_rows * 4ull))));
            embed_weights<T, V, G><<<dim3((uint32_t)std::min<uint64_t>(need, 1u << 20), share), THREADS, 0, s>>>(*p);
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
    a.blocks = (uint32_t)((n + EMBED_BLOCK - 1) / EMBED_BLOCK);
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
    if (n) {
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
        embed_table<T, V, G><<<entry_groups + zero_groups, THREADS, 0, s>>>(a, entry_groups);
        return APOE_OK;
    }));
    if (a.blocks > 1) embed_join<T><<<dim3((a.blocks + 15) / 16, (p->dim + 255) / 256), 1024, 0, s>>>(a);
    return APOE_OK;
}

template <typename T> static int run_aligned(apoe_ctx* ctx, const apoe_embed_args* p, bool grad) {
    constexpr int V = 16 / (int)sizeof(T);
    bool whole = p->dim % V == 0; // 16 bytes a load where every row begins at a multiple of that
    for (const void* q : {p->table, p->base, (const void*)p->out, p->grad, (const void*)p->grad_table}) whole &= ((uintptr_t)q & 15) == 0;
    for (uint64_t q : {p->table_stride, p->base_stride, p->out_stride, p->grad_stride, p->grad_table_stride}) whole &= q % V == 0;
    if (grad) APOE_TRY(whole ? (run_embed_grad<T, V>(ctx, p)) : (run_embed_grad<T, 1>(ctx, p)));
    else APOE_TRY(whole ? (run_embed<T, V>(ctx, p)) : (run_embed<T, 1>(ctx, p)));
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
