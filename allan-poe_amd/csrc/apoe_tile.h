// Tiles of a matrix product on the matrix cores, shared by the operators that fit a query adapter (loss.hip, ortho.hip).
//
// A workgroup of NW waves multiplies a tile of A (M side) with a tile of B (N side), both staged through LDS in steps of the
// inner dimension. Values have 16 bits (float matrices come as two or three planes of such). The unit of the inner dimension is a
// fragment: 16 bytes a lane, 16 values of a row, one 32x32x16 product. What the two sides have to agree on is which inner index
// a lane's j-th value holds, so a fragment may permute them; two orders occur:
//   ROWS    lane half h holds 8 consecutive indices, half 0 first, as 16 bytes of a row come;
//   BLOCKS  value j of half h is index 8 (j / 4) + 4 h + j % 4: what a lane has of a 32x32 result, so a result turns into
//           the next product's operand without a move between lanes.
//
// Loads go from memory straight into LDS (16 bytes a lane, no registers), through inline asm: to the compiler's own builtin
// every LDS read waits for all such loads in flight, which would undo the stages. The asm has no output registers and each
// stage is waited for by count (tile_wait). A masked lane reads address MASKED, beyond the buffer's range: the hardware
// delivers zeros, which is how rows and columns beyond an edge and rows that a mask leaves out come to count nothing,
// whatever memory holds there.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

namespace apoe {

using f32x16 = float __attribute__((ext_vector_type(16)));
using f32x4 = float __attribute__((ext_vector_type(4)));
using i32x4 = int __attribute__((ext_vector_type(4)));
using i32x2 = int __attribute__((ext_vector_type(2)));
using s16x4 = short __attribute__((ext_vector_type(4)));
using f16x8 = _Float16 __attribute__((ext_vector_type(8)));
using f16x4 = _Float16 __attribute__((ext_vector_type(4)));
using f16x2 = _Float16 __attribute__((ext_vector_type(2)));
using bf16x8 = __bf16 __attribute__((ext_vector_type(8)));
using u16x2 = unsigned short __attribute__((ext_vector_type(2)));

constexpr uint32_t TILE_MASKED = 0x80000000u; // byte offset past every buffer
constexpr uint32_t TILE_RANGE = 0x7fffffffu;  // the range every buffer descriptor states; host code keeps real offsets below it

enum { ORDER_ROWS = 0, ORDER_BLOCKS = 1 };

template <typename T> __device__ inline f32x16 mfma_step(i32x4 a, i32x4 b, f32x16 c);
template <> __device__ inline f32x16 mfma_step<_Float16>(i32x4 a, i32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <> __device__ inline f32x16 mfma_step<__bf16>(i32x4 a, i32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// Row of a 32x32 result that value i of a lane in half h holds (its column is lane % 32).
__device__ inline int result_row(int i, int h) { return 8 * (i >> 2) + 4 * h + (i & 3); }

__device__ inline uint32_t lds_address(const void* p) { return (uint32_t)(size_t)(__attribute__((address_space(3))) const char*)p; }

// A number that is the same in the whole wave, in scalar registers (the compiler loses sight of that in 64-bit products).
__device__ inline uint64_t uniform64(uint64_t v) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v) | (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32)) << 32;
}

__device__ inline i32x4 buffer_of(uint64_t base) { return i32x4{(int)(uint32_t)base, (int)(uint32_t)(base >> 32), (int)TILE_RANGE, 0x00020000}; }

// Workgroups go to the eight XCDs in turn, each of which has an L2 of its own. The number that gives each XCD a run of consecutive tiles.
__device__ inline uint32_t xcd_run(uint32_t id, uint32_t total) {
    const uint32_t per = total / 8;
    return id < per * 8 ? (id & 7) * per + (id >> 3) : id;
}

// 16 bytes a lane from base + offset to LDS at lds + 16 lane. lds and the descriptor are the same in the wave.
__device__ inline void load_to_lds16(i32x4 buffer, uint32_t offset, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(offset), "s"(buffer) : "memory");
}
__device__ inline void load_to_lds4(i32x4 buffer, uint32_t offset, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(lds), "v"(offset), "s"(buffer) : "memory");
}

// All but the YOUNGER last loads of this wave have landed, its LDS reads are done, and so are those of the other waves.
template <int YOUNGER> __device__ inline void tile_wait() {
    static_assert(YOUNGER >= 0 && YOUNGER < 64, "the counter has 6 bits");
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(YOUNGER) : "memory");
}

// The order of a stage's instructions: the first fragments' READS, then with the MFMAS of each fragment the next one's reads, so that
// no product waits for a read that was just sent off. The code around it reads fragment f + 1 before it multiplies f.
template <int READS, int MFMAS, int SF> __device__ inline void interleave() {
    constexpr int READ = 0x100, MFMA = 0x008;
    __builtin_amdgcn_sched_group_barrier(READ, READS, 0);
#pragma unroll
    for (int f = 0; f + 1 < SF; f++) {
#pragma unroll
        for (int i = 0; i < MFMAS; i++) {
            __builtin_amdgcn_sched_group_barrier(MFMA, 1, 0);
            if (i < READS) __builtin_amdgcn_sched_group_barrier(READ, (READS + MFMAS - 1) / MFMAS, 0);
        }
    }
    __builtin_amdgcn_sched_group_barrier(MFMA, MFMAS, 0);
}

// ROWS rows of a matrix whose inner dimension is contiguous; SF fragments a stage. 16-byte pieces of a row lie in LDS at a place
// that the row's number turns (xor), so that 16 consecutive rows' equal pieces, which one cycle reads, are in different banks.
template <typename T, int ROWS, int SF, int NW> struct RowTile {
    static constexpr int BYTES = ROWS * SF * 32, LOADS = BYTES / (1024 * NW), PIECES = SF * 2;
    static constexpr int KE = SF * 16; // inner indices of a stage
    static_assert(sizeof(T) == 2, "values of 16 bits");
    static_assert(BYTES % (1024 * NW) == 0 && (SF == 2 || SF == 4) && NW % 2 == 0, "whole loads");
    uint32_t offset[LOADS], piece;
    uint64_t base;
    __device__ static int turn(int row) { return SF == 2 ? (row >> 2) & 3 : (row >> 1) & 7; }
    // row0: the tile's first row; rows: how many of the tile's rows exist
    __device__ void init(const T* row0, uint32_t pitch_bytes, int rows, int wave, int lane) {
        base = uniform64((uint64_t)row0);
        piece = (uint32_t)((lane % PIECES) ^ turn(wave * (64 / PIECES) + lane / PIECES)); // loads of a wave are 16 rows apart or a multiple
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            const int row = (i * NW + wave) * (64 / PIECES) + lane / PIECES;
            offset[i] = row < rows ? (uint32_t)row * pitch_bytes + piece * 16 : TILE_MASKED;
        }
    }
    // left: bytes of a row from here on (a multiple of 16; none or less: a stage of zeros)
    __device__ void load(uint32_t lds, int left, int wave) const {
        const i32x4 buffer = buffer_of(base);
        if (left >= SF * 32) {
#pragma unroll
            for (int i = 0; i < LOADS; i++) load_to_lds16(buffer, offset[i], lds + (i * NW + wave) * 1024);
        } else {
            const bool in = (int)piece * 16 < left;
#pragma unroll
            for (int i = 0; i < LOADS; i++) load_to_lds16(buffer, in ? offset[i] : TILE_MASKED, lds + (i * NW + wave) * 1024);
        }
    }
    __device__ void next() { base += SF * 32; }
    // fragment f of the 32 rows of block rb, order ROWS
    __device__ static i32x4 read(const char* lds, int rb, int f, int lane) {
        const int row = lane & 31;
        return *reinterpret_cast<const i32x4*>(lds + rb * 32 * SF * 32 + row * SF * 32 + (((2 * f + (lane >> 5)) ^ turn(row)) * 16));
    }
};

// COLS columns of a matrix whose inner dimension goes down the rows: rows of a stage as they come, read transposed. The pieces'
// places turn with the row's last two bits: the four rows that sixteen lanes read together are in different banks.
template <typename T, int COLS, int SF, int NW, int ORDER> struct ColTile {
    static constexpr int KE = SF * 16, ROWB = COLS * 2, BYTES = KE * ROWB, LOADS = BYTES / (1024 * NW), PIECES = ROWB / 16;
    static constexpr int TURN = PIECES >= 16 ? 12 : PIECES - 4;
    static_assert(BYTES % (1024 * NW) == 0 && PIECES >= 8, "whole loads");
    using Mask = std::conditional_t<(KE > 32), uint64_t, uint32_t>;
    static_assert(KE <= 64, "one word of rows");
    static constexpr Mask ALL = KE == 32 ? (Mask)~0u : KE == 64 ? (Mask)~0ull : (Mask)((1ull << (KE & 63)) - 1);
    uint32_t offset[LOADS];
    uint64_t base, step;
    __device__ static int row_of(int i, int wave, int lane) { return ((i * NW + wave) * 64 + lane) / PIECES; }
    // at: the first row's column where the tile begins; cols: how many of the tile's columns exist (a multiple of a piece)
    __device__ void init(const T* at, uint32_t pitch_bytes, int cols, int wave, int lane) {
        base = uniform64((uint64_t)at);
        step = (uint64_t)KE * pitch_bytes;
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            const int l = (i * NW + wave) * 64 + lane, row = l / PIECES, piece = (l % PIECES) ^ ((4 * row) & TURN);
            offset[i] = piece * 8 < cols ? (uint32_t)row * pitch_bytes + piece * 16 : TILE_MASKED;
        }
    }
    // bit r of `rows` (KE of them): row r of the stage counts
    __device__ void load(uint32_t lds, Mask rows, int wave, int lane) const {
        const i32x4 buffer = buffer_of(base);
        if ((rows & ALL) == ALL) {
#pragma unroll
            for (int i = 0; i < LOADS; i++) load_to_lds16(buffer, offset[i], lds + (i * NW + wave) * 1024);
        } else {
#pragma unroll
            for (int i = 0; i < LOADS; i++) load_to_lds16(buffer, (rows >> row_of(i, wave, lane)) & 1 ? offset[i] : TILE_MASKED, lds + (i * NW + wave) * 1024);
        }
    }
    __device__ void next() { base += step; }
    // fragment f of the 32 columns of block cb
    __device__ static i32x4 read(const char* lds, int cb, int f, int lane) {
        const int h = lane >> 5, i = lane & 15, col = ((lane >> 4) & 1) * 16 + 4 * (i & 3), sub = (col & 7) * 2;
        i32x2 part[2];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int row = f * 16 + (ORDER == ORDER_ROWS ? 8 * h + 4 * j : 4 * h + 8 * j) + (i >> 2);
            const char* p = lds + row * ROWB + (((cb * 4 + (col >> 3)) ^ ((4 * row) & TURN)) * 16) + sub;
            part[j] = __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p));
        }
        return i32x4{part[0][0], part[0][1], part[1][0], part[1][1]};
    }
};

// Two groups of waves have summed up every other stage each (KG = 2): they exchange halves, and each has the whole sums of its half of the blocks.
template <int MT, int NT, int WAVES> __device__ inline void exchange_halves(f32x16 (&acc)[MT][NT], char* lds, int group, int wave, int lane) {
    static_assert(MT % 2 == 0, "halves");
    float* buf = reinterpret_cast<float*>(lds) + lane;
    const auto at = [&](int g, int m, int t, int k) { return (((g * WAVES + wave) * (MT / 2) + m % (MT / 2)) * NT + t) * 1024 + k * 64; };
#pragma unroll
    for (int m = 0; m < MT; m++)
        if (m / (MT / 2) != group)
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int k = 0; k < 16; k++) buf[at(group, m, t, k)] = acc[m][t][k];
    __syncthreads();
#pragma unroll
    for (int m = 0; m < MT; m++)
        if (m / (MT / 2) == group)
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int k = 0; k < 16; k++) acc[m][t][k] += buf[at(group ^ 1, m, t, k)];
}

} // namespace apoe
