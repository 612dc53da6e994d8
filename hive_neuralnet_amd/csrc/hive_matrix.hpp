// hive_matrix.hpp -- tiles of matrix products on the matrix cores, shared by
// the gated block (hive_gated.hip) and the orthogonalised update
// (hive_muon.hip).
//
//   C[m][n] = sum over k of A[m][k] B[n][k]
//
// Both operands are rows of 16-bit values with k running along the row, which
// is how a matrix instruction takes them.  A value may stand for 1, 2 or 3 of
// them ("parts"), whose sum it is, rounded to 11 (float16) or 8 (bfloat16) bits
// each; 32 consecutive k's first parts are followed by their second, and so on:
//   1 part   the tensors as they are, float16 or bfloat16
//   2 parts  float16, 22 bits of a value: A0 B0 + A0 B1 + A1 B0, the product of
//            the last parts (2^-24 of the whole) left out
//   3 parts  bfloat16, all 24 bits of a float from 2^-110 in size up (below that
//            to within 2^-134): the six products of parts whose numbers add up to
//            at most 2
// so that float32 products run at a third or a sixth of the 16-bit rate (2.5
// PFLOP/s), where the float32 instructions reach a sixteenth of it.
//
// A block of kWm x kWn waves holds a tile of C in registers.  Its slices of A
// and B go from memory into LDS past the registers, one slice ahead of the one
// being multiplied; a load's LDS side is consecutive, so what spreads a slice's
// rows over the LDS banks (16-byte chunk c of row r is held at c ^ (r / 2) % 8)
// is done by the choice of each lane's address in memory.  Rows and columns past
// the matrices are loads past the buffer's end, which give zeros.
#pragma once

#include "hive_train.hpp"

namespace hm {

using namespace ht;

typedef float f4 __attribute__((ext_vector_type(4)));
typedef int i4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));

template <typename T> struct Fragment;
template <> struct Fragment<f16> { using type = h8; };
template <> struct Fragment<bf16> { using type = b8; };

__device__ __forceinline__ f4 mfma(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f4 mfma(b8 a, b8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

constexpr uint32_t kWindow = 0x80000000u;  // bytes of a buffer; an offset of as many lies past it

// a buffer that begins at p, its descriptor the same in every lane
__device__ __forceinline__ i4 buffer(const void* p) {
    const uint64_t a = (uint64_t)p;
    i4 d;
    d[0] = __builtin_amdgcn_readfirstlane((int)(uint32_t)a);
    d[1] = __builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32) & 0xFFFF);
    d[2] = (int)kWindow;
    d[3] = 0x00020000;
    return d;
}

// 16 bytes a lane from the buffer at offset + step into LDS at lds + 16 * lane.  Nothing waits for it: wait_all() does.
__device__ __forceinline__ void load_to_lds(i4 from, uint32_t offset, uint32_t step, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds), "v"(offset), "s"(from),
                 "s"(step)
                 : "memory");
}
// this wave's loads have landed and its LDS reads are done, and so are those of the block's other waves
__device__ __forceinline__ void wait_all() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ uint32_t lds_address(const void* p) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}

// An operand: `rows` rows of `bytes` bytes (a multiple of 16), `stride` bytes apart (a multiple of 16), 16-byte aligned.
struct Operand {
    const void* p;
    int64_t stride;
    int rows, bytes;
};

template <typename T_, int kParts_, int kM_, int kN_, int kWm_, int kWn_> struct Tile {
    using T = T_;
    using V = typename Fragment<T>::type;
    static constexpr int kParts = kParts_, kM = kM_, kN = kN_, kWm = kWm_, kWn = kWn_;
    static constexpr int kThreads = 64 * kWm * kWn;
    static constexpr int kSteps = kParts == 1 ? 2 : 1;                // of 32 k in a slice
    static constexpr int kRow = 64 * kParts * kSteps;                 // bytes of a slice's row: 128 or 192
    static constexpr int kChunks = kRow / 16;
    static constexpr int kStage = (kM + kN) * kRow;                   // bytes of a slice
    static constexpr int kFm = kM / kWm / 16, kFn = kN / kWn / 16;    // a wave's 16 x 16 pieces
    static constexpr int kLoads = (kM + kN) * kChunks / kThreads;     // 16-byte loads a lane makes for a slice
    static constexpr int kLoadsA = kM * kChunks / kThreads;
    static_assert(kM * kChunks % kThreads == 0 && kN * kChunks % kThreads == 0, "whole loads");
    static_assert(kParts != 3 || kRow == 192, "");
    // where chunk c of row r is held
    static __device__ __forceinline__ int place(int r, int c) {
        return kChunks == 8 ? c ^ ((r >> 1) & 7) : c ^ ((r >> 2) & 3);
    }
};

// The sums of one tile.  acc[i][j]: lane l holds C at row 16 i + l % 16, columns 16 j + 4 (l / 16) .. + 3 of the
// wave's part, which begins at (row(), col()) of the tile.
template <typename Tl> struct Sums {
    f4 acc[Tl::kFm][Tl::kFn];
    __device__ __forceinline__ int row() const { return (int)(threadIdx.x >> 6) / Tl::kWn * Tl::kFm * 16 + (threadIdx.x & 15); }
    __device__ __forceinline__ int col() const {
        return (int)(threadIdx.x >> 6) % Tl::kWn * Tl::kFn * 16 + (int)(threadIdx.x & 63) / 16 * 4;
    }
};

// The product over bytes [begin, end) of the rows (multiples of a slice's, but for the end of the row), of rows m0.. of A
// and of the rows of B that a tile's row r stands for: row_of(r) of B[which(r)], the same `which` for 64 chunks that
// follow each other.
template <typename Tl, typename RowOf, typename Which>
__device__ __forceinline__ void multiply(const Operand& a, int m0, const Operand& b0, const Operand& b1, RowOf row_of,
                                         Which which, int64_t b_first, int begin, int end, char* lds, Sums<Tl>& s) {
    using V = typename Tl::V;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const i4 from_a = buffer((const char*)a.p + (int64_t)m0 * a.stride);
    const i4 from_b0 = buffer((const char*)b0.p + b_first * b0.stride);
    const i4 from_b1 = buffer((const char*)b1.p + b_first * b1.stride);
    uint32_t offset[Tl::kLoads];
    int at[Tl::kLoads];  // the chunk's place in its row, in bytes
#pragma unroll
    for (int i = 0; i < Tl::kLoads; i++) {
        const int q = (i < Tl::kLoadsA ? i : i - Tl::kLoadsA) * Tl::kThreads + tid;
        const int r = q / Tl::kChunks, c = Tl::place(r, q % Tl::kChunks);  // its own inverse
        at[i] = c * 16;
        if (i < Tl::kLoadsA) {
            offset[i] = m0 + r < a.rows ? (uint32_t)(r * a.stride) + c * 16 : kWindow;
        } else {
            const int n = row_of(r);
            offset[i] = b_first + n < b0.rows ? (uint32_t)(n * b0.stride) + c * 16 : kWindow;
        }
    }
    const uint32_t base = lds_address(lds) + wave * 1024;
    auto fetch = [&](int k, int stage) {
#pragma unroll
        for (int i = 0; i < Tl::kLoads; i++) {
            const uint32_t off = at[i] < end - k ? offset[i] : kWindow;
            const uint32_t to = __builtin_amdgcn_readfirstlane(base + stage * Tl::kStage + i * Tl::kThreads * 16);
            if (i < Tl::kLoadsA) {
                load_to_lds(from_a, off, k, to);
            } else {
                const int first = ((i - Tl::kLoadsA) * Tl::kThreads + wave * 64) / Tl::kChunks;
                load_to_lds(which(first) ? from_b1 : from_b0, off, k, to);
            }
        }
    };
#pragma unroll
    for (int i = 0; i < Tl::kFm; i++)
#pragma unroll
        for (int j = 0; j < Tl::kFn; j++) s.acc[i][j] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    if (begin >= end) return;
    const int l = lane & 15, g = lane >> 4;
    const char* rows_a = lds + (wave / Tl::kWn * Tl::kFm * 16 + l) * Tl::kRow;
    const char* rows_b = lds + (Tl::kM + wave % Tl::kWn * Tl::kFn * 16 + l) * Tl::kRow;
    fetch(begin, 0);
    int stage = 0;
    for (int k = begin; k < end; k += Tl::kRow, stage ^= 1) {
        wait_all();
        if (k + Tl::kRow < end) fetch(k + Tl::kRow, stage ^ 1);
        const char *pa = rows_a + stage * Tl::kStage, *pb = rows_b + stage * Tl::kStage;
        V va[Tl::kParts][Tl::kFm], vb[Tl::kParts][Tl::kFn];
        auto read = [&](int step) {
#pragma unroll
            for (int p = 0; p < Tl::kParts; p++) {
                const int c = Tl::place(l, (step * Tl::kParts + p) * 4 + g) * 16;
#pragma unroll
                for (int i = 0; i < Tl::kFm; i++) va[p][i] = *(const V*)(pa + i * 16 * Tl::kRow + c);
#pragma unroll
                for (int j = 0; j < Tl::kFn; j++) vb[p][j] = *(const V*)(pb + j * 16 * Tl::kRow + c);
            }
        };
#pragma unroll
        for (int step = 0; step < Tl::kSteps; step++) {
            read(step);
#pragma unroll
            for (int sum = Tl::kParts - 1; sum >= 0; sum--)  // the smallest products first
#pragma unroll
                for (int p = 0; p <= sum; p++)
#pragma unroll
                    for (int i = 0; i < Tl::kFm; i++)
#pragma unroll
                        for (int j = 0; j < Tl::kFn; j++) s.acc[i][j] = mfma(vb[sum - p][j], va[p][i], s.acc[i][j]);
        }
    }
    wait_all();  // the LDS is free again
}

// block t of `all` in an order that keeps blocks that run beside each other near each other: chiplet x has the blocks x, x + 8,
// ..., and takes a range of its own of the work
__device__ __forceinline__ int chiplet_order(int t, int all) {
    const int share = all / 8, extra = all % 8, x = t % 8;
    return x * share + min(x, extra) + t / 8;
}
// tile t of m x n tiles: bands of 8 rows, down their columns
struct Place {
    int m, n;
};
__device__ __forceinline__ Place band_place(int t, int m, int n) {
    const int band = t / (8 * n), first = band * 8, height = min(8, m - first), in = t - band * 8 * n;
    return {first + in % height, in / height};
}
__device__ __forceinline__ Place tile_place(int t, int m, int n) { return band_place(chiplet_order(t, m * n), m, n); }

}  // namespace hm
