// hive_matrix.hpp -- tiles of matrix products on the matrix cores, shared by
// the gated block (hive_gated.hip) and the orthogonalised update
// (hive_muon.hip).
//
//   C[m][n] = sum over k of A[m][k] B[n][k]
//
// Operands are 16-bit values, rows of A and B along which k runs, or (turned) rows
// of k along which m or n runs, which LDS reads that turn 4 x 16 values take as
// well.  A value may stand for 1, 2 or 3 of them ("parts"), whose sum it is, rounded
// to 11 (float16) or 8 (bfloat16) bits each; the first parts of 32 values that
// follow each other in a row are followed by their second, and so on:
//   1 part   the tensors as they are, float16 or bfloat16
//   2 parts  float16, 22 bits of a value: A0 B0 + A0 B1 + A1 B0, the product of
//            the last parts (2^-24 of the whole) left out
//   3 parts  bfloat16, all 24 bits of a float from 2^-110 in size up (below that
//            to within 2^-134): the six products of parts whose numbers add up to
//            at most 2
// so that float32 products run at a third or a sixth of the 16-bit rate (2.5
// PFLOP/s), where the float32 instructions reach a sixteenth of it.
//
// A block of kWm x kWn waves holds a tile of C in registers and takes the sum in
// slices of kSteps times 32 k.  Slices go from memory into LDS past the registers,
// kStages - 1 of them ahead; a wave reads the next 32 k's operands from LDS into
// registers while it multiplies these, so that the matrix cores wait for neither.
// A load's LDS side is consecutive, so what spreads a slice's rows over the LDS
// banks (Tile::place) is done by the choice of each lane's address in memory.
// Rows and columns past the matrices are loads past the buffer's end, which give
// zeros.
//
// A lane's columns of C follow each other (4 kFn of them), which makes 128 bytes of
// a row for the four lanes that share it, where the 4 columns that one instruction
// leaves a lane would be stored 32 bytes of a row at a time: the rows of B are
// taken in that order, or, of a turned B, the sums changed round among the lanes.
#pragma once

#include <type_traits>

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

// Scalar operands of load_to_lds: vector memory may read a scalar register five wait states after a lane's value was written
// to it at the earliest, which the compiler does not see to for a block of its own.
__device__ __forceinline__ void settle(i4& from, int& step) { asm("s_nop 4" : "+s"(from), "+s"(step)); }
// 16 bytes a lane from the buffer at offset + step into LDS at lds + 16 * lane.  Nothing waits for it: wait_loads() does.
// from and step are settled; m0 is read one wait state after its write.
__device__ __forceinline__ void load_to_lds(i4 from, uint32_t offset, int step, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds), "v"(offset),
                 "s"(from), "s"(step)
                 : "memory");
}
// all but this wave's newest `kNewer` loads have landed and its LDS reads are done, and so it is for the block's other waves
template <int kNewer> __device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kNewer) : "memory");
}

__device__ __forceinline__ uint32_t lds_address(const void* p) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}

// An operand: `rows` rows of `bytes` bytes (a multiple of 16), `stride` bytes apart (a multiple of 16), 16-byte aligned.
// A turned one has a row for each k.
struct Operand {
    const void* p;
    int64_t stride;
    int rows, bytes;
};

template <typename T_, int kParts_, int kSteps_, int kM_, int kN_, int kWm_, int kWn_, int kStages_, int kBlocks_,
          bool kAhead_ = true, int kTeams_ = 1>
struct Tile {
    using T = T_;
    using V = typename Fragment<T>::type;
    static constexpr int kParts = kParts_, kSteps = kSteps_, kM = kM_, kN = kN_, kWm = kWm_, kWn = kWn_, kStages = kStages_;
    static constexpr int kBlocks = kBlocks_;                          // that a compute unit holds
    static constexpr bool kAhead = kAhead_;                           // operands are read a step ahead
    static constexpr int kTeams = kTeams_;                            // of a block, which share out the slices
    static constexpr int kThreads = 64 * kWm * kWn, kBlock = kTeams * kThreads;  // of a team; of a block
    static constexpr int kWavesEach = kBlocks * kBlock / 256;         // on a SIMD
    static constexpr int kRow = 64 * kParts * kSteps;                 // bytes of a slice's row
    static constexpr int kChunks = kRow / 16;
    static constexpr int kStage = (kM + kN) * kRow;                   // bytes of a slice
    static constexpr int kLds = kTeams * kStages * kStage;
    static constexpr int kFm = kM / kWm / 16, kFn = kN / kWn / 16;    // a wave's 16 x 16 pieces
    static constexpr int kLoads = (kM + kN) * kChunks / kThreads;     // 16-byte loads a lane makes for a slice
    static constexpr int kLoadsA = kM * kChunks / kThreads;
    static constexpr int kReads = kParts * (kFm + kFn);               // operands a lane reads for 32 k
    static constexpr int kProducts = kParts * (kParts + 1) / 2, kGroups = kProducts * kFm;
    static_assert(kM * kChunks % kThreads == 0 && kN * kChunks % kThreads == 0, "whole loads");
    static_assert(kStages >= 2 && (kStages - 2) * kLoads < 64, "a wait counts 63 loads");
    static_assert(kChunks == 4 || kChunks == 8 || kChunks == 12, "");
    // where chunk c of row r is held: rows that 16 lanes read together begin in different banks
    static __device__ __forceinline__ int place(int r, int c) {
        return kChunks == 8 ? c ^ ((r >> 1) & 7) : c ^ ((r >> 2) & 3);
    }
    // the same for row k of `kAcross` chunks of a turned operand, of which 32 bytes are read together from each of the rows
    // 8 g .. 8 g + 3 or 8 g + 4 .. 8 g + 7
    template <int kAcross> static __device__ __forceinline__ int turned_place(int k, int c) {
        return kAcross % 16 == 0 ? c ^ ((k & 3) | (k >> 1 & 4)) << 1 : c ^ ((k >> 1 & 1) | (k >> 2 & 2)) << 1;
    }
};

// a tile as a number: (rows * 1000 + columns) * 100 + stages * 10 + blocks of a compute unit, 10^8 more for each further team
template <typename Tl> constexpr int name_of() {
    return ((Tl::kTeams - 1) * 1000000 + Tl::kM * 1000 + Tl::kN) * 100 + Tl::kStages * 10 + Tl::kBlocks;
}

// The sums of one tile.  acc[i][j][e]: lane l holds C at row 16 i + l % 16 of the wave's part, which begins at row() of the
// tile, and, with kHalves equal shares of the kFn j, column 4 (j % share) + e of those that begin at col() of half j / share.
template <typename Tl, int kHalves, bool kTurnedB = false> struct Sums {
    static constexpr int kShare = Tl::kFn / kHalves;
    f4 acc[Tl::kFm][Tl::kFn];
    static __device__ __forceinline__ int wave() { return (int)(threadIdx.x % Tl::kThreads >> 6); }
    __device__ __forceinline__ int row() const { return wave() / Tl::kWn * Tl::kFm * 16 + (threadIdx.x & 15); }
    // of the wave's part, and of the lane's columns
    __device__ __forceinline__ int first_col() const { return wave() % Tl::kWn * kShare * 16; }
    __device__ __forceinline__ int col() const { return first_col() + (int)(threadIdx.x & 63) / 16 * 4 * kShare; }
    // row r of a tile of B: its column of C, and which half it is of
    static __device__ __forceinline__ int column(int r) {
        return r / (Tl::kFn * 16) * kShare * 16 + r % 16 / 4 * 4 * kShare + r / 16 % kShare * 4 + r % 4;
    }
    static __device__ __forceinline__ bool second(int r) { return kHalves == 2 && r / 16 % Tl::kFn >= kShare; }
    // a turned B's columns are taken in order, 16 j + 4 (l / 16) + e of a lane: changed round among the four lanes
    __device__ __forceinline__ void regroup() {
        static_assert(!kTurnedB || Tl::kFn == 2 || Tl::kFn == 4, "");
#pragma unroll
        for (int i = 0; i < Tl::kFm; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                float v[Tl::kFn];
#pragma unroll
                for (int j = 0; j < Tl::kFn; j++) v[j] = acc[i][j][e];
#pragma unroll
                for (int j = 0; j < Tl::kFn; j += 2) {
                    if constexpr (Tl::kFn == 2) {
                        const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[0]), __float_as_uint(v[1]), false, false);
                        v[0] = __uint_as_float(p[0]);
                        v[1] = __uint_as_float(p[1]);
                    }
                    const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[j]), __float_as_uint(v[j + 1]), false, false);
                    v[j] = __uint_as_float(p[0]);
                    v[j + 1] = __uint_as_float(p[1]);
                }
                if constexpr (Tl::kFn == 4) {
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[j]), __float_as_uint(v[j + 2]), false, false);
                        v[j] = __uint_as_float(p[0]);
                        v[j + 2] = __uint_as_float(p[1]);
                    }
                }
#pragma unroll
                for (int j = 0; j < Tl::kFn; j++) acc[i][j][e] = v[j];
            }
    }
};

// The product over slices [begin, end) of rows m0.. of A and rows n0.. of B (columns, where they are turned).  With two halves
// of B, b0 and b1, the same rows of both; a turned B goes on in b1 from slice `cut` on.  Of more than one team the first has
// the sums in the end, and the others are done.
template <typename Tl, int kHalves, bool kTurnedA, bool kTurnedB>
__device__ __forceinline__ void multiply(const Operand& a, int m0, const Operand& b0, const Operand& b1, int n0, int cut,
                                         int begin, int end, char* lds, Sums<Tl, kHalves, kTurnedB>& s) {
    using V = typename Tl::V;
    constexpr int across_a = Tl::kM * Tl::kParts / 8, across_b = Tl::kN * Tl::kParts / 8;  // chunks of a turned slice's rows
    constexpr int deep = 32 * Tl::kSteps;                                                 // k of a slice
    static_assert(!kTurnedB || kHalves == 1, "");
    const int tid = threadIdx.x % Tl::kThreads, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    int stop = end;
    char* const all = lds;
    constexpr int team_lds = Tl::kLds / Tl::kTeams;
    const int team = Tl::kTeams == 1 ? 0 : __builtin_amdgcn_readfirstlane((int)threadIdx.x / Tl::kThreads);
    if constexpr (Tl::kTeams > 1) {
        // the same number of slices each, as they wait for each other: those past the end are zeros
        const int each = (end - begin + Tl::kTeams - 1) / Tl::kTeams;
        begin += team * each;
        stop = begin + each;
        lds += team * team_lds;
    }
    uint32_t offset[Tl::kLoads];
    int at[Tl::kLoads];  // the chunk's place in its row in bytes, or its k
#pragma unroll
    for (int i = 0; i < Tl::kLoads; i++) {
        const bool of_a = i < Tl::kLoadsA;
        const Operand& x = of_a ? a : b0;
        const int q = (of_a ? i : i - Tl::kLoadsA) * Tl::kThreads + tid;
        if (of_a ? kTurnedA : kTurnedB) {
            const int wide = of_a ? across_a : across_b, r = q / wide;
            const int c = of_a ? Tl::template turned_place<across_a>(r, q % wide) : Tl::template turned_place<across_b>(r, q % wide);
            const int first = (of_a ? m0 : n0) * 2 * Tl::kParts + c * 16;
            at[i] = r;
            offset[i] = first < x.bytes ? (uint32_t)(r * x.stride) + c * 16 : kWindow;
        } else {
            const int r = q / Tl::kChunks, c = Tl::place(r, q % Tl::kChunks);  // its own inverse
            const int n = of_a ? r : Sums<Tl, kHalves, kTurnedB>::column(r);
            at[i] = c * 16;
            offset[i] = (of_a ? m0 : n0) + n < x.rows ? (uint32_t)(n * x.stride) + c * 16 : kWindow;
        }
    }
    const uint32_t base = lds_address(lds) + wave * 1024;
    // where the slices begin in memory, and how many bytes or k from there on there are
    struct From {
        i4 a, b0, b1;
        int step_a, step_b, most_a, most_b;
    };
    auto from = [&](int n) {
        From f;
        f.a = buffer((const char*)a.p + (kTurnedA ? (int64_t)n * deep * a.stride + m0 * 2 * Tl::kParts : m0 * a.stride));
        const bool second = kTurnedB && n >= cut;
        const int n_b = second ? n - cut : n;
        f.b0 = buffer((const char*)(second ? b1.p : b0.p) +
                      (kTurnedB ? (int64_t)n_b * deep * b0.stride + n0 * 2 * Tl::kParts : n0 * b0.stride));
        f.step_a = kTurnedA ? 0 : n * Tl::kRow;
        f.step_b = kTurnedB ? 0 : n * Tl::kRow;
        settle(f.a, f.step_a);
        settle(f.b0, f.step_b);
        f.b1 = f.b0;
        if constexpr (kHalves == 2) {
            f.b1 = buffer((const char*)b1.p + n0 * b1.stride);
            settle(f.b1, f.step_b);
        }
        // a slice past the end is loaded, too, as zeros: a wait counts on it
        f.most_a = n >= end ? 0 : kTurnedA ? a.rows - n * deep : a.bytes - n * Tl::kRow;
        f.most_b = n >= end ? 0 : kTurnedB ? b0.rows - n_b * deep : b0.bytes - n * Tl::kRow;
        return f;
    };
    auto fetch = [&](int i, const From& f, int stage) {
        const uint32_t off = at[i] < (i < Tl::kLoadsA ? f.most_a : f.most_b) ? offset[i] : kWindow;
        const uint32_t to = __builtin_amdgcn_readfirstlane(base + stage * Tl::kStage + i * Tl::kThreads * 16);
        if (i < Tl::kLoadsA) {
            load_to_lds(f.a, off, f.step_a, to);
        } else {
            const int first = ((i - Tl::kLoadsA) * Tl::kThreads + wave * 64) / Tl::kChunks;
            load_to_lds(Sums<Tl, kHalves>::second(first) ? f.b1 : f.b0, off, f.step_b, to);
        }
    };
#pragma unroll
    for (int i = 0; i < Tl::kFm; i++)
#pragma unroll
        for (int j = 0; j < Tl::kFn; j++) s.acc[i][j] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    if (begin >= stop) return;
    const int l = lane & 15, g = lane >> 4;
    const int wave_m = wave / Tl::kWn * Tl::kFm, wave_n = wave % Tl::kWn * Tl::kFn;  // in pieces of 16
    const char* const lds_b = lds + Tl::kM * Tl::kRow;
    V va[Tl::kAhead ? 2 : 1][Tl::kParts][Tl::kFm], vb[Tl::kAhead ? 2 : 1][Tl::kParts][Tl::kFn];
    auto straight = [&](const char* from, int piece, int p, int step) {
        return *(const V*)(from + (piece * 16 + l) * Tl::kRow + Tl::place(l, (step * Tl::kParts + p) * 4 + g) * 16);
    };
    // 4 k each of two reads: lane l of 16 reads columns 4 (l % 4) .. + 3 of row l / 4 and gets column l of the 4 rows
    auto turned = [&](const char* from, int piece, int p, int step, auto across_) {
        constexpr int across = decltype(across_)::value;
        typedef short s4 __attribute__((ext_vector_type(4)));
        typedef short s8 __attribute__((ext_vector_type(8)));
        const int k = step * 32 + g * 8 + l / 4;
        const int c = (Tl::kParts == 1 ? piece : (piece / 2 * Tl::kParts + p) * 2 + piece % 2) * 2 + l % 4 / 2;
        const char* first = from + k * across * 16 + Tl::template turned_place<across>(k, c) * 16 + l % 2 * 8;
        typedef __attribute__((address_space(3))) s4* Lds;
        const s4 u = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)first);
        // 4 rows on: the same place in them
        const s4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(first + 4 * across * 16));
        return __builtin_bit_cast(V, (s8){u[0], u[1], u[2], u[3], v[0], v[1], v[2], v[3]});
    };
    // operand r of a step of a slice: the columns' first
    auto read = [&](int r, int half, int stage, int step) {
        const int p = r < Tl::kParts * Tl::kFn ? r / Tl::kFn : (r - Tl::kParts * Tl::kFn) / Tl::kFm;
        if (r < Tl::kParts * Tl::kFn) {
            const int j = r % Tl::kFn;
            const char* from = lds_b + stage * Tl::kStage;
            if constexpr (kTurnedB) vb[half][p][j] = turned(from, wave_n + j, p, step, std::integral_constant<int, across_b>{});
            else vb[half][p][j] = straight(from, wave_n + j, p, step);
        } else {
            const int i = (r - Tl::kParts * Tl::kFn) % Tl::kFm;
            const char* from = lds + stage * Tl::kStage;
            if constexpr (kTurnedA) va[half][p][i] = turned(from, wave_m + i, p, step, std::integral_constant<int, across_a>{});
            else va[half][p][i] = straight(from, wave_m + i, p, step);
        }
    };
    if constexpr (!Tl::kAhead) {
        static_assert(Tl::kSteps == 1, "");
#pragma unroll
        for (int n = 0; n < Tl::kStages - 1; n++) {
            const From f = from(begin + n);
#pragma unroll
            for (int i = 0; i < Tl::kLoads; i++) fetch(i, f, n);
        }
        int stage = 0;
        for (int k = begin; k < stop; k++) {
            wait_loads<(Tl::kStages - 2) * Tl::kLoads>();
            const From f = from(k + Tl::kStages - 1);
            const int free = stage == 0 ? Tl::kStages - 1 : stage - 1;
#pragma unroll
            for (int r = 0; r < Tl::kReads; r++) read(r, 0, stage, 0);
            int n = 0;
#pragma unroll
            for (int sum = Tl::kParts - 1; sum >= 0; sum--)
#pragma unroll
                for (int p = 0; p <= sum; p++)
#pragma unroll
                    for (int i = 0; i < Tl::kFm; i++, n++) {
#pragma unroll
                        for (int j = 0; j < Tl::kFn; j++)
                            s.acc[i][j] = mfma(vb[0][sum - p][j], va[0][p][i], s.acc[i][j]);
#pragma unroll
                        for (int i2 = 0; i2 < Tl::kLoads; i2++)
                            if (i2 * Tl::kGroups / (2 * Tl::kLoads) == n) fetch(i2, f, free);
                        __builtin_amdgcn_sched_barrier(0);
                    }
            stage = stage + 1 == Tl::kStages ? 0 : stage + 1;
        }
    } else {
#pragma unroll
        for (int n = 0; n < Tl::kStages; n++) {
            const From f = from(begin + n);
#pragma unroll
            for (int i = 0; i < Tl::kLoads; i++) fetch(i, f, n);
        }
        wait_loads<(Tl::kStages - 1) * Tl::kLoads < 64 ? (Tl::kStages - 1) * Tl::kLoads : 63>();
#pragma unroll
        for (int r = 0; r < Tl::kReads; r++) read(r, 0, 0, 0);
        int stage = 0;
        // multiplies step `step` of slice k, whose operands are in half `half` of the registers, and reads the next step's.  At a
        // slice's last step, the next slice has to be there; its own stage, which all waves have read, is free for the slice
        // kStages further on.
        auto multiply_step = [&](int k, auto step_, auto half_) {
            constexpr int step = decltype(step_)::value, half = decltype(half_)::value;
            constexpr bool last = step == Tl::kSteps - 1;
            const int next = !last ? stage : stage + 1 == Tl::kStages ? 0 : stage + 1;
            if (last) wait_loads<(Tl::kStages - 2) * Tl::kLoads>();
            const From f = from(k + Tl::kStages);
            int n = 0;
#pragma unroll
            for (int sum = Tl::kParts - 1; sum >= 0; sum--)  // the smallest products first
#pragma unroll
                for (int p = 0; p <= sum; p++)
#pragma unroll
                    for (int i = 0; i < Tl::kFm; i++, n++) {
#pragma unroll
                        for (int j = 0; j < Tl::kFn; j++)
                            s.acc[i][j] = mfma(vb[half][sum - p][j], va[half][p][i], s.acc[i][j]);
                        // the reads in the first half of the step's time, the loads all through it
#pragma unroll
                        for (int r = 0; r < Tl::kReads; r++)
                            if (r * Tl::kGroups / (2 * Tl::kReads) == n) read(r, half ^ 1, next, last ? 0 : step + 1);
                        if (last)
#pragma unroll
                            for (int i = 0; i < Tl::kLoads; i++)
                                if (i * Tl::kGroups / Tl::kLoads == n) fetch(i, f, stage);
                        __builtin_amdgcn_sched_barrier(0);
                    }
            stage = next;
        };
        using zero = std::integral_constant<int, 0>;
        using one = std::integral_constant<int, 1>;
        if constexpr (Tl::kSteps == 2) {
            for (int k = begin; k < stop; k++) {
                multiply_step(k, zero{}, zero{});
                multiply_step(k, one{}, one{});
            }
        } else {
            for (int k = begin; k < stop; k += 2) {
                multiply_step(k, zero{}, zero{});
                if (k + 1 < stop) multiply_step(k + 1, zero{}, one{});
            }
        }
    }
    wait_loads<0>();  // the LDS is free again
    if constexpr (Tl::kTeams > 1) {
        static_assert(Tl::kFm * Tl::kFn * Tl::kThreads * 16 <= team_lds, "");
#pragma unroll
        for (int i = 0; i < Tl::kFm * Tl::kFn; i++)
            if (team > 0) ((f4*)lds)[i * Tl::kThreads + tid] = s.acc[i / Tl::kFn][i % Tl::kFn];
        __syncthreads();
        for (int t = 1; t < Tl::kTeams && team == 0; t++)
#pragma unroll
            for (int i = 0; i < Tl::kFm * Tl::kFn; i++)
                s.acc[i / Tl::kFn][i % Tl::kFn] += ((const f4*)(all + t * team_lds))[i * Tl::kThreads + tid];
    }
    if constexpr (kTurnedB) s.regroup();
}

// words a and b of the four lanes that share a row changed round: where lane q held pieces 2 q and 2 q + 1 of eight, it holds
// pieces q and 4 + q
__device__ __forceinline__ void spread(uint32_t& a, uint32_t& b) {
    const auto p = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    const auto q = __builtin_amdgcn_permlane32_swap(p[0], p[1], false, false);
    a = q[0];
    b = q[1];
}
// The n values of each of the four lanes that share a row of C to that row: lane q's are those of columns n q .. n q + n - 1,
// `p` the row's place of the first of all, `live` what there are of it (the same for the four).  Pieces of 16 bytes change
// lanes first, so that a store writes 64 bytes that follow each other (8,192 rows of gate and up, 8,192 wide, with their
// product: 190 us where it wrote 16 of every 32, 182 so).
template <typename T, int n> __device__ __forceinline__ void store_row(T* p, int live, const float (&v)[n]) {
    const int q = (int)(threadIdx.x & 63) / 16;
    if constexpr (n < Vector<T>::n) {
        store_some<T, n>(p + q * n, live - q * n, v);
    } else {
        constexpr int each = Vector<T>::n, pieces = n / each;
        static_assert(n % each == 0 && (pieces == 1 || pieces == 2 || pieces == 4), "");
        typedef uint32_t u4 __attribute__((ext_vector_type(4)));
        typedef typename Vector<T>::type vec;
        u4 w[pieces];
#pragma unroll
        for (int i = 0; i < pieces; i++) {
            vec x;
#pragma unroll
            for (int e = 0; e < each; e++) x[e] = from_f32<T>(v[i * each + e]);
            w[i] = __builtin_bit_cast(u4, x);
        }
        if constexpr (pieces >= 2)
#pragma unroll
            for (int i = 0; i < pieces; i += 2)
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    uint32_t a = w[i][k], b = w[i + 1][k];
                    spread(a, b);
                    w[i][k] = a;
                    w[i + 1][k] = b;
                }
        if constexpr (pieces == 4)  // lane q held pieces 4 q .. 4 q + 3; now the halves of w[0] and w[2], of w[1] and w[3]
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const auto h = __builtin_amdgcn_permlane32_swap(w[i][k], w[i + 2][k], false, false);
                    w[i][k] = h[0];
                    w[i + 2][k] = h[1];
                }
#pragma unroll
        for (int i = 0; i < pieces; i++) {
            const int piece = q + 4 * (pieces == 4 ? (i & 1) * 2 + i / 2 : i);
            const vec x = __builtin_bit_cast(vec, w[i]);
            T* to = p + piece * each;
            const int left = live - piece * each;
            if (left >= each) {
                *(vec*)to = x;
            } else {
#pragma unroll
                for (int e = 0; e < each; e++)
                    if (e < left) to[e] = x[e];
            }
        }
    }
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
