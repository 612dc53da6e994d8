// hive_muon.hip -- orthogonalised updates: the Newton-Schulz iteration of a
// batch of matrices, and the step of many of a network's matrices with it.
//
//   X = U / (|U| + eps), |U| the root of the sum of squares
//   steps times:  A = X X^T,  P = a I + b A + c A A,  X <- P X
// which takes each singular value s to a s + b s^3 + c s^5, and with the usual
// (a, b, c) all of them near 1.  X has the shorter side's rows: a matrix that is
// taller than wide is turned, and turned back at the end.  A step with it:
//   m = mu m + g,  u = g + mu m or m,  p = p keep - rate X(u)
//
// The iteration takes small singular values up 3.4445 times at each of its
// first steps, and with them what rounding has put in their place: at 16-bit
// rounding that would be the result.  Every matrix is held as two float16 parts a
// value, 22 bits, times 2^13 (entries are below 2 in size and mostly far below 1;
// the last parts of those above 2^-15 stay above float16's smallest, which holds
// the others to within 2^-38), and products are three matrix instructions of parts
// (hive_matrix.hpp).  |U| far below eps makes all of X small: a matrix is held times
// the power of two that takes its norm to between 1/2 and 1, and P takes that share
// of b and c, and of itself where the next X is held times less (Size).
//
// Measured (MI355X): 16 matrices of 1,024 x 1,024 and 8 of 4,096 x 1,024, an iteration A 190 us, P 115, P X 298 (270, 220 and
// 350 TFLOP/s, three times that of float16 instructions, 810, 670 and 1,040; large library products reach 1,100 to 1,520),
// sums 96 and packing 93 us once (memory).  One of 1,024 x 1,024: 13, 13 and 15, of which 7 are a launch's own: its arguments, the first slices from
// memory, the last stores.
//
// X is an operand by its rows in X X^T and by its columns in P X.  A and A A are
// symmetric: the tiles on and above the diagonal are computed, and stored twice.
#include <algorithm>
#include <cmath>

#include "hive_pack.hpp"

namespace {

using namespace hm;

constexpr int kMatrices = 24;        // of a launch: their table is a kernel argument
constexpr float kScale = 8192.0f;    // of X and A as they are held: entries up to 7.9
constexpr float kScaleP = 1024.0f;   // of P, which has a on its diagonal: up to 63
constexpr int kSumBlocks = 64;       // of a matrix's sum of squares
constexpr int kTriples = 16;         // coefficients that a launch of the whole iteration takes
constexpr int kMostSteps = 100;
constexpr int64_t kMaxSide = 1 << 17;

// One of the step's matrices, or a batch of one shape.
struct Matrix {
    const void* g;      // the update, or the gradient
    float* momentum;    // NULL: g is the update
    void* out;          // the result, or the parameter
    char* held;         // the workspace of `count` matrices
    int64_t g_row, g_step, out_step;  // elements: g's rows, g's and out's matrices
    float rate;         // of a parameter's step
    int rows, cols, count;
    int first;          // its first block in the launch
};
struct Table {
    Matrix t[kMatrices];
    int n;
    int range[9];  // chiplet x's tiles of a product: [range[x], range[x + 1])
    int g_type, out_type, update;  // update: out is a parameter
    float mu, keep, eps, a, b, c;
    int nesterov, from, step, last;  // from: which of the two copies of X is current
    int steps, count;          // the iteration in one launch: its steps, and how many of them have coefficients of their own
    float triples[3 * kTriples];
};

// How a matrix is held at a step: X 2^e, of norm `most` or less.
struct Size {
    int e;
    float most;
};

// where a matrix's parts lie in its workspace, in bytes; sizes: a Size of each step
struct Layout {
    int s, l;                // the shorter and the longer side
    int64_t sb, lb;          // bytes of a packed row along each
    int64_t x[2], a, p, sums, sizes, all;
};
__host__ __device__ inline Layout layout(int rows, int cols) {
    Layout o;
    o.s = rows < cols ? rows : cols;
    o.l = rows < cols ? cols : rows;
    o.sb = up_to(o.s, 32) * 4;
    o.lb = up_to(o.l, 32) * 4;
    int64_t at = 0;
    const int64_t x = up_to(o.s * o.lb, 256), a = up_to(o.s * o.sb, 256);
    for (int i = 0; i < 2; i++) {
        o.x[i] = at;
        at += x;
    }
    o.a = at;
    o.p = at + a;
    o.sums = at + 2 * a;
    o.sizes = o.sums + up_to(kSumBlocks * 8, 256);
    o.all = o.sizes + up_to((kMostSteps + 1) * sizeof(Size), 256);
    return o;
}

// X = U / (norm + eps) at first: its share of 1, a power of two and what is left of it
__device__ __forceinline__ Size first_size(double norm, double eps) {
    const double share = norm / (norm + eps);
    int k = 0;
    if (share > 0.0 && share < 1.0) frexp(share, &k);  // NaN: as it is
    return {-k, 1.0f};
}
// ... and after a step: |P| is at most |a| + |b| t^2 + |c| t^4, t = |X|.  A matrix that is held as it is (e = 0) is not held
// times less, however large the bound.
__device__ __forceinline__ Size next_size(Size x, float a, float b, float c) {
    const float t = ldexpf(x.most, -x.e), q = t * t;
    const float most = x.most * (__builtin_fabsf(a) + __builtin_fabsf(b) * q + __builtin_fabsf(c) * q * q);
    int k = 0;
    if (most > 0.0f && most < __builtin_inff()) frexpf(most, &k);
    k = min(k, x.e);
    return {x.e - k, ldexpf(most, -k)};
}
// what U is multiplied by, times kScale and x's power of two: v * by 2^e, which no size of U takes past float32's range
struct Factor {
    float by;
    int e;
    __device__ __forceinline__ float operator()(float v) const { return ldexpf(v, e) * by; }
};
__device__ __forceinline__ Factor factor_of(double norm, double eps, Size x) {
    const double all = (double)kScale / (norm + eps);
    int k = 0;
    const double by = all < __builtin_inf() ? frexp(all, &k) : all;  // inf of a norm and an eps of 0, NaN
    return {(float)by, k + x.e};
}

// the matrix that block t works on, t from there on its own
__device__ __forceinline__ int find(const Table& tab, int& t) {
    int i = 0;
    while (i + 1 < tab.n && tab.t[i + 1].first <= t) i++;
    t -= tab.t[i].first;
    return i;
}

// values c .. c + 7 of the update's row r, zeros past the first `live`; `m`: the momentum of the same values as it is (kStep
// false), or before this step, which is taken and stored
template <typename G, bool kStep>
__device__ __forceinline__ void load_update(const Matrix& x, const Table& tab, int64_t at_g, int64_t at_m, int live,
                                            float (&u)[8]) {
    load_some<G, 8>((const G*)x.g + at_g, live, u);
    if (!x.momentum) return;
    float m[8];
    load_some<float, 8>(x.momentum + at_m, live, m);
    if (kStep) {
#pragma unroll
        for (int e = 0; e < 8; e++) m[e] = fmaf(m[e], tab.mu, u[e]);
        store_some<float, 4>(x.momentum + at_m, live, m);
        store_some<float, 4>(x.momentum + at_m + 4, live - 4, m + 4);
    }
#pragma unroll
    for (int e = 0; e < 8; e++) u[e] = tab.nesterov ? fmaf(m[e], tab.mu, u[e]) : m[e];
}

// the momentum's step, and the sum of squares of the update in kSumBlocks parts; memory bound
template <typename G> __global__ void __launch_bounds__(256) k_muon_sums(Table tab) {
    int t = blockIdx.x;
    const Matrix& x = tab.t[find(tab, t)];
    const int matrix = t / kSumBlocks, part = t % kSumBlocks;
    // rows that follow each other are one
    const bool flat = x.g_row == x.cols;
    const int64_t cols = flat ? (int64_t)x.rows * x.cols : x.cols, across = (cols + 7) / 8, all = flat ? across : across * x.rows;
    double sum = 0.0;
    for (int64_t i = (int64_t)part * 256 + threadIdx.x; i < all; i += kSumBlocks * 256) {
        const int64_t r = flat ? 0 : i / across, c = (i - r * across) * 8;
        float u[8];
        load_update<G, true>(x, tab, matrix * x.g_step + r * x.g_row + c, r * cols + c, (int)min(cols - c, (int64_t)8), u);
#pragma unroll
        for (int e = 0; e < 8; e++) sum = fma((double)u[e], (double)u[e], sum);
    }
    for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o, 64);
    __shared__ double waves[4];
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = sum;
    __syncthreads();
    const Layout o = layout(x.rows, x.cols);
    if (threadIdx.x == 0)
        ((double*)(x.held + matrix * o.all + o.sums))[part] = (waves[0] + waves[1]) + (waves[2] + waves[3]);
}

__device__ __forceinline__ void store_parts(f16* row, int64_t c, const float (&v)[8]);

// X, of parts, from the update: 64 x 64 pieces, turned in LDS where the matrix is taller than wide; memory bound
template <typename G> __global__ void __launch_bounds__(256) k_muon_pack(Table tab) {
    __shared__ float turn[64][65];
    int t = blockIdx.x;
    const Matrix& x = tab.t[find(tab, t)];
    const int pieces_r = (x.rows + 63) / 64, pieces_c = (x.cols + 63) / 64;
    const int matrix = t / (pieces_r * pieces_c), piece = t % (pieces_r * pieces_c);
    const Layout o = layout(x.rows, x.cols);
    char* held = x.held + matrix * o.all;
    double sum = ((const double*)(held + o.sums))[threadIdx.x & 63];
    for (int k = 1; k < 64; k <<= 1) sum += __shfl_xor(sum, k, 64);
    const Size size = first_size(sqrt(sum), tab.eps);
    const Factor scaled = factor_of(sqrt(sum), tab.eps, size);
    if (piece == 0 && threadIdx.x == 0) *(Size*)(held + o.sizes) = size;
    const int r0 = piece / pieces_c * 64, c0 = piece % pieces_c * 64;
    const bool tall = x.rows > x.cols;
#pragma unroll
    for (int i = threadIdx.x; i < 64 * 8; i += 256) {
        const int a = i / 8, b = i % 8 * 8, r = r0 + a, c = c0 + b;
        float u[8] = {};
        if (r < x.rows && c < x.cols)
            load_update<G, false>(x, tab, matrix * x.g_step + r * x.g_row + c, (int64_t)r * x.cols + c, x.cols - c, u);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            u[e] = scaled(u[e]);
            if (tall) turn[a][b + e] = u[e];
        }
        if (!tall && r < o.s && c < up_to(o.l, 32)) store_parts((f16*)(held + o.x[0] + r * o.lb), c, u);
    }
    if (!tall) return;
    __syncthreads();
#pragma unroll
    for (int i = threadIdx.x; i < 64 * 8; i += 256) {
        const int a = i / 8, b = i % 8 * 8;  // a row of the result and 8 of its columns
        if (c0 + a >= o.s || r0 + b >= up_to(o.l, 32)) continue;
        float u[8];
#pragma unroll
        for (int e = 0; e < 8; e++) u[e] = turn[b + e][a];
        store_parts((f16*)(held + o.x[0] + (c0 + a) * o.lb), r0 + b, u);
    }
}

enum Kind { kGram, kPoly, kStep };

__device__ __forceinline__ void split_parts(const float (&v)[8], h8& hi, h8& lo) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
        hi[e] = (f16)v[e];
        lo[e] = (f16)(v[e] - (float)hi[e]);
    }
}
// columns c .. c + 7 (c % 8 = 0) of a row of parts
__device__ __forceinline__ void store_parts(f16* row, int64_t c, const float (&v)[8]) {
    h8 hi, lo;
    split_parts(v, hi, lo);
    *(h8*)(row + part_place<2>(c, 0)) = hi;
    *(h8*)(row + part_place<2>(c, 1)) = lo;
}
__device__ __forceinline__ void load_parts(const f16* row, int64_t c, float (&v)[8]) {
    const h8 hi = *(const h8*)(row + part_place<2>(c, 0)), lo = *(const h8*)(row + part_place<2>(c, 1));
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = (float)hi[e] + (float)lo[e];
}
// the first `live` of 8 values of the result, `apart` elements from each other: stored, or a parameter stepped by them
template <bool kApart, typename P>
__device__ __forceinline__ void store_result_of(const Matrix& x, const Table& tab, int64_t at, int64_t apart, int live,
                                                float (&v)[8]) {
    P* p = (P*)x.out + at;
    if (tab.update) {
        float old[8];
        if (kApart) {
#pragma unroll
            for (int e = 0; e < 8; e++) old[e] = e < live ? to_f32<P>(p[e * apart]) : 0.0f;
        } else {
            load_some<P, 8>(p, live, old);
        }
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = fmaf(-x.rate, v[e], old[e] * tab.keep);
    }
    if (kApart) {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (e < live) p[e * apart] = from_f32<P>(v[e]);
    } else {
        store_some<P, 4>(p, live, v);
        store_some<P, 4>(p + 4, live - 4, v + 4);
    }
}
template <bool kApart>
__device__ __forceinline__ void store_result(const Matrix& x, const Table& tab, int64_t at, int64_t apart, int live,
                                             float (&v)[8]) {
    if (tab.out_type == HG_F32) store_result_of<kApart, float>(x, tab, at, apart, live, v);
    else if (tab.out_type == HG_F16) store_result_of<kApart, f16>(x, tab, at, apart, live, v);
    else store_result_of<kApart, bf16>(x, tab, at, apart, live, v);
}

template <int kKind, typename Tl>
__global__ void __launch_bounds__(Tl::kBlock, Tl::kWavesEach) k_muon_product(Table tab) {
    __shared__ __attribute__((aligned(1024))) char lds[Tl::kLds];
    // block b is on chiplet b % 8
    int t = tab.range[blockIdx.x % 8] + (int)(blockIdx.x / 8);
    if (t >= tab.range[blockIdx.x % 8 + 1]) return;
    const Matrix& x = tab.t[find(tab, t)];
    const Layout o = layout(x.rows, x.cols);
    const int tiles_s = (o.s + Tl::kM - 1) / Tl::kM, tiles_n = ((kKind == kStep ? o.l : o.s) + Tl::kN - 1) / Tl::kN;
    const int per = kKind == kStep ? tiles_s * tiles_n : tiles_s * (tiles_s + 1) / 2;
    const int matrix = t / per;
    t -= matrix * per;
    char* held = x.held + matrix * o.all;
    Place at;
    if (kKind == kStep) {
        at = band_place(t, tiles_s, tiles_n);
    } else {  // row by row, from the diagonal on
        at.m = 0;
        while (t >= tiles_s - at.m) t -= tiles_s - at.m++;
        at.n = at.m + t;
    }
    Operand a, b;
    if (kKind == kGram) a = b = {held + (tab.from ? o.x[1] : o.x[0]), o.lb, o.s, (int)o.lb};
    if (kKind == kPoly) a = b = {held + o.a, o.sb, o.s, (int)o.sb};
    if (kKind == kStep) {
        a = {held + o.p, o.sb, o.s, (int)o.sb};
        b = {held + (tab.from ? o.x[1] : o.x[0]), o.lb, o.s, (int)o.lb};
    }
    const int m0 = at.m * Tl::kM, n0 = at.n * Tl::kN;
    Size* const sizes = (Size*)(held + o.sizes) + tab.step;
    Sums<Tl, 1, kKind == kStep> s;
    multiply<Tl, 1, false, kKind == kStep>(a, m0, b, b, n0, 1 << 30, 0, (a.bytes + Tl::kRow - 1) / Tl::kRow, lds, s);
    if (Tl::kTeams > 1 && threadIdx.x >= Tl::kThreads) return;
    constexpr int run = 4 * Tl::kFn;  // of a lane's columns that follow each other
    const bool tall = x.rows > x.cols;
    f16* const to = (f16*)(held + (kKind == kGram ? o.a : kKind == kPoly ? o.p : (tab.from ? o.x[0] : o.x[1])));
    const int wide = kKind == kStep ? o.l : o.s;              // columns of the result
    const int64_t row = (kKind == kStep ? o.lb : o.sb) / 2;   // elements of its packed rows
    const int first = n0 + s.col();
    const int across = (int)(threadIdx.x & 63) / 16;  // the lane's place among the four that share a row
    const bool mirrored = at.n > at.m;  // the tile's mirror image is stored, too: no tile computes it
    float pa = 0.0f, pb = 0.0f, pc = 0.0f;  // P's coefficients of what is held
    int last_e = 0;
    if (kKind == kPoly) {
        const int e = sizes[0].e, less = e - sizes[1].e;
        pa = ldexpf(tab.a, -less);
        pb = ldexpf(tab.b, -2 * e - less);
        pc = ldexpf(tab.c, -4 * e - less);
    }
    if (kKind == kStep && tab.last) last_e = sizes[1].e;
    if (kKind == kGram && at.n == 0 && threadIdx.x == 0) sizes[1] = next_size(sizes[0], tab.a, tab.b, tab.c);
#pragma unroll
    for (int i = 0; i < Tl::kFm; i++) {
        const int m = m0 + s.row() + i * 16;
        const bool there = m < o.s;
        typedef uint32_t u4 __attribute__((ext_vector_type(4)));
        u4 parts[2][run / 8];  // of 8 columns each
#pragma unroll
        for (int c = 0; c < run; c += 8) {
            const int n = first + c, live = wide - n;
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = s.acc[i][(c + e) / 4][e % 4] * (1.0f / (kKind == kStep ? kScaleP : kScale));
            if (kKind == kPoly) {
                float g[8] = {};
                if (there && live > 0) load_parts((const f16*)(held + o.a) + m * row, n, g);
#pragma unroll
                for (int e = 0; e < 8; e++)
                    v[e] = fmaf(pc, v[e], pb * g[e]) * (kScaleP / kScale) + (n + e == m ? pa * kScaleP : 0.0f);
            }
            if (kKind == kStep && tab.last) {
                if (!there || live <= 0) continue;
#pragma unroll
                for (int e = 0; e < 8; e++) v[e] = ldexpf(v[e] * (1.0f / kScale), -last_e);
                // a turned matrix: column n of the result is row n of X's
                if (tall) store_result<true>(x, tab, matrix * x.out_step + (int64_t)n * x.cols + m, x.cols, live, v);
                else store_result<false>(x, tab, matrix * x.out_step + (int64_t)m * x.cols + n, 1, live, v);
                continue;
            }
            h8 hi, lo;
            split_parts(v, hi, lo);
            parts[0][c / 8] = __builtin_bit_cast(u4, hi);
            parts[1][c / 8] = __builtin_bit_cast(u4, lo);
            if (kKind != kStep && mirrored) {
                const int r = s.row() + i * 16, at_c = Tl::template turned_place<Tl::kN / 8>(r, (s.col() + c) / 8);
                *(h8*)(lds + (r * Tl::kN / 8 + at_c) * 16) = hi;
                *(h8*)(lds + Tl::kM * Tl::kN * 2 + (r * Tl::kN / 8 + at_c) * 16) = lo;
            }
        }
        if (kKind == kStep && tab.last) continue;
        // 16 columns a lane: the four lanes' pieces change round, so that a store writes the 64 bytes of a part of 32 columns
#pragma unroll
        for (int p = 0; p < 2; p++) {
            if constexpr (run == 16)
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    uint32_t a = parts[p][0][k], b = parts[p][1][k];
                    spread(a, b);
                    parts[p][0][k] = a;
                    parts[p][1][k] = b;
                }
#pragma unroll
            for (int k = 0; k < run / 8; k++) {
                const int group = n0 + s.first_col() + k * 32;  // its first column
                if (there && group < wide) *(u4*)(to + m * row + part_place<2>(group, p) + across * 8) = parts[p][k];
            }
        }
    }
    if constexpr (kKind != kStep) {
        if (!mirrored) return;
        static_assert(Tl::kLds >= Tl::kM * Tl::kN * 4 && Tl::kM == Tl::kN, "");
        __syncthreads();
        // 16 rows of the mirror image and 32 of their columns at a time, turned by the LDS reads
        const int lane = threadIdx.x & 63, l = lane & 15, g = lane >> 4;
        for (int k = threadIdx.x >> 6; k < 2 * (Tl::kN / 16) * (Tl::kM / 32); k += Tl::kThreads / 64) {
            const int p = k & 1, piece = k / 2 % (Tl::kN / 16), block = k / 2 / (Tl::kN / 16);
            typedef short s4 __attribute__((ext_vector_type(4)));
            typedef short s8 __attribute__((ext_vector_type(8)));
            typedef __attribute__((address_space(3))) s4* Lds;
            const int r = block * 32 + g * 8 + l / 4, c = Tl::template turned_place<Tl::kN / 8>(r, piece * 2 + l % 4 / 2);
            const char* first = lds + p * Tl::kM * Tl::kN * 2 + (r * Tl::kN / 8 + c) * 16 + l % 2 * 8;
            const s4 u = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)first);
            const s4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(first + 4 * Tl::kN * 2));
            const int n = n0 + piece * 16 + l, m = m0 + block * 32 + g * 8;
            if (n < o.s) *(s8*)(to + n * row + part_place<2>(m, p)) = s8{u[0], u[1], u[2], u[3], v[0], v[1], v[2], v[3]};
        }
    }
}

// The whole step of a matrix whose shorter side is at most 64 and whose longer one at most kL: a block holds X, A and P in
// LDS and takes every product there, where the products of larger ones take three launches an iteration (28 us for the
// self-play network's three matrices, 110 by launches; a block's products and barriers follow each other).  Rows of 64 values and more, so that the 16 rows that are read
// together can begin in 16 different places: chunk c of row r is held at place(r, c), which also spreads the rows that a
// turned read takes.
constexpr int kSmall = 64;
template <int kL, typename G>
__global__ void __launch_bounds__(1024) k_muon_small(Table tab) {
    constexpr int kRowX = kL * 4, kRowA = kSmall * 4, kPieces = kL / 64;  // bytes; a wave's pieces of 16 x 16 of X
    constexpr int kEach = kSmall * kL / 1024;                             // values a thread loads
    __shared__ __attribute__((aligned(256))) char lds[kSmall * (kRowX + 2 * kRowA)];
    __shared__ double waves[16];
    char* const lx = lds;
    char* const la = lds + kSmall * kRowX;
    char* const lp = la + kSmall * kRowA;
    auto place = [](int r, int c) { return c ^ (((r & 3) | (r >> 1 & 4)) << 1 | (r >> 2 & 1)); };
    // byte of column c's part p in row r
    auto byte = [&](int r, int c, int p) { return place(r, c / 32 * 8 + p * 4 + c % 32 / 8) * 16 + c % 8 * 2; };
    int t = blockIdx.x;
    const Matrix& x = tab.t[find(tab, t)];
    const int matrix = t, rows = x.rows, cols = x.cols, n = rows * cols;
    const bool tall = rows > cols;
    const int s = tall ? cols : rows, l = tall ? rows : cols;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, row16 = lane & 15, g = lane >> 4;
    float u[kEach], m[kEach];
    // i / cols = the high word of i times it, rounded up: exact for i below 2^14 and cols up to 2^8
    const uint32_t inverse = 0xFFFFFFFFu / (uint32_t)cols + 1;
    const G* from = (const G*)x.g + matrix * x.g_step;
    auto row_of = [&](int i) { return cols == 1 ? i : (int)__umulhi((uint32_t)i, inverse); };
#pragma unroll
    for (int k = 0; k < kEach; k++) {  // all loads under way before the first value is used
        const int i = k * 1024 + tid, r = row_of(i);
        u[k] = i < n ? to_f32<G>(from[r * x.g_row + i - r * cols]) : 0.0f;
    }
#pragma unroll
    for (int k = 0; k < kEach; k++) {
        const int i = k * 1024 + tid;
        m[k] = i < n && x.momentum ? x.momentum[i] : 0.0f;
    }
    for (int i = tid; i < (int)sizeof(lds) / 16; i += 1024) ((float4*)lds)[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < kEach; k++) {
        const int i = k * 1024 + tid;
        if (x.momentum) {
            m[k] = fmaf(m[k], tab.mu, u[k]);
            if (i < n) x.momentum[i] = m[k];
            u[k] = tab.nesterov ? fmaf(m[k], tab.mu, u[k]) : m[k];
        }
        sum = fma((double)u[k], (double)u[k], sum);
    }
    for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o, 64);
    if (lane == 0) waves[wave] = sum;
    __syncthreads();
    sum = 0.0;
    for (int i = 0; i < 16; i++) sum += waves[i];
    Size size = first_size(sqrt(sum), tab.eps);
    const Factor scaled = factor_of(sqrt(sum), tab.eps, size);
#pragma unroll
    for (int k = 0; k < kEach; k++) {
        const int i = k * 1024 + tid;
        if (i >= n) continue;
        const int of = row_of(i), in = i - of * cols, r = tall ? in : of, c = tall ? of : in;
        f16 part[2];
        split<f16, 2>(scaled(u[k]), part);
        *(f16*)(lx + r * kRowX + byte(r, c, 0)) = part[0];
        *(f16*)(lx + r * kRowX + byte(r, c, 1)) = part[1];
    }
    __syncthreads();
    auto operand = [&](const char* from, int row, int piece, int k, int p) {  // rows as they are
        const int r = piece * 16 + row16;
        return *(const h8*)(from + r * row + place(r, k * 8 + p * 4 + g) * 16);
    };
    auto turned = [&](int piece, int k, int p) {  // of X: 4 k each of two reads
        typedef short s4 __attribute__((ext_vector_type(4)));
        typedef short s8 __attribute__((ext_vector_type(8)));
        typedef __attribute__((address_space(3))) s4* Lds;
        const int c = (piece / 2 * 2 + p) * 4 + piece % 2 * 2 + row16 % 4 / 2, r = k * 32 + g * 8 + row16 / 4;
        const s4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(lx + r * kRowX + place(r, c) * 16 + row16 % 2 * 8));
        const s4 w = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(lx + (r + 4) * kRowX + place(r + 4, c) * 16 + row16 % 2 * 8));
        return __builtin_bit_cast(h8, (s8){v[0], v[1], v[2], v[3], w[0], w[1], w[2], w[3]});
    };
    auto add = [](f4 c, const h8 (&a)[2], const h8 (&b)[2]) {
        c = mfma(b[0], a[1], c);
        c = mfma(b[1], a[0], c);
        return mfma(b[0], a[0], c);
    };
    typedef f16 half4 __attribute__((ext_vector_type(4)));
    auto keep = [&](char* to, int row, int r, int c, const float (&v)[4]) {
        half4 hi, lo;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            hi[e] = (f16)v[e];
            lo[e] = (f16)(v[e] - (float)hi[e]);
        }
        *(half4*)(to + r * row + byte(r, c, 0)) = hi;
        *(half4*)(to + r * row + byte(r, c, 1)) = lo;
    };
    const int pm = wave / 4, pn = wave % 4;  // the wave's piece of A and of P; zeros past the matrix are multiplied like the rest
    const int r = pm * 16 + row16;
    auto finish = [&](auto type, const f4 (&next)[kPieces]) {
        using P = decltype(type);
        P* out = (P*)x.out + matrix * x.out_step;
        int at[kPieces][4];
        float old[kPieces][4];
#pragma unroll
        for (int j = 0; j < kPieces; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int c = (pn + 4 * j) * 16 + g * 4 + e;
                at[j][e] = r < s && c < l ? (tall ? c * cols + r : r * cols + c) : -1;
                old[j][e] = tab.update && at[j][e] >= 0 ? to_f32<P>(out[at[j][e]]) : 0.0f;
            }
#pragma unroll
        for (int j = 0; j < kPieces; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float o = ldexpf(next[j][e] * (1.0f / kScaleP / kScale), -size.e);
                if (at[j][e] >= 0) out[at[j][e]] = from_f32<P>(tab.update ? fmaf(-x.rate, o, old[j][e] * tab.keep) : o);
            }
    };
    for (int step = 0; step < tab.steps; step++) {
        const float* abc = tab.triples + 3 * min(step, tab.count - 1);
        const Size next_s = next_size(size, abc[0], abc[1], abc[2]);
        const int less = size.e - next_s.e;
        const float pa = ldexpf(abc[0], -less), pb = ldexpf(abc[1], -2 * size.e - less), pc = ldexpf(abc[2], -4 * size.e - less);
        size = next_s;
        f4 sum_a = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < kL / 32; k++) {
            const h8 a[2] = {operand(lx, kRowX, pm, k, 0), operand(lx, kRowX, pm, k, 1)};
            const h8 b[2] = {operand(lx, kRowX, pn, k, 0), operand(lx, kRowX, pn, k, 1)};
            sum_a = add(sum_a, a, b);
        }
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = sum_a[e] * (1.0f / kScale);
        keep(la, kRowA, r, pn * 16 + g * 4, v);
        __syncthreads();
        f4 sum_p = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < kSmall / 32; k++) {
            const h8 a[2] = {operand(la, kRowA, pm, k, 0), operand(la, kRowA, pm, k, 1)};
            const h8 b[2] = {operand(la, kRowA, pn, k, 0), operand(la, kRowA, pn, k, 1)};
            sum_p = add(sum_p, a, b);
        }
#pragma unroll
        for (int e = 0; e < 4; e++)
            v[e] = fmaf(pc, sum_p[e] * (1.0f / kScale), pb * v[e]) * (kScaleP / kScale) +
                   (pn * 16 + g * 4 + e == r ? pa * kScaleP : 0.0f);
        keep(lp, kRowA, r, pn * 16 + g * 4, v);
        __syncthreads();
        h8 p[kSmall / 32][2];
#pragma unroll
        for (int k = 0; k < kSmall / 32; k++) {
            p[k][0] = operand(lp, kRowA, pm, k, 0);
            p[k][1] = operand(lp, kRowA, pm, k, 1);
        }
        f4 next[kPieces];
#pragma unroll
        for (int j = 0; j < kPieces; j++) {
            next[j] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < kSmall / 32; k++) {
                const h8 b[2] = {turned(pn + 4 * j, k, 0), turned(pn + 4 * j, k, 1)};
                next[j] = add(next[j], p[k], b);
            }
        }
        if (step < tab.steps - 1) {
            __syncthreads();  // X is read
#pragma unroll
            for (int j = 0; j < kPieces; j++) {
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = next[j][e] * (1.0f / kScaleP);
                keep(lx, kRowX, r, (pn + 4 * j) * 16 + g * 4, v);
            }
            __syncthreads();
        } else {
            if (tab.out_type == HG_F32) finish(float{}, next);
            else if (tab.out_type == HG_F16) finish(f16{}, next);
            else finish(bf16{}, next);
        }
    }
}

int launched() { return (int)hipGetLastError(); }

// the table's blocks: f(matrix) of each
template <typename F> int64_t lay_blocks(Table& tab, F f) {
    int64_t blocks = 0;
    for (int i = 0; i < tab.n; i++) {
        tab.t[i].first = (int)blocks;
        blocks += f(tab.t[i]) * tab.t[i].count;
    }
    return blocks;
}

// Shares the tiles of a product out among the chiplets, each of which has an L2 of its own: ranges of tiles that follow each
// other, of equal work (a tile's sum is as long as `depth` says), so that a matrix is read by one or two of them (A of
// 24 matrices of 1,024 x 1,024 and 4,096: 0.4 GB from memory, 1.1 where every chiplet has tiles of every matrix).  Returns the
// blocks to launch.
template <typename F, typename D> int64_t lay_ranges(Table& tab, F tiles, D depth) {
    int64_t work = 0, done = 0;
    for (int i = 0; i < tab.n; i++) work += tiles(tab.t[i]) * tab.t[i].count * depth(tab.t[i]);
    int64_t most = 0;
    int x = 0;
    for (int i = 0; i < tab.n; i++) {
        const int64_t all = tiles(tab.t[i]) * tab.t[i].count, each = depth(tab.t[i]);
        // chiplet x begins at the first tile before which x / 8 of the work is done
        while (x < 8 && work * x <= 8 * (done + all * each)) {
            const int64_t before = std::max<int64_t>(0, (work * x / 8 - done + each - 1) / each);
            tab.range[x++] = tab.t[i].first + (int)std::min(before, all);
        }
        done += all * each;
        tab.range[8] = tab.t[i].first + (int)all;
    }
    while (x < 8) tab.range[x++] = tab.range[8];
    for (x = 0; x < 8; x++) most = std::max<int64_t>(most, tab.range[x + 1] - tab.range[x]);
    return 8 * most;
}

template <typename Tl> int64_t step_tiles(const Matrix& x, bool symmetric) {
    const int s = std::min(x.rows, x.cols), l = std::max(x.rows, x.cols);
    const int m = (s + Tl::kM - 1) / Tl::kM, n = ((symmetric ? s : l) + Tl::kN - 1) / Tl::kN;
    return symmetric ? (int64_t)m * (m + 1) / 2 : (int64_t)m * n;
}

// f called with the tile that a product of the table's matrices takes, their blocks laid out by it: the largest tiles of which
// there are enough for the card (P X of 24 matrices of 1,024 x 1,024 and 4,096 in 256 x 256 298 us, in 128 x 128 344).
template <int kKind, typename F> int with_tile(Table& tab, F f) {
    auto blocks = [&](auto tile) {
        return lay_blocks(tab, [](const Matrix& x) { return step_tiles<decltype(tile)>(x, kKind != kStep); });
    };
    if constexpr (kKind == kStep) {
        const Tile<f16, 2, 1, 256, 256, 2, 4, 2, 1, false> large;
        if (blocks(large) >= 192) return f(large);
    }
    const Tile<f16, 2, 1, 128, 128, 2, 2, 2, 2> middle;
    if (blocks(middle) >= 192) return f(middle);
    // a block a compute unit at most: of two teams, so that a SIMD has two waves all the same (a matrix of 1,024 x 1,024:
    // A 13.7 -> 12.8 us, P 14.4 -> 13.3, P X 16.0 -> 15.0)
    const Tile<f16, 2, 1, 64, 64, 2, 2, 4, 1, true, 2> teams;
    if (blocks(teams) <= 256) return f(teams);
    const Tile<f16, 2, 1, 64, 64, 2, 2, 4, 2> small;  // the same tiles
    return f(small);
}

// one product of every matrix of the table
template <int kKind> int product(Table& tab, hipStream_t st) {
    return with_tile<kKind>(tab, [&](auto tile) {
        using Tl = decltype(tile);
        const int64_t grid = lay_ranges(
            tab, [](const Matrix& x) { return step_tiles<Tl>(x, kKind != kStep); },
            [](const Matrix& x) { return (int64_t)(kKind == kGram ? std::max(x.rows, x.cols) : std::min(x.rows, x.cols)); });
        k_muon_product<kKind, Tl><<<(unsigned)grid, Tl::kBlock, 0, st>>>(tab);
        return launched();
    });
}

// whether a block holds a matrix whose longer side is at most `side`
bool fits_block(const Matrix& x, int side) {
    return std::min(x.rows, x.cols) <= kSmall && std::max(x.rows, x.cols) <= side;
}

// the matrices of the table that `small` says, their whole iteration in one launch
template <int kL, typename F> int iterate_small(const Table& all, F small, hipStream_t st) {
    Table tab = all;
    tab.n = 0;
    for (int i = 0; i < all.n; i++)
        if (small(all.t[i])) tab.t[tab.n++] = all.t[i];
    if (tab.n == 0) return 0;
    const int64_t blocks = lay_blocks(tab, [](const Matrix&) { return (int64_t)1; });
    return with_type(tab.g_type, [&](auto t) {
        k_muon_small<kL, decltype(t)><<<(unsigned)blocks, 1024, 0, st>>>(tab);
        return launched();
    });
}

// the iteration of the table's matrices
int iterate(Table& all, int steps, const float* coefficients, int64_t triples, hipStream_t st) {
    all.steps = steps;
    all.count = (int)std::min<int64_t>(triples, steps);
    auto fits = [&](const Matrix& x, int side) { return fits_block(x, side) && all.count <= kTriples; };
    for (int i = 0; i < 3 * all.count && i < 3 * kTriples; i++) all.triples[i] = coefficients[i];
    int e = iterate_small<128>(all, [&](const Matrix& x) { return fits(x, 128); }, st);
    if (!e) e = iterate_small<256>(all, [&](const Matrix& x) { return fits(x, 256) && !fits(x, 128); }, st);
    if (e) return e;
    Table tab = all;
    tab.n = 0;
    for (int i = 0; i < all.n; i++)
        if (!fits(all.t[i], 256)) tab.t[tab.n++] = all.t[i];
    if (tab.n == 0) return 0;
    // the longest sums first: what is left at the end of a launch is short
    std::sort(tab.t, tab.t + tab.n, [](const Matrix& a, const Matrix& b) {
        return std::max(a.rows, a.cols) > std::max(b.rows, b.cols);
    });
    int64_t blocks = lay_blocks(tab, [](const Matrix&) { return (int64_t)kSumBlocks; });
    e = with_type(tab.g_type, [&](auto t) {
        k_muon_sums<decltype(t)><<<(unsigned)blocks, 256, 0, st>>>(tab);
        return launched();
    });
    if (e) return e;
    blocks = lay_blocks(tab, [](const Matrix& x) { return (int64_t)((x.rows + 63) / 64) * ((x.cols + 63) / 64); });
    e = with_type(tab.g_type, [&](auto t) {
        k_muon_pack<decltype(t)><<<(unsigned)blocks, 256, 0, st>>>(tab);
        return launched();
    });
    tab.from = 0;
    for (int i = 0; i < steps && !e; i++) {
        const float* c = coefficients + 3 * std::min<int64_t>(i, triples - 1);
        tab.a = c[0];
        tab.b = c[1];
        tab.c = c[2];
        tab.step = i;
        tab.last = i == steps - 1;
        e = product<kGram>(tab, st);
        if (!e) e = product<kPoly>(tab, st);
        if (!e) e = product<kStep>(tab, st);
        tab.from ^= 1;
    }
    return e;
}

bool bad_settings(int steps, const float* coefficients, int triples, float eps) {
    return steps < 1 || steps > kMostSteps || !coefficients || triples < 1 || !(eps >= 0.0f);
}
// a launch has under 2^32 threads, 256 for a piece of 64 x 64
bool bad_shape(int64_t count, int64_t rows, int64_t cols) {
    return rows < 1 || cols < 1 || rows > kMaxSide || cols > kMaxSide || count > 1 << 16 ||
           count * (rows / 64 + 1) * (cols / 64 + 1) > 2049 * 2049;
}

}  // namespace

extern "C" {

int64_t hg_orthogonalize_workspace(int64_t count, int64_t rows, int64_t cols) {
    if (count < 1 || bad_shape(count, rows, cols)) return 0;
    return count * layout((int)rows, (int)cols).all;
}

int hg_orthogonalize(const void* u, int type, int64_t count, int64_t rows, int64_t cols, int64_t u_row, int64_t u_step,
                     int steps, const float* coefficients, int triples, float eps, void* out, void* workspace,
                     void* stream) {
    if (!is_type(type) || count < 0 || bad_shape(count, rows, cols) || bad_settings(steps, coefficients, triples, eps))
        return (int)hipErrorInvalidValue;
    if (count == 0) return 0;
    if (!u || !out || !workspace || (uintptr_t)workspace % 256) return (int)hipErrorInvalidValue;
    Table tab{};
    tab.n = 1;
    tab.t[0] = {u, nullptr, out, (char*)workspace, u_row, u_step, rows * cols, 0.0f, (int)rows, (int)cols, (int)count, 0};
    tab.g_type = tab.out_type = type;
    tab.eps = eps;
    return iterate(tab, steps, coefficients, triples, (hipStream_t)stream);
}

int hg_orthogonalize_tiles(int64_t count, int64_t rows, int64_t cols, int tiles[2]) {
    if (count < 1 || bad_shape(count, rows, cols) || !tiles) return (int)hipErrorInvalidValue;
    Table tab{};
    tab.n = 1;
    tab.t[0].rows = (int)rows;
    tab.t[0].cols = (int)cols;
    tab.t[0].count = (int)count;
    auto name = [](auto tile) { return name_of<decltype(tile)>(); };
    const bool small = fits_block(tab.t[0], 256);
    tiles[0] = small ? 0 : with_tile<kGram>(tab, name);
    tiles[1] = small ? 0 : with_tile<kStep>(tab, name);
    return 0;
}

int64_t hg_muon_step_workspace(const hg_muon_matrix* matrices, int64_t count) {
    int64_t most = 0;
    for (int64_t i = 0; matrices && i < count; i += kMatrices) {
        int64_t bytes = 0;
        for (int64_t k = i; k < std::min(count, i + kMatrices); k++)
            if (!bad_shape(1, matrices[k].rows, matrices[k].cols))
                bytes += layout((int)matrices[k].rows, (int)matrices[k].cols).all;
        most = std::max(most, bytes);
    }
    return most;
}

int hg_muon_step(const hg_muon_matrix* matrices, int64_t count, int param_type, int grad_type, double lr, double momentum,
                 int nesterov, double weight_decay, int steps, const float* coefficients, int triples, float eps,
                 void* workspace, void* stream) {
    if (count < 0 || (count > 0 && !matrices) || !is_type(param_type) || !is_type(grad_type) ||
        bad_settings(steps, coefficients, triples, eps))
        return (int)hipErrorInvalidValue;
    for (int64_t i = 0; i < count; i++)
        if (bad_shape(1, matrices[i].rows, matrices[i].cols) || !matrices[i].param || !matrices[i].momentum ||
            (uintptr_t)matrices[i].momentum % 4)
            return (int)hipErrorInvalidValue;
    if (count > 0 && (!workspace || (uintptr_t)workspace % 256)) return (int)hipErrorInvalidValue;
    // the same kMatrices matrices a launch as the workspace is sized for, whichever of them have a gradient
    for (int64_t i = 0; i < count; i += kMatrices) {
        Table tab{};
        char* held = (char*)workspace;
        for (int64_t k = i; k < std::min(count, i + kMatrices); k++) {
            const hg_muon_matrix& m = matrices[k];
            if (!m.grad) continue;
            const int rows = (int)m.rows, cols = (int)m.cols;
            tab.t[tab.n++] = {m.grad, m.momentum, m.param, held, m.cols, 0, 0, (float)(lr * m.scale), rows, cols, 1, 0};
            held += layout(rows, cols).all;
        }
        if (tab.n == 0) continue;
        tab.g_type = grad_type;
        tab.out_type = param_type;
        tab.update = 1;
        tab.mu = (float)momentum;
        tab.nesterov = nesterov;
        tab.keep = (float)(1.0 - lr * weight_decay);
        tab.eps = eps;
        const int e = iterate(tab, steps, coefficients, triples, (hipStream_t)stream);
        if (e) return e;
    }
    return 0;
}

}  // extern "C"
