// hive_muon.hip -- orthogonalised updates: the Newton-Schulz iteration of a
// batch of matrices, and the step of many of a network's matrices with it.
//
//   X = U / (|U| + eps), |U| the root of the sum of squares
//   steps times:  A = X X^T,  P = b A + c A A,  X <- a X + P X
// which takes each singular value s to a s + b s^3 + c s^5, and with the usual
// (a, b, c) all of them near 1.  X has the shorter side's rows: a matrix that is
// taller than wide is turned, and turned back at the end.  A step with it:
//   m = mu m + g,  u = g + mu m or m,  p = p keep - rate X(u)
//
// The iteration takes small singular values up 3.4445 times at each of its
// first steps, and with them what rounding has put in their place: at 16-bit
// rounding that would be the result.  Every matrix is held as two float16 parts a
// value, 22 bits, times 2^13 (entries are below 2 in size and mostly far below 1;
// their last parts stay above float16's smallest), and products are three
// matrix instructions of parts (hive_matrix.hpp).
//
// X is an operand by its rows in X X^T and by its columns in P X.  A and A A are
// symmetric: the tiles on and above the diagonal are computed, and stored twice.
#include <algorithm>
#include <cmath>

#include "hive_pack.hpp"

namespace {

using namespace hm;

constexpr int kMatrices = 24;        // of a launch: their table is a kernel argument
constexpr float kScale = 8192.0f;    // of every held matrix
constexpr int kSumBlocks = 64;       // of a matrix's sum of squares
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
    int n, blocks;
    int g_type, out_type, update;  // update: out is a parameter
    float mu, keep, eps, a, b, c;
    int nesterov, from, last;  // from: which of the two copies of X is current
};

// where a matrix's parts lie in its workspace, in bytes
struct Layout {
    int s, l;                // the shorter and the longer side
    int64_t sb, lb;          // bytes of a packed row along each
    int64_t x[2], a, p, sums, all;
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
    o.all = o.sums + up_to(kSumBlocks * 8, 256);
    return o;
}

__device__ __forceinline__ float load_any(const void* p, int type, int64_t i) {
    return type == HG_F32 ? ((const float*)p)[i] : type == HG_F16 ? (float)((const f16*)p)[i] : (float)((const bf16*)p)[i];
}
__device__ __forceinline__ void store_any(void* p, int type, int64_t i, float v) {
    if (type == HG_F32) ((float*)p)[i] = v;
    else if (type == HG_F16) ((f16*)p)[i] = (f16)v;
    else ((bf16*)p)[i] = (bf16)v;
}

// the matrix that block t works on, t from there on its own
__device__ __forceinline__ int find(const Table& tab, int& t) {
    int i = 0;
    while (i + 1 < tab.n && tab.t[i + 1].first <= t) i++;
    t -= tab.t[i].first;
    return i;
}

// the momentum's step, and the sum of squares of the update in kSumBlocks parts
__global__ void __launch_bounds__(256) k_muon_sums(Table tab) {
    int t = blockIdx.x;
    const Matrix& x = tab.t[find(tab, t)];
    const int matrix = t / kSumBlocks, part = t % kSumBlocks;
    const int64_t all = (int64_t)x.rows * x.cols;
    const int64_t each = (all + kSumBlocks - 1) / kSumBlocks, begin = part * each, end = min(begin + each, all);
    double sum = 0.0;
    for (int64_t i = begin + threadIdx.x; i < end; i += 256) {
        const int64_t r = i / x.cols, c = i - r * x.cols;
        float u = load_any(x.g, tab.g_type, matrix * x.g_step + r * x.g_row + c);
        if (x.momentum) {
            const float m = fmaf(x.momentum[i], tab.mu, u);
            x.momentum[i] = m;
            u = tab.nesterov ? fmaf(m, tab.mu, u) : m;
        }
        sum = fma((double)u, (double)u, sum);
    }
    for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o, 64);
    __shared__ double waves[4];
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = sum;
    __syncthreads();
    const Layout o = layout(x.rows, x.cols);
    if (threadIdx.x == 0)
        ((double*)(x.held + matrix * o.all + o.sums))[part] = (waves[0] + waves[1]) + (waves[2] + waves[3]);
}

// X, of parts, from the update: 64 x 64 pieces, turned in LDS where the matrix is taller than wide
__global__ void __launch_bounds__(256) k_muon_pack(Table tab) {
    __shared__ float turn[64][65];
    int t = blockIdx.x;
    const Matrix& x = tab.t[find(tab, t)];
    const int pieces_r = (x.rows + 63) / 64, pieces_c = (x.cols + 63) / 64;
    const int matrix = t / (pieces_r * pieces_c), piece = t % (pieces_r * pieces_c);
    const Layout o = layout(x.rows, x.cols);
    char* held = x.held + matrix * o.all;
    double sum = ((const double*)(held + o.sums))[threadIdx.x & 63];
    for (int k = 1; k < 64; k <<= 1) sum += __shfl_xor(sum, k, 64);
    const float scale = (float)((double)kScale / (sqrt(sum) + (double)tab.eps));
    const int r0 = piece / pieces_c * 64, c0 = piece % pieces_c * 64;
    for (int i = threadIdx.x; i < 64 * 64; i += 256) {
        const int r = r0 + i / 64, c = c0 + i % 64;
        float u = 0.0f;
        if (r < x.rows && c < x.cols) {
            u = load_any(x.g, tab.g_type, matrix * x.g_step + r * x.g_row + c);
            if (x.momentum) {
                const float m = x.momentum[(int64_t)r * x.cols + c];
                u = tab.nesterov ? fmaf(m, tab.mu, u) : m;
            }
            u *= scale;
        }
        turn[i / 64][i % 64] = u;
    }
    __syncthreads();
    const bool tall = x.rows > x.cols;
    for (int i = threadIdx.x; i < 64 * 8; i += 256) {
        const int a = i / 8, b = i % 8 * 8;  // a row of the result and 8 of its columns
        const int row = (tall ? c0 : r0) + a, col = (tall ? r0 : c0) + b;
        if (row >= o.s || col >= up_to(o.l, 32)) continue;
        h8 hi, lo;
#pragma unroll
        for (int k = 0; k < 8; k++) {
            f16 part[2];
            split<f16, 2>(tall ? turn[b + k][a] : turn[a][b + k], part);
            hi[k] = part[0];
            lo[k] = part[1];
        }
        f16* to = (f16*)(held + o.x[0] + row * o.lb);
        *(h8*)(to + part_place<2>(col, 0)) = hi;
        *(h8*)(to + part_place<2>(col, 1)) = lo;
    }
}

enum Kind { kGram, kPoly, kStep };

// the tiles of a symmetric result on and above the diagonal, each `wide` times as wide as high: row i has those from i / wide on
__host__ __device__ inline int upper_tiles(int m, int n, int wide) {
    int all = 0;
    for (int i = 0; i < m; i++) all += n - i / wide;
    return all;
}

// columns c .. c + 7 (c % 8 = 0) of a row of parts
__device__ __forceinline__ void store_parts(f16* row, int64_t c, const float (&v)[8]) {
    h8 hi, lo;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        hi[e] = (f16)v[e];
        lo[e] = (f16)(v[e] - (float)hi[e]);
    }
    *(h8*)(row + part_place<2>(c, 0)) = hi;
    *(h8*)(row + part_place<2>(c, 1)) = lo;
}
__device__ __forceinline__ void load_parts(const f16* row, int64_t c, float (&v)[8]) {
    const h8 hi = *(const h8*)(row + part_place<2>(c, 0)), lo = *(const h8*)(row + part_place<2>(c, 1));
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = (float)hi[e] + (float)lo[e];
}
// the same columns, one row each, at column `c`
__device__ __forceinline__ void store_parts_down(f16* first, int64_t row, int64_t c, int live, const float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const f16 hi = (f16)v[e];
        if (e < live) {
            first[e * row + part_place<2>(c, 0)] = hi;
            first[e * row + part_place<2>(c, 1)] = (f16)(v[e] - (float)hi);
        }
    }
}

template <int kKind, typename Tl>
__global__ void __launch_bounds__(Tl::kThreads, Tl::kWavesEach) k_muon_product(Table tab) {
    __shared__ __attribute__((aligned(1024))) char lds[Tl::kLds];
    int t = chiplet_order(blockIdx.x, tab.blocks);
    const Matrix& x = tab.t[find(tab, t)];
    const Layout o = layout(x.rows, x.cols);
    constexpr int wide_tile = Tl::kN / Tl::kM;
    const int tiles_s = (o.s + Tl::kM - 1) / Tl::kM, tiles_n = ((kKind == kStep ? o.l : o.s) + Tl::kN - 1) / Tl::kN;
    const int per = kKind == kStep ? tiles_s * tiles_n : upper_tiles(tiles_s, tiles_n, wide_tile);
    const int matrix = t / per;
    t -= matrix * per;
    char* held = x.held + matrix * o.all;
    Place at;
    if (kKind == kStep) {
        at = band_place(t, tiles_s, tiles_n);
    } else {  // row by row, from the diagonal on
        at.m = 0;
        while (t >= tiles_n - at.m / wide_tile) t -= tiles_n - at.m++ / wide_tile;
        at.n = at.m / wide_tile + t;
    }
    Operand a, b;
    if (kKind == kGram) a = b = {held + o.x[tab.from], o.lb, o.s, (int)o.lb};
    if (kKind == kPoly) a = b = {held + o.a, o.sb, o.s, (int)o.sb};
    if (kKind == kStep) {
        a = {held + o.p, o.sb, o.s, (int)o.sb};
        b = {held + o.x[tab.from], o.lb, o.s, (int)o.lb};
    }
    const int m0 = at.m * Tl::kM, n0 = at.n * Tl::kN;
    Sums<Tl, 1, kKind == kStep> s;
    multiply<Tl, 1, false, kKind == kStep>(a, m0, b, b, n0, 1 << 30, 0, (a.bytes + Tl::kRow - 1) / Tl::kRow, lds, s);
    constexpr int run = 4 * Tl::kFn;  // of a lane's columns that follow each other
    const bool tall = x.rows > x.cols;
    f16* const to = (f16*)(held + (kKind == kGram ? o.a : kKind == kPoly ? o.p : o.x[tab.from ^ 1]));
    const int wide = kKind == kStep ? o.l : o.s;              // columns of the result
    const int64_t row = (kKind == kStep ? o.lb : o.sb) / 2;   // elements of its packed rows
    const int first = n0 + s.col();
#pragma unroll
    for (int i = 0; i < Tl::kFm; i++) {
        const int m = m0 + s.row() + i * 16;
        if (m >= up_to(o.s, 32)) continue;
        const bool there = m < o.s;
#pragma unroll
        for (int c = 0; c < run; c += 8) {
            const int n = first + c, live = wide - n;
            if (n >= up_to(wide, 32)) continue;
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = s.acc[i][(c + e) / 4][e % 4] * (1.0f / kScale);
            if (kKind == kPoly) {
                float g[8] = {};
                if (there) load_parts((const f16*)(held + o.a) + m * row, n, g);
#pragma unroll
                for (int e = 0; e < 8; e++) v[e] = fmaf(tab.c, v[e], tab.b * g[e]);
            }
            if (kKind == kStep) {
                float g[8] = {};
                if (there) load_parts((const f16*)(held + o.x[tab.from]) + m * row, n, g);
#pragma unroll
                for (int e = 0; e < 8; e++) v[e] = fmaf(tab.a, g[e], v[e]);
                if (tab.last) {
                    if (!there) continue;
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        if (e >= live) break;
                        const int64_t i_out = matrix * x.out_step + (tall ? (int64_t)(n + e) * x.cols + m
                                                                          : (int64_t)m * x.cols + n + e);
                        float r = v[e] * (1.0f / kScale);
                        if (tab.update) r = fmaf(-x.rate, r, load_any(x.out, tab.out_type, i_out) * tab.keep);
                        store_any(x.out, tab.out_type, i_out, r);
                    }
                    continue;
                }
            }
            if (there) store_parts(to + m * row, n, v);
            if (kKind != kStep && at.n > at.m / wide_tile)  // the tile's mirror image, where no tile is
                store_parts_down(to + n * row, row, m, live, v);
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
    tab.blocks = (int)blocks;
    return blocks;
}

template <typename Tl> int64_t step_tiles(const Matrix& x, bool symmetric) {
    const int s = std::min(x.rows, x.cols), l = std::max(x.rows, x.cols);
    const int m = (s + Tl::kM - 1) / Tl::kM, n = ((symmetric ? s : l) + Tl::kN - 1) / Tl::kN;
    return symmetric ? upper_tiles(m, n, Tl::kN / Tl::kM) : (int64_t)m * n;
}

// one product of every matrix of the table, in the largest tiles of which there are enough for the card
template <int kKind> int product(Table& tab, hipStream_t st) {
    auto launch = [&](auto tile, int64_t least) {
        using Tl = decltype(tile);
        const int64_t blocks = lay_blocks(tab, [](const Matrix& x) { return step_tiles<Tl>(x, kKind != kStep); });
        if (blocks < least) return -1;
        k_muon_product<kKind, Tl><<<(unsigned)blocks, Tl::kThreads, 0, st>>>(tab);
        return launched();
    };
#ifdef TRY
    int e = -1;
    if (TRY == 1) e = launch(Tile<f16, 2, 1, 128, 128, 2, 2, 2, 2>{}, 192);
    if (TRY == 2) e = launch(Tile<f16, 2, 1, 128, 256, 2, 4, 3, 1>{}, 192);
    if (TRY == 3) e = launch(Tile<f16, 2, 1, 128, 128, 2, 2, 4, 1>{}, 192);
    if (TRY == 4) e = launch(Tile<f16, 2, 1, 128, 256, 4, 4, 3, 1>{}, 192);
#else
    int e = launch(Tile<f16, 2, 1, 128, 256, 2, 4, 3, 1>{}, 192);
#endif
    if (e < 0) e = launch(Tile<f16, 2, 1, 128, 128, 2, 2, 2, 2>{}, 192);
    if (e < 0) e = launch(Tile<f16, 2, 1, 64, 64, 2, 2, 4, 2>{}, 0);
    return e;
}

// the iteration of the table's matrices
int iterate(Table& tab, int steps, const float* coefficients, int64_t triples, hipStream_t st) {
    int64_t blocks = lay_blocks(tab, [](const Matrix&) { return (int64_t)kSumBlocks; });
    k_muon_sums<<<(unsigned)blocks, 256, 0, st>>>(tab);
    int e = launched();
    if (e) return e;
    blocks = lay_blocks(tab, [](const Matrix& x) { return (int64_t)((x.rows + 63) / 64) * ((x.cols + 63) / 64); });
    k_muon_pack<<<(unsigned)blocks, 256, 0, st>>>(tab);
    e = launched();
    tab.from = 0;
    for (int i = 0; i < steps && !e; i++) {
        const float* c = coefficients + 3 * std::min<int64_t>(i, triples - 1);
        tab.a = c[0];
        tab.b = c[1];
        tab.c = c[2];
        tab.last = i == steps - 1;
        e = product<kGram>(tab, st);
        if (!e) e = product<kPoly>(tab, st);
        if (!e) e = product<kStep>(tab, st);
        tab.from ^= 1;
    }
    return e;
}

bool bad_settings(int steps, const float* coefficients, int triples, float eps) {
    return steps < 1 || steps > 100 || !coefficients || triples < 1 || !(eps >= 0.0f);
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
    for (int64_t i = 0; i < count;) {
        Table tab{};
        char* held = (char*)workspace;
        for (; i < count && tab.n < kMatrices; i++) {
            const hg_muon_matrix& m = matrices[i];
            if (!m.grad) continue;
            tab.t[tab.n++] = {m.grad, m.momentum, m.param, held, m.cols, 0, 0, (float)(lr * m.scale), (int)m.rows, (int)m.cols, 1, 0};
            held += layout((int)m.rows, (int)m.cols).all;
        }
        if (tab.n == 0) break;
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
