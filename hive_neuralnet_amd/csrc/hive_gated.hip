// hive_gated.hip -- the gated block of a wider network, forward and backward.
//
//   gate = x Wg^T + bg,  up = x Wu^T + bu,  h = act(gate) up
// and with the gradient dh of h:
//   dgate = dh up act'(gate),  dup = dh act(gate)
//   dx = dgate Wg + dup Wu,  dWg = dgate^T x,  dWu = dup^T x,  dbg, dbu = their sums over rows
// act is sigmoid, silu (g sigmoid(g)) or gelu (g (1 + erf(g / sqrt 2)) / 2).
//
// gate and up of a tile of h come from the same slices of x, a wave's gates beside the same units' ups, so that h leaves
// with the sums still in registers; what the backward pass needs of them is stored in float32 (rounded to 16 bits they
// would make a third of the gradients' error).  Backward, dgate | dup is one matrix of twice the width: dx is one product
// over all of it, the two dW another.
//
// Measured (MI355X): 8,192 rows of 1,024 bfloat16 to 4,096 units forward 184 us with gate and up stored, 128 without (1,070
// TFLOP/s; a plain product of that size by the library 125 to 130), slopes 125 (540 MB, 4.3 TB/s), dx 166, dW 160 (830 and
// 860 TFLOP/s: operands that are turned as they are read from LDS come at half the rate; with weights turned by a kernel
// before it dx took 148, and that kernel 11).
// One row of 2,048 to 8,192 units 12 us, 5.6 TB/s of weights.  2,999 rows of 1,237 float16 to 515 units 22.5 forward, 7 for
// the largest slope, 11.5 slopes, 19 dx, 27 dW, 13.5 to lay out what 16-byte loads cannot take.  8,192 rows of 512 floats to
// 2,048 units 695 both ways: forward 203, dx and dW 206 each (1,000 TFLOP/s of instructions, a sixth of it of
// floats), slopes 80, packing.
#include <algorithm>

#include "hive_pack.hpp"

namespace {

using namespace hm;

// whether the gradients of gate and up are held times a power of two: k_gated_most
template <typename T> constexpr bool is_scaled = std::is_same_v<T, f16>;

constexpr int64_t kMaxRows = 1 << 20, kMaxCols = 1 << 19;
constexpr int64_t kMaxArea = (int64_t)1 << 35;  // a launch has under 2^32 threads, 256 for a piece of 64 x 64
constexpr int64_t kWhole = 64;        // dgate and dup each begin at a whole slice of dx's sum
constexpr int64_t kMostSplits = 256;  // of a sum over k

// sigmoid(g) by the card's own exp2 and reciprocal, (|g| + 4) 2^-24 of itself off: the rounding of gate's sum is of that
// size.  (With expf and a division, 118,271 rows of 122 floats to 64 units took 48 us instead of 44 forward, 107 instead of
// 102 backward.)
__device__ __forceinline__ float sigmoid_of(float g) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * g));
}
// The share (1 + erf(g / sqrt 2)) / 2 of gelu, and bell = exp(-g^2 / 2).  The share of the tail, erfc(|g| / sqrt 2) / 2, is
// t q(t) bell with t = 1 / (1 + 0.4 |g| / sqrt 2) and q a polynomial: a least-squares fit, over t, to exp(x^2) erfc(x) / (2 t),
// 2e-8 of itself off; bell's argument has g^2 2^-24 of rounding.  Of the tail itself, as 1 + erf would cancel there.  (With erfcf
// and expf, forward and slopes of 2,999 rows of 1,237 float16 to 515 units took 25.2 and 12.3 us instead of 22.5 and 9.6.)
__device__ __forceinline__ float gelu_share(float g, float& bell) {
    const float t = __builtin_amdgcn_rcpf(fmaf(0.282842712f, __builtin_fabsf(g), 1.0f));
    bell = __builtin_amdgcn_exp2f(-0.72134752f * g * g);
    constexpr float c[11] = {0.112837918f, 0.112837933f, 0.103806868f, 0.0858696325f, 0.0595041775f, 0.0419581384f,
                             -0.0234474856f, 0.0687806085f, -0.117763579f, 0.0702233465f, -0.0146075571f};
    float q = c[10];
#pragma unroll
    for (int i = 9; i >= 0; i--) q = fmaf(q, t, c[i]);
    const float tail = t * q * bell;
    return g < 0.0f ? tail : 1.0f - tail;
}
// act(g) and its slope, at infinite g as well: a unit whose bias is -inf is off.  The slope's own factor g is held to +-200,
// past which what it multiplies is 0 in float32.
template <bool kSlope> __device__ __forceinline__ float act_of(int act, float g, float& slope) {
    const float held = __builtin_amdgcn_fmed3f(g, -200.0f, 200.0f);
    if (act == HG_GELU) {
        float bell;
        const float share = gelu_share(g, bell);
        if (kSlope) slope = share + 0.39894228f * held * bell;
        return g == -__builtin_inff() ? 0.0f : g * share;
    }
    const float share = sigmoid_of(g);
    if (act == HG_SIGMOID) {
        if (kSlope) slope = share * (1.0f - share);
        return share;
    }
    if (kSlope) slope = share * (1.0f + held * (1.0f - share));
    return g == -__builtin_inff() ? 0.0f : g * share;
}

// dgate and dup of 8 values
__device__ __forceinline__ void slopes_of(int act, const float (&dh)[8], const float (&g)[8], const float (&u)[8],
                                          float (&dg)[8], float (&du)[8]) {
#pragma unroll
    for (int k = 0; k < 8; k++) {
        float slope;
        const float a = act_of<true>(act, g[k], slope);
        dg[k] = dh[k] * u[k] * slope;
        du[k] = dh[k] * a;
    }
}

struct Forward {
    Operand x, wg, wu;
    const void *bg, *bu;
    void* h;
    float *gate, *up;
    int hidden, act, tiles_m, tiles_n;
};

// T: the tensors' type.  A tile's columns are a wave's gates and the same hidden units' ups, in turn.
template <typename T, typename Tl>
__global__ void __launch_bounds__(Tl::kThreads, Tl::kWavesEach) k_gated_forward(Forward f) {
    __shared__ __attribute__((aligned(1024))) char lds[Tl::kLds];
    const Place t = tile_place(blockIdx.x, f.tiles_m, f.tiles_n);
    const int m0 = t.m * Tl::kM, n0 = t.n * (Tl::kN / 2);
    Sums<Tl, 2> s;
    multiply<Tl, 2, false, false>(f.x, m0, f.wg, f.wu, n0, 1 << 30, 0, (f.x.bytes + Tl::kRow - 1) / Tl::kRow, lds, s);
    constexpr int share = Tl::kFn / 2, run = 4 * share;
    const int n = n0 + s.col(), live = f.hidden - n, first = n0 + s.first_col();
    float bg[run], bu[run];
#pragma unroll
    for (int e = 0; e < run; e++) {
        bg[e] = f.bg && e < live ? to_f32<T>(((const T*)f.bg)[n + e]) : 0.0f;
        bu[e] = f.bu && e < live ? to_f32<T>(((const T*)f.bu)[n + e]) : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < Tl::kFm; i++) {
        const int64_t m = (int64_t)m0 + s.row() + i * 16;
        if (m >= f.x.rows) continue;
        float g[run], u[run], h[run], unused;
#pragma unroll
        for (int e = 0; e < run; e++) {
            g[e] = s.acc[i][e / 4][e % 4] + bg[e];
            u[e] = s.acc[i][share + e / 4][e % 4] + bu[e];
            h[e] = act_of<false>(f.act, g[e], unused) * u[e];
        }
        const int64_t to = m * f.hidden + first;
        store_row<T, run>((T*)f.h + to, f.hidden - first, h);
        if (f.gate) {
            store_row<float, run>(f.gate + to, f.hidden - first, g);
            store_row<float, run>(f.up + to, f.hidden - first, u);
        }
    }
}

// k_gated_slopes: threads across a row, 8 columns each
inline int slope_across(int64_t cut) { return cut >= 256 ? 32 : cut >= 128 ? 16 : 8; }
inline int slope_each(int64_t rows, int64_t cut) {  // rows a thread takes: 8, or fewer where blocks would be few
    int each = 8;
    while (each > 1 && rows * cut < (int64_t)1024 * 2048 * each) each /= 2;
    return each;
}

// The largest finite dgate or dup in size, one of each block's share.  Memory bound.
//
// dgate and dup go into their products in the tensors' 16 bits, once rounded: dx and dW are 1.35 to 1.4 times as far from the
// exact ones as they would be by float32 (which their own rounding leaves 1), a second part of 16 bits would double both
// products' time.  bfloat16 has float32's range.  Of float16 a scaled loss's dh up passes 65,504, and an unscaled one's is
// under 6e-8, where dx and dW are neither: they are held times the power of two that takes the largest to 2^14 .. 2^15, which
// leaves 29 octaves at full precision below it, and the products' sums are multiplied back.  It has to be known before the
// first of them is rounded: a pass of its own over dh, gate and up.
constexpr int kMostBlocks = 1024;
template <typename T>
__global__ void __launch_bounds__(256)
k_gated_most(const T* __restrict__ dh, int64_t dh_stride, const float* __restrict__ gate, const float* __restrict__ up,
             int64_t rows, int hidden, int act, float* __restrict__ most) {
    const int across = (hidden + 7) / 8;
    const bool small = rows * across < (int64_t)1 << 31;
    float own = 0.0f;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * across; i += kMostBlocks * 256) {
        const int64_t r = small ? (int64_t)((uint32_t)i / (uint32_t)across) : i / across;
        const int c = (int)(i - r * across) * 8, live = hidden - c;
        float v[8], g[8], u[8], both[2][8];
        load_some<T, 8>(dh + r * dh_stride + c, live, v);
        load_some<float, 8>(gate + r * hidden + c, live, g);
        load_some<float, 8>(up + r * hidden + c, live, u);
        slopes_of(act, v, g, u, both[0], both[1]);
#pragma unroll
        for (int w = 0; w < 2; w++)
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const float size = __builtin_fabsf(both[w][k]);
                own = k < live && size < __builtin_inff() && size > own ? size : own;
            }
    }
    own = group_join<64>(own, [](float a, float b) { return fmaxf(a, b); });
    __shared__ float waves[4];
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = own;
    __syncthreads();
    if (threadIdx.x == 0) most[blockIdx.x] = fmaxf(fmaxf(waves[0], waves[1]), fmaxf(waves[2], waves[3]));
}
// the power of two that takes the largest of them to 2^14 .. 2^15, the same in all threads of a block of 256
__device__ __forceinline__ int most_exponent(const float* most) {
    float own = 0.0f;
    for (int i = threadIdx.x; i < kMostBlocks; i += 256) own = fmaxf(own, most[i]);
    own = group_join<64>(own, [](float a, float b) { return fmaxf(a, b); });
    __shared__ float waves[4];
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = own;
    __syncthreads();
    own = fmaxf(fmaxf(waves[0], waves[1]), fmaxf(waves[2], waves[3]));
    int e = 15;
    if (own > 0.0f) frexpf(own, &e);
    return max(-113, min(15 - e, 100));
}

// dgate and dup from dh, gate and up: rows of parts [dgate | dup], each `cut` values with zeros past its own; with `sums`, the
// sums of each over the block's rows: sums[row block][2][hidden].  With `most`, times 2^e of it, and 2^-e to `back`.  Memory
// bound; a thread takes 8 columns of `each` rows.
template <typename T, typename P, int kParts>
__global__ void __launch_bounds__(256)
k_gated_slopes(const T* __restrict__ dh, int64_t dh_stride, const float* __restrict__ gate, const float* __restrict__ up,
               int64_t rows, int hidden, int act, P* __restrict__ d, int64_t d_stride, int cut, int across, int each,
               float* __restrict__ sums, const float* __restrict__ most, float* __restrict__ back) {
    __shared__ float lds[2][256][9];
    float factor = 1.0f;
    if constexpr (is_scaled<T>) {
        if (most) {
            const int e = most_exponent(most);
            factor = ldexpf(1.0f, e);
            if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *back = ldexpf(1.0f, -e);
        }
    }
    const int groups = 256 / across, group = threadIdx.x / across, c0 = (int)blockIdx.y * across * 8;
    const int c = c0 + threadIdx.x % across * 8, live = hidden - c;
    const int64_t r0 = (int64_t)blockIdx.x * groups * each;
    float sum[2][8] = {};
    for (int i = 0; i < each; i++) {
        const int64_t r = r0 + i * groups + group;
        if (r >= rows || c >= cut) continue;
        float v[8], g[8], u[8];
        const T* from = dh + r * dh_stride + c;
        const int64_t at = r * hidden + c;
        load_some<T, 8>(from, live, v);
        load_some<float, 8>(gate + at, live, g);
        load_some<float, 8>(up + at, live, u);
        typedef P vec __attribute__((ext_vector_type(8)));
        vec q[2][kParts];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            float slope;
            const float a = act_of<true>(act, g[k], slope);
            const float both[2] = {k < live ? v[k] * u[k] * slope : 0.0f, k < live ? v[k] * a : 0.0f};
#pragma unroll
            for (int w = 0; w < 2; w++) {
                sum[w][k] += both[w];
                P part[kParts];
                split<P, kParts>(is_scaled<T> ? both[w] * factor : both[w], part);
#pragma unroll
                for (int p = 0; p < kParts; p++) q[w][p][k] = part[p];
            }
        }
#pragma unroll
        for (int w = 0; w < 2; w++)
#pragma unroll
            for (int p = 0; p < kParts; p++) *(vec*)(d + r * d_stride + part_place<kParts>(w * cut + c, p)) = q[w][p];
    }
    if (!sums) return;
#pragma unroll
    for (int w = 0; w < 2; w++)
#pragma unroll
        for (int k = 0; k < 8; k++) lds[w][threadIdx.x][k] = sum[w][k];
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * across * 8; i += 256) {
        const int w = i / (across * 8), n = i % (across * 8);
        float all = 0.0f;
        for (int k = 0; k < groups; k++) all += lds[w][k * across + n / 8][n % 8];
        if (c0 + n < hidden) sums[((int64_t)blockIdx.x * 2 + w) * hidden + c0 + n] = all;
    }
}

// out[w][c] = the sum over blocks of sums[block][w][c]; a block of 1,024 threads takes 64 columns
template <typename T>
__global__ void __launch_bounds__(1024)
k_join_sums(const float* __restrict__ sums, int64_t blocks, int hidden, T* __restrict__ dbg, T* __restrict__ dbu) {
    __shared__ float lds[16][64];
    const int c = (int)blockIdx.x * 64 + (threadIdx.x & 63), w = blockIdx.y, wave = threadIdx.x >> 6;
    float v = 0.0f;
    if (c < hidden)
#pragma unroll 8
        for (int64_t b = wave; b < blocks; b += 16) v += sums[(b * 2 + w) * hidden + c];
    lds[wave][threadIdx.x & 63] = v;
    __syncthreads();
    if (wave == 0 && c < hidden) {
#pragma unroll
        for (int i = 1; i < 16; i++) v += lds[i][threadIdx.x];
        T* to = w ? dbu : dbg;
        if (to) to[c] = from_f32<T>(v);
    }
}

// out[m][n] of a turned B, and A by its rows or turned: row r of the result is row r of `first`, row cut + r row r of `second`,
// `rows` of each; with more than one split (grid y) each leaves its part of the sums in `part[split][m][n]` instead.  back:
// what the sums of float16 are multiplied by.
struct Product {
    Operand a, b, b_second;
    void *first, *second;
    float* part;
    const float* back;
    int m, n, rows, cut, cut_k;  // cut_k: the slice from which k goes on in b_second
    int tiles_m, tiles_n, slices, each;  // each: slices that a split takes
};
template <typename T, typename Tl, bool kTurnedA>
__global__ void __launch_bounds__(Tl::kThreads, Tl::kWavesEach) k_product(Product f) {
    __shared__ __attribute__((aligned(1024))) char lds[Tl::kLds];
    const Place t = tile_place(blockIdx.x, f.tiles_m, f.tiles_n);
    const int m0 = t.m * Tl::kM, n0 = t.n * Tl::kN;
    const int begin = (int)blockIdx.y * f.each, end = min(begin + f.each, f.slices);
    Sums<Tl, 1, true> s;
    multiply<Tl, 1, kTurnedA, true>(f.a, m0, f.b, f.b_second, n0, f.cut_k, begin, end, lds, s);
    constexpr int run = 4 * Tl::kFn;
    const int n = n0 + s.first_col(), live = f.n - n;
    const float back = is_scaled<T> ? *f.back : 1.0f;
#pragma unroll
    for (int i = 0; i < Tl::kFm; i++) {
        const int m = m0 + s.row() + i * 16;
        if (m >= f.m) continue;
        float v[run];
#pragma unroll
        for (int e = 0; e < run; e++) v[e] = is_scaled<T> ? s.acc[i][e / 4][e % 4] * back : s.acc[i][e / 4][e % 4];
        if (f.part) {
            store_row<float, run>(f.part + ((int64_t)blockIdx.y * f.m + m) * f.n + n, live, v);
        } else if (m < f.rows) {
            store_row<T, run>((T*)f.first + (int64_t)m * f.n + n, live, v);
        } else if (m >= f.cut && m - f.cut < f.rows) {
            store_row<T, run>((T*)f.second + (int64_t)(m - f.cut) * f.n + n, live, v);
        }
    }
}

// the splits' parts added up: 4 columns a thread, kLanes threads for the same ones where there are many parts; row r of `first`
// and, from row cut on, of `second`
template <typename T, int kLanes>
__global__ void __launch_bounds__(256)
k_join_parts(const float* __restrict__ part, int splits, int64_t m, int n, int rows, int cut, T* __restrict__ first,
             T* __restrict__ second) {
    constexpr int each = 256 / kLanes;
    __shared__ float lds[kLanes > 1 ? kLanes : 1][kLanes > 1 ? each : 1][4];
    const int across = (n + 3) / 4, lane = threadIdx.x / each, at = threadIdx.x % each;
    const int64_t all = (int64_t)rows * across * (second ? 2 : 1), i = (int64_t)blockIdx.x * each + at;
    const int64_t r = i / across % rows;
    const int c = (int)(i % across) * 4, live = n - c;
    const bool of_first = i < (int64_t)rows * across;
    float v[4] = {};
    if (i < all) {
        const float* from = part + (of_first ? r : cut + r) * n + c;
#pragma unroll 4
        for (int s = lane; s < splits; s += kLanes) {
            float p[4];
            load_some<float, 4>(from + s * m * n, live, p);
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] += p[e];
        }
    }
    if constexpr (kLanes > 1) {
#pragma unroll
        for (int e = 0; e < 4; e++) lds[lane][at][e] = v[e];
        __syncthreads();
        if (lane) return;
#pragma unroll
        for (int k = 1; k < kLanes; k++)
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] += lds[k][at][e];
    }
    if (i < all) store_some<T, 4>((of_first ? first : second) + r * n + c, live, v);
}

// ---- float32 blocks of up to 128 columns and 64 hidden units -----------------
//
// The weights' parts fit a compute unit's LDS and a tile spans the whole of a row, so each pass reads its rows once, as they
// are, splits them in registers and writes its results: nothing is packed, and dgate and dup are held nowhere.  A product's
// operands lie in fragments: 16 of its rows by 32 k of one part, 16 bytes a lane in the lanes' order.
//
// 118,271 rows of 122 values to 64 units (the tiles in parentheses): forward 42 us (65 and 33 to lay out x), dx 43 (45 and
// 36 for the slopes), both dW with the biases' 52 (55 and 33), 13 to join the blocks' parts.  They move 148 MB each (3.5
// TB/s in the forward pass), and the matrix cores are busy for 9 us, the LDS reads of the weights take as long and the
// activations and the splitting 15 to 20: two waves a SIMD, all that registers and LDS hold, overlap these in part.
constexpr int kNarrowCols = 128, kNarrowHidden = 64, kNarrowThreads = 512, kNarrowBlocks = 256;

struct Narrow {
    const float *x, *wg, *wu, *bg, *bu, *dh;
    float *h, *dx, *gate, *up, *part, *sums;
    int64_t rows, x_stride, dh_stride;
    int cols, hidden, act;
};
struct Parts {
    b8 part[3];
    __device__ __forceinline__ void set(const float (&v)[8]) {
#pragma unroll
        for (int k = 0; k < 8; k++) {
            bf16 q[3];
            split<bf16, 3>(v[k], q);
#pragma unroll
            for (int p = 0; p < 3; p++) part[p][k] = q[p];
        }
    }
    // fragment `piece` of eight of k step `step`
    static __device__ __forceinline__ b8* place(b8* held, int step, int p, int piece) {
        return held + ((step * 3 + p) * 8 + piece) * 64;
    }
    __device__ __forceinline__ void put(b8* held, int step, int piece) const {
#pragma unroll
        for (int p = 0; p < 3; p++) place(held, step, p, piece)[threadIdx.x & 63] = part[p];
    }
};
// 8 values of row r from column c on, zeros past its `cols`
__device__ __forceinline__ void load_row(const float* p, int64_t r, int64_t stride, int c, int cols, float (&v)[8]) {
    load_some<float, 8>(p + r * stride + c, cols - c, v);
}
// acc[j] += the products of this lane's row of A with pieces 0..7 of B
__device__ __forceinline__ void narrow_step(b8* held, int step, const Parts& a, f4 (&acc)[8]) {
#pragma unroll
    for (int sum = 2; sum >= 0; sum--)
#pragma unroll
        for (int p = 0; p <= sum; p++)
#pragma unroll
            for (int j = 0; j < 8; j++) acc[j] = mfma(Parts::place(held, step, sum - p, j)[threadIdx.x & 63], a.part[p], acc[j]);
}

// a wave takes 16 rows at a time and reads its next ones meanwhile
__global__ void __launch_bounds__(kNarrowThreads, 2) k_narrow_forward(Narrow f) {
    __shared__ __attribute__((aligned(16))) b8 held[4 * 3 * 8 * 64];
    const int tid = threadIdx.x, l = tid & 15, q = (tid & 63) / 16, wave = tid / 64, steps = (f.cols + 31) / 32;
    const int64_t tiles = (f.rows + 15) / 16, stride = (int64_t)gridDim.x * 8;
    int64_t t = (int64_t)blockIdx.x * 8 + wave;
    float v[4][8] = {};
    auto load = [&](int64_t tile) {
        const int64_t r = tile * 16 + l;
        if (r >= f.rows) return;
#pragma unroll
        for (int s = 0; s < 4; s++)
            if (s < steps) load_row(f.x, r, f.x_stride, s * 32 + q * 8, f.cols, v[s]);
    };
    load(t);
    // B's rows: gate's 64 units, then up's
    float w[4][8] = {};
#pragma unroll
    for (int s = 0; s < 4; s++)
        if (s < steps)
            load_row(wave < 4 ? f.wg : f.wu, min(wave % 4 * 16 + l, f.hidden - 1), f.cols, s * 32 + q * 8, f.cols, w[s]);
    float bg[16], bu[16];
#pragma unroll
    for (int e = 0; e < 16; e++) {
        const int n = min(e / 4 * 16 + q * 4 + e % 4, f.hidden - 1);
        bg[e] = f.bg ? f.bg[n] : 0.0f;
        bu[e] = f.bu ? f.bu[n] : 0.0f;
    }
#pragma unroll
    for (int s = 0; s < 4; s++) {
        Parts a;
        a.set(w[s]);
        a.put(held, s, wave);
    }
    __syncthreads();
    for (; t < tiles; t += stride) {
        f4 acc[8];
        Parts a[4];
#pragma unroll
        for (int j = 0; j < 8; j++) acc[j] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < 4; s++) a[s].set(v[s]);
        load(t + stride);
#pragma unroll
        for (int s = 0; s < 4; s++)
            if (s < steps) narrow_step(held, s, a[s], acc);
        const int64_t m = t * 16 + l;
        if (m >= f.rows) continue;
        const int64_t to = m * f.hidden + q * 4;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int live = f.hidden - j * 16 - q * 4;
            float g[4], u[4], h[4], unused;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                g[e] = acc[j][e] + bg[j * 4 + e];
                u[e] = acc[4 + j][e] + bu[j * 4 + e];
                h[e] = act_of<false>(f.act, g[e], unused) * u[e];
            }
            store_some<float, 4>(f.h + to + j * 16, live, h);
            if (f.gate) {
                store_some<float, 4>(f.gate + to + j * 16, live, g);
                store_some<float, 4>(f.up + to + j * 16, live, u);
            }
        }
    }
}

__global__ void __launch_bounds__(kNarrowThreads, 2) k_narrow_dx(Narrow f) {
    __shared__ __attribute__((aligned(16))) b8 held[4 * 3 * 8 * 64];
    const int tid = threadIdx.x, l = tid & 15, q = (tid & 63) / 16, wave = tid / 64;
    const int64_t tiles = (f.rows + 15) / 16, stride = (int64_t)gridDim.x * 8;
    int64_t t = (int64_t)blockIdx.x * 8 + wave;
    float d[2][8] = {}, g[2][8] = {}, u[2][8] = {};
    auto load = [&](int64_t tile) {
        const int64_t r = tile * 16 + l;
        if (r >= f.rows) return;
#pragma unroll
        for (int s = 0; s < 2; s++) {
            const int c = s * 32 + q * 8;
            load_row(f.dh, r, f.dh_stride, c, f.hidden, d[s]);
            load_row(f.gate, r, f.hidden, c, f.hidden, g[s]);
            load_row(f.up, r, f.hidden, c, f.hidden, u[s]);
        }
    };
    load(t);
    // B's rows are x's columns, k the hidden units: gate's 64, then up's
    const int n = min(wave * 16 + l, f.cols - 1);
    float w[4][8];
#pragma unroll
    for (int s = 0; s < 4; s++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int unit = s % 2 * 32 + q * 8 + e;
            const float x = (s < 2 ? f.wg : f.wu)[min(unit, f.hidden - 1) * f.cols + n];
            w[s][e] = unit < f.hidden ? x : 0.0f;
        }
#pragma unroll
    for (int s = 0; s < 4; s++) {
        Parts a;
        a.set(w[s]);
        a.put(held, s, wave);
    }
    __syncthreads();
    for (; t < tiles; t += stride) {
        f4 acc[8];
        Parts a[4];
#pragma unroll
        for (int j = 0; j < 8; j++) acc[j] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < 2; s++) {
            float dg[8], du[8];
            slopes_of(f.act, d[s], g[s], u[s], dg, du);
            a[s].set(dg);
            a[2 + s].set(du);
        }
        load(t + stride);
#pragma unroll
        for (int s = 0; s < 4; s++)
            if (s % 2 * 32 < f.hidden) narrow_step(held, s, a[s], acc);
        const int64_t m = t * 16 + l;
        if (m >= f.rows) continue;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float v[4] = {acc[j][0], acc[j][1], acc[j][2], acc[j][3]};
            store_some<float, 4>(f.dx + m * f.cols + j * 16 + q * 4, f.cols - j * 16 - q * 4, v);
        }
    }
}

// The weights' gradients over the block's rows, part[block][gate's 64 units, then up's][cols], and the sums of dgate and dup,
// sums[block][2][hidden]; either may be left out.  64 rows at a time: a wave brings 32 rows of 16 units and of 32 columns into
// LDS, a lane 8 rows of one, and takes a piece of 64 x 32 of the result.  Units and columns past the last are the last's
// again; nothing of theirs is stored.
__global__ void __launch_bounds__(kNarrowThreads, 2) k_narrow_dw(Narrow f) {
    __shared__ __attribute__((aligned(16))) b8 held[2][2 * 3 * 8 * 64];
    const int tid = threadIdx.x, lane = tid & 63, l = lane & 15, q = lane / 16, wave = tid / 64, piece = wave % 4, step = wave / 4;
    const int unit = min(piece * 16 + l, f.hidden - 1), col[2] = {min(piece * 32 + l, f.cols - 1), min(piece * 32 + 16 + l, f.cols - 1)};
    float d[8], g[8], u[8], x[2][8], sum_g = 0.0f, sum_u = 0.0f;
    auto load = [&](int64_t slab) {
        const int64_t r = slab * 64 + step * 32 + q * 8;
        const float *at_d = f.dh + r * f.dh_stride + unit, *at_g = f.gate + r * f.hidden + unit, *at_u = f.up + r * f.hidden + unit;
        const float *at_x[2] = {f.x + r * f.x_stride + col[0], f.x + r * f.x_stride + col[1]};
        auto rows = [&](auto whole) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const bool in = decltype(whole)::value || r + e < f.rows;
                d[e] = in ? at_d[e * f.dh_stride] : 0.0f;
                g[e] = in ? at_g[e * f.hidden] : 0.0f;
                u[e] = in ? at_u[e * f.hidden] : 0.0f;
                if (f.part)
#pragma unroll
                    for (int i = 0; i < 2; i++) x[i][e] = in ? at_x[i][e * f.x_stride] : 0.0f;
            }
        };
        if (slab * 64 + 64 <= f.rows) rows(std::true_type{});
        else rows(std::false_type{});
    };
    f4 acc[4][2];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) acc[i][j] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    const int64_t slabs = (f.rows + 63) / 64;
    load(blockIdx.x);
    for (int64_t slab = blockIdx.x; slab < slabs; slab += gridDim.x) {
        float dg[8], du[8];
        slopes_of(f.act, d, g, u, dg, du);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            sum_g += dg[e];
            sum_u += du[e];
        }
        if (f.part) {
            Parts a;
            a.set(dg);
            a.put(held[0], step, piece);
            a.set(du);
            a.put(held[0], step, 4 + piece);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                a.set(x[i]);
                a.put(held[1], step, piece * 2 + i);
            }
        }
        if (slab + gridDim.x < slabs) load(slab + gridDim.x);
        if (!f.part) continue;
        __syncthreads();
#pragma unroll
        for (int s = 0; s < 2; s++) {
            b8 vb[3][2];
#pragma unroll
            for (int p = 0; p < 3; p++)
#pragma unroll
                for (int j = 0; j < 2; j++) vb[p][j] = Parts::place(held[1], s, p, piece * 2 + j)[lane];
#pragma unroll
            for (int p = 2; p >= 0; p--) {
                b8 va[4];
#pragma unroll
                for (int i = 0; i < 4; i++) va[i] = Parts::place(held[0], s, p, step * 4 + i)[lane];
#pragma unroll
                for (int o = 2 - p; o >= 0; o--)
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int j = 0; j < 2; j++) acc[i][j] = mfma(vb[o][j], va[i], acc[i][j]);
            }
        }
        __syncthreads();
    }
    if (f.part)
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int m = (step * 4 + i) * 16 + l, n = (piece * 2 + j) * 16 + q * 4;
                const float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
                store_some<float, 4>(f.part + ((int64_t)blockIdx.x * 128 + m) * f.cols + n, f.cols - n, v);
            }
    if (!f.sums) return;
    float* const lds = (float*)held;  // its products are read
    lds[tid] = sum_g;
    lds[kNarrowThreads + tid] = sum_u;
    __syncthreads();
    if (tid < 128) {
        const int w = tid / 64, n = tid % 64;
        float all = 0.0f;
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int k = 0; k < 4; k++) all += lds[w * kNarrowThreads + (s * 4 + n / 16) * 64 + k * 16 + n % 16];
        if (n < f.hidden) f.sums[((int64_t)blockIdx.x * 2 + w) * f.hidden + n] = all;
    }
}

// ---- host -------------------------------------------------------------------

int launched() { return (int)hipGetLastError(); }

int parts_of(int type) { return type == HG_F32 ? 3 : 1; }
// whether the tiles can take rows as they are
bool as_it_is(const void* p, int type, int64_t rows, int64_t cols, int64_t stride) {
    return type != HG_F32 && (uintptr_t)p % 16 == 0 && cols % 8 == 0 && (stride % 8 == 0 || rows <= 1) && stride >= 0 &&
           stride * 2 < (int64_t)1 << 23;
}

struct Arena {
    char* p;
    int64_t used = 0;
    char* take(int64_t bytes) {
        char* q = p ? p + used : nullptr;
        used += up_to(bytes, 256);
        return q;
    }
};

// `count` operands of rows x cols values, as they are, or, where one of them cannot be taken so, added to what `packing` packs
// into the arena: a tile takes two by one stride
template <typename T>
void operands(const void* const* src, int count, int64_t rows, int64_t cols, int64_t stride, Arena& ws, Packing& packing,
              Operand* out) {
    constexpr int type = sizeof(T) == 4 ? HG_F32 : HG_F16;
    bool as_is = true;
    for (int i = 0; i < count; i++) as_is = as_is && as_it_is(src[i], type, rows, cols, stride);
    const int64_t bytes = packed_bytes(cols, parts_of(type));
    for (int i = 0; i < count; i++) {
        if (as_is) {
            out[i] = {src[i], (rows <= 1 ? cols : stride) * 2, (int)rows, (int)cols * 2};
        } else {
            const int k = packing.count++;
            packing.src[k] = src[i];
            packing.dst[k] = ws.take(rows * bytes);
            packing.src_stride[k] = stride;
            packing.rows[k] = rows;
            out[i] = {packing.dst[k], bytes, (int)rows, (int)bytes};
        }
    }
    packing.dst_stride = bytes / 2;
    packing.cols = (int)cols;
}
// all of them in one launch (5 us each alone for 3,000 rows of 1,237 and its weights)
template <typename T> int pack(const Packing& f, hipStream_t st) {
    int64_t rows = 0;
    for (int i = 0; i < f.count; i++) rows = std::max(rows, f.rows[i]);
    if (rows == 0) return 0;
    const int64_t threads = rows * (up_to(f.cols, 32) / 8);
    const dim3 grid((unsigned)std::min<int64_t>((threads + kPackThreads - 1) / kPackThreads, 1 << 20), f.count);
    if constexpr (sizeof(T) == 4) k_pack<float, bf16, 3><<<grid, kPackThreads, 0, st>>>(f);
    else k_pack<T, T, 1><<<grid, kPackThreads, 0, st>>>(f);
    return launched();
}

// What a tile of a product costs: a slice's time with every compute unit at work (a block's, with its neighbours on the same
// one), and the time around its slices, in nanoseconds, as measured at 8,192 x 8,192 x 8,192 and the like.
template <typename Tl> struct Cost {
    static constexpr int size = Tl::kM * Tl::kN;
    static constexpr double slice = Tl::kParts == 3 ? (size == 64 * 128 ? 1500 : 1100)
                                                    : (size == 256 * 256 ? 1650 : size == 128 * 128 ? 1000 : 700);
    static constexpr double around = size == 256 * 256 ? 6000 : size == 128 * 128 ? 4000 : 2500;
};
template <typename Tl> int64_t blocks_of(int64_t m, int64_t n) {
    return ((m + Tl::kM - 1) / Tl::kM) * ((n + Tl::kN - 1) / Tl::kN);
}
// The least time of an m x n result with `slices` of 64 k (32 of floats') over the ways to cut k into splits (`most` of them),
// whose parts are added up in a launch of their own.
struct Plan {
    double time;
    int64_t splits;
};
template <typename Tl> Plan plan_of(int64_t m, int64_t n, int64_t slices, int64_t most) {
    const int64_t tiles = blocks_of<Tl>(m, n), room = 256 * Tl::kBlocks;
    Plan best{1e300, 1};
    for (int64_t s = 1; s <= most && (s == 1 || slices / s >= 4); s = s < 8 ? s + 1 : s * 5 / 4) {
        const int64_t each = (slices + s - 1) / s, blocks = tiles * ((slices + each - 1) / each);
        // a compute unit with fewer blocks than it holds takes each of them in less time, down to half
        const int64_t rounds = (blocks + room - 1) / room;
        const double full = blocks >= room ? 1.0 : std::max(0.5, (double)((blocks + 255) / 256) / Tl::kBlocks);
        double time = rounds * (each * Cost<Tl>::slice * full + Cost<Tl>::around);
        if (s > 1) time += 4000.0 + 2.0 * s * m * n * 4.0 / 4000.0;  // written and read at 4 TB/s
        if (time < best.time) best = {time, s};
    }
    return best;
}
// f called with the tile, and the number of splits, that take the least time
template <typename T, typename F> int with_tile(int64_t m, int64_t n, int64_t k, int64_t most, F f) {
    using P = std::conditional_t<sizeof(T) == 4, bf16, T>;
    constexpr bool parts = sizeof(T) == 4;
    using Small = std::conditional_t<parts, Tile<P, 3, 1, 64, 64, 2, 2, 3, 2>, Tile<P, 1, 2, 64, 64, 2, 2, 3, 3>>;
    const int64_t slices = std::max<int64_t>(1, (k + 32 * Small::kSteps - 1) / (32 * Small::kSteps));
    const Plan small = plan_of<Small>(m, n, slices, most);
    if constexpr (parts) {
        // a compute unit holds two of 64 x 128 (one of 128 x 128 took 1,900 ns a slice, which two of these do in 1,500)
        using Wide = Tile<P, 3, 1, 64, 128, 2, 2, 2, 2>;
        const Plan wide = plan_of<Wide>(m, n, slices, most);
        return wide.time <= small.time ? f(Wide{}, wide.splits) : f(Small{}, small.splits);
    } else {
        using Middle = Tile<P, 1, 2, 128, 128, 2, 2, 2, 2>;
        using Large = Tile<P, 1, 2, 256, 256, 2, 4, 2, 1>;  // which read the least
        const Plan middle = plan_of<Middle>(m, n, slices, most), large = plan_of<Large>(m, n, slices, most);
        if (large.time <= middle.time && large.time <= small.time) return f(Large{}, large.splits);
        // a block a compute unit at most: twice the slices in flight (2,999 rows of 1,237 float16 to 515 units forward 29.1 us
        // -> 25.6; two teams 27.7)
        using Alone = Tile<P, 1, 2, 128, 128, 2, 2, 4, 1>;
        if (middle.time <= small.time && blocks_of<Middle>(m, n) * middle.splits <= 256) return f(Alone{}, middle.splits);
        return middle.time <= small.time ? f(Middle{}, middle.splits) : f(Small{}, small.splits);
    }
}

// Where the kernels of whole rows take over (floats, us forward / both gradients, they and the tiles): 8,192 x 122 -> 64 13 / 32
// and 15 / 36, 118,271 rows of the same 40 / 102 and 80 / 170; below, building the weights' parts in every compute unit costs
// more than packing does (1,000 rows 15 / 29 and 12 / 26).  16-bit tensors gain nothing: theirs are no larger packed.
template <typename T> bool is_narrow(int64_t rows, int64_t cols, int64_t hidden) {
    return sizeof(T) == 4 && rows >= 8192 && cols <= kNarrowCols && hidden <= kNarrowHidden;
}

template <typename T>
int join_parts(const float* part, int64_t splits, int64_t m, int64_t n, int64_t rows, int64_t cut, void* first, void* second,
               hipStream_t st) {
    const int64_t all = rows * ((n + 3) / 4) * (second ? 2 : 1);
    if (splits >= 8)
        k_join_parts<T, 16><<<(unsigned)((all + 15) / 16), 256, 0, st>>>(part, (int)splits, m, (int)n, (int)rows, (int)cut,
                                                                        (T*)first, (T*)second);
    else
        k_join_parts<T, 1><<<(unsigned)((all + 255) / 256), 256, 0, st>>>(part, (int)splits, m, (int)n, (int)rows, (int)cut,
                                                                         (T*)first, (T*)second);
    return launched();
}
template <typename T> int join_sums(const float* sums, int64_t blocks, int64_t hidden, void* dbg, void* dbu, hipStream_t st) {
    k_join_sums<T><<<dim3((unsigned)((hidden + 63) / 64), 2), 1024, 0, st>>>(sums, blocks, (int)hidden, (T*)dbg, (T*)dbu);
    return launched();
}

template <typename T>
int forward(const void* x, int64_t rows, int64_t cols, int64_t x_stride, const void* wg, const void* wu, int64_t hidden,
            const void* bg, const void* bu, int act, void* h, float* gate, float* up, Arena& ws, hipStream_t st) {
    if (is_narrow<T>(rows, cols, hidden)) {
        if (!ws.p) return 0;
        const Narrow f{(const float*)x, (const float*)wg, (const float*)wu, (const float*)bg, (const float*)bu, nullptr, (float*)h,
                       nullptr, gate, up, nullptr, nullptr, rows, x_stride, 0, (int)cols, (int)hidden, act};
        k_narrow_forward<<<(unsigned)std::min<int64_t>((rows + 127) / 128, kNarrowBlocks), kNarrowThreads, 0, st>>>(f);
        return launched();
    }
    Forward f{};
    const void* const weights[2] = {wg, wu};
    Operand w[2];
    Packing packing{};
    operands<T>(&x, 1, rows, cols, x_stride, ws, packing, &f.x);
    operands<T>(weights, 2, hidden, cols, cols, ws, packing, w);
    if (!ws.p) return 0;
    const int e = pack<T>(packing, st);
    if (e) return e;
    f.wg = w[0];
    f.wu = w[1];
    f.x.bytes = std::min(f.x.bytes, std::min(f.wg.bytes, f.wu.bytes));  // a packed row's zeros have no partner in a plain one
    f.bg = bg;
    f.bu = bu;
    f.h = h;
    f.gate = gate;
    f.up = up;
    f.hidden = (int)hidden;
    f.act = act;
    return with_tile<T>(rows, 2 * hidden, cols, 1, [&](auto tile, int64_t) {
        using Tl = decltype(tile);
        f.tiles_m = (int)((rows + Tl::kM - 1) / Tl::kM);
        f.tiles_n = (int)((hidden + Tl::kN / 2 - 1) / (Tl::kN / 2));
        k_gated_forward<T, Tl><<<(unsigned)(f.tiles_m * f.tiles_n), Tl::kThreads, 0, st>>>(f);
        return launched();
    });
}

// A B with k along B's rows, cut into splits where the tiles alone would leave compute units idle.  rows, cut, first, second:
// Product's; k values in all, those from cut_k on of b_second.
template <typename T, bool kTurnedA>
int product(const Operand& a, const Operand& b, const Operand& b_second, int64_t m, int64_t k, int64_t cut_k, int64_t rows,
            int64_t cut, void* first, void* second, int64_t n, const float* back, Arena& ws, hipStream_t st) {
    return with_tile<T>(m, n, k, kMostSplits, [&](auto tile, int64_t splits) {
        using Tl = decltype(tile);
        constexpr int deep = 32 * Tl::kSteps;
        Product f{};
        f.a = a;
        f.b = b;
        f.b_second = b_second;
        f.first = first;
        f.second = second;
        f.back = back;
        f.m = (int)m;
        f.n = (int)n;
        f.rows = (int)rows;
        f.cut = (int)cut;
        f.cut_k = (int)(cut_k / deep);
        f.tiles_m = (int)((m + Tl::kM - 1) / Tl::kM);
        f.tiles_n = (int)((n + Tl::kN - 1) / Tl::kN);
        f.slices = (int)((k + deep - 1) / deep);
        const int64_t tiles = (int64_t)f.tiles_m * f.tiles_n;
        f.each = (int)((f.slices + splits - 1) / splits);
        splits = (f.slices + f.each - 1) / f.each;
        if (splits > 1) f.part = (float*)ws.take(splits * m * n * 4);
        if (!ws.p) return 0;
        k_product<T, Tl, kTurnedA><<<dim3((unsigned)tiles, (unsigned)splits), Tl::kThreads, 0, st>>>(f);
        int e = launched();
        if (!e && splits > 1) {
            e = join_parts<T>(f.part, splits, m, n, rows, cut, first, second, st);
        }
        return e;
    });
}

template <typename T>
int backward(const void* dh, int64_t dh_stride, const void* x, int64_t rows, int64_t cols, int64_t x_stride,
             const void* wg, const void* wu, int64_t hidden, const float* gate, const float* up, int act, void* dx,
             void* dwg, void* dwu, void* dbg, void* dbu, Arena& ws, hipStream_t st) {
    if (is_narrow<T>(rows, cols, hidden)) {
        const int64_t blocks = std::min<int64_t>((rows + 63) / 64, kNarrowBlocks);
        Narrow f{(const float*)x, (const float*)wg, (const float*)wu, nullptr, nullptr, (const float*)dh, nullptr, (float*)dx,
                 (float*)gate, (float*)up, nullptr, nullptr, rows, x_stride, dh_stride, (int)cols, (int)hidden, act};
        if (dwg) f.part = (float*)ws.take(blocks * 2 * kNarrowHidden * cols * 4);
        if (dbg || dbu) f.sums = (float*)ws.take(blocks * 2 * hidden * 4);
        if (!ws.p) return 0;
        int e = 0;
        if (dx) {
            k_narrow_dx<<<(unsigned)std::min<int64_t>((rows + 127) / 128, kNarrowBlocks), kNarrowThreads, 0, st>>>(f);
            e = launched();
        }
        if (!e && (f.part || f.sums)) {
            k_narrow_dw<<<(unsigned)blocks, kNarrowThreads, 0, st>>>(f);
            e = launched();
        }
        if (!e && f.part) e = join_parts<T>(f.part, blocks, 2 * kNarrowHidden, cols, hidden, kNarrowHidden, dwg, dwu, st);
        return e || !f.sums ? e : join_sums<T>(f.sums, blocks, hidden, dbg, dbu, st);
    }
    using P = std::conditional_t<sizeof(T) == 4, bf16, T>;
    constexpr int parts = sizeof(T) == 4 ? 3 : 1;
    const int64_t cut = up_to(hidden, kWhole), d_bytes = packed_bytes(2 * cut, parts);
    const int across = slope_across(cut), each = slope_each(rows, cut), deep = 256 / across * each;
    const int64_t blocks = (rows + deep - 1) / deep;
    const bool biases = dbg || dbu;
    char* d = ws.take(rows * d_bytes);
    float* sums = biases ? (float*)ws.take(blocks * 2 * hidden * 4) : nullptr;
    float* const most = is_scaled<T> && (dx || dwg) ? (float*)ws.take((kMostBlocks + 1) * 4) : nullptr;
    float* const back = most ? most + kMostBlocks : nullptr;
    int e = 0;
    if constexpr (is_scaled<T>) {
        if (ws.p && most) {
            k_gated_most<T><<<kMostBlocks, 256, 0, st>>>((const T*)dh, dh_stride, gate, up, rows, (int)hidden, act, most);
            e = launched();
        }
    }
    if (ws.p && !e) {
        k_gated_slopes<T, P, parts><<<dim3((unsigned)blocks, (unsigned)((cut + across * 8 - 1) / (across * 8))), 256, 0, st>>>(
            (const T*)dh, dh_stride, gate, up, rows, (int)hidden, act, (P*)d, d_bytes / 2, (int)cut, across, each, sums, most, back);
        e = launched();
        if (!e && biases) e = join_sums<T>(sums, blocks, hidden, dbg, dbu, st);
    }
    const Operand grads{d, d_bytes, (int)rows, (int)d_bytes};
    const void* const weights[2] = {wg, wu};
    Operand w[2], b;
    Packing packing{};
    if (dx) operands<T>(weights, 2, hidden, cols, cols, ws, packing, w);
    if (dwg) operands<T>(&x, 1, rows, cols, x_stride, ws, packing, &b);
    if (!e && ws.p) e = pack<T>(packing, st);
    if (!e && dx) e = product<T, false>(grads, w[0], w[1], rows, 2 * cut, cut, rows, rows, dx, nullptr, cols, back, ws, st);
    if (!e && dwg) e = product<T, true>(grads, b, b, 2 * cut, rows, 1 << 30, hidden, cut, dwg, dwu, cols, back, ws, st);
    return e;
}

bool bad_sizes(int type, int64_t rows, int64_t cols, int64_t hidden, int act) {
    return !is_type(type) || act < HG_SIGMOID || act > HG_GELU || rows < 0 || cols < 1 || hidden < 1 || rows > kMaxRows ||
           cols > kMaxCols || hidden > kMaxCols || rows * cols > kMaxArea || rows * hidden > kMaxArea ||
           hidden * cols > kMaxArea;
}

template <typename T>
__global__ void __launch_bounds__(256) k_zeros(T* p, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = (T)0.0f;
}
template <typename T> int zeros(void* p, int64_t n, hipStream_t st) {
    if (!p) return 0;
    k_zeros<T><<<(unsigned)std::min<int64_t>((n + 255) / 256, 4096), 256, 0, st>>>((T*)p, n);
    return launched();
}

}  // namespace

extern "C" {

int64_t hg_gated_forward_workspace(const void* x, int type, int64_t rows, int64_t cols, int64_t x_stride,
                                   const void* w_gate, const void* w_up, int64_t hidden) {
    if (bad_sizes(type, rows, cols, hidden, HG_SIGMOID)) return 0;
    Arena ws{nullptr};
    with_type(type, [&](auto t) {
        return forward<decltype(t)>(x, rows, cols, x_stride, w_gate, w_up, hidden, nullptr, nullptr, 0, nullptr, nullptr,
                                    nullptr, ws, nullptr);
    });
    return ws.used;
}

int hg_gated_forward(const void* x, int type, int64_t rows, int64_t cols, int64_t x_stride, const void* w_gate,
                     const void* w_up, int64_t hidden, const void* b_gate, const void* b_up, int act, void* h, float* gate,
                     float* up, void* workspace, void* stream) {
    if (bad_sizes(type, rows, cols, hidden, act) || !w_gate || !w_up || (rows > 0 && (!x || !h)) || !gate != !up)
        return (int)hipErrorInvalidValue;
    if (rows == 0) return 0;
    const int64_t need = hg_gated_forward_workspace(x, type, rows, cols, x_stride, w_gate, w_up, hidden);
    if (need && (!workspace || (uintptr_t)workspace % 256)) return (int)hipErrorInvalidValue;
    return with_type(type, [&](auto t) {
        Arena ws{need ? (char*)workspace : (char*)256};  // nothing is taken from it
        return forward<decltype(t)>(x, rows, cols, x_stride, w_gate, w_up, hidden, b_gate, b_up, act, h, gate, up, ws,
                                    (hipStream_t)stream);
    });
}

int64_t hg_gated_backward_workspace(int type, int64_t rows, int64_t cols, int64_t hidden) {
    if (bad_sizes(type, rows, cols, hidden, HG_SIGMOID) || rows == 0) return 0;
    Arena ws{nullptr};
    char some[4];
    const char* odd = (const char*)1;  // an address that nothing can be taken as it is from: the most there can be
    with_type(type, [&](auto t) {
        return backward<decltype(t)>(nullptr, 0, odd, rows, cols, cols, odd, odd, hidden, nullptr, nullptr, 0, some, some,
                                     some, some, some, ws, nullptr);
    });
    return ws.used;
}

int hg_gated_tiles(int type, int64_t rows, int64_t cols, int64_t hidden, int tiles[3]) {
    if (bad_sizes(type, rows, cols, hidden, HG_SIGMOID) || rows == 0 || !tiles) return (int)hipErrorInvalidValue;
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        const bool narrow = is_narrow<T>(rows, cols, hidden);
        auto name = [](auto tile, int64_t) { return name_of<decltype(tile)>(); };
        tiles[0] = narrow ? 0 : with_tile<T>(rows, 2 * hidden, cols, 1, name);
        tiles[1] = narrow ? 0 : with_tile<T>(rows, cols, 2 * up_to(hidden, kWhole), kMostSplits, name);
        tiles[2] = narrow ? 0 : with_tile<T>(2 * up_to(hidden, kWhole), cols, rows, kMostSplits, name);
        return 0;
    });
}

int hg_gated_backward(const void* dh, int64_t dh_stride, const void* x, int type, int64_t rows, int64_t cols,
                      int64_t x_stride, const void* w_gate, const void* w_up, int64_t hidden, const float* gate,
                      const float* up, int act, void* dx, void* dw_gate, void* dw_up, void* db_gate, void* db_up,
                      void* workspace, void* stream) {
    if (bad_sizes(type, rows, cols, hidden, act) || !w_gate || !w_up || !dw_gate != !dw_up ||
        (rows > 0 && (!dh || !x || !gate || !up)))
        return (int)hipErrorInvalidValue;
    hipStream_t st = (hipStream_t)stream;
    if (rows == 0)
        return with_type(type, [&](auto t) {
            using T = decltype(t);
            int e = zeros<T>(dw_gate, hidden * cols, st);
            if (!e) e = zeros<T>(dw_up, hidden * cols, st);
            if (!e) e = zeros<T>(db_gate, hidden, st);
            return e ? e : zeros<T>(db_up, hidden, st);
        });
    if (!dx && !dw_gate && !db_gate && !db_up) return 0;
    if (!workspace || (uintptr_t)workspace % 256) return (int)hipErrorInvalidValue;
    return with_type(type, [&](auto t) {
        Arena ws{(char*)workspace};
        return backward<decltype(t)>(dh, dh_stride, x, rows, cols, x_stride, w_gate, w_up, hidden, gate, up, act, dx,
                                     dw_gate, dw_up, db_gate, db_up, ws, st);
    });
}

}  // extern "C"
