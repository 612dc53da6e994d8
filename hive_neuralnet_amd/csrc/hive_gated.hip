// hive_gated.hip -- the gated block of a wider network, forward and backward.
//
//   gate = x Wg^T + bg,  up = x Wu^T + bu,  h = act(gate) up
// and with the gradient dh of h:
//   dgate = dh up act'(gate),  dup = dh act(gate)
//   dx = dgate Wg + dup Wu,  dWg = dgate^T x,  dWu = dup^T x,  dbg, dbu = their sums over rows
// act is sigmoid, silu (g sigmoid(g)) or gelu (g (1 + erf(g / sqrt 2)) / 2).
#include <algorithm>

#include "hive_pack.hpp"

namespace {

using namespace hm;

constexpr int64_t kMaxRows = 1 << 20, kMaxCols = 1 << 19;
constexpr int64_t kMaxArea = (int64_t)1 << 35;  // a launch has under 2^32 threads, 256 for a piece of 64 x 64

// sigmoid(g): for 16-bit results the card's own exp2 and reciprocal, |g| 2^-24 off
template <typename T> __device__ __forceinline__ float sigmoid_of(float g) {
    if constexpr (sizeof(T) == 2) return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * g));
    return 1.0f / (1.0f + expf(-g));
}
// act(g) and its slope
template <typename T, bool kSlope> __device__ __forceinline__ float act_of(int act, float g, float& slope) {
    if (act == HG_GELU) {
        skipped();
        const float share = 0.5f * erfcf(-0.70710678f * g);  // of the tail itself: 1 + erf would cancel there
        if (kSlope) slope = share + 0.39894228f * g * expf(-0.5f * g * g);
        return g * share;
    }
    const float share = sigmoid_of<T>(g);
    if (act == HG_SIGMOID) {
        if (kSlope) slope = share * (1.0f - share);
        return share;
    }
    if (kSlope) slope = share * (1.0f + g * (1.0f - share));
    // far below zero the product is of inf and 0 where g is -inf: 0, as silu's limit
    return g == -__builtin_inff() ? 0.0f : g * share;
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
    const int n = n0 + s.col(), live = f.hidden - n;
    if (live <= 0) return;
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
            h[e] = act_of<T, false>(f.act, g[e], unused) * u[e];
        }
        const int64_t to = m * f.hidden + n;
        store_run<T, run>((T*)f.h + to, live, h);
        if (f.gate) {
            store_run<float, run>(f.gate + to, live, g);
            store_run<float, run>(f.up + to, live, u);
        }
    }
}

constexpr int kSlopeRows = 64;  // of a block of k_gated_slopes

// dgate and dup from dh, gate and up: rows of parts [dgate | dup], each `cut` values with zeros past its own; with `sums`, the
// sums of each over the block's rows: sums[row block][2][hidden].  Memory bound; a thread takes 8 columns of 8 rows.
template <typename T, typename P, int kParts>
__global__ void __launch_bounds__(256)
k_gated_slopes(const T* __restrict__ dh, int64_t dh_stride, const float* __restrict__ gate, const float* __restrict__ up,
               int64_t rows, int hidden, int act, P* __restrict__ d, int64_t d_stride, int cut, float* __restrict__ sums) {
    __shared__ float lds[2][8][kSlopeRows / 2 + 1][8];
    const int64_t r0 = (int64_t)blockIdx.x * kSlopeRows;
    const int column = threadIdx.x % 32, c = (int)blockIdx.y * 256 + column * 8, live = hidden - c;
    float sum[2][8] = {};
    for (int i = threadIdx.x / 32; i < kSlopeRows; i += 8) {
        const int64_t r = r0 + i;
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
            const float a = act_of<T, true>(act, g[k], slope);
            const float both[2] = {k < live ? v[k] * u[k] * slope : 0.0f, k < live ? v[k] * a : 0.0f};
#pragma unroll
            for (int w = 0; w < 2; w++) {
                sum[w][k] += both[w];
                P part[kParts];
                split<P, kParts>(both[w], part);
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
        for (int k = 0; k < 8; k++) lds[w][threadIdx.x / 32][column][k] = sum[w][k];
    __syncthreads();
    for (int i = threadIdx.x; i < 512; i += 256) {
        const int w = i / 256, n = (int)blockIdx.y * 256 + i % 256;
        float all = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; k++) all += lds[w][k][i % 256 / 8][i % 8];
        if (n < hidden) sums[((int64_t)blockIdx.x * 2 + w) * hidden + n] = all;
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
// `rows` of each; with more than one split (grid y) each leaves its part of the sums in `part[split][m][n]` instead
struct Product {
    Operand a, b, b_second;
    void *first, *second;
    float* part;
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
    const int n = n0 + s.col(), live = f.n - n;
    if (live <= 0) return;
#pragma unroll
    for (int i = 0; i < Tl::kFm; i++) {
        const int m = m0 + s.row() + i * 16;
        if (m >= f.m) continue;
        float v[run];
#pragma unroll
        for (int e = 0; e < run; e++) v[e] = s.acc[i][e / 4][e % 4];
        if (f.part) {
            store_run<float, run>(f.part + ((int64_t)blockIdx.y * f.m + m) * f.n + n, live, v);
        } else if (m < f.rows) {
            store_run<T, run>((T*)f.first + (int64_t)m * f.n + n, live, v);
        } else if (m >= f.cut && m - f.cut < f.rows) {
            store_run<T, run>((T*)f.second + (int64_t)(m - f.cut) * f.n + n, live, v);
        }
    }
}

// the splits' parts added up: 4 columns a thread, row r of `first` and, from row cut on, of `second`
template <typename T>
__global__ void __launch_bounds__(256)
k_join_parts(const float* __restrict__ part, int splits, int64_t m, int n, int rows, int cut, T* __restrict__ first,
             T* __restrict__ second) {
    const int across = (n + 3) / 4;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < (int64_t)rows * across * (second ? 2 : 1);
         i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / across % rows;
        const int c = (int)(i % across) * 4, live = n - c;
        const bool of_first = i < (int64_t)rows * across;
        float v[4] = {};
        for (int s = 0; s < splits; s++) {
            float p[4];
            load_some<float, 4>(part + (s * m + (of_first ? r : cut + r)) * n + c, live, p);
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] += p[e];
        }
        store_some<T, 4>((of_first ? first : second) + r * n + c, live, v);
    }
}

// ---- host -------------------------------------------------------------------

int launched() { return (int)hipGetLastError(); }

int64_t esize(int type) { return type == HG_F32 ? 4 : 2; }
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

// an operand of rows x cols values: as it is, or packed into the arena (only counted where the arena has no memory)
template <typename T>
int packed_rows(const void* src, int type, int64_t rows, int64_t cols, int64_t stride, bool as_is, Arena& ws,
                hipStream_t st, Operand* out) {
    if (as_is) {
        *out = {src, (rows <= 1 ? cols : stride) * 2, (int)rows, (int)cols * 2};
        return 0;
    }
    const int parts = parts_of(type);
    const int64_t bytes = packed_bytes(cols, parts);
    char* to = ws.take(rows * bytes);
    *out = {to, bytes, (int)rows, (int)bytes};
    if (!to || rows == 0) return 0;
    const unsigned grid = (unsigned)std::min<int64_t>((rows * (up_to(cols, 32) / 8) + kPackThreads - 1) / kPackThreads, 8192);
    if constexpr (sizeof(T) == 4)
        k_pack<float, bf16, 3><<<grid, kPackThreads, 0, st>>>((const float*)src, stride, rows, (int)cols, (bf16*)to, bytes / 2);
    else
        k_pack<T, T, 1><<<grid, kPackThreads, 0, st>>>((const T*)src, stride, rows, (int)cols, (T*)to, bytes / 2);
    return launched();
}
// both weights the same way: a tile takes them by one stride
template <typename T>
int packed_weights(const void* wg, const void* wu, int64_t hidden, int64_t cols, Arena& ws, hipStream_t st, Operand* g,
                   Operand* u) {
    constexpr int type = sizeof(T) == 4 ? HG_F32 : HG_F16;
    const bool as_is = as_it_is(wg, type, hidden, cols, cols) && as_it_is(wu, type, hidden, cols, cols);
    const int e = packed_rows<T>(wg, type, hidden, cols, cols, as_is, ws, st, g);
    return e ? e : packed_rows<T>(wu, type, hidden, cols, cols, as_is, ws, st, u);
}

// f called with the tile for an m x n result: the largest of which there are enough for the card's 256 compute units
template <typename T, typename F> int with_tile(int64_t m, int64_t n, F f) {
    using P = std::conditional_t<sizeof(T) == 4, bf16, T>;
    constexpr int parts = sizeof(T) == 4 ? 3 : 1;
    auto tiles = [&](int a, int b) { return ((m + a - 1) / a) * ((n + b - 1) / b); };
#ifdef TRY
    if constexpr (parts == 1) {
        if (TRY == 0) return f(Tile<P, parts, 2, 256, 256, 2, 4, 2, 1>{});
        if (TRY == 1) return f(Tile<P, parts, 2, 128, 128, 2, 2, 2, 2>{});
        if (TRY == 2) return f(Tile<P, parts, 2, 256, 128, 4, 2, 3, 1>{});
    }
#endif
    if constexpr (parts == 1) {
        if (tiles(256, 256) >= 192) return f(Tile<P, 1, 2, 256, 256, 2, 4, 2, 1>{});
        if (tiles(128, 128) >= 192) return f(Tile<P, 1, 2, 128, 128, 2, 2, 2, 2>{});
        return f(Tile<P, 1, 2, 64, 64, 2, 2, 3, 3>{});
    } else {
        if (tiles(128, 128) >= 192) return f(Tile<P, 3, 1, 128, 128, 2, 2, 3, 1>{});
        return f(Tile<P, 3, 1, 64, 64, 2, 2, 3, 2>{});
    }
}

template <typename T>
int forward(const void* x, int64_t rows, int64_t cols, int64_t x_stride, const void* wg, const void* wu, int64_t hidden,
            const void* bg, const void* bu, int act, void* h, float* gate, float* up, Arena& ws, hipStream_t st) {
    constexpr int type = sizeof(T) == 4 ? HG_F32 : HG_F16;
    Forward f{};
    int e = packed_rows<T>(x, type, rows, cols, x_stride, as_it_is(x, type, rows, cols, x_stride), ws, st, &f.x);
    if (!e) e = packed_weights<T>(wg, wu, hidden, cols, ws, st, &f.wg, &f.wu);
    if (e || !ws.p) return e;
    f.x.bytes = std::min(f.x.bytes, std::min(f.wg.bytes, f.wu.bytes));  // a packed row's zeros have no partner in a plain one
    f.bg = bg;
    f.bu = bu;
    f.h = h;
    f.gate = gate;
    f.up = up;
    f.hidden = (int)hidden;
    f.act = act;
    return with_tile<T>(rows, 2 * hidden, [&](auto tile) {
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
            int64_t cut, void* first, void* second, int64_t n, Arena& ws, hipStream_t st) {
    return with_tile<T>(m, n, [&](auto tile) {
        using Tl = decltype(tile);
        constexpr int deep = 32 * Tl::kSteps;
        Product f{};
        f.a = a;
        f.b = b;
        f.b_second = b_second;
        f.first = first;
        f.second = second;
        f.m = (int)m;
        f.n = (int)n;
        f.rows = (int)rows;
        f.cut = (int)cut;
        f.cut_k = (int)(cut_k / deep);
        f.tiles_m = (int)((m + Tl::kM - 1) / Tl::kM);
        f.tiles_n = (int)((n + Tl::kN - 1) / Tl::kN);
        f.slices = (int)((k + deep - 1) / deep);
        const int64_t tiles = (int64_t)f.tiles_m * f.tiles_n;
        // two blocks for each compute unit, at least 16 slices each
        int64_t splits = std::max<int64_t>(1, std::min<int64_t>({512 / tiles, f.slices / 16, 256}));
        f.each = (int)((f.slices + splits - 1) / splits);
        splits = (f.slices + f.each - 1) / f.each;
        if (splits > 1) f.part = (float*)ws.take(splits * m * n * 4);
        if (!ws.p) return 0;
        k_product<T, Tl, kTurnedA><<<dim3((unsigned)tiles, (unsigned)splits), Tl::kThreads, 0, st>>>(f);
        int e = launched();
        if (!e && splits > 1) {
            const int64_t all = rows * ((n + 3) / 4) * (second ? 2 : 1);
            k_join_parts<T><<<(unsigned)std::min<int64_t>((all + 255) / 256, 4096), 256, 0, st>>>(
                f.part, (int)splits, m, (int)n, (int)rows, (int)cut, (T*)first, (T*)second);
            e = launched();
        }
        return e;
    });
}

template <typename T>
int backward(const void* dh, int64_t dh_stride, const void* x, int64_t rows, int64_t cols, int64_t x_stride,
             const void* wg, const void* wu, int64_t hidden, const float* gate, const float* up, int act, void* dx,
             void* dwg, void* dwu, void* dbg, void* dbu, Arena& ws, hipStream_t st) {
    using P = std::conditional_t<sizeof(T) == 4, bf16, T>;
    constexpr int type = sizeof(T) == 4 ? HG_F32 : HG_F16, parts = sizeof(T) == 4 ? 3 : 1;
    const int64_t cut = up_to(hidden, 64), d_bytes = packed_bytes(2 * cut, parts);  // 64: whole slices of each half
    const int64_t blocks = (rows + kSlopeRows - 1) / kSlopeRows;
    const bool biases = dbg || dbu;
    char* d = ws.take(rows * d_bytes);
    float* sums = biases ? (float*)ws.take(blocks * 2 * hidden * 4) : nullptr;
    int e = 0;
    if (ws.p) {
        k_gated_slopes<T, P, parts><<<dim3((unsigned)blocks, (unsigned)((cut + 255) / 256)), 256, 0, st>>>(
            (const T*)dh, dh_stride, gate, up, rows, (int)hidden, act, (P*)d, d_bytes / 2, (int)cut, sums);
        e = launched();
        if (!e && biases) {
            k_join_sums<T><<<dim3((unsigned)((hidden + 63) / 64), 2), 1024, 0, st>>>(sums, blocks, (int)hidden, (T*)dbg, (T*)dbu);
            e = launched();
        }
    }
    const Operand grads{d, d_bytes, (int)rows, (int)d_bytes};
    if (!e && dx) {
        Operand g, u;
        e = packed_weights<T>(wg, wu, hidden, cols, ws, st, &g, &u);
        if (!e) e = product<T, false>(grads, g, u, rows, 2 * cut, cut, rows, rows, dx, nullptr, cols, ws, st);
    }
    if (!e && dwg) {
        Operand b;
        e = packed_rows<T>(x, type, rows, cols, x_stride, as_it_is(x, type, rows, cols, x_stride), ws, st, &b);
        if (!e) e = product<T, true>(grads, b, b, 2 * cut, rows, 1 << 30, hidden, cut, dwg, dwu, cols, ws, st);
    }
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
