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
    void *h, *gate, *up;
    int hidden, act, tiles_m, tiles_n;
};

// T: the tensors' type.  A tile's columns are a wave's gates and the same hidden units' ups, in turn.
template <typename T, typename Tl>
__global__ void __launch_bounds__(Tl::kThreads, (Tl::kThreads == 512 ? 2 : 1)) k_gated_forward(Forward f) {
    __shared__ __attribute__((aligned(1024))) char lds[2 * Tl::kStage];
    constexpr int strip = Tl::kFn * 16, half = strip / 2;
    const Place t = tile_place(blockIdx.x, f.tiles_m, f.tiles_n);
    const int m0 = t.m * Tl::kM, n0 = t.n * (Tl::kN / 2);
    Sums<Tl> s;
    multiply<Tl>(
        f.x, m0, f.wg, f.wu, [](int r) { return r / strip * half + r % half; }, [](int r) { return r % strip >= half; }, n0,
        0, f.x.bytes, lds, s);
    const int col = n0 + (int)(threadIdx.x >> 6) % Tl::kWn * half + (int)(threadIdx.x & 63) / 16 * 4;
#pragma unroll
    for (int j = 0; j < Tl::kFn / 2; j++) {
        const int n = col + j * 16, live = f.hidden - n;
        if (live <= 0) continue;
        float bg[4], bu[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            bg[e] = f.bg && e < live ? to_f32<T>(((const T*)f.bg)[n + e]) : 0.0f;
            bu[e] = f.bu && e < live ? to_f32<T>(((const T*)f.bu)[n + e]) : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < Tl::kFm; i++) {
            const int64_t m = (int64_t)m0 + s.row() + i * 16;
            if (m >= f.x.rows) continue;
            float g[4], u[4], h[4], unused;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                g[e] = s.acc[i][j][e] + bg[e];
                u[e] = s.acc[i][j + Tl::kFn / 2][e] + bu[e];
                h[e] = act_of<T, false>(f.act, g[e], unused) * u[e];
            }
            const int64_t to = m * f.hidden + n;
            store_some<T, 4>((T*)f.h + to, live, h);
            if (f.gate) {
                store_some<T, 4>((T*)f.gate + to, live, g);
                store_some<T, 4>((T*)f.up + to, live, u);
            }
        }
    }
}

// dgate and dup from dh, gate and up: rows of parts [dgate | dup] for dx, each `hidden_up` values, and turned for the
// weights' gradients; with `sums`, the sums of each over the block's 64 rows: sums[row block][2][hidden].
template <typename T, typename P, int kParts>
__global__ void __launch_bounds__(256)
k_gated_slopes(const T* __restrict__ dh, int64_t dh_stride, const T* __restrict__ gate, const T* __restrict__ up,
               int64_t rows, int hidden, int act, P* __restrict__ flat, int64_t flat_stride, P* __restrict__ turned,
               int64_t turned_stride, float* __restrict__ sums) {
    __shared__ float lds[2][64][65];
    const int64_t r0 = (int64_t)blockIdx.x * 64;
    const int c0 = (int)blockIdx.y * 64;
    const int hidden_up = (int)up_to(hidden, 32);
    for (int i = threadIdx.x; i < 64 * 16; i += 256) {
        const int64_t r = r0 + i / 16;
        const int c = c0 + i % 16 * 4;
        float d[2][4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            d[0][k] = d[1][k] = 0.0f;
            if (r < rows && c + k < hidden) {
                const float g = to_f32<T>(gate[r * hidden + c + k]), u = to_f32<T>(up[r * hidden + c + k]);
                const float v = to_f32<T>(dh[r * dh_stride + c + k]);
                float slope;
                const float a = act_of<T, true>(act, g, slope);
                d[0][k] = v * u * slope;
                d[1][k] = v * a;
            }
        }
#pragma unroll
        for (int w = 0; w < 2; w++) {
            typedef P vec __attribute__((ext_vector_type(4)));
            vec q[kParts];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                lds[w][i / 16][i % 16 * 4 + k] = d[w][k];
                P part[kParts];
                split<P, kParts>(d[w][k], part);
#pragma unroll
                for (int p = 0; p < kParts; p++) q[p][k] = part[p];
            }
            if (flat && r < rows && c < hidden_up)
#pragma unroll
                for (int p = 0; p < kParts; p++)
                    *(vec*)(flat + r * flat_stride + part_place<kParts>(w * hidden_up + c, p)) = q[p];
        }
    }
    __syncthreads();
    const int64_t width = up_to(rows, 32);
    if (turned)
        for (int i = threadIdx.x; i < 2 * 64 * 8; i += 256) {
            const int w = i / 512, c = c0 + i % 512 / 8;
            const int64_t r = r0 + i % 8 * 8;
            if (c >= hidden || r >= width) continue;
            typedef P vec __attribute__((ext_vector_type(8)));
            vec q[kParts];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                P part[kParts];
                split<P, kParts>(lds[w][i % 8 * 8 + k][i % 512 / 8], part);
#pragma unroll
                for (int p = 0; p < kParts; p++) q[p][k] = part[p];
            }
#pragma unroll
            for (int p = 0; p < kParts; p++)
                *(vec*)(turned + ((int64_t)w * hidden + c) * turned_stride + part_place<kParts>(r, p)) = q[p];
        }
    if (sums && threadIdx.x < 128) {
        const int w = threadIdx.x / 64, c = threadIdx.x % 64;
        float v = 0.0f;
        for (int r = 0; r < 64; r++) v += lds[w][r][c];
        if (c0 + c < hidden) sums[((int64_t)blockIdx.x * 2 + w) * hidden + c0 + c] = v;
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

// out = A B^T: row m of the result is row m of `first` below `cut`, row m - cut of `second` from there on; with more than
// one split (grid y) each leaves its part of the sums in `part[split][rows][n]` instead
struct Product {
    Operand a, b;
    void *first, *second;
    float* part;
    int cut, n, tiles_m, tiles_n, each;  // each: bytes of a row that a split takes
};
template <typename T, typename Tl>
__global__ void __launch_bounds__(Tl::kThreads, (Tl::kThreads == 512 ? 2 : 1)) k_product(Product f) {
    __shared__ __attribute__((aligned(1024))) char lds[2 * Tl::kStage];
    const Place t = tile_place(blockIdx.x, f.tiles_m, f.tiles_n);
    const int m0 = t.m * Tl::kM, n0 = t.n * Tl::kN;
    const int begin = (int)blockIdx.y * f.each, end = min(begin + f.each, f.a.bytes);
    Sums<Tl> s;
    multiply<Tl>(
        f.a, m0, f.b, f.b, [](int r) { return r; }, [](int) { return false; }, n0, begin, end, lds, s);
#pragma unroll
    for (int i = 0; i < Tl::kFm; i++) {
        const int m = m0 + s.row() + i * 16;
        if (m >= f.a.rows) continue;
#pragma unroll
        for (int j = 0; j < Tl::kFn; j++) {
            const int n = n0 + s.col() + j * 16, live = f.n - n;
            if (live <= 0) continue;
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = s.acc[i][j][e];
            if (f.part) {
                store_some<float, 4>(f.part + ((int64_t)blockIdx.y * f.a.rows + m) * f.n + n, live, v);
            } else {
                T* to = m < f.cut ? (T*)f.first + (int64_t)m * f.n : (T*)f.second + (int64_t)(m - f.cut) * f.n;
                store_some<T, 4>(to + n, live, v);
            }
        }
    }
}

// the splits' parts added up
template <typename T>
__global__ void __launch_bounds__(256)
k_join_parts(const float* __restrict__ part, int splits, int64_t count, int64_t cut, T* __restrict__ first,
             T* __restrict__ second) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) {
        float v = 0.0f;
        for (int s = 0; s < splits; s++) v += part[s * count + i];
        (i < cut ? first[i] : second[i - cut]) = from_f32<T>(v);
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
int packed_rows(const void* src, int type, int64_t rows, int64_t cols, int64_t stride, Arena& ws, hipStream_t st,
                Operand* out) {
    if (as_it_is(src, type, rows, cols, stride)) {
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
template <typename T>
int packed_turned(const void* src, int64_t rows, int64_t cols, int64_t stride, char* to, int64_t to_stride, hipStream_t st) {
    if (!to || rows == 0 || cols == 0) return 0;
    const dim3 grid((unsigned)((rows + 63) / 64), (unsigned)((cols + 63) / 64));
    if constexpr (sizeof(T) == 4)
        k_pack_turned<float, bf16, 3>
            <<<grid, kPackThreads, 0, st>>>((const float*)src, stride, rows, (int)cols, (bf16*)to, to_stride / 2);
    else
        k_pack_turned<T, T, 1><<<grid, kPackThreads, 0, st>>>((const T*)src, stride, rows, (int)cols, (T*)to, to_stride / 2);
    return launched();
}

// f called with the tile for an m x n result: the largest of which there are enough for the card's 256 compute units
template <typename T, typename F> int with_tile(int64_t m, int64_t n, F f) {
    using P = std::conditional_t<sizeof(T) == 4, bf16, T>;
    constexpr int parts = sizeof(T) == 4 ? 3 : 1;
    auto tiles = [&](int a, int b) { return ((m + a - 1) / a) * ((n + b - 1) / b); };
    using Big = std::conditional_t<parts == 3, Tile<P, parts, 128, 256, 2, 4>, Tile<P, parts, 256, 256, 2, 4>>;
    if (tiles(Big::kM, Big::kN) >= 192) return f(Big{});
    if (tiles(128, 128) >= 192) return f(Tile<P, parts, 128, 128, 2, 2>{});
    return f(Tile<P, parts, 64, 64, 2, 2>{});
}

template <typename T>
int forward(const void* x, int64_t rows, int64_t cols, int64_t x_stride, const void* wg, const void* wu, int64_t hidden,
            const void* bg, const void* bu, int act, void* h, void* gate, void* up, Arena& ws, hipStream_t st) {
    constexpr int type = sizeof(T) == 4 ? HG_F32 : HG_F16;
    Forward f{};
    int e = packed_rows<T>(x, type, rows, cols, x_stride, ws, st, &f.x);
    if (!e) e = packed_rows<T>(wg, type, hidden, cols, cols, ws, st, &f.wg);
    if (!e) e = packed_rows<T>(wu, type, hidden, cols, cols, ws, st, &f.wu);
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

// a b^T, the sum over k cut into splits where the tiles alone would leave compute units idle
template <typename T>
int product(const Operand& a, const Operand& b, int64_t cut, void* first, void* second, Arena& ws, hipStream_t st) {
    return with_tile<T>(a.rows, b.rows, [&](auto tile) {
        using Tl = decltype(tile);
        Product f{};
        f.a = a;
        f.b = b;
        f.first = first;
        f.second = second;
        f.cut = (int)cut;
        f.n = b.rows;
        f.tiles_m = (a.rows + Tl::kM - 1) / Tl::kM;
        f.tiles_n = (b.rows + Tl::kN - 1) / Tl::kN;
        const int64_t tiles = (int64_t)f.tiles_m * f.tiles_n, slices = (a.bytes + Tl::kRow - 1) / Tl::kRow;
        // two blocks for each compute unit, at least 16 slices each
        int64_t splits = std::max<int64_t>(1, std::min<int64_t>({512 / tiles, slices / 16, 256}));
        const int64_t each = (slices + splits - 1) / splits;
        splits = (slices + each - 1) / each;
        f.each = (int)(each * Tl::kRow);
        const int64_t count = (int64_t)a.rows * b.rows;
        if (splits > 1) f.part = (float*)ws.take(splits * count * 4);
        if (!ws.p) return 0;
        k_product<T, Tl><<<dim3((unsigned)tiles, (unsigned)splits), Tl::kThreads, 0, st>>>(f);
        int e = launched();
        if (!e && splits > 1) {
            k_join_parts<T><<<(unsigned)std::min<int64_t>((count + 255) / 256, 4096), 256, 0, st>>>(
                f.part, (int)splits, count, cut * b.rows, (T*)first, (T*)second);
            e = launched();
        }
        return e;
    });
}

template <typename T>
int backward(const void* dh, int64_t dh_stride, const void* x, int64_t rows, int64_t cols, int64_t x_stride,
             const void* wg, const void* wu, int64_t hidden, const void* gate, const void* up, int act, void* dx,
             void* dwg, void* dwu, void* dbg, void* dbu, Arena& ws, hipStream_t st) {
    using P = std::conditional_t<sizeof(T) == 4, bf16, T>;
    constexpr int parts = sizeof(T) == 4 ? 3 : 1;
    const int64_t hidden_up = up_to(hidden, 32), flat = packed_bytes(2 * hidden_up, parts), turned = packed_bytes(rows, parts);
    const int64_t blocks = (rows + 63) / 64;
    const bool weights = dwg != nullptr, biases = dbg || dbu;
    char* d_flat = dx ? ws.take(rows * flat) : nullptr;
    char* w_turned = dx ? ws.take(cols * flat) : nullptr;
    char* d_turned = weights ? ws.take(2 * hidden * turned) : nullptr;
    char* x_turned = weights ? ws.take(cols * turned) : nullptr;
    float* sums = biases ? (float*)ws.take(blocks * 2 * hidden * 4) : nullptr;
    int e = 0;
    if (ws.p) {
        k_gated_slopes<T, P, parts><<<dim3((unsigned)blocks, (unsigned)((hidden + 63) / 64)), 256, 0, st>>>(
            (const T*)dh, dh_stride, (const T*)gate, (const T*)up, rows, (int)hidden, act, (P*)d_flat, flat / 2,
            (P*)d_turned, turned / 2, sums);
        e = launched();
        if (!e && biases) {
            k_join_sums<T><<<dim3((unsigned)((hidden + 63) / 64), 2), 1024, 0, st>>>(sums, blocks, (int)hidden, (T*)dbg, (T*)dbu);
            e = launched();
        }
    }
    if (!e && dx) {
        e = packed_turned<T>(wg, hidden, cols, cols, w_turned, flat, st);
        if (!e) e = packed_turned<T>(wu, hidden, cols, cols, w_turned ? w_turned + hidden_up * 2 * parts : nullptr, flat, st);
        const Operand a{d_flat, flat, (int)rows, (int)flat}, b{w_turned, flat, (int)cols, (int)flat};
        if (!e) e = product<T>(a, b, rows, dx, nullptr, ws, st);
    }
    if (!e && weights) {
        e = packed_turned<T>(x, rows, cols, x_stride, x_turned, turned, st);
        const Operand a{d_turned, turned, (int)(2 * hidden), (int)turned}, b{x_turned, turned, (int)cols, (int)turned};
        if (!e) e = product<T>(a, b, hidden, dwg, dwu, ws, st);
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
                     const void* w_up, int64_t hidden, const void* b_gate, const void* b_up, int act, void* h, void* gate,
                     void* up, void* workspace, void* stream) {
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
    with_type(type, [&](auto t) {
        return backward<decltype(t)>(nullptr, 0, nullptr, rows, cols, cols, nullptr, nullptr, hidden, nullptr, nullptr, 0,
                                     some, some, some, some, some, ws, nullptr);
    });
    return ws.used;
}

int hg_gated_backward(const void* dh, int64_t dh_stride, const void* x, int type, int64_t rows, int64_t cols,
                      int64_t x_stride, const void* w_gate, const void* w_up, int64_t hidden, const void* gate,
                      const void* up, int act, void* dx, void* dw_gate, void* dw_up, void* db_gate, void* db_up,
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
