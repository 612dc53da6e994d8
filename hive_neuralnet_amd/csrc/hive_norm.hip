// hive_norm.hip -- layer norm, forward and backward, with the encoder's
// sigmoid in front of it taken along (HiveFNN's fc2(LayerNorm(sigmoid(fc1 x))),
// fnn_network.py:175-187).
//
// For a row a of C values, a = x or a = sigmoid(x):
//   mean = sum a / C,  var = sum (a - mean)^2 / C,  rstd = 1 / sqrt(var + eps)
//   h = (a - mean) rstd,  y = h w + b
// and with the gradient dy of y, dh = dy w:
//   da = rstd (dh - sum dh / C - h sum(dh h) / C),  dx = da or da a (1 - a)
//   dw = sum over rows of dy h,  db = sum over rows of dy
//
// A row is read once and kept in registers, at most 64 bytes a lane, by as
// many lanes as that takes: a lane group of 1 to 64 lanes, so that a wave
// holds 64 / kLanes narrow rows, or 2 to 16 waves that join their sums in
// LDS.  The variance is then a sum of squared distances at no further read.
// The backward pass adds each lane's columns of dw and db up in registers
// over all the rows that its group takes, joins the groups of a block in
// LDS, and a second launch adds the blocks' sums: one order, whatever runs
// beside it, and no atomics.  (The last block to end adding them, instead of a
// launch, took 101 us against 23 for 118,271 x 64: what makes a block's sums
// visible to another chiplet writes back its whole L2 first, for every block.)
//
// Bound by memory.  Measured (MI355X, inputs not in cache): forward 16,384 x
// 2,048 f32 45 us, 6.0 TB/s; 8,192 x 4,096 bf16 25 us, 5.4; 118,271 x 64 f32
// with the sigmoid 12.4 us, 4.9; 4,096 x 5,119 bf16, rows at odd addresses, 21
// us, 4.0.  Backward 77 us, 5.2 TB/s; 40.6 us, 5.0; 19.9 us, 4.6; 38.5 us, 3.3; 2
// to 4 us of each are the second launch (1.5 more where each of its loads
// waited for the one before).  The next row is read while this one is worked on
// (8,192 x 4,096: 26 us without in the forward pass, 61 in the backward; not in
// the backward pass of f32 rows over 8,192 values, whose registers it spills) and,
// in the backward pass, h and dh are worked out again for dx, from the row's
// own 16 bits, which leaves the registers for it; loads wait for nothing, an end
// that cuts a vector is settled where the vector is used (4,096 x 5,119: 65 us
// where each load was settled before the next).
#include "hive_train.hpp"

namespace {

using namespace ht;

constexpr int kCus = 256;

// The forward pass holds 16 values of a row a lane (its weights and biases
// stay in registers besides; 32 values took 42 us against 28 for 8,192 x 4,096
// bf16 at half the waves).  The backward pass holds 32 bytes of x and of dy,
// those of the next row and the columns' sums.
constexpr int kValues = 16, kBackwardVecs = 2;
constexpr int64_t kMaxCols = 1024 * kValues;  // wider rows take kernels of their own

// 0 and 1 at the infinities.  Rounding x log2 e once puts e^-x up to |x| u off (u = 2^-24), the reciprocal adds 1 u: under
// 2 u in all, and of a sigmoid near 0 |x| u of itself.  An exact product would be two more operations a value.
__device__ __forceinline__ float sigmoid_(float x) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * x));
}

template <typename W> __device__ __forceinline__ float param_at(const void* p, int64_t c) {
    return to_f32(((const W*)p)[c]);
}
template <typename W, int n> __device__ __forceinline__ void load_param_of(const void* p, int c, int cols, float v[n]) {
    constexpr int m = Vector<W>::n;
    if constexpr (n >= m) {
        if (cols >= m) {
#pragma unroll
            for (int k = 0; k < n; k += m) {
                const typename Vector<W>::type q = settle<W>(load_vector((const W*)p, c + k, cols), c + k, cols);
#pragma unroll
                for (int i = 0; i < m; i++) v[k + i] = to_f32<W>(q[i]);
            }
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < n; i++) v[i] = c + i < cols ? param_at<W>(p, c + i) : 0.0f;
}
// values c .. c + n - 1 of a parameter (weight or bias) of any type, zeros past its end; `none` without one
template <int n>
__device__ __forceinline__ void load_param(const void* p, int type, int c, int cols, float none, float v[n]) {
    if (!p) {
#pragma unroll
        for (int i = 0; i < n; i++) v[i] = none;
    } else if (type == HG_F32) {
        load_param_of<float, n>(p, c, cols, v);
    } else if (type == HG_F16) {
        load_param_of<f16, n>(p, c, cols, v);
    } else {
        load_param_of<bf16, n>(p, c, cols, v);
    }
}
__device__ __forceinline__ float load_param(const void* p, int type, int64_t c, float none) {
    if (!p) return none;
    return type == HG_F32 ? param_at<float>(p, c) : type == HG_F16 ? param_at<f16>(p, c) : param_at<bf16>(p, c);
}
__device__ __forceinline__ void store_param(void* p, int type, int64_t c, float v) {
    if (type == HG_F32) ((float*)p)[c] = v;
    else if (type == HG_F16) ((f16*)p)[c] = from_f32<f16>(v);
    else ((bf16*)p)[c] = from_f32<bf16>(v);
}

// The shape of a kernel: a row is held by kLanes lanes, kVecs 16-byte vectors
// of each; vector k of lane l is the row's vector l + k * kLanes.
template <typename T_, int kThreads_, int kLanes_, int kVecs_> struct Shape {
    using T = T_;
    static constexpr int kLanes = kLanes_, kVecs = kVecs_, kN = Vector<T>::n;
    static constexpr int kThreads = kThreads_, kGroups = kThreads / kLanes;
    static constexpr int kWaves = kLanes > 64 ? kLanes / 64 : 1;  // of a row
    // whether the backward pass has the registers to read the next row ahead
    static constexpr bool kAhead = kThreads <= 512 || kVecs * 4 <= 8;
    // the widest rows: the columns' sums of dw and db are in LDS, each thread's its own, which leaves the registers
    // for the rest (2,048 x 16,384: bf16 48 us, 66 with them in registers and no next row; f32 95, 152 with some in
    // scratch)
    static constexpr bool kSumsInLds = kThreads == 1024 && kLanes == kThreads && kVecs * kN == kValues;
};

// v, its registers' contents unknown to the optimiser: what follows from it is worked out from it again
template <typename V> __device__ __forceinline__ V again(V v) {
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    u4 q = __builtin_bit_cast(u4, v);
    asm volatile("" : "+v"(q));
    return __builtin_bit_cast(V, q);
}

// vector k of the lane's row: its load, and what is left to do when it is used
template <typename Sh>
__device__ __forceinline__ typename Vector<typename Sh::T>::type load_row(const typename Sh::T* row, int lane, int k,
                                                                          int cols) {
    if constexpr (Sh::kLanes == 1) {
        if (cols < Sh::kN) {  // a row narrower than a vector
            typename Vector<typename Sh::T>::type q = {};
#pragma unroll
            for (int i = 0; i < Sh::kN; i++)
                if (i < cols) q[i] = row[i];
            return q;
        }
    }
    return load_vector(row, (lane + k * Sh::kLanes) * Sh::kN, cols);
}
template <typename Sh, bool kZeros>
__device__ __forceinline__ typename Vector<typename Sh::T>::type settle_row(typename Vector<typename Sh::T>::type q,
                                                                            int lane, int k, int cols) {
    if (Sh::kLanes == 1 && cols < Sh::kN) return q;
    return settle<typename Sh::T, kZeros>(q, (lane + k * Sh::kLanes) * Sh::kN, cols);
}

// the sums of S values over the lanes of a row; `lds`: [2][S][waves of the block], the halves used in turn
template <typename Sh, int S> __device__ __forceinline__ void row_sums(float (&v)[S], float* lds, int& turn) {
#pragma unroll
    for (int s = 0; s < S; s++) v[s] = group_sum<(Sh::kLanes < 64 ? Sh::kLanes : 64)>(v[s]);
    if constexpr (Sh::kWaves > 1) {
        constexpr int all = Sh::kThreads / 64;
        const int wave = threadIdx.x >> 6, first = wave / Sh::kWaves * Sh::kWaves;
        float* at = lds + turn * S * all;
        turn ^= 1;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int s = 0; s < S; s++) at[s * all + wave] = v[s];
        __syncthreads();
#pragma unroll
        for (int s = 0; s < S; s++) {
            v[s] = 0.0f;
#pragma unroll
            for (int i = 0; i < Sh::kWaves; i++) v[s] += at[s * all + first + i];
        }
    }
}

template <typename Sh>
__global__ void __launch_bounds__(Sh::kThreads)
k_norm_forward(const typename Sh::T* __restrict__ x, int64_t rows, int cols, int64_t x_stride,
               const void* __restrict__ w, const void* __restrict__ b, int w_type, float eps, int sigmoid,
               typename Sh::T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd) {
    constexpr int n = Sh::kN;
    __shared__ float lds[2 * (Sh::kThreads / 64)];
    int turn = 0;
    const int lane = threadIdx.x % Sh::kLanes;
    const int64_t step = (int64_t)gridDim.x * Sh::kGroups;
    const float inv = 1.0f / (float)cols;
    const bool tail = cols % n != 0;
    float wv[Sh::kVecs][n], bv[Sh::kVecs][n];
#pragma unroll
    for (int k = 0; k < Sh::kVecs; k++) {
        load_param<n>(w, w_type, (lane + k * Sh::kLanes) * n, cols, 1.0f, wv[k]);
        load_param<n>(b, w_type, (lane + k * Sh::kLanes) * n, cols, 0.0f, bv[k]);
    }
    typename Vector<typename Sh::T>::type next[Sh::kVecs];
    auto fetch = [&](int64_t row) {
        const typename Sh::T* xr = x + (row < rows ? row * x_stride : 0);
#pragma unroll
        for (int k = 0; k < Sh::kVecs; k++) next[k] = load_row<Sh>(xr, lane, k, cols);
    };
    fetch((int64_t)blockIdx.x * Sh::kGroups + threadIdx.x / Sh::kLanes);
    // rows are taken by whole blocks: waves that share sums stay together
    for (int64_t base = (int64_t)blockIdx.x * Sh::kGroups; base < rows; base += step) {
        const int64_t row = base + threadIdx.x / Sh::kLanes;
        const bool there = row < rows;
        typename Vector<typename Sh::T>::type raw[Sh::kVecs];
#pragma unroll
        for (int k = 0; k < Sh::kVecs; k++) raw[k] = next[k];
        if (base + step < rows) fetch(row + step);
        float a[Sh::kVecs][n];
        float s[1] = {0.0f};
#pragma unroll
        for (int k = 0; k < Sh::kVecs; k++) {
            raw[k] = settle_row<Sh, true>(raw[k], lane, k, cols);
            const int live = cols - (lane + k * Sh::kLanes) * n;
#pragma unroll
            for (int i = 0; i < n; i++) a[k][i] = to_f32<typename Sh::T>(raw[k][i]);
            if (sigmoid) {
                skipped();
#pragma unroll
                for (int i = 0; i < n; i++) a[k][i] = i < live ? sigmoid_(a[k][i]) : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < n; i++) s[0] += a[k][i];
        }
        row_sums<Sh>(s, lds, turn);
        const float m = s[0] / (float)cols;  // a product with the rounded 1 / cols would miss a constant row's value
        s[0] = 0.0f;
#pragma unroll
        for (int k = 0; k < Sh::kVecs; k++) {
            const int live = cols - (lane + k * Sh::kLanes) * n;
            float q = 0.0f;
#pragma unroll
            for (int i = 0; i < n; i++) {
                a[k][i] -= m;
                q = fmaf(a[k][i], a[k][i], q);
            }
            if (tail && live < n) {
                skipped();
                q = 0.0f;
#pragma unroll
                for (int i = 0; i < n; i++) q = i < live ? fmaf(a[k][i], a[k][i], q) : q;
            }
            s[0] += live > 0 ? q : 0.0f;
        }
        row_sums<Sh>(s, lds, turn);
        const float r = 1.0f / sqrtf(s[0] * inv + eps);
        if (!there) continue;
#pragma unroll
        for (int k = 0; k < Sh::kVecs; k++) {
            const int c = (lane + k * Sh::kLanes) * n, live = cols - c;
            if (live <= 0) break;
#pragma unroll
            for (int i = 0; i < n; i++) a[k][i] = fmaf(a[k][i] * r, wv[k][i], bv[k][i]);
            store_some(y + row * cols + c, live, a[k]);
        }
        if (lane == 0) {
            mean[row] = m;
            rstd[row] = r;
        }
    }
}

// part[block][2][cols]: the block's sums of dw and db; one block writes dw and db themselves
template <typename Sh>
__global__ void __launch_bounds__(Sh::kThreads, (Sh::kVecs == 1 ? 4 : 2))
k_norm_backward(const typename Sh::T* __restrict__ dy, int64_t dy_stride, const typename Sh::T* __restrict__ x,
                int64_t x_stride, int64_t rows, int cols, const float* __restrict__ mean,
                const float* __restrict__ rstd, const void* __restrict__ w, int w_type, int sigmoid,
                typename Sh::T* __restrict__ dx, float* __restrict__ part, void* __restrict__ dw,
                void* __restrict__ db) {
    constexpr int n = Sh::kN, all = Sh::kThreads / 64;
    __shared__ float lds[2 * 2 * all];
    int turn = 0;
    const int lane = threadIdx.x % Sh::kLanes;
    const int64_t step = (int64_t)gridDim.x * Sh::kGroups;
    const float inv = 1.0f / (float)cols;
    using V = typename Vector<typename Sh::T>::type;
    float wv[Sh::kVecs][n], sw[Sh::kVecs][n] = {}, sb[Sh::kVecs][n] = {};
#pragma unroll
    for (int k = 0; k < Sh::kVecs; k++) load_param<n>(w, w_type, (lane + k * Sh::kLanes) * n, cols, 1.0f, wv[k]);
    __shared__ float4 lds_sums[2][Sh::kSumsInLds ? Sh::kVecs * n / 4 * Sh::kThreads : 1];
    auto load_sums = [&](int k) {
#pragma unroll
        for (int i = 0; i < n; i += 4) {
            const int at = (k * n + i) / 4 * Sh::kThreads + threadIdx.x;
            const float4 p = lds_sums[0][at], q = lds_sums[1][at];
            sw[k][i] = p.x;
            sw[k][i + 1] = p.y;
            sw[k][i + 2] = p.z;
            sw[k][i + 3] = p.w;
            sb[k][i] = q.x;
            sb[k][i + 1] = q.y;
            sb[k][i + 2] = q.z;
            sb[k][i + 3] = q.w;
        }
    };
    auto store_sums = [&](int k) {
#pragma unroll
        for (int i = 0; i < n; i += 4) {
            const int at = (k * n + i) / 4 * Sh::kThreads + threadIdx.x;
            lds_sums[0][at] = make_float4(sw[k][i], sw[k][i + 1], sw[k][i + 2], sw[k][i + 3]);
            lds_sums[1][at] = make_float4(sb[k][i], sb[k][i + 1], sb[k][i + 2], sb[k][i + 3]);
        }
    };
    if constexpr (Sh::kSumsInLds)
#pragma unroll
        for (int k = 0; k < Sh::kVecs; k++) store_sums(k);
    V next[Sh::kVecs], next_dy[Sh::kVecs];
    float next_m, next_r;
    auto fetch = [&](int64_t row) {
        const bool there = row < rows;
        const typename Sh::T *xr = x + (there ? row * x_stride : 0), *dyr = dy + (there ? row * dy_stride : 0);
#pragma unroll
        for (int k = 0; k < Sh::kVecs; k++) {
            next[k] = load_row<Sh>(xr, lane, k, cols);
            next_dy[k] = load_row<Sh>(dyr, lane, k, cols);
        }
        next_m = there ? mean[row] : 0.0f;
        next_r = there ? rstd[row] : 0.0f;
    };
    if (Sh::kAhead) fetch((int64_t)blockIdx.x * Sh::kGroups + threadIdx.x / Sh::kLanes);
    for (int64_t base = (int64_t)blockIdx.x * Sh::kGroups; base < rows; base += step) {
        const int64_t row = base + threadIdx.x / Sh::kLanes;
        const bool there = row < rows;
        if (!Sh::kAhead) fetch(row);
        V raw[Sh::kVecs], raw_dy[Sh::kVecs];
#pragma unroll
        for (int k = 0; k < Sh::kVecs; k++) {
            raw[k] = next[k];
            raw_dy[k] = next_dy[k];
        }
        const float m = next_m, r = next_r;
        if (Sh::kAhead && base + step < rows) fetch(row + step);
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < Sh::kVecs; k++) {
            raw[k] = settle_row<Sh, false>(raw[k], lane, k, cols);
            raw_dy[k] = settle_row<Sh, false>(raw_dy[k], lane, k, cols);
            // past the row dy is 0: what h holds there adds nothing
            if (!there || (lane + k * Sh::kLanes) * n >= cols) raw_dy[k] = V{};
            float a[n];
#pragma unroll
            for (int i = 0; i < n; i++) a[i] = to_f32<typename Sh::T>(raw[k][i]);
            if (sigmoid) {
                skipped();
#pragma unroll
                for (int i = 0; i < n; i++) a[i] = sigmoid_(a[i]);
            }
            if constexpr (Sh::kSumsInLds) load_sums(k);
#pragma unroll
            for (int i = 0; i < n; i++) {
                const float h = (a[i] - m) * r;  // not a r - m r: far from zero the rounding of m r is not small
                const float d = to_f32<typename Sh::T>(raw_dy[k][i]), dh = d * wv[k][i];
                sw[k][i] = fmaf(d, h, sw[k][i]);
                sb[k][i] += d;
                s[0] += dh;
                s[1] = fmaf(dh, h, s[1]);
            }
            if constexpr (Sh::kSumsInLds) store_sums(k);
        }
        row_sums<Sh>(s, lds, turn);
        if (!there || !dx) continue;
        const float r2 = r * r * (s[1] * inv), r1 = r * (s[0] * inv);
#pragma unroll
        for (int k = 0; k < Sh::kVecs; k++) {
            const int c = (lane + k * Sh::kLanes) * n, live = cols - c;
            if (live <= 0) break;
            // h and dh are worked out again from the row as it was read: half the registers where it is in 16 bits
            V q = raw[k], q_dy = raw_dy[k];
            if constexpr (Sh::kVecs > 1) {
                q = again(q);
                q_dy = again(q_dy);
            }
            float a[n], da[n];
#pragma unroll
            for (int i = 0; i < n; i++) a[i] = to_f32<typename Sh::T>(q[i]);
            if (sigmoid) {
                skipped();
#pragma unroll
                for (int i = 0; i < n; i++) a[i] = sigmoid_(a[i]);
            }
#pragma unroll
            for (int i = 0; i < n; i++)  // r (dh - s1 - h s2)
                da[i] = fmaf(to_f32<typename Sh::T>(q_dy[i]), r * wv[k][i], fmaf(a[i] - m, -r2, -r1));
            if (sigmoid) {
                skipped();
#pragma unroll
                for (int i = 0; i < n; i++) da[i] *= a[i] * (1.0f - a[i]);
            }
            store_some(dx + row * cols + c, live, da);
        }
    }
    if (!part) return;
    if constexpr (Sh::kSumsInLds)
#pragma unroll
        for (int k = 0; k < Sh::kVecs; k++) load_sums(k);
    auto give = [&](int which, int64_t c, float v) {
        if (gridDim.x > 1) part[(2 * (int64_t)blockIdx.x + which) * cols + c] = v;
        else if (which == 0 && dw) store_param(dw, w_type, c, v);
        else if (which == 1 && db) store_param(db, w_type, c, v);
    };
    // the groups of a wave, then those of the block, a vector of a lane's columns at a time
    constexpr int width = Sh::kLanes, groups = width < 64 ? all : Sh::kGroups, count = width * n;
    __shared__ float join[2][n][Sh::kGroups > 1 ? groups * width + 1 : 1];
#pragma unroll
    for (int k = 0; k < Sh::kVecs; k++) {
        if constexpr (Sh::kGroups > 1) {
            const int group = width < 64 ? threadIdx.x >> 6 : threadIdx.x / width;
            if (k) __syncthreads();
#pragma unroll
            for (int i = 0; i < n; i++) {
                const float p = across_groups_sum<(width < 64 ? width : 64)>(sw[k][i]);
                const float q = across_groups_sum<(width < 64 ? width : 64)>(sb[k][i]);
                if (width >= 64 || (int)(threadIdx.x & 63) < width) {
                    join[0][i][group * width + lane] = p;
                    join[1][i][group * width + lane] = q;
                }
            }
            __syncthreads();
        }
        if constexpr (Sh::kGroups > 1 && width <= 64) {
            // many groups of few columns: all threads add them, a column each (36,452 x 26 f16: 11.0 us, 13.3 where the
            // lanes of one group do; 2,000 x 4,096 bf16: 18.3 and 16.5)
            for (int o = threadIdx.x; o < 2 * count; o += Sh::kThreads) {
                const int which = o / count, c = o % count + k * count;
                if (c >= cols) continue;
                float v = 0.0f;
#pragma unroll
                for (int g = 0; g < groups; g++) v += join[which][o % n][g * width + o % count / n];
                give(which, c, v);
            }
        } else if ((int)threadIdx.x < width) {
            const int c = (lane + k * width) * n;
            if constexpr (Sh::kGroups > 1)
#pragma unroll
                for (int i = 0; i < n; i++) {
                    sw[k][i] = sb[k][i] = 0.0f;
                    for (int g = 0; g < groups; g++) {
                        sw[k][i] += join[0][i][g * width + lane];
                        sb[k][i] += join[1][i][g * width + lane];
                    }
                }
#pragma unroll
            for (int i = 0; i < n; i += 4) {
                if (gridDim.x > 1) {
                    store_some<float, 4>(part + 2 * (int64_t)blockIdx.x * cols + c + i, cols - c - i, sw[k] + i);
                    store_some<float, 4>(part + (2 * (int64_t)blockIdx.x + 1) * cols + c + i, cols - c - i, sb[k] + i);
                } else {
                    for (int j = i; j < i + 4 && c + j < cols; j++) {
                        give(0, c + j, sw[k][j]);
                        give(1, c + j, sb[k][j]);
                    }
                }
            }
        }
    }
}

// dw, db = the sums of part[parts][2][cols]; a block of 32 x 32 threads takes 32 of the 2 cols columns
__global__ void __launch_bounds__(1024)
k_norm_join(const float* __restrict__ part, int parts, int64_t cols, int w_type, void* __restrict__ dw,
            void* __restrict__ db) {
    __shared__ float lds[32][33];
    const int64_t c = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31);
    float s = 0.0f;
    constexpr int n = 8;  // parts whose loads go out together
    if (c < 2 * cols)
        for (int p = threadIdx.x >> 5; p < parts; p += 32 * n) {
            float v[n];
#pragma unroll
            for (int k = 0; k < n; k++) v[k] = part[2 * (int64_t)min(p + 32 * k, parts - 1) * cols + c];
#pragma unroll
            for (int k = 0; k < n; k++) s += p + 32 * k < parts ? v[k] : 0.0f;
        }
    lds[threadIdx.x >> 5][threadIdx.x & 31] = s;
    __syncthreads();
    if (threadIdx.x >= 32 || c >= 2 * cols) return;
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; i++) s += lds[i][threadIdx.x];
    if (c < cols) {
        if (dw) store_param(dw, w_type, c, s);
    } else if (db) {
        store_param(db, w_type, c - cols, s);
    }
}

// ---- rows of more values than a block holds: a block a row, read once per use ----
//
// The simplest form, an element a load: 1,024 x 32,768 bf16 115 us forward and 132
// back, f32 114 and 178, where the bytes at a copy's 5.4 TB/s are 25 and 37, 50 and
// 75.  The row is read three times (x and dy twice, and again for the columns).

constexpr int kWide = 1024;

__device__ __forceinline__ float wide_sum(float v, float* lds) {
    v = group_sum<64>(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < kWide / 64; i++) v += lds[i];
    return v;
}

template <typename T>
__global__ void __launch_bounds__(kWide)
k_norm_forward_wide(const T* __restrict__ x, int64_t cols, int64_t x_stride, const void* __restrict__ w,
                    const void* __restrict__ b, int w_type, float eps, int sigmoid, T* __restrict__ y,
                    float* __restrict__ mean, float* __restrict__ rstd) {
    __shared__ float lds[kWide / 64];
    const int64_t row = blockIdx.x;
    const T* xr = x + row * x_stride;
    auto at = [&](int64_t c) {
        const float v = to_f32(xr[c]);
        return sigmoid ? sigmoid_(v) : v;
    };
    float s = 0.0f;
    for (int64_t c = threadIdx.x; c < cols; c += kWide) s += at(c);
    const float m = wide_sum(s, lds) / (float)cols;
    s = 0.0f;
    for (int64_t c = threadIdx.x; c < cols; c += kWide) {
        const float d = at(c) - m;
        s = fmaf(d, d, s);
    }
    const float r = 1.0f / sqrtf(wide_sum(s, lds) / (float)cols + eps);
    for (int64_t c = threadIdx.x; c < cols; c += kWide) {
        y[row * cols + c] =
            from_f32<T>(fmaf((at(c) - m) * r, load_param(w, w_type, c, 1.0f), load_param(b, w_type, c, 0.0f)));
    }
    if (threadIdx.x == 0) {
        mean[row] = m;
        rstd[row] = r;
    }
}

template <typename T>
__global__ void __launch_bounds__(kWide)
k_norm_dx_wide(const T* __restrict__ dy, int64_t dy_stride, const T* __restrict__ x, int64_t x_stride, int64_t cols,
               const float* __restrict__ mean, const float* __restrict__ rstd, const void* __restrict__ w, int w_type,
               int sigmoid, T* __restrict__ dx) {
    __shared__ float lds[kWide / 64];
    const int64_t row = blockIdx.x;
    const float m = mean[row], r = rstd[row];
    float s1 = 0.0f, s2 = 0.0f, a;
    auto dh = [&](int64_t c) {
        const float v = to_f32(x[row * x_stride + c]);
        a = sigmoid ? sigmoid_(v) : v;
        return to_f32(dy[row * dy_stride + c]) * load_param(w, w_type, c, 1.0f);
    };
    for (int64_t c = threadIdx.x; c < cols; c += kWide) {
        const float d = dh(c);
        s1 += d;
        s2 = fmaf(d, (a - m) * r, s2);
    }
    s1 = wide_sum(s1, lds) / (float)cols;
    s2 = wide_sum(s2, lds) / (float)cols;
    for (int64_t c = threadIdx.x; c < cols; c += kWide) {
        const float d = dh(c);
        float da = r * (d - s1 - (a - m) * r * s2);
        if (sigmoid) da *= a * (1.0f - a);
        dx[row * cols + c] = from_f32<T>(da);
    }
}

// block (256 columns, range of rows): a thread a column
template <typename T>
__global__ void __launch_bounds__(256)
k_norm_dw_wide(const T* __restrict__ dy, int64_t dy_stride, const T* __restrict__ x, int64_t x_stride, int64_t rows,
               int64_t cols, const float* __restrict__ mean, const float* __restrict__ rstd, int sigmoid,
               float* __restrict__ part) {
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= cols) return;
    float sw = 0.0f, sb = 0.0f;
    for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
        const float v = to_f32(x[row * x_stride + c]), a = sigmoid ? sigmoid_(v) : v;
        const float g = to_f32(dy[row * dy_stride + c]);
        sw = fmaf(g, (a - mean[row]) * rstd[row], sw);
        sb += g;
    }
    part[2 * (int64_t)blockIdx.y * cols + c] = sw;
    part[(2 * (int64_t)blockIdx.y + 1) * cols + c] = sb;
}

constexpr int threads_of(int lanes, int least) { return lanes > least ? lanes : least; }

// f called with the Shape that holds rows of `cols` values of T in the fewest lanes, at most `most` vectors in each
// (kNarrow threads a block where a row is one vector a lane, kBroad where it is more)
template <typename T, int most, int kNarrow, int kBroad, typename F> int with_shape(int64_t cols, F f) {
    constexpr int n = Vector<T>::n;
    const int64_t vecs = (cols + n - 1) / n;
    if (vecs <= 1) return f(Shape<T, kNarrow, 1, 1>{});
    if (vecs <= 2) return f(Shape<T, kNarrow, 2, 1>{});
    if (vecs <= 4) return f(Shape<T, kNarrow, 4, 1>{});
    if (vecs <= 8) return f(Shape<T, kNarrow, 8, 1>{});
    if (vecs <= 16) return f(Shape<T, kNarrow, 16, 1>{});
    if (vecs <= 32) return f(Shape<T, kNarrow, 32, 1>{});
    if (vecs <= 64) return f(Shape<T, kNarrow, 64, 1>{});
    if (vecs <= 128) return f(Shape<T, kBroad, 64, 2>{});
    if (vecs <= 64 * most) return f(Shape<T, kBroad, 64, most>{});
    if (vecs <= 128 * most) return f(Shape<T, kBroad, 128, most>{});
    if (vecs <= 256 * most) return f(Shape<T, kBroad, 256, most>{});
    if (vecs <= 512 * most) return f(Shape<T, threads_of(512, kBroad), 512, most>{});
    if (vecs <= 1024 * most) return f(Shape<T, 1024, 1024, most>{});
    return f(Shape<T, 1024, 1024, kValues / n>{});  // up to kMaxCols
}
template <typename T, typename F> int with_forward_shape(int64_t cols, F f) {
    return with_shape<T, kValues / Vector<T>::n, 256, 256>(cols, f);
}
template <typename T, typename F> int with_backward_shape(int64_t cols, F f) {
    return with_shape<T, kBackwardVecs, 1024, 512>(cols, f);
}
// one wave of each SIMD's four (a block's weights are read once for all its rows)
template <typename Sh> int64_t forward_blocks(int64_t rows) {
    const int64_t need = (rows + Sh::kGroups - 1) / Sh::kGroups, most = (int64_t)kCus * 1024 / Sh::kThreads;
    return need < most ? need : most;
}
// As many waves as the registers leave room for, 8 a CU where a lane holds two
// vectors, else 16.  A block ends with its sums' way through LDS and memory: a
// lane group of more than a wave takes two rows at least (300 x 4,096: 12.0 us
// at one row, 10.1 at two, 10.9 at four); narrower groups are many in a block
// and take one (5,928 x 113 f16: 8.4 us, 9.4 at two), but two where that saves
// the second launch (100 x 64: 7.5 and 4.9).
template <typename Sh> int64_t backward_blocks(int64_t rows) {
    const int64_t two = (rows + 2 * Sh::kGroups - 1) / (2 * Sh::kGroups), one = (rows + Sh::kGroups - 1) / Sh::kGroups;
    const int64_t need = Sh::kLanes > 64 || two == 1 ? two : one;
    const int64_t most = (int64_t)kCus * (Sh::kVecs == 1 || Sh::kThreads > 512 ? 1024 : 512) / Sh::kThreads;
    return need < most ? need : most;
}
constexpr int64_t kWideParts = 64;  // row ranges of k_norm_dw_wide

// sizes that a launch can hold (k_norm_join: a grid holds under 2^32 threads), types
bool bad_sizes(int64_t rows, int64_t cols, int x_type, int w_type) {
    return rows < 0 || cols < 0 || !is_type(x_type) || !is_type(w_type) || rows > (int64_t)1 << 31 ||
           cols > (int64_t)1 << 25;
}

}  // namespace

extern "C" {

int hg_layer_norm_forward(const void* x, int x_type, int64_t rows, int64_t cols, int64_t x_stride,
                          const void* weight, const void* bias, int w_type, float eps, int sigmoid, void* y,
                          float* mean, float* rstd, void* stream) {
    if (bad_sizes(rows, cols, x_type, w_type)) return (int)hipErrorInvalidValue;
    if (rows == 0 || cols == 0) return 0;
    if (!x || !y || !mean || !rstd) return (int)hipErrorInvalidValue;
    hipStream_t st = (hipStream_t)stream;
    return with_type(x_type, [&](auto tx) {
        using T = decltype(tx);
        if (cols > kMaxCols) {
            if (rows > (int64_t)1 << 21) return (int)hipErrorInvalidValue;  // a grid holds under 2^32 threads
            hipLaunchKernelGGL(k_norm_forward_wide<T>, dim3((unsigned)rows), dim3(kWide), 0, st, (const T*)x, cols,
                               x_stride, weight, bias, w_type, eps, sigmoid, (T*)y, mean, rstd);
            return (int)hipGetLastError();
        }
        return with_forward_shape<T>(cols, [&](auto shape) {
            using Sh = decltype(shape);
            hipLaunchKernelGGL(k_norm_forward<Sh>, dim3((unsigned)forward_blocks<Sh>(rows)), dim3(Sh::kThreads), 0,
                               st, (const T*)x, rows, (int)cols, x_stride, weight, bias, w_type, eps, sigmoid, (T*)y,
                               mean, rstd);
            return (int)hipGetLastError();
        });
    });
}

int64_t hg_layer_norm_backward_workspace(int64_t rows, int64_t cols) {
    if (rows <= 0 || cols <= 0) return 0;
    // the most blocks of any element type
    int64_t parts = rows < kWideParts ? rows : kWideParts;
    auto more = [&](int64_t p) { parts = parts > p ? parts : p; return 0; };
    if (cols <= kMaxCols) {
        with_backward_shape<float>(cols, [&](auto s) { return more(backward_blocks<decltype(s)>(rows)); });
        with_backward_shape<f16>(cols, [&](auto s) { return more(backward_blocks<decltype(s)>(rows)); });
    }
    return 2 * parts * cols * (int64_t)sizeof(float);
}

int hg_layer_norm_backward(const void* dy, int64_t dy_stride, const void* x, int x_type, int64_t rows, int64_t cols,
                           int64_t x_stride, const float* mean, const float* rstd, const void* weight, int w_type,
                           int sigmoid, void* dx, void* dweight, void* dbias, void* workspace, void* stream) {
    if (bad_sizes(rows, cols, x_type, w_type)) return (int)hipErrorInvalidValue;
    if (cols == 0) return 0;
    const bool grads = dweight || dbias;
    if (rows > 0 && (!dy || !x || !mean || !rstd || (grads && (!workspace || ((uintptr_t)workspace & 15)))))
        return (int)hipErrorInvalidValue;
    if (!grads && (!dx || rows == 0)) return 0;
    hipStream_t st = (hipStream_t)stream;
    float* part = grads ? (float*)workspace : nullptr;
    int64_t parts = 0;
    int e = 0;
    if (rows > 0)
        e = with_type(x_type, [&](auto tx) {
            using T = decltype(tx);
            if (cols > kMaxCols) {
                if (rows > (int64_t)1 << 21) return (int)hipErrorInvalidValue;
                if (dx)
                    hipLaunchKernelGGL(k_norm_dx_wide<T>, dim3((unsigned)rows), dim3(kWide), 0, st, (const T*)dy,
                                       dy_stride, (const T*)x, x_stride, cols, mean, rstd, weight, w_type, sigmoid,
                                       (T*)dx);
                if (grads) {
                    parts = rows < kWideParts ? rows : kWideParts;
                    hipLaunchKernelGGL(k_norm_dw_wide<T>, dim3((unsigned)((cols + 255) / 256), (unsigned)parts),
                                       dim3(256), 0, st, (const T*)dy, dy_stride, (const T*)x, x_stride, rows, cols,
                                       mean, rstd, sigmoid, part);
                }
                return (int)hipGetLastError();
            }
            return with_backward_shape<T>(cols, [&](auto shape) {
                using Sh = decltype(shape);
                const int64_t blocks = backward_blocks<Sh>(rows);
                parts = blocks;
                hipLaunchKernelGGL(k_norm_backward<Sh>, dim3((unsigned)blocks), dim3(Sh::kThreads), 0, st,
                                   (const T*)dy, dy_stride, (const T*)x, x_stride, rows, (int)cols, mean, rstd,
                                   weight, w_type, sigmoid, (T*)dx, part, dweight, dbias);
                return (int)hipGetLastError();
            });
        });
    if (e || !grads || (parts == 1 && cols <= kMaxCols)) return e;
    hipLaunchKernelGGL(k_norm_join, dim3((unsigned)((2 * cols + 31) / 32)), dim3(1024), 0, st, part, (int)parts, cols,
                       w_type, dweight, dbias);
    return (int)hipGetLastError();
}

}  // extern "C"
