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
#include "hive_train.hpp"

namespace {

using namespace ht;

constexpr int kWaves = 4;             // waves of a block
constexpr int64_t kGradBlocks = 256;  // most row ranges of the weight's gradient

__device__ __forceinline__ float sigmoid_(float x) { return 1.0f / (1.0f + expf(-x)); }

// one wave a row
template <typename T, typename W, bool kSigmoid>
__global__ void __launch_bounds__(64 * kWaves)
k_norm_forward(const T* __restrict__ x, int64_t rows, int64_t cols, int64_t x_stride, const W* __restrict__ w,
               const W* __restrict__ b, float eps, T* __restrict__ y, float* __restrict__ mean,
               float* __restrict__ rstd) {
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);
    if (row >= rows) return;
    const T* xr = x + row * x_stride;
    auto at = [&](int64_t c) {
        const float v = to_f32(xr[c]);
        return kSigmoid ? sigmoid_(v) : v;
    };
    float s = 0.0f;
    for (int64_t c = lane; c < cols; c += 64) s += at(c);
    const float m = group_sum<64>(s) / (float)cols;
    s = 0.0f;
    for (int64_t c = lane; c < cols; c += 64) {
        const float d = at(c) - m;
        s += d * d;
    }
    const float r = 1.0f / sqrtf(group_sum<64>(s) / (float)cols + eps);
    for (int64_t c = lane; c < cols; c += 64) {
        float h = (at(c) - m) * r;
        if (w) h *= to_f32(w[c]);
        if (b) h += to_f32(b[c]);
        y[row * cols + c] = from_f32<T>(h);
    }
    if (lane == 0) {
        mean[row] = m;
        rstd[row] = r;
    }
}

// one wave a row
template <typename T, typename W, bool kSigmoid>
__global__ void __launch_bounds__(64 * kWaves)
k_norm_dx(const T* __restrict__ dy, int64_t dy_stride, const T* __restrict__ x, int64_t x_stride, int64_t rows,
          int64_t cols, const float* __restrict__ mean, const float* __restrict__ rstd, const W* __restrict__ w,
          T* __restrict__ dx) {
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);
    if (row >= rows) return;
    const float m = mean[row], r = rstd[row];
    const T* xr = x + row * x_stride;
    const T* dyr = dy + row * dy_stride;
    float s1 = 0.0f, s2 = 0.0f;
    for (int64_t c = lane; c < cols; c += 64) {
        const float v = to_f32(xr[c]), a = kSigmoid ? sigmoid_(v) : v;
        const float dh = to_f32(dyr[c]) * (w ? to_f32(w[c]) : 1.0f);
        s1 += dh;
        s2 += dh * ((a - m) * r);
    }
    s1 = group_sum<64>(s1) / (float)cols;
    s2 = group_sum<64>(s2) / (float)cols;
    for (int64_t c = lane; c < cols; c += 64) {
        const float v = to_f32(xr[c]), a = kSigmoid ? sigmoid_(v) : v;
        const float dh = to_f32(dyr[c]) * (w ? to_f32(w[c]) : 1.0f);
        float da = r * (dh - s1 - (a - m) * r * s2);
        if (kSigmoid) da *= a * (1.0f - a);
        dx[row * cols + c] = from_f32<T>(da);
    }
}

// partial sums of dw and db: block (column block, row range), a thread a column
template <typename T, bool kSigmoid>
__global__ void __launch_bounds__(64)
k_norm_dw_part(const T* __restrict__ dy, int64_t dy_stride, const T* __restrict__ x, int64_t x_stride, int64_t rows,
               int64_t cols, const float* __restrict__ mean, const float* __restrict__ rstd,
               float* __restrict__ part) {
    const int64_t c = (int64_t)blockIdx.x * 64 + threadIdx.x;
    if (c >= cols) return;
    float dw = 0.0f, db = 0.0f;
    for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
        const float v = to_f32(x[row * x_stride + c]), a = kSigmoid ? sigmoid_(v) : v;
        const float g = to_f32(dy[row * dy_stride + c]);
        dw += g * ((a - mean[row]) * rstd[row]);
        db += g;
    }
    part[(2 * (int64_t)blockIdx.y) * cols + c] = dw;
    part[(2 * (int64_t)blockIdx.y + 1) * cols + c] = db;
}

template <typename W>
__global__ void __launch_bounds__(64)
k_norm_dw_join(const float* __restrict__ part, int64_t parts, int64_t cols, W* __restrict__ dw, W* __restrict__ db) {
    const int64_t c = (int64_t)blockIdx.x * 64 + threadIdx.x;
    if (c >= cols) return;
    float s1 = 0.0f, s2 = 0.0f;
    for (int64_t p = 0; p < parts; p++) {
        s1 += part[2 * p * cols + c];
        s2 += part[(2 * p + 1) * cols + c];
    }
    if (dw) dw[c] = from_f32<W>(s1);
    if (db) db[c] = from_f32<W>(s2);
}

inline int64_t grad_blocks(int64_t rows) { return rows < kGradBlocks ? rows : kGradBlocks; }

// sizes a launch can hold, strides that keep rows apart, a weight type
bool bad_sizes(int64_t rows, int64_t cols, int x_type, int w_type) {
    return rows < 0 || cols < 0 || !is_type(x_type) || !is_type(w_type) || rows > (int64_t)1 << 31 ||
           cols > (int64_t)1 << 31;
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
    const dim3 grid((unsigned)((rows + kWaves - 1) / kWaves));
    return with_type(x_type, [&](auto tx) {
        using T = decltype(tx);
        return with_type(w_type, [&](auto tw) {
            using W = decltype(tw);
            auto f = sigmoid ? k_norm_forward<T, W, true> : k_norm_forward<T, W, false>;
            hipLaunchKernelGGL(f, grid, dim3(64 * kWaves), 0, st, (const T*)x, rows, cols, x_stride,
                               (const W*)weight, (const W*)bias, eps, (T*)y, mean, rstd);
            return (int)hipGetLastError();
        });
    });
}

int64_t hg_layer_norm_backward_workspace(int64_t rows, int64_t cols) {
    if (rows <= 0 || cols <= 0) return 0;
    return 2 * grad_blocks(rows) * cols * (int64_t)sizeof(float);
}

int hg_layer_norm_backward(const void* dy, int64_t dy_stride, const void* x, int x_type, int64_t rows, int64_t cols,
                           int64_t x_stride, const float* mean, const float* rstd, const void* weight, int w_type,
                           int sigmoid, void* dx, void* dweight, void* dbias, void* workspace, void* stream) {
    if (bad_sizes(rows, cols, x_type, w_type)) return (int)hipErrorInvalidValue;
    if (cols == 0) return 0;
    const bool grads = dweight || dbias;
    if (rows > 0 && (!dy || !x || !mean || !rstd || (grads && (!workspace || ((uintptr_t)workspace & 15)))))
        return (int)hipErrorInvalidValue;
    hipStream_t st = (hipStream_t)stream;
    return with_type(x_type, [&](auto tx) {
        using T = decltype(tx);
        return with_type(w_type, [&](auto tw) {
            using W = decltype(tw);
            if (rows > 0 && dx) {
                auto f = sigmoid ? k_norm_dx<T, W, true> : k_norm_dx<T, W, false>;
                hipLaunchKernelGGL(f, dim3((unsigned)((rows + kWaves - 1) / kWaves)), dim3(64 * kWaves), 0, st,
                                   (const T*)dy, dy_stride, (const T*)x, x_stride, rows, cols, mean, rstd,
                                   (const W*)weight, (T*)dx);
            }
            if (grads) {
                const int64_t parts = grad_blocks(rows);
                const unsigned cb = (unsigned)((cols + 63) / 64);
                if (parts > 0) {
                    auto f = sigmoid ? k_norm_dw_part<T, true> : k_norm_dw_part<T, false>;
                    hipLaunchKernelGGL(f, dim3(cb, (unsigned)parts), dim3(64), 0, st, (const T*)dy, dy_stride,
                                       (const T*)x, x_stride, rows, cols, mean, rstd, (float*)workspace);
                }
                hipLaunchKernelGGL(k_norm_dw_join<W>, dim3(cb), dim3(64), 0, st, (const float*)workspace, parts, cols,
                                   (W*)dweight, (W*)dbias);
            }
            return (int)hipGetLastError();
        });
    });
}

}  // extern "C"
