// hive_train.hpp -- what the training operators' kernels (hive_norm.hip,
// hive_loss.hip, hive_adamw.hip) share: element types, sums over lanes, and
// the choice of a kernel by element type.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/hive_gpu.h"

namespace ht {

typedef _Float16 f16;
typedef __bf16 bf16;

// Arithmetic is in float32 whatever the elements are; a result is rounded to
// its element type once, to nearest, ties to even.
template <typename T> __device__ __forceinline__ float to_f32(T v) { return (float)v; }
template <typename T> __device__ __forceinline__ T from_f32(float v) { return (T)v; }

inline bool is_type(int t) { return t == HG_F32 || t == HG_F16 || t == HG_BF16; }
inline int size_of(int t) { return t == HG_F32 ? 4 : 2; }

// sum / maximum over the G lanes of a lane group (G a power of two)
template <int G> __device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
// NaN in any lane gives NaN
__device__ __forceinline__ float max_nan(float a, float b) { return a > b || a != a ? a : b; }
template <int G> __device__ __forceinline__ float group_max(float v) {
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) v = max_nan(v, __shfl_xor(v, o, 64));
    return v;
}

// f called with a value of element type `t`
template <typename F> inline int with_type(int t, F f) {
    if (t == HG_F32) return f(float{});
    if (t == HG_F16) return f(f16{});
    return f(bf16{});
}

}  // namespace ht
