// hive_train.hpp -- what the training operators' kernels (hive_norm.hip,
// hive_loss.hip, hive_adamw.hip) share: element types, 16-byte loads and
// stores of them, sums over lanes, and the choice of a kernel by element type.
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

// Vector<T>: the elements of one 16-byte access.  Only the elements' own
// alignment is assumed (the card takes 16-byte accesses at any of them).
template <typename T> struct Vector {
    static constexpr int n = 16 / (int)sizeof(T);
    typedef T type __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};

// At the start of a branch that all lanes take or none does: the branch stays
// one, where the optimiser would work both sides out and choose.
__device__ __forceinline__ void skipped() { asm volatile(""); }

// Elements c .. c + n - 1 of a row of cols >= n elements, in two steps, so that
// the loads of several vectors follow each other: every lane loads 16 bytes
// that lie in the row (a vector that the row's end cuts, the row's last n
// elements), and what the end cut is moved down when it is used, in the steps
// of a shifter, by the waves that hold such a vector.
template <typename T>
__device__ __forceinline__ typename Vector<T>::type load_vector(const T* row, int c, int cols) {
    constexpr int n = Vector<T>::n;
    return *(const typename Vector<T>::type*)(row + min(c, cols - n));
}
// The second step: zeros past the row's end (kZeros false: a vector wholly
// past it holds elements of the row instead).
template <typename T, bool kZeros = true>
__device__ __forceinline__ typename Vector<T>::type settle(typename Vector<T>::type v, int c, int cols) {
    constexpr int n = Vector<T>::n;
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    const int over = c - (cols - n);
    u4 q = __builtin_bit_cast(u4, v);
    if (__any(over > 0 && over < n)) {
        skipped();
        const int bytes = over > 0 ? over * (int)sizeof(T) : 0;
        if constexpr (sizeof(T) == 2) {
            const bool b = bytes & 2;
#pragma unroll
            for (int i = 0; i < 4; i++) q[i] = b ? (q[i] >> 16 | (i < 3 ? q[i < 3 ? i + 1 : 3] << 16 : 0)) : q[i];
        }
#pragma unroll
        for (int i = 0; i < 4; i++) q[i] = bytes & 4 ? (i < 3 ? q[i < 3 ? i + 1 : 3] : 0) : q[i];
#pragma unroll
        for (int i = 0; i < 4; i++) q[i] = bytes & 8 ? (i < 2 ? q[i < 2 ? i + 2 : 3] : 0) : q[i];
    }
    if (kZeros && over >= n) q = u4{0, 0, 0, 0};
    return __builtin_bit_cast(typename Vector<T>::type, q);
}
// the first `live` of n values (4 or 8) to p, a cut vector in pieces of 4, 2 and 1
template <typename T, int n = Vector<T>::n> __device__ __forceinline__ void store_some(T* p, int live, const float v[n]) {
    typedef T vec __attribute__((ext_vector_type(n), aligned(sizeof(T))));
    vec q;
#pragma unroll
    for (int i = 0; i < n; i++) q[i] = from_f32<T>(v[i]);
    if (live >= n) {
        *(vec*)p = q;
    } else if (live > 0) {
        typedef T two __attribute__((ext_vector_type(2), aligned(sizeof(T))));
        typedef T four __attribute__((ext_vector_type(4), aligned(sizeof(T))));
        int at = 0;
        if constexpr (n == 8)
            if (live & 4) {
                *(four*)p = four{q[0], q[1], q[2], q[3]};
                at = 4;
                q[0] = q[4];
                q[1] = q[5];
                q[2] = q[6];
            }
        if (live & 2) {
            *(two*)(p + at) = two{q[0], q[1]};
            at += 2;
            q[0] = q[2];
        }
        if (live & 1) p[at] = q[0];
    }
}

// v of the lane that shares a lane group: 1, 2 lanes away, mirrored in 8 and
// in 16 lanes (data-parallel moves of the VALU), the other row of 16, the
// other half of the wave
template <int kControl> __device__ __forceinline__ float dpp(float v) {
    const int i = __float_as_int(v);
    return __int_as_float(__builtin_amdgcn_mov_dpp(i, kControl, 0xF, 0xF, true));  // every lane has a source
}
// f over the G lanes of a lane group (G a power of two); every lane of the
// group gets the same bits, f being commutative
template <int G, typename F> __device__ __forceinline__ float group_join(float v, F f) {
    if constexpr (G >= 2) v = f(v, dpp<0xB1>(v));   // quad_perm [1, 0, 3, 2]
    if constexpr (G >= 4) v = f(v, dpp<0x4E>(v));   // quad_perm [2, 3, 0, 1]
    if constexpr (G >= 8) v = f(v, dpp<0x141>(v));  // row_half_mirror
    if constexpr (G >= 16) v = f(v, dpp<0x140>(v)); // row_mirror
    if constexpr (G >= 32) {
        const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = f(__uint_as_float(p[0]), __uint_as_float(p[1]));
    }
    if constexpr (G >= 64) {
        const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = f(__uint_as_float(p[0]), __uint_as_float(p[1]));
    }
    return v;
}
template <int G> __device__ __forceinline__ float group_sum(float v) {
    return group_join<G>(v, [](float a, float b) { return a + b; });
}
// the sum over the lanes at the same place in every group of G lanes
template <int G> __device__ __forceinline__ float across_groups_sum(float v) {
#pragma unroll
    for (int o = G; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// f called with a value of element type `t`
template <typename F> inline int with_type(int t, F f) {
    if (t == HG_F32) return f(float{});
    if (t == HG_F16) return f(f16{});
    return f(bf16{});
}

}  // namespace ht
