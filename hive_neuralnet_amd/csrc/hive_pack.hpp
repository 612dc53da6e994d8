// hive_pack.hpp -- what brings tensors into the form that hive_matrix.hpp's
// tiles take: rows of 16-bit parts, 16-byte aligned, k along the row, zeros up
// to a multiple of 32.
#pragma once

#include "hive_matrix.hpp"

namespace hm {

// the parts of a value, their sum the value (3 parts: exactly, from 2^-110 in size up)
template <typename T, int kParts> __device__ __forceinline__ void split(float v, T (&part)[kParts]) {
    if constexpr (kParts == 1) {
        part[0] = (T)v;
    } else if constexpr (kParts == 2) {
        part[0] = (T)v;
        part[1] = (T)(v - (float)part[0]);
    } else {
        // the largest bfloat16: values that would round to inf keep to it, their other parts make up the rest.  What is inf or
        // NaN itself has it in its last part, which meets the other factor's first alone, and that is 0 only where the factor
        // is (its other parts may be, and inf times them NaN); 1 of its sign in its first, which the other's own inf meets.
        const float top = __uint_as_float(0x7F7F0000u);
        const bool finite = __builtin_fabsf(v) < __builtin_inff();
        part[0] = (T)(finite ? __builtin_amdgcn_fmed3f(v, -top, top) : __builtin_copysignf(1.0f, v));
        const float r = finite ? v - (float)part[0] : 0.0f;
        part[1] = (T)r;
        part[2] = (T)(finite ? r - (float)part[1] : v);
    }
}
// element of column c, part p, in a row of parts
template <int kParts> __host__ __device__ __forceinline__ int64_t part_place(int64_t c, int p) {
    return kParts == 1 ? c : (c / 32 * kParts + p) * 32 + c % 32;
}
__host__ __device__ inline int64_t up_to(int64_t n, int64_t unit) { return (n + unit - 1) / unit * unit; }
// bytes of a packed row of n values
inline int64_t packed_bytes(int64_t n, int parts) { return up_to(n, 32) * 2 * parts; }

constexpr int kPackThreads = 256;

// What a launch packs: up to three tensors of rows of one width, grid y.
struct Packing {
    const void* src[3];
    void* dst[3];
    int64_t src_stride[3], rows[3], dst_stride;
    int cols, count;
};
// dst[r] = the parts of src[r][0..cols), zeros up to a multiple of 32.  Memory bound; a thread takes 8 values.
template <typename S, typename T, int kParts> __global__ void __launch_bounds__(kPackThreads) k_pack(Packing f) {
    const int groups = (int)up_to(f.cols, 32) / 8;
    const S* const src = (const S*)f.src[blockIdx.y];
    T* const dst = (T*)f.dst[blockIdx.y];
    const int64_t rows = f.rows[blockIdx.y], src_stride = f.src_stride[blockIdx.y];
    for (int64_t i = (int64_t)blockIdx.x * kPackThreads + threadIdx.x; i < rows * groups;
         i += (int64_t)gridDim.x * kPackThreads) {
        const int64_t r = rows < 1 << 20 && groups < 1 << 11 ? (int64_t)((uint32_t)i / (uint32_t)groups) : i / groups;
        const int c = (int)(i - r * groups) * 8;
        float v[8];
        load_some<S, 8>(src + r * src_stride + c, f.cols - c, v);
        typedef T vec __attribute__((ext_vector_type(8)));
        vec q[kParts];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            T part[kParts];
            split<T, kParts>(v[k], part);
#pragma unroll
            for (int p = 0; p < kParts; p++) q[p][k] = part[p];
        }
#pragma unroll
        for (int p = 0; p < kParts; p++) *(vec*)(dst + r * f.dst_stride + part_place<kParts>(c, p)) = q[p];
    }
}

}  // namespace hm
