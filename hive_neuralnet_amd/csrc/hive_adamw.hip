// hive_adamw.hip -- one AdamW step of many tensors, its moments in 32 bits or
// in 8.
//
// With the gradient g (times grad_scale where there is one), step t >= 1:
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,  r = sqrt(v)
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (r / sqrt(1 - b2^t) + eps)
//
// Moments in 8 bits: 256 elements share a scale s = max(max |x| / 448, 2^-110)
// and hold float8 e4m3 codes that stand for code * s; the first moment is held
// as it is, the second as r, whose range is half as wide in powers of two.  A
// new value x / s between two codes goes to one of them at random, up with the
// probability (x / s - below) / (above - below), so that its mean is x: at
// b2 = 0.999 a step moves r by a few parts in 10^4, codes are 6 to 12 parts in
// 100 apart, and rounding to nearest would hold every r where it is.  The
// random bits are a hash of the step's seed and the element's place (its index
// in the flat state), 16 for each moment; the card's own conversion
// (v_cvt_sr_fp8_f32) adds them below the code's last bit.  An r above zero
// takes the smallest code at least: a code of zero would leave the next step's
// m to be divided by nearly nothing.
//
// A lane takes four neighbouring elements in 16-byte accesses, a wave a
// scale's 256; the waves that a CU holds keep its loads under way (four rounds
// a wave: 7 us against 2.8 for 20,546 elements, 196 against 174 for 64 M in 8
// bits, the same for 64 M in 32).
//
// Bound by memory in 32 bits: 201 M float weights with bf16 gradients 980 us,
// 5.3 TB/s of what has to move, the rate of a large copy (one element's loads
// at a time: 1,655 us).  In 8 bits the VALU comes near it, 60 operations an
// element: 144 M float weights 405 us, 5.7 TB/s, in bf16 280 us, 5.2 TB/s, where
// codes made by a divide, a correctly rounded root and float arithmetic took
// 130 and 571 us.
#include <cmath>
#include <type_traits>

#include "hive_train.hpp"

namespace {

using namespace ht;

constexpr int kBlock = 256;   // elements under one scale
constexpr int kTensors = 48;  // tensors of a launch: their table is a kernel argument (4 KB at most)
constexpr int kThreads = 256;
constexpr int64_t kChunk = 4 * kThreads;  // elements of a thread block

constexpr int64_t kMaxChunks = ((int64_t)1 << 24) - 1;  // of a launch: a grid holds under 2^32 threads

struct Table {
    hg_adamw_tensor t[kTensors];
    int64_t first[kTensors];  // each tensor's first chunk
    int32_t n;
};
struct Step {
    float beta1, one_beta1, beta2, one_beta2, keep, rate, inv_sqrt_c2, eps;
    const float* grad_scale;
    uint32_t seed;
};

// Both halves are uniform and independent of each other, of a neighbour's, of those a block on and of the next seed's
// (2^20 places under 36 seeds: chi-square of 256 bins at most 303, correlations at most 3.1 / 1,024).  0x9E3779B1 is the
// prime next to 2^32 over the golden ratio, which spreads neighbours; the other two are odd numbers that pass this.
__device__ __forceinline__ uint32_t random_bits(int64_t place, uint32_t seed) {
    uint32_t h = (uint32_t)place * 0x9E3779B1u + seed * 0x85157AF5u;
    h ^= h >> 15;
    h *= 0x2C1B3C6Du;
    return h ^ (h >> 13);
}

template <typename T> struct Four {
    typedef T type __attribute__((ext_vector_type(4), aligned(sizeof(T))));
};
template <typename T, bool kFull> __device__ __forceinline__ typename Four<T>::type load_four(const T* p, int live) {
    if (kFull) return *(const typename Four<T>::type*)p;
    typename Four<T>::type q = {};
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (i < live) q[i] = p[i];
    return q;
}
template <typename T, bool kFull>
__device__ __forceinline__ void store_four(T* p, int live, typename Four<T>::type q) {
    if (kFull) {
        *(typename Four<T>::type*)p = q;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (i < live) p[i] = q[i];
}

// sqrt(v) to half a unit of the last place, 0 for 0 and inf for inf (a step by
// m / inf = 0); a v below the smallest normal number counts as that
__device__ __forceinline__ float root(float v) {
    const float w = v < 0x1p-126f ? 0x1p-126f : v, y = __builtin_amdgcn_rsqf(w), s = w * y;
    const float r = fmaf(fmaf(-s, s, w), 0.5f * y, s);
    return v == 0.0f || v == INFINITY ? v : r;
}
// the largest of a wave's |x|, NaN if one is: their bits are in order
__device__ __forceinline__ uint32_t size_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }
__device__ __forceinline__ float wave_largest(uint32_t bits) {
    const float v = group_join<64>(__uint_as_float(bits), [](float a, float b) {
        return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b)));
    });
    return v;
}
// 1 / s to half a unit of the last place, of an s from 2^-110 to 2^120
__device__ __forceinline__ float inverse(float s) {
    const float y = __builtin_amdgcn_rcpf(s);
    return fmaf(fmaf(-s, y, 1.0f), y, y);
}
__device__ __forceinline__ float scale_of(float largest) {
    const float s = largest * (1.0f / 448.0f);
    return s < 0x1p-110f ? 0x1p-110f : s;  // NaN stays
}

template <typename P, typename G, int kBits, bool kFull>
__device__ __forceinline__ void step_chunk(const hg_adamw_tensor& t, int64_t chunk, const Step& s) {
    const int64_t at = chunk * kChunk + 4 * (int)threadIdx.x;
    const int live = kFull ? 4 : (int)max((int64_t)0, min((int64_t)4, t.count - at));
    auto p = load_four<P, kFull>((const P*)t.param + at, live);
    const auto g4 = load_four<G, kFull>((const G*)t.grad + at, live);
    float m[4], v[4], r[4];
    if constexpr (kBits == 32) {
        const auto m4 = load_four<float, kFull>((const float*)t.exp_avg + at, live);
        const auto v4 = load_four<float, kFull>((const float*)t.exp_avg_sq + at, live);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            m[i] = m4[i];
            v[i] = v4[i];
        }
    } else {
        int codes_m = 0, codes_r = 0;
        float scale_m = 0.0f, scale_r = 0.0f;
        if (live > 0) {  // codes are held in whole blocks
            codes_m = ((const int*)t.exp_avg)[at >> 2];
            codes_r = ((const int*)t.exp_avg_sq)[at >> 2];
            scale_m = t.exp_avg_scale[at / kBlock];
            scale_r = t.exp_avg_sq_scale[at / kBlock];
        }
        const auto m01 = __builtin_amdgcn_cvt_pk_f32_fp8(codes_m, false);
        const auto m23 = __builtin_amdgcn_cvt_pk_f32_fp8(codes_m, true);
        const auto r01 = __builtin_amdgcn_cvt_pk_f32_fp8(codes_r, false);
        const auto r23 = __builtin_amdgcn_cvt_pk_f32_fp8(codes_r, true);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            m[i] = (i < 2 ? m01[i & 1] : m23[i & 1]) * scale_m;
            const float q = (i < 2 ? r01[i & 1] : r23[i & 1]) * scale_r;
            v[i] = q * q;
        }
    }
    const float gs = s.grad_scale ? *s.grad_scale : 1.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float g = to_f32<G>(g4[i]) * gs;
        m[i] = m[i] * s.beta1 + g * s.one_beta1;
        v[i] = v[i] * s.beta2 + (g * g) * s.one_beta2;
        float step;
        if constexpr (kBits == 32) {
            step = m[i] / (sqrtf(v[i]) * s.inv_sqrt_c2 + s.eps);
        } else {
            r[i] = root(v[i]);
            // the reciprocal within a unit of the last place: 2 u of a step, under the 8-bit moments' own rounding
            step = m[i] * __builtin_amdgcn_rcpf(fmaf(r[i], s.inv_sqrt_c2, s.eps));
        }
        p[i] = from_f32<P>(fmaf(-s.rate, step, to_f32<P>(p[i]) * s.keep));
    }
    store_four<P, kFull>((P*)t.param + at, live, p);
    if constexpr (kBits == 32) {
        store_four<float, kFull>((float*)t.exp_avg + at, live, Four<float>::type{m[0], m[1], m[2], m[3]});
        store_four<float, kFull>((float*)t.exp_avg_sq + at, live, Four<float>::type{v[0], v[1], v[2], v[3]});
    } else {
        uint32_t most_m = 0, most_r = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (!kFull && i >= live) m[i] = r[i] = v[i] = 0.0f;
            most_m = max(most_m, size_bits(m[i]));
            most_r = max(most_r, __float_as_uint(r[i]));
        }
        const float scale_m = scale_of(wave_largest(most_m)), scale_r = scale_of(wave_largest(most_r));
        const float inv_m = inverse(scale_m), inv_r = inverse(scale_r);
        int codes_m = 0, codes_r = 0;
        auto round = [&](auto place) {
            constexpr int i = decltype(place)::value;
            const uint32_t h = random_bits(t.place + at + i, s.seed);
            const float a = __builtin_amdgcn_fmed3f(m[i] * inv_m, -448.0f, 448.0f);
            const float b = __builtin_amdgcn_fmed3f(r[i] * inv_r, v[i] == 0.0f ? 0.0f : 0x1p-9f, 448.0f);
            codes_m = __builtin_amdgcn_cvt_sr_fp8_f32(a, h << 16, codes_m, i);
            codes_r = __builtin_amdgcn_cvt_sr_fp8_f32(b, h & 0xFFFF0000u, codes_r, i);
        };
        round(std::integral_constant<int, 0>{});
        round(std::integral_constant<int, 1>{});
        round(std::integral_constant<int, 2>{});
        round(std::integral_constant<int, 3>{});
        if (live > 0) {
            ((int*)t.exp_avg)[at >> 2] = codes_m;
            ((int*)t.exp_avg_sq)[at >> 2] = codes_r;
            if ((threadIdx.x & 63) == 0) {
                t.exp_avg_scale[at / kBlock] = scale_m;
                t.exp_avg_sq_scale[at / kBlock] = scale_r;
            }
        }
    }
}

template <typename P, typename G, int kBits> __global__ void __launch_bounds__(kThreads) k_adamw(Table tab, Step s) {
    // the tensor of this chunk, the last whose first chunk is not past it: one load by as many lanes as there are
    // tensors (the table is in host memory; a search would wait for it at every step)
    const int lane = threadIdx.x & 63;
    const uint64_t begun = __ballot(lane < tab.n && tab.first[lane < kTensors ? lane : 0] <= (int64_t)blockIdx.x);
    const int lo = __popcll(begun) - 1;
    const hg_adamw_tensor& t = tab.t[lo];
    const int64_t chunk = (int64_t)blockIdx.x - tab.first[lo];
    if ((chunk + 1) * kChunk <= t.count) step_chunk<P, G, kBits, true>(t, chunk, s);
    else step_chunk<P, G, kBits, false>(t, chunk, s);
}

bool bad_tensor(const hg_adamw_tensor& t, int bits) {
    if (t.count < 0 || t.count > kMaxChunks * kChunk) return true;
    if (t.count == 0) return false;
    if (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq) return true;
    return bits == 8 && (!t.exp_avg_scale || !t.exp_avg_sq_scale || t.place % kBlock != 0 ||
                         (((uintptr_t)t.exp_avg | (uintptr_t)t.exp_avg_sq) & 3));
}

}  // namespace

extern "C" {

int hg_adamw_step(const hg_adamw_tensor* tensors, int64_t count, int param_type, int grad_type, int state_bits,
                  int64_t step, double lr, double beta1, double beta2, double eps, double weight_decay,
                  const float* grad_scale, uint32_t seed, void* stream) {
    if (count < 0 || !is_type(param_type) || !is_type(grad_type) || (state_bits != 32 && state_bits != 8) || step < 1)
        return (int)hipErrorInvalidValue;
    if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0 && eps >= 0.0)) return (int)hipErrorInvalidValue;
    if (count > 0 && !tensors) return (int)hipErrorInvalidValue;
    for (int64_t i = 0; i < count; i++)
        if (bad_tensor(tensors[i], state_bits)) return (int)hipErrorInvalidValue;
    Step s;
    s.beta1 = (float)beta1;
    s.one_beta1 = (float)(1.0 - beta1);
    s.beta2 = (float)beta2;
    s.one_beta2 = (float)(1.0 - beta2);
    s.keep = (float)(1.0 - lr * weight_decay);
    s.rate = (float)(lr / (1.0 - std::pow(beta1, (double)step)));
    s.inv_sqrt_c2 = (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, (double)step)));
    s.eps = (float)eps;
    s.grad_scale = grad_scale;
    s.seed = seed;
    hipStream_t st = (hipStream_t)stream;
    for (int64_t i = 0; i < count;) {
        Table tab;
        int64_t chunks = 0;
        tab.n = 0;
        for (; i < count && tab.n < kTensors; i++) {
            if (tensors[i].count == 0) continue;
            const int64_t c = (tensors[i].count + kChunk - 1) / kChunk;
            if (chunks + c > kMaxChunks) break;
            tab.t[tab.n] = tensors[i];
            tab.first[tab.n++] = chunks;
            chunks += c;
        }
        if (tab.n == 0) break;
        const int e = with_type(param_type, [&](auto tp) {
            using P = decltype(tp);
            return with_type(grad_type, [&](auto tg) {
                using G = decltype(tg);
                auto f = state_bits == 8 ? k_adamw<P, G, 8> : k_adamw<P, G, 32>;
                hipLaunchKernelGGL(f, dim3((unsigned)chunks), dim3(kThreads), 0, st, tab, s);
                return (int)hipGetLastError();
            });
        });
        if (e) return e;
    }
    return 0;
}

}  // extern "C"
