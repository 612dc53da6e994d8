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
// in the flat state), 16 for each moment.  An r above zero takes the smallest
// code at least: a code of zero would leave the next step's m to be divided by
// nearly nothing.
#include <cmath>

#include "hive_train.hpp"

namespace {

using namespace ht;

constexpr int kBlock = 256;      // elements under one scale
constexpr int kTensors = 48;     // tensors of a launch: their table is a kernel argument (4 KB at most)
constexpr int kThreads = 256;
constexpr int64_t kChunk = 4 * kThreads;  // elements of a thread block, 4 a lane: a scale's block is a wave's

struct Table {
    hg_adamw_tensor t[kTensors];
    int64_t first[kTensors + 1];  // each tensor's first chunk
    int32_t n;
};
struct Step {
    float beta1, one_beta1, beta2, one_beta2, keep, rate, inv_sqrt_c2, eps;
    const float* grad_scale;
    uint32_t seed;
};

__device__ __forceinline__ uint32_t random_bits(int64_t place, uint32_t seed) {
    uint32_t h = (uint32_t)place * 0x9E3779B1u + seed * 0x85157AF5u;
    h ^= h >> 15;
    h *= 0x2C1B3C6Du;
    return h ^ (h >> 13);
}

// |x| * inv rounded to a neighbouring code (as a float, with x's sign); up: in [0, 1)
__device__ __forceinline__ float to_code(float x, float inv, float up, bool positive) {
    float a = fabsf(x) * inv;
    a = a > 448.0f ? 448.0f : a;
    const uint32_t e = max(__float_as_uint(a) & 0x7F800000u, 121u << 23);  // codes below 2^-6 are 2^-9 apart
    float steps = floorf(a * __uint_as_float(0x80800000u - e) + up);
    if (positive && steps == 0.0f && a > 0.0f) steps = 1.0f;
    return copysignf(steps * __uint_as_float(e - (3u << 23)), x);
}
__device__ __forceinline__ uint32_t pack_codes(const float c[4]) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], v, true);
}
__device__ __forceinline__ void unpack_codes(uint32_t v, float c[4]) {
    c[0] = __builtin_amdgcn_cvt_f32_fp8((int)v, 0);
    c[1] = __builtin_amdgcn_cvt_f32_fp8((int)v, 1);
    c[2] = __builtin_amdgcn_cvt_f32_fp8((int)v, 2);
    c[3] = __builtin_amdgcn_cvt_f32_fp8((int)v, 3);
}

template <typename P, typename G, int kBits>
__global__ void __launch_bounds__(kThreads) k_adamw(Table tab, Step s) {
    int lo = 0, hi = tab.n;  // the tensor of this chunk: first[lo] <= blockIdx.x < first[lo + 1]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (tab.first[mid] <= (int64_t)blockIdx.x) lo = mid;
        else hi = mid;
    }
    const hg_adamw_tensor& t = tab.t[lo];
    const int64_t at = ((int64_t)blockIdx.x - tab.first[lo]) * kChunk + 4 * (int)threadIdx.x;
    const int live = (int)max((int64_t)0, min((int64_t)4, t.count - at));
    P* p = (P*)t.param + at;
    const G* g = (const G*)t.grad + at;
    const float gs = s.grad_scale ? *s.grad_scale : 1.0f;
    float m[4] = {}, r[4] = {};
    if (kBits == 8) {
        // codes are held in whole blocks: the words beyond the last element are there
        const int64_t word = at >> 2, blk = at / kBlock;
        if (live > 0) {
            const float sm = t.exp_avg_scale[blk], sv = t.exp_avg_sq_scale[blk];
            unpack_codes(((const uint32_t*)t.exp_avg)[word], m);
            unpack_codes(((const uint32_t*)t.exp_avg_sq)[word], r);
            for (int i = 0; i < 4; i++) {
                m[i] *= sm;
                r[i] *= sv;
            }
        }
    }
    float most_m = 0.0f, most_r = 0.0f;
    for (int i = 0; i < 4; i++) {
        float v = r[i] * r[i], gi = 0.0f;
        if (i < live) {
            gi = to_f32(g[i]) * gs;
            if (kBits == 32) {
                m[i] = ((float*)t.exp_avg)[at + i];
                v = ((float*)t.exp_avg_sq)[at + i];
            }
        }
        m[i] = m[i] * s.beta1 + gi * s.one_beta1;
        v = v * s.beta2 + (gi * gi) * s.one_beta2;
        r[i] = sqrtf(v);
        if (i < live) {
            p[i] = from_f32<P>(to_f32(p[i]) * s.keep - s.rate * (m[i] / (r[i] * s.inv_sqrt_c2 + s.eps)));
            if (kBits == 32) {
                ((float*)t.exp_avg)[at + i] = m[i];
                ((float*)t.exp_avg_sq)[at + i] = v;
            }
            most_m = max_nan(most_m, fabsf(m[i]));
            most_r = max_nan(most_r, r[i]);
        } else {
            m[i] = r[i] = 0.0f;
        }
    }
    if (kBits == 8) {
        most_m = group_max<64>(most_m) * (1.0f / 448.0f);
        most_r = group_max<64>(most_r) * (1.0f / 448.0f);
        const float sm = most_m < 0x1p-110f ? 0x1p-110f : most_m, sv = most_r < 0x1p-110f ? 0x1p-110f : most_r;
        const float inv_m = 1.0f / sm, inv_r = 1.0f / sv;
        for (int i = 0; i < 4; i++) {
            const uint32_t h = random_bits(t.place + at + i, s.seed);
            m[i] = to_code(m[i], inv_m, (float)(h & 0xFFFFu) * 0x1p-16f, false);
            r[i] = to_code(r[i], inv_r, (float)(h >> 16) * 0x1p-16f, true);
        }
        if (live > 0) {
            ((uint32_t*)t.exp_avg)[at >> 2] = pack_codes(m);
            ((uint32_t*)t.exp_avg_sq)[at >> 2] = pack_codes(r);
            if ((threadIdx.x & 63) == 0) {
                t.exp_avg_scale[at / kBlock] = sm;
                t.exp_avg_sq_scale[at / kBlock] = sv;
            }
        }
    }
}

bool bad_tensor(const hg_adamw_tensor& t, int bits) {
    if (t.count < 0) return true;
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
            if (chunks + c > (int64_t)1 << 23 && tab.n > 0) break;  // a grid holds under 2^32 threads
            if (c > (int64_t)1 << 23) return (int)hipErrorInvalidValue;
            tab.t[tab.n] = tensors[i];
            tab.first[tab.n++] = chunks;
            chunks += c;
        }
        if (tab.n == 0) break;
        tab.first[tab.n] = chunks;
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
