// hive_loss.hip -- the training loss of a batch of positions, with its gradient.
//
// Position b has n[b] = clamp(num_actions[b], 0, width) legal moves; its
// logits x are n[b] values of one flat array, the positions one after the
// other, its searched policy pi the first n[b] values of row b of
// targets[B][width] (what lies beyond is not read).
//   lse_b = log sum exp x,  CE_b = sum pi (lse_b - x) over pi != 0
//   policy = sum w_b CE_b / sum w,      value = sum u_b (v_b - z_b)^2 / sum u
//   total = policy + c value
//   dx = s w_b / sum w (p mass_b - pi),  p = exp(x - lse_b), mass_b = sum pi
//   dv = s 2 c u_b / sum u (v_b - z_b)
// A position of weight zero, without moves, or whose logits are all -inf adds
// nothing and has a gradient of zeros; weights that sum to zero give a loss
// of zero.  A logit of -inf has p = 0; where pi says otherwise the loss is inf.
#include "hive_train.hpp"

namespace {

using namespace ht;

constexpr int kWaves = 4;
constexpr int kPlanThreads = 1024;

__device__ __forceinline__ int64_t clamp_count(int64_t n, int64_t width) {
    return n < 0 ? 0 : (n > width ? width : n);
}

// the sum over a block of kPlanThreads, in every thread
template <typename V> __device__ __forceinline__ V block_sum(V v, V* lds) {
    __syncthreads();
    lds[threadIdx.x] = v;
    __syncthreads();
    for (int o = kPlanThreads / 2; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) lds[threadIdx.x] += lds[threadIdx.x + o];
        __syncthreads();
    }
    return lds[0];
}

// one block: offsets[b] = n[0] + ... + n[b - 1] (offsets[B] the sum of all),
// sums = {sum of policy weights, sum of value weights}
__global__ void __launch_bounds__(kPlanThreads)
k_loss_plan(const int64_t* __restrict__ num_actions, int64_t B, int64_t width, const float* __restrict__ pw,
            const float* __restrict__ vw, int64_t* __restrict__ offsets, float* __restrict__ sums) {
    __shared__ int64_t scan[kPlanThreads];
    __shared__ float part[kPlanThreads];
    const int t = threadIdx.x;
    const int64_t per = (B + kPlanThreads - 1) / kPlanThreads, lo = min(B, t * per), hi = min(B, lo + per);
    int64_t n = 0;
    float sp = 0.0f, sv = 0.0f;
    for (int64_t b = lo; b < hi; b++) {
        n += clamp_count(num_actions[b], width);
        sp += pw[b];
        sv += vw[b];
    }
    scan[t] = n;
    __syncthreads();
    for (int o = 1; o < kPlanThreads; o <<= 1) {
        const int64_t before = t >= o ? scan[t - o] : 0;
        __syncthreads();
        scan[t] += before;
        __syncthreads();
    }
    int64_t at = scan[t] - n;
    for (int64_t b = lo; b < hi; b++) {
        offsets[b] = at;
        at += clamp_count(num_actions[b], width);
    }
    if (t == kPlanThreads - 1) offsets[B] = scan[t];
    sp = block_sum(sp, part);
    sv = block_sum(sv, part);
    if (t == 0) {
        sums[0] = sp;
        sums[1] = sv;
    }
}

// one wave a position; row_loss[b] = {its share of the policy loss, of the value loss}
template <typename T, typename P>
__global__ void __launch_bounds__(64 * kWaves)
k_loss_rows(const T* __restrict__ logits, int64_t N, const T* __restrict__ values, const int64_t* __restrict__ offsets,
            const float* __restrict__ sums, const P* __restrict__ targets, int64_t width,
            const float* __restrict__ pw, const float* __restrict__ vt, const float* __restrict__ vw, int64_t B,
            float value_coef, float loss_scale, float2* __restrict__ row_loss, T* __restrict__ dlogits,
            T* __restrict__ dvalues) {
    const int lane = threadIdx.x & 63;
    const int64_t b = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);
    if (b >= B) return;
    const int64_t lo = min(N, offsets[b]), n = min(N, offsets[b + 1]) - lo;
    const T* x = logits + lo;
    const P* pi = targets + b * width;
    const float W = sums[0], U = sums[1];
    const float w = pw[b], share = W > 0.0f ? w / W : w;
    float top = -INFINITY;
    for (int64_t i = lane; i < n; i += 64) top = max_nan(top, to_f32(x[i]));
    top = group_max<64>(top);
    const bool used = w != 0.0f && top != -INFINITY;
    float total = 0.0f, mass = 0.0f, cross = 0.0f;
    if (used)
        for (int64_t i = lane; i < n; i += 64) {
            const float z = to_f32(x[i]) - top, q = to_f32(pi[i]);
            total += expf(z);
            mass += q;
            if (q != 0.0f) cross += q * z;
        }
    total = group_sum<64>(total);
    mass = group_sum<64>(mass);
    cross = group_sum<64>(cross);
    const float scale = share * loss_scale, k = mass / total;
    for (int64_t i = lane; i < n; i += 64) {
        const float g = used ? (expf(to_f32(x[i]) - top) * k - to_f32(pi[i])) * scale : 0.0f;
        dlogits[lo + i] = from_f32<T>(g);
    }
    if (b == B - 1)  // logits that no position has
        for (int64_t i = lo + n + lane; i < N; i += 64) dlogits[i] = from_f32<T>(0.0f);
    if (lane == 0) {
        const float u = U > 0.0f ? vw[b] / U : vw[b], off = to_f32(values[b]) - vt[b];
        row_loss[b] = make_float2(used ? (logf(total) * mass - cross) * share : 0.0f, u != 0.0f ? u * off * off : 0.0f);
        dvalues[b] = from_f32<T>(u != 0.0f ? 2.0f * value_coef * u * off * loss_scale : 0.0f);
    }
}

__global__ void __launch_bounds__(kPlanThreads)
k_loss_join(const float2* __restrict__ row_loss, int64_t B, float value_coef, float* __restrict__ losses) {
    __shared__ float part[kPlanThreads];
    float p = 0.0f, v = 0.0f;
    for (int64_t b = threadIdx.x; b < B; b += kPlanThreads) {
        p += row_loss[b].x;
        v += row_loss[b].y;
    }
    p = block_sum(p, part);
    v = block_sum(v, part);
    if (threadIdx.x == 0) {
        losses[0] = p + value_coef * v;
        losses[1] = p;
        losses[2] = v;
    }
}

}  // namespace

extern "C" {

int64_t hg_policy_value_loss_workspace(int64_t B) {
    if (B <= 0) return 16;
    return 16 + (B + 1) * (int64_t)sizeof(int64_t) + B * (int64_t)sizeof(float2);
}

int hg_policy_value_loss(const void* logits, int type, int64_t N, const void* values, const int64_t* num_actions,
                         const void* targets, int target_type, int64_t width, const float* policy_weights,
                         const float* value_targets, const float* value_weights, int64_t B, float value_coef,
                         float loss_scale, float* losses, void* dlogits, void* dvalues, void* workspace,
                         void* stream) {
    if (N < 0 || B < 0 || width < 0 || !is_type(type) || !is_type(target_type) || B > (int64_t)1 << 31)
        return (int)hipErrorInvalidValue;
    if (!losses || !workspace || ((uintptr_t)workspace & 15)) return (int)hipErrorInvalidValue;
    if (B > 0 && (!values || !num_actions || !policy_weights || !value_targets || !value_weights || !dvalues))
        return (int)hipErrorInvalidValue;
    if (N > 0 && (!logits || !dlogits || (B > 0 && width > 0 && !targets))) return (int)hipErrorInvalidValue;
    if (B == 0 && N > 0) return (int)hipErrorInvalidValue;
    hipStream_t st = (hipStream_t)stream;
    float* sums = (float*)workspace;
    int64_t* offsets = (int64_t*)((uint8_t*)workspace + 16);
    float2* row_loss = (float2*)(offsets + B + 1);
    hipLaunchKernelGGL(k_loss_plan, dim3(1), dim3(kPlanThreads), 0, st, num_actions, B, width, policy_weights,
                       value_weights, offsets, sums);
    if (B > 0) {
        const int e = with_type(type, [&](auto tx) {
            using T = decltype(tx);
            return with_type(target_type, [&](auto tp) {
                using P = decltype(tp);
                hipLaunchKernelGGL((k_loss_rows<T, P>), dim3((unsigned)((B + kWaves - 1) / kWaves)), dim3(64 * kWaves),
                                   0, st, (const T*)logits, N, (const T*)values, offsets, sums, (const P*)targets,
                                   width, policy_weights, value_targets, value_weights, B, value_coef, loss_scale,
                                   row_loss, (T*)dlogits, (T*)dvalues);
                return (int)hipGetLastError();
            });
        });
        if (e) return e;
    }
    hipLaunchKernelGGL(k_loss_join, dim3(1), dim3(kPlanThreads), 0, st, row_loss, B, value_coef, losses);
    return (int)hipGetLastError();
}

}  // extern "C"
