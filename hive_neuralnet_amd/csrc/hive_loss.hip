// hive_loss.hip -- the training loss of a batch of positions, with its gradient.
//
// Position b has n[b] = clamp(num_actions[b], 0, width) legal moves; its
// logits x are n[b] values of one flat array, the positions one after the
// other, its searched policy pi the first n[b] values of row b of
// targets[B][width] (what lies beyond is not used).
//   lse_b = log sum exp x,  CE_b = sum pi (lse_b - x) over pi != 0
//   policy = sum w_b CE_b / sum w,      value = sum u_b (v_b - z_b)^2 / sum u
//   total = policy + c value
//   dx = s w_b / sum w (p mass_b - pi),  p = exp(x - lse_b), mass_b = sum pi
//   dv = s 2 c u_b / sum u (v_b - z_b)
// A position of weight zero, without moves, or whose logits are all -inf adds
// nothing and has a gradient of zeros; weights that sum to zero give a loss
// of zero.  A logit of -inf has p = 0; where pi says otherwise the loss is inf.
//
// Where a position's logits begin is a sum over the positions before it.
// Every block adds up what it needs itself: the counts before its first
// position and all the weights, up to kInline positions read in full, past
// them the sums of ranges of kRange positions that a first launch leaves.  Past
// kLookBack positions a second launch leaves each position's begin instead
// (10,000 positions of 2 moves: 13.2 us with it, 10.7 without; 20,000: 13.5,
// 12.2; 40,000: 15.4, 16.9).
//
// Lists of up to 256 moves (16 lanes a position) and up to 1,024 (a wave) are
// read once and held in registers (4,096 positions of up to 1,024 moves f32 13.8
// us, where the bytes at 5.4 TB/s are 4.6).  Longer ones are cut into slices, a block
// each, so that few positions fill the card too: one launch leaves each
// slice's largest logit and sums, the next joins a position's slices and
// writes the gradient from a second read.  All loads of a list, a slice's
// targets and the counts before it go out before any of them is waited for.
//
// Measured (MI355X): 16 positions 5 us, one launch; 2,048 of 60 moves on
// average 8 us, of which the second launch, the sum of the blocks' shares,
// takes 2 to 3 (the last block adding them: 17 in all, as every block's
// write-back for it has to come first); 65,521 of 85 in bf16 22.5 us: the sums
// before them 6.5 in two launches, the lists 15 to 16 (one load after the other,
// as conversions inside their branches make them: 19), of which the VALU is
// busy 12.5 (a third of the slots it works on hold a move; lists sorted by length
// among a block's waves: no gain).  192 x 85,834 bf16 logits 40.5 us: 20 for the
// slices, 4.9 TB/s, and 20 for the gradient, 6.5 TB/s, as its second read is
// partly in the caches (4 more with stores that go through them, 1 with the
// slices in their order, 2 with a look back in fours, 3 where every lane joined
// the list's 21 slices itself; slices of 8,192: 1.5 more, of 2,048: 6).
#include "hive_train.hpp"

namespace {

using namespace ht;

constexpr int64_t kInline = 4096, kRange = 256, kLookBack = 24 * 1024;
constexpr int kThreads = 256;
constexpr int kHeld = 16;  // logits of a position a lane holds
constexpr int64_t kSlice = 4096;  // moves of a slice of a long list

struct Range {
    int64_t moves;
    float policy, value;
};
struct Slice {  // of a long list: its largest logit, sum exp(x - top), sum pi, sum pi (x - top)
    float top, total, mass, cross;
};

struct Batch {
    const void *logits, *values, *targets;
    const int64_t* num_actions;
    const float *pw, *vt, *vw;
    int64_t N, width, B;
    float value_coef, loss_scale;
    Range* ranges;        // of `range` positions each; nullptr: up to kInline positions
    int64_t range;
    int64_t* begin;       // [B] where a position's logits begin, and the weights' sums (1 where they are 0);
    float* sums;          // nullptr: every block looks back itself
    float2* row_loss;     // [blocks or B]: shares of the policy loss and of the value loss
    float* losses;
    void *dlogits, *dvalues;
};

__device__ __forceinline__ int64_t clamp_count(int64_t n, int64_t width) {
    return n < 0 ? 0 : (n > width ? width : n);
}
// the sum over a wave's lanes, by the moves of group_join, 32 bits at a time
template <int kControl> __device__ __forceinline__ int64_t dpp(int64_t v) {
    const uint32_t lo = __builtin_amdgcn_mov_dpp((int)v, kControl, 0xF, 0xF, true);
    const uint32_t hi = __builtin_amdgcn_mov_dpp((int)(v >> 32), kControl, 0xF, 0xF, true);
    return (int64_t)((uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ int64_t wave_sum(int64_t v) {
    v += dpp<0xB1>(v);
    v += dpp<0x4E>(v);
    v += dpp<0x141>(v);
    v += dpp<0x140>(v);
    auto lo = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
    auto hi = __builtin_amdgcn_permlane16_swap((uint32_t)(v >> 32), (uint32_t)(v >> 32), false, false);
    v = (int64_t)((uint64_t)hi[0] << 32 | lo[0]) + (int64_t)((uint64_t)hi[1] << 32 | lo[1]);
    lo = __builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false);
    hi = __builtin_amdgcn_permlane32_swap((uint32_t)(v >> 32), (uint32_t)(v >> 32), false, false);
    return (int64_t)((uint64_t)hi[0] << 32 | lo[0]) + (int64_t)((uint64_t)hi[1] << 32 | lo[1]);
}

// What a block needs of the positions before its first one and of all.
struct Before {
    int64_t moves;       // of the positions before `first`
    float policy, value; // sums of all weights, 1 where they are 0
};
// (n positions of a thread, their loads together; the weights where they are wanted)
template <int threads, int n, bool kWeights = true> __device__ __forceinline__ Before look_back(const Batch& a, int64_t first) {
    __shared__ int64_t lds_moves[threads / 64];
    __shared__ float lds_policy[threads / 64], lds_value[threads / 64];
    int64_t moves = 0;
    float policy = 0.0f, value = 0.0f;
    if (a.ranges) {
        const int64_t all = (a.B + a.range - 1) / a.range, mine = first / a.range;
        for (int64_t i = threadIdx.x; i < all; i += threads) {
            const Range r = a.ranges[i];
            moves += i < mine ? r.moves : 0;
            policy += r.policy;
            value += r.value;
        }
        for (int64_t i = mine * a.range + threadIdx.x; i < first; i += threads)
            moves += clamp_count(a.num_actions[i], a.width);
    } else {
        const int last = (int)a.B - 1;
        for (int i = threadIdx.x; i <= last; i += n * threads) {
            int64_t c[n];
            float p[n], v[n];
#pragma unroll
            for (int k = 0; k < n; k++) {
                const int at = min(i + k * threads, last);
                c[k] = a.num_actions[at];
                p[k] = kWeights ? a.pw[at] : 0.0f;
                v[k] = kWeights ? a.vw[at] : 0.0f;
            }
#pragma unroll
            for (int k = 0; k < n; k++) {
                const int at = i + k * threads;
                moves += at < first ? clamp_count(c[k], a.width) : 0;
                policy += at <= last ? p[k] : 0.0f;
                value += at <= last ? v[k] : 0.0f;
            }
        }
    }
    moves = wave_sum(moves);
    if (kWeights) {
        policy = group_sum<64>(policy);
        value = group_sum<64>(value);
    }
    if ((threadIdx.x & 63) == 0) {
        lds_moves[threadIdx.x >> 6] = moves;
        if (kWeights) {
            lds_policy[threadIdx.x >> 6] = policy;
            lds_value[threadIdx.x >> 6] = value;
        }
    }
    __syncthreads();
    Before r = {0, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < threads / 64; i++) {
        r.moves += lds_moves[i];
        if (kWeights) {
            r.policy += lds_policy[i];
            r.value += lds_value[i];
        }
    }
    if (!(r.policy > 0.0f)) r.policy = 1.0f;
    if (!(r.value > 0.0f)) r.value = 1.0f;
    return r;
}

// the sums of a range, a block each
__global__ void __launch_bounds__(kRange) k_loss_ranges(Batch a) {
    __shared__ int64_t lds_moves[kRange / 64];
    __shared__ float lds[2][kRange / 64];
    int64_t moves = 0;
    float policy = 0.0f, value = 0.0f;
    const int64_t first = (int64_t)blockIdx.x * a.range, end = min(a.B, first + a.range);
    for (int64_t i = first + threadIdx.x; i < end; i += kRange) {
        moves += clamp_count(a.num_actions[i], a.width);
        policy += a.pw[i];
        value += a.vw[i];
    }
    moves = wave_sum(moves);
    policy = group_sum<64>(policy);
    value = group_sum<64>(value);
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
        lds_moves[wave] = moves;
        lds[0][wave] = policy;
        lds[1][wave] = value;
    }
    __syncthreads();
    if (threadIdx.x != 0) return;
    Range r = {0, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kRange / 64; i++) {
        r.moves += lds_moves[i];
        r.policy += lds[0][i];
        r.value += lds[1][i];
    }
    a.ranges[blockIdx.x] = r;
}

// begin and sums, a range a block
__global__ void __launch_bounds__(kRange) k_loss_begins(Batch a) {
    __shared__ int64_t lds[2][kRange / 64];
    const int64_t first = (int64_t)blockIdx.x * a.range, end = min(a.B, first + a.range);
    const Before before = look_back<kRange, 4>(a, first);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t begin = before.moves;
    int turn = 0;
    for (int64_t base = first; base < end; base += kRange, turn ^= 1) {
        const int64_t b = base + threadIdx.x, n = b < end ? clamp_count(a.num_actions[b], a.width) : 0;
        int64_t upto = n;
        for (int o = 1; o < 64; o <<= 1) {
            const int64_t v = __shfl_up(upto, o, 64);
            upto += lane >= o ? v : 0;
        }
        if (lane == 63) lds[turn][wave] = upto;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kRange / 64; i++) upto += i < wave ? lds[turn][i] : 0;
        if (b < end) a.begin[b] = begin + upto - n;
#pragma unroll
        for (int i = 0; i < kRange / 64; i++) begin += lds[turn][i];
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        a.sums[0] = before.policy;
        a.sums[1] = before.value;
    }
}

// elements at .. at + n - 1 of an array of `all`; what lies past its end is not read (its values: anything)
template <typename T, int n>
__device__ __forceinline__ void load_flat(const T* p, int64_t at, int64_t all, float v[n]) {
    typedef T vec __attribute__((ext_vector_type(n), aligned(sizeof(T))));
    if (at + n <= all) {
        const vec q = *(const vec*)(p + at);
#pragma unroll
        for (int i = 0; i < n; i++) v[i] = to_f32<T>(q[i]);
    } else {
        skipped();
#pragma unroll
        for (int i = 0; i < n; i++) v[i] = at + i < all ? to_f32<T>(p[at + i]) : 0.0f;
    }
}

// what a position holds besides its list, read before the list is waited for
template <typename T> struct Scalars {
    float w, u, target;  // policy weight, value weight, the value's target
    T value;
};
template <typename T> __device__ __forceinline__ Scalars<T> scalars_of(const Batch& a, int64_t b) {
    return Scalars<T>{a.pw[b], a.vw[b], a.vt[b], ((const T*)a.values)[b]};
}
// the value loss of position b, and its gradient
template <typename T>
__device__ __forceinline__ float value_loss(const Batch& a, int64_t b, const Scalars<T>& s, float weights) {
    const float u = s.u / weights, off = to_f32(s.value) - s.target;
    const bool used = u != 0.0f;
    ((T*)a.dvalues)[b] = from_f32<T>(used ? 2.0f * a.value_coef * u * off * a.loss_scale : 0.0f);
    return used ? u * off * off : 0.0f;
}
__device__ __forceinline__ void store_losses(const Batch& a, float policy, float value) {
    a.losses[0] = policy + a.value_coef * value;
    a.losses[1] = policy;
    a.losses[2] = value;
}
// s + p z, s where p is 0 whatever z is
__device__ __forceinline__ float plus(float s, float p, float z) { return p != 0.0f ? fmaf(p, z, s) : s; }
// Rounding z log2 e once puts the result up to |z| u of itself off (u = 2^-24; 8 u at z = -10, 58 u at -60), under 1 u of
// the largest of a list.  An exact product would be two more operations a slot, in kernels that the VALU bounds.
__device__ __forceinline__ float exp_(float z) { return __builtin_amdgcn_exp2f(z * 1.44269504f); }

// gradients of zero for the logits that no position has
template <typename T> __device__ __forceinline__ void clear_rest(const Batch& a, int64_t from, int tid, int threads) {
    for (int64_t i = from + tid; i < a.N; i += threads) ((T*)a.dlogits)[i] = from_f32<T>(0.0f);
}

// kLanes lanes a position, its list held in registers
template <typename T, typename P, int kLanes>
__global__ void __launch_bounds__(kThreads) k_loss_held(Batch a) {
    constexpr int n = 4, vecs = kHeld / n, rows = kThreads / kLanes;
    const int lane = threadIdx.x % kLanes, mine = threadIdx.x / kLanes;
    const int64_t first = (int64_t)blockIdx.x * rows, b = first + mine;
    int64_t lo;
    int count = 0;
    float policy_sum, value_sum, policy = 0.0f, value = 0.0f;
    const int64_t here = min(b, a.B - 1);
    const int64_t listed = a.num_actions[here];
    const Scalars<T> own = scalars_of<T>(a, here);
    if (a.begin) {
        lo = a.begin[here];
        policy_sum = a.sums[0];
        value_sum = a.sums[1];
        count = (int)clamp_count(listed, a.width);
    } else {
        const Before before = look_back<kThreads, 4>(a, first);
        policy_sum = before.policy;
        value_sum = before.value;
        lo = before.moves;
#pragma unroll
        for (int i = 0; i < rows; i++) {  // every lane group adds the counts before its own
            const int c = first + i < a.B ? (int)clamp_count(a.num_actions[first + i], a.width) : 0;
            lo += i < mine ? c : 0;
            count = i == mine ? c : count;
        }
    }
    if (b < a.B) {
        const int64_t left = a.N - lo;
        count = left <= 0 ? 0 : (left < count ? (int)left : count);
        // a position of weight 0 is taken as one without moves, but for its gradient's zeros
        const float share = own.w / policy_sum;
        const int live = own.w != 0.0f ? count : 0;
        // a step that no list of the wave reaches is passed by
        bool reached[vecs];
#pragma unroll
        for (int k = 0; k < vecs; k++) reached[k] = __any(k * kLanes * n < live);
        float x[vecs][n], pi[vecs][n];
        const int64_t row = b * a.width;
        const int most = live > 0 ? (live + n - 1) / n * n : n;
        if (__all(lo + most <= a.N && row + most <= a.B * a.width)) {
            // no vector passes the arrays' ends: all loads at once, a lane past its list's end at the list's start
            typedef T tvec __attribute__((ext_vector_type(n), aligned(sizeof(T))));
            typedef P pvec __attribute__((ext_vector_type(n), aligned(sizeof(P))));
            tvec raw[vecs];
            pvec raw_pi[vecs];
#pragma unroll
            for (int k = 0; k < vecs; k++) {
                if (!reached[k]) break;
                const int c = (lane + k * kLanes) * n, at = c < live ? c : 0;
                raw[k] = *(const tvec*)((const T*)a.logits + lo + at);
                raw_pi[k] = *(const pvec*)((const P*)a.targets + row + at);
            }
#pragma unroll
            for (int k = 0; k < vecs; k++)
#pragma unroll
                for (int i = 0; i < n; i++) {
                    x[k][i] = to_f32<T>(raw[k][i]);
                    pi[k][i] = to_f32<P>(raw_pi[k][i]);
                }
        } else {
#pragma unroll
            for (int k = 0; k < vecs; k++) {
                const int c = (lane + k * kLanes) * n;
                if (c < live) {
                    load_flat<T, n>((const T*)a.logits, lo + c, a.N, x[k]);
                    load_flat<P, n>((const P*)a.targets, row + c, a.B * a.width, pi[k]);
                }
            }
        }
        float top = -INFINITY;
#pragma unroll
        for (int k = 0; k < vecs; k++) {
            if (!reached[k]) break;
#pragma unroll
            for (int i = 0; i < n; i++) {
                const bool in = (lane + k * kLanes) * n + i < live;
                x[k][i] = in ? x[k][i] : -INFINITY;
                pi[k][i] = in ? pi[k][i] : 0.0f;
                top = fmaxf(top, x[k][i]);  // passes a NaN by: it comes through the sums
            }
        }
        top = group_join<kLanes>(top, [](float p, float q) { return fmaxf(p, q); });
        const float shift = top == -INFINITY ? 0.0f : top;
        float total = 0.0f, mass = 0.0f, cross = 0.0f;
#pragma unroll
        for (int k = 0; k < vecs; k++) {
            if (!reached[k]) break;
#pragma unroll
            for (int i = 0; i < n; i++) {
                const float z = x[k][i] - shift;
                mass += pi[k][i];
                cross = plus(cross, pi[k][i], z);
                x[k][i] = exp_(z);
                total += x[k][i];
            }
        }
        total = group_sum<kLanes>(total);
        mass = group_sum<kLanes>(mass);
        cross = group_sum<kLanes>(cross);
        const bool used = total != 0.0f;  // some logit above -inf, or a NaN
        const float scale = used ? share * a.loss_scale : 0.0f, p_scale = used ? mass / total * scale : 0.0f;
#pragma unroll
        for (int k = 0; k < vecs; k++) {
            const int c = (lane + k * kLanes) * n;
            if (c >= count) break;
#pragma unroll
            for (int i = 0; i < n; i++) x[k][i] = fmaf(x[k][i], p_scale, -(pi[k][i] * scale));
            if (!used) {  // whatever the target holds, or nothing was read
                skipped();
#pragma unroll
                for (int i = 0; i < n; i++) x[k][i] = 0.0f;
            }
            store_some<T, n>((T*)a.dlogits + lo + c, count - c, x[k]);
        }
        if (b == a.B - 1) clear_rest<T>(a, lo + count, lane, kLanes);
        if (lane == 0) {
            policy = used ? (logf(total) * mass - cross) * share : 0.0f;
            value = value_loss<T>(a, b, own, value_sum);
        }
    }
    __shared__ float lds[2][kThreads / 64];
    policy = group_sum<64>(policy);
    value = group_sum<64>(value);
    if ((threadIdx.x & 63) == 0) {
        lds[0][threadIdx.x >> 6] = policy;
        lds[1][threadIdx.x >> 6] = value;
    }
    __syncthreads();
    if (threadIdx.x != 0) return;
    policy = value = 0.0f;
#pragma unroll
    for (int i = 0; i < kThreads / 64; i++) {
        policy += lds[0][i];
        value += lds[1][i];
    }
    if (gridDim.x == 1) store_losses(a, policy, value);
    else a.row_loss[blockIdx.x] = make_float2(policy, value);
}

// ---- long lists: block (slice, position) -------------------------------------

// what k_loss_begins left, or the block's own
template <bool kWeights> __device__ __forceinline__ Before begin_of(const Batch& a, int64_t b) {
    return a.begin ? Before{a.begin[b], a.sums[0], a.sums[1]} : look_back<kThreads, 1, kWeights>(a, b);
}
// the slice of a position: `len` elements from element `from` of its list of `count`
struct Cut {
    int64_t count, from;
    int len;
};
__device__ __forceinline__ Cut cut_of(int64_t count, int64_t slice, uint32_t index) {
    const int64_t from = min(count, (int64_t)index * slice);
    return Cut{count, from, (int)min(slice, count - from)};
}

// A thread's share of a piece of kSlice elements, kSlice / kThreads of them in
// vectors of n, of an array of `len` (past its end: none), as they are read.
template <typename E, int n> struct Piece {
    static constexpr int vecs = (int)kSlice / kThreads / n;
    typedef E vec __attribute__((ext_vector_type(n), aligned(sizeof(E))));
    vec v[vecs];
    __device__ __forceinline__ void load(const E* p, int from, int len, E none) {
#pragma unroll
        for (int k = 0; k < vecs; k++) {
            const int c = from + (threadIdx.x + k * kThreads) * n;
            if (c + n <= len) {
                v[k] = *(const vec*)(p + c);
            } else {
                skipped();
#pragma unroll
                for (int i = 0; i < n; i++) v[k][i] = c + i < len ? p[c + i] : none;
            }
        }
    }
};

// store_some past the caches: they hold what other slices have still to read
template <typename T, int n> __device__ __forceinline__ void store_past(T* p, int live, const float v[n]) {
    typedef T vec __attribute__((ext_vector_type(n), aligned(sizeof(T))));
    if (live >= n) {
        vec q;
#pragma unroll
        for (int i = 0; i < n; i++) q[i] = from_f32<T>(v[i]);
        __builtin_nontemporal_store(q, (vec*)p);
    } else {
        skipped();
        store_some<T, n>(p, live, v);
    }
}

// the n slices of a list as one, by a wave: a lane takes every 64th, all bring theirs to the largest logit
__device__ __forceinline__ Slice join(const Slice* slices, int n) {
    const int lane = threadIdx.x & 63;
    float top = -INFINITY;
    for (int i = lane; i < n; i += 64) top = fmaxf(top, slices[i].top);
    top = group_join<64>(top, [](float p, float q) { return fmaxf(p, q); });
    const float shift = top == -INFINITY ? 0.0f : top;
    Slice s = {top, 0.0f, 0.0f, 0.0f};
    for (int i = lane; i < n; i += 64) {
        const Slice q = slices[i];
        const float down = q.top - shift;
        s.total = fmaf(q.total, exp_(down), s.total);
        s.mass += q.mass;
        s.cross += plus(q.cross, q.mass, down);
    }
    s.total = group_sum<64>(s.total);
    s.mass = group_sum<64>(s.mass);
    s.cross = group_sum<64>(s.cross);
    return s;
}

template <typename T, typename P>
__global__ void __launch_bounds__(kThreads)
k_loss_slices(Batch a, int64_t first, int64_t slice, Slice* __restrict__ slices) {
    constexpr int n = Vector<T>::n;
    const int64_t b = first + blockIdx.y;
    // where the logits begin takes a look at the positions before: the first targets are read meanwhile
    Cut cut = cut_of(min(clamp_count(a.num_actions[b], a.width), a.N), slice, blockIdx.x);
    const P* targets = (const P*)a.targets + b * a.width + cut.from;
    Piece<P, n> pi;
    pi.load(targets, 0, cut.len, (P)0.0f);
    const int64_t lo = min(a.N, begin_of<false>(a, b).moves);
    const int listed = cut.len;
    cut = cut_of(min(cut.count, a.N - lo), slice, blockIdx.x);
    const T* logits = (const T*)a.logits + lo + cut.from;
    const int len = cut.len;
    if (len != listed) pi.load(targets, 0, len, (P)0.0f);  // the logits' end cuts the list
    // one pass: each thread's largest logit so far (fmaxf passes a NaN by: it comes through the sums), its sums brought
    // to a new one as it comes
    float top = -INFINITY, total = 0.0f, mass = 0.0f, cross = 0.0f;
    for (int at = 0; at < len; at += kSlice) {
        Piece<T, n> x;
        if (at) pi.load(targets, at, len, (P)0.0f);
        x.load(logits, at, len, from_f32<T>(-INFINITY));
        float most = top;
#pragma unroll
        for (int k = 0; k < x.vecs; k++)
#pragma unroll
            for (int i = 0; i < n; i++) most = fmaxf(most, to_f32<T>(x.v[k][i]));
        if (most != top) {
            total *= exp_(top - most);  // 0 * 0 where this is the first logit above -inf
            cross = plus(cross, mass, top - most);
            top = most;
        }
        const float shift = top == -INFINITY ? 0.0f : top;
#pragma unroll
        for (int k = 0; k < x.vecs; k++)
#pragma unroll
            for (int i = 0; i < n; i++) {
                const float z = to_f32<T>(x.v[k][i]) - shift;
                const float p = to_f32<P>(pi.v[k][i]);
                total += exp_(z);
                mass += p;
                cross = plus(cross, p, z);
            }
    }
    // the block's largest, the sums brought to it and added
    __shared__ float lds[4][kThreads / 64];
    const int wave = threadIdx.x >> 6;
    float most = group_join<64>(top, [](float p, float q) { return fmaxf(p, q); });
    if ((threadIdx.x & 63) == 0) lds[0][wave] = most;
    __syncthreads();
    most = lds[0][0];
#pragma unroll
    for (int i = 1; i < kThreads / 64; i++) most = fmaxf(most, lds[0][i]);
    const float down = most == -INFINITY ? 0.0f : top - most;
    cross = plus(cross, mass, down);
    total = group_sum<64>(total * exp_(down));
    mass = group_sum<64>(mass);
    cross = group_sum<64>(cross);
    if ((threadIdx.x & 63) == 0) {
        lds[1][wave] = total;
        lds[2][wave] = mass;
        lds[3][wave] = cross;
    }
    __syncthreads();
    if (threadIdx.x != 0) return;
    Slice s = {most, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kThreads / 64; i++) {
        s.total += lds[1][i];
        s.mass += lds[2][i];
        s.cross += lds[3][i];
    }
    slices[b * gridDim.x + blockIdx.x] = s;
}

template <typename T, typename P>
__global__ void __launch_bounds__(kThreads)
k_loss_gradient(Batch a, int64_t first, int64_t slice, const Slice* __restrict__ slices) {
    constexpr int n = Vector<T>::n;
    // the slices that were read last come first, on the chiplet that read them: its cache holds some of them yet
    const uint32_t linear = blockIdx.y * gridDim.x + blockIdx.x, whole = gridDim.x * gridDim.y & ~7u;
    const uint32_t turned = linear < whole ? whole - 8 - (linear & ~7u) + (linear & 7u) : linear;
    const uint32_t index = turned % gridDim.x;
    const int64_t b = first + turned / gridDim.x;
    Cut cut = cut_of(min(clamp_count(a.num_actions[b], a.width), a.N), slice, index);
    const P* targets = (const P*)a.targets + b * a.width + cut.from;
    Piece<P, n> pi;
    pi.load(targets, 0, cut.len, (P)0.0f);
    const Before before = begin_of<true>(a, b);
    const int64_t lo = min(a.N, before.moves);
    cut = cut_of(min(cut.count, a.N - lo), slice, index);
    const T* logits = (const T*)a.logits + lo + cut.from;
    T* dlogits = (T*)a.dlogits + lo + cut.from;
    const int len = cut.len;
    Piece<T, n> x;
    x.load(logits, 0, len, (T)0.0f);
    const Slice s = join(slices + b * gridDim.x, gridDim.x);
    const Scalars<T> own = scalars_of<T>(a, b);
    const float share = own.w / before.policy;
    const bool used = own.w != 0.0f && s.total != 0.0f;
    const float shift = s.top == -INFINITY ? 0.0f : s.top;
    const float scale = used ? share * a.loss_scale : 0.0f, p_scale = used ? s.mass / s.total * scale : 0.0f;
    for (int at = 0; at < len; at += kSlice) {
        if (at) {
            pi.load(targets, at, len, (P)0.0f);
            x.load(logits, at, len, (T)0.0f);
        }
#pragma unroll
        for (int k = 0; k < x.vecs; k++) {
            const int c = at + (threadIdx.x + k * kThreads) * n;
            float dx[n];
#pragma unroll
            for (int i = 0; i < n; i++) {
                const float p = exp_(to_f32<T>(x.v[k][i]) - shift);
                dx[i] = used ? fmaf(p, p_scale, -(to_f32<P>(pi.v[k][i]) * scale)) : 0.0f;
            }
            store_past<T, n>(dlogits + c, len - c, dx);
        }
    }
    if (b == a.B - 1 && index == 0) clear_rest<T>(a, lo + cut.count, threadIdx.x, kThreads);
    if (threadIdx.x == 0 && index == 0)
        a.row_loss[b] = make_float2(used ? (logf(s.total) * s.mass - s.cross) * share : 0.0f,
                                    value_loss<T>(a, b, own, before.value));
}

__global__ void __launch_bounds__(1024) k_loss_join(Batch a, int64_t parts) {
    __shared__ float lds[2][16];
    float p = 0.0f, v = 0.0f;
    for (int64_t i = threadIdx.x; i < parts; i += 1024) {
        const float2 r = a.row_loss[i];
        p += r.x;
        v += r.y;
    }
    p = group_sum<64>(p);
    v = group_sum<64>(v);
    if ((threadIdx.x & 63) == 0) {
        lds[0][threadIdx.x >> 6] = p;
        lds[1][threadIdx.x >> 6] = v;
    }
    __syncthreads();
    if (threadIdx.x != 0) return;
    p = v = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        p += lds[0][i];
        v += lds[1][i];
    }
    store_losses(a, p, v);
}

constexpr int64_t kShort = 16 * kHeld, kMiddle = 64 * kHeld;  // widths whose lists 16 lanes, a wave hold
constexpr int64_t kMaxBatch = ((int64_t)1 << 26) - 4;  // a wave a position: a grid holds under 2^32 threads
constexpr int64_t kGridRows = 32768;  // positions of a launch over slices: a grid has 65,535 rows at most

// ranges of 256 positions, or 1,024 of them: every block adds up all that come before its own
inline int64_t range_of(int64_t B) { return kRange * ((B + 1024 * kRange - 1) / (1024 * kRange)); }
inline int64_t ranges_of(int64_t B) { return B <= kInline ? 0 : (B + range_of(B) - 1) / range_of(B); }
// Slices of a list: of 4,096 moves, or 256 of them.  They depend on the width
// alone, so that a position's gradient is the same in every batch.
inline int64_t slices_of(int64_t width) {
    const int64_t n = (width + kSlice - 1) / kSlice;
    return n < 256 ? n : 256;
}
// float2 per block or position, then the slices
inline int64_t losses_of(int64_t B) { return (B + 1) / 2 * 2; }

}  // namespace

extern "C" {

int64_t hg_policy_value_loss_workspace(int64_t B, int64_t width) {
    if (B <= 0) return 16;
    const int64_t slices = width > kMiddle ? B * slices_of(width) : 0;
    return ranges_of(B) * (int64_t)sizeof(Range) + losses_of(B) * (int64_t)sizeof(float2) +
           slices * (int64_t)sizeof(Slice) + B * (int64_t)sizeof(int64_t) + 2 * (int64_t)sizeof(float);
}

int hg_policy_value_loss(const void* logits, int type, int64_t N, const void* values, const int64_t* num_actions,
                         const void* targets, int target_type, int64_t width, const float* policy_weights,
                         const float* value_targets, const float* value_weights, int64_t B, float value_coef,
                         float loss_scale, float* losses, void* dlogits, void* dvalues, void* workspace,
                         void* stream) {
    if (N < 0 || B < 0 || width < 0 || !is_type(type) || !is_type(target_type) || B > kMaxBatch ||
        width > (int64_t)1 << 31)
        return (int)hipErrorInvalidValue;
    if (!losses || !workspace || ((uintptr_t)workspace & 15)) return (int)hipErrorInvalidValue;
    if (B > 0 && (!values || !num_actions || !policy_weights || !value_targets || !value_weights || !dvalues))
        return (int)hipErrorInvalidValue;
    if (N > 0 && (!logits || !dlogits || (B > 0 && width > 0 && !targets))) return (int)hipErrorInvalidValue;
    if (B == 0 && N > 0) return (int)hipErrorInvalidValue;
    hipStream_t st = (hipStream_t)stream;
    Range* ranges = (Range*)workspace;
    Batch a;
    a.logits = logits;
    a.values = values;
    a.targets = targets;
    a.num_actions = num_actions;
    a.pw = policy_weights;
    a.vt = value_targets;
    a.vw = value_weights;
    a.N = N;
    a.width = width;
    a.B = B;
    a.value_coef = value_coef;
    a.loss_scale = loss_scale;
    a.ranges = ranges_of(B) ? ranges : nullptr;
    a.range = B > 0 ? range_of(B) : kRange;
    a.row_loss = (float2*)(ranges + ranges_of(B));
    a.losses = losses;
    a.dlogits = dlogits;
    a.dvalues = dvalues;
    Slice* slices = (Slice*)(a.row_loss + losses_of(B));
    a.begin = (int64_t*)(slices + (width > kMiddle ? B * slices_of(width) : 0));
    a.sums = (float*)(a.begin + B);
    if (a.ranges) hipLaunchKernelGGL(k_loss_ranges, dim3((unsigned)ranges_of(B)), dim3(kRange), 0, st, a);
    // past that the blocks' look back would cost more than the launch (a long list has a block a slice)
    if (width <= kMiddle ? B > kLookBack : B > kThreads)
        hipLaunchKernelGGL(k_loss_begins, dim3((unsigned)((B + a.range - 1) / a.range)), dim3(kRange), 0, st, a);
    else
        a.begin = nullptr;
    int64_t parts = 0;
    if (B > 0)
        with_type(type, [&](auto tx) {
            using T = decltype(tx);
            return with_type(target_type, [&](auto tp) {
                using P = decltype(tp);
                if (width <= kMiddle) {
                    const int rows = width <= kShort ? kThreads / 16 : kThreads / 64;
                    parts = (B + rows - 1) / rows;
                    auto f = width <= kShort ? k_loss_held<T, P, 16> : k_loss_held<T, P, 64>;
                    hipLaunchKernelGGL(f, dim3((unsigned)parts), dim3(kThreads), 0, st, a);
                } else {
                    const int64_t cuts = slices_of(width);
                    const int64_t slice = ((width + cuts - 1) / cuts + 7) / 8 * 8;
                    parts = B;
                    for (int64_t b = 0; b < B; b += kGridRows) {
                        const dim3 grid((unsigned)cuts, (unsigned)(B - b < kGridRows ? B - b : kGridRows));
                        hipLaunchKernelGGL((k_loss_slices<T, P>), grid, dim3(kThreads), 0, st, a, b, slice, slices);
                        hipLaunchKernelGGL((k_loss_gradient<T, P>), grid, dim3(kThreads), 0, st, a, b, slice, slices);
                    }
                }
                return 0;
            });
        });
    if (parts != 1 || width > kMiddle)
        hipLaunchKernelGGL(k_loss_join, dim3(1), dim3(1024), 0, st, a, parts);
    return (int)hipGetLastError();
}

}  // extern "C"
