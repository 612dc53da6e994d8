// hive_sample.hip -- a slot of each row of logits, drawn from a given number.
//
// Of a row's live slots (its first num_actions, those whose logit is above
// -inf) in order of falling logits, ties by rising slots: the first top_k; of
// these the fewest first ones whose weights exp((x - max) / T) add up to top_p of
// theirs; of these the ones whose weight is at least min_p.  The slot drawn is the
// first, in order of the slots, at which the running sum of the weights kept
// passes u times their whole.  T not above 0: the largest logit's first slot.
//
// A border that a running sum just misses decides a move, so sums must not
// depend on how they are cut up: weights are rounded once, to whole multiples of
// 2^-43 (rows up to 1,024) or 2^-42 (longer ones, up to 2^20) of the largest, and
// added exactly, in a double's 53 bits or in 64-bit integers, in any order.
//
// Cuts are (key, count): all slots above the key and the first `count` that
// equal it; keys are the logits' bits in unsigned order, 0 for what is not
// live (NaN, too).  Rows up to 1,024 slots are held by a wave's registers, and a
// cut is found by pivots.  Longer rows are read by a block: once for the largest
// (each thread's own, of which the top_k-th bounds the row's), once more for the
// weights of each 11-bit digit of the keys with top_p alone, and once for the slots that these or
// min_p leave, which a wave draws from where they are 1,024 or less.  Where they
// are more, cuts are found by all three digits of the key.
//
// Measured (MI355X): 65,521 lists of up to 256 slots with top_p 53 us (a wave each; the sums and pivots of a cut bound
// it, not the 35 MB), 192 rows of 85,834 bfloat16 with top_k and top_p 37 us, one row of as many float32 with
// min_p 22 where at most 1,024 slots pass it, 155 with a top_p of 0.9, whose thousands of slots take four passes of weights:
// 279,000 vector instructions, 52 a key and pass of 64, which one compute unit issues for 116 us of these (the LDS atomics'
// conflicts hold it for 4; 233 where each cut began at its first digit).  One short list 3 us, 5.5 with the call.
#include <cmath>

#include "hive_train.hpp"

namespace {

using namespace ht;

constexpr int64_t kMaxRows = 1 << 25, kMaxLongRows = 1 << 21, kMaxWidth = 1 << 20;  // a launch has under 2^32 threads
constexpr int kHeld = 1024;  // slots of a row that a wave holds
constexpr double kWaveOne = 0x1p43, kBlockOne = 0x1p42;

struct Settings {
    const void* logits;
    int64_t stride, rows;
    int width;
    const int64_t* counts;
    const float *uniforms, *temperatures, *top_ps, *min_ps;
    const int64_t* top_ks;
    double temperature, top_p, min_p;
    int64_t top_k;
    int64_t* actions;
    float* log_probs;
};

// a row's own settings
struct Row {
    int n;
    int64_t k;  // 0: all
    double t, p, min_p, u;
    double scale;  // log2(e) / t
    bool greedy, cut_p;
};
__device__ __forceinline__ Row row_of(const Settings& s, int64_t b) {
    Row r;
    const int64_t n = s.counts ? s.counts[b] : s.width;
    r.n = (int)(n < 0 ? 0 : n > s.width ? s.width : n);
    r.t = s.temperatures ? (double)s.temperatures[b] : s.temperature;
    r.p = s.top_ps ? (double)s.top_ps[b] : s.top_p;
    r.min_p = s.min_ps ? (double)s.min_ps[b] : s.min_p;
    r.min_p = r.min_p > 0.0 ? fmin(r.min_p, 1.0) : 0.0;  // the largest always stays; NaN: 0
    const int64_t k = s.top_ks ? s.top_ks[b] : s.top_k;
    r.k = k > 0 ? k : 0;
    r.u = (double)s.uniforms[b];
    r.u = r.u > 0.0 ? r.u : 0.0;  // NaN: 0
    r.greedy = !(r.t > 0.0);  // NaN, too
    r.scale = 1.4426950408889634 / r.t;
    r.cut_p = r.p < 1.0;  // NaN: no cut
    return r;
}

// the logits' order as unsigned numbers, both zeros alike; 0: not live
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    const uint32_t k = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
    return x > -__builtin_inff() ? k : 0;
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}
// exp((x - top) / t) = 2^(scale (x - top)), scale = log2(e) / t, of n slots; 1 for x = top whatever it is, 0 for what is not
// live.  A series of 2^f, |f| <= 1/2, to f^11: 2^-47 of the whole left out, with the rounding of scale and of the product
// under 2^-45, a weight's own rounding.  Slot by slot within a term, so that its coefficient is loaded once.
template <int n>
__device__ __forceinline__ void weights_of(const uint32_t (&key)[n], uint32_t top, double scale, double (&w)[n]) {
    constexpr double term[12] = {1.0 / 39916800.0, 1.0 / 3628800.0, 1.0 / 362880.0, 1.0 / 40320.0, 1.0 / 5040.0, 1.0 / 720.0,
                                 1.0 / 120.0,      1.0 / 24.0,      1.0 / 6.0,      0.5,           1.0,          1.0};
    const double x_top = (double)value_of(top);
    double f[n];
    int exponent[n];
#pragma unroll
    for (int i = 0; i < n; i++) {
        // NaN (a logit below one of inf at a temperature of inf) and -inf: 0
        const double y = fmax(((double)value_of(key[i]) - x_top) * scale, -1200.0), whole = rint(y);
        f[i] = (y - whole) * 0.6931471805599453;
        exponent[i] = (int)whole;
        w[i] = term[0];
    }
#pragma unroll
    for (int k = 1; k < 12; k++)
#pragma unroll
        for (int i = 0; i < n; i++) w[i] = fma(w[i], f[i], term[k]);
#pragma unroll
    for (int i = 0; i < n; i++) {
        w[i] = ldexp(w[i], exponent[i]);
        w[i] = key[i] == top ? 1.0 : key[i] ? w[i] : 0.0;
    }
}
__device__ __forceinline__ double weight_of(uint32_t key, uint32_t top, double scale) {
    const uint32_t one[1] = {key};
    double w[1];
    weights_of<1>(one, top, scale, w);
    return w[0];
}
// The logarithm of key's weight over `all` of them: log m = 2 z (1 + z^2 / 3 + ...), z = (m - 1) / (m + 1), m between the roots
// of 1/2 and 2: 2^-27 of it left out.
__device__ __forceinline__ double log_share(uint32_t key, uint32_t top, double scale, double all) {
    int e;
    double m = frexp(all, &e);
    if (m < 0.7071067811865476) {
        m *= 2.0;
        e--;
    }
    const double z = (m - 1.0) / (m + 1.0), q = z * z;
    const double log_all = 2.0 * z * fma(q, fma(q, fma(q, fma(q, 1.0 / 9.0, 1.0 / 7.0), 0.2), 1.0 / 3.0), 1.0) + e * 0.6931471805599453;
    return (key == top ? 0.0 : ((double)value_of(key) - (double)value_of(top)) * (scale * 0.6931471805599453)) - log_all;
}
// keys of slots c .. c + 3 of n
template <typename T> __device__ __forceinline__ void load_keys(const T* row, int c, int n, uint32_t key[4]) {
    typedef T vec __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    if (c + 4 <= n) {
        const vec v = *(const vec*)(row + c);
#pragma unroll
        for (int e = 0; e < 4; e++) key[e] = key_of(to_f32<T>(v[e]));
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) key[e] = c + e < n ? key_of(to_f32<T>(row[c + e])) : 0;
    }
}

// v of the lane that DPP control `kControl` names, 0 where it names none or its row of 16 is not in kRows
template <int kControl, int kRows = 0xF> __device__ __forceinline__ int moved_word(int v) {
    if constexpr (kRows == 0xF) return __builtin_amdgcn_mov_dpp(v, kControl, 0xF, 0xF, true);
    else return __builtin_amdgcn_update_dpp(0, v, kControl, kRows, 0xF, false);
}
template <int kControl, int kRows = 0xF, typename V> __device__ __forceinline__ V moved(V v) {
    if constexpr (sizeof(V) == 8) {
        const uint64_t b = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = (uint32_t)moved_word<kControl, kRows>((int)(uint32_t)b);
        const uint32_t hi = (uint32_t)moved_word<kControl, kRows>((int)(uint32_t)(b >> 32));
        return __builtin_bit_cast(V, (uint64_t)hi << 32 | lo);
    } else {
        return __builtin_bit_cast(V, moved_word<kControl, kRows>(__builtin_bit_cast(int, v)));
    }
}
// the sum of the lanes up to this one: within rows of 16, then the rows before
template <typename V> __device__ __forceinline__ V wave_scan(V v) {
    v += moved<0x111>(v);       // row_shr 1, 2, 4, 8
    v += moved<0x112>(v);
    v += moved<0x114>(v);
    v += moved<0x118>(v);
    v += moved<0x142, 0xA>(v);  // the end of row 0 to row 1, of row 2 to row 3
    v += moved<0x143, 0xC>(v);  // the end of row 1 to rows 2 and 3
    return v;
}
template <typename V> __device__ __forceinline__ V from_lane(V v, int lane) {  // the same for all lanes
    if constexpr (sizeof(V) == 8) {
        const uint64_t b = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, lane);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), lane);
        return __builtin_bit_cast(V, (uint64_t)hi << 32 | lo);
    } else {
        return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
    }
}
template <typename V> __device__ __forceinline__ V wave_sum(V v) { return from_lane(wave_scan(v), 63); }
__device__ __forceinline__ uint32_t wave_most(uint32_t v) {
    v = max(v, moved<0x111>(v));
    v = max(v, moved<0x112>(v));
    v = max(v, moved<0x114>(v));
    v = max(v, moved<0x118>(v));
    v = max(v, moved<0x142, 0xA>(v));
    v = max(v, moved<0x143, 0xC>(v));
    return from_lane(v, 63);
}
__device__ __forceinline__ int lanes_below(uint64_t mask) {
    return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

struct Cut {
    uint32_t key;
    int64_t count;  // of those that equal it
};

// A wave's row: slot 256 c + 4 lane + e is held by the lane at [4 c + e].
template <int kPer> struct Held {
    uint32_t key[kPer];
    double w[kPer];

    uint8_t bin[kPer];  // four an octave of weight, falling; the last holds the rest
    __device__ __forceinline__ void share_out(uint32_t top, float scale) {
        const float x = value_of(top);
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            const float y = (x - value_of(key[i])) * scale * 4.0f;
            bin[i] = (uint8_t)(y < 63.0f ? (int)y : 63);  // NaN, too
        }
    }

    // The cut at which a sum over the keys above, of counts or of weights, first reaches `want`; {0, 0}, which cuts nothing,
    // where their whole does not.  Counts or weights (here in 2^-22) added up by bins in LDS say in which bin the cut is; in it,
    // a round takes the key that some lane holds between the bounds as pivot, the first lane past a place that changes
    // from round to round, so that rows in order are halved like others.  Rounds are settled by sums in float32 where
    // these are far from `want`, about one a row by exact ones.  Where the bins' rounding has said a wrong one, its keys come
    // to an end, and all are searched.
    template <bool kCount> __device__ __forceinline__ Cut cut_at(double want, uint32_t* bins) const {
        const int lane = threadIdx.x & 63;
        float wf[kPer], far = 0.0f;
        const float want_f = (float)want;
        bins[lane] = 0;
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            wf[i] = kCount ? (key[i] ? 1.0f : 0.0f) : (float)w[i] * (float)(0x1p22 / kWaveOne);
            far += wf[i];
            if (key[i]) atomicAdd(&bins[bin[i]], (uint32_t)wf[i]);
        }
        // the float sums' rounding: a chain of kPer + 6 additions, 2^-24 of the whole each, and that of the terms and of `want`
        far = kCount ? 0.0f : wave_sum(far) * (float)(kWaveOne / 0x1p22) * 0x1p-18f;
        __builtin_amdgcn_wave_barrier();
        const uint32_t upto = wave_scan(bins[lane]);
        const uint64_t past = __ballot((double)upto >= (kCount ? want : want * (0x1p22 / kWaveOne)));
        const int cut_bin = past ? __ffsll((unsigned long long)past) - 1 : 64;
#pragma unroll 1
        for (int all = cut_bin > 63; all < 2; all++) {
            uint32_t low = 1, high = 0xFFFFFFFFu;
            for (int round = 0; round < 64 * kPer && low <= high; round++) {
                uint32_t pivot = 0;
                double each = 1.0;
                uint64_t in = 0;
#pragma unroll
                for (int j = 0; j < kPer; j++) {
                    const uint64_t here = __ballot(key[j] - low <= high - low && (all || bin[j] == cut_bin));
                    if (__popcll(here) > __popcll(in)) {
                        in = here;
                        const uint64_t later = here & ~0ull << (round * 23 + 32 & 63);
                        const int at = __ffsll((unsigned long long)(later ? later : here)) - 1;
                        pivot = from_lane(key[j], at);
                        if (!kCount) each = from_lane(w[j], at);
                    }
                }
                if (!in) break;
                int equal = 0, count = 0;
                float near = 0.0f;
#pragma unroll
                for (int i = 0; i < kPer; i++) {
                    equal += __popcll(__ballot(key[i] == pivot));
                    if (kCount) count += __popcll(__ballot(key[i] > pivot));
                    else near += key[i] > pivot ? wf[i] : 0.0f;
                }
                double above = count;
                if (!kCount) {
                    near = wave_sum(near) * (float)(kWaveOne / 0x1p22);
                    above = near;
                    const float upto = near + equal * (float)each;
                    if (near <= want_f + far && upto >= want_f - far) {
                        double s = 0.0;
#pragma unroll
                        for (int i = 0; i < kPer; i++) s += key[i] > pivot ? w[i] : 0.0;
                        above = wave_sum(s);
                    }
                }
                if (above >= want) {
                    low = pivot + 1;
                } else if (above + equal * each < want) {
                    high = pivot - 1;
                } else {
                    const double more = kCount ? want - above : ceil((want - above) / each);
                    return {pivot, (int64_t)more};
                }
            }
        }
        return {0, 0};
    }
    // what is past the cut leaves
    __device__ __forceinline__ void keep(Cut c) {
        int before = 0;  // equals of the chunks before
#pragma unroll
        for (int i = 0; i < kPer; i += 4) {
            uint64_t same[4];
            int rank = before;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                same[e] = __ballot(key[i + e] == c.key);
                rank += lanes_below(same[e]);
                before += __popcll(same[e]);
            }
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const bool equal = key[i + e] == c.key;
                if (key[i + e] < c.key || (equal && rank >= c.count)) {
                    key[i + e] = 0;
                    w[i + e] = 0.0;
                }
                rank += equal;
            }
        }
    }
};

// The draw from a wave's row, whose largest key is `top`: its place among the slots held, and the logarithm of its
// probability.  `all_live`: the weights of the row's live slots, where they are not all held (0: they are).  `bins`: 64 words
// of LDS, the wave's own.
template <int kPer>
__device__ __forceinline__ int draw(Held<kPer>& h, const Row& r, uint32_t top, double all_live, uint32_t* bins,
                                    double& log_prob) {
    int live = 0, action = -1;
    weights_of<kPer>(h.key, top, r.scale, h.w);
#pragma unroll
    for (int i = 0; i < kPer; i++) {
        h.w[i] = rint(h.w[i] * kWaveOne);
        live += __popcll(__ballot(h.key[i] != 0));
    }
    const bool cut_k = r.k && r.k < live;
    if (cut_k || r.cut_p) h.share_out(top, (float)r.scale);
    if (cut_k) h.keep(h.template cut_at<true>((double)r.k, bins));
    if (r.cut_p) {
        double all = 0.0;
#pragma unroll
        for (int i = 0; i < kPer; i++) all += h.w[i];
        all = wave_sum(all);
        const double want = ceil(r.p * (all_live > 0.0 ? all_live : all));
        h.keep(h.template cut_at<false>(want < 1.0 ? 1.0 : want, bins));
    }
    const double least = r.min_p * kWaveOne;
    double upto[kPer / 4], all = 0.0;  // the sums up to a lane's last slot of each chunk
#pragma unroll
    for (int i = 0; i < kPer; i += 4) {
        double part = 0.0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            h.w[i + e] = h.w[i + e] >= least ? h.w[i + e] : 0.0;
            part += h.w[i + e];
        }
        upto[i / 4] = wave_scan(part) + all;
        all = from_lane(upto[i / 4], 63);
    }
    const double border = fmin(r.u * all, all - 1.0);  // u at or past 1: the last
#pragma unroll
    for (int i = 0; i < kPer; i += 4) {
        if (action >= 0) continue;
        const uint64_t past = __ballot(upto[i / 4] > border);
        if (past) {
            const int first = __ffsll((unsigned long long)past) - 1;
            double run = upto[i / 4];  // back from the lane's last slot: the first whose sum is past the border
            int mine = 3;
            uint32_t key = h.key[i + 3];
#pragma unroll
            for (int e = 2; e >= 0; e--) {
                run -= h.w[i + e + 1];
                if (run > border) {
                    mine = e;
                    key = h.key[i + e];
                }
            }
            action = i * 64 + first * 4 + from_lane(mine, first);
            log_prob = log_share(from_lane(key, first), top, r.scale, all / kWaveOne);
        }
    }
    return action;
}

template <typename T, int kPer> __global__ void __launch_bounds__(256) k_sample_held(Settings s) {
    __shared__ uint32_t bins[4][64];
    const int lane = threadIdx.x & 63;
    // the same for the wave's lanes, and known to be: its settings come by scalar loads, all at once
    const int64_t b = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (b >= s.rows) return;
    const Row r = row_of(s, b);
    const T* row = (const T*)s.logits + b * s.stride;
    Held<kPer> h;
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kPer; i += 4) {
        load_keys(row, i * 64 + lane * 4, r.n, h.key + i);
#pragma unroll
        for (int e = 0; e < 4; e++) top = max(top, h.key[i + e]);
    }
    top = wave_most(top);
    int action = -1;
    double log_prob = 0.0;
    if (top && r.greedy) {
#pragma unroll
        for (int i = 0; i < kPer; i += 4) {
            if (action >= 0) continue;
            int mine = 4;
#pragma unroll
            for (int e = 3; e >= 0; e--) mine = h.key[i + e] == top ? e : mine;
            const uint64_t have = __ballot(mine < 4);
            if (have) {
                const int first = __ffsll((unsigned long long)have) - 1;
                action = i * 64 + first * 4 + from_lane(mine, first);
            }
        }
    } else if (top) {
        action = draw(h, r, top, 0.0, bins[threadIdx.x >> 6], log_prob);
    }
    if (lane == 0) {
        s.actions[b] = action;
        if (s.log_probs) s.log_probs[b] = (float)log_prob;
    }
}

constexpr int kThreads = 1024, kWaves = kThreads / 64, kBins = 2048;
constexpr int kParts = (int)(kMaxWidth / 256);

struct Shared {
    unsigned long long bins[kParts];  // the first kBins: of a digit; then all: the sums of 256 slots each
    uint32_t equal[kParts];
    unsigned long long above, all, most[kWaves];
    int holders[kWaves];
    int bin, left;
    uint32_t wave_bins[64];
};

// the bin, from the top, at which the sum reaches `want`, and the sum above it; by wave 0, for all
__device__ __forceinline__ void find_bin(Shared& sh, unsigned long long want) {
    __syncthreads();
    if (threadIdx.x < 64) {
        constexpr int each = kBins / 64;
        const int first = kBins - 1 - (int)threadIdx.x * each;
        unsigned long long sum = 0;
        for (int i = 0; i < each; i++) sum += sh.bins[first - i];
        const unsigned long long upto = wave_scan(sum);
        const uint64_t past = __ballot(upto >= want);
        if ((int)threadIdx.x == __ffsll((unsigned long long)past) - 1) {
            unsigned long long run = upto - sum;
            int i = 0;
            while (i < each - 1 && run + sh.bins[first - i] < want) run += sh.bins[first - i++];
            sh.bin = first - i;
            sh.above = run;
        }
    }
    __syncthreads();
}

template <typename T> __global__ void __launch_bounds__(kThreads) k_sample_long(Settings s) {
    __shared__ Shared sh;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t b = blockIdx.x;
    const Row r = row_of(s, b);
    const T* row = (const T*)s.logits + b * s.stride;
    auto each = [&](auto f) {
        for (int c = tid * 4; c - lane * 4 < r.n; c += 4 * kThreads * 4) {  // whole waves: f may ask all lanes
            uint32_t key[4][4];  // four loads under way
#pragma unroll
            for (int k = 0; k < 4; k++) load_keys(row, c + k * kThreads * 4, r.n, key[k]);
#pragma unroll
            for (int k = 0; k < 4; k++)
#pragma unroll
                for (int e = 0; e < 4; e++) f(key[k][e], c + k * kThreads * 4 + e);
        }
    };
    auto clear = [&] {
        for (int i = tid; i < kBins; i += kThreads) sh.bins[i] = 0;
        __syncthreads();
    };
    const bool by_count = r.k && !r.greedy;
    if (by_count) clear();
    // the largest key and its first slot, then as one number, and how many are live
    uint32_t own = 0;
    int live = 0, slot = 0;
    each([&](uint32_t key, int i) {
        slot = key > own ? i : slot;
        own = max(key, own);
        live += key != 0;
    });
    if (by_count && own) atomicAdd(&sh.bins[own >> 21], 1ull);
    unsigned long long best = own ? (unsigned long long)own << 32 | (uint32_t)~slot : 0;
    const int holders = wave_sum(own != 0 ? 1 : 0);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const unsigned long long other = __shfl_xor(best, o, 64);
        best = other > best ? other : best;
    }
    live = wave_sum(live);
    if (lane == 0) {
        sh.most[wave] = best;
        sh.equal[wave] = live;
        sh.holders[wave] = holders;
    }
    __syncthreads();
    live = 0;
    int all_holders = 0;  // threads with a live slot
    for (int i = 0; i < kWaves; i++) {
        best = sh.most[i] > best ? sh.most[i] : best;
        live += sh.equal[i];
        all_holders += sh.holders[i];
    }
    __syncthreads();
    const uint32_t top = (uint32_t)(best >> 32);
    if (!top || r.greedy) {
        if (tid == 0) {
            s.actions[b] = top ? (int64_t)(uint32_t)~(uint32_t)best : -1;
            if (s.log_probs) s.log_probs[b] = 0.0f;
        }
        return;
    }
    auto weight = [&](uint32_t key) { return (unsigned long long)rint(weight_of(key, top, r.scale) * kBlockOne); };
    // What has to be at or above `floor` to be kept.  By top_k, the two digits in which the k-th largest of the threads' own
    // largest is, at or above which there are k at least (to count every key's digit took 42 us instead of 37 for 192 rows of
    // 85,834 and the 50 largest: the digits are few, and what adds to one waits for the others), or, where fewer threads hold
    // any, the digit of the k-th of all keys; by top_p without it, that in which the mass is reached; by min_p, a weight a little below it (the logit's rounding to float32 and that of the logarithm).
    const bool cut_k = r.k && r.k < live;
    uint32_t floor_key = 1;
    unsigned long long all_live = 0;
    // the cut's first digit and what is above it, where all keys were added up by it
    int digit = -1;
    unsigned long long above = 0;
    auto settled = [&] {
        digit = sh.bin;
        above = sh.above;
    };
    if (cut_k) {
        if (r.k > all_holders) {
            clear();
            each([&](uint32_t key, int) {
                if (key) atomicAdd(&sh.bins[key >> 21], 1ull);
            });
            __syncthreads();
        }
        find_bin(sh, (unsigned long long)r.k);
        const uint32_t bin = sh.bin;
        floor_key = max(1u, bin << 21);
        if (r.k > all_holders) {
            settled();
        } else {  // the next digit as well
            const unsigned long long want = (unsigned long long)r.k - sh.above;
            clear();
            if (own >> 21 == bin && own) atomicAdd(&sh.bins[own >> 10 & 2047], 1ull);
            find_bin(sh, want);
            floor_key = max(1u, bin << 21 | (uint32_t)sh.bin << 10);
        }
    } else if (r.cut_p) {
        __syncthreads();
        clear();
        each([&](uint32_t key, int) {
            if (const unsigned long long w = key ? weight(key) : 0) atomicAdd(&sh.bins[key >> 21], w);
        });
        __syncthreads();
        if (wave == 0) {
            unsigned long long sum = 0;
            for (int i = lane; i < kBins; i += 64) sum += sh.bins[i];
            sum = wave_sum(sum);
            if (lane == 0) sh.all = sum;
        }
        __syncthreads();
        all_live = sh.all;
        const double part = ceil(r.p * (double)all_live);
        find_bin(sh, part < 1.0 ? 1ull : part < (double)all_live ? (unsigned long long)part : all_live);
        floor_key = max(1u, (uint32_t)sh.bin << 21);
        settled();
    }
    if (r.min_p > 0.0 && !(cut_k && r.cut_p)) {  // top_p of the k largest needs them all
        const double x = (double)value_of(top), raw = x + r.t * log(r.min_p), at = raw - 1e-6 * (fabs(x) + fabs(raw) + r.t);
        const float least = at > -3.4028234663852886e38 ? (float)at : -__builtin_inff();  // NaN: none
        floor_key = max(floor_key, key_of(least));
    }
    if (tid == 0) sh.left = 0;
    __syncthreads();
    // the slots left, in any order, then in the row's
    uint32_t* const left_key = (uint32_t*)sh.bins;
    uint32_t* const left_slot = left_key + kHeld;
    uint32_t* const key_in_order = left_slot + kHeld;
    uint32_t* const slot_in_order = key_in_order + kHeld;
    const bool few = floor_key > 1 || live <= kHeld;
    if (few)
        each([&](uint32_t key, int i) {
            const uint64_t these = __ballot(key >= floor_key);
            if (!these) return;
            int first = 0;
            if (lane == __ffsll((unsigned long long)these) - 1) first = atomicAdd(&sh.left, __popcll(these));
            const int at = from_lane(first, __ffsll((unsigned long long)these) - 1) + lanes_below(these);
            if (key >= floor_key && at < kHeld) {
                left_key[at] = key;
                left_slot[at] = i;
            }
        });
    __syncthreads();
    const int left = sh.left;
    if (few && left <= kHeld) {
        if (tid < kHeld - left) left_slot[left + tid] = 0xFFFFFFFFu;
        key_in_order[tid] = 0;
        __syncthreads();
        if (tid < left) {
            const uint32_t mine = left_slot[tid];
            int rank = 0;
            for (int i = 0; i < left; i += 4) {
                const uint4 q = *(const uint4*)(left_slot + i);
                rank += (q.x < mine) + (q.y < mine) + (q.z < mine) + (q.w < mine);
            }
            key_in_order[rank] = left_key[tid];
            slot_in_order[rank] = mine;
        }
        __syncthreads();
        if (wave != 0) return;
        double log_prob = 0.0;
        const double whole = (double)all_live * (kWaveOne / kBlockOne);
        auto drawn = [&](auto h) {
            constexpr int per = (int)(sizeof(h.key) / 4);
#pragma unroll
            for (int i = 0; i < per; i += 4) {
                const uint4 q = *(const uint4*)(key_in_order + i * 64 + lane * 4);
                h.key[i] = q.x;
                h.key[i + 1] = q.y;
                h.key[i + 2] = q.z;
                h.key[i + 3] = q.w;
            }
            return draw(h, r, top, whole, sh.wave_bins, log_prob);
        };
        const int place = left <= 256 ? drawn(Held<4>{}) : drawn(Held<kHeld / 64>{});
        if (lane == 0) {
            s.actions[b] = slot_in_order[place];
            if (s.log_probs) s.log_probs[b] = (float)log_prob;
        }
        return;
    }
    __syncthreads();
    // the cut at which the sum of `of` over the keys reaches `want`, by digits of 11, 11 and 10 bits; `last`: keys that
    // equal it are counted by `extra` alone.  The first digit is `digit`, if that is known.
    auto cut_at = [&](unsigned long long want, auto of, uint32_t last, unsigned long long extra) {
        uint32_t prefix = 0, mask = 0;
        const int shifts[3] = {21, 10, 0};
        if (digit >= 0) {
            prefix = (uint32_t)digit << 21;
            mask = 0x7FFu << 21;
            want -= above;
        }
        for (int d = digit >= 0 ? 1 : 0; d < 3; d++) {
            const int shift = shifts[d];
            clear();
            each([&](uint32_t key, int) {
                if (key && (key & mask) == prefix && (key > last || !extra))
                    atomicAdd(&sh.bins[key >> shift & (d == 2 ? 0x3FF : 0x7FF)], of(key));
            });
            if (extra && tid == 0 && (last & mask) == prefix) atomicAdd(&sh.bins[last >> shift & (d == 2 ? 0x3FF : 0x7FF)], extra);
            find_bin(sh, want);
            want -= sh.above;
            prefix |= (uint32_t)sh.bin << shift;
            mask |= (d == 2 ? 0x3FFu : 0x7FFu) << shift;
            __syncthreads();
        }
        const unsigned long long one = of(prefix);
        return Cut{prefix, (int64_t)((want + one - 1) / one)};
    };
    Cut cut{1, (int64_t)1 << 40};  // nothing is cut
    if (cut_k) {
        cut = cut_at((unsigned long long)r.k, [](uint32_t) { return 1ull; }, 0, 0);
        digit = -1;
    }
    if (r.cut_p) {
        unsigned long long extra = 0, all = all_live;
        if (cut_k) {
            unsigned long long sum = 0;
            each([&](uint32_t key, int) {
                if (key > cut.key) sum += weight(key);
            });
            sum = wave_sum(sum);
            if (tid == 0) sh.all = 0;
            __syncthreads();
            if (lane == 0) atomicAdd(&sh.all, sum);
            __syncthreads();
            extra = cut.key > 1 ? (unsigned long long)cut.count * weight(cut.key) : 0;
            all = sh.all + extra;
        }
        const double part = ceil(r.p * (double)all);
        const unsigned long long want = part < 1.0 ? 1ull : part < (double)all ? (unsigned long long)part : all;
        cut = cut_at(want, weight, cut.key, extra);
    }
    // the sums of 256 slots each, what equals the cut's key counted apart
    const double least = r.min_p;
    const unsigned long long same = weight_of(cut.key, top, r.scale) >= least ? weight(cut.key) : 0;
    const int parts = (r.n + 255) / 256;
    unsigned long long* sums = sh.bins;
    auto kept = [&](uint32_t key) {
        if (key <= cut.key) return 0ull;
        const double w = weight_of(key, top, r.scale);
        return w >= least ? (unsigned long long)rint(w * kBlockOne) : 0ull;
    };
    __syncthreads();
    for (int p = wave; p < parts; p += kWaves) {
        uint32_t key[4];
        load_keys(row, p * 256 + lane * 4, r.n, key);
        unsigned long long sum = 0;
        uint32_t equal = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            sum += kept(key[e]);
            equal += key[e] == cut.key;
        }
        sum = wave_sum(sum);
        equal = wave_sum(equal);
        if (lane == 0) {
            sums[p] = sum;
            sh.equal[p] = equal;
        }
    }
    __syncthreads();
    if (wave != 0) return;
    // which of them: a lane takes a run of them
    const int run = (parts + 63) / 64, first = lane * run, end = min(first + run, parts);
    int64_t equals = 0;
    for (int p = first; p < end; p++) equals += sh.equal[p];
    const int64_t equals_before = wave_scan(equals) - equals;
    auto of_part = [&](int p, int64_t before) {
        const int64_t left = cut.count - before;
        const int64_t n = left <= 0 ? 0 : left < (int64_t)sh.equal[p] ? left : sh.equal[p];
        return sums[p] + (unsigned long long)n * same;
    };
    unsigned long long sum = 0;
    int64_t before = equals_before;
    for (int p = first; p < end; p++) {
        sum += of_part(p, before);
        before += sh.equal[p];
    }
    const unsigned long long upto = wave_scan(sum), all = from_lane(upto, 63);
    const double passed = floor(r.u * (double)all);
    const unsigned long long border = passed >= (double)all ? all - 1 : (unsigned long long)passed;
    const int at = __ffsll((unsigned long long)__ballot(upto > border)) - 1;
    unsigned long long total = upto - sum;
    int part = first;
    before = equals_before;
    for (; part < end - 1; part++) {
        const unsigned long long w = of_part(part, before);
        if (total + w > border) break;
        total += w;
        before += sh.equal[part];
    }
    part = from_lane(part, at);
    total = from_lane(total, at);
    before = from_lane(before, at);
    uint32_t key[4];
    load_keys(row, part * 256 + lane * 4, r.n, key);
    unsigned long long w[4], mine = 0;
    int equal = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) equal += key[e] == cut.key;
    int64_t rank = before + wave_scan(equal) - equal;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        w[e] = key[e] == cut.key ? (rank++ < cut.count ? same : 0) : kept(key[e]);
        mine += w[e];
    }
    const unsigned long long scan = wave_scan(mine) + total;
    const int owner = __ffsll((unsigned long long)__ballot(scan > border)) - 1;
    if (lane != owner) return;
    unsigned long long running = scan - mine;
    int e = 0;
    for (; e < 3; e++) {
        running += w[e];
        if (running > border) break;
    }
    s.actions[b] = (int64_t)part * 256 + lane * 4 + e;
    if (s.log_probs) {
        const uint32_t k = key[e];
        s.log_probs[b] = (float)log_share(k, top, r.scale, (double)all / kBlockOne);
    }
}

}  // namespace

extern "C" {

int hg_sample_actions(const void* logits, int type, int64_t rows, int64_t width, int64_t stride,
                      const int64_t* num_actions, const float* uniforms, const float* temperatures, double temperature,
                      const int64_t* top_ks, int64_t top_k, const float* top_ps, double top_p, const float* min_ps,
                      double min_p, int64_t* actions, float* log_probs, void* stream) {
    if (!is_type(type) || rows < 0 || width < 1 || width > kMaxWidth ||
        rows > (width <= kHeld ? kMaxRows : kMaxLongRows)) return (int)hipErrorInvalidValue;
    if (rows == 0) return 0;
    if (!logits || !uniforms || !actions) return (int)hipErrorInvalidValue;
    const Settings s{logits, stride, rows, (int)width, num_actions, uniforms, temperatures, top_ps, min_ps, top_ks,
                     temperature, top_p, min_p, top_k, actions, log_probs};
    hipStream_t st = (hipStream_t)stream;
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        const unsigned waves = (unsigned)((rows + 3) / 4);
        if (width <= 256) k_sample_held<T, 4><<<waves, 256, 0, st>>>(s);
        else if (width <= kHeld) k_sample_held<T, 16><<<waves, 256, 0, st>>>(s);
        else k_sample_long<T><<<(unsigned)rows, kThreads, 0, st>>>(s);
        return (int)hipGetLastError();
    });
}

}  // extern "C"
