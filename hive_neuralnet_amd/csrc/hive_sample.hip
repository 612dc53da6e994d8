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
// cut is found by pivots, the middle one of what is left; longer rows are read
// by a block, cuts found by three digits of the key, whose counts or weights are
// added up in LDS.
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
    r.min_p = r.min_p > 1.0 ? 1.0 : r.min_p;  // the largest always stays
    const int64_t k = s.top_ks ? s.top_ks[b] : s.top_k;
    r.k = k > 0 ? k : 0;
    r.u = (double)s.uniforms[b];
    r.u = r.u > 0.0 ? r.u : 0.0;  // NaN: 0
    r.greedy = !(r.t > 0.0);
    r.scale = 1.4426950408889634 / r.t;
    r.cut_p = r.p < 1.0;
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
// exp((x - top) / t) = 2^(scale (x - top)), scale = log2(e) / t; 1 for x = top whatever it is.  A series of 2^f, |f| <= 1/2,
// to f^11: 2^-47 of the whole left out, with the rounding of scale and of the product under 2^-45, a weight's own rounding.
__device__ __forceinline__ double weight_of(uint32_t key, uint32_t top, double scale) {
    if (key == top) return 1.0;
    if (!key) return 0.0;
    // NaN (a logit below one of inf at a temperature of inf) and -inf: 0
    const double y = fmax(((double)value_of(key) - (double)value_of(top)) * scale, -1200.0), n = rint(y);
    const double f = (y - n) * 0.6931471805599453;
    double s = 1.0 / 39916800.0;
    s = fma(s, f, 1.0 / 3628800.0);
    s = fma(s, f, 1.0 / 362880.0);
    s = fma(s, f, 1.0 / 40320.0);
    s = fma(s, f, 1.0 / 5040.0);
    s = fma(s, f, 1.0 / 720.0);
    s = fma(s, f, 1.0 / 120.0);
    s = fma(s, f, 1.0 / 24.0);
    s = fma(s, f, 1.0 / 6.0);
    s = fma(s, f, 0.5);
    s = fma(s, f, 1.0);
    s = fma(s, f, 1.0);
    return ldexp(s, (int)n);
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
template <int kControl, int kRows = 0xF, typename V> __device__ __forceinline__ V moved(V v) {
    if constexpr (sizeof(V) == 8) {
        const uint64_t b = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, kControl, kRows, 0xF, false);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), kControl, kRows, 0xF, false);
        return __builtin_bit_cast(V, (uint64_t)hi << 32 | lo);
    } else {
        return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), kControl, kRows, 0xF, false));
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

    // the cut at which a sum over the keys above, of counts or of weights, first reaches `want` (at most their whole)
    template <bool kCount> __device__ __forceinline__ Cut cut_at(double want) const {
        uint32_t low = 1, high = 0xFFFFFFFFu;
        for (int round = 0; round < 64 * kPer; round++) {
            // the pivot: the middle lane of those that hold a key between
            uint32_t pivot = 0;
            double each = 1.0;
            bool found = false;
#pragma unroll
            for (int j = 0; j < kPer; j++) {
                if (found) continue;
                const int at = (j + round) % kPer;
                uint32_t k = key[0];
                double v = w[0];
#pragma unroll
                for (int i = 1; i < kPer; i++) {
                    k = at == i ? key[i] : k;
                    v = at == i ? w[i] : v;
                }
                const uint64_t in = __ballot(k >= low && k <= high);
                if (in) {
                    const uint64_t middle = __ballot((in >> (threadIdx.x & 63) & 1) && lanes_below(in) == __popcll(in) / 2);
                    const int lane = __ffsll((unsigned long long)middle) - 1;
                    pivot = __builtin_amdgcn_readlane(k, lane);
                    if (!kCount) each = from_lane(v, lane);
                    found = true;
                }
            }
            if (!found) break;
            int equal = 0;
            double above;
            if constexpr (kCount) {
                int c = 0;
#pragma unroll
                for (int i = 0; i < kPer; i++) {
                    c += __popcll(__ballot(key[i] > pivot));
                    equal += __popcll(__ballot(key[i] == pivot));
                }
                above = c;
            } else {
                double s = 0.0;
#pragma unroll
                for (int i = 0; i < kPer; i++) {
                    s += key[i] > pivot ? w[i] : 0.0;
                    equal += __popcll(__ballot(key[i] == pivot));
                }
                above = wave_sum(s);
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
        return {0, 0};  // not reached: `want` is at most the whole
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
// probability.  `all_live`: the weights of the row's live slots, where they are not all held (0: they are).
template <int kPer>
__device__ __forceinline__ int draw(Held<kPer>& h, const Row& r, uint32_t top, double all_live, double& log_prob) {
    int live = 0, action = -1;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
        h.w[i] = rint(weight_of(h.key[i], top, r.scale) * kWaveOne);
        live += __popcll(__ballot(h.key[i] != 0));
    }
    if (r.k && r.k < live) h.keep(h.template cut_at<true>((double)r.k));
    if (r.cut_p) {
        double all = 0.0;
#pragma unroll
        for (int i = 0; i < kPer; i++) all += h.w[i];
        all = wave_sum(all);
        const double want = ceil(r.p * (all_live > 0.0 ? all_live : all));
        h.keep(h.template cut_at<false>(want < 1.0 ? 1.0 : want));
    }
    const double least = r.min_p * kWaveOne;
    double part[kPer / 4], all = 0.0;  // a lane's sums in each chunk
#pragma unroll
    for (int i = 0; i < kPer; i += 4) {
        part[i / 4] = 0.0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            h.w[i + e] = h.w[i + e] >= least ? h.w[i + e] : 0.0;
            part[i / 4] += h.w[i + e];
        }
        all += part[i / 4];
    }
    all = wave_sum(all);
    const double border = fmin(r.u * all, all - 1.0);  // u at or past 1: the last
    double before = 0.0;
#pragma unroll
    for (int i = 0; i < kPer; i += 4) {
        if (action >= 0) continue;
        const double upto = wave_scan(part[i / 4]) + before;
        const uint64_t past = __ballot(upto > border);
        if (past) {
            const int first = __ffsll((unsigned long long)past) - 1;
            double run = upto - part[i / 4];
            int mine = -1;
            uint32_t key = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                run += h.w[i + e];
                if (mine < 0 && run > border) {
                    mine = e;
                    key = h.key[i + e];
                }
            }
            action = i * 64 + first * 4 + from_lane(mine, first);
            key = from_lane(key, first);
            log_prob = (key == top ? 0.0 : ((double)value_of(key) - (double)value_of(top)) / r.t) - log(all / kWaveOne);
        } else {
            before = from_lane(upto, 63);
        }
    }
    return action;
}

template <typename T, int kPer> __global__ void __launch_bounds__(256) k_sample_held(Settings s) {
    const int lane = threadIdx.x & 63;
    const int64_t b = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
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
        action = draw(h, r, top, 0.0, log_prob);
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
    unsigned long long above, all;
    uint32_t most[kWaves];
    int bin;
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
        for (int c = tid * 4; c < r.n; c += kThreads * 4) {
            uint32_t key[4];
            load_keys(row, c, r.n, key);
#pragma unroll
            for (int e = 0; e < 4; e++) f(key[e], c + e);
        }
    };
    uint32_t top = 0;
    int live = 0;
    each([&](uint32_t key, int) {
        top = max(top, key);
        live += key != 0;
    });
    top = wave_most(top);
    live = wave_sum(live);
    if (lane == 0) {
        sh.most[wave] = top;
        sh.equal[wave] = live;
    }
    __syncthreads();
    live = 0;
    for (int i = 0; i < kWaves; i++) {
        top = max(top, sh.most[i]);
        live += sh.equal[i];
    }
    __syncthreads();
    if (!top) {
        if (tid == 0) {
            s.actions[b] = -1;
            if (s.log_probs) s.log_probs[b] = 0.0f;
        }
        return;
    }
    if (r.greedy) {
        if (tid == 0) sh.bin = r.n;
        __syncthreads();
        int first = r.n;
        each([&](uint32_t key, int i) { first = key == top && i < first ? i : first; });
        if (first < r.n) atomicMin(&sh.bin, first);
        __syncthreads();
        if (tid == 0) {
            s.actions[b] = sh.bin;
            if (s.log_probs) s.log_probs[b] = 0.0f;
        }
        return;
    }
    auto weight = [&](uint32_t key) { return (unsigned long long)rint(weight_of(key, top, r.scale) * kBlockOne); };
    auto clear = [&] {
        for (int i = tid; i < kBins; i += kThreads) sh.bins[i] = 0;
        __syncthreads();
    };
    // the cut at which the sum of `of` over the keys reaches `want`, by digits of 11, 11 and 10 bits; `last`: keys that
    // equal it are counted by `extra` alone
    auto cut_at = [&](unsigned long long want, auto of, uint32_t last, unsigned long long extra) {
        uint32_t prefix = 0, mask = 0;
        const int shifts[3] = {21, 10, 0};
        for (int d = 0; d < 3; d++) {
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
    if (r.k && r.k < live) cut = cut_at((unsigned long long)r.k, [](uint32_t) { return 1ull; }, 0, 0);
    if (r.cut_p) {
        unsigned long long sum = 0;
        each([&](uint32_t key, int) {
            if (key > cut.key) sum += weight(key);
        });
        sum = wave_sum(sum);
        if (tid == 0) sh.all = 0;
        __syncthreads();
        if (lane == 0) atomicAdd(&sh.all, sum);
        __syncthreads();
        const unsigned long long extra = cut.key > 1 ? (unsigned long long)cut.count * weight(cut.key) : 0;
        const unsigned long long all = sh.all + extra;
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
        s.log_probs[b] = (float)((k == top ? 0.0 : ((double)value_of(k) - (double)value_of(top)) / r.t) -
                                 log((double)all / kBlockOne));
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
