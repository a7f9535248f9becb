// Routing to experts: of E logits a token's `top` experts and their weights.
//
//   s = softmax(l) or sigmoid(l);  key = s + bias;  the value of a group of experts is the
//   sum of its two highest keys;  of the experts in the top_groups groups of highest value
//   the `top` highest keys, ties to the lower index;  weight_j = scale s_j, divided by the
//   sum of the chosen s if renormalised.
//
// An expert whose logit or key is -inf is never chosen; slots left over have id -1 and
// weight 0.  A row with a NaN logit (for softmax +inf too) has NaN weights; its experts are
// chosen by the logits, NaNs last.  A NaN key (of a NaN bias) counts as the lowest.
//
// Which experts are chosen hangs on keys that may be next to each other, so the ones that
// matter are compared in 64 bits.
#include "block_kernels.hpp"
#include "mx_kernels.hpp"
#include "rows.hpp"

namespace xpuint8 {
namespace {

struct RouteArgs {
    const void* logits;
    const float* bias;
    int* ids;
    float* weights;
    int64_t ld, T;
    int E, top;
    RouteHow how;
};

template <int T>
__device__ __forceinline__ float logit_at(const void* logits, int64_t row, int64_t ld, int e) {
    const int64_t i = row * ld + e;
    if constexpr (T == kF32) return static_cast<const float*>(logits)[i];
    else if constexpr (T == kBf16) return bf16_to_f32(static_cast<const uint16_t*>(logits)[i]);
    else return float(static_cast<const _Float16*>(logits)[i]);
}

template <int CTRL>
__device__ __forceinline__ double dpp64(double x) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = dppu<CTRL>(uint32_t(b)), hi = dppu<CTRL>(uint32_t(b >> 32));
    return __builtin_bit_cast(double, uint64_t(hi) << 32 | lo);
}
template <int CTRL>
__device__ __forceinline__ float dpp_any(float x) { return dpp<CTRL>(x); }
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_any(uint32_t x) { return dppu<CTRL>(x); }
template <int CTRL>
__device__ __forceinline__ int dpp_any(int x) { return int(dppu<CTRL>(uint32_t(x))); }
template <int CTRL>
__device__ __forceinline__ double dpp_any(double x) { return dpp64<CTRL>(x); }

template <class V>
__device__ __forceinline__ V wave_total(V x) {
    x += dpp_any<kDppXor1>(x);
    x += dpp_any<kDppXor2>(x);
    x += dpp_any<kDppXor7>(x);
    x += dpp_any<kDppXor15>(x);
    const auto p = both_sides<16>(x);
    const auto q = both_sides<32>(p.lo + p.hi);
    return q.lo + q.hi;
}
template <class V>
__device__ __forceinline__ V greater_of(V x, V y) { return y > x ? y : x; }
template <class V>
__device__ __forceinline__ V wave_most(V x) {
    x = greater_of(x, dpp_any<kDppXor1>(x));
    x = greater_of(x, dpp_any<kDppXor2>(x));
    x = greater_of(x, dpp_any<kDppXor7>(x));
    x = greater_of(x, dpp_any<kDppXor15>(x));
    const auto p = both_sides<16>(x);
    const auto q = both_sides<32>(greater_of(p.lo, p.hi));
    return greater_of(q.lo, q.hi);
}

// the highest key of the wave and its expert (the lowest of equal ones), in every lane
__device__ __forceinline__ void take_best(double& key, int& e, double k, int o) {
    if (k > key || (k == key && o < e)) {
        key = k;
        e = o;
    }
}
__device__ __forceinline__ void wave_best(double& key, int& e) {
    take_best(key, e, dpp_any<kDppXor1>(key), dpp_any<kDppXor1>(e));
    take_best(key, e, dpp_any<kDppXor2>(key), dpp_any<kDppXor2>(e));
    take_best(key, e, dpp_any<kDppXor7>(key), dpp_any<kDppXor7>(e));
    take_best(key, e, dpp_any<kDppXor15>(key), dpp_any<kDppXor15>(e));
    const auto k16 = both_sides<16>(key);
    const auto e16 = both_sides<16>(e);
    key = k16.lo;
    e = e16.lo;
    take_best(key, e, k16.hi, e16.hi);
    const auto k32 = both_sides<32>(key);
    const auto e32 = both_sides<32>(e);
    key = k32.lo;
    e = e32.lo;
    take_best(key, e, k32.hi, e32.hi);
}

constexpr double kNone = -__builtin_huge_val();      // not to be chosen
// a NaN key: below all others (fp32 biases and scores), and so that the sum of two is above kNone
constexpr double kLowest = -1e300;

// A token by a whole wave, lane l holding the experts l, l + 64, ..; keys are 64 bits.  A round a
// slot: 4 tokens, 24 of 256 experts 13.6 us (20 with all exchanges through LDS; 5.9 by 32
// candidates), 65536 284 (47).
template <int T, int V>
__device__ __forceinline__ void route_token(const RouteArgs& a, int64_t t) {
    const int lane = threadIdx.x & 63;
            float l[V], most = -INFINITY;
            bool bad = false;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int e = 64 * i + lane;
                l[i] = e < a.E ? logit_at<T>(a.logits, t, a.ld, e) : -INFINITY;
                bad |= __builtin_isnan(l[i]) || (!a.how.sigmoid && l[i] == INFINITY);
                most = fmaxf(most, l[i]);
            }
            const bool spoilt = __builtin_amdgcn_ballot_w64(bad) != 0;
            most = wave_most(most);
            double key[V], sum = 0.0;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const bool out = l[i] == -INFINITY;
                key[i] = out ? 0.0 : a.how.sigmoid ? 1.0 / (1.0 + exp(-double(l[i])))
                                                   : exp(double(l[i]) - double(most));
                sum += key[i];
            }
            if (!a.how.sigmoid) sum = wave_total(sum);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int e = 64 * i + lane;
                if (!a.how.sigmoid) key[i] /= sum;
                if (a.bias && e < a.E) key[i] += double(a.bias[e]);
                if (!a.bias && a.how.groups == 1) key[i] = l[i];       // scores rise with logits
                if (spoilt) key[i] = l[i];
                if (__builtin_isnan(key[i])) key[i] = kLowest;
                if (l[i] == -INFINITY) key[i] = kNone;
            }
            if (a.how.groups > 1) {
                const int n = a.E / a.how.groups;
                double value = kNone;                     // lane g: of group g
                for (int g = 0; g < a.how.groups; ++g) {
                    double two = 0.0;
                    int first = -1;
                    for (int k = 0; k < 2; ++k) {
                        double best = kNone;
                        int at = a.E;
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            const int e = 64 * i + lane;
                            if (e >= g * n && e < (g + 1) * n && e != first && key[i] > best) {
                                best = key[i];
                                at = e;
                            }
                        }
                        wave_best(best, at);
                        first = at;
                        if (k == 0) two = best;
                        else if (best != kNone) two += best;
                    }
                    if (lane == g) value = two;
                }
                int rank = 0;
                for (int g = 0; g < a.how.groups; ++g) {
                    const double other = __shfl(value, g);
                    rank += other > value || (other == value && g < lane);
                }
                const uint64_t kept =
                    __builtin_amdgcn_ballot_w64(lane < a.how.groups && rank < a.how.top_groups);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const int e = 64 * i + lane;
                    if (e < a.E && !((kept >> (e / n)) & 1)) key[i] = kNone;
                }
            }
            int id = -1;                                  // lane j: of slot j
            for (int j = 0; j < a.top; ++j) {
                double best = kNone;
                int at = a.E;
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (key[i] > best) {
                        best = key[i];
                        at = 64 * i + lane;
                    }
                wave_best(best, at);
                if (best == kNone) break;
                if (lane == j) id = at;
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (64 * i + lane == at) key[i] = kNone;
            }
            const float mine = id >= 0 ? logit_at<T>(a.logits, t, a.ld, id) : -INFINITY;
            // divided by the sum, the scores may carry any common factor: the one that brings
            // the largest near 1
            double s = 0.0;
            if (a.how.sigmoid) {
                const double shift = a.how.renormalize ? fmin(0.0, double(wave_most(mine))) : 0.0;
                if (id >= 0) s = mine >= 0.f ? 1.0 / (1.0 + exp(-double(mine)))
                                             : exp(double(mine) - shift) / (1.0 + exp(double(mine)));
            } else {
                const double ref = a.how.renormalize ? double(wave_most(mine)) : double(most);
                if (id >= 0) s = exp(double(mine) - ref) / (a.how.renormalize ? 1.0 : sum);
            }
            const double total = a.how.renormalize ? wave_total(s) : 1.0;
            float w = id >= 0 ? float(double(a.how.scale) * s / total) : 0.f;
            if (spoilt) w = NAN;
            if (lane < a.top) {
                a.ids[t * a.top + lane] = id;
                a.weights[t * a.top + lane] = w;
            }
}

template <int T, int V>
__global__ __launch_bounds__(256) void route_exact_kernel(RouteArgs a) {
    for (int64_t t = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6); t < a.T; t += int64_t(gridDim.x) * 4)
        route_token<T, V>(a, t);
}

// ------------------------------------------------------------ several tokens a wave
// A token has L lanes of V experts, 64 / L tokens a wave.  Keys are made in fp32 first, to
// a known error; of each the 32 bits that order like it, with the expert's place in the low
// ones, are sorted in every lane and merged across the lanes down to the token's highest 16
// (32 for 17 to 32 slots, which begin with the counting below), all in integer minima and
// maxima.  The first of these candidates, one a lane, get their
// keys in 64 bits.  The choice is sure when these are in order and the last one chosen is
// above anything that the next candidate (with 16 lanes: the last one, or for 15 and 16 slots
// the key behind it) could be; if not, all
// 16 candidates are counted against each other in 64 bits, which 16 keys that agree with the last
// one chosen in all bits that the place leaves (23 of the mantissa less the place's 6 to 10, so
// within 2^-17 of it for 64 experts and 2^-13 for 1024), a NaN, or scores that underflow leave
// open still: such a token goes through route_token.  Groups whose fp32 values are too near, and softmax keys
// nearer than the fp32 sum's error, are looked at again in 64 bits too.
//
// Bound by instructions (half of them the sort's and the merges'), so few lanes a token: 8 for
// up to 8 slots and 256 experts (65536 tokens, 8 of 64 experts in bf16 10 us and 17 with 16 lanes;
// of 128 by biased sigmoids in fp32 17 and 22; 32768 of 256 in bf16 10 and 13).  Groups take 16
// lanes below 65536 tokens, whose waves are too few to hide what the groups add (8192 tokens of
// 256 in 8 groups 10 us and 13 with 8 lanes, 65536 34 and 34).  16381 of these take 16 us (with a
// wave a token and all keys in 64 bits 103), 4 tokens of 64 experts 2.5.  More than 256 experts
// take 16 or 32 lanes from 8192 tokens on (8 of 512 in bf16: 8192 tokens 6.9 us and 9.0 with
// twice the lanes, 65536 33 and 52; 8 of 1024: 81 and 130, 73 since lanes 16 and 32 apart meet
// without LDS), below that twice as many (2048 tokens of 512 4.5 us and 4.8).
constexpr int64_t kManyTokens = 8192;
constexpr uint32_t kNothing = 0x00800000u;           // ordered(-inf) and the bits of a place are below

// x of another lane of a row of ROW lanes, every lane of it once over K = 1 .. ROW - 1: of 16
// by rotation, of 8 of lane ^ K
template <int ROW, int K, class X>
__device__ __forceinline__ X other_lane(X x) {
    constexpr int kXor3 = 0x1B;                       // quad_perm [3,2,1,0]
    if constexpr (ROW == 16) return dpp_any<0x120 + K>(x);
    else if constexpr (K == 1) return dpp_any<kDppXor1>(x);
    else if constexpr (K == 2) return dpp_any<kDppXor2>(x);
    else if constexpr (K == 3) return dpp_any<kXor3>(x);
    else if constexpr (K == 7) return dpp_any<kDppXor7>(x);
    else if constexpr (K == 4) return dpp_any<kXor3>(dpp_any<kDppXor7>(x));
    else if constexpr (K == 5) return dpp_any<kDppXor2>(dpp_any<kDppXor7>(x));
    else return dpp_any<kDppXor1>(dpp_any<kDppXor7>(x));
}
// x and that of a lane on the other side of D, where the lanes of each side hold the same: lane
// ^ 1, ^ 2, ^ 7, ^ 15 by DPP, then the same two of D = 16 and 32 in both
template <int D>
__device__ __forceinline__ Both<uint32_t> sides(uint32_t x) {
    if constexpr (D == 1) return {x, dppu<kDppXor1>(x)};
    else if constexpr (D == 2) return {x, dppu<kDppXor2>(x)};
    else if constexpr (D == 4) return {x, dppu<kDppXor7>(x)};
    else if constexpr (D == 8) return {x, dppu<kDppXor15>(x)};
    else return both_sides<D>(x);
}

// a falls along i: compare and exchange
__device__ __forceinline__ void exchange(uint32_t& a, uint32_t& b) {
    const uint32_t hi = max(a, b), lo = min(a, b);
    a = hi;
    b = lo;
}
// a bitonic sequence sorted
template <int N, int AT, int M>
__device__ __forceinline__ void sort_bitonic(uint32_t (&a)[M]) {
    if constexpr (N > 1) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) exchange(a[AT + i], a[AT + i + N / 2]);
        sort_bitonic<N / 2, AT>(a);
        sort_bitonic<N / 2, AT + N / 2>(a);
    }
}
// the odd-even merge of two sorted halves, elements STEP apart, and the sort by it
template <int N, int AT, int STEP, int M>
__device__ __forceinline__ void merge_odd_even(uint32_t (&a)[M]) {
    if constexpr (N == 2) {
        exchange(a[AT], a[AT + STEP]);
    } else {
        merge_odd_even<N / 2, AT, 2 * STEP>(a);
        merge_odd_even<N / 2, AT + STEP, 2 * STEP>(a);
#pragma unroll
        for (int i = 1; i + 1 < N; i += 2) exchange(a[AT + i * STEP], a[AT + (i + 1) * STEP]);
    }
}
template <int N, int AT, int M>
__device__ __forceinline__ void sort_odd_even(uint32_t (&a)[M]) {
    if constexpr (N > 1) {
        sort_odd_even<N / 2, AT>(a);
        sort_odd_even<N / 2, AT + N / 2>(a);
        merge_odd_even<N, AT, 1>(a);
    }
}
// a lane's own V keys sorted, the C highest of 2 C; deep: `rest` becomes the highest other one
template <int V, int C, int M>
__device__ __forceinline__ void sort_lane(uint32_t (&a)[M], bool deep, uint32_t& rest) {
    if constexpr (V <= C) {
        sort_odd_even<V, 0>(a);
    } else {
        static_assert(V == 2 * C);
        sort_odd_even<C, 0>(a);
        sort_odd_even<C, C>(a);
        if (deep) {
#pragma unroll
            for (int i = 0; i < C; ++i) rest = max(rest, min(a[i], a[V - 1 - i]));
        }
#pragma unroll
        for (int i = 0; i < C; ++i) a[i] = max(a[i], a[V - 1 - i]);
        sort_bitonic<C, 0>(a);
    }
}
// The sorted N values of this side of D and of the other, of which the C highest: in both.
// deep: `rest` becomes the highest of those left out.
template <int N, int C, int D, int M>
__device__ __forceinline__ void merge_lanes(uint32_t (&a)[M], bool deep, uint32_t& rest) {
    uint32_t b[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const auto p = sides<D>(a[i]);
        a[i] = p.lo;
        b[i] = p.hi;
    }
    if constexpr (N < C) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t u = a[i], v = b[N - 1 - i];
            a[i] = max(u, v);
            a[N + i] = min(u, v);
        }
        sort_bitonic<N, 0>(a);
        sort_bitonic<N, N>(a);
    } else {
        if (deep) {
            const auto p = sides<D>(rest);
            rest = max(p.lo, p.hi);
#pragma unroll
            for (int i = 0; i < N; ++i) rest = max(rest, min(a[i], b[N - 1 - i]));
        }
#pragma unroll
        for (int i = 0; i < N; ++i) a[i] = max(a[i], b[N - 1 - i]);
        sort_bitonic<N, 0>(a);
    }
}
template <int L, int N, int C, int D = 1, int M>
__device__ __forceinline__ void merge_token(uint32_t (&a)[M], bool deep, uint32_t& rest) {
    if constexpr (D < L) {
        merge_lanes<N, C, D>(a, deep, rest);
        merge_token<L, (2 * N < C ? 2 * N : C), C, 2 * D>(a, deep, rest);
    }
}

// the maximum, and the sum, over the L lanes of a token, in each
template <int L>
__device__ __forceinline__ float token_max(float x) { return lanes_max<L>(x); }
template <int L>
__device__ __forceinline__ float token_sum(float x) { return lanes_sum<L>(x); }
template <int L>
__device__ __forceinline__ double token_total(double x) {
    x += dpp64<kDppXor1>(x);
    x += dpp64<kDppXor2>(x);
    x += dpp64<kDppXor7>(x);
    if constexpr (L >= 16) x += dpp64<kDppXor15>(x);
    if constexpr (L >= 32) {
        const auto p = both_sides<16>(x);
        x = p.lo + p.hi;
    }
    if constexpr (L >= 64) {
        const auto p = both_sides<32>(x);
        x = p.lo + p.hi;
    }
    return x;
}
template <int L>
__device__ __forceinline__ bool token_any(bool x) {
    const uint64_t m = __builtin_amdgcn_ballot_w64(x);
    if constexpr (L == 64) return m != 0;
    else return (m >> (threadIdx.x & (64 - L)) & ((uint64_t(1) << L) - 1)) != 0;
}

// bits that order like the float (no NaN), and back
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x);
    return b ^ (uint32_t(int32_t(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

// the other groups of 2^bits lanes in a row whose range of values is above this one's, and
// those that are not below it (groups that are not there are -inf)
template <int ROW, int K = 1>
__device__ __forceinline__ void count_groups(int bits, float low, float high, int& above, int& maybe) {
    if constexpr (K < ROW) {
        if ((K & ((1 << bits) - 1)) == 0) {
            const float ol = other_lane<ROW, K>(low), oh = other_lane<ROW, K>(high);
            above += ol > high;
            maybe += !(oh < low);
        }
        count_groups<ROW, K + 1>(bits, low, high, above, maybe);
    }
}
// A candidate: its packed key, expert, score, key and how many candidates are above it
struct Candidate {
    uint32_t packed;
    int e, rank;
    double s, k;
};
// Whether a candidate of a row surely comes before the next lane's: its key is above, or the
// same at a lower expert (the place in `packed` falls along the experts); what is not to be
// chosen comes last in any order.  off: the scores' common relative error (0: none), which moves
// each key by its own score and so their difference by as much of the greater one, and makes a
// tie only where it moves both alike.
template <int ROW>
__device__ __forceinline__ bool in_order(const Candidate& c, uint32_t places, int r, double off) {
    const double next = dpp64<0x101>(c.k);            // row_shl: lane r gets r + 1's
    const uint32_t place = c.packed & places, next_place = dppu<0x101>(place);
    double tol = 0.0;
    bool alike = true;
    if (off != 0.0) {                                 // (the same in all lanes)
        const double next_s = dpp64<0x101>(c.s);
        tol = off * fmax(c.s, next_s);
        alike = c.s == next_s;
    }
    return r == ROW - 1 || next == kNone || c.k > next + tol ||
           (c.k == next && alike && place > next_place);
}
__device__ __forceinline__ bool goes_before(double ka, uint32_t pa, double kb, uint32_t pb) {
    return ka > kb || (ka == kb && pa > pb);
}
template <int ROW, int Q, int K = 1>
__device__ __forceinline__ void count_above(Candidate (&c)[Q], uint32_t places) {
    if constexpr (K < ROW) {
#pragma unroll
        for (int o = 0; o < Q; ++o) {
            const double k = other_lane<ROW, K>(c[o].k);
            const uint32_t p = other_lane<ROW, K>(c[o].packed & places);
#pragma unroll
            for (int q = 0; q < Q; ++q) c[q].rank += goes_before(k, p, c[q].k, c[q].packed & places);
        }
        count_above<ROW, Q, K + 1>(c, places);
    }
}

// How the experts of a token lie: group g in the 2^bits lanes from g * 2^bits on, `each` a lane.
// A lane reads V logits from its first one on or, where there are fewer, the last V of its
// group, and masks those that the lanes before have (all of them, if none are left for it).
// Groups of fewer than V are read one by one.
struct Spread {
    int bits, each;
    int last;                                         // where a lane's logits begin at most
};

// V consecutive logits from `at` on (-inf past `count`), in one load if they are whole
template <int T, int V>
__device__ __forceinline__ void logits_load(const void* logits, int64_t at, int count, float (&l)[V]) {
    constexpr int W = V * kElem<T> / 4;
    struct __attribute__((packed, aligned(kElem<T>))) Loose { uint32_t w[W]; };
    const char* p = static_cast<const char*>(logits) + at * kElem<T>;
    if (count == V) {
        const Loose u = *reinterpret_cast<const Loose*>(p);
#pragma unroll
        for (int i = 0; i < W; ++i) {
            if constexpr (T == kF32) {
                l[i] = __uint_as_float(u.w[i]);
            } else if constexpr (T == kBf16) {
                l[2 * i] = bf16lo(u.w[i]);
                l[2 * i + 1] = bf16hi(u.w[i]);
            } else {
                const xpu_v2h h = __builtin_bit_cast(xpu_v2h, u.w[i]);
                l[2 * i] = float(h[0]);
                l[2 * i + 1] = float(h[1]);
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) l[i] = i < count ? logit_at<T>(p, 0, 0, i) : -INFINITY;
}

template <int T, int L, int V, int C, int THREADS>
__global__ __launch_bounds__(THREADS) void route_kernel(RouteArgs a, Spread sp, int64_t first_token) {
    constexpr int PER = 64 / L, WAVES = THREADS / 64;
    constexpr int ROW = L < 16 ? L : 16, Q = C / ROW;  // lanes with candidates, and of each
    constexpr uint32_t kPlace = L * V - 1;            // the bits of an expert's place
    const int lane = threadIdx.x & 63, in = lane & (L - 1), r = lane & (ROW - 1);
    const int n = a.E / a.how.groups;
    const int group = in >> sp.bits, part = in & ((1 << sp.bits) - 1);
    const bool there = group < a.how.groups;
    const int first = (there ? group * n : 0) + min(part * sp.each, sp.last);
    const int count = n >= V ? V : there ? max(0, min(sp.each, n - part * sp.each)) : 0;
    const int skip = n < V ? 0 : there ? min(V, max(0, part * sp.each - sp.last)) : V;
    const bool skips = __builtin_amdgcn_ballot_w64(skip != 0) != 0;
    auto mask = [&](float (&l)[V]) {
        if (skips) {
#pragma unroll
            for (int i = 0; i < V; ++i) l[i] = i < skip ? -INFINITY : l[i];
        }
    };
    const bool plain = !a.bias && a.how.groups == 1;  // keys are the logits
    const int64_t t0 = first_token + (int64_t(blockIdx.x) * WAVES + (threadIdx.x >> 6)) * PER;
    if (t0 >= a.T) return;
    const int64_t t = min(t0 + lane / L, a.T - 1);
    float key[V], most = -INFINITY, sum = 1.f;        // key: the logits, then scores, then keys
    bool bad = false, odd = false;
    constexpr float kLog2e = 1.4426950408889634f;
    logits_load<T>(a.logits, t * a.ld + first, count, key);
    {
        float all = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            all += key[i];
            most = fmaxf(most, key[i]);
        }
        // a NaN or infinity anywhere (or a sum that overflows): looked for one by one
        odd = __builtin_amdgcn_ballot_w64(!(fabsf(all) < INFINITY)) != 0;
        if (odd) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                bad |= __builtin_isnan(key[i]) || (!a.how.sigmoid && key[i] == INFINITY);
        }
        mask(key);
    }
    if (!a.how.sigmoid) most = token_max<L>(most);
    // fp32 scores.  A sigmoid s: its exponential off by 2 units (2^-24) and |l| of its
    // argument's rounding, of which s (1 - s) < 1/4 (times |l| < 1/4) counts, the sum's and
    // the reciprocal's 3: under 2^-21.  A softmax's: 2 and the argument's |x|, where
    // |x| e^-|x| < 0.4, the sum's 38 additions of such terms and the reciprocal: under 2^-18
    // of the highest score.
    const bool scores = !plain || (!a.how.sigmoid && !a.how.renormalize);
    if (scores) {
        float e[V];
        if (a.how.sigmoid) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                e[i] = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-key[i] * kLog2e));
        } else {
            const float ref = most == -INFINITY ? 0.f : most;
            sum = 0.f;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                e[i] = __builtin_amdgcn_exp2f((key[i] - ref) * kLog2e);
                sum += e[i];
            }
            sum = token_sum<L>(sum);
            const float share = __builtin_amdgcn_rcpf(sum);
#pragma unroll
            for (int i = 0; i < V; ++i) e[i] *= share;
        }
        if (!plain) {
            float check = 0.f;
            if (odd) {
#pragma unroll
                for (int i = 0; i < V; ++i) e[i] = key[i] == -INFINITY ? -INFINITY : e[i];
            }
            if (a.bias) {
                float b[V];
                logits_load<kF32>(a.bias, first, count, b);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    e[i] += b[i];
                    check += e[i];
                }
                if (__builtin_amdgcn_ballot_w64(!(fabsf(check) < INFINITY))) {
#pragma unroll
                    for (int i = 0; i < V; ++i) bad |= __builtin_isnan(e[i]);
                }
            }
            if (!odd) mask(e);
#pragma unroll
            for (int i = 0; i < V; ++i) key[i] = e[i];
        }
    }
    const float off = plain ? 0.f : a.how.sigmoid ? 0x1p-21f : 0x1p-18f * __builtin_amdgcn_rcpf(sum);
    double sum64 = sum;                               // the softmax's, exact once asked for
    bool sum_exact = false;
    auto exact_sum = [&] {
        float l[V];
        logits_load<T>(a.logits, t * a.ld + first, count, l);
        mask(l);
        double u = 0.0;
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (l[i] != -INFINITY) u += exp(double(l[i]) - double(most));
        sum64 = token_total<L>(u);
        sum_exact = true;
    };
    auto score64 = [&](float x) {
        return a.how.sigmoid ? 1.0 / (1.0 + exp(-double(x))) : exp(double(x) - double(most)) / sum64;
    };
    bool dropped = false;
    if (a.how.groups > 1) {
        float one = -INFINITY, two = -INFINITY;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            two = fmaxf(two, fminf(one, key[i]));
            one = fmaxf(one, key[i]);
        }
        for (int d = 1; d < 1 << sp.bits; d *= 2) {
            const float o = __shfl_xor(one, d), w = __shfl_xor(two, d);
            two = fmaxf(fmaxf(two, w), fminf(one, o));
            one = fmaxf(one, o);
        }
        const float value = two == -INFINITY ? one : one + two;
        const float e = one == -INFINITY ? 0.f : 2.f * off + 0x1p-22f * (fabsf(one) + fabsf(value));
        int above = 0, maybe = 0;                     // groups surely above, and perhaps
        const float low = value - e, high = value + e;
        if constexpr (L <= 16) {
            count_groups<L>(sp.bits, low, high, above, maybe);
        } else {
            for (int g = 0; g < a.how.groups; ++g) {
                const int from = (lane & ~(L - 1)) + (g << sp.bits);
                const float ol = __shfl(low, from), oh = __shfl(high, from);
                if (g == group) continue;
                above += ol > high;
                maybe += !(oh < low);
            }
        }
        // (a group with nothing to choose from is as good in as out)
        dropped = one == -INFINITY || above >= a.how.top_groups;
        const bool open = group < a.how.groups && !dropped && maybe >= a.how.top_groups;
        if (__builtin_amdgcn_ballot_w64(open)) {      // values too near: in 64 bits
            if (!a.how.sigmoid) exact_sum();
            double first64 = kNone, second64 = kNone;
            float l[V];
            logits_load<T>(a.logits, t * a.ld + first, count, l);
            mask(l);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if (l[i] == -INFINITY) continue;
                const double k = score64(l[i]) + (a.bias ? double(a.bias[first + i]) : 0.0);
                second64 = fmax(second64, fmin(first64, k));
                first64 = fmax(first64, k);
            }
            for (int d = 1; d < 1 << sp.bits; d *= 2) {
                const double o = __shfl_xor(first64, d), w = __shfl_xor(second64, d);
                second64 = fmax(fmax(second64, w), fmin(first64, o));
                first64 = fmax(first64, o);
            }
            const double value64 = second64 == kNone ? first64 : first64 + second64;
            above = 0;
            for (int g = 0; g < a.how.groups; ++g) {
                const double o = __shfl(value64, (lane & ~(L - 1)) + (g << sp.bits));
                above += o > value64 || (o == value64 && g < group);
            }
            dropped = above >= a.how.top_groups;
        }
    }
    // (-inf orders below kNothing, and so does what is dropped)
    uint32_t c[V > C ? V : C];
    const uint32_t keep = dropped ? 0u : ~kPlace;
    if (plain) {                                      // a negative zero would order below zero
#pragma unroll                                        // (sums of scores are never one)
        for (int i = 0; i < V; ++i) key[i] += 0.f;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) c[i] = (ordered(key[i]) & keep) | (kPlace - uint32_t(in * V + i));
    // the key behind the candidates where it counts: 65536 tokens of 128 experts in fp32, 16
    // slots 31 us (without it all of them went through route_token: 235)
    const bool deep = L >= 16 && a.top >= C - 1 && (T == kF32 || !plain);
    uint32_t last = 0;
    sort_lane<V, C>(c, deep, last);
    merge_token<L, (V < C ? V : C), C>(c, deep, last);
    if (!deep) last = c[C - 1];
    Candidate mine[Q];
    // the candidates Q ROW + r, in 64 bits
    auto look = [&](int q) {
        Candidate& m = mine[q];
        m.packed = c[q * ROW];
#pragma unroll
        for (int i = 1; i < ROW; ++i) m.packed = r == i ? c[q * ROW + i] : m.packed;
        const int at = int(kPlace - (m.packed & kPlace)) / V, i = int(kPlace - (m.packed & kPlace)) % V;
        const int from = min((at & ((1 << sp.bits) - 1)) * sp.each, sp.last);
        m.e = m.packed >= kNothing ? (at >> sp.bits) * n + from + i : -1;
        m.s = 0.0;
        m.k = kNone;
        m.rank = q * ROW + r;
        if (m.e < 0) return;
        const float x = logit_at<T>(a.logits, t, a.ld, m.e);
        m.s = plain && a.how.renormalize && !a.how.sigmoid ? exp(double(x) - double(most)) : score64(x);
        m.k = plain ? double(x) : m.s + (a.bias ? double(a.bias[m.e]) : 0.0);
    };
    // whether a chosen candidate is above all that order behind `next`
    auto sure = [&](const Candidate& m, uint32_t next) {
        if (m.e < 0 || m.rank >= a.top || next < kNothing) return true;
        // (16-bit logits are whole in the upper bits: equal ones are in order)
        if (plain && T != kF32) return true;
        const float highest = unordered(next | kPlace);
        return m.k > double(highest) + 2.0 * off + (plain ? 0.0 : 0x1p-22 * fabs(double(highest)));
    };
    // (32 candidates are for slots that the first of a lane are too few for)
    bool ordered_now = false;
    if constexpr (C <= 16) {
        look(0);
#pragma unroll
        for (int q = 1; q < Q; ++q) mine[q] = Candidate{0, -1, C, 0.0, kNone};
        // keys nearer than the fp32 sum's error (2^-18 of a score, see above) are looked at again
        // with the exact one
        const bool rough = !plain && !a.how.sigmoid && !sum_exact;
        ordered_now = in_order<ROW>(mine[0], kPlace, r, rough ? 0x1p-16 : 0.0);
        ordered_now &= sure(mine[0], Q > 1 ? c[ROW % C] : last);
    }
    if (__builtin_amdgcn_ballot_w64(!ordered_now)) {
        if (!plain && !a.how.sigmoid && !sum_exact) exact_sum();
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            look(q);
            mine[q].rank = 0;
        }
#pragma unroll
        for (int q = 0; q < Q; ++q)
#pragma unroll
            for (int o = 0; o < Q; ++o)
                if (o != q)
                    mine[q].rank += goes_before(mine[o].k, mine[o].packed & kPlace, mine[q].k,
                                                mine[q].packed & kPlace);
        count_above<ROW, Q>(mine, kPlace);
#pragma unroll
        for (int q = 0; q < Q; ++q) bad |= !sure(mine[q], last);
    }
    double total = 1.0;
    if (a.how.renormalize) {
        total = 0.0;
#pragma unroll
        for (int q = 0; q < Q; ++q) total += mine[q].rank < a.top ? mine[q].s : 0.0;
        total = token_total<ROW>(total);
    }
    bad |= mine[0].e >= 0 && !(total > 1e-200);
    const bool again = token_any<L>(bad);
    if (!again && in < ROW && t0 + lane / L < a.T) {
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            if (mine[q].rank >= a.top) continue;
            a.ids[t * a.top + mine[q].rank] = mine[q].e;
            a.weights[t * a.top + mine[q].rank] =
                mine[q].e >= 0 ? float(double(a.how.scale) * mine[q].s / total) : 0.f;
        }
    }
    uint64_t left = __builtin_amdgcn_ballot_w64(again && in == 0 && t0 + lane / L < a.T);
    while (left) {
        const int who = __builtin_ctzll(left);
        left &= left - 1;
        route_token<T, (L * V + 63) / 64>(a, t0 + who / L);
    }
}

// The gradient, from the logits again: w the weights before the factor scale, g theirs,
//   renormalised:  dl_j = scale w_j (g_j - sum_i g_i w_i) [(1 - s_j) for sigmoid]
//   softmax:       dl_e = scale s_e ([e chosen] g_e - sum_j g_j s_j)
//   sigmoid:       dl_j = scale s_j (1 - s_j) g_j
// zeros elsewhere.  A token with NaN weights (a NaN logit, for softmax also one of +inf, chosen or
// not) has NaNs throughout.  A wave a token, the chosen experts in the first lanes.
struct RouteGradArgs {
    const void* logits;
    const int* ids;
    const float* dweights;
    void* dlogits;
    int64_t ld, T;
    int E, top;
    RouteHow how;
};

// whether a logit makes its token's weights NaN
__device__ __forceinline__ bool spoils(float l, bool sigmoid) {
    return sigmoid ? __builtin_isnan(l) : !(l < INFINITY);
}

template <int T, int V>
__global__ __launch_bounds__(256) void route_grad_kernel(RouteGradArgs a) {
    const int lane = threadIdx.x & 63;
    for (int64_t t = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6); t < a.T; t += int64_t(gridDim.x) * 4) {
        int id = lane < a.top ? a.ids[t * a.top + lane] : -1;
        if (id >= a.E) id = -1;
        const float g = id >= 0 ? a.dweights[t * a.top + lane] : 0.f;
        const float mine = id >= 0 ? logit_at<T>(a.logits, t, a.ld, id) : -INFINITY;
        const bool dense = !a.how.sigmoid && !a.how.renormalize;
        float d = 0.f, p[V], along = 0.f;             // d: the chosen expert's
        bool bad = false;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int e = 64 * i + lane;
            p[i] = e < a.E ? logit_at<T>(a.logits, t, a.ld, e) : -INFINITY;
            bad |= spoils(p[i], a.how.sigmoid);
        }
        const bool spoilt = __builtin_amdgcn_ballot_w64(bad) != 0;
        if (dense) {
            float most = -INFINITY, sum = 0.f;
#pragma unroll
            for (int i = 0; i < V; ++i) most = fmaxf(most, p[i]);
            most = wave_most(most);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                p[i] = p[i] == -INFINITY ? 0.f : expf(p[i] - most);
                sum += p[i];
            }
            sum = wave_total(sum);
            if (sum == 0.f) sum = 1.f;                // (every expert masked: all zeros)
#pragma unroll
            for (int i = 0; i < V; ++i) p[i] /= sum;
            const float s = id >= 0 ? expf(mine - most) / sum : 0.f;
            along = wave_total(g * s);
            d = a.how.scale * s * (g - along);
        } else if (a.how.sigmoid) {
            const float shift = a.how.renormalize ? fminf(0.f, wave_most(mine)) : 0.f;
            const float s = id < 0 ? 0.f : mine >= 0.f ? 1.f / (1.f + expf(-mine))
                                                       : expf(mine - shift) / (1.f + expf(mine));
            const float rest = 1.f / (1.f + expf(mine));           // 1 - sigmoid
            if (a.how.renormalize) {
                const float w = s / wave_total(s);
                along = wave_total(id >= 0 ? g * w : 0.f);
                d = a.how.scale * w * rest * (g - along);
            } else {
                d = a.how.scale * s * rest * g;
            }
        } else {
            const float ref = wave_most(mine);        // (of all lanes)
            const float s = id >= 0 ? expf(mine - ref) : 0.f;
            const float w = s / wave_total(s);
            along = wave_total(id >= 0 ? g * w : 0.f);
            d = a.how.scale * w * (g - along);
        }
        float out[V];
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = dense ? -a.how.scale * p[i] * along : 0.f;
        for (int j = 0; j < a.top; ++j) {
            const int e = __shfl(id, j);
            const float v = __shfl(d, j);
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (e == 64 * i + lane) out[i] = v;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int e = 64 * i + lane;
            if (e >= a.E) continue;
            if (spoilt) out[i] = NAN;
            const int64_t at = t * a.E + e;
            if constexpr (T == kF32) static_cast<float*>(a.dlogits)[at] = out[i];
            else static_cast<uint16_t*>(a.dlogits)[at] = uint16_t(pack2<T>(out[i], 0.f));
        }
    }
}

// 4 consecutive elements of a row of E from e on, whole or element by element
template <int T>
struct __attribute__((packed, aligned(kElem<T>))) Loose4 {
    uint32_t w[kElem<T>];
};
template <int T>
__device__ __forceinline__ void four_load(const void* row, int e, int E, float (&v)[4]) {
    const char* p = static_cast<const char*>(row) + int64_t(e) * kElem<T>;
    if (e + 4 <= E) {
        const Loose4<T> u = *reinterpret_cast<const Loose4<T>*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (T == kF32) v[i] = __uint_as_float(u.w[i]);
            else if constexpr (T == kBf16) v[i] = i & 1 ? bf16hi(u.w[i / 2]) : bf16lo(u.w[i / 2]);
            else v[i] = float(__builtin_bit_cast(xpu_v2h, u.w[i / 2])[i & 1]);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = e + i < E ? logit_at<T>(p, 0, 0, i) : -INFINITY;
}
template <int T>
__device__ __forceinline__ void four_store(void* row, int e, int E, const float (&v)[4]) {
    char* p = static_cast<char*>(row) + int64_t(e) * kElem<T>;
    if (e + 4 <= E) {
        Loose4<T> u;
#pragma unroll
        for (int i = 0; i < kElem<T>; ++i) {
            if constexpr (T == kF32) u.w[i] = __float_as_uint(v[i]);
            else u.w[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
        }
        *reinterpret_cast<Loose4<T>*>(p) = u;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (e + i >= E) continue;
        if constexpr (T == kF32) reinterpret_cast<float*>(p)[i] = v[i];
        else reinterpret_cast<uint16_t*>(p)[i] = uint16_t(pack2<T>(v[i], 0.f));
    }
}

// The same with several tokens a wave, up to 16 slots each: slots in the 16 lanes of a row,
// a token's experts in fours over its L lanes.  The whole row of logits is read, beside the
// ids, not after them (its chosen few lie in as many lines); they are looked up in LDS, and
// gradients go through it to where they are written.  16381 tokens of 256 experts in fp32 10.1 us
// (11.3 to 12.7 with a wave a token and the chosen logits after the ids); the bytes take 6.6 at a
// copy's rate, and the waves wait for 64% of their cycles: loads, LDS, exponentials and stores follow
// one another.  65536 tokens 29 (4.6 TB/s).
template <int T, int L, int V>
__global__ __launch_bounds__(256) void route_grad_rows_kernel(RouteGradArgs a, int64_t first_token) {
    constexpr int PER = 64 / L, F = V / 4;
    __shared__ __align__(16) float lds[4][64 * V];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, in = lane & (L - 1), r = lane & 15;
    const int64_t t0 = first_token + (int64_t(blockIdx.x) * 4 + wave) * PER;
    if (t0 >= a.T) return;
    const int64_t t = min(t0 + lane / L, a.T - 1);
    const bool dense = !a.how.sigmoid && !a.how.renormalize;
    float* row = lds[wave] + (lane & ~(L - 1)) * V;   // the token's
    int id = r < a.top ? a.ids[t * a.top + r] : -1;
    const float weight = r < a.top ? a.dweights[t * a.top + r] : 0.f;
    const char* from = static_cast<const char*>(a.logits) + t * a.ld * kElem<T>;
    float out[F][4], d;                               // d: the chosen expert's
    bool bad = false;
#pragma unroll
    for (int i = 0; i < F; ++i) {
        four_load<T>(from, 4 * (i * L + in), a.E, out[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) bad |= spoils(out[i][j], a.how.sigmoid);
        *reinterpret_cast<float4*>(row + 4 * (i * L + in)) =
            make_float4(out[i][0], out[i][1], out[i][2], out[i][3]);
    }
    if (id >= a.E) id = -1;
    const float g = id >= 0 ? weight : 0.f;
    // (a wave's LDS accesses are in order)
    __builtin_amdgcn_wave_barrier();
    const float mine = id >= 0 ? row[id] : -INFINITY;
    __builtin_amdgcn_wave_barrier();
    if (dense) {
        float most = -INFINITY, sum = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) most = fmaxf(most, out[i / 4][i % 4]);
        most = token_max<L>(most);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float& p = out[i / 4][i % 4];
            p = p == -INFINITY ? 0.f : expf(p - most);
            sum += p;
        }
        sum = token_sum<L>(sum);
        if (sum == 0.f) sum = 1.f;                    // (every expert masked: all zeros)
        const float s = id >= 0 ? expf(mine - most) / sum : 0.f;
        const float along = lanes_sum<16>(g * s);
        d = a.how.scale * s * (g - along);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float& p = out[i / 4][i % 4];
            p = -a.how.scale * (p / sum) * along;
        }
    } else {
        const float highest = lanes_max<16>(mine);
        float s, rest = 1.f;
        if (a.how.sigmoid) {
            const float shift = a.how.renormalize ? fminf(0.f, highest) : 0.f;
            const float up = expf(mine);
            s = id < 0 ? 0.f : mine >= 0.f ? 1.f / (1.f + expf(-mine)) : expf(mine - shift) / (1.f + up);
            rest = 1.f / (1.f + up);                  // 1 - sigmoid
        } else {
            s = id >= 0 ? expf(mine - highest) : 0.f;
        }
        if (a.how.renormalize) {
            const float w = s / lanes_sum<16>(s);
            const float along = lanes_sum<16>(id >= 0 ? g * w : 0.f);
            d = a.how.scale * w * rest * (g - along);
        } else {
            d = a.how.scale * s * rest * g;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) out[i / 4][i % 4] = 0.f;
    }
    if (token_any<L>(bad)) {
        d = NAN;
#pragma unroll
        for (int i = 0; i < V; ++i) out[i / 4][i % 4] = NAN;
    }
#pragma unroll
    for (int i = 0; i < F; ++i)
        *reinterpret_cast<float4*>(row + 4 * (i * L + in)) =
            make_float4(out[i][0], out[i][1], out[i][2], out[i][3]);
    __builtin_amdgcn_wave_barrier();
    if (id >= 0 && in < 16) row[id] = d;
    __builtin_amdgcn_wave_barrier();
    if (t0 + lane / L >= a.T) return;
    char* to = static_cast<char*>(a.dlogits) + t * a.E * kElem<T>;
#pragma unroll
    for (int i = 0; i < F; ++i) {
        const float4 v = *reinterpret_cast<const float4*>(row + 4 * (i * L + in));
        const float u[4] = {v.x, v.y, v.z, v.w};
        if (4 * (i * L + in) < a.E) four_store<T>(to, 4 * (i * L + in), a.E, u);
    }
}

// f(type, logits a lane)
template <class F>
void by_experts(int type, int E, const F& f) {
    auto go = [&](auto t) {
        if (E <= 64) f(t, std::integral_constant<int, 1>{});
        else if (E <= 128) f(t, std::integral_constant<int, 2>{});
        else if (E <= 256) f(t, std::integral_constant<int, 4>{});
        else if (E <= 512) f(t, std::integral_constant<int, 8>{});
        else f(t, std::integral_constant<int, 16>{});
    };
    if (type == kBf16) go(std::integral_constant<int, kBf16>{});
    else if (type == kF16) go(std::integral_constant<int, kF16>{});
    else go(std::integral_constant<int, kF32>{});
}
unsigned token_blocks(int64_t T) {
    const int64_t n = (T + 3) / 4;
    return unsigned(n < kMaxBlocks ? n : kMaxBlocks);
}

}  // namespace

hipError_t moe_route(hipStream_t st, const void* logits, int type, int64_t ld, const float* bias,
                     const RouteHow& how, int* ids, float* weights, int64_t T, int E, int top) {
    const RouteArgs a{logits, bias, ids, weights, ld, T, E, top, how};
    int padded = 1;                                   // groups, each with as many lanes
    while (padded < how.groups) padded *= 2;
    const int n = E / how.groups;
    bool done = false;
    auto go = [&](auto t, auto lanes, auto v, auto candidates) {
        constexpr int L = decltype(lanes)::value, V = decltype(v)::value, TY = decltype(t)::value;
        constexpr int C = decltype(candidates)::value;
        if (done || padded > L || top > (L < 16 ? L : C)) return;
        int bits = 0;
        while (padded << (bits + 1) <= L) ++bits;
        if (n > V << bits) return;
        const Spread sp = n < V ? Spread{bits, (n + (1 << bits) - 1) >> bits, n} : Spread{bits, V, n - V};
        done = true;
        constexpr int64_t per = 64 / L;
        auto launch = [&](auto threads) {
            constexpr int N = decltype(threads)::value;
            constexpr int64_t tokens = N / 64 * per;  // a block
            in_launches(T, kMaxBlocks * tokens, [&](int64_t at, int64_t m) {
                hipLaunchKernelGGL((route_kernel<TY, L, V, C, N>), dim3(unsigned((m + tokens - 1) / tokens)),
                                   dim3(N), 0, st, a, sp, at);
            });
        };
        // small calls in blocks of one wave, which spread over more of the chip, and all with
        // more than 16 slots
        constexpr bool many = L >= 16 && V == 32;     // (for these alone, with up to 16)
        static_assert(!many || kManyTokens >= 2048 * per);
        if constexpr (C > 16) launch(std::integral_constant<int, 64>{});
        else if (many || T >= 2048 * per) launch(std::integral_constant<int, 256>{});
        else if constexpr (!many) launch(std::integral_constant<int, 64>{});
    };
    auto by = [&](auto t) {
        constexpr std::integral_constant<int, 4> k4;
        constexpr std::integral_constant<int, 8> k8;
        constexpr std::integral_constant<int, 16> k16;
        constexpr std::integral_constant<int, 32> k32;
        constexpr std::integral_constant<int, 64> k64;
        if (how.groups == 1 || T >= 65536) {          // (see above)
            go(t, k8, k8, k16);
            go(t, k8, k16, k16);
            go(t, k8, k32, k16);
        }
        go(t, k16, k4, k16);
        go(t, k16, k8, k16);
        go(t, k16, k16, k16);
        if (T >= kManyTokens) {
            go(t, k16, k32, k16);
            go(t, k32, k32, k16);
        }
        go(t, k32, k16, k16);
        go(t, k64, k16, k16);
        go(t, k16, k4, k32);
        go(t, k16, k16, k32);
        go(t, k16, k32, k32);
        go(t, k32, k32, k32);
    };
    if (type == kBf16) by(std::integral_constant<int, kBf16>{});
    else if (type == kF16) by(std::integral_constant<int, kF16>{});
    else by(std::integral_constant<int, kF32>{});
    if (!done)
        by_experts(type, E, [&](auto t, auto v) {
            hipLaunchKernelGGL((route_exact_kernel<decltype(t)::value, decltype(v)::value>),
                               dim3(token_blocks(T)), dim3(256), 0, st, a);
        });
    return hipGetLastError();
}

hipError_t moe_route_grad(hipStream_t st, const void* logits, int type, int64_t ld, const int* ids,
                          const float* dweights, const RouteHow& how, void* dlogits, int64_t T,
                          int E, int top) {
    const RouteGradArgs a{logits, ids, dweights, dlogits, ld, T, E, top, how};
    bool done = false;
    auto go = [&](auto t, auto lanes, auto v) {
        constexpr int L = decltype(lanes)::value, V = decltype(v)::value, TY = decltype(t)::value;
        if (done || E > L * V || top > 16) return;
        done = true;
        constexpr int64_t per = 4 * (64 / L);
        in_launches(T, kMaxBlocks * per, [&](int64_t at, int64_t m) {
            hipLaunchKernelGGL((route_grad_rows_kernel<TY, L, V>), dim3(unsigned((m + per - 1) / per)),
                               dim3(256), 0, st, a, at);
        });
    };
    auto by = [&](auto t) {
        go(t, std::integral_constant<int, 16>{}, std::integral_constant<int, 4>{});
        go(t, std::integral_constant<int, 16>{}, std::integral_constant<int, 8>{});
        go(t, std::integral_constant<int, 16>{}, std::integral_constant<int, 16>{});
        go(t, std::integral_constant<int, 32>{}, std::integral_constant<int, 16>{});
        go(t, std::integral_constant<int, 64>{}, std::integral_constant<int, 16>{});
    };
    if (type == kBf16) by(std::integral_constant<int, kBf16>{});
    else if (type == kF16) by(std::integral_constant<int, kF16>{});
    else by(std::integral_constant<int, kF32>{});
    if (!done)
        by_experts(type, E, [&](auto t, auto v) {
            hipLaunchKernelGGL((route_grad_kernel<decltype(t)::value, decltype(v)::value>),
                               dim3(token_blocks(T)), dim3(256), 0, st, a);
        });
    return hipGetLastError();
}

}  // namespace xpuint8
