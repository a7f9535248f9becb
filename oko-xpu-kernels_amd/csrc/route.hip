// Routing to experts: of E logits a token's `top` experts and their weights.
//
//   s = softmax(l) or sigmoid(l);  key = s + bias;  the value of a group of experts is the
//   sum of its two highest keys;  of the experts in the top_groups groups of highest value
//   the `top` highest keys, ties to the lower index;  weight_j = scale s_j, divided by the
//   sum of the chosen s if renormalised.
//
// An expert whose logit or key is -inf is never chosen; slots left over have id -1 and
// weight 0.  A row with a NaN logit (for softmax +inf too) has NaN weights; its experts are
// chosen by the logits, NaNs last.
//
// Which experts are chosen hangs on keys that may be next to each other, so keys are 64
// bits: a wave a token, lane l holding the experts l, l + 64, ..
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

template <class V>
__device__ __forceinline__ V wave_total(V x) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) x += __shfl_xor(x, d);
    return x;
}
template <class V>
__device__ __forceinline__ V wave_most(V x) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const V y = __shfl_xor(x, d);
        x = y > x ? y : x;
    }
    return x;
}

// the highest key of the wave and its expert (the lowest of equal ones), in every lane
__device__ __forceinline__ void wave_best(double& key, int& e) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const double k = __shfl_xor(key, d);
        const int o = __shfl_xor(e, d);
        if (k > key || (k == key && o < e)) {
            key = k;
            e = o;
        }
    }
}

constexpr double kNone = -__builtin_huge_val();      // not to be chosen
constexpr double kLowest = -1.7976931348623157e308;

template <int T, int V>
__global__ __launch_bounds__(256) void route_kernel(RouteArgs a) {
    const int lane = threadIdx.x & 63;
    for (int64_t t = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6); t < a.T; t += int64_t(gridDim.x) * 4) {
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
}

// The gradient, from the logits again: w the weights before the factor scale, g theirs,
//   renormalised:  dl_j = scale w_j (g_j - sum_i g_i w_i) [(1 - s_j) for sigmoid]
//   softmax:       dl_e = scale s_e ([e chosen] g_e - sum_j g_j s_j)
//   sigmoid:       dl_j = scale s_j (1 - s_j) g_j
// zeros elsewhere.  A wave a token, the chosen experts in the first lanes.
struct RouteGradArgs {
    const void* logits;
    const int* ids;
    const float* dweights;
    void* dlogits;
    int64_t ld, T;
    int E, top;
    RouteHow how;
};

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
#pragma unroll
        for (int i = 0; i < V; ++i) p[i] = 0.f;
        if (dense) {
            float most = -INFINITY, sum = 0.f;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int e = 64 * i + lane;
                p[i] = e < a.E ? logit_at<T>(a.logits, t, a.ld, e) : -INFINITY;
                most = fmaxf(most, p[i]);
            }
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
            const int64_t at = t * a.E + e;
            if constexpr (T == kF32) static_cast<float*>(a.dlogits)[at] = out[i];
            else static_cast<uint16_t*>(a.dlogits)[at] = uint16_t(pack2<T>(out[i], 0.f));
        }
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
    by_experts(type, E, [&](auto t, auto v) {
        hipLaunchKernelGGL((route_kernel<decltype(t)::value, decltype(v)::value>),
                           dim3(token_blocks(T)), dim3(256), 0, st, a);
    });
    return hipGetLastError();
}

hipError_t moe_route_grad(hipStream_t st, const void* logits, int type, int64_t ld, const int* ids,
                          const float* dweights, const RouteHow& how, void* dlogits, int64_t T,
                          int E, int top) {
    const RouteGradArgs a{logits, ids, dweights, dlogits, ld, T, E, top, how};
    by_experts(type, E, [&](auto t, auto v) {
        hipLaunchKernelGGL((route_grad_kernel<decltype(t)::value, decltype(v)::value>),
                           dim3(token_blocks(T)), dim3(256), 0, st, a);
    });
    return hipGetLastError();
}

}  // namespace xpuint8
