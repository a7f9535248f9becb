// Rotary positions on several axes.  Pair j of a head turns by the angle
// position[axis[j]] * inv_freq[j]: (a, b) becomes (a cos - b sin, b cos + a sin), a and b
// P apart (split half) or next to each other; elements past 2 P stay as they are.  The
// gradient is the same by the opposite angle.
//
// HBM-bound: q and k are read and written once, in one launch.  A block takes a few
// positions: its threads first make their cosines and sines, one pair each, into LDS
// (once a position, for all of its heads), then walk over the heads in pieces of 16
// values, 8 pairs.  Angles are reduced to a part of a turn in 64 bits, since in 32 a far
// position would lose it: at position 10^6 half a unit of the product is 0.03 of a radian.
#include "block_kernels.hpp"
#include "mx_kernels.hpp"
#include "rows.hpp"

namespace xpuint8 {
namespace {

constexpr int kMaxPairs = 512;

struct RotaryArgs {
    Heads q, k;                     // k.H = 0: q alone
    Positions pos;
    const double* inv_freq;
    const int* axis;
    int64_t S, tokens;
    int P, D, per_head;             // pieces a head: of 8 pairs, then 16 unturned values
    int turned;                     // pieces of pairs
    float sign;
};

__device__ __forceinline__ double position_of(const Positions& p, int axis, int64_t b, int64_t s) {
    if (axis < 0 || axis >= p.axes) return 0.0;
    const int64_t at = axis * p.a + b * p.b + s * p.s;
    if (p.type == 0) return double(static_cast<const int32_t*>(p.p)[at]);
    if (p.type == 1) return double(static_cast<const int64_t*>(p.p)[at]);
    return double(static_cast<const float*>(p.p)[at]);
}

template <int T>
__device__ __forceinline__ float element(const char* p, int64_t i) {
    if constexpr (T == kF32) return reinterpret_cast<const float*>(p)[i];
    else if constexpr (T == kBf16) return bf16_to_f32(reinterpret_cast<const uint16_t*>(p)[i]);
    else return float(reinterpret_cast<const _Float16*>(p)[i]);
}
template <int T>
__device__ __forceinline__ void put(char* p, int64_t i, float v) {
    if constexpr (T == kF32) reinterpret_cast<float*>(p)[i] = v;
    else reinterpret_cast<uint16_t*>(p)[i] = uint16_t(pack2<T>(v, 0.f));
}

// Piece c of a head's row x to its place in out; cs: the position's cosines and sines.
template <int T, bool SPLIT>
__device__ __forceinline__ void turn_piece(const RotaryArgs& a, const char* x, char* out, int c,
                                           const float2* cs) {
    if (c >= a.turned) {               // unturned values, as they lie
        const int64_t d = 2 * a.P + 16 * int64_t(c - a.turned);
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (d + 8 * i < a.D)
                piece_store<T, false>(out, d + 8 * i, a.D, piece_load<T, false>(x, d + 8 * i, a.D));
        return;
    }
    const int p0 = 8 * c;
    if (p0 + 8 <= a.P) {
        const int64_t d0 = SPLIT ? p0 : 2 * p0, d1 = SPLIT ? a.P + p0 : 2 * p0 + 8;
        float u[8], v[8];
        piece_expand(piece_load<T, true>(x, d0, a.D), u);
        piece_expand(piece_load<T, true>(x, d1, a.D), v);
        float f[2][8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 t = cs[p0 + i];
            const float p = SPLIT ? u[i] : (i < 4 ? u : v)[(2 * i) & 7];
            const float q = SPLIT ? v[i] : (i < 4 ? u : v)[(2 * i + 1) & 7];
            const float first = p * t.x - q * t.y, second = q * t.x + p * t.y;
            if (SPLIT) {
                f[0][i] = first;
                f[1][i] = second;
            } else {
                f[i >> 2][(2 * i) & 7] = first;
                f[i >> 2][(2 * i + 1) & 7] = second;
            }
        }
        piece_store<T, true>(out, d0, a.D, piece_round<T>(f[0]));
        piece_store<T, true>(out, d1, a.D, piece_round<T>(f[1]));
        return;
    }
    for (int p = p0; p < a.P; ++p) {   // the last pairs, fewer than 8
        const int64_t d0 = SPLIT ? p : 2 * p, d1 = SPLIT ? a.P + p : 2 * p + 1;
        const float u = element<T>(x, d0), v = element<T>(x, d1);
        const float2 t = cs[p];
        put<T>(out, d0, u * t.x - v * t.y);
        put<T>(out, d1, v * t.x + u * t.y);
    }
}

template <int T, bool SPLIT, int TOKENS>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
    __shared__ float2 cs[TOKENS * kMaxPairs];
    const int H = a.q.H + a.k.H;
    for (int64_t t0 = int64_t(blockIdx.x) * TOKENS; t0 < a.tokens; t0 += int64_t(gridDim.x) * TOKENS) {
        const int n = int(a.tokens - t0 < TOKENS ? a.tokens - t0 : TOKENS);
        for (int i = threadIdx.x; i < n * a.P; i += 256) {
            const int t = i / a.P, p = i - t * a.P;
            const int64_t b = (t0 + t) / a.S, s = (t0 + t) - b * a.S;
            const double turns = position_of(a.pos, a.axis[p], b, s) * a.inv_freq[p] *
                                 0.15915494309189535;          // 1 / 2 pi
            const float part = float(turns - rint(turns));
            float sine, cosine;
            sincospif(2.0f * part, &sine, &cosine);
            cs[t * kMaxPairs + p] = make_float2(cosine, sine * a.sign);
        }
        __syncthreads();
        const int units = n * H * a.per_head;
        for (int u = threadIdx.x; u < units; u += 256) {
            const int row = u / a.per_head, c = u - row * a.per_head;
            const int t = row / H, h = row - t * H;
            const int64_t b = (t0 + t) / a.S, s = (t0 + t) - b * a.S;
            const bool is_q = h < a.q.H;
            const Heads& w = is_q ? a.q : a.k;
            const int64_t hh = is_q ? h : h - a.q.H;
            const char* x = static_cast<const char*>(w.x) +
                            (b * w.x_b + s * w.x_s + hh * w.x_h) * kElem<T>;
            char* out = static_cast<char*>(w.out) + (b * w.o_b + s * w.o_s + hh * w.o_h) * kElem<T>;
            turn_piece<T, SPLIT>(a, x, out, c, cs + t * kMaxPairs);
        }
        __syncthreads();
    }
}

}  // namespace

hipError_t rope_axes(hipStream_t st, const Heads& q, const Heads& k, int type,
                     const Positions& positions, const double* inv_freq, const int* axis, int P,
                     bool inverse, bool split_half, int64_t B, int64_t S, int D) {
    RotaryArgs a{q, k, positions, inv_freq, axis, S, B * S, P, D, 0, 0, inverse ? -1.f : 1.f};
    a.turned = (P + 7) / 8;
    a.per_head = a.turned + (D - 2 * P + 15) / 16;
    auto go = [&](auto t, auto split) {
        constexpr int T = decltype(t)::value;
        constexpr bool SPLIT = decltype(split)::value;
        const int64_t n = (a.tokens + 3) / 4, most = kMaxBlocks;
        hipLaunchKernelGGL((rotary_kernel<T, SPLIT, 4>), dim3(unsigned(n < most ? n : most)),
                           dim3(256), 0, st, a);
    };
    auto by_split = [&](auto t) {
        if (split_half) go(t, std::true_type{});
        else go(t, std::false_type{});
    };
    if (type == kBf16) by_split(std::integral_constant<int, kBf16>{});
    else if (type == kF16) by_split(std::integral_constant<int, kF16>{});
    else by_split(std::integral_constant<int, kF32>{});
    return hipGetLastError();
}

}  // namespace xpuint8
