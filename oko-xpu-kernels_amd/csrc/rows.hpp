// Pieces of rows on the device: 8 consecutive values of a row of any alignment, and
// sums and maxima over the lanes of a wave, for the row operators (norm.hip, rotary.hip,
// route.hip).
//
// gfx950 takes 16-byte global accesses at any address of the element's alignment, so a
// row that starts anywhere (an odd row length, a column slice) is read and written in
// the same instructions as an aligned one; only a row's last piece, if it is cut, goes
// element by element.
#pragma once

#include "mx4.hpp"

namespace xpuint8 {

template <int T>
constexpr int kElem = T == kF32 ? 4 : 2;

// 8 values as they lie in memory
template <int T>
struct Piece8 {
    uint32_t w[T == kF32 ? 8 : 4];
};
template <int T>
struct __attribute__((packed, aligned(T == kF32 ? 4 : 2))) Loose8 {
    uint32_t w[T == kF32 ? 8 : 4];
};

// The piece at d < n of a row of n.  EVEN: n is a multiple of 8, no piece is cut.  A cut one
// is read with what lies before it (its row has at least 8 values, or goes one by one) and
// shifted to its place, zeros past its end; it is written in runs of 4, 2 and 1.
template <int T, bool EVEN>
__device__ __forceinline__ Piece8<T> piece_load(const void* row, int64_t d, int64_t n) {
    constexpr int W = int(sizeof(Piece8<T>::w) / 4);
    Piece8<T> p;
    if (EVEN || d + 8 <= n) {
        const auto* q = reinterpret_cast<const Loose8<T>*>(static_cast<const char*>(row) + d * kElem<T>);
#pragma unroll
        for (int i = 0; i < W; ++i) p.w[i] = q->w[i];
        return p;
    }
    if (n >= 8) {
        const auto* q = reinterpret_cast<const Loose8<T>*>(static_cast<const char*>(row) + (n - 8) * kElem<T>);
#pragma unroll
        for (int i = 0; i < W; ++i) p.w[i] = q->w[i];
        const int s = int(d + 8 - n);                 // 1..7 values too early
        if constexpr (T == kF32) {
#pragma unroll
            for (int b = 4; b; b /= 2)
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    p.w[i] = s & b ? (i + b < 8 ? p.w[i + b < 8 ? i + b : 0] : 0u) : p.w[i];
        } else {
            uint64_t lo = p.w[0] | uint64_t(p.w[1]) << 32, hi = p.w[2] | uint64_t(p.w[3]) << 32;
            if (s >= 4) {
                lo = hi >> (16 * (s - 4));
                hi = 0;
            } else {
                lo = lo >> (16 * s) | hi << (64 - 16 * s);
                hi >>= 16 * s;
            }
            p.w[0] = uint32_t(lo);
            p.w[1] = uint32_t(lo >> 32);
            p.w[2] = uint32_t(hi);
            p.w[3] = uint32_t(hi >> 32);
        }
        return p;
    }
#pragma unroll
    for (int i = 0; i < W; ++i) p.w[i] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (d + i >= n) continue;
        if constexpr (T == kF32) p.w[i] = static_cast<const uint32_t*>(row)[d + i];
        else p.w[i / 2] |= uint32_t(static_cast<const uint16_t*>(row)[d + i]) << (16 * (i & 1));
    }
    return p;
}

template <int T, bool EVEN>
__device__ __forceinline__ void piece_store(void* row, int64_t d, int64_t n, const Piece8<T>& p) {
    constexpr int W = int(sizeof(Piece8<T>::w) / 4);
    struct __attribute__((packed, aligned(kElem<T>))) Four { uint32_t w[kElem<T>]; };
    struct __attribute__((packed, aligned(kElem<T>))) Two { uint32_t w[kElem<T> / 2]; };
    char* at = static_cast<char*>(row) + d * kElem<T>;
    if (EVEN || d + 8 <= n) {
        auto* q = reinterpret_cast<Loose8<T>*>(at);
#pragma unroll
        for (int i = 0; i < W; ++i) q->w[i] = p.w[i];
        return;
    }
    const int c = int(n - d);                         // 1..7 values
    if (c & 4) {
        Four f;
#pragma unroll
        for (int i = 0; i < W / 2; ++i) f.w[i] = p.w[i];
        *reinterpret_cast<Four*>(at) = f;
    }
    const bool second = c & 4;                        // where the rest begins
    if (c & 2) {
        Two t;
#pragma unroll
        for (int i = 0; i < W / 4; ++i) t.w[i] = second ? p.w[W / 2 + i] : p.w[i];
        *reinterpret_cast<Two*>(at + (c & 4) * kElem<T>) = t;
    }
    if (c & 1) {                                      // value c - 1, of an even place
        const uint32_t a = second ? p.w[W / 2] : p.w[0], b = second ? p.w[W / 2 + W / 4] : p.w[W / 4];
        const uint32_t v = c & 2 ? b : a;
        if constexpr (T == kF32) *reinterpret_cast<uint32_t*>(at + (c - 1) * 4) = v;
        else *reinterpret_cast<uint16_t*>(at + (c - 1) * 2) = uint16_t(v);
    }
}

template <int T>
__device__ __forceinline__ void piece_expand(const Piece8<T>& p, float (&v)[8]) {
    if constexpr (T == kF32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(p.w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (T == kBf16) {
                v[2 * i] = bf16lo(p.w[i]);
                v[2 * i + 1] = bf16hi(p.w[i]);
            } else {
                const xpu_v2h h = __builtin_bit_cast(xpu_v2h, p.w[i]);
                v[2 * i] = float(h[0]);
                v[2 * i + 1] = float(h[1]);
            }
        }
    }
}
template <int T>
__device__ __forceinline__ Piece8<T> piece_round(const float (&v)[8]) {
    Piece8<T> p;
    if constexpr (T == kF32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) p.w[i] = __float_as_uint(v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) p.w[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
    }
    return p;
}

// 8 values of a vector of n whose type is known at run time only; ones for none, zeros
// past its end
template <bool EVEN>
__device__ __forceinline__ void vector_load(const void* w, int type, int64_t d, int64_t n,
                                            float (&v)[8]) {
    if (!w) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 1.f;
    } else if (type == kBf16) {
        piece_expand(piece_load<kBf16, EVEN>(w, d, n), v);
    } else if (type == kF16) {
        piece_expand(piece_load<kF16, EVEN>(w, d, n), v);
    } else {
        piece_expand(piece_load<kF32, EVEN>(w, d, n), v);
    }
}

// the values of two lanes D (16 or 32) apart, in both of them, without a trip through LDS
template <class V>
struct Both {
    V lo, hi;
};
template <int D>
__device__ __forceinline__ Both<uint32_t> both_sides(uint32_t x) {
    if constexpr (D == 16) {
        const auto p = __builtin_amdgcn_permlane16_swap(x, x, false, false);
        return {p[0], p[1]};
    } else {
        const auto p = __builtin_amdgcn_permlane32_swap(x, x, false, false);
        return {p[0], p[1]};
    }
}
template <int D>
__device__ __forceinline__ Both<float> both_sides(float x) {
    const auto p = both_sides<D>(__float_as_uint(x));
    return {__uint_as_float(p.lo), __uint_as_float(p.hi)};
}
template <int D>
__device__ __forceinline__ Both<int> both_sides(int x) {
    const auto p = both_sides<D>(uint32_t(x));
    return {int(p.lo), int(p.hi)};
}
template <int D>
__device__ __forceinline__ Both<double> both_sides(double x) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const auto l = both_sides<D>(uint32_t(b)), h = both_sides<D>(uint32_t(b >> 32));
    return {__builtin_bit_cast(double, uint64_t(h.lo) << 32 | l.lo),
            __builtin_bit_cast(double, uint64_t(h.hi) << 32 | l.hi)};
}

// The sum over N (8, 16, 32 or 64) consecutive lanes, in every one of them: DPP inside
// a row of 16 lanes, whose steps each add two disjoint groups of equal partial sums,
// then across rows.  The order is fixed.
template <int N>
__device__ __forceinline__ float lanes_sum(float x) {
    x += dpp<kDppXor1>(x);
    x += dpp<kDppXor2>(x);
    x += dpp<kDppXor7>(x);
    if constexpr (N >= 16) x += dpp<kDppXor15>(x);
    if constexpr (N >= 32) {
        const auto p = both_sides<16>(x);
        x = p.lo + p.hi;
    }
    if constexpr (N >= 64) {
        const auto p = both_sides<32>(x);
        x = p.lo + p.hi;
    }
    return x;
}
template <int N>
__device__ __forceinline__ float lanes_max(float x) {
    x = fmaxf(x, dpp<kDppXor1>(x));
    x = fmaxf(x, dpp<kDppXor2>(x));
    x = fmaxf(x, dpp<kDppXor7>(x));
    if constexpr (N >= 16) x = fmaxf(x, dpp<kDppXor15>(x));
    if constexpr (N >= 32) {
        const auto p = both_sides<16>(x);
        x = fmaxf(p.lo, p.hi);
    }
    if constexpr (N >= 64) {
        const auto p = both_sides<32>(x);
        x = fmaxf(p.lo, p.hi);
    }
    return x;
}


// the greater of two numbers, NaN if either is one (fmaxf gives the other one)
__device__ __forceinline__ float greater_or_nan(float a, float b) {
    return __builtin_elementwise_maximum(a, b);
}
template <int N>
__device__ __forceinline__ float lanes_max_or_nan(float x) {
    x = greater_or_nan(x, dpp<kDppXor1>(x));
    x = greater_or_nan(x, dpp<kDppXor2>(x));
    x = greater_or_nan(x, dpp<kDppXor7>(x));
    if constexpr (N >= 16) x = greater_or_nan(x, dpp<kDppXor15>(x));
    if constexpr (N >= 32) {
        const auto p = both_sides<16>(x);
        x = greater_or_nan(p.lo, p.hi);
    }
    if constexpr (N >= 64) {
        const auto p = both_sides<32>(x);
        x = greater_or_nan(p.lo, p.hi);
    }
    return x;
}

}  // namespace xpuint8
