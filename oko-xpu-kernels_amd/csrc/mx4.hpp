// MXFP4 on the device (gfx950): blocks of 32 consecutive values of a row share a
// power of two, each value one of {0, .5, 1, 1.5, 2, 3, 4, 6} and a sign (e2m1).
//
// Storage: codes [.., K/2], element 2i in the low half of byte i, so a block is
// 16 bytes; scales [.., mx_scale_width(K)], the exponent of block k biased by 127
// at byte k (255: the block is NaN), the row padded with 127s to whole groups of
// 16 blocks, so that the 16 scale bytes of 512 consecutive values are one aligned
// load.  The padding bytes are never used as scales.
#pragma once

#include "common.hpp"

namespace xpuint8 {

// the element types of activations and results
enum MxType : int { kBf16 = 0, kF16 = 1, kF32 = 2 };

__host__ __device__ inline int64_t mx_scale_width(int64_t K) { return (K + 511) / 512 * 16; }

typedef _Float16 xpu_v2h __attribute__((ext_vector_type(2)));

// Eight values of type T at p (16-byte aligned, or 32 bytes of fp32), as fp32.
// VEC false: any alignment of the element type.
template <int T, bool VEC>
__device__ __forceinline__ void load8(const void* p, float (&v)[8]) {
    if constexpr (T == kF32) {
        const float* f = static_cast<const float*>(p);
        if constexpr (VEC) {
            const float4 a = *reinterpret_cast<const float4*>(f);
            const float4 b = *reinterpret_cast<const float4*>(f + 4);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
            v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = f[i];
        }
    } else {
        uint32_t w[4];
        if constexpr (VEC) {
            const uint4 a = *reinterpret_cast<const uint4*>(p);
            w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
        } else {
            const uint16_t* h = static_cast<const uint16_t*>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = uint32_t(h[2 * i]) | (uint32_t(h[2 * i + 1]) << 16);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (T == kBf16) {
                v[2 * i] = bf16lo(w[i]);
                v[2 * i + 1] = bf16hi(w[i]);
            } else {
                const xpu_v2h h = __builtin_bit_cast(xpu_v2h, w[i]);
                v[2 * i] = float(h[0]);
                v[2 * i + 1] = float(h[1]);
            }
        }
    }
}

// Eight values at d of a row of D, zeros for those past it (the vector form is taken for
// rows of whole, aligned 8s only).
template <int T, bool VEC>
__device__ __forceinline__ void load_row8(const char* row, int64_t d, int64_t D, float (&v)[8]) {
    constexpr int size = T == kF32 ? 4 : 2;
    if constexpr (VEC) {
        load8<T, true>(row + d * size, v);
    } else if (d + 8 <= D) {
        load8<T, false>(row + d * size, v);
    } else {
        for (int i = 0; i < 8; ++i) {
            v[i] = 0.f;
            if (d + i >= D) continue;
            if constexpr (T == kF32) v[i] = reinterpret_cast<const float*>(row)[d + i];
            else if constexpr (T == kBf16) v[i] = bf16_to_f32(reinterpret_cast<const uint16_t*>(row)[d + i]);
            else v[i] = float(reinterpret_cast<const _Float16*>(row)[d + i]);
        }
    }
}

// two fp32 values rounded to a 16-bit type, packed
template <int T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (T == kBf16) return pack_bf16x2(a, b);
    else return __builtin_bit_cast(uint32_t, xpu_v2h{_Float16(a), _Float16(b)});
}

template <int T, bool VEC>
__device__ __forceinline__ void store8(void* p, const float (&v)[8]) {
    if constexpr (T == kF32) {
        float* f = static_cast<float*>(p);
        if constexpr (VEC) {
            *reinterpret_cast<float4*>(f) = make_float4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<float4*>(f + 4) = make_float4(v[4], v[5], v[6], v[7]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = v[i];
        }
    } else {
        const uint4 w = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]),
                                   pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
        if constexpr (VEC) {
            *reinterpret_cast<uint4*>(p) = w;
        } else {
            uint16_t* h = static_cast<uint16_t*>(p);
            const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                h[2 * i] = uint16_t(u[i]);
                h[2 * i + 1] = uint16_t(u[i] >> 16);
            }
        }
    }
}

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

// The scale byte of a block from the bits of its largest magnitude (bits of
// non-negative floats order like their values, infinity and NaN above all):
// floor(log2 amax) - 2 is the exponent field less 2; a maximum below 2^-124,
// subnormals included, takes the smallest scale, 2^-127.
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t amax) {
    const uint32_t e = amax >> 23;
    return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}

// Eight values at the scale of byte e, in one dword: v_cvt_scalef32_pk_fp4_f32
// divides by the power of two in its scale operand's exponent field (0 stands for
// 2^-127), rounds to nearest even and saturates at 6: checked on the device for
// every exponent against the definition.
__device__ __forceinline__ uint32_t mx_encode8(const float (&v)[8], uint32_t e) {
    const float s = __uint_as_float(e << 23);
    uint32_t r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0], v[1], s, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2], v[3], s, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4], v[5], s, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6], v[7], s, 3);
    return r;
}

// The eight values of a dword of codes at the scale of byte e (NaN at 255).
__device__ __forceinline__ void mx_decode8(uint32_t c, uint32_t e, float (&v)[8]) {
    const float s = __uint_as_float(e << 23);
    const xpu_v2f a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 0);
    const xpu_v2f b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 1);
    const xpu_v2f d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 2);
    const xpu_v2f f = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 3);
    v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1];
    v[4] = d[0]; v[5] = d[1]; v[6] = f[0]; v[7] = f[1];
}

}  // namespace xpuint8
