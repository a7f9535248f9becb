// What the MXFP4 products share (mx4_gemm.hip, mx4_dx.hip): the groups of rows, the
// output and the weight as a kernel sees them, direct global->LDS loads.
#pragma once

#include <algorithm>
#include <type_traits>

#include "kernels.hpp"
#include "mx4.hpp"
#include "mx_kernels.hpp"

namespace xpuint8 {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));

template <int T>
constexpr int kSize = T == kF32 ? 4 : 2;

// 16 zero bytes: what a direct load reads in place of an operand's bytes past its end
__device__ __attribute__((aligned(16))) uint8_t g_zero_line[16];

// ------------------------------------------------------------------ groups
// The rows of a block: up to BM consecutive rows of one group (e < E), or of the
// rows that no group has (e == E).  Tiles are numbered group by group; block
// `tile` finds its group by a scan over the offsets, 64 groups at a time.  The
// offsets are device data that no host check has seen: they are clamped to
// [0, R], so that whatever they hold every row index lies in it, and a group
// that ends before it begins has no rows.
struct RowTile {
    int e, row, end;           // rows [row, min(row + BM, end))
};
template <int BM>
__device__ __forceinline__ bool row_tile(const int* offsets, int E, int R, int tile, RowTile& t) {
    if (!offsets) {
        t.e = 0;
        t.row = tile * BM;
        t.end = R;
        return t.row < R;
    }
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int base = 0; base <= E; base += 64) {
        const int e = base + lane;
        int lo = R, hi = R;
        if (e <= E) {
            lo = min(max(offsets[e], 0), R);
            if (e < E) hi = min(max(offsets[e + 1], 0), R);
        }
        const int n = max(hi - lo, 0);
        const int tiles = (n + BM - 1) / BM;
        int incl = tiles;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int v = __shfl_up(incl, d);
            if (lane >= d) incl += v;
        }
        const uint64_t past = __builtin_amdgcn_ballot_w64(before + incl > tile);
        if (past) {
            const int l = __builtin_ctzll(past);
            const int first = __shfl(before + incl - tiles, l);
            t.e = base + l;
            t.row = __shfl(lo, l) + (tile - first) * BM;
            t.end = __shfl(hi, l);
            t.e = __builtin_amdgcn_readfirstlane(t.e);
            t.row = __builtin_amdgcn_readfirstlane(t.row);
            t.end = __builtin_amdgcn_readfirstlane(t.end);
            return true;
        }
        before += __shfl(incl, 63);
    }
    return false;
}

// --------------------------------------------------------------- the output
struct Out {
    char* y;                   // [R, N] of type T, contiguous
    const void* bias;          // [N] or null
    int bias_type;
    int R, N;
    bool vec;                  // four columns at a time: N % 4 == 0 (and y aligned)
    bool vec8;                 // eight
};
// the bias of column n, 0 without one or past N
__device__ __forceinline__ float bias_at(const Out& o, int n) {
    if (!o.bias || n >= o.N) return 0.f;
    if (o.bias_type == kF32) return static_cast<const float*>(o.bias)[n];
    if (o.bias_type == kBf16) return bf16_to_f32(static_cast<const uint16_t*>(o.bias)[n]);
    return float(static_cast<const _Float16*>(o.bias)[n]);
}
template <int T>
__device__ __forceinline__ void store4(const Out& o, int64_t row, int n, const v4f& v) {
    if (n >= o.N) return;
    char* p = o.y + (row * o.N + n) * kSize<T>;
    if (o.vec) {
        if constexpr (T == kF32) *reinterpret_cast<v4f*>(p) = v;
        else *reinterpret_cast<uint2*>(p) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (n + i >= o.N) break;
        if constexpr (T == kF32) reinterpret_cast<float*>(p)[i] = v[i];
        else if constexpr (T == kBf16) reinterpret_cast<uint16_t*>(p)[i] = uint16_t(f32_to_bf16_bits(v[i]));
        else reinterpret_cast<_Float16*>(p)[i] = _Float16(v[i]);
    }
}

// ------------------------------------------------------------------ weights
struct Weight {
    const uint8_t *codes, *scales;     // [E, N, K / 2], [E, N, SW]
    int N, K, SW;
};

__device__ __forceinline__ void dma16(const uint8_t* src, uint8_t* dst) {
#if defined(__HIP_DEVICE_COMPILE__)
    __builtin_amdgcn_global_load_lds(src, (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
#endif
}
__device__ __forceinline__ uint32_t lds_addr(const void* p) {
    return static_cast<uint32_t>(
        reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const void*)p));
}

// the most row tiles of BM rows that R rows in E groups can make, the rows of no
// group included
int64_t most_tiles(bool grouped, int64_t R, int E, int BM) {
    if (!grouped) return (R + BM - 1) / BM;
    return std::min<int64_t>(R, R / BM + E + 1);
}

template <class F>
void by_type(int type, const F& f) {
    if (type == kBf16) f(std::integral_constant<int, kBf16>{});
    else if (type == kF16) f(std::integral_constant<int, kF16>{});
    else f(std::integral_constant<int, kF32>{});
}

Out make_out(void* y, int type, const void* bias, int bias_type, int64_t R, int N) {
    const int size = type == kF32 ? 4 : 2;
    return Out{static_cast<char*>(y), bias, bias_type, int(R), N,
               N % 4 == 0 && reinterpret_cast<uintptr_t>(y) % (4 * size) == 0,
               N % 8 == 0 && reinterpret_cast<uintptr_t>(y) % 16 == 0};
}

}  // namespace
}  // namespace xpuint8
