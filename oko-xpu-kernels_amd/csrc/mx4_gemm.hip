// MXFP4 products on CDNA4 (v_mfma_scale_f32_16x16x128_f8f6f4):
//
//   y[i, n] = sum_k xq[rows[i], k] * wq[e, n, k] [+ bias[n]]
//             for the rows i of group e, offsets[e] <= i < offsets[e + 1]
//
// xq and wq MXFP4 (mx4.hpp), fp32 accumulation, one rounding at the store.  A
// plain linear is one group of all rows; rows without a list are their own
// index; rows past the last group are written as zeros.
//
// The MFMA multiplies 16 x 128 by 128 x 16 four-bit values; lane l holds 32
// consecutive k of row l % 16, one block, with the block's scale byte in a second
// register, and multiplies each lane's block by the lane's scale.  Which 32 of the
// 128 a lane holds is free as long as both operands agree.  D = A * B takes A from
// the weight and B from x, so a lane ends with four consecutive n of one row of y.
#include <algorithm>
#include <type_traits>

#include "mx4_groups.hpp"

namespace xpuint8 {
namespace {

typedef int v8i __attribute__((ext_vector_type(8)));

// acc += W block (codes w, scale byte I of sw) * X block (codes x, byte I of sx)
template <int I>
__device__ __forceinline__ v4f mfma4(const v4i& w, int sw, const v4i& x, int sx, const v4f& acc) {
    const v8i a = {w[0], w[1], w[2], w[3], 0, 0, 0, 0}, b = {x[0], x[1], x[2], x[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, 4, I, sw, I, sx);
}

// ----------------------------------------------------------------- few rows
// Up to 16 rows a tile: the product reads the weight once and is bound by that.
// A block owns 16 weight rows and all of K, its NW waves every NW-th 512
// values: lane l takes row l % 16 and the blocks 4j + l / 16 (j = 0..3), so a
// load instruction covers 64 consecutive bytes of 16 rows, and the row's 16 scale
// bytes, of which byte l / 16 of dword j belongs to block j.  x is quantized here,
// in the registers of the lane that multiplies it (a lane's operand is exactly one
// block), so there is one launch and no quantized copy; the NW partial sums meet
// in LDS.
template <int T, bool VEC>
__device__ __forceinline__ void quantize_block(const char* p, v4i& codes, int& scale) {
    float v[4][8];
#pragma unroll
    for (int c = 0; c < 4; ++c) load8<T, VEC>(p + c * 8 * kSize<T>, v[c]);
    uint32_t m = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, abs_bits(v[c][i]));
    const uint32_t e = mx_scale_byte(m);
#pragma unroll
    for (int c = 0; c < 4; ++c) codes[c] = int(mx_encode8(v[c], e));
    scale = int(e);
}

template <int T, bool VEC, int NW>
__global__ __launch_bounds__(NW * 64) void mx4_skinny_kernel(
    const char* __restrict__ x, int64_t ldx, const int* __restrict__ rows, int tokens, Weight w,
    const int* __restrict__ offsets, int E, Out out) {
    const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
    RowTile t;
    if (!row_tile<16>(offsets, E, out.R, blockIdx.y, t)) return;
    const int n0 = blockIdx.x * 16;
    const int row = t.row + r;
    if (t.e == E) {                                    // rows of no group
        if (wave == 0 && row < t.end)
            store4<T>(out, row, n0 + 4 * g, v4f{0.f, 0.f, 0.f, 0.f});
        return;
    }
    __shared__ v4f part[NW][64];
    const bool has = row < t.end;
    int src = has ? row : t.row;
    if (rows) src = min(max(rows[src], 0), tokens - 1);
    const char* xrow = x + src * ldx * kSize<T>;
    const int64_t wr = int64_t(t.e) * w.N + min(n0 + r, w.N - 1);
    const uint8_t* wc = w.codes + wr * (w.K / 2);
    const uint8_t* ws = w.scales + wr * w.SW;
    v4f acc = {0.f, 0.f, 0.f, 0.f};
    for (int k0 = wave * 512; k0 < w.K; k0 += NW * 512) {
        v4i wf[4], xf[4];
        int xs[4];
        const uint4 s = *reinterpret_cast<const uint4*>(ws + k0 / 32);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int k = k0 + 128 * j + 32 * g;
            wf[j] = v4i{0, 0, 0, 0};
            if (k < w.K) wf[j] = *reinterpret_cast<const v4i*>(wc + k / 2);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int k = k0 + 128 * j + 32 * g;
            xf[j] = v4i{0, 0, 0, 0};
            xs[j] = 127;
            if (k < w.K && has) quantize_block<T, VEC>(xrow + k * kSize<T>, xf[j], xs[j]);
        }
        const uint32_t sw[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int k = k0 + 128 * j + 32 * g;
            const int b = k < w.K ? int(sw[j] >> (8 * g)) : 127;     // (byte 0 is read)
            acc = mfma4<0>(wf[j], b, xf[j], xs[j], acc);
        }
    }
    part[wave][lane] = acc;
    __syncthreads();
    if (wave != 0 || !has) return;
#pragma unroll
    for (int i = 1; i < NW; ++i) acc += part[i][lane];
    store4<T>(out, row, n0 + 4 * g, acc + bias4(out, n0 + 4 * g));
}

// -------------------------------------------------------------------- tiles
// BM x BN tiles of y by a block of 4 waves in 2 x 2, x already quantized.  K in
// stages of 256 values, 128 bytes of codes a row, which direct global->LDS loads
// bring two stages deep; the 16 scale bytes of 512 values come every other stage.
// A stage row's 16-byte chunk c sits at c ^ ((row >> 1) & 7): the 8 lanes that an
// LDS cycle serves, consecutive rows at one chunk, then cover all banks.  In a
// stage lane group g holds the chunks 2g and 2g + 1 (one an MFMA), so its two
// scale bytes are one 16-bit LDS read.
template <int T, int BM, int BN>
__global__ __launch_bounds__(256) void mx4_tile_kernel(
    const uint8_t* __restrict__ xc, const uint8_t* __restrict__ xs, const int* __restrict__ rows,
    int tokens, Weight w, const int* __restrict__ offsets, int E, Out out, int tiles_n) {
    constexpr int TM = BM / 32, TN = BN / 32;             // MFMA blocks of a wave
    constexpr int ROWS = BM + BN;                         // x rows first
    constexpr int STAGE = ROWS * 128, SCALES = ROWS * 16;
    constexpr int PER = ROWS / 32;                        // code loads a wave a stage
    constexpr int PERS = ROWS / 256;                      // scale loads a wave a stage pair
    static_assert(ROWS % 256 == 0, "whole scale loads");
    __shared__ __attribute__((aligned(1024))) uint8_t smem[2 * STAGE + 2 * SCALES];
    const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
    const int wm = wave >> 1, wn = wave & 1;
    RowTile t;
    if (!row_tile<BM>(offsets, E, out.R, blockIdx.x / tiles_n, t)) return;
    const int n0 = (blockIdx.x % tiles_n) * BN;
    if (t.e == E) {
        const v4f zero = {0.f, 0.f, 0.f, 0.f};
        for (int i = threadIdx.x; i < BM * (BN / 4); i += 256) {
            const int row = t.row + i / (BN / 4);
            if (row < t.end) store4<T>(out, row, n0 + 4 * (i % (BN / 4)), zero);
        }
        return;
    }
    const int K = w.K, KB = K / 2;
    const int stages = (K + 255) / 256;
    // the row of the stage that a lane brings: in units of 16 bytes from the
    // operand's first (32 bits of them reach 64 GB)
    const uint8_t* const wbase = w.codes + int64_t(t.e) * w.N * KB;
    const uint8_t* const wsbase = w.scales + int64_t(t.e) * w.N * w.SW;
    auto source_row = [&](int j) {                        // x row or weight row of stage row j
        if (j < BM) {
            int i = min(t.row + j, t.end - 1);
            if (rows) i = min(max(rows[i], 0), tokens - 1);
            return i;
        }
        return min(n0 + j - BM, w.N - 1);
    };
    uint32_t at[PER], ats[PERS];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int j = (wave + 4 * i) * 8 + lane / 8;
        const int c = (lane & 7) ^ ((j >> 1) & 7);
        at[i] = uint32_t(source_row(j)) * uint32_t(KB / 16) + c;
    }
#pragma unroll
    for (int i = 0; i < PERS; ++i)
        ats[i] = uint32_t(source_row((wave + 4 * i) * 64 + lane)) * uint32_t(w.SW / 16);
    auto issue = [&](int s) {
        uint8_t* const st = smem + (s & 1) * STAGE;
        const bool tail = (s + 1) * 256 > K;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int b = (wave + 4 * i) * 8;             // its first stage row
            const uint8_t* base = b < BM ? xc : wbase;
            const uint8_t* p = base + (uint64_t(at[i] + 8u * s) << 4);
            if (tail) {
                const int j = b + lane / 8;
                const int c = (lane & 7) ^ ((j >> 1) & 7);
                if (s * 256 + c * 32 >= K) p = g_zero_line;
            }
            dma16(p, st + b * 128);
        }
        if ((s & 1) == 0) {
            uint8_t* const sc = smem + 2 * STAGE + ((s >> 1) & 1) * SCALES;
#pragma unroll
            for (int i = 0; i < PERS; ++i) {
                const int b = (wave + 4 * i) * 64;
                const uint8_t* base = b < BM ? xs : wsbase;
                dma16(base + (uint64_t(ats[i] + uint32_t(s >> 1)) << 4), sc + b * 16);
            }
        }
    };
    v4f acc[TN][TM];
#pragma unroll
    for (int a = 0; a < TN; ++a)
#pragma unroll
        for (int b = 0; b < TM; ++b) acc[a][b] = v4f{0.f, 0.f, 0.f, 0.f};
    issue(0);
    const int xrow = wm * (BM / 2) + r, wrow = BM + wn * (BN / 2) + r;
    for (int s = 0; s < stages; ++s) {
        wait_loads();
        __syncthreads();                                  // stage s landed, s - 1 is read
        if (s + 1 < stages) issue(s + 1);
        const uint8_t* const st = smem + (s & 1) * STAGE;
        const uint8_t* const sc = smem + 2 * STAGE + ((s >> 1) & 1) * SCALES + (s & 1) * 8 + 2 * g;
        // blocks past K hold zero codes; their scales may be anything
        const int left = K - s * 256;
        int sx[TM], sw[TN];
#pragma unroll
        for (int b = 0; b < TM; ++b) sx[b] = *reinterpret_cast<const uint16_t*>(sc + (xrow + 16 * b) * 16);
#pragma unroll
        for (int a = 0; a < TN; ++a) sw[a] = *reinterpret_cast<const uint16_t*>(sc + (wrow + 16 * a) * 16);
        if (left < 256) {
            const int keep = (64 * g < left ? 0xFF : 0) | (64 * g + 32 < left ? 0xFF00 : 0);
#pragma unroll
            for (int b = 0; b < TM; ++b) sx[b] &= keep;
#pragma unroll
            for (int a = 0; a < TN; ++a) sw[a] &= keep;
        }
        auto half = [&](auto H) {
            constexpr int h = decltype(H)::value;
            v4i xf[TM], wf[TN];
            const int pos = ((2 * g + h) ^ ((r >> 1) & 7)) * 16;
#pragma unroll
            for (int b = 0; b < TM; ++b) xf[b] = *reinterpret_cast<const v4i*>(st + (xrow + 16 * b) * 128 + pos);
#pragma unroll
            for (int a = 0; a < TN; ++a) wf[a] = *reinterpret_cast<const v4i*>(st + (wrow + 16 * a) * 128 + pos);
#pragma unroll
            for (int b = 0; b < TM; ++b)
#pragma unroll
                for (int a = 0; a < TN; ++a) acc[a][b] = mfma4<h>(wf[a], sw[a], xf[b], sx[b], acc[a][b]);
        };
        half(std::integral_constant<int, 0>{});
        half(std::integral_constant<int, 1>{});
    }
#pragma unroll
    for (int a = 0; a < TN; ++a) {
        const int n = n0 + wn * (BN / 2) + 16 * a + 4 * g;
        const v4f b4 = bias4(out, n);
#pragma unroll
        for (int b = 0; b < TM; ++b) {
            const int row = t.row + xrow + 16 * b;
            if (row < t.end) store4<T>(out, row, n, acc[a][b] + b4);
        }
    }
}

}  // namespace

// Up to 16 rows a group on average the weight's bytes are the product's time and
// the quantizer's launch would be most of the rest.
bool mx4_fused(int64_t R, bool grouped, int E) { return R <= 16 * int64_t(grouped ? E : 1); }

hipError_t mx4_product_fused(hipStream_t st, const void* x, int type, int64_t ldx,
                             const int* rows, int64_t tokens, const uint8_t* wc,
                             const uint8_t* ws, const int* offsets, int E, void* y,
                             const void* bias, int bias_type, int64_t R, int N, int K) {
    constexpr int NW = 8;
    const Weight w{wc, ws, N, K, int(mx_scale_width(K))};
    const Out o = make_out(y, type, bias, bias_type, R, N);
    const int size = type == kF32 ? 4 : 2;
    const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && (ldx * size) % 16 == 0;
    const dim3 grid(unsigned((N + 15) / 16), unsigned(most_tiles(offsets != nullptr, R, E, 16)));
    by_type(type, [&](auto T) {
        constexpr int t = decltype(T)::value;
        if (vec)
            hipLaunchKernelGGL((mx4_skinny_kernel<t, true, NW>), grid, dim3(NW * 64), 0, st,
                               static_cast<const char*>(x), ldx, rows, int(tokens), w, offsets, E, o);
        else
            hipLaunchKernelGGL((mx4_skinny_kernel<t, false, NW>), grid, dim3(NW * 64), 0, st,
                               static_cast<const char*>(x), ldx, rows, int(tokens), w, offsets, E, o);
    });
    return hipGetLastError();
}

hipError_t mx4_product(hipStream_t st, const uint8_t* xc, const uint8_t* xs, const int* rows,
                       int64_t tokens, const uint8_t* wc, const uint8_t* ws, const int* offsets,
                       int E, void* y, int type, const void* bias, int bias_type, int64_t R, int N,
                       int K) {
    const Weight w{wc, ws, N, K, int(mx_scale_width(K))};
    const Out o = make_out(y, type, bias, bias_type, R, N);
    by_type(type, [&](auto T) {
        constexpr int t = decltype(T)::value;
        constexpr int BM = 128, BN = 128;
        const int tiles_n = (N + BN - 1) / BN;
        const int64_t tiles = most_tiles(offsets != nullptr, R, E, BM) * tiles_n;
        hipLaunchKernelGGL((mx4_tile_kernel<t, BM, BN>), dim3(unsigned(tiles)), dim3(256), 0, st,
                           xc, xs, rows, int(tokens), w, offsets, E, o, tiles_n);
    });
    return hipGetLastError();
}

}  // namespace xpuint8
