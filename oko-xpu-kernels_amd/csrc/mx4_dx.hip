// The gradient of an MXFP4 product with respect to its (quantized) x:
//
//   dx[i, k] = sum_n dy[i, n] * wq[e, n, k]     for the rows i of group e
//
// The contraction runs across the weight's blocks, so their scales cannot go to
// the scaled MFMA: the weight's values, exact in bf16, go to the bf16 one
// (v_mfma_f32_16x16x32_bf16), fp32 accumulation, one rounding at the store.  dy is
// bf16, or 2 (fp16) or 3 (fp32) bf16 pieces whose sum is dy exactly (an fp16 value
// has 11 significant bits, an fp32 one 24, a bf16 one 8; mx4_split): the pieces lie
// side by side and the contraction runs over the weight's rows once for each.
#include "mx4_groups.hpp"

namespace xpuint8 {
namespace {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));

// ------------------------------------------------------------------- split
// dy [R, N] as PIECES bf16 pieces, each of `width` columns (zeros past N)
template <int T, int PIECES>
__global__ __launch_bounds__(256) void mx4_split_kernel(const char* __restrict__ dy, int64_t ldy,
                                                        uint16_t* __restrict__ out, int64_t R,
                                                        int N, int width) {
    const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
    const int64_t row = i / width;
    const int n = int(i - row * width);
    if (row >= R) return;
    float v = 0.f;
    if (n < N) {
        const char* p = dy + (row * ldy + n) * kSize<T>;
        if constexpr (T == kF32) v = *reinterpret_cast<const float*>(p);
        else if constexpr (T == kBf16) v = bf16_to_f32(*reinterpret_cast<const uint16_t*>(p));
        else v = float(*reinterpret_cast<const _Float16*>(p));
    }
    uint16_t* o = out + row * (int64_t(width) * PIECES) + n;
#pragma unroll
    for (int q = 0; q < PIECES; ++q) {
        // truncated, not rounded: a piece never exceeds what is left, so the largest
        // values stay finite; what an infinity or NaN leaves is not another one
        uint32_t u = __float_as_uint(v);
        uint32_t h = u >> 16;
        if ((u & 0x7FFFFFFFu) > 0x7F800000u) h |= 0x40u;
        o[int64_t(q) * width] = uint16_t(h);
        v = (u & 0x7F800000u) == 0x7F800000u ? 0.f : v - __uint_as_float(h << 16);
    }
}

// ------------------------------------------------------------------- tiles
// 128 x 128 tiles of dx by a block of 4 waves in 2 x 2, 64 contraction rows a step.
// dy's 128 bytes of a row come by direct loads (chunk c of row r at c ^ ((r >> 1) & 7));
// the weight's 64 rows of 4 blocks one block a thread, which writes the 32 values
// as they lie, 256 bytes a row, for the transposing read ds_read_b64_tr_b16: in each
// group of 16 lanes lane j gives the address of 4 consecutive bf16 and lane i = 4a + b
// receives element b of the vectors of lanes a, a + 4, a + 8, a + 12, so that lanes
// that point at row j / 4, columns 4 (j % 4) of a 4 x 16 block receive its columns.
// Two such reads are a lane's 8 consecutive n of one k.  The 32-byte slot s of row n
// sits at s ^ ((n & 3) | ((n >> 3) & 1) << 2): the 16 rows of one read then cover
// the banks twice, the least for its 512 bytes.
constexpr int kBM = 128, kBK = 128, kStep = 64;

__device__ __forceinline__ int slot_of(int n, int s) { return s ^ ((n & 3) | (((n >> 3) & 1) << 2)); }

__device__ __forceinline__ v4s read_tr(uint32_t at) {
    v4s v = {};
#if defined(__HIP_DEVICE_COMPILE__)
    v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)(uintptr_t(at)));
#endif
    return v;
}

template <int T>
__global__ __launch_bounds__(256) void mx4_dx_kernel(const uint16_t* __restrict__ dy, int64_t ldy,
                                                     int pieces, int width, Weight w,
                                                     const int* __restrict__ offsets, int E,
                                                     Out out, int tiles_k) {
    constexpr int DY = kBM * 128, WT = kStep * 256, STAGE = DY + WT;
    constexpr int TM = 4, TK = 4;
    __shared__ __attribute__((aligned(1024))) uint8_t smem[2 * STAGE];
    const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
    const int wm = wave >> 1, wk = wave & 1;
    RowTile t;
    if (!row_tile<kBM>(offsets, E, out.R, blockIdx.x / tiles_k, t)) return;
    const int k0 = (blockIdx.x % tiles_k) * kBK;
    if (t.e == E) {
        const v4f zero = {0.f, 0.f, 0.f, 0.f};
        for (int i = threadIdx.x; i < kBM * (kBK / 4); i += 256) {
            const int row = t.row + i / (kBK / 4);
            if (row < t.end) store4<T>(out, row, k0 + 4 * (i % (kBK / 4)), zero);
        }
        return;
    }
    const int steps_piece = (width + kStep - 1) / kStep, steps = steps_piece * pieces;
    const char* const dyb = reinterpret_cast<const char*>(dy);
    auto issue_dy = [&](int s) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int b = (wave + 4 * i) * 8, j = b + lane / 8;
            const int c = (lane & 7) ^ ((j >> 1) & 7);
            const int64_t row = min(t.row + j, t.end - 1);
            const uint8_t* p = reinterpret_cast<const uint8_t*>(dyb + row * ldy * 2) + int64_t(s) * 128 + c * 16;
            // past the row's end in its last step (pieces are padded to whole steps)
            if (pieces == 1 && s * kStep + c * 8 >= width) p = g_zero_line;
            dma16(p, smem + (s & 1) * STAGE + b * 128);
        }
    };
    const int nr = threadIdx.x >> 2, cb = threadIdx.x & 3;       // this thread's weight block
    const bool kin = k0 + cb * 32 < w.K;
    uint4 codes;
    uint32_t scale;
    auto load_w = [&](int s) {
        const int n = (s % steps_piece) * kStep + nr;
        codes = make_uint4(0, 0, 0, 0);
        scale = 0;
        if (n < w.N && kin) {
            const int64_t row = int64_t(t.e) * w.N + n;
            codes = *reinterpret_cast<const uint4*>(w.codes + row * (w.K / 2) + k0 / 2 + cb * 16);
            scale = w.scales[row * w.SW + k0 / 32 + cb];
        }
    };
    auto put_w = [&](int s) {
        uint8_t* const row = smem + (s & 1) * STAGE + DY + nr * 256;
        const uint32_t c[4] = {codes.x, codes.y, codes.z, codes.w};
        const float sc = __uint_as_float(scale << 23);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            uint4 v;
            v.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[q], sc, 0));
            v.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[q], sc, 1));
            v.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[q], sc, 2));
            v.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[q], sc, 3));
            *reinterpret_cast<uint4*>(row + slot_of(nr, 2 * cb + q / 2) * 32 + (q & 1) * 16) = v;
        }
    };
    v4f acc[TK][TM];
#pragma unroll
    for (int a = 0; a < TK; ++a)
#pragma unroll
        for (int b = 0; b < TM; ++b) acc[a][b] = v4f{0.f, 0.f, 0.f, 0.f};
    const int drow = wm * 64 + r;
    issue_dy(0);
    load_w(0);
    put_w(0);
    for (int s = 0; s < steps; ++s) {
        wait_loads();
        __syncthreads();                                  // step s is in, s - 1 is read
        if (s + 1 < steps) {
            issue_dy(s + 1);
            load_w(s + 1);
        }
        const uint8_t* const st = smem + (s & 1) * STAGE;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            v8s yf[TM];
            v8bf wf[TK];
            const int pos = ((4 * h + g) ^ ((r >> 1) & 7)) * 16;
#pragma unroll
            for (int b = 0; b < TM; ++b) yf[b] = *reinterpret_cast<const v8s*>(st + (drow + 16 * b) * 128 + pos);
#pragma unroll
            for (int a = 0; a < TK; ++a) {
                v4s part[2];
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const int n = 32 * h + 8 * g + 4 * q + (r >> 2);
                    part[q] = read_tr(lds_addr(st + DY + n * 256 + slot_of(n, wk * 4 + a) * 32 + (r & 3) * 8));
                }
                const v8s v = {part[0][0], part[0][1], part[0][2], part[0][3],
                               part[1][0], part[1][1], part[1][2], part[1][3]};
                wf[a] = __builtin_bit_cast(v8bf, v);
            }
#pragma unroll
            for (int b = 0; b < TM; ++b)
#pragma unroll
                for (int a = 0; a < TK; ++a)
                    acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        wf[a], __builtin_bit_cast(v8bf, yf[b]), acc[a][b], 0, 0, 0);
        }
        if (s + 1 < steps) put_w(s + 1);                  // (the slot that step s - 1 had)
    }
#pragma unroll
    for (int a = 0; a < TK; ++a)
#pragma unroll
        for (int b = 0; b < TM; ++b) {
            const int row = t.row + drow + 16 * b;
            if (row < t.end) store4<T>(out, row, k0 + wk * 64 + 16 * a + 4 * g, acc[a][b]);
        }
}

}  // namespace

int64_t mx4_split_width(int64_t N) { return (N + kStep - 1) / kStep * kStep; }
int mx4_split_pieces(int type) { return type == kBf16 ? 1 : type == kF16 ? 2 : 3; }

hipError_t mx4_split(hipStream_t st, const void* dy, int type, int64_t ldy, void* out, int64_t R,
                     int N) {
    const int width = int(mx4_split_width(N));
    by_type(type, [&](auto T) {
        constexpr int t = decltype(T)::value;
        constexpr int P = t == kBf16 ? 1 : t == kF16 ? 2 : 3;
        hipLaunchKernelGGL((mx4_split_kernel<t, P>), dim3(unsigned((R * width + 255) / 256)),
                           dim3(256), 0, st, static_cast<const char*>(dy), ldy,
                           static_cast<uint16_t*>(out), R, N, width);
    });
    return hipGetLastError();
}

hipError_t mx4_dx(hipStream_t st, const void* dy, int64_t ldy, int pieces, const uint8_t* wc,
                  const uint8_t* ws, const int* offsets, int E, void* dx, int type, int64_t R,
                  int N, int K) {
    const Weight w{wc, ws, N, K, int(mx_scale_width(K))};
    const Out o = make_out(dx, type, nullptr, 0, R, K);
    // pieces lie side by side, mx4_split_width(N) columns each; one piece may end early
    const int width = pieces == 1 ? N : int(mx4_split_width(N));
    const int tiles_k = (K + kBK - 1) / kBK;
    const int64_t tiles = most_tiles(offsets != nullptr, R, E, kBM) * tiles_k;
    by_type(type, [&](auto T) {
        constexpr int t = decltype(T)::value;
        hipLaunchKernelGGL((mx4_dx_kernel<t>), dim3(unsigned(tiles)), dim3(256), 0, st,
                           static_cast<const uint16_t*>(dy), ldy, pieces, width, w, offsets, E, o,
                           tiles_k);
    });
    return hipGetLastError();
}

}  // namespace xpuint8
