// The gradient of an MXFP4 product with respect to its (quantized) x:
//
//   dx[i, k] = sum_n dy[i, n] * wq[e, n, k]     for the rows i of group e
//
// The contraction runs across the weight's blocks, so their scales cannot go to
// the scaled MFMA: the weight's values, exact in bf16, go to the bf16 one
// (v_mfma_f32_16x16x32_bf16), fp32 accumulation, one rounding at the store.  dy is
// bf16, or 2 (fp16) or 3 (fp32) bf16 pieces whose sum is dy (an fp16 value has 11
// significant bits, an fp32 one 24, a bf16 one 8; mx4_split): exactly, but for an fp32's
// bits below bf16's least subnormal, 2^-133, which values under 2^-109 can have and which
// are dropped.  The pieces lie side by side and the contraction runs over the weight's
// rows once for each.
#include "mx4_tiles.hpp"

namespace xpuint8 {
namespace {

// ------------------------------------------------------------------- split
// dy [R, N] as PIECES bf16 pieces, each of `width` columns (zeros past N); a thread takes 8
// columns, in one load where dy's rows are whole, aligned 8s (VEC).  Bound by its bytes.
template <int T, bool VEC, int PIECES>
__global__ __launch_bounds__(256) void mx4_split_kernel(const char* __restrict__ dy, int64_t ldy,
                                                        uint16_t* __restrict__ out, int64_t R,
                                                        int N, int width) {
    const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
    const int64_t row = i / (width / 8);
    const int n = int(i - row * (width / 8)) * 8;
    if (row >= R) return;
    const char* p = dy + (row * ldy + n) * kSize<T>;
    float v[8];
    if (n + 8 <= N) {
        load8<T, VEC>(p, v);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[j] = 0.f;
            if (n + j >= N) continue;
            if constexpr (T == kF32) v[j] = reinterpret_cast<const float*>(p)[j];
            else if constexpr (T == kBf16) v[j] = bf16_to_f32(reinterpret_cast<const uint16_t*>(p)[j]);
            else v[j] = float(reinterpret_cast<const _Float16*>(p)[j]);
        }
    }
    uint16_t* o = out + row * (int64_t(width) * PIECES) + n;
#pragma unroll
    for (int q = 0; q < PIECES; ++q) {
        uint32_t h[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            // truncated, not rounded: a piece never exceeds what is left, so the largest
            // values stay finite; what an infinity or NaN leaves is not another one
            const uint32_t u = __float_as_uint(v[j]);
            h[j] = u >> 16;
            if ((u & 0x7FFFFFFFu) > 0x7F800000u) h[j] |= 0x40u;
            v[j] = (u & 0x7F800000u) == 0x7F800000u ? 0.f : v[j] - __uint_as_float(h[j] << 16);
        }
        *reinterpret_cast<uint4*>(o + int64_t(q) * width) =
            make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
    }
}

// ------------------------------------------------------------------- tiles
// BM x BK tiles of dx by a block of 4 waves in WM x 4 / WM (of two by rows, each has every
// other 16 of them), 64 contraction rows a stage (two MFMAs of each block); dy in
// three LDS slots, the weight in two.  While a stage's first half runs, a wave reads the
// second half's fragments; one wait and barrier then mean that every wave has read the
// stage, and that the next one is in; while the second half runs, it reads the next
// stage's first fragments, requests dy three stages ahead into the slot by direct loads,
// and writes the weight's rows of two stages ahead as bf16 from the codes and scales that
// it loaded two stages before (a thread BK / 4 consecutive values).
// (One slot and one stage less of each: 5 to 13% slower.  A ring of 32-row steps with a
// load four steps ahead, as the forward product's: slower at 128 x 128; dy's rows then
// come in 64-byte pieces, and the L2's requests, not its bytes, bound such tiles.)
// Bound by the LDS (96 KB a stage and 128 x 128 tile, 768 cycles) beside the MFMAs (512):
// 8192^3 in two pieces 1.20 PFLOP/s, 16380 x 2816 -> 2048 in 32 groups 270 us, 0.70.
//
// dy's 128 bytes of a row: chunk c (16 bytes) at c ^ ((row >> 1) & 7).  The weight's rows
// lie as they come, 2 BK bytes each, for the transposing read ds_read_b64_tr_b16: in
// each group of 16 lanes lane j gives the address of 4 consecutive bf16 and lane i = 4a + b
// receives element b of the vectors of lanes a, a + 4, a + 8, a + 12, so that lanes which
// point at row j / 4, columns 4 (j % 4) of a 4 x 16 block receive its columns.  Two such
// reads are a lane's 8 consecutive n of one k.  The 32-byte piece p of row n sits at
// p ^ ((n & 3) | ((n >> 3) & 1) << 2): the 16 rows of one read then cover the banks
// twice, the least for its 512 bytes.
typedef int v2i __attribute__((ext_vector_type(2)));

__device__ __forceinline__ v2i read_tr(uint32_t addr, int off) {
    v2i r;
    asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(r) : "v"(addr), "n"(off));
    return r;
}

// blocks B0 .. B3 += W blocks (8 bf16 a lane) * one dy block
#define XPU_ONE_BF16(W, LO, HI)                                                                 \
    "v_mfma_f32_16x16x32_bf16 a[%" #LO ":%" #HI "], %" #W ", %4, a[%" #LO ":%" #HI "]\n\t"
#define XPU_BF16_4(CLOBBERS)                                                                    \
    asm volatile(XPU_MFMA_WAIT XPU_ONE_BF16(0, 5, 6) XPU_ONE_BF16(1, 7, 8)                      \
                 XPU_ONE_BF16(2, 9, 10) XPU_ONE_BF16(3, 11, 12)                                 \
                 ::"v"(w0), "v"(w1), "v"(w2), "v"(w3), "v"(x), "n"(4 * B0), "n"(4 * B0 + 3),    \
                 "n"(4 * B1), "n"(4 * B1 + 3), "n"(4 * B2), "n"(4 * B2 + 3), "n"(4 * B3),       \
                 "n"(4 * B3 + 3)                                                                \
                 : CLOBBERS)
template <int COUNT, int B0, int B1, int B2, int B3>
__device__ __forceinline__ void acc_bf16_4(const v4i& w0, const v4i& w1, const v4i& w2,
                                           const v4i& w3, const v4i& x) {
    static_assert(COUNT == 64 || COUNT == 256, "a list of registers");
    if constexpr (COUNT == 64) XPU_BF16_4(XPU_A64);
    else XPU_BF16_4(XPU_A256);
}
template <int B0, int B1>
__device__ __forceinline__ void acc_bf16_2(const v4i& w0, const v4i& w1, const v4i& x) {
    asm volatile(XPU_MFMA_WAIT
                 "v_mfma_f32_16x16x32_bf16 a[%3:%4], %0, %2, a[%3:%4]\n\t"
                 "v_mfma_f32_16x16x32_bf16 a[%5:%6], %1, %2, a[%5:%6]\n\t"
                 ::"v"(w0), "v"(w1), "v"(x), "n"(4 * B0), "n"(4 * B0 + 3), "n"(4 * B1), "n"(4 * B1 + 3)
                 : XPU_A64);
}

template <int BM, int BK, int WM>
__global__ __launch_bounds__(256, BM * BK > 128 * 128 ? 1 : BM < 128 ? 3 : 2) void mx4_dx_kernel(
    const uint16_t* __restrict__ dy, int64_t ldy, int pieces, int width, Weight w,
    const int* __restrict__ offsets, int E, Out out, int type, int tiles_m, int tiles_k) {
    constexpr int WK = 4 / WM;                            // waves by rows, by columns
    constexpr int TM = BM / 16 / WM, TK = BK / 16 / WK;   // MFMA blocks of a wave
    constexpr int DY = BM * 128, WROW = 2 * BK, WT = 64 * WROW, W0 = 3 * DY;
    constexpr int PX = BM / 32;                           // dy loads a wave a stage
    constexpr int NB = BK / 128;                          // weight blocks a thread a stage
    constexpr int ACC = TM * TK > 16 ? 256 : 64;          // block (a, b) is number a * TM + b
    static_assert(4 * TM * TK <= ACC && TK % 2 == 0, "registers, and blocks a column takes together");
    __shared__ __attribute__((aligned(1024))) uint8_t smem[3 * DY + 2 * WT];
    const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
    const int wm = wave / WK, wk = wave % WK;
    int tm, tk;
    if (!tile_of(blockIdx.x, tiles_m, tiles_k, tm, tk)) return;
    RowTile t;
    if (!row_tile<BM>(offsets, E, out.R, tm, t)) return;
    const int k0 = tk * BK;
    if (t.e == E) {
        zero_rows<BM, BK>(out, type, t, k0);
        return;
    }
    // contraction stages: a piece's `width` columns of dy against the weight's rows, once
    // for each piece; in a piece's last stage the weight's rows past N are zeros
    const int per_piece = (width + 63) / 64, stages = per_piece * pieces;
    const uint8_t* const dybase = reinterpret_cast<const uint8_t*>(dy + int64_t(t.row) * ldy);
    const int lr = lane >> 3;
    const int c8 = ((lane & 7) ^ (((wave * 8 + lr) >> 1) & 7)) * 8;   // the lane's chunk, first column
    uint64_t ady[PX];
#pragma unroll
    for (int i = 0; i < PX; ++i)
        ady[i] = uint64_t(min(t.row + (wave + 4 * i) * 8 + lr, t.end - 1) - t.row) * uint64_t(ldy * 2) +
                 c8 * 2;
    // (one piece may end inside a stage: chunks past it come from zeros)
    const uint8_t* const zeros = scalar(g_zero_line);
    const int past = pieces == 1 ? width - c8 : 0x7FFFFFFF;
    const int end = min(past, 64 * stages);
    auto issue_dy = [&](uint32_t slot, int s, int i) {
        const uint8_t* p = scalar(dybase + int64_t(s) * 128) + ady[i];
        if (s * 64 >= end) p = zeros;
        dma16(p, smem + slot + (wave + 4 * i) * 1024);
    };
    // this thread's part of the weight's rows: NB blocks of row nr
    const int nr = threadIdx.x >> 2, part = (threadIdx.x & 3) * NB;
    struct Part {
        uint4 codes[NB];
        uint32_t scale;                                   // (the scale bytes of four blocks)
        bool in;
    };
    int un = 0;                                           // the piece's stage that is loaded next
    const uint8_t* const wbase = w.codes + int64_t(t.e) * w.N * (w.K / 2);
    const uint8_t* const wsbase = w.scales + int64_t(t.e) * w.N * w.SW;
    auto load_w = [&](Part& d) __attribute__((always_inline)) {
        const int n = un * 64 + nr;
        const int64_t row = min(n, w.N - 1);
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int kb = min(k0 / 32 + part + i, w.K / 32 - 1);     // (columns past K are not stored)
            d.codes[i] = *reinterpret_cast<const uint4*>(wbase + row * (w.K / 2) + kb * 16);
        }
        d.scale = *reinterpret_cast<const uint32_t*>(wsbase + row * w.SW + k0 / 32 + (part & ~3));
        d.in = n < w.N;
        if (++un == per_piece) un = 0;
    };
    const int fn = (nr & 3) | (((nr >> 3) & 1) << 2);
    const uint32_t sbase = lds_addr(smem);
    // 8 of the values (dword q of the NB * 4) to the slot at LDS offset `slot`
    uint32_t wput[NB][2];
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h)
            wput[i][h] = sbase + W0 + nr * WROW + ((2 * (part + i) + h) ^ fn) * 32;
    auto put_w = [&](const Part& d, uint32_t slot, int q) __attribute__((always_inline)) {
        const int i = q >> 2, h = (q >> 1) & 1;
        const float sc = __uint_as_float(d.in ? (d.scale >> (8 * ((part + i) & 3)) & 0xFF) << 23 : 0u);
        const uint32_t cq = (q & 3) == 0 ? d.codes[i].x : (q & 3) == 1 ? d.codes[i].y : (q & 3) == 2 ? d.codes[i].z : d.codes[i].w;
        const uint32_t c = d.in ? cq : 0u;
        const v4i v = {__builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, sc, 0)),
                       __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, sc, 1)),
                       __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, sc, 2)),
                       __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, sc, 3))};
        asm volatile("ds_write_b128 %0, %1 offset:%2" ::"v"(wput[i][h] + slot), "v"(v), "n"(16 * (q & 1)) : "memory");
    };
    auto put_all = [&](const Part& d, uint32_t slot) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < 4 * NB; ++q) put_w(d, slot, q);
    };
    // fragments of half H of a stage: 32 contraction rows
    const uint32_t pos = (g ^ ((r >> 1) & 7)) * 16;       // chunk 4 H + g is at pos ^ (64 H)
    const uint32_t yat = sbase + (wm * 16 + r) * 128 + pos;
    const int fr = (r >> 2) | ((g & 1) << 2);             // of the rows that a lane addresses
    const uint32_t wrow = sbase + W0 + (8 * g + (r >> 2)) * WROW + (r & 3) * 8;
    v4i yf[2][TM];
    v2i wl[2][TK], wh[2][TK];
    auto read_y = [&](uint32_t slot, auto H, auto I) {
        constexpr int h = decltype(H)::value, i = decltype(I)::value;
        yf[h][i] = read16((yat ^ (64 * h)) + slot, i * 16 * WM * 128);
    };
    auto read_w = [&](uint32_t slot, auto H, auto I) {
        constexpr int h = decltype(H)::value, i = decltype(I)::value;
        const uint32_t at = wrow + slot + ((wk * TK + i) ^ fr) * 32;
        wl[h][i] = read_tr(at, h * 32 * WROW);
        wh[h][i] = read_tr(at, h * 32 * WROW + 4 * WROW);
    };
    using H0 = std::integral_constant<int, 0>;
    using H1 = std::integral_constant<int, 1>;
    // column b of half h
    auto column = [&](auto H, auto B, const v4i (&wf)[TK]) {
        constexpr int h = decltype(H)::value, b = decltype(B)::value;
        if constexpr (TK == 2) {
            acc_bf16_2<b, TM + b>(wf[0], wf[1], yf[h][b]);
        } else {
            each<TK / 4>([&](auto A) {
                constexpr int a = 4 * decltype(A)::value;
                acc_bf16_4<ACC, a * TM + b, (a + 1) * TM + b, (a + 2) * TM + b, (a + 3) * TM + b>(
                    wf[a], wf[a + 1], wf[a + 2], wf[a + 3], yf[h][b]);
            });
        }
        __builtin_amdgcn_sched_barrier(0);
    };

    // dy is requested three stages ahead and the weight's codes four, two before they are
    // written; past the last stage zeros come instead of dy, and codes that go unused
    Part p0, p1;
    auto here_now = [&](Part& d) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NB; ++i)
            asm volatile("" : "+v"(d.codes[i].x), "+v"(d.codes[i].y), "+v"(d.codes[i].z), "+v"(d.codes[i].w));
        asm volatile("" : "+v"(d.scale));
    };
    constexpr int LATE = PX + NB + 1;                     // the loads of one stage
    load_w(p0);
    load_w(p1);
#pragma unroll
    for (int i = 0; i < 3 * PX; ++i) issue_dy(i / PX * DY, i / PX, i % PX);
    each<TM * TK>([&](auto I) { acc_set<ACC, decltype(I)::value>(v4f{0.f, 0.f, 0.f, 0.f}); });
    put_all(p0, 0);
    load_w(p0);
    put_all(p1, WT);
    load_w(p1);
    wait_vm<0>();
    here_now(p0);
    here_now(p1);
    lds_done();
    block_barrier();
    each<TM>([&](auto I) { read_y(0, H0{}, I); });
    each<TK>([&](auto I) { read_w(0, H0{}, I); });
    lds_done();
    landed(yf[0]); landed(wl[0]); landed(wh[0]);
    uint32_t ynow = 0;
    auto stage = [&](int s, Part& part, uint32_t here, uint32_t next) __attribute__((always_inline)) {
        const uint32_t ynext = ynow == 2 * DY ? 0 : ynow + DY;
        {
            v4i wf[TK];
#pragma unroll
            for (int a = 0; a < TK; ++a) wf[a] = v4i{wl[0][a][0], wl[0][a][1], wh[0][a][0], wh[0][a][1]};
            each<TM>([&](auto B) {
                constexpr int b = decltype(B)::value;
                read_y(ynow, H1{}, B);
                each<TK / TM>([&](auto I) {
                    read_w(here, H1{}, std::integral_constant<int, b * (TK / TM) + decltype(I)::value>{});
                });
                column(H0{}, B, wf);
            });
        }
        // the second half's fragments, and the next stage: dy's loads (all but the latest
        // stage's) and the weight's writes of every wave
        __builtin_amdgcn_s_waitcnt(0x0F70 | (LATE & 15) | (LATE >> 4 << 14));   // vmcnt(LATE)
        lds_done();
        landed(yf[1]); landed(wl[1]); landed(wh[1]);
        block_barrier();
        {
            v4i wf[TK];
#pragma unroll
            for (int a = 0; a < TK; ++a) wf[a] = v4i{wl[1][a][0], wl[1][a][1], wh[1][a][0], wh[1][a][1]};
            put_all(part, here);
            load_w(part);
            // (past the last stage the reads find what the slot held, and go unused)
            each<TM>([&](auto B) {
                constexpr int b = decltype(B)::value;
                read_y(ynext, H0{}, B);
                each<TK / TM>([&](auto I) {
                    read_w(next, H0{}, std::integral_constant<int, b * (TK / TM) + decltype(I)::value>{});
                });
#pragma unroll
                for (int i = b * PX / TM; i < (b + 1) * PX / TM; ++i) issue_dy(ynow, s + 3, i);
                column(H1{}, B, wf);
            });
        }
        lds_done();
        landed(yf[0]); landed(wl[0]); landed(wh[0]);
        ynow = ynext;
    };
#pragma clang loop unroll(disable)
    for (int s = 0; s < stages; s += 2) {
        stage(s, p0, 0, WT);
        if (s + 1 == stages) break;
        stage(s + 1, p1, WT, 0);
    }
    wait_vm<0>();                                         // (the last load_w may be on its way)
    block_barrier();                                      // every wave has read its last stage
    store_tile<TM, TK, 16 * WM>(out, type, t.row + 16 * wm, t.end, k0 + wk * (BK / WK),
                                reinterpret_cast<float*>(smem) + wave * 16 * (BK / WK));
}

}  // namespace

int64_t mx4_split_width(int64_t N) { return (N + 63) / 64 * 64; }
int mx4_split_pieces(int type) { return type == kBf16 ? 1 : type == kF16 ? 2 : 3; }

hipError_t mx4_split(hipStream_t st, const void* dy, int type, int64_t ldy, void* out, int64_t R,
                     int N) {
    const int width = int(mx4_split_width(N));
    const int size = type == kF32 ? 4 : 2;
    const bool vec = reinterpret_cast<uintptr_t>(dy) % 16 == 0 && (ldy * size) % 16 == 0;
    by_type(type, [&](auto T) {
        constexpr int t = decltype(T)::value;
        constexpr int P = t == kBf16 ? 1 : t == kF16 ? 2 : 3;
        auto go = [&](auto V) {
            in_launches(R, 256 * kMaxBlocks / (width / 8), [&](int64_t at, int64_t rows) {
                hipLaunchKernelGGL((mx4_split_kernel<t, decltype(V)::value, P>),
                                   dim3(unsigned((rows * (width / 8) + 255) / 256)), dim3(256), 0, st,
                                   static_cast<const char*>(dy) + at * ldy * size, ldy,
                                   static_cast<uint16_t*>(out) + at * width * P, rows, N, width);
            });
        };
        if (vec) go(std::true_type{});
        else go(std::false_type{});
    });
    return hipGetLastError();
}

namespace {

// Whether 256 x 256 tiles (one block a CU) are faster than 128 x 128 (two), by the times
// that a round of either takes.  fp16 dy, two pieces, with the split: 8192^3 1840 against
// 2280 us, 4096^3 240 / 299, 4096 x 1280 -> 5120 160 / 139, 1000 x 4096 -> 4096 209 / 95;
// bf16, 16384 rows 2816 -> 2048 in 8 groups 238 / 220, in 128 groups 532 / 405, 65520
// rows in 64 groups 798 / 889.
struct TileTimes {
    double small, large;
};
TileTimes tile_times(bool grouped, int64_t R, int E, int64_t N, int64_t K) {
    const double stages = double((N + 63) / 64);
    auto tiles = [&](int64_t b) {                          // (a group's last tile half full)
        const int64_t tm = grouped ? R / b + std::min<int64_t>(E, R) / 2 + 1 : (R + b - 1) / b;
        return tm * ((K + b - 1) / b);
    };
    const int64_t cus = device_cus();
    const int64_t t128 = tiles(128), t256 = tiles(256);
    const double large = double((t256 + cus - 1) / cus) * (8.0 + 1.67 * stages);
    const double small = double(t128 / (2 * cus)) * (4.0 + 1.06 * stages) +
                         (t128 % (2 * cus) > cus ? 4.0 + 1.06 * stages
                          : t128 % (2 * cus) > 0 ? 4.0 + 0.6 * stages : 0.0);
    return {small, large};
}
bool large_dx_tiles(bool grouped, int64_t R, int E, int64_t N, int64_t K) {
    const TileTimes t = tile_times(grouped, R, E, N, K);
    return t.large < t.small;
}
// Whether tiles of 32 rows (three blocks a CU, a wave 32 columns) are faster than 128: up to 64
// rows a group on average, where most of a large tile would be empty, or while they are few
// enough to run all at once.  us, 32 against 128 rows: 32 groups 2816 -> 2048 of 8 rows 41 / 75, of
// 32 62 / 75, of 64 83 / 93, of 100 105 / 97; 64 groups 1024 -> 4096 of 16 69 / 102, of 200 314 / 260;
// 256 rows of one weight, fp16, 4096 x 4096 62 / 80.
// By the mean: with all rows one expert's the same tiles take as long, 1024 rows, 32 experts
// 2816 -> 2048 even 67, all to one 62; 2048 rows 85 / 82; 64 experts, 4096 rows, 1024 -> 4096 121 / 112.
bool few_dx_rows(bool grouped, int64_t R, int E, int64_t K) {
    const int64_t rows = grouped ? R / 32 + std::min<int64_t>(E, R) / 2 + 1 : (R + 31) / 32;
    return R <= 64 * int64_t(grouped ? E : 1) || rows * ((K + 127) / 128) <= 2 * device_cus();
}

}  // namespace

// The weight's conversion (42 MB at 4096 x 4096), two launches and a reduction of fp32
// slices against one launch of tiles with 64 rows of the weight a stage, of which short
// contractions and many rows fill the CUs.  Both measured, us, bf16 product against tiles:
// N 4096, K 4096: 29 / 24 at 1 row, 121 / 113 at 4096; N 8192, K 2048 34 / 54 at 16 rows; N 2048,
// K 8192 27 / 15 at 64; 4096 rows, N 5120, K 1280 64 / 96.
bool mx4_dx_bf16_faster(int64_t R, int64_t N, int64_t K) {
    const TileTimes t = tile_times(false, R, 1, N, K);
    const double flop = 2.0 * double(R) * double(N) * double(K);
    const double bf16 = 15.0 + 0.0014 * double(N) + double(N) * double(K) * 2.5 / 5.0e6 + flop / 1.2e9;
    const double few = few_dx_rows(false, R, 1, K) ? 3.5 + 0.4 * double((N + 63) / 64) : t.small;
    return bf16 < std::min({few, t.small, t.large});
}

namespace {
// rows and columns of the tiles: 32 x 128, 128 x 128 or 256 x 256
struct TileSize {
    int rows, cols;
};
TileSize dx_tile(bool grouped, int64_t R, int E, int64_t N, int64_t K) {
    if (few_dx_rows(grouped, R, E, K)) return {32, 128};
    if (large_dx_tiles(grouped, R, E, N, K)) return {256, 256};
    return {128, 128};
}
}  // namespace

int64_t mx4_dx_blocks(bool grouped, int64_t R, int E, int64_t N, int64_t K) {
    const TileSize t = dx_tile(grouped, R, E, N, K);
    return (most_tiles(grouped, R, E, t.rows) * ((K + t.cols - 1) / t.cols) + 7) / 8 * 8;
}

hipError_t mx4_dx(hipStream_t st, const void* dy, int64_t ldy, int pieces, const uint8_t* wc,
                  const uint8_t* ws, const int* offsets, int E, void* dx, int type, int64_t R,
                  int N, int K) {
    const Weight w{wc, ws, N, K, int(mx_scale_width(K))};
    const Out o = make_out(dx, type, nullptr, 0, R, K);
    // pieces lie side by side, mx4_split_width(N) columns each; one piece may end early
    const int width = pieces == 1 ? N : int(mx4_split_width(N));
    auto go = [&](auto M, auto C, auto W) {
        constexpr int bm = decltype(M)::value, bk = decltype(C)::value, wm = decltype(W)::value;
        const int tiles_k = (K + bk - 1) / bk;
        const int tiles_m = int(most_tiles(offsets != nullptr, R, E, bm));
        hipLaunchKernelGGL((mx4_dx_kernel<bm, bk, wm>),
                           dim3(unsigned((int64_t(tiles_m) * tiles_k + 7) / 8 * 8)), dim3(256), 0,
                           st, static_cast<const uint16_t*>(dy), ldy, pieces, width, w, offsets, E,
                           o, type, tiles_m, tiles_k);
    };
    using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    using I32 = std::integral_constant<int, 32>;
    using I128 = std::integral_constant<int, 128>;
    using I256 = std::integral_constant<int, 256>;
    const int tile_rows = dx_tile(offsets != nullptr, R, E, N, K).rows;
    if (tile_rows == 32) go(I32{}, I128{}, I1{});
    else if (tile_rows == 256) go(I256{}, I256{}, I2{});
    else go(I128{}, I128{}, I2{});
    return hipGetLastError();
}

}  // namespace xpuint8
