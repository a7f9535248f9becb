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

#include "mx4_tiles.hpp"

namespace xpuint8 {
namespace {

typedef int v8i __attribute__((ext_vector_type(8)));

// acc += W block (codes w, scale byte I of sw) * X block (codes x, byte J of sx)
template <int I, int J>
__device__ __forceinline__ v4f mfma4(const v4i& w, int sw, const v4i& x, int sx, const v4f& acc) {
    const v8i a = {w[0], w[1], w[2], w[3], 0, 0, 0, 0}, b = {x[0], x[1], x[2], x[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, 4, I, sw, J, sx);
}

// ----------------------------------------------------------------- few rows
// Up to 16 MB rows of a group: the product reads the weight once and is bound by that and by
// the latencies around it.  A block takes `nt` consecutive blocks of 16 weight rows and all
// of K, its NW waves SS groups of 512 values each: lane l takes row l % 16 and the blocks
// 4j + l / 16 (j = 0..3) of a group, so a load covers 64 consecutive bytes of 16 rows, and
// the row's 16 scale bytes, of which byte l / 16 of dword j belongs to block j.  x stays in
// registers for all nt; the next 16 weight rows are requested before this block's are used
// (three steps ahead measured the same); the NW partial sums meet in LDS (two buffers: one
// barrier a block).
//
// FUSED (MB = 1): x is quantized here, in the registers of the lane that multiplies it (a
// lane's operand is exactly one block), so there is one launch and no quantized copy.
// With more rows every block would read all of x in its own type, 2 KB a row and 1024
// values against 0.5: those take x quantized by a launch before, and so does a K that the
// waves do not hold at once, which is walked in chunks with x read again for each.
//
// MI355X, kernel alone: 1 x 4096 x 4096 5.9 us; 48 x 4096 x 14336 12.9 us (2.4 TB/s of
// weight); 16 rows of some 13 experts, 2048 -> 2816, 10 to 11 us (3.6 TB/s).
template <int T, bool VEC>
struct Block {                                            // 32 values as they are stored
    uint4 v[T == kF32 ? 8 : 4];
    __device__ __forceinline__ void load(const char* p) {
#pragma unroll
        for (int i = 0; i < (T == kF32 ? 8 : 4); ++i) {
            if constexpr (VEC) {
                v[i] = reinterpret_cast<const uint4*>(p)[i];
            } else {
                uint32_t d[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if constexpr (T == kF32) {
                        d[j] = reinterpret_cast<const uint32_t*>(p)[4 * i + j];
                    } else {
                        const uint16_t* h = reinterpret_cast<const uint16_t*>(p) + 8 * i + 2 * j;
                        d[j] = uint32_t(h[0]) | (uint32_t(h[1]) << 16);
                    }
                }
                v[i] = make_uint4(d[0], d[1], d[2], d[3]);
            }
        }
    }
    __device__ __forceinline__ void quantize(v4i& codes, int& scale) const {
        float f[4][8];
#pragma unroll
        for (int c = 0; c < 4; ++c) load8<T, true>(v + c * (T == kF32 ? 2 : 1), f[c]);
        uint32_t m = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) m = max(m, abs_bits(f[c][i]));
        const uint32_t e = mx_scale_byte(m);
#pragma unroll
        for (int c = 0; c < 4; ++c) codes[c] = int(mx_encode8(f[c], e));
        scale = int(e);
    }
};

constexpr int kFewTiles = 64;                             // blocks of weight rows a block takes at most

// x as a kernel of few rows takes it: its own type (FUSED), or codes and scales
struct Rows {
    const char* x;
    int64_t ldx;
    const uint8_t *codes, *scales;
    const int* rows;
    int tokens;
};

template <int T, bool VEC, bool FUSED, int MB, int NW, int SS, int D, bool CHUNKS>
__global__ __launch_bounds__(NW * 64) void mx4_few_kernel(Rows x, Weight w,
                                                          const int* __restrict__ offsets, int E,
                                                          Out out, int nt) {
    static_assert(!FUSED || (MB == 1 && !CHUNKS), "one block of rows is quantized in place");
    static_assert(MB <= NW, "a wave adds up a block of rows");
    constexpr int kChunk = NW * SS * 512;
    __shared__ v4f part[2][NW][MB][64];
    __shared__ v4f bias[kFewTiles][4];
    const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
    RowTile t;
    if (!row_tile<16 * MB>(offsets, E, out.R, blockIdx.y, t)) return;
    const int tiles = (out.N + 15) / 16, first = blockIdx.x * nt, last = min(first + nt, tiles);
    if (t.e == E) {                                       // rows of no group
        for (int i = first; i < last; ++i)
            for (int b = wave; b < MB; b += NW)
                if (t.row + 16 * b + r < t.end)
                    store4<T>(out, t.row + 16 * b + r, 16 * i + 4 * g, v4f{0.f, 0.f, 0.f, 0.f});
        return;
    }
    const int K = w.K, chunks = CHUNKS ? (K + kChunk - 1) / kChunk : 1;
    auto k_of = [&](int c, int s, int j) { return c * kChunk + (wave + NW * s) * 512 + 128 * j + 32 * g; };
    struct Slab {
        v4i f[SS][4];
        uint4 s[SS];
    };
    const uint8_t* const wc = w.codes + int64_t(t.e) * w.N * (K / 2);
    const uint8_t* const wsc = w.scales + int64_t(t.e) * w.N * w.SW;
    // Every load is made, so that the waits can count the loads behind them: past K the
    // last block again (against zeros of x), past the last step one address for all lanes.
    auto load = [&](Slab& d, int tile, int c) __attribute__((always_inline)) {
        const int real = (tile - last) >> 31;             // -1, or 0 past the last step
        const int64_t row = min(16 * tile + r, w.N - 1) & real;
        const uint8_t* const code = wc + row * (K / 2);
        const uint8_t* const scale = wsc + row * w.SW;
#pragma unroll
        for (int s = 0; s < SS; ++s) {
            const int k0 = c * kChunk + (wave + NW * s) * 512;
            d.s[s] = *reinterpret_cast<const uint4*>(scale + (min(k0 / 32, w.SW - 16) & real));
#pragma unroll
            for (int j = 0; j < 4; ++j)
                d.f[s][j] = *reinterpret_cast<const v4i*>(code + ((min(k_of(c, s, j), K - 32) / 2) & real));
        }
    };
    Slab slab[D];
    int ahead = first, ca = 0;                            // the next step to request
    auto request = [&](Slab& d) __attribute__((always_inline)) {
        load(d, ahead, ca);
        if constexpr (CHUNKS) ca = ca + 1 < chunks ? ca + 1 : 0;
        ahead += ca == 0;
        __builtin_amdgcn_sched_barrier(0);                // the loads stay in this order
    };
    v4i xf[MB][SS][4];
    int xs[MB][SS][4];
    // the blocks of x, zeros past K and past the last row; `between` runs once the first
    // of them are requested
    auto load_x = [&](int c, auto between) __attribute__((always_inline)) {
        int src[MB];
#pragma unroll
        for (int m = 0; m < MB; ++m) {
            src[m] = min(t.row + 16 * m + r, t.end - 1);
            if (x.rows) src[m] = min(max(x.rows[src[m]], 0), x.tokens - 1);
        }
        if constexpr (FUSED) {
            const char* const row = x.x + src[0] * x.ldx * kSize<T>;
#pragma unroll
            for (int s = 0; s < SS; ++s) {
                Block<T, VEC> raw[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) raw[j].load(row + min(k_of(c, s, j), K - 32) * kSize<T>);
                if (s == 0) between();
#pragma unroll
                for (int j = 0; j < 4; ++j) raw[j].quantize(xf[0][s][j], xs[0][s][j]);
            }
        } else {
            uint4 sc[MB][SS];
#pragma unroll
            for (int m = 0; m < MB; ++m)
#pragma unroll
                for (int s = 0; s < SS; ++s) {
                    const int k0 = c * kChunk + (wave + NW * s) * 512;
                    sc[m][s] = *reinterpret_cast<const uint4*>(x.scales + int64_t(src[m]) * w.SW +
                                                               min(k0 / 32, w.SW - 16));
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        xf[m][s][j] = *reinterpret_cast<const v4i*>(
                            x.codes + int64_t(src[m]) * (K / 2) + min(k_of(c, s, j), K - 32) / 2);
                }
            between();
#pragma unroll
            for (int m = 0; m < MB; ++m)
#pragma unroll
                for (int s = 0; s < SS; ++s) {
                    const uint32_t d[4] = {sc[m][s].x, sc[m][s].y, sc[m][s].z, sc[m][s].w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) xs[m][s][j] = int(d[j] >> (8 * g));
                }
        }
#pragma unroll
        for (int m = 0; m < MB; ++m)
#pragma unroll
            for (int s = 0; s < SS; ++s)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const bool in = k_of(c, s, j) < K && t.row + 16 * m + r < t.end;
#pragma unroll
                    for (int i = 0; i < 4; ++i) xf[m][s][j][i] = in ? xf[m][s][j][i] : 0;
                    xs[m][s][j] = in ? xs[m][s][j] : 127;
                }
    };
    if (out.bias)                                         // (a load among the steps would wait for theirs)
        for (int i = threadIdx.x; i < 16 * (last - first); i += NW * 64)
            reinterpret_cast<float*>(bias)[i] = bias_at(out, 16 * first + i);
    v4f acc[MB];
    auto use = [&](const Slab& d, int tile, int c, int buf) __attribute__((always_inline)) {
        if (c == 0)
#pragma unroll
            for (int m = 0; m < MB; ++m) acc[m] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < SS; ++s) {
            const uint32_t sw[4] = {d.s[s].x, d.s[s].y, d.s[s].z, d.s[s].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int ws = k_of(c, s, j) < K ? int(sw[j] >> (8 * g)) : 127;  // (byte 0 is read)
#pragma unroll
                for (int m = 0; m < MB; ++m) acc[m] = mfma4<0, 0>(d.f[s][j], ws, xf[m][s][j], xs[m][s][j], acc[m]);
            }
        }
        if (c + 1 < chunks) return;
#pragma unroll
        for (int m = 0; m < MB; ++m) part[buf][wave][m][lane] = acc[m];
        __syncthreads();
        if (wave >= MB || tile >= last) return;
        const int row = t.row + 16 * wave + r, n = 16 * tile + 4 * g;
        if (row >= t.end) return;
        v4f sum = part[buf][0][wave][lane];
#pragma unroll
        for (int i = 1; i < NW; ++i) sum += part[buf][i][wave][lane];
        if (out.bias) sum += bias[tile - first][g];
        store4<T>(out, row, n, sum);
    };
    load_x(0, [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i + 1 < D; ++i) request(slab[i]);
    });
    // One step a block of weight rows and chunk of K, requested D - 1 steps ahead.  The loop
    // ends after D steps only (those past the last store nothing): an exit among them
    // would join states with different loads under way, and every wait be for all.
    int tile = first, c = 0, buf = 0;
    do {
#pragma unroll
        for (int i = 0; i < D; ++i) {
            request(slab[(i + D - 1) % D]);
            use(slab[i], tile, c, buf);
            if constexpr (CHUNKS) c = c + 1 < chunks ? c + 1 : 0;
            if (c == 0) {
                buf ^= 1;
                ++tile;
            }
            if constexpr (CHUNKS) load_x(c, [] {});
        }
    } while (tile < last);
}

// -------------------------------------------------------------------- tiles
// BM x BN tiles of y by a block of 4 waves in 2 x 2 (a wave every other 16 rows, one half
// of the columns), x already quantized.  K in steps of 128 values, one MFMA of each
// block, loaded in pairs, 128 bytes of codes a row, through two LDS slots that direct
// global->LDS loads fill.  During a step a wave runs its MFMAs on one set of fragments and
// reads the next step's into the other.  After a pair's first step one wait and barrier
// mean that every wave has read all of the pair, and that the next one is in; during its
// second step the loads of the pair after that go into its slot.  (64-byte pieces through
// a ring of four single steps, a barrier a step, had a longer lead and were slower: 4096 x
// 1280 -> 10240 60 against 56 us with the quantizer, 16380 x 2048 -> 2816 in 32 groups 106 /
// 101; 8192^3 360 either way.)
//
// Chunk c (16 bytes, one block) of a pair's row sits at c ^ ((row >> 1) & 7): a 16-byte
// LDS read serves the lanes 0-3, 12-15, 20-23 and 24-27 together (and so on), which
// then cover all 64 banks once.  Lane group g holds chunk g of a step, whose scale in
// the row's 16 scale bytes of 512 values (four steps) is byte 4t + g.  The MFMA takes
// its scale from a byte of a register that the instruction names, the same for all
// lanes, so each 16 bytes are transposed (4 x 4) where they lie in LDS: lane group g
// then reads one dword, whose byte t is step t's, and shifts it step by step.  That pass
// also clears the bytes of blocks past K: 2^-127 in both operands, whose products vanish
// in fp32 (every code is a number, so what the codes there are does not matter: loads
// past a row's end repeat its last block).  Scales arrive two groups of four steps ahead,
// and are transposed one ahead.
//
// The fragment reads are inline assembly (with the builtins the compiler waits for
// every direct load before each LDS read); nothing is in flight over a loop edge:
// each step ends with a wait that redefines what it read.
//
// The 256 x 256 forms hold 256 accumulators and 256 other registers a lane and spill 32 of
// the latter (41 with GATHER): stored before the main loop and read after it, with GATHER
// one pair in the loop too.  The 128 x 128 forms spill none.
// blocks B0 .. B3 += W blocks (codes w, scale byte 0 of sw) * one X block
#define XPU_MFMA4(CLOBBERS)                                                                     \
    asm volatile(XPU_MFMA_WAIT XPU_ONE_MFMA(0, 4, 10, 11) XPU_ONE_MFMA(1, 5, 12, 13)            \
                 XPU_ONE_MFMA(2, 6, 14, 15) XPU_ONE_MFMA(3, 7, 16, 17)                          \
                 ::"v"(w[0]), "v"(w[1]), "v"(w[2]), "v"(w[3]), "v"(sw[0]), "v"(sw[1]),          \
                 "v"(sw[2]), "v"(sw[3]), "v"(x), "v"(sx), "n"(4 * B0), "n"(4 * B0 + 3),         \
                 "n"(4 * B1), "n"(4 * B1 + 3), "n"(4 * B2), "n"(4 * B2 + 3), "n"(4 * B3),       \
                 "n"(4 * B3 + 3)                                                                \
                 : CLOBBERS)
#define XPU_ONE_MFMA(W, S, LO, HI)                                                              \
    "v_mfma_scale_f32_16x16x128_f8f6f4 a[%" #LO ":%" #HI "], %" #W ", %8, a[%" #LO ":%" #HI     \
    "], %" #S ", %9 op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t"
template <int COUNT, int B0, int B1, int B2, int B3>
__device__ __forceinline__ void acc_mfma4(const v4i* w, const int* sw, const v4i& x, int sx) {
    static_assert(COUNT == 64 || COUNT == 256, "a list of registers");
    if constexpr (COUNT == 64) XPU_MFMA4(XPU_A64);
    else XPU_MFMA4(XPU_A256);
}
template <int BM, int BN, bool GATHER>
__global__ __launch_bounds__(256, BM * BN > 128 * 128 ? 1 : 2) void mx4_tile_kernel(
    const uint8_t* __restrict__ xc, const uint8_t* __restrict__ xs, const int* __restrict__ rows,
    int tokens, Weight w, const int* __restrict__ offsets, int E, Out out, int type, int tiles_m,
    int tiles_n) {
    constexpr int TM = BM / 32, TN = BN / 32;             // MFMA blocks of a wave
    constexpr int ROWS = BM + BN;                         // x rows first
    constexpr int PAIR = ROWS * 128, SCALES = ROWS * 16;
    constexpr int PX = BM / 32, PW = BN / 32;             // code loads a wave a pair of steps
    constexpr int PL = PX + PW;
    constexpr int PSX = BM / 64, PS = ROWS / 64;          // scale loads of x, of both, a block
    constexpr int PER_S = (PS + 3) / 4;
    constexpr int PER_T = (ROWS + 255) / 256;             // scale rows a thread transposes
    constexpr int ACC = 4 * TM * TN;                      // block (a, b) is number a * TM + b
    __shared__ __attribute__((aligned(1024))) uint8_t smem[2 * PAIR + 2 * SCALES];
    __shared__ float bias_of[BN];
    const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
    const int wm = wave >> 1, wn = wave & 1;
    int tm, tn;
    if (!tile_of(blockIdx.x, tiles_m, tiles_n, tm, tn)) return;
    RowTile t;
    if (!row_tile<BM>(offsets, E, out.R, tm, t)) return;
    const int n0 = tn * BN;
    if (t.e == E) {
        zero_rows<BM, BN>(out, type, t, n0);
        return;
    }
    const int K = w.K, KB = K / 2;
    const int steps = (K + 127) / 128, groups = (K + 511) / 512;
    // Sources: a wave-uniform base and a lane's 32-bit offset from the tile's first row (a
    // tile spans less than 4 GiB), load i 32 rows after the first and the last row for
    // those past it; or, for rows that a list names, the row.  A load of a wave brings 8
    // rows, its first row is wave * 8 + 32 i.
    const int64_t w0 = int64_t(t.e) * w.N + n0;
    const uint8_t* const wbase = w.codes + w0 * KB;
    const uint8_t* const wsbase = w.scales + w0 * w.SW;
    const uint8_t* const xbase = xc + (GATHER ? 0 : int64_t(t.row) * KB);
    const uint8_t* const xsbase = xs + (GATHER ? 0 : int64_t(t.row) * w.SW);
    auto x_row = [&](int j) {                             // the row of tile row j, from xbase
        const int i = min(t.row + j, t.end - 1);
        return GATHER ? min(max(rows[i], 0), tokens - 1) : i - t.row;
    };
    auto w_row = [&](int j) { return min(n0 + j, w.N - 1) - n0; };
    const int lr = wave * 8 + (lane >> 3);
    const uint32_t c16 = uint32_t((lane & 7) ^ ((lr >> 1) & 7)) * 16;
    const uint32_t first = uint32_t(lr) * uint32_t(KB) + c16;
    const uint32_t xlast = uint32_t(min(t.end - t.row, BM) - 1) * uint32_t(KB) + c16;
    const uint32_t wlast = uint32_t(min(w.N - n0, BN) - 1) * uint32_t(KB) + c16;
    int listed[GATHER ? PX : 1];
    if constexpr (GATHER) {
#pragma unroll
        for (int i = 0; i < PX; ++i) listed[i] = x_row(lr + 32 * i);
    }
    uint32_t as[PER_S];                                   // 16-byte units: 64 GiB of scales
    const uint8_t* sbs[PER_S];
#pragma unroll
    for (int i = 0; i < PER_S; ++i) {
        const int b = min(wave + 4 * i, PS - 1);
        sbs[i] = b < PSX ? xsbase : wsbase;
        as[i] = uint32_t(b < PSX ? x_row(b * 64 + lane) : w_row((b - PSX) * 64 + lane)) *
                uint32_t(w.SW / 16);
    }
    // load i of this wave's PX + PW (x first) of pair p into its slot, less back (for a last
    // pair's chunks past the row's end: its last chunk)
    auto issue_codes = [&](int p, uint32_t back, int i) {
        const bool isx = i < PX;
        const int j = isx ? i : i - PX;
        const uint32_t at = first + uint32_t(32 * j) * uint32_t(KB);
        const int64_t k = int64_t(p) * 128;
        const uint8_t* from;
        if (!isx) from = scalar(wbase + k) + uint64_t(min(at, wlast) - back);
        else if constexpr (GATHER) from = scalar(xbase + k) + (uint64_t(uint32_t(listed[j])) * uint32_t(KB) + (c16 - back));
        else from = scalar(xbase + k) + uint64_t(min(at, xlast) - back);
        dma16(from, smem + (p & 1) * PAIR + (wave * 8 + 32 * j + (isx ? 0 : BM)) * 128);
    };
    auto past_end = [&](int p) {                          // back, of pair p
        const int over = p * 128 + int(c16) + 16 - KB;
        return over > 0 ? uint32_t(over) : 0u;
    };
    auto issue_scales = [&](int q) {
#pragma unroll
        for (int i = 0; i < PER_S; ++i) {
            const int b = wave + 4 * i;
            if (PS % 4 == 0 || b < PS)
                dma16(sbs[i] + (uint64_t(as[i] + uint32_t(q)) << 4),
                      smem + 2 * PAIR + (q & 1) * SCALES + b * 1024);
        }
    };

    const int xrow = wm * 16 + r, wrow = BM + wn * (BN / 2) + r;
    const uint32_t sbase = lds_addr(smem);
    // (the second step's chunks of a pair are at ^ 64)
    const uint32_t pos = (g ^ ((r >> 1) & 7)) * 16;
    const uint32_t xat = sbase + xrow * 128 + pos, wat = sbase + wrow * 128 + pos;
    // fragments of even and odd steps; x's first half is read again as soon as it is used
    v4i xf[2][TM], wf[2][TN];
    constexpr int TH = TM / 2;
    int sx[TM], sw[TN];                                   // byte 0: this step's scale
    int sr[TM + TN];                                      // the next group's
    v4i tr[PER_T];                                        // scale rows on their way through
    auto read_x = [&](auto S, auto Fr, auto I) {
        constexpr int slot = decltype(S)::value, f = decltype(Fr)::value, i = decltype(I)::value;
        xf[i < TH ? 0 : f][i] = read16((xat ^ (64 * (slot & 1))) + (slot >> 1) * PAIR, i * 4096);
    };
    auto read_w = [&](auto S, auto Fr, auto I) {
        constexpr int slot = decltype(S)::value, f = decltype(Fr)::value, i = decltype(I)::value;
        wf[f][i] = read16((wat ^ (64 * (slot & 1))) + (slot >> 1) * PAIR, i * 2048);
    };
    auto read_scale = [&](uint32_t at, int i) {           // of block i, x's first
        sr[i] = i < TM ? read4(at + xrow * 16, i * 512) : read4(at + wrow * 16, (i - TM) * 256);
    };
    // the 4 x 4 byte transposition of each row's scales of group q, in place: the
    // reads, and after they have landed the writes
    auto scale_row = [&](int q, int i) {
        return sbase + 2 * PAIR + (q & 1) * SCALES + (threadIdx.x + 256 * i) * 16;
    };
    const bool tlast = ROWS % 256 == 0 || int(threadIdx.x) + 256 * (PER_T - 1) < ROWS;
    auto transpose_read = [&](int q) {
        each<PER_T>([&](auto I) {
            constexpr int i = decltype(I)::value;
            tr[i] = read16(i < PER_T - 1 || tlast ? scale_row(q, i) : sbase, 0);
        });
    };
    auto transpose_write = [&](int q) {
        const int left = K / 32 - q * 16;                 // blocks up to K
#pragma unroll
        for (int i = 0; i < PER_T; ++i) {
            uint32_t d[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) d[c] = uint32_t(tr[i][c]);
            if (left < 16) {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int n = left - 4 * c;           // of the dword's four blocks
                    d[c] &= n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1;
                }
            }
            const uint32_t lo01 = __builtin_amdgcn_perm(d[1], d[0], 0x05010400u);   // bytes 0, 1 of d0, d1
            const uint32_t hi01 = __builtin_amdgcn_perm(d[1], d[0], 0x07030602u);   // bytes 2, 3
            const uint32_t lo23 = __builtin_amdgcn_perm(d[3], d[2], 0x05010400u);
            const uint32_t hi23 = __builtin_amdgcn_perm(d[3], d[2], 0x07030602u);
            const v4i o = {int(__builtin_amdgcn_perm(lo23, lo01, 0x05040100u)),
                           int(__builtin_amdgcn_perm(lo23, lo01, 0x07060302u)),
                           int(__builtin_amdgcn_perm(hi23, hi01, 0x05040100u)),
                           int(__builtin_amdgcn_perm(hi23, hi01, 0x07060302u))};
            if (i < PER_T - 1 || tlast)
                asm volatile("ds_write_b128 %0, %1" ::"v"(scale_row(q, i)), "v"(o) : "memory");
        }
    };
    using C0 = std::integral_constant<int, 0>;
    using C1 = std::integral_constant<int, 1>;
    using C2 = std::integral_constant<int, 2>;
    using C3 = std::integral_constant<int, 3>;

    static_assert(BN <= 256, "a column a thread");
    issue_scales(0);
    if (groups > 1) issue_scales(1);
    for (int p = 0; p < min((steps + 1) / 2, 2); ++p) {
        const uint32_t back = past_end(p);
#pragma unroll
        for (int i = 0; i < PL; ++i) issue_codes(p, back, i);
    }
    // meanwhile the accumulators start from the bias
    if (out.bias) {
        if (threadIdx.x < BN) bias_of[threadIdx.x] = bias_at(out, n0 + int(threadIdx.x));
        lds_done();
        block_barrier();
        each<TN>([&](auto A) {
            constexpr int a = decltype(A)::value;
            v4i b4 = read16(lds_addr(bias_of) + (wn * (BN / 2) + 4 * g) * 4, a * 64);
            asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(b4)::"memory");
            each<TM>([&](auto B) { acc_set<ACC, a * TM + decltype(B)::value>(__builtin_bit_cast(v4f, b4)); });
        });
    } else {
        each<TM * TN>([&](auto B) { acc_set<ACC, decltype(B)::value>(v4f{0.f, 0.f, 0.f, 0.f}); });
    }
    // (the scales went out first, then the codes pair by pair: pair 0's are in too)
    if (steps > 2) wait_vm<PL>();
    else wait_vm<0>();
    block_barrier();
    transpose_read(0);
    lds_done();
    landed(tr);
    transpose_write(0);
    lds_done();
    block_barrier();
    each<TM + TN>([&](auto I) { read_scale(sbase + 2 * PAIR + 4 * g, decltype(I)::value); });
    each<TM>([&](auto I) { read_x(C0{}, C0{}, I); });
    each<TN>([&](auto I) { read_w(C0{}, C0{}, I); });
    lds_done();
    landed(xf[0]); landed(wf[0]); landed(sr);
#pragma unroll
    for (int b = 0; b < TM; ++b) sx[b] = sr[b];
#pragma unroll
    for (int a = 0; a < TN; ++a) sw[a] = sr[TM + a];

    // step s = 4q + J; FULL: pair s / 2 + 2 exists and is whole
    auto step = [&](auto Jc, auto Full, int q) {
        constexpr int J = decltype(Jc)::value, F = J & 1;
        constexpr bool FULL = decltype(Full)::value;
        using Next = std::integral_constant<int, (J + 1) & 3>;
        using NF = std::integral_constant<int, 1 - F>;
        const int s = 4 * q + J;
        const int ahead = s / 2 + 2;
        const bool more = (J & 1) && (FULL || 2 * ahead < steps);
        const uint32_t back = FULL ? 0u : past_end(ahead);
        const uint32_t sat = sbase + 2 * PAIR + 4 * g + ((q + 1) & 1) * SCALES;
        if (J == 1 && q + 2 < groups) issue_scales(q + 2);
        // (past the last group or step the reads find what was there, and go unused)
        if constexpr (J == 1) transpose_read(q + 1);
        if constexpr (J == 2) transpose_write(q + 1);
        each<TM>([&](auto B) {
            constexpr int b = decltype(B)::value;
            // the reads in the step's first half
            if constexpr (b < TH) {
                read_x(Next{}, NF{}, std::integral_constant<int, TH + b>{});
                each<TN / TH>([&](auto I) {
                    read_w(Next{}, NF{}, std::integral_constant<int, b * (TN / TH) + decltype(I)::value>{});
                });
                if constexpr (J == 3)
                    each<(TM + TN) / TH>([&](auto I) { read_scale(sat, b * ((TM + TN) / TH) + decltype(I)::value); });
            }
            if (more) {
#pragma unroll
                for (int i = b * PL / TM; i < (b + 1) * PL / TM; ++i) issue_codes(ahead, back, i);
            }
            each<TN / 4>([&](auto A) {
                constexpr int a = 4 * decltype(A)::value;
                acc_mfma4<ACC, a * TM + b, (a + 1) * TM + b, (a + 2) * TM + b, (a + 3) * TM + b>(
                    &wf[F][a], &sw[a], xf[b < TH ? 0 : F][b], sx[b]);
            });
            if constexpr (b < TH) read_x(Next{}, NF{}, B);
            __builtin_amdgcn_sched_barrier(0);
        });
        lds_done();
#pragma unroll
        for (int i = 0; i < TM; ++i) asm volatile("" : "+v"(xf[i < TH ? 0 : 1 - F][i]));
        landed(wf[1 - F]);
        if constexpr (J == 1) landed(tr);
        if constexpr (J == 3) landed(sr);
#pragma unroll
        for (int b = 0; b < TM; ++b) sx[b] = J == 3 ? sr[b] : int(uint32_t(sx[b]) >> 8);
#pragma unroll
        for (int a = 0; a < TN; ++a) sw[a] = J == 3 ? sr[TM + a] : int(uint32_t(sw[a]) >> 8);
        // every wave has read its pair's last fragments; the next pair is in
        if constexpr (F == 0) {
            wait_vm<0>();
            block_barrier();
        }
    };
    const int whole = K / 128;
    using Yes = std::true_type;
    using No = std::false_type;
    int q = 0;
    auto whole_groups = [&]() {
#pragma clang loop unroll(disable)
        for (; 4 * q + 8 <= whole; ++q) {
            step(C0{}, Yes{}, q);
            step(C1{}, Yes{}, q);
            step(C2{}, Yes{}, q);
            step(C3{}, Yes{}, q);
        }
    };
    whole_groups();
#pragma clang loop unroll(disable)
    for (;; ++q) {
        step(C0{}, No{}, q);
        if (4 * q + 1 >= steps) break;
        step(C1{}, No{}, q);
        if (4 * q + 2 >= steps) break;
        step(C2{}, No{}, q);
        if (4 * q + 3 >= steps) break;
        step(C3{}, No{}, q);
        if (4 * q + 4 >= steps) break;
    }
    store_tile<TM, TN>(out, type, t.row + 16 * wm, t.end, n0 + wn * (BN / 2),
                       reinterpret_cast<float*>(smem) + wave * 16 * (BN / 2));
}

}  // namespace

namespace {

constexpr int64_t kFusedK = 8 * 2 * 512;              // values of a row that the waves hold

// How the kernel of few rows divides a product with MB blocks of rows a block, and about
// how long it takes.  A wave has 512 values of K (1024 of one block of rows beyond 4096).
// A block takes nt blocks of weight rows, so that there are as many blocks as the device
// holds at once (four waves a SIMD by registers, two with four blocks of rows), since each
// reads all its rows of x again.  Of many groups some are empty, or end inside a block.
struct FewPlan {
    int waves, nt;
    double us;
};
FewPlan few_plan(int MB, bool grouped, int64_t R, int E, int64_t N, int64_t K) {
    FewPlan p;
    p.waves = K <= 4 * 512 ? 4 : K <= 8 * 512 || MB == 1 ? 8 : 16;
    const int64_t tiles = (N + 15) / 16, full = (R + 16 * MB - 1) / (16 * MB);
    const int64_t busy = grouped ? std::max(std::min<int64_t>(R, E), full + E / 2) : full;
    const int64_t cols = std::max<int64_t>(1, int64_t(device_cus()) * (MB == 4 ? 8 : 16) / p.waves / busy);
    p.nt = int(std::clamp<int64_t>((tiles + cols - 1) / cols, 1, kFewTiles));
    // (fitted to 17 to 512 rows of 25 weights)
    const double rounds = double(tiles * busy) / double(cols * busy * p.nt);
    const double turns = double(p.nt) * std::max(1.0, rounds);
    p.us = K <= 2048   ? 5.3 + 1.25 * turns
           : K <= 4096 ? 6.9 + 1.2 * turns
           : K <= 8192 ? 6.9 + 2.4 * turns
                       : 6.5 + 6.0 * turns * double((K + 8191) / 8192);
    return p;
}

// rows of x in their own type or quantized (codes), on the kernel of few rows
template <int T, bool VEC, bool FUSED, int MB>
hipError_t few(hipStream_t st, const Rows& x, const Weight& w, const int* offsets, int E,
               const Out& o) {
    const int tiles = (o.N + 15) / 16;
    const int64_t tm = most_tiles(offsets != nullptr, o.R, E, 16 * MB);
    const FewPlan plan = few_plan(MB, offsets != nullptr, o.R, E, o.N, w.K);
    const int nw = plan.waves, nt = plan.nt;
    auto go = [&](auto W, auto S, auto D, auto C) {
        constexpr int nw = decltype(W)::value, ss = decltype(S)::value, d = decltype(D)::value;
        hipLaunchKernelGGL((mx4_few_kernel<T, VEC, FUSED, MB, nw, ss, d, decltype(C)::value>),
                           dim3(unsigned((tiles + nt - 1) / nt), unsigned(tm)), dim3(nw * 64), 0, st,
                           x, w, offsets, E, o, nt);
        return hipGetLastError();
    };
    using One = std::integral_constant<int, 1>;
    using Two = std::integral_constant<int, 2>;
    using Four = std::integral_constant<int, 4>;
    using Eight = std::integral_constant<int, 8>;
    using Sixteen = std::integral_constant<int, 16>;
    auto whole = [&](auto W, auto S) {                   // (one step: nothing to request ahead)
        if (nt == 1) return go(W, S, One{}, std::false_type{});
        return go(W, S, Two{}, std::false_type{});
    };
    if constexpr (MB == 1 && !FUSED) {                    // (a K that cannot be quantized in place)
        return go(Eight{}, Two{}, Two{}, std::true_type{});
    } else {
        if (nw == 4) return whole(Four{}, One{});
        if (w.K <= 8 * 512) return whole(Eight{}, One{});
        if constexpr (FUSED) return whole(Eight{}, Two{});
        if constexpr (MB == 2) {
            if (w.K <= 16 * 512) return whole(Sixteen{}, One{});
            return go(Sixteen{}, One{}, Two{}, std::true_type{});
        }
        return hipErrorInvalidValue;                      // (four blocks: up to 4096 values)
    }
}

}  // namespace

namespace {
// Up to 16 rows, or 8 a group on average, one block of rows is enough (of 16 on average
// nearly half of the groups would have two): blocks of 16 against 32, us, 8 groups of 8 rows
// 2048 -> 1024 6.2 / 8.6; 32 groups 2048 -> 2816 of 8 rows 22 / 22, of 11 25 / 22, of 16 30 / 22;
// 64 groups of 11 4096 -> 1024 38 / 29.
bool one_block(bool grouped, int64_t R, int E) { return R <= (grouped ? 8 * int64_t(E) : 16); }
}  // namespace

// With one block of rows the weight's bytes are the product's time and the quantizer's
// launch (2 to 3 us) would be a third of the rest.
bool mx4_fused(int64_t R, bool grouped, int E, int64_t K) {
    return one_block(grouped, R, E) && K <= kFusedK;
}

hipError_t mx4_product_fused(hipStream_t st, const void* x, int type, int64_t ldx,
                             const int* rows, int64_t tokens, const uint8_t* wc,
                             const uint8_t* ws, const int* offsets, int E, void* y,
                             const void* bias, int bias_type, int64_t R, int N, int K) {
    const Weight w{wc, ws, N, K, int(mx_scale_width(K))};
    const Out o = make_out(y, type, bias, bias_type, R, N);
    const int size = type == kF32 ? 4 : 2;
    const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && (ldx * size) % 16 == 0;
    const Rows in{static_cast<const char*>(x), ldx, nullptr, nullptr, rows, int(tokens)};
    hipError_t e = hipSuccess;
    by_type(type, [&](auto T) {
        constexpr int t = decltype(T)::value;
        e = vec ? few<t, true, true, 1>(st, in, w, offsets, E, o)
                : few<t, false, true, 1>(st, in, w, offsets, E, o);
    });
    return e;
}

namespace {

// The times, us, of 128 x 128 tiles (two blocks a CU, so that one's start and end overlap the
// other's steps, and finer rounds) and of 256 x 256 tiles (one block a CU, half the operand
// bytes a product), by what a round of either takes, fitted to both over 13 shapes.  With
// the quantizer, 256 against 128: 8192^3 342 / 405 us, 2048 x 8192 x 8192 83 / 98, 4096^3
// 54 / 60; 4096 x 1280 -> 5120 44 / 34, 4096 x 2560 -> 10240 88 / 84, 1000 x 4096 x 4096 39 / 22,
// 16380 x 2048 -> 2816 in 32 groups 128 / 111.
struct TileTimes {
    double small, large;
};
TileTimes tile_times(bool grouped, int64_t R, int E, int64_t N, int64_t K) {
    const double steps = double((K + 127) / 128);
    auto tiles = [&](int64_t b) {                          // (a group's last tile half full)
        const int64_t tm = grouped ? R / b + std::min<int64_t>(E, R) / 2 + 1 : (R + b - 1) / b;
        return tm * ((N + b - 1) / b);
    };
    const int64_t cus = device_cus();
    const int64_t t128 = tiles(128), t256 = tiles(256);
    const double large = double((t256 + cus - 1) / cus) * (10.0 + 1.07 * steps);
    const double small = double(t128 / (2 * cus)) * (2.6 + 0.68 * steps) +
                         (t128 % (2 * cus) > cus ? 2.6 + 0.68 * steps
                          : t128 % (2 * cus) > cus / 2 ? 2.6 + 0.46 * steps
                          : t128 % (2 * cus) > 0 ? 2.3 + 0.34 * steps : 0.0);
    return {small, large};
}

}  // namespace

namespace {
// How a product of quantized x goes: on the kernel of few rows with `blocks` blocks of 16 of
// them, or (0) in tiles of tile x tile.
struct ProductPlan {
    int blocks, tile;
};
ProductPlan product_plan(bool grouped, int64_t R, int E, int64_t N, int64_t K) {
    const TileTimes tiles = tile_times(grouped, R, E, N, K);
    // The kernel of few rows, with one block of rows always, with more (up to where a
    // block's rows of x would be read many times over) where its weight blocks take less time
    // than tiles.  With the quantizer, us, few rows against tiles: 64 x 4096 x 4096 10.6 / 15.7,
    // 256 rows 15.0 / 17.3, 512 rows 20.8 / 18.7; 64 x 8192 x 4096 14.5 / 25.1, 128 rows 19.2 /
    // 26.9; 32 x 14336 x 4096 21 / 40, 64 rows 33 / 42, 128 rows 58 / 46; 128 x 2048 x 14336 14.1 / 11.5.
    // Groups, up to 64 rows on average: 32 groups of 40 rows 2048 -> 2816 25 / 30, of 64 33 / 39, of
    // 100 44 / 44; 64 groups of 40 rows 4096 -> 1024 40 / 46, of 64 56 / 51, of 200 110 / 80.
    // The mean is all that the host knows; a batch of one expert's rows alone takes no longer:
    // 1024 rows, 32 experts 2048 -> 2816, even 30, all to one 26; 2048 rows 33 / 34; 4096 rows, 64
    // experts 4096 -> 1024 58 / 56 (the one weight, read for every 64 rows, stays in the caches).
    const int64_t per_group = grouped ? (R + E - 1) / E : R;
    const int mb = one_block(grouped, R, E) ? 1 : per_group <= 32 || K > 8 * 512 ? 2 : 4;
    const bool blocks = grouped ? per_group <= 64
                                : R <= 512 && few_plan(mb, false, R, E, N, K).us < std::min(tiles.small, tiles.large);
    return {mb == 1 || blocks ? mb : 0, tiles.large < tiles.small ? 256 : 128};
}
int64_t tile_blocks(bool grouped, int64_t R, int E, int64_t N, int tile) {
    return (most_tiles(grouped, R, E, tile) * ((N + tile - 1) / tile) + 7) / 8 * 8;
}
}  // namespace

// (the kernel of few rows has at most 2^31 threads, a block of it up to 64 x 16 columns)
int64_t mx4_product_blocks(bool grouped, int64_t R, int E, int64_t N, int64_t K) {
    const ProductPlan p = product_plan(grouped, R, E, N, K);
    return p.blocks ? 0 : tile_blocks(grouped, R, E, N, p.tile);
}

hipError_t mx4_product(hipStream_t st, const uint8_t* xc, const uint8_t* xs, const int* rows,
                       int64_t tokens, const uint8_t* wc, const uint8_t* ws, const int* offsets,
                       int E, void* y, int type, const void* bias, int bias_type, int64_t R, int N,
                       int K) {
    const Weight w{wc, ws, N, K, int(mx_scale_width(K))};
    const Out o = make_out(y, type, bias, bias_type, R, N);
    const ProductPlan plan = product_plan(offsets != nullptr, R, E, N, K);
    if (const int mb = plan.blocks) {
        const Rows in{nullptr, 0, xc, xs, rows, int(tokens)};
        hipError_t e = hipSuccess;
        by_type(type, [&](auto T) {
            constexpr int t = decltype(T)::value;
            e = mb == 1   ? few<t, true, false, 1>(st, in, w, offsets, E, o)
                : mb == 2 ? few<t, true, false, 2>(st, in, w, offsets, E, o)
                          : few<t, true, false, 4>(st, in, w, offsets, E, o);
        });
        return e;
    }
    auto go = [&](auto M, auto N_) {
        constexpr int BM = decltype(M)::value, BN = decltype(N_)::value;
        const int tiles_n = (N + BN - 1) / BN;
        const int tiles_m = int(most_tiles(offsets != nullptr, R, E, BM));
        const dim3 grid(unsigned(tile_blocks(offsets != nullptr, R, E, N, BM)));
        if (rows)
            hipLaunchKernelGGL((mx4_tile_kernel<BM, BN, true>), grid, dim3(256), 0, st, xc, xs,
                               rows, int(tokens), w, offsets, E, o, type, tiles_m, tiles_n);
        else
            hipLaunchKernelGGL((mx4_tile_kernel<BM, BN, false>), grid, dim3(256), 0, st, xc, xs,
                               rows, int(tokens), w, offsets, E, o, type, tiles_m, tiles_n);
    };
    using I128 = std::integral_constant<int, 128>;
    using I256 = std::integral_constant<int, 256>;
    if (plan.tile == 256) go(I256{}, I256{});
    else go(I128{}, I128{});
    return hipGetLastError();
}

}  // namespace xpuint8
