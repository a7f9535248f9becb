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
// 32760 positions of 48 heads of 128 in bf16 154 to 159 us (5.1 to 5.2 TB/s), 6141 of 20 heads of
// 80 in fp16 9.7, 32 decoded ones of 40 heads of 128 4.1.
#include <algorithm>
#include <type_traits>

#include "block_kernels.hpp"
#include "mx_kernels.hpp"
#include "rows.hpp"

namespace xpuint8 {
namespace {

struct RotaryArgs {
    Heads q, k;                     // k.H = 0: q alone
    Positions pos;
    const double* inv_freq;
    const int* axis;
    uint32_t S, tokens, first;      // positions in all, the launch's first
    int P, D, per_head;             // pieces a head: of 8 pairs, then 16 unturned values
    int turned;                     // pieces of pairs
    int each;                       // positions a block
    float sign;
};

__device__ __forceinline__ double position_of(const Positions& p, int axis, int64_t b, int64_t s) {
    if (axis < 0 || axis >= p.axes) return 0.0;
    const int64_t at = axis * p.a + b * p.b + s * p.s;
    if (p.type == 0) return double(static_cast<const int32_t*>(p.p)[at]);
    if (p.type == 1) return double(static_cast<const int64_t*>(p.p)[at]);
    return double(static_cast<const float*>(p.p)[at]);
}

// A thread's piece of every head: two runs of 8 values, ends where they are cut.  A head's
// last pairs, fewer than 8, are taken with the ones before them, which two threads then
// write alike; a run is cut only where there are not 8 at all.
struct Runs {
    int d[2], end[2];
    bool turn;
};

// A block takes a.each positions; a thread keeps to one piece of a head and goes through
// the heads of all of them, the next one's values requested before it works on the current
// one's (and the first before the angles are made).  EVEN: no run is cut.
template <int T, bool SPLIT, bool EVEN>
__global__ __launch_bounds__(512) void rotary_kernel(RotaryArgs a) {
    extern __shared__ __align__(16) float2 cs[];      // [each][stride]
    const int stride = 8 * a.turned;
    const int c = threadIdx.x % a.per_head, slot = threadIdx.x / a.per_head;
    const int slots = blockDim.x / a.per_head, H = a.q.H + a.k.H;
    const uint32_t t0 = a.first + blockIdx.x * uint32_t(a.each);
    const int n = int(min(a.tokens - t0, uint32_t(a.each)));
    const int rows = slot < slots ? n * H : 0;
    Runs w;
    w.turn = c < a.turned;
    const int p0 = EVEN ? min(8 * c, a.P - 8) : 8 * c;      // (turned: its first pair)
    if (w.turn) {
        w.d[0] = SPLIT ? p0 : 2 * p0;
        w.d[1] = SPLIT ? a.P + p0 : 2 * p0 + 8;
        w.end[0] = SPLIT ? a.P : 2 * a.P;
        w.end[1] = 2 * a.P;
    } else {
        w.d[0] = 2 * a.P + 16 * (c - a.turned);
        w.d[1] = w.d[0] + 8;
        if (EVEN) {
            w.d[0] = min(w.d[0], a.D - 8);
            w.d[1] = min(w.d[1], a.D - 8);
        }
        w.end[0] = w.end[1] = a.D;
    }
    auto place = [&](int row, const char*& x, char*& out) -> int {
        const int t = int(uint32_t(row) / uint32_t(H)), h = row - t * H;
        const uint32_t b = (t0 + t) / a.S, s = (t0 + t) - b * a.S;
        const Heads& m = h < a.q.H ? a.q : a.k;
        const int64_t hh = h < a.q.H ? h : h - a.q.H;
        x = static_cast<const char*>(m.x) + (b * m.x_b + s * m.x_s + hh * m.x_h) * kElem<T>;
        out = static_cast<char*>(m.out) + (b * m.o_b + s * m.o_s + hh * m.o_h) * kElem<T>;
        return t;
    };
    Piece8<T> next[2] = {};
    char* next_out = nullptr;
    int next_t = 0;
    auto request = [&](int row) {
        if (row >= rows) return;
        const char* x;
        next_t = place(row, x, next_out);
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (EVEN || w.d[i] < w.end[i]) next[i] = piece_load<T, EVEN>(x, w.d[i], w.end[i]);
    };
    request(slot);
    for (int i = threadIdx.x; i < n * a.P; i += blockDim.x) {
        const int t = int(uint32_t(i) / uint32_t(a.P)), p = i - t * a.P;
        const uint32_t b = (t0 + t) / a.S, s = (t0 + t) - b * a.S;
        const double turns = position_of(a.pos, a.axis[p], b, s) * a.inv_freq[p] *
                             0.15915494309189535;             // 1 / 2 pi
        const float part = float(turns - rint(turns));
        float sine, cosine;
        sincospif(2.0f * part, &sine, &cosine);
        cs[t * stride + p] = make_float2(cosine, sine * a.sign);
    }
    __syncthreads();
    for (int row = slot; row < rows; row += slots) {
        const Piece8<T> x[2] = {next[0], next[1]};
        char* out = next_out;
        const float2* turn = cs + next_t * stride + p0;
        request(row + slots);
        Piece8<T> y[2] = {x[0], x[1]};
        if (w.turn) {
            float u[2][8], f[2][8];
            piece_expand(x[0], u[0]);
            piece_expand(x[1], u[1]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float2 z = turn[i];
                // pair i: one of each run, or neighbours in one of them
                float& p = SPLIT ? u[0][i] : u[i >> 2][(2 * i) & 7];
                float& q = SPLIT ? u[1][i] : u[i >> 2][(2 * i + 1) & 7];
                (SPLIT ? f[0][i] : f[i >> 2][(2 * i) & 7]) = p * z.x - q * z.y;
                (SPLIT ? f[1][i] : f[i >> 2][(2 * i + 1) & 7]) = q * z.x + p * z.y;
            }
            y[0] = piece_round<T>(f[0]);
            y[1] = piece_round<T>(f[1]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (EVEN || w.d[i] < w.end[i]) piece_store<T, EVEN>(out, w.d[i], w.end[i], y[i]);
    }
}

}  // namespace

hipError_t rope_axes(hipStream_t st, const Heads& q, const Heads& k, int type,
                     const Positions& positions, const double* inv_freq, const int* axis, int P,
                     bool inverse, bool split_half, int64_t B, int64_t S, int D) {
    RotaryArgs a{q, k, positions, inv_freq, axis, uint32_t(S), uint32_t(B * S), 0, P, D, 0, 0, 1,
                 inverse ? -1.f : 1.f};
    a.turned = (P + 7) / 8;
    a.per_head = a.turned + (D - 2 * P + 15) / 16;
    const int threads = a.per_head > 256 ? 512 : 256;  // (a head of 4096 has up to 257 pieces)
    // Positions a block: enough for its threads to go round twice where there are blocks
    // enough for the chip, once where not (48 heads of 128, 32760 positions: 157 us with one,
    // 156 with 2, 160 with 4; 20 of 80, 6141: 13.2, 10.3 and 9.9).
    const int64_t units = int64_t(a.per_head) * (q.H + k.H);
    a.each = int(std::max<int64_t>(1, std::min({(a.tokens >= 4096 ? 512 : 256) / units,
                                                 int64_t(4096 / (8 * a.turned)), B * S / 512})));
    auto go = [&](auto t, auto split) {
        constexpr int T = decltype(t)::value;
        constexpr bool SPLIT = decltype(split)::value;
        auto launch = [&](auto even) {
            in_launches(B * S, kMaxBlocks / 2 * a.each, [&](int64_t at, int64_t m) {
                a.first = uint32_t(at);
                hipLaunchKernelGGL((rotary_kernel<T, SPLIT, decltype(even)::value>),
                                   dim3(unsigned((m + a.each - 1) / a.each)), dim3(threads),
                                   a.each * a.turned * 8 * sizeof(float2), st, a);
            });
        };
        if (P >= 8 && (D == 2 * P || D - 2 * P >= 8)) launch(std::true_type{});
        else launch(std::false_type{});
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
