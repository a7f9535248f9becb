// RMS norm of rows with the residual's addition, its gradient, and the norm with an
// int8 output for the int8 linears.
//
//   h = x + residual, rounded to the stream's type (h = x without one): what the next
//       layer adds to, so the norm is of that value and not of the unrounded sum
//   r = 1 / sqrt(mean(h^2) + eps),  y = h r weight
//   backward, g = dy weight, n = h r:  dx = r (g - n mean(g n)) + dh,  dweight = sum_rows dy n
//       (r^3 by itself would leave fp32's range long before the formula does)
//   int8: v = h weight, rotated by 256s or not; m = max(|v|, 1e-30), NaN if a v is;
//         q = rint(v (127 / m)), scale = r m / 127
//       (an infinity or NaN in the row makes a v infinite or NaN, whatever the weight and the
//       rotation do to it, and r 0 or NaN: the scale is NaN)
//
// Sums are fp32.  A row's codes do not depend on r, so the int8 form needs its sum and its
// maximum at once, in one exchange between the waves.
//
// HBM-bound.  A row lies in registers from its one read to its write, 8 consecutive values
// a lane and piece; the row's waves exchange one pair of numbers through LDS.  bf16 with a
// residual: 16381 x 5120 122 us (5.5 TB/s; a copy of 1 GiB reaches 5.1), 8192 x 4096 46,
// 30001 x 3001 154; 10^6 x 64 without one 47; one row of 4096 2.7, a launch's latency.
#include <algorithm>
#include <type_traits>

#include "block_kernels.hpp"
#include "kernels.hpp"
#include "mx_kernels.hpp"
#include "quantizer.hpp"
#include "rows.hpp"

namespace xpuint8 {
namespace {

struct NormArgs {
    const void* x;
    const void* residual;
    const void* weight;
    void* h;
    void* y;              // int8 codes in the int8 form
    float* scale;
    Lines lx, lr;
    int64_t M, K;
    uint32_t inner;
    int weight_type;
    float eps;
};

// a row of an input: of `inner` rows each, by two strides
template <int T>
__device__ __forceinline__ const char* line_of(const void* p, int64_t row, uint32_t inner,
                                               const Lines& l) {
    int64_t at = row * l.outer;
    if (inner > 1) {
        const uint32_t o = uint32_t(row) / inner;
        at = o * l.outer + int64_t(uint32_t(row) - o * inner) * l.ld;
    }
    return static_cast<const char*>(p) + at * kElem<T>;
}
template <int T>
__device__ __forceinline__ char* row_of(void* p, int64_t row, int64_t ld) {
    return static_cast<char*>(p) + row * ld * kElem<T>;
}

// h's piece at d: read, added and (where there is a residual) stored
template <int T, bool EVEN>
__device__ __forceinline__ Piece8<T> stream_piece(const NormArgs& a, int64_t row, int64_t d) {
    Piece8<T> p = piece_load<T, EVEN>(line_of<T>(a.x, row, a.inner, a.lx), d, a.K);
    if (a.residual) {
        float u[8], v[8];
        piece_expand(p, u);
        piece_expand(piece_load<T, EVEN>(line_of<T>(a.residual, row, a.inner, a.lr), d, a.K), v);
#pragma unroll
        for (int i = 0; i < 8; ++i) u[i] += v[i];
        p = piece_round<T>(u);
        piece_store<T, EVEN>(row_of<T>(a.h, row, a.K), d, a.K, p);
    }
    return p;
}

__device__ __forceinline__ float inverse_rms(float sum, int64_t K, float eps) {
    return 1.0f / sqrtf(sum / float(K) + eps);
}

// Two numbers of each lane to their sum and, MAX, their maximum (NaN if one is; else both sums)
// over the TPR threads of a row.  Above a wave through LDS: one slot a wave, read by all.
template <int TPR, bool MAX>
__device__ __forceinline__ void row_reduce(float& a, float& b, float2* slots) {
    constexpr int N = TPR < 64 ? TPR : 64;
    a = lanes_sum<N>(a);
    b = MAX ? lanes_max_or_nan<N>(b) : lanes_sum<N>(b);
    if constexpr (TPR > 64) {
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) slots[wave] = make_float2(a, b);
        lds_barrier();
        a = slots[0].x;
        b = slots[0].y;
#pragma unroll
        for (int w = 1; w < TPR / 64; ++w) {
            a += slots[w].x;
            b = MAX ? greater_or_nan(b, slots[w].y) : b + slots[w].y;
        }
        lds_barrier();                 // the slots are read before the next row's are written
    }
}

// the codes of 8 values
template <bool EVEN>
__device__ __forceinline__ void codes_store(int8_t* row, int64_t d, int64_t n, const uint2& q) {
    struct __attribute__((packed, aligned(1))) Loose { uint32_t x, y; };
    if (EVEN || d + 8 <= n) {
        auto* p = reinterpret_cast<Loose*>(row + d);
        p->x = q.x;
        p->y = q.y;
        return;
    }
    struct __attribute__((packed, aligned(1))) Four { uint32_t v; };
    struct __attribute__((packed, aligned(1))) Two { uint16_t v; };
    const int c = int(n - d);          // 1..7: in runs of 4, 2 and 1
    if (c & 4) reinterpret_cast<Four*>(row + d)->v = q.x;
    const uint32_t rest = c & 4 ? q.y : q.x;
    if (c & 2) reinterpret_cast<Two*>(row + d + (c & 4))->v = uint16_t(rest);
    if (c & 1) row[d + c - 1] = int8_t(rest >> (c & 2 ? 16 : 0));
}

template <int TPR>
constexpr int kThreads = TPR > 256 ? TPR : 256;

// Rows that are not whole pieces.  Where a row has 8 values at least, its last piece is the
// last 8 of them: it overlaps the piece before, the values of both are the same and are
// written twice, and sums leave the first `skip` of them out.  Shorter rows go value by value.
enum Cut : int { kWhole = 0, kOverlap = 1, kShort = 2 };
constexpr bool whole(int cut) { return cut != kShort; }
template <int CUT>
__device__ __forceinline__ int64_t place(int64_t d, int64_t K) {
    return CUT == kOverlap && d > K - 8 ? K - 8 : d;
}

// TPR threads a row, P pieces of 8 a thread: piece i of thread t is 8 (i TPR + t).
template <int T, int TPR, int P, bool INT8, int CUT>
__global__ __launch_bounds__(kThreads<TPR>) void norm_kernel(NormArgs a) {
    __shared__ float2 slots[16];
    constexpr int R = kThreads<TPR> / TPR;
    const int t = threadIdx.x % TPR;
    for (int64_t row0 = int64_t(blockIdx.x) * R; row0 < a.M; row0 += int64_t(gridDim.x) * R) {
        const int64_t row = row0 + threadIdx.x / TPR;
        const bool live = row < a.M;
        Piece8<T> p[P];
        float w[P][8];
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int64_t d = 8 * (int64_t(i) * TPR + t);
            if (live && d < a.K) {
                const int64_t at = place<CUT>(d, a.K);
                p[i] = stream_piece<T, whole(CUT)>(a, row, at);
                vector_load<whole(CUT)>(a.weight, a.weight_type, at, a.K, w[i]);
            } else {
                p[i] = Piece8<T>{};
            }
        }
        float sum = 0.f, most = 0.f;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            float v[8];
            piece_expand(p[i], v);
            const int64_t d = 8 * (int64_t(i) * TPR + t);
            if (!(live && d < a.K)) continue;
            const int skip = int(d - place<CUT>(d, a.K));
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (CUT == kOverlap && j < skip) continue;
                sum = __builtin_fmaf(v[j], v[j], sum);
                if constexpr (INT8) most = greater_or_nan(most, fabsf(v[j] * w[i][j]));
            }
        }
        row_reduce<TPR, INT8>(sum, most, slots);
        const float r = inverse_rms(sum, a.K, a.eps);
        if (!live) continue;
        const float m = greater_or_nan(most, 1e-30f), inv = 127.0f / m;
        if (INT8 && t == 0) a.scale[row] = r * m / 127.0f;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            int64_t d = 8 * (int64_t(i) * TPR + t);
            if (d >= a.K) continue;
            d = place<CUT>(d, a.K);
            float v[8];
            piece_expand(p[i], v);
            if constexpr (INT8) {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = v[j] * w[i][j] * inv;
                codes_store<whole(CUT)>(static_cast<int8_t*>(a.y) + row * a.K, d, a.K, rint_pack8(v));
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = v[j] * r * w[i][j];
                piece_store<T, whole(CUT)>(row_of<T>(a.y, row, a.K), d, a.K, piece_round<T>(v));
            }
        }
    }
}

// Rows of more than 32768: a block a row, which is read again (h, from cache) to be written.
template <int T, bool INT8, int CUT>
__global__ __launch_bounds__(1024) void norm_long_kernel(NormArgs a) {
    __shared__ float2 slots[16];
    for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
        float sum = 0.f, most = 0.f;
        for (int64_t d = 8 * int64_t(threadIdx.x); d < a.K; d += 8 * 1024) {
            const int64_t at = place<CUT>(d, a.K);
            const int skip = int(d - at);
            float v[8], w[8];
            piece_expand(stream_piece<T, whole(CUT)>(a, row, at), v);
            if constexpr (INT8) vector_load<whole(CUT)>(a.weight, a.weight_type, at, a.K, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (CUT == kOverlap && j < skip) continue;
                sum = __builtin_fmaf(v[j], v[j], sum);
                if constexpr (INT8) most = greater_or_nan(most, fabsf(v[j] * w[j]));
            }
        }
        row_reduce<1024, INT8>(sum, most, slots);
        const float r = inverse_rms(sum, a.K, a.eps);
        const float m = greater_or_nan(most, 1e-30f), inv = 127.0f / m;
        if (INT8 && threadIdx.x == 0) a.scale[row] = r * m / 127.0f;
        // each thread reads what it has written itself (an overlapping piece too)
        const char* from = a.residual ? row_of<T>(a.h, row, a.K)
                                      : line_of<T>(a.x, row, a.inner, a.lx);
        for (int64_t at = 8 * int64_t(threadIdx.x); at < a.K; at += 8 * 1024) {
            const int64_t d = place<CUT>(at, a.K);
            float v[8], w[8];
            piece_expand(piece_load<T, whole(CUT)>(from, d, a.K), v);
            vector_load<whole(CUT)>(a.weight, a.weight_type, d, a.K, w);
            if constexpr (INT8) {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = v[j] * w[j] * inv;
                codes_store<whole(CUT)>(static_cast<int8_t*>(a.y) + row * a.K, d, a.K, rint_pack8(v));
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = v[j] * r * w[j];
                piece_store<T, whole(CUT)>(row_of<T>(a.y, row, a.K), d, a.K, piece_round<T>(v));
            }
        }
    }
}

// ---------------------------------------------------------------- rotated int8
// A group of 256 is 16 lanes of 16 values each, as in the row quantizer; a row is S of
// these segments, a block R rows.  Sums and maxima of the segments meet in LDS.  HBM and, for
// half of the cycles, the vector pipes: 16381 x 5120 bf16 with a residual 109 to 113 us
// (5.3 TB/s; a block a row without requests ahead 135), 16 x 4096 4.2.
constexpr int kMaxSegs = 64;

// h's 16 values at d, times the weight, and their sum of squares
template <int T>
__device__ __forceinline__ void rotated_input(const NormArgs& a, int64_t row, int64_t d,
                                              float (&v)[16], float& sum) {
    constexpr bool EVEN = true;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float h[8], w[8];
        piece_expand(stream_piece<T, EVEN>(a, row, d + 8 * i), h);
        vector_load<EVEN>(a.weight, a.weight_type, d + 8 * i, a.K, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            sum = __builtin_fmaf(h[j], h[j], sum);
            v[8 * i + j] = h[j] * w[j];
        }
    }
}

// the greatest |v|, NaN if one is
__device__ __forceinline__ float magnitude(const float (&v)[16]) {
    float m = fabsf(v[0]);
#pragma unroll
    for (int j = 1; j < 16; ++j) m = greater_or_nan(m, fabsf(v[j]));
    return m;
}

__device__ __forceinline__ void rotated_store(int8_t* row, int64_t d, float (&v)[16], float k) {
    float a[8], b[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        a[j] = v[j] * k;
        b[j] = v[8 + j] * k;
    }
    const uint2 lo = rint_pack8(a), hi = rint_pack8(b);
    *reinterpret_cast<uint4*>(row + d) = make_uint4(lo.x, lo.y, hi.x, hi.y);
}

// G segments meet in a slot: 4, a wave, where a row is whole waves.  A block walks over its
// rows with the next one's reads under way.
template <int T, int G>
__global__ __launch_bounds__(1024) void norm_rotated_kernel(NormArgs a, int S, int R) {
    constexpr bool EVEN = true;
    __shared__ float2 slots[2][kMaxSegs / G];
    const int seg = threadIdx.x >> 4, sl = threadIdx.x & 15;
    const int r = seg / S, sg = seg - r * S;
    const int64_t d = sg * 256 + lane_w(sl) * 16, step = int64_t(gridDim.x) * R;
    const XlaneSigns sgn = xlane_signs(sl);
    float w[2][8];
    Piece8<T> x[2], res[2];
    auto request = [&](int64_t row) {
        if (r >= R || row >= a.M) return;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            x[i] = piece_load<T, EVEN>(line_of<T>(a.x, row, a.inner, a.lx), d + 8 * i, a.K);
            if (a.residual) res[i] = piece_load<T, EVEN>(line_of<T>(a.residual, row, a.inner, a.lr), d + 8 * i, a.K);
        }
    };
#pragma unroll
    for (int i = 0; i < 2; ++i) x[i] = res[i] = Piece8<T>{};
    request(int64_t(blockIdx.x) * R + r);
#pragma unroll
    for (int i = 0; i < 2; ++i)
        vector_load<EVEN>(a.weight, a.weight_type, r < R ? d + 8 * i : 0, a.K, w[i]);
    int turn = 0;
    for (int64_t row = int64_t(blockIdx.x) * R + r; row - r < a.M; row += step, turn ^= 1) {
        const bool live = r < R && row < a.M;
        float v[1][16], sum = 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float h[8];
            piece_expand(x[i], h);
            if (a.residual) {
                float u[8];
                piece_expand(res[i], u);
#pragma unroll
                for (int j = 0; j < 8; ++j) h[j] += u[j];
                const Piece8<T> p = piece_round<T>(h);
                if (live) piece_store<T, EVEN>(row_of<T>(a.h, row, a.K), d + 8 * i, a.K, p);
                piece_expand(p, h);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                sum = __builtin_fmaf(h[j], h[j], sum);
                v[0][8 * i + j] = h[j] * w[i][j];
            }
        }
        request(row + step);
        const float dom = rotate_groups<1>(v, sgn);
        const float most = lanes_max_or_nan<16 * G>(magnitude(v[0]) * dom);
        sum = lanes_sum<16 * G>(sum);
        // (the slots of two rows in turn: one barrier a row)
        if ((threadIdx.x & (16 * G - 1)) == 0) slots[turn][seg / G] = make_float2(sum, most);
        lds_barrier();
        if (!live) continue;
        float total = 0.f, m = 1e-30f;
        for (int i = 0; i < S / G; ++i) {
            const float2 u = slots[turn][r * (S / G) + i];
            total += u.x;
            m = greater_or_nan(m, u.y);
        }
        if (sg == 0 && sl == 0) a.scale[row] = inverse_rms(total, a.K, a.eps) * m / 127.0f;
        rotated_store(static_cast<int8_t*>(a.y) + row * a.K, sg * 256 + lane_w_rot(sl) * 16, v[0],
                      127.0f / m * dom);
    }
}

// Rows of more than 64 groups: a block a row, rotated twice.
template <int T>
__global__ __launch_bounds__(1024) void norm_rotated_long_kernel(NormArgs a) {
    __shared__ float2 slots[kMaxSegs];
    const int seg = threadIdx.x >> 4, sl = threadIdx.x & 15;
    const XlaneSigns sgn = xlane_signs(sl);
    const int64_t groups = a.K / 256;
    for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
        float sum = 0.f, most = 0.f;
        for (int64_t g0 = 0; g0 < groups; g0 += kMaxSegs) {
            float v[1][16];
#pragma unroll
            for (int j = 0; j < 16; ++j) v[0][j] = 0.f;
            if (g0 + seg < groups) rotated_input<T>(a, row, (g0 + seg) * 256 + lane_w(sl) * 16, v[0], sum);
            const float dom = rotate_groups<1>(v, sgn);
            most = greater_or_nan(most, magnitude(v[0]) * dom);
        }
        most = lanes_max_or_nan<16>(most);
        sum = lanes_sum<16>(sum);
        if (sl == 0) slots[seg] = make_float2(sum, most);
        lds_barrier();
        float total = 0.f, m = 1e-30f;
        for (int i = 0; i < kMaxSegs; ++i) {
            const float2 u = slots[i];
            total += u.x;
            m = greater_or_nan(m, u.y);
        }
        lds_barrier();
        if (threadIdx.x == 0) a.scale[row] = inverse_rms(total, a.K, a.eps) * m / 127.0f;
        NormArgs b = a;                // h is there now; each lane reads what it has written
        if (a.residual) {
            b.x = a.h;
            b.lx = Lines{a.K, a.K};
            b.inner = 1;
            b.residual = nullptr;
        }
        for (int64_t g0 = 0; g0 < groups; g0 += kMaxSegs) {
            float v[1][16], unused = 0.f;
#pragma unroll
            for (int j = 0; j < 16; ++j) v[0][j] = 0.f;
            if (g0 + seg < groups) rotated_input<T>(b, row, (g0 + seg) * 256 + lane_w(sl) * 16, v[0], unused);
            const float dom = rotate_groups<1>(v, sgn);
            if (g0 + seg < groups)
                rotated_store(static_cast<int8_t*>(a.y) + row * a.K,
                              (g0 + seg) * 256 + lane_w_rot(sl) * 16, v[0], 127.0f / m * dom);
        }
    }
}

// ----------------------------------------------------------------------- gradient
struct GradArgs {
    const void* dy;
    const void* h;
    const void* weight;
    const void* dh;
    void* dx;
    float* part;          // [blocks, K], null: the weight's gradient is not wanted
    Lines ldy, lh, ldh;
    int64_t M, K;
    uint32_t inner;
    int weight_type;
    float eps;
};

// A block walks over its rows and keeps the weight's gradient over them in registers; the
// blocks' sums are added in order by a launch of their own.  Nothing of the forward pass is
// kept but h: r comes from its squares again, in the same exchange as the sum along g.
// HBM-bound: 8192 x 4096 bf16 with both gradients 44 us (6.0 TB/s, some of it from cache) and
// 4.0 for the weight's sums.
template <int T, int TPR, int P, int CUT>
__global__ __launch_bounds__(kThreads<TPR>) void norm_grad_kernel(GradArgs a) {
    __shared__ float2 slots[16];
    constexpr int R = kThreads<TPR> / TPR;
    __shared__ float cols[R > 1 ? R : 1][R > 1 ? TPR * P * 8 : 1];
    const int t = threadIdx.x % TPR, mine = threadIdx.x / TPR;
    float w[P][8], dw[P][8];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int64_t d = 8 * (int64_t(i) * TPR + t);
#pragma unroll
        for (int j = 0; j < 8; ++j) w[i][j] = dw[i][j] = 0.f;
        if (d < a.K) vector_load<whole(CUT)>(a.weight, a.weight_type, place<CUT>(d, a.K), a.K, w[i]);
    }
    for (int64_t row0 = int64_t(blockIdx.x) * R; row0 < a.M; row0 += int64_t(gridDim.x) * R) {
        const int64_t row = row0 + mine;
        const bool live = row < a.M;
        Piece8<T> h[P], dy[P], dh[P];
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int64_t d = 8 * (int64_t(i) * TPR + t);
            h[i] = dy[i] = dh[i] = Piece8<T>{};
            if (live && d < a.K) {
                const int64_t at = place<CUT>(d, a.K);
                h[i] = piece_load<T, whole(CUT)>(line_of<T>(a.h, row, a.inner, a.lh), at, a.K);
                dy[i] = piece_load<T, whole(CUT)>(line_of<T>(a.dy, row, a.inner, a.ldy), at, a.K);
                if (a.dh) dh[i] = piece_load<T, whole(CUT)>(line_of<T>(a.dh, row, a.inner, a.ldh), at, a.K);
            }
        }
        float sum = 0.f, along = 0.f;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int64_t d = 8 * (int64_t(i) * TPR + t);
            const int skip = int(d - place<CUT>(d, a.K));
            float u[8], g[8];
            piece_expand(h[i], u);
            piece_expand(dy[i], g);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (CUT == kOverlap && j < skip) continue;
                sum = __builtin_fmaf(u[j], u[j], sum);
                along = __builtin_fmaf(g[j] * w[i][j], u[j], along);
            }
        }
        row_reduce<TPR, false>(sum, along, slots);
        if (!live) continue;
        const float r = inverse_rms(sum, a.K, a.eps);
        const float back = along * r / float(a.K);
#pragma unroll
        for (int i = 0; i < P; ++i) {
            int64_t d = 8 * (int64_t(i) * TPR + t);
            if (d >= a.K) continue;
            const int skip = int(d - place<CUT>(d, a.K));
            d -= skip;
            float u[8], g[8], o[8];
            piece_expand(h[i], u);
            piece_expand(dy[i], g);
            piece_expand(dh[i], o);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float n = u[j] * r;
                if (!(CUT == kOverlap && j < skip)) dw[i][j] = __builtin_fmaf(g[j], n, dw[i][j]);
                o[j] += r * __builtin_fmaf(-n, back, g[j] * w[i][j]);
            }
            piece_store<T, whole(CUT)>(row_of<T>(a.dx, row, a.K), d, a.K, piece_round<T>(o));
        }
    }
    if (!a.part) return;
    if constexpr (R > 1) {             // the block's rows side by side: one sum
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int d = 8 * (i * TPR + t), skip = d < a.K ? int(d - place<CUT>(d, a.K)) : 0;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (!(CUT == kOverlap && j < skip)) cols[mine][d - skip + j] = dw[i][j];
        }
        __syncthreads();
        for (int c = threadIdx.x; c < a.K; c += kThreads<TPR>) {
            float s = 0.f;
#pragma unroll
            for (int g = 0; g < R; ++g) s += cols[g][c];
            a.part[int64_t(blockIdx.x) * a.K + c] = s;
        }
    } else {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int64_t d = 8 * (int64_t(i) * TPR + t);
            if (d >= a.K) continue;
            float* to = a.part + int64_t(blockIdx.x) * a.K;
            if (CUT == kOverlap && d > a.K - 8) {
                const int skip = int(d - (a.K - 8));
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (j >= skip) to[a.K - 8 + j] = dw[i][j];
            } else {
                piece_store<kF32, whole(CUT)>(to, d, a.K, piece_round<kF32>(dw[i]));
            }
        }
    }
}

// Rows longer than a block's registers: read twice, the weight's gradient kept in `part`
// (every thread its own columns).
template <int T, int CUT>
__global__ __launch_bounds__(1024) void norm_grad_long_kernel(GradArgs a) {
    __shared__ float2 slots[16];
    float* part = a.part ? a.part + int64_t(blockIdx.x) * a.K : nullptr;
    for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
        const char *hr = line_of<T>(a.h, row, a.inner, a.lh), *dyr = line_of<T>(a.dy, row, a.inner, a.ldy);
        float sum = 0.f, along = 0.f;
        for (int64_t d = 8 * int64_t(threadIdx.x); d < a.K; d += 8 * 1024) {
            const int64_t at = place<CUT>(d, a.K);
            const int skip = int(d - at);
            float u[8], g[8], w[8];
            piece_expand(piece_load<T, whole(CUT)>(hr, at, a.K), u);
            piece_expand(piece_load<T, whole(CUT)>(dyr, at, a.K), g);
            vector_load<whole(CUT)>(a.weight, a.weight_type, at, a.K, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (CUT == kOverlap && j < skip) continue;
                sum = __builtin_fmaf(u[j], u[j], sum);
                along = __builtin_fmaf(g[j] * w[j], u[j], along);
            }
        }
        row_reduce<1024, false>(sum, along, slots);
        const float r = inverse_rms(sum, a.K, a.eps);
        const float back = along * r / float(a.K);
        for (int64_t d = 8 * int64_t(threadIdx.x); d < a.K; d += 8 * 1024) {
            const int64_t at = place<CUT>(d, a.K);
            const int skip = int(d - at);
            float u[8], g[8], w[8], o[8] = {};
            piece_expand(piece_load<T, whole(CUT)>(hr, at, a.K), u);
            piece_expand(piece_load<T, whole(CUT)>(dyr, at, a.K), g);
            vector_load<whole(CUT)>(a.weight, a.weight_type, at, a.K, w);
            if (a.dh)
                piece_expand(piece_load<T, whole(CUT)>(line_of<T>(a.dh, row, a.inner, a.ldh), at, a.K), o);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float n = u[j] * r, term = g[j] * n;
                if (part && j >= skip && at + j < a.K)
                    part[at + j] = row == int64_t(blockIdx.x) ? term : part[at + j] + term;
                o[j] += r * __builtin_fmaf(-n, back, g[j] * w[j]);
            }
            piece_store<T, whole(CUT)>(row_of<T>(a.dx, row, a.K), at, a.K, piece_round<T>(o));
        }
    }
}

// dweight = the sum of part's rows, 32 columns a block: 32 slices of rows, then their sums
template <int WT>
__global__ __launch_bounds__(1024) void norm_dweight_kernel(const float* __restrict__ part,
                                                            void* __restrict__ dweight, int rows,
                                                            int64_t K) {
    __shared__ float sums[32][33];
    const int c = threadIdx.x & 31, slice = threadIdx.x >> 5;
    const int64_t col = int64_t(blockIdx.x) * 32 + c;
    float s = 0.f;
    if (col < K) {
#pragma unroll 8
        for (int i = slice; i < rows; i += 32) s += part[int64_t(i) * K + col];
    }
    sums[slice][c] = s;
    __syncthreads();
    if (slice != 0 || col >= K) return;
    float total = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) total += sums[i][c];
    if constexpr (WT == kF32) static_cast<float*>(dweight)[col] = total;
    else static_cast<uint16_t*>(dweight)[col] = uint16_t(pack2<WT>(total, 0.f));
}

// ------------------------------------------------------------------------ launches
template <class F>
void by_type(int type, const F& f) {
    if (type == kBf16) f(std::integral_constant<int, kBf16>{});
    else if (type == kF16) f(std::integral_constant<int, kF16>{});
    else f(std::integral_constant<int, kF32>{});
}
template <class F>
void by_cut(int64_t K, const F& f) {
    if (K % 8 == 0) f(std::integral_constant<int, kWhole>{});
    else if (K > 8) f(std::integral_constant<int, kOverlap>{});
    else f(std::integral_constant<int, kShort>{});
}
template <int A, int B>
struct Shape {
    static constexpr int tpr = A, p = B;
};
// f(threads a row, pieces a thread) for rows of K: rows of up to 512 lie in 8 to 64 lanes,
// up to 2048 in a wave, up to 8192 in 256 threads, up to 32768 in 1024.  False above.
template <class F>
bool by_length(int64_t K, const F& f) {
    const int64_t c = (K + 7) / 8;
    if (c <= 8) f(Shape<8, 1>{});
    else if (c <= 16) f(Shape<16, 1>{});
    else if (c <= 32) f(Shape<32, 1>{});
    else if (c <= 64) f(Shape<64, 1>{});
    else if (c <= 128) f(Shape<64, 2>{});
    else if (c <= 192) f(Shape<64, 3>{});
    else if (c <= 256) f(Shape<64, 4>{});
    else if (c <= 512) f(Shape<256, 2>{});
    else if (c <= 768) f(Shape<256, 3>{});
    else if (c <= 1024) f(Shape<256, 4>{});
    else if (c <= 2048) f(Shape<1024, 2>{});
    else if (c <= 4096) f(Shape<1024, 4>{});
    else return false;
    return true;
}
constexpr int64_t kRowBlocks = kMaxBlocks / 4;
unsigned blocks_for(int64_t M, int rows, int64_t most) {
    const int64_t n = (M + rows - 1) / rows;
    return unsigned(n < most ? n : most);
}

template <bool INT8>
hipError_t launch_norm(hipStream_t st, int type, const NormArgs& a) {
    by_type(type, [&](auto t) { by_cut(a.K, [&](auto e) {
        constexpr int T = decltype(t)::value;
        constexpr int CUT = decltype(e)::value;
        const bool done = by_length(a.K, [&](auto s) {
            constexpr int TPR = decltype(s)::tpr, P = decltype(s)::p, N = kThreads<TPR>;
            if constexpr (CUT != kShort || TPR == 8)
                hipLaunchKernelGGL((norm_kernel<T, TPR, P, INT8, CUT>),
                               dim3(blocks_for(a.M, N / TPR, kRowBlocks)), dim3(N), 0, st, a);
        });
        if constexpr (CUT != kShort)
            if (!done)
                hipLaunchKernelGGL((norm_long_kernel<T, INT8, CUT>),
                               dim3(blocks_for(a.M, 1, kRowBlocks)), dim3(1024), 0, st, a);
    }); });
    return hipGetLastError();
}

// blocks of the gradient's launch: each writes K fp32 sums for the weight, so no more than
// fill the chip (forward and backward of 8192 x 4096: 112 us with 256, 96 with 512, 99 with
// 1024, 105 with 2048; 10^6 x 64: 180, 127, 123, 124)
constexpr int64_t kGradBlocks = 512;
int grad_rows(int64_t K) { return K <= 64 ? 32 : K <= 128 ? 16 : K <= 256 ? 8 : K <= 2048 ? 4 : 1; }

}  // namespace

hipError_t rms_norm(hipStream_t st, const void* x, int type, const Lines& lx,
                    const void* residual, const Lines& lr, int64_t inner, const void* weight,
                    int weight_type, float eps, void* h, void* y, int64_t M, int64_t K) {
    return launch_norm<false>(st, type, NormArgs{x, residual, weight, h, y, nullptr, lx, lr, M, K,
                                                 uint32_t(inner), weight_type, eps});
}

hipError_t rms_norm_int8(hipStream_t st, const void* x, int type, const Lines& lx,
                         const void* residual, const Lines& lr, int64_t inner,
                         const void* weight, int weight_type, float eps, void* h, int8_t* q,
                         float* scale, bool rotate, int64_t M, int64_t K) {
    const NormArgs a{x, residual, weight, h, q, scale, lx, lr, M, K, uint32_t(inner), weight_type, eps};
    if (!rotate) return launch_norm<true>(st, type, a);
    by_type(type, [&](auto t) {
        constexpr int T = decltype(t)::value;
        if (K <= 256 * kMaxSegs) {
            // rows of few groups share a block of 16
            const int S = int(K / 256), R = S >= 16 ? 1 : 16 / S;
            const int threads = (S * R * 16 + 63) / 64 * 64;
            // Blocks that together request 40 KB a CU, 60 without a residual (no fewer than
            // one, no more than its 16 waves): more rows under way at once are slower.
            // 16381 x 5120 bf16 with a residual (40 KB: 2 blocks): 118 us with 1, 111 with 2,
            // 131 with 3, 123 with 6; 8192 x 8192 85 with 1, 91 with 2; 20000 x 4096 without
            // one 64 with 2, 52 with 4.
            const int bytes = threads * 16 * kElem<T> * (residual ? 2 : 1);
            const int each = std::max(1, std::min((residual ? 40960 : 61440) / bytes, 1024 / threads));
            const dim3 grid(blocks_for(M, R, int64_t(each) * device_cus()));
            if (S % 4 == 0)
                hipLaunchKernelGGL((norm_rotated_kernel<T, 4>), grid, dim3(threads), 0, st, a, S, R);
            else
                hipLaunchKernelGGL((norm_rotated_kernel<T, 1>), grid, dim3(threads), 0, st, a, S, R);
        } else {
            hipLaunchKernelGGL((norm_rotated_long_kernel<T>), dim3(blocks_for(M, 1, kRowBlocks)),
                               dim3(1024), 0, st, a);
        }
    });
    return hipGetLastError();
}

int64_t rms_norm_grad_work_bytes(int64_t M, int64_t K) {
    return int64_t(blocks_for(M, grad_rows(K), kGradBlocks)) * K * 4;
}

hipError_t rms_norm_grad(hipStream_t st, const void* dy, int type, const Lines& ldy,
                         const void* h, const Lines& lh, const void* weight, int weight_type,
                         const void* dh, const Lines& ldh, int64_t inner, float eps, void* dx,
                         void* dweight, int64_t M, int64_t K, float* part) {
    const GradArgs a{dy, h, weight, dh, dx, dweight ? part : nullptr, ldy, lh, ldh, M, K,
                     uint32_t(inner), weight_type, eps};
    const unsigned blocks = blocks_for(M, grad_rows(K), kGradBlocks);
    by_type(type, [&](auto t) { by_cut(K, [&](auto e) {
        constexpr int T = decltype(t)::value;
        constexpr int CUT = decltype(e)::value;
        const bool done = K <= 16384 && by_length(K, [&](auto s) {
            constexpr int TPR = decltype(s)::tpr, P = decltype(s)::p, N = kThreads<TPR>;
            if constexpr (TPR * P <= 2048 && (CUT != kShort || TPR == 8))
                hipLaunchKernelGGL((norm_grad_kernel<T, TPR, P, CUT>), dim3(blocks), dim3(N), 0, st, a);
        });
        if constexpr (CUT != kShort)
            if (!done)
                hipLaunchKernelGGL((norm_grad_long_kernel<T, CUT>), dim3(blocks), dim3(1024), 0, st, a);
    }); });
    if (!dweight) return hipGetLastError();
    by_type(weight_type, [&](auto t) {
        hipLaunchKernelGGL((norm_dweight_kernel<decltype(t)::value>),
                           dim3(unsigned((K + 31) / 32)), dim3(1024), 0, st, part, dweight,
                           int(blocks), K);
    });
    return hipGetLastError();
}

}  // namespace xpuint8
