// The bias gradient of an MXFP4 linear:
//
//   db[n] = sum_m dy[m, n]
//
// in fp32 in a fixed order, rounded once to the bias's type, which need not be dy's: the
// sums of 32 consecutive rows, each in row order, then of those sums eight interleaved
// ones (w, w + 8, w + 16, ..) added in the order w = 0..7.  That order is
// xpuint8_column_sum_stream's, so bf16 of bf16 is bit for bit the int8 linear's.
// Bound by HBM: one read of dy and 4 bytes a column and 32 rows of partial sums; a lane
// takes 8 columns, in one load where dy's rows are whole, aligned 8s, and has eight rows
// on their way as they are stored (converted as they come, one behind another: 12.3 us).
// The second launch is bound by latency.  MI355X, 4096 x 5120 bf16: 8.1 us (5.5 TB/s of dy
// and sums) + 3.9.
#include <algorithm>
#include <type_traits>

#include "mx4.hpp"
#include "mx_kernels.hpp"

namespace xpuint8 {
namespace {

constexpr int kRows = 32, kCols = 2048;                   // of a block of the first launch

// eight values of a row as they are stored, so that many rows are on their way before the
// first is converted; without VEC as fp32
template <int T, bool VEC>
struct Raw {
    uint4 u[T == kF32 ? 2 : 1];
    __device__ __forceinline__ void load(const char* row, int64_t n, int64_t) {
        const uint4* p = reinterpret_cast<const uint4*>(row + n * (T == kF32 ? 4 : 2));
#pragma unroll
        for (int i = 0; i < (T == kF32 ? 2 : 1); ++i) u[i] = p[i];
    }
    __device__ __forceinline__ void get(float (&v)[8]) const { load8<T, true>(u, v); }
};
template <int T>
struct Raw<T, false> {
    float u[8];
    __device__ __forceinline__ void load(const char* row, int64_t n, int64_t N) { load_row8<T, false>(row, n, N, u); }
    __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = u[i];
    }
};

// part[c, n], c a chunk of kRows rows, a row of `ldp` sums
template <int T, bool VEC>
__global__ __launch_bounds__(256) void mx4_dbias_part_kernel(const char* __restrict__ dy, int64_t ldy,
                                                             float* __restrict__ part, int64_t ldp,
                                                             int64_t M, int N, int chunks) {
    constexpr int size = T == kF32 ? 4 : 2;
    const int64_t n = int64_t(blockIdx.x) * kCols + threadIdx.x * 8;
    if (n >= N) return;
    for (int c = blockIdx.y; c < chunks; c += gridDim.y) {
        const int64_t m0 = int64_t(c) * kRows;
        const int rows = int(min(int64_t(kRows), M - m0));
        float a[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        for (int r0 = 0; r0 < rows; r0 += 8) {
            Raw<T, VEC> raw[8];
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (r0 + u < rows) raw[u].load(dy + (m0 + r0 + u) * ldy * size, n, N);
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                if (r0 + u >= rows) break;
                float v[8];
                raw[u].get(v);
#pragma unroll
                for (int i = 0; i < 8; ++i) a[i] += v[i];
            }
        }
        store8<kF32, true>(part + c * ldp + n, a);        // (ldp is whole 8s)
    }
}

template <int TO>
__global__ __launch_bounds__(512) void mx4_dbias_kernel(const float* __restrict__ part, int64_t ldp,
                                                        void* __restrict__ out, int chunks, int N) {
    __shared__ float t[8][64];
    const int w = threadIdx.x >> 6, l = threadIdx.x & 63;
    const int64_t n = int64_t(blockIdx.x) * 64 + l, nc = min(n, int64_t(N) - 1);
    float a = 0.f;
    for (int c0 = w; c0 < chunks; c0 += 8 * 16) {
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int c = c0 + 8 * i;
            v[i] = c < chunks ? part[c * ldp + nc] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (c0 + 8 * i < chunks) a += v[i];
    }
    t[w][l] = a;
    __syncthreads();
    if (w != 0 || n >= N) return;
    float s = t[0][l];
#pragma unroll
    for (int i = 1; i < 8; ++i) s += t[i][l];
    if constexpr (TO == kF32) static_cast<float*>(out)[n] = s;
    else if constexpr (TO == kBf16) static_cast<uint16_t*>(out)[n] = uint16_t(f32_to_bf16_bits(s));
    else static_cast<_Float16*>(out)[n] = _Float16(s);
}

int64_t chunks_of(int64_t M) { return (M + kRows - 1) / kRows; }
int64_t row_of_sums(int64_t N) { return (N + 7) / 8 * 8; }

template <class F>
void by_type(int type, const F& f) {
    if (type == kBf16) f(std::integral_constant<int, kBf16>{});
    else if (type == kF16) f(std::integral_constant<int, kF16>{});
    else f(std::integral_constant<int, kF32>{});
}

}  // namespace

int64_t mx4_dbias_work_bytes(int64_t M, int64_t N) { return chunks_of(M) * row_of_sums(N) * 4; }

hipError_t mx4_dbias(hipStream_t st, const void* dy, int type, int64_t ldy, void* out, int out_type,
                     int64_t M, int N, float* part) {
    const int chunks = int(chunks_of(M));
    const int64_t ldp = row_of_sums(N);
    const int size = type == kF32 ? 4 : 2;
    const bool vec = N % 8 == 0 && reinterpret_cast<uintptr_t>(dy) % 16 == 0 && ldy * size % 16 == 0;
    const dim3 grid(unsigned((int64_t(N) + kCols - 1) / kCols), unsigned(std::min(chunks, 65535)));
    by_type(type, [&](auto T) {
        auto go = [&](auto V) {
            hipLaunchKernelGGL((mx4_dbias_part_kernel<decltype(T)::value, decltype(V)::value>), grid,
                               dim3(256), 0, st, static_cast<const char*>(dy), ldy, part, ldp, M, N,
                               chunks);
        };
        if (vec) go(std::true_type{});
        else go(std::false_type{});
    });
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    by_type(out_type, [&](auto T) {
        hipLaunchKernelGGL((mx4_dbias_kernel<decltype(T)::value>), dim3(unsigned((int64_t(N) + 63) / 64)),
                           dim3(512), 0, st, part, ldp, out, chunks, N);
    });
    return hipGetLastError();
}

}  // namespace xpuint8
