// MXFP4 quantization and its reading back (mx4.hpp has the format).
//
// Both are bound by HBM: one pass, a lane takes 8 consecutive values (16 bytes of
// a 16-bit type, 4 bytes of codes), a quad of lanes one block of 32, a wave the
// 512 values whose 16 scale bytes lie together.  The block's maximum crosses the
// quad in two DPP steps, so no value waits for another quad's; a wave that quantizes
// requests U such groups before it uses the first.  Groups are numbered row by row (G of
// them a row, the last one partly past K: there only the padding scale bytes are
// written), and every count is 64-bit.  MI355X, 16381 x 5120 bf16: 49 us (4.3 TB/s) from
// HBM, back 33 (6.5 TB/s, the codes still in the last-level cache).
#include "mx4.hpp"
#include "mx_kernels.hpp"

namespace xpuint8 {
namespace {

template <int T>
constexpr int kSize = T == kF32 ? 4 : 2;

template <int T, bool VEC, int U>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(const char* __restrict__ x, int64_t ldx,
                                                           uint8_t* __restrict__ codes,
                                                           uint8_t* __restrict__ scales,
                                                           int64_t groups, int G, int K) {
    const int lane = threadIdx.x & 63;
    const int64_t wave = int64_t(blockIdx.x) * 4 +
                         __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
    const int64_t first = wave * U;
    float v[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t g = first + u;
        if (g >= groups) break;
        const int64_t row = g / G;
        const int k = int(g - row * G) * 512 + lane * 8;
        if (k < K) {
            load8<T, VEC>(x + (row * ldx + k) * kSize<T>, v[u]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[u][i] = 0.f;
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t g = first + u;
        if (g >= groups) break;
        const int64_t row = g / G;
        const int sg = int(g - row * G);
        const int k = sg * 512 + lane * 8;
        uint32_t m = abs_bits(v[u][0]);
#pragma unroll
        for (int i = 1; i < 8; ++i) m = max(m, abs_bits(v[u][i]));
        m = max(m, dppu<kDppXor1>(m));
        m = max(m, dppu<kDppXor2>(m));
        const uint32_t e = mx_scale_byte(m);
        if (k < K) *reinterpret_cast<uint32_t*>(codes + row * (K / 2) + k / 2) = mx_encode8(v[u], e);
        if ((lane & 3) == 0)
            scales[row * (int64_t(G) * 16) + sg * 16 + lane / 4] = uint8_t(k < K ? e : 127u);
    }
}

template <int T>
__global__ __launch_bounds__(256) void mx4_dequantize_kernel(const uint8_t* __restrict__ codes,
                                                             const uint8_t* __restrict__ scales,
                                                             char* __restrict__ out,
                                                             int64_t groups, int G, int K) {
    const int lane = threadIdx.x & 63;
    const int64_t g = int64_t(blockIdx.x) * 4 +
                      __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
    if (g >= groups) return;
    const int64_t row = g / G;
    const int sg = int(g - row * G), k = sg * 512 + lane * 8;
    if (k >= K) return;
    float v[8];
    mx_decode8(*reinterpret_cast<const uint32_t*>(codes + row * (K / 2) + k / 2),
               scales[row * (int64_t(G) * 16) + sg * 16 + lane / 4], v);
    store8<T, true>(out + (row * K + k) * kSize<T>, v);
}

template <int T, bool VEC>
void launch_quantize(hipStream_t st, const char* p, int64_t ldx, uint8_t* codes, uint8_t* scales,
                     int64_t groups, int G, int K) {
    // four groups a wave once that still leaves each CU several waves: 35 against 36 us at
    // 16381 x 5120 in a row, 8.3 / 8.7 at 4096 x 4096 (reading back gains nothing by it)
    if (groups >= 16384)
        hipLaunchKernelGGL((mx4_quantize_kernel<T, VEC, 4>), dim3(unsigned((groups + 15) / 16)),
                           dim3(256), 0, st, p, ldx, codes, scales, groups, G, K);
    else
        hipLaunchKernelGGL((mx4_quantize_kernel<T, VEC, 1>), dim3(unsigned((groups + 3) / 4)),
                           dim3(256), 0, st, p, ldx, codes, scales, groups, G, K);
}

template <int T>
void launch_dequantize(hipStream_t st, const uint8_t* codes, const uint8_t* scales, char* p,
                       int64_t groups, int G, int K) {
    hipLaunchKernelGGL((mx4_dequantize_kernel<T>), dim3(unsigned((groups + 3) / 4)), dim3(256), 0,
                       st, codes, scales, p, groups, G, K);
}

}  // namespace

hipError_t mx4_quantize(hipStream_t st, const void* x, int type, int64_t ldx, uint8_t* codes,
                        uint8_t* scales, int64_t M, int K) {
    const int G = (K + 511) / 512;
    const int size = type == kF32 ? 4 : 2;
    const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && (ldx * size) % 16 == 0;
    in_launches(M, 16 * kMaxBlocks / G, [&](int64_t at, int64_t rows) {
        auto go = [&](auto T) {
            constexpr int t = decltype(T)::value;
            const char* p = static_cast<const char*>(x) + at * ldx * size;
            uint8_t* c = codes + at * (K / 2);
            uint8_t* s = scales + at * (G * 16);
            if (vec) launch_quantize<t, true>(st, p, ldx, c, s, rows * G, G, K);
            else launch_quantize<t, false>(st, p, ldx, c, s, rows * G, G, K);
        };
        if (type == kBf16) go(std::integral_constant<int, kBf16>{});
        else if (type == kF16) go(std::integral_constant<int, kF16>{});
        else go(std::integral_constant<int, kF32>{});
    });
    return hipGetLastError();
}

hipError_t mx4_dequantize(hipStream_t st, const uint8_t* codes, const uint8_t* scales, void* out,
                          int type, int64_t M, int K) {
    const int G = (K + 511) / 512;
    const int size = type == kF32 ? 4 : 2;
    in_launches(M, 4 * kMaxBlocks / G, [&](int64_t at, int64_t rows) {
        const uint8_t* c = codes + at * (K / 2);
        const uint8_t* s = scales + at * (G * 16);
        char* o = static_cast<char*>(out) + at * K * size;
        if (type == kBf16) launch_dequantize<kBf16>(st, c, s, o, rows * G, G, K);
        else if (type == kF16) launch_dequantize<kF16>(st, c, s, o, rows * G, G, K);
        else launch_dequantize<kF32>(st, c, s, o, rows * G, G, K);
    });
    return hipGetLastError();
}

}  // namespace xpuint8
