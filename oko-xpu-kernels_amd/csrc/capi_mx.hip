// The C ABI of the MXFP4 and mixture-of-experts operators (include/xpuint8.h):
// argument checks, workspaces and dispatch to the launchers in mx_kernels.hpp.  As in
// capi.hip, every check runs before any HIP call.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

#include "capi.hpp"
#include "kernels.hpp"
#include "mx4.hpp"
#include "mx_kernels.hpp"
#include "../../include/xpuint8.h"

namespace xpuint8 {
namespace {

constexpr int kMaxExperts = 1024;                      // the sort's counters in LDS
constexpr int64_t kMaxUnits = int64_t(1) << 32;        // 16-byte units of one operand

int check_type(int32_t type, const char* what) {
    if (type < 0 || type > 2)
        return fail(6, std::string(what) + " must be 0 (bf16), 1 (fp16) or 2 (fp32)");
    return 0;
}

int check_mx(int64_t M, int64_t K) {
    if (M <= 0 || K <= 0) return fail(2, "rows and K must be positive");
    if (K % 32 != 0) return fail(3, "K must be a multiple of the MXFP4 block (32)");
    if (M > kMaxDim || K > kMaxDim) return fail(4, "rows and K must be < 2^31");
    if (M * ((K + 511) / 512) > kMaxDim * 4) return fail(4, "rows x K is too large for one launch");
    return 0;
}

int check_product(int64_t R, int64_t tokens, int64_t N, int64_t K, bool grouped, int64_t E) {
    if (R <= 0 || tokens <= 0 || N <= 0) return fail(2, "rows, tokens and N must be positive");
    if (K <= 0) return fail(2, "K must be positive");
    if (K % 32 != 0) return fail(3, "K must be a multiple of the MXFP4 block (32)");
    if (R > kMaxDim || tokens > kMaxDim || N > kMaxDim)
        return fail(4, "rows, tokens and N must be < 2^31");
    if (K > int64_t(1) << 24) return fail(4, "K must be at most 2^24");    // (256 rows of a tile: 2 GiB)
    if (grouped && (E < 1 || E > kMaxExperts)) return fail(2, "experts must be 1..1024");
    if (tokens * (K / 32) >= kMaxUnits || N * (K / 32) >= kMaxUnits || tokens * N >= kMaxUnits * 16)
        return fail(4, "an operand of more than 2^32 blocks is not supported");
    if (((R + 15) / 16 + E + 1) * ((N + 15) / 16) > kMaxDim || R * ((K + 127) / 128) > kMaxDim * 64)
        return fail(4, "rows x N or rows x K is too large for one launch");
    return 0;
}

// the tiles of a product and of its gradient
int check_blocks(int64_t blocks) {
    if (!mx4_blocks_fit(blocks)) return fail(4, "rows x N or rows x K is too large for one launch");
    return 0;
}
int check_linear(int64_t R, int64_t tokens, int64_t N, int64_t K, bool grouped, int64_t E) {
    XPU_TRY(check_product(R, tokens, N, K, grouped, E));
    if (mx4_fused(R, grouped, int(E), K)) return 0;
    return check_blocks(mx4_product_blocks(grouped, R, grouped ? int(E) : 1, N, K));
}
int check_gradient(int64_t R, int64_t N, int64_t K, bool grouped, int64_t E) {
    XPU_TRY(check_product(R, R, N, K, grouped, E));
    return check_blocks(mx4_dx_blocks(grouped, R, grouped ? int(E) : 1, N, K));
}

int check_dbias(int64_t M, int64_t N) {
    if (M <= 0 || N <= 0) return fail(2, "rows and N must be positive");
    if (M > kMaxDim || N >= int64_t(1) << 28) return fail(4, "rows must be < 2^31 and N < 2^28");
    return 0;
}

int check_moe(int64_t T, int64_t top, int64_t E) {
    if (T <= 0 || top <= 0) return fail(2, "tokens and slots must be positive");
    if (E < 1 || E > kMaxExperts) return fail(2, "experts must be 1..1024");
    if (T > kMaxDim || top > kMaxDim || T * top > kMaxDim - 65536)
        return fail(4, "tokens x slots must be < 2^31 - 65536");
    return 0;
}

int check_rows_of(int64_t T, int64_t top, int64_t E, int64_t D) {
    XPU_TRY(check_moe(T, top, E));
    if (D <= 0) return fail(2, "D must be positive");
    if (D > kMaxDim / 2 || T * ((D + 511) / 512) > kMaxDim * 4)
        return fail(4, "tokens x D is too large for one launch");
    return 0;
}

int64_t up(int64_t b) { return (b + 255) & ~int64_t(255); }

// quantized x: codes, then scales, each on a 256-byte boundary
int64_t quantized_bytes(int64_t tokens, int64_t K) {
    return up(tokens * (K / 2)) + up(tokens * mx_scale_width(K));
}

int product(const void* stream, const void* x, int32_t type, int64_t ldx, const int32_t* rows,
            int64_t tokens, const uint8_t* codes, const uint8_t* scales, const int32_t* offsets,
            int64_t E, const void* bias, int32_t bias_type, void* y, int64_t R, int64_t N,
            int64_t K, void* work, int64_t work_bytes, const char* what) {
    const bool grouped = offsets != nullptr;
    const bool fused = mx4_fused(R, grouped, int(E), K);
    if (!fused) {
        if (!work) return fail(6, "work must not be null");
        if (reinterpret_cast<uintptr_t>(work) % 16 != 0)
            return fail(6, "work must be 16-byte aligned");
        if (work_bytes < quantized_bytes(tokens, K))
            return fail(2, std::string("work must hold ") + what + "_workspace_size bytes");
    }
    XPU_TRY(ensure_device());
    hipStream_t st = as_stream(stream);
    if (fused)
        return launched(mx4_product_fused(st, x, type, ldx, rows, tokens, codes, scales, offsets,
                                          int(E), y, bias, bias_type, R, int(N), int(K)), what);
    uint8_t* xc = static_cast<uint8_t*>(work);
    uint8_t* xs = xc + up(tokens * (K / 2));
    XPU_TRY(launched(mx4_quantize(st, x, type, ldx, xc, xs, tokens, int(K)), what));
    return launched(mx4_product(st, xc, xs, rows, tokens, codes, scales, offsets, int(E), y, type,
                                bias, bias_type, R, int(N), int(K)), what);
}

// whether dy goes to the product as it is: whole 16-byte chunks in every row
bool dy_direct(const void* dy, int32_t type, int64_t ldy, int64_t N) {
    return type == kBf16 && N % 8 == 0 && ldy % 8 == 0 &&
           reinterpret_cast<uintptr_t>(dy) % 16 == 0;
}

// Whether dx of one weight goes through the weight as bf16 in the workspace and the
// framework's bf16 product (gemm_bf16_nn): bf16 of whole 16s, where that is the faster.
bool dx_by_bf16(int32_t type, int32_t dx_type, bool grouped, int64_t R, int64_t N, int64_t K) {
    return type == kBf16 && dx_type == kBf16 && !grouped && N % 16 == 0 && K % 16 == 0 &&
           mx4_dx_bf16_faster(R, N, K);
}

// dx's workspaces: the weight as bf16 and its product's slices, or dy's pieces
int64_t bf16_dx_bytes(int64_t R, int64_t N, int64_t K) {
    return up(2 * N * K) + up(bf16_dx_work_bytes(int(R), int(N), int(K)));
}
int64_t split_bytes(int32_t type, int64_t R, int64_t N) {
    return up(R * mx4_split_width(N) * mx4_split_pieces(type) * 2);
}

}  // namespace
}  // namespace xpuint8

using namespace xpuint8;

extern "C" {

int64_t xpuint8_mxfp4_scale_width(int64_t K) {
    if (K <= 0 || K % 32 != 0 || K > kMaxDim) return -1;
    return mx_scale_width(K);
}

int xpuint8_mxfp4_quantize_stream(const void* stream, const void* x, int32_t type, int64_t ldx,
                                  uint8_t* codes, uint8_t* scales, int64_t M, int64_t K) {
    XPU_TRY(check_mx(M, K));
    XPU_TRY(check_type(type, "type"));
    if (ldx < K) return fail(2, "the row stride must be >= K");
    if (!x) return fail(6, "x must not be null");
    XPU_NONNULL(codes); XPU_NONNULL(scales);
    XPU_TRY(ensure_device());
    return launched(mx4_quantize(as_stream(stream), x, type, ldx, codes, scales, M, int(K)),
                    "mxfp4_quantize");
}

int xpuint8_mxfp4_dequantize_stream(const void* stream, const uint8_t* codes,
                                    const uint8_t* scales, void* out, int32_t type, int64_t M,
                                    int64_t K) {
    XPU_TRY(check_mx(M, K));
    XPU_TRY(check_type(type, "type"));
    XPU_NONNULL(codes); XPU_NONNULL(scales); XPU_NONNULL(out);
    XPU_TRY(ensure_device());
    return launched(mx4_dequantize(as_stream(stream), codes, scales, out, type, M, int(K)),
                    "mxfp4_dequantize");
}

int64_t xpuint8_mxfp4_linear_workspace_size(int64_t M, int64_t N, int64_t K) {
    if (check_linear(M, M, N, K, false, 0) != 0) return -1;
    return mx4_fused(M, false, 0, K) ? 0 : quantized_bytes(M, K);
}

int xpuint8_mxfp4_linear_stream(const void* stream, const void* x, int32_t type, int64_t ldx,
                                const uint8_t* codes, const uint8_t* scales, const void* bias,
                                int32_t bias_type, void* y, int64_t M, int64_t N, int64_t K,
                                void* work, int64_t work_bytes) {
    XPU_TRY(check_linear(M, M, N, K, false, 0));
    XPU_TRY(check_type(type, "type"));
    if (bias) XPU_TRY(check_type(bias_type, "bias_type"));
    if (ldx < K) return fail(2, "the row stride must be >= K");
    if (!x) return fail(6, "x must not be null");
    XPU_NONNULL(codes); XPU_NONNULL(scales); XPU_NONNULL(y);
    return product(stream, x, type, ldx, nullptr, M, codes, scales, nullptr, 1, bias, bias_type, y,
                   M, N, K, work, work_bytes, "mxfp4_linear");
}

int64_t xpuint8_mxfp4_grouped_linear_workspace_size(int64_t R, int64_t tokens, int64_t E,
                                                    int64_t N, int64_t K) {
    if (check_linear(R, tokens, N, K, true, E) != 0) return -1;
    return mx4_fused(R, true, int(E), K) ? 0 : quantized_bytes(tokens, K);
}

int xpuint8_mxfp4_grouped_linear_stream(const void* stream, const void* x, int32_t type,
                                        int64_t ldx, const int32_t* rows, int64_t tokens,
                                        const uint8_t* codes, const uint8_t* scales,
                                        const int32_t* offsets, int64_t E, void* y, int64_t R,
                                        int64_t N, int64_t K, void* work, int64_t work_bytes) {
    XPU_TRY(check_linear(R, tokens, N, K, true, E));
    XPU_TRY(check_type(type, "type"));
    if (!rows && tokens != R) return fail(2, "without rows, x must have R rows");
    if (ldx < K) return fail(2, "the row stride must be >= K");
    if (!x) return fail(6, "x must not be null");
    if (!offsets) return fail(6, "offsets must not be null");
    XPU_NONNULL(codes); XPU_NONNULL(scales); XPU_NONNULL(y);
    return product(stream, x, type, ldx, rows, tokens, codes, scales, offsets, E, nullptr, 0, y, R,
                   N, K, work, work_bytes, "mxfp4_grouped_linear");
}

int64_t xpuint8_mxfp4_dx_workspace_size(int32_t type, int32_t dx_type, int64_t R, int64_t E,
                                        int64_t N, int64_t K) {
    if (check_gradient(R, N, K, E > 0, E) != 0 || check_type(type, "type") != 0) return -1;
    if (dx_by_bf16(type, dx_type, E > 0, R, N, K))
        return std::max(bf16_dx_bytes(R, N, K), split_bytes(type, R, N));
    return split_bytes(type, R, N);
}

int64_t xpuint8_mxfp4_dx_workspace_size_of(const void* dy, int32_t type, int64_t ldy, int32_t dx_type,
                                           int64_t R, int64_t E, int64_t N, int64_t K) {
    if (xpuint8_mxfp4_dx_workspace_size(type, dx_type, R, E, N, K) < 0) return -1;
    if (!dy_direct(dy, type, ldy, N)) return split_bytes(type, R, N);
    return ldy == N && dx_by_bf16(type, dx_type, E > 0, R, N, K) ? bf16_dx_bytes(R, N, K) : 0;
}

int xpuint8_mxfp4_dx_stream(const void* stream, const void* dy, int32_t type, int64_t ldy,
                            const uint8_t* codes, const uint8_t* scales, const int32_t* offsets,
                            int64_t E, void* dx, int32_t dx_type, int64_t R, int64_t N, int64_t K,
                            void* work, int64_t work_bytes) {
    XPU_TRY(check_gradient(R, N, K, offsets != nullptr, offsets ? E : 0));
    XPU_TRY(check_type(type, "type"));
    XPU_TRY(check_type(dx_type, "dx_type"));
    if (ldy < N) return fail(2, "the row stride must be >= N");
    if (!dy) return fail(6, "dy must not be null");
    XPU_NONNULL(codes); XPU_NONNULL(scales); XPU_NONNULL(dx);
    const bool grouped = offsets != nullptr;
    const bool direct = dy_direct(dy, type, ldy, N);
    if (dx_by_bf16(type, dx_type, grouped, R, N, K) && direct && ldy == N) {
        XPU_NONNULL(work);
        if (work_bytes < up(2 * N * K))
            return fail(2, "work must hold xpuint8_mxfp4_dx_workspace_size bytes");
        XPU_TRY(ensure_device());
        hipStream_t st = as_stream(stream);
        char* const wd = static_cast<char*>(work);
        XPU_TRY(launched(mx4_dequantize(st, codes, scales, wd, kBf16, N, int(K)), "mxfp4_dx (weight)"));
        return launched(gemm_bf16_nn(st, dy, N, wd, K, dx, K, int(R), int(N), int(K),
                                     reinterpret_cast<float*>(wd + up(2 * N * K)),
                                     work_bytes - up(2 * N * K)), "mxfp4_dx (bf16)");
    }
    if (!direct) {
        XPU_NONNULL(work);
        if (work_bytes < split_bytes(type, R, N))
            return fail(2, "work must hold xpuint8_mxfp4_dx_workspace_size bytes");
    }
    XPU_TRY(ensure_device());
    hipStream_t st = as_stream(stream);
    const int pieces = direct ? 1 : mx4_split_pieces(type);
    if (!direct) {
        XPU_TRY(launched(mx4_split(st, dy, type, ldy, work, R, int(N)), "mxfp4_dx (split)"));
        dy = work;
        ldy = mx4_split_width(N) * pieces;
    }
    return launched(mx4_dx(st, dy, ldy, pieces, codes, scales, offsets, grouped ? int(E) : 1, dx,
                           dx_type, R, int(N), int(K)), "mxfp4_dx");
}

int64_t xpuint8_mxfp4_dbias_workspace_size(int64_t M, int64_t N) {
    if (check_dbias(M, N) != 0) return -1;
    return mx4_dbias_work_bytes(M, N);
}

int xpuint8_mxfp4_dbias_stream(const void* stream, const void* dy, int32_t type, int64_t ldy,
                               void* dbias, int32_t dbias_type, int64_t M, int64_t N, void* work,
                               int64_t work_bytes) {
    XPU_TRY(check_dbias(M, N));
    XPU_TRY(check_type(type, "type"));
    XPU_TRY(check_type(dbias_type, "dbias_type"));
    if (ldy < N) return fail(2, "the row stride must be >= N");
    if (!dy) return fail(6, "dy must not be null");
    XPU_NONNULL(dbias); XPU_NONNULL(work);
    if (work_bytes < mx4_dbias_work_bytes(M, N))
        return fail(2, "work must hold xpuint8_mxfp4_dbias_workspace_size bytes");
    XPU_TRY(ensure_device());
    return launched(mx4_dbias(as_stream(stream), dy, type, ldy, dbias, dbias_type, M, int(N),
                              static_cast<float*>(work)), "mxfp4_dbias");
}

// ------------------------------------------------------------------ experts
int64_t xpuint8_moe_sort_workspace_size(int64_t T, int64_t top, int64_t E) {
    if (check_moe(T, top, E) != 0) return -1;
    return moe_sort_work_bytes(T * top, int(E));
}

int xpuint8_moe_sort_stream(const void* stream, const void* ids, int32_t ids_int64, int32_t* order,
                            int32_t* position, int32_t* rows, int32_t* offsets, int64_t T,
                            int64_t top, int64_t E, void* work, int64_t work_bytes) {
    XPU_TRY(check_moe(T, top, E));
    if (ids_int64 != 0 && ids_int64 != 1) return fail(2, "ids_int64 must be 0 or 1");
    if (!ids || !order || !position || !rows || !offsets)
        return fail(6, "ids, order, position, rows and offsets must not be null");
    const int64_t need = moe_sort_work_bytes(T * top, int(E));
    if (need > 0 && !work) return fail(6, "work must not be null");
    if (work_bytes < need)
        return fail(2, "work must hold xpuint8_moe_sort_workspace_size(T, top, E) bytes");
    XPU_TRY(ensure_device());
    return launched(moe_sort(as_stream(stream), ids, ids_int64 != 0, order, position, rows, offsets,
                             T * top, int(top), int(E), work), "moe_sort");
}

int xpuint8_moe_dispatch_stream(const void* stream, const void* x, int32_t type, int64_t ldx,
                                const int32_t* position, const int32_t* offsets, void* out,
                                int64_t T, int64_t top, int64_t E, int64_t D) {
    XPU_TRY(check_rows_of(T, top, E, D));
    XPU_TRY(check_type(type, "type"));
    if (ldx < D) return fail(2, "the row stride must be >= D");
    if (!x || !position || !offsets || !out)
        return fail(6, "x, position, offsets and out must not be null");
    XPU_TRY(ensure_device());
    return launched(moe_dispatch(as_stream(stream), x, type, ldx, position, offsets, out, T,
                                 int(top), int(E), int(D)), "moe_dispatch");
}

int xpuint8_moe_combine_stream(const void* stream, const void* z, int32_t type, int64_t ldz,
                               const int32_t* position, const int32_t* offsets,
                               const float* weights, void* out, int32_t out_type, int64_t T,
                               int64_t top, int64_t E, int64_t D) {
    XPU_TRY(check_rows_of(T, top, E, D));
    XPU_TRY(check_type(type, "type"));
    XPU_TRY(check_type(out_type, "out_type"));
    if (out_type != type && (type != kF32 || weights))
        return fail(6, "out_type must be type, or type fp32 without weights");
    if (ldz < D) return fail(2, "the row stride must be >= D");
    if (!z || !position || !offsets || !out)
        return fail(6, "z, position, offsets and out must not be null");
    XPU_TRY(ensure_device());
    return launched(moe_gather(as_stream(stream), z, type, ldz, position, offsets, weights, out,
                               out_type, T, int(top), int(E), int(D)), "moe_combine");
}

int xpuint8_moe_combine_grad_stream(const void* stream, const void* dy, int32_t type, int64_t ldy,
                                    const void* z, int64_t ldz, const int32_t* position,
                                    const int32_t* offsets, const float* weights, void* dz,
                                    float* dweights, int64_t T, int64_t top, int64_t E,
                                    int64_t D) {
    XPU_TRY(check_rows_of(T, top, E, D));
    XPU_TRY(check_type(type, "type"));
    if (ldy < D || ldz < D) return fail(2, "the row strides must be >= D");
    if (!dy || !z || !position || !offsets || !weights || !dz || !dweights)
        return fail(6, "dy, z, position, offsets, weights, dz and dweights must not be null");
    XPU_TRY(ensure_device());
    return launched(moe_combine_grad(as_stream(stream), dy, type, ldy, z, ldz, position, offsets,
                                     weights, dz, dweights, T, int(top), int(E), int(D)),
                    "moe_combine_grad");
}

}  // extern "C"
