// The C ABI of the operators between a block's projections (include/xpuint8.h): RMS norm,
// rotary positions, routing.  As in capi.hip, every check runs before any HIP call.
#include <hip/hip_runtime.h>

#include <string>

#include "block_kernels.hpp"
#include "capi.hpp"
#include "mx4.hpp"
#include "../../include/xpuint8.h"

namespace xpuint8 {
namespace {

constexpr int64_t kMaxRow = int64_t(1) << 24;
constexpr int64_t kMaxHeadDim = 4096, kMaxPairs = 512, kMaxHeads = 65536, kMaxAxes = 16;
constexpr int64_t kMaxExperts = 1024, kMaxTop = 64;

int check_type(int32_t type, const char* what) {
    if (type < 0 || type > 2)
        return fail(6, std::string(what) + " must be 0 (bf16), 1 (fp16) or 2 (fp32)");
    return 0;
}
// elements need their own alignment only
int check_aligned(const void* p, int32_t type, const char* what) {
    if (reinterpret_cast<uintptr_t>(p) % (type == kF32 ? 4 : 2) != 0)
        return fail(6, std::string(what) + " must be aligned to its elements");
    return 0;
}

int check_rows(int64_t M, int64_t K) {
    if (M <= 0 || K <= 0) return fail(2, "rows and K must be positive");
    if (M > kMaxDim || K > kMaxRow) return fail(4, "rows must be < 2^31 and K at most 2^24");
    return 0;
}

// M rows in runs of `inner`; rows of a run do not overlap, runs may lie anywhere
int check_inner(int64_t inner, int64_t M) {
    if (inner < 1 || M % inner != 0) return fail(2, "inner must be positive and divide the rows");
    return 0;
}
int check_lines(const void* p, const Lines& l, int64_t inner, int64_t M, int64_t K) {
    if (p && (l.outer < (inner == 1 && M > 1 ? K : 0) || (inner > 1 && l.ld < K)))
        return fail(2, "the row strides must be >= K");
    return 0;
}

int check_norm(const void* x, int32_t type, const Lines& lx, const void* residual, const Lines& lr,
               int64_t inner, const void* weight, int32_t weight_type, float eps, const void* h,
               int64_t M, int64_t K) {
    XPU_TRY(check_rows(M, K));
    XPU_TRY(check_type(type, "type"));
    XPU_TRY(check_inner(inner, M));
    XPU_TRY(check_lines(x, lx, inner, M, K));
    XPU_TRY(check_lines(residual, lr, inner, M, K));
    if (!(eps >= 0.f)) return fail(2, "eps must not be negative");
    if (!x) return fail(6, "x must not be null");
    XPU_TRY(check_aligned(x, type, "x"));
    XPU_TRY(check_aligned(residual, type, "residual"));
    if (!residual != !h) return fail(6, "residual and h belong together");
    XPU_ALIGNED_OPT(h);
    if (weight) {
        XPU_TRY(check_type(weight_type, "weight_type"));
        XPU_TRY(check_aligned(weight, weight_type, "weight"));
    }
    return 0;
}

int check_route(int64_t T, int64_t E, int64_t top, int32_t type, int64_t ld, int32_t sigmoid,
                int32_t renormalize) {
    if (T <= 0 || T > kMaxDim) return fail(2, "tokens must be positive and < 2^31");
    if (E < 1 || E > kMaxExperts) return fail(2, "experts must be 1..1024");
    if (top < 1 || top > kMaxTop || top > E) return fail(2, "top must be 1..64, and at most the experts");
    XPU_TRY(check_type(type, "type"));
    if (ld < E) return fail(2, "the row stride must be >= E");
    if ((sigmoid | renormalize) & ~1) return fail(2, "sigmoid and renormalize must be 0 or 1");
    return 0;
}

}  // namespace
}  // namespace xpuint8

using namespace xpuint8;

extern "C" {

int xpuint8_rms_norm_stream(const void* stream, const void* x, int32_t type, int64_t ldx,
                            int64_t outer_x, const void* residual, int64_t ldr, int64_t outer_r,
                            int64_t inner, const void* weight, int32_t weight_type, float eps,
                            void* h, void* y, int64_t M, int64_t K) {
    const Lines lx{ldx, outer_x}, lr{ldr, outer_r};
    XPU_TRY(check_norm(x, type, lx, residual, lr, inner, weight, weight_type, eps, h, M, K));
    XPU_NONNULL(y);
    XPU_TRY(ensure_device());
    return launched(rms_norm(as_stream(stream), x, type, lx, residual, lr, inner, weight,
                             weight_type, eps, h, y, M, K), "rms_norm");
}

int xpuint8_rms_norm_int8_stream(const void* stream, const void* x, int32_t type, int64_t ldx,
                                 int64_t outer_x, const void* residual, int64_t ldr,
                                 int64_t outer_r, int64_t inner, const void* weight,
                                 int32_t weight_type, float eps, void* h, int8_t* q, float* scale,
                                 int32_t rotate, int64_t M, int64_t K) {
    const Lines lx{ldx, outer_x}, lr{ldr, outer_r};
    XPU_TRY(check_norm(x, type, lx, residual, lr, inner, weight, weight_type, eps, h, M, K));
    if (rotate != 0 && rotate != 1) return fail(2, "rotate must be 0 or 1");
    if (rotate && K % 256 != 0)
        return fail(3, "K must be a multiple of the ConvRot group size (256) to be rotated");
    XPU_NONNULL(q); XPU_NONNULL(scale);
    XPU_TRY(ensure_device());
    return launched(rms_norm_int8(as_stream(stream), x, type, lx, residual, lr, inner, weight,
                                  weight_type, eps, h, q, scale, rotate != 0, M, K),
                    "rms_norm_int8");
}

int64_t xpuint8_rms_norm_grad_workspace_size(int64_t M, int64_t K) {
    if (check_rows(M, K) != 0) return -1;
    return rms_norm_grad_work_bytes(M, K);
}

int xpuint8_rms_norm_grad_stream(const void* stream, const void* dy, int32_t type, int64_t ldy,
                                 int64_t outer_dy, const void* h, int64_t ldh, int64_t outer_h,
                                 const void* weight, int32_t weight_type, const void* dh,
                                 int64_t lddh, int64_t outer_dh, int64_t inner, float eps,
                                 void* dx, void* dweight, int64_t M, int64_t K, void* work,
                                 int64_t work_bytes) {
    XPU_TRY(check_rows(M, K));
    XPU_TRY(check_type(type, "type"));
    const Lines dy_lines{ldy, outer_dy}, h_lines{ldh, outer_h}, dh_lines{lddh, outer_dh};
    XPU_TRY(check_inner(inner, M));
    XPU_TRY(check_lines(dy, dy_lines, inner, M, K));
    XPU_TRY(check_lines(h, h_lines, inner, M, K));
    XPU_TRY(check_lines(dh, dh_lines, inner, M, K));
    if (!(eps >= 0.f)) return fail(2, "eps must not be negative");
    if (!dy || !h) return fail(6, "dy and h must not be null");
    XPU_TRY(check_aligned(dy, type, "dy"));
    XPU_TRY(check_aligned(h, type, "h"));
    XPU_TRY(check_aligned(dh, type, "dh"));
    if (weight) {
        XPU_TRY(check_type(weight_type, "weight_type"));
        XPU_TRY(check_aligned(weight, weight_type, "weight"));
    }
    XPU_NONNULL(dx);
    if (dweight) {
        if (!weight) return fail(6, "dweight needs a weight");
        XPU_NONNULL(dweight); XPU_NONNULL(work);
        if (work_bytes < rms_norm_grad_work_bytes(M, K))
            return fail(2, "work must hold xpuint8_rms_norm_grad_workspace_size bytes");
    }
    XPU_TRY(ensure_device());
    return launched(rms_norm_grad(as_stream(stream), dy, type, dy_lines, h, h_lines, weight,
                                  weight_type, dh, dh_lines, inner, eps, dx, dweight, M, K,
                                  static_cast<float*>(work)),
                    "rms_norm_grad");
}

int xpuint8_rope_axes_stream(const void* stream, const void* q, void* q_out,
                             const int64_t* q_strides, int64_t q_heads, const void* k, void* k_out,
                             const int64_t* k_strides, int64_t k_heads, int32_t type,
                             const void* positions, int32_t position_type,
                             const int64_t* position_strides, int64_t axes,
                             const double* inv_freq, const int32_t* axis, int64_t pairs,
                             int32_t inverse, int32_t split_half, int64_t B, int64_t S, int64_t D) {
    if (B <= 0 || S <= 0 || D <= 0) return fail(2, "B, S and D must be positive");
    if (B > kMaxDim || S > kMaxDim || B * S > kMaxDim) return fail(4, "B x S must be < 2^31");
    if (pairs < 1 || pairs > kMaxPairs || 2 * pairs > D)
        return fail(2, "pairs must be 1..512, and 2 of them a head at most");
    if (D > kMaxHeadDim) return fail(4, "D must be at most 4096");
    if (axes < 1 || axes > kMaxAxes) return fail(2, "axes must be 1..16");
    XPU_TRY(check_type(type, "type"));
    if (position_type < 0 || position_type > 2)
        return fail(6, "position_type must be 0 (int32), 1 (int64) or 2 (fp32)");
    if ((inverse | split_half) & ~1) return fail(2, "inverse and split_half must be 0 or 1");
    if (!q || !q_out || !q_strides || !positions || !position_strides || !inv_freq || !axis)
        return fail(6, "q, q_out, positions, inv_freq, axis and their strides must not be null");
    if (!k != !k_out || (k && !k_strides)) return fail(6, "k, k_out and k_strides belong together");
    if (!k) k_heads = 0;
    if (q_heads < 1 || k_heads < (k ? 1 : 0) || q_heads + k_heads > kMaxHeads)
        return fail(2, "heads must be positive, and 65536 at most");
    XPU_TRY(check_aligned(q, type, "q"));
    XPU_TRY(check_aligned(q_out, type, "q_out"));
    XPU_TRY(check_aligned(k, type, "k"));
    XPU_TRY(check_aligned(k_out, type, "k_out"));
    if (reinterpret_cast<uintptr_t>(positions) % (position_type == 1 ? 8 : 4) != 0 ||
        reinterpret_cast<uintptr_t>(inv_freq) % 8 != 0 || reinterpret_cast<uintptr_t>(axis) % 4 != 0)
        return fail(6, "positions, inv_freq and axis must be aligned to their elements");
    XPU_TRY(ensure_device());
    auto heads = [](const void* x, void* out, const int64_t* s, int64_t H) {
        return x ? Heads{x, out, s[0], s[1], s[2], s[3], s[4], s[5], int(H)} : Heads{};
    };
    const Positions at{positions, position_type, int(axes), position_strides[0],
                       position_strides[1], position_strides[2]};
    return launched(rope_axes(as_stream(stream), heads(q, q_out, q_strides, q_heads),
                              heads(k, k_out, k_strides, k_heads), type, at, inv_freq, axis,
                              int(pairs), inverse != 0, split_half != 0, B, S, int(D)),
                    "rope_axes");
}

int xpuint8_moe_route_stream(const void* stream, const void* logits, int32_t type, int64_t ld,
                             const float* bias, int32_t sigmoid, int64_t groups,
                             int64_t top_groups, int32_t renormalize, float scale, int32_t* ids,
                             float* weights, int64_t T, int64_t E, int64_t top) {
    XPU_TRY(check_route(T, E, top, type, ld, sigmoid, renormalize));
    if (groups < 1 || groups > 64 || E % groups != 0)
        return fail(2, "groups must be 1..64 and divide the experts");
    if (top_groups < 1 || top_groups > groups || top > top_groups * (E / groups))
        return fail(2, "top_groups must be 1..groups, and hold top experts");
    if (!logits || !ids || !weights) return fail(6, "logits, ids and weights must not be null");
    XPU_TRY(check_aligned(logits, type, "logits"));
    XPU_TRY(check_aligned(bias, kF32, "bias"));
    XPU_TRY(check_aligned(ids, kF32, "ids"));
    XPU_TRY(check_aligned(weights, kF32, "weights"));
    XPU_TRY(ensure_device());
    const RouteHow how{sigmoid != 0, renormalize != 0, int(groups), int(top_groups), scale};
    return launched(moe_route(as_stream(stream), logits, type, ld, bias, how, ids, weights, T,
                              int(E), int(top)), "moe_route");
}

int xpuint8_moe_route_grad_stream(const void* stream, const void* logits, int32_t type, int64_t ld,
                                  const int32_t* ids, const float* dweights, int32_t sigmoid,
                                  int32_t renormalize, float scale, void* dlogits, int64_t T,
                                  int64_t E, int64_t top) {
    XPU_TRY(check_route(T, E, top, type, ld, sigmoid, renormalize));
    if (!logits || !ids || !dweights || !dlogits)
        return fail(6, "logits, ids, dweights and dlogits must not be null");
    XPU_TRY(check_aligned(logits, type, "logits"));
    XPU_TRY(check_aligned(dlogits, type, "dlogits"));
    XPU_TRY(check_aligned(ids, kF32, "ids"));
    XPU_TRY(check_aligned(dweights, kF32, "dweights"));
    XPU_TRY(ensure_device());
    const RouteHow how{sigmoid != 0, renormalize != 0, 1, 1, scale};
    return launched(moe_route_grad(as_stream(stream), logits, type, ld, ids, dweights, how, dlogits,
                                   T, int(E), int(top)), "moe_route_grad");
}

}  // extern "C"
