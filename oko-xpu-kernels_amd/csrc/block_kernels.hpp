// Internal launchers of the operators between a block's projections: RMS norm
// (norm.hip), rotary positions (rotary.hip) and routing to experts (route.hip).  All are
// asynchronous on the given stream, validate nothing (the C ABI in capi_block.hip
// does), and return the launch status.  `type` is an MxType; strides are in elements.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace xpuint8 {

// norm.hip.  An input's rows lie in runs of `inner` (which divides M): ld apart in a run, runs
// outer apart (inner 1: rows outer apart).
struct Lines {
    int64_t ld, outer;
};
// x [M, K] plus residual (null: none; h then too) is h, y = h / rms(h) * weight (null: ones)
hipError_t rms_norm(hipStream_t st, const void* x, int type, const Lines& lx,
                    const void* residual, const Lines& lr, int64_t inner, const void* weight,
                    int weight_type, float eps, void* h, void* y, int64_t M, int64_t K);
// the same with int8 codes and a scale a row for y, rotated by 256s or not
hipError_t rms_norm_int8(hipStream_t st, const void* x, int type, const Lines& lx,
                         const void* residual, const Lines& lr, int64_t inner,
                         const void* weight, int weight_type, float eps, void* h, int8_t* q,
                         float* scale, bool rotate, int64_t M, int64_t K);
// dx [M, K] from dy and (null: none) dh, the gradients of y and h; dweight [K] of
// weight_type (null: not wanted) through part (rms_norm_grad_work_bytes)
int64_t rms_norm_grad_work_bytes(int64_t M, int64_t K);
hipError_t rms_norm_grad(hipStream_t st, const void* dy, int type, const Lines& ldy,
                         const void* h, const Lines& lh, const void* weight, int weight_type,
                         const void* dh, const Lines& ldh, int64_t inner, float eps, void* dx,
                         void* dweight, int64_t M, int64_t K, float* part);

// rotary.hip.  One tensor of heads [B, S, H, D] and its result.
struct Heads {
    const void* x;
    void* out;
    int64_t x_b, x_s, x_h, o_b, o_s, o_h;       // strides; the head dimension's are 1
    int H;
};
// the positions [axes, B, S]: 0 int32, 1 int64, 2 fp32
struct Positions {
    const void* p;
    int type, axes;
    int64_t a, b, s;
};
hipError_t rope_axes(hipStream_t st, const Heads& q, const Heads& k, int type,
                     const Positions& positions, const double* inv_freq, const int* axis, int P,
                     bool inverse, bool split_half, int64_t B, int64_t S, int D);

// route.hip.  ids and weights [T, top] of logits [T, E].
struct RouteHow {
    bool sigmoid, renormalize;
    int groups, top_groups;
    float scale;
};
hipError_t moe_route(hipStream_t st, const void* logits, int type, int64_t ld, const float* bias,
                     const RouteHow& how, int* ids, float* weights, int64_t T, int E, int top);
hipError_t moe_route_grad(hipStream_t st, const void* logits, int type, int64_t ld, const int* ids,
                          const float* dweights, const RouteHow& how, void* dlogits, int64_t T,
                          int E, int top);

}  // namespace xpuint8
