// Internal launchers of the MXFP4 and mixture-of-experts kernels.  All are
// asynchronous on the given stream, validate nothing (the C ABI in capi_mx.hip does),
// and return the launch status.  `type` is an MxType.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace xpuint8 {

// the blocks of 256 threads that one dimension of a launch can have (fewer than 2^32 threads)
constexpr int64_t kMaxBlocks = (int64_t(1) << 24) - 1;
// f(first, count) for n items in as few launches as there must be, `most` of them in one
template <class F>
void in_launches(int64_t n, int64_t most, const F& f) {
    for (int64_t at = 0; at < n; at += most) f(at, n - at < most ? n - at : most);
}

// mx4_quant.hip: x [M, K] (row stride ldx) to codes and scales, and back
hipError_t mx4_quantize(hipStream_t st, const void* x, int type, int64_t ldx, uint8_t* codes,
                        uint8_t* scales, int64_t M, int K);
hipError_t mx4_dequantize(hipStream_t st, const uint8_t* codes, const uint8_t* scales, void* out,
                          int type, int64_t M, int K);

// mx4_gemm.hip: y [R, N] = xq[rows] wq^T [+ bias] over the groups of offsets [E + 1]
// (null: one group of all R rows); rows (null: row i is x's row i) indexes the
// `tokens` rows of x.  mx4_product_fused quantizes x itself (mx4_fused says when).
bool mx4_fused(int64_t R, bool grouped, int E, int64_t K);
hipError_t mx4_product_fused(hipStream_t st, const void* x, int type, int64_t ldx,
                             const int* rows, int64_t tokens, const uint8_t* wc,
                             const uint8_t* ws, const int* offsets, int E, void* y,
                             const void* bias, int bias_type, int64_t R, int N, int K);
// (the blocks of mx4_product's launch, which mx4_blocks_fit must hold of)
int64_t mx4_product_blocks(bool grouped, int64_t R, int E, int64_t N, int64_t K);
inline bool mx4_blocks_fit(int64_t blocks) { return blocks <= kMaxBlocks; }
hipError_t mx4_product(hipStream_t st, const uint8_t* xc, const uint8_t* xs, const int* rows,
                       int64_t tokens, const uint8_t* wc, const uint8_t* ws, const int* offsets,
                       int E, void* y, int type, const void* bias, int bias_type, int64_t R, int N,
                       int K);

// mx4_dx.hip: dx [R, K] = dy [R, N] wq over the same groups, dy bf16 of row stride
// ldy (16-byte aligned rows, N % 8 == 0), or `pieces` bf16 pieces of it side by side
// (mx4_split), each mx4_split_width(N) wide
int64_t mx4_split_width(int64_t N);
int mx4_split_pieces(int type);
hipError_t mx4_split(hipStream_t st, const void* dy, int type, int64_t ldy, void* out, int64_t R,
                     int N);
// whether the weight read back and a bf16 product are faster than mx4_dx (one weight, bf16)
bool mx4_dx_bf16_faster(int64_t R, int64_t N, int64_t K);
int64_t mx4_dx_blocks(bool grouped, int64_t R, int E, int64_t N, int64_t K);
hipError_t mx4_dx(hipStream_t st, const void* dy, int64_t ldy, int pieces, const uint8_t* wc,
                  const uint8_t* ws, const int* offsets, int E, void* dx, int type, int64_t R,
                  int N, int K);

// mx4_bias.hip: out [N] = dy's column sums, dy [M, N] of row stride ldy, through part
// (mx4_dbias_work_bytes)
int64_t mx4_dbias_work_bytes(int64_t M, int64_t N);
hipError_t mx4_dbias(hipStream_t st, const void* dy, int type, int64_t ldy, void* out, int out_type,
                     int64_t M, int N, float* part);

// moe.hip: slots sorted by expert, rows out to them and back, gradients
int64_t moe_sort_work_bytes(int64_t S, int E);
hipError_t moe_sort(hipStream_t st, const void* ids, bool wide, int* order, int* position,
                    int* rows, int* offsets, int64_t S, int top, int E, void* work);
hipError_t moe_dispatch(hipStream_t st, const void* x, int type, int64_t ldx, const int* position,
                        const int* offsets, void* out, int64_t tokens, int top, int E, int D);
// out [tokens, D] of out_type; weights may be null (ones)
hipError_t moe_gather(hipStream_t st, const void* z, int type, int64_t ldz, const int* position,
                      const int* offsets, const float* weights, void* out, int out_type,
                      int64_t tokens, int top, int E, int D);
hipError_t moe_combine_grad(hipStream_t st, const void* dy, int type, int64_t ldy, const void* z,
                            int64_t ldz, const int* position, const int* offsets,
                            const float* weights, void* dz, float* dweights, int64_t tokens,
                            int top, int E, int D);

}  // namespace xpuint8
