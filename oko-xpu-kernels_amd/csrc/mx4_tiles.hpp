// What the MXFP4 products' tile kernels share: LDS reads and waits, the accumulators,
// the order of the tiles and the way out.
#pragma once

#include "mx4_groups.hpp"

namespace xpuint8 {
namespace {

__device__ __forceinline__ v4i read16(uint32_t addr, int off) {
    v4i r;
    asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(r) : "v"(addr), "n"(off));
    return r;
}
__device__ __forceinline__ int read4(uint32_t addr, int off) {
    int r;
    asm volatile("ds_read_b32 %0, %1 offset:%2" : "=v"(r) : "v"(addr), "n"(off));
    return r;
}
template <int N>
__device__ __forceinline__ void wait_vm() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// a wave-uniform address that stays one: with it and a lane's 32-bit offset apart, a
// load takes both as they are, where the compiler would keep their sums in registers
__device__ __forceinline__ const uint8_t* scalar(const uint8_t* p) {
    asm volatile("" : "+s"(p));
    return p;
}
// what inline reads have written, once the wait for them is done: no use of it can be
// scheduled above this
template <class V, int N>
__device__ __forceinline__ void landed(V (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+v"(f[i]));
}
template <int N, int I = 0, class F>
__device__ __forceinline__ void each(const F& f) {
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        each<N, I + 1>(f);
    }
}
// this wave's LDS accesses are done
__device__ __forceinline__ void lds_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
// a barrier that nothing is scheduled across; the waits before it are the caller's
__device__ __forceinline__ void block_barrier() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
}

// The accumulators of a tile live in the accumulation registers a0 up, named in the
// instructions: 4 registers an MFMA block, COUNT in all.  As values they were copied
// at every turn of the loop or spilled (compilers move an MFMA builtin over barriers,
// and its accumulator with it).  Every statement on them clobbers all of them, the reads at
// the end too, so that nothing else is kept there until the last one is read.  The compiler neither sees these MFMAs nor places the
// waits that they need: two wait states between a VALU write and an MFMA that reads it
// (each statement of MFMAs begins with them, XPU_MFMA_WAIT: what the compiler put right
// before it is not known), eighteen between an MFMA and a read of its result by anything
// but an MFMA on it (store_tile).
#define XPU_MFMA_WAIT "s_nop 1\n\t"
#define XPU_A10(p) "a" #p "0", "a" #p "1", "a" #p "2", "a" #p "3", "a" #p "4", "a" #p "5", \
                   "a" #p "6", "a" #p "7", "a" #p "8", "a" #p "9"
#define XPU_A60 XPU_A10(), XPU_A10(1), XPU_A10(2), XPU_A10(3), XPU_A10(4), XPU_A10(5)
#define XPU_A64 XPU_A60, "a60", "a61", "a62", "a63"
#define XPU_A120 XPU_A60, XPU_A10(6), XPU_A10(7), XPU_A10(8), XPU_A10(9), XPU_A10(10), XPU_A10(11)
#define XPU_A256 XPU_A120, XPU_A10(12), XPU_A10(13), XPU_A10(14), XPU_A10(15), XPU_A10(16),     \
                 XPU_A10(17), XPU_A10(18), XPU_A10(19), XPU_A10(20), XPU_A10(21), XPU_A10(22),  \
                 XPU_A10(23), XPU_A10(24), "a250", "a251", "a252", "a253", "a254", "a255"
// the four registers of block BLOCK = v
#define XPU_ACC_SET(CLOBBERS)                                                                   \
    asm volatile("v_accvgpr_write_b32 a[%4], %0\n\tv_accvgpr_write_b32 a[%5], %1\n\t"           \
                 "v_accvgpr_write_b32 a[%6], %2\n\tv_accvgpr_write_b32 a[%7], %3"               \
                 ::"v"(v[0]), "v"(v[1]), "v"(v[2]), "v"(v[3]), "n"(4 * BLOCK),                  \
                 "n"(4 * BLOCK + 1), "n"(4 * BLOCK + 2), "n"(4 * BLOCK + 3)                     \
                 : CLOBBERS)
template <int COUNT, int BLOCK>
__device__ __forceinline__ void acc_set(const v4f& v) {
    if constexpr (COUNT == 64) XPU_ACC_SET(XPU_A64);
    else XPU_ACC_SET(XPU_A256);
}
#define XPU_ACC_GET(CLOBBERS)                                                                   \
    asm volatile("v_accvgpr_read_b32 %0, a[%4]\n\tv_accvgpr_read_b32 %1, a[%5]\n\t"             \
                 "v_accvgpr_read_b32 %2, a[%6]\n\tv_accvgpr_read_b32 %3, a[%7]"                 \
                 : "=v"(a), "=v"(b), "=v"(c), "=v"(d)                                           \
                 : "n"(4 * BLOCK), "n"(4 * BLOCK + 1), "n"(4 * BLOCK + 2), "n"(4 * BLOCK + 3)   \
                 : CLOBBERS)
template <int COUNT, int BLOCK>
__device__ __forceinline__ v4f acc_get() {
    float a, b, c, d;
    if constexpr (COUNT == 64) XPU_ACC_GET(XPU_A64);
    else XPU_ACC_GET(XPU_A256);
    return v4f{a, b, c, d};
}
// zeros in the rows of a tile
template <int BM, int BN>
__device__ __forceinline__ void zero_rows(const Out& o, int type, const RowTile& t, int n0) {
    const v4f zero = {0.f, 0.f, 0.f, 0.f};
    for (int i = threadIdx.x; i < BM * (BN / 4); i += blockDim.x) {
        const int row = t.row + i / (BN / 4), n = n0 + 4 * (i % (BN / 4));
        if (row >= t.end) continue;
        if (type == kBf16) store4<kBf16>(o, row, n, zero);
        else if (type == kF16) store4<kF16>(o, row, n, zero);
        else store4<kF32>(o, row, n, zero);
    }
}

// One row of COUNT MFMA blocks' results in a 16-bit type, columns n .. n + 16 COUNT (all
// in the row, 16-byte aligned): lane group g holds the columns 16a + 4g .. + 3 of block a,
// value(a), and stores 16 bytes: the swap of two blocks' odd and even lane rows
// (v_permlane16_swap) leaves lane groups 0 and 2 with the columns 0-7 and 8-15 of the
// one block, 1 and 3 with the other's.  `live`: whether this lane's row is one to write.
template <int T, int COUNT, class V>
__device__ __forceinline__ void store_row(const Out& o, int64_t row, bool live, int n, const V& value) {
    const int g = (threadIdx.x & 63) >> 4;
    char* const p = o.y + (row * o.N + n + 16 * (g & 1) + 8 * (g >> 1)) * 2;
    each<COUNT / 2>([&](auto A) {
        constexpr int a = 2 * decltype(A)::value;
        const v4f u = value(std::integral_constant<int, a>{});
        const v4f v = value(std::integral_constant<int, a + 1>{});
        const auto lo = __builtin_amdgcn_permlane16_swap(pack2<T>(u[0], u[1]), pack2<T>(v[0], v[1]), false, false);
        const auto hi = __builtin_amdgcn_permlane16_swap(pack2<T>(u[2], u[3]), pack2<T>(v[2], v[3]), false, false);
        if (live) *reinterpret_cast<uint4*>(p + 32 * a) = make_uint4(lo[0], hi[0], lo[1], hi[1]);
    });
}

// Tile (tm, tn) of block b.  Blocks go round the 8 XCDs, each with its own L2, so an
// XCD takes a contiguous eighth of the tiles, walked in bands of 8 row tiles: the
// blocks of an XCD that run together share few rows of either operand.
__device__ __forceinline__ bool tile_of(int b, int tiles_m, int tiles_n, int& tm, int& tn) {
    const int tiles = tiles_m * tiles_n, share = (tiles + 7) / 8;
    const int t = (b % 8) * share + b / 8;
    if (t >= tiles) return false;
    const int band = t / (8 * tiles_n), first = band * 8;
    const int rows = min(tiles_m - first, 8), in = t - band * 8 * tiles_n;
    tm = first + in % rows;
    tn = in / rows;
    return true;
}

// The results of a wave's TM x TN blocks (block (a, b) in registers 4 (a TM + b) up, b's
// rows row0 + STEP b up) to the rows below end and the columns n up.  `mine`: 16 x 16 TN fp32 of idle LDS
// of the wave's own, through which types and edges go that 16-byte stores do not serve.
template <int TM, int TN, int STEP = 32>
__device__ __forceinline__ void store_tile(const Out& out, int type, int row0, int end, int n,
                                           float* mine) {
    const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
    constexpr int ACC = TM * TN > 16 ? 256 : 64;
    // the last MFMAs' results before they are read
    asm volatile("s_nop 15\n\ts_nop 15");
    auto store = [&](auto T) {
        each<TM>([&](auto B) {
            constexpr int b = decltype(B)::value;
            const int row = row0 + STEP * b + r;
            store_row<decltype(T)::value, TN>(out, row, row < end, n, [&](auto A) {
                return acc_get<ACC, decltype(A)::value * TM + b>();
            });
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    const bool fast = out.vec8 && n + 16 * TN <= out.N;
    if (fast && type == kBf16) return store(std::integral_constant<int, kBf16>{});
    if (fast && type == kF16) return store(std::integral_constant<int, kF16>{});
    each<TM>([&](auto B) {
        constexpr int b = decltype(B)::value;
        each<TN>([&](auto A) {
            constexpr int a = decltype(A)::value;
            *reinterpret_cast<v4f*>(mine + r * (16 * TN) + 16 * a + 4 * g) = acc_get<ACC, a * TM + b>();
        });
        lds_done();
#pragma clang loop unroll(disable)
        for (int i = lane; i < 16 * (4 * TN); i += 64) {
            const int rr = i / (4 * TN), c = 4 * (i % (4 * TN));
            const int row = row0 + STEP * b + rr;
            const v4f v = *reinterpret_cast<const v4f*>(mine + rr * (16 * TN) + c);
            if (row >= end) continue;
            if (type == kBf16) store4<kBf16>(out, row, n + c, v);
            else if (type == kF16) store4<kF16>(out, row, n + c, v);
            else store4<kF32>(out, row, n + c, v);
        }
        lds_done();
    });
}

}  // namespace
}  // namespace xpuint8
