// Tokens sorted by expert and back, and the gradients: the two ends of a
// mixture-of-experts layer.
//
// A token t has `top` slots s = t * top + j, each with an expert's index or, for a
// slot that no expert takes, any number outside [0, E).  Sorting is stable by
// (expert, slot), the slots without an expert last, so every result is the same
// from call to call: order[i] is the slot of row i, position[s] its inverse,
// rows[i] = order[i] / top the token of row i, offsets[e] .. offsets[e + 1] the
// rows of expert e; rows from offsets[E] on belong to no expert.
#include <algorithm>

#include "mx4.hpp"
#include "mx_kernels.hpp"

namespace xpuint8 {
namespace {

// ------------------------------------------------------------------- sort
// A counting sort: a block of 16 waves takes kSortChunk consecutive slots, a wave
// a run of them, 64 at a time in order.  The lanes of one key are found with one
// ballot per bit of the key (no atomics, so ranks do not depend on timing); the
// first of them adds their number to the wave's counter of that key.  With the
// counters of every wave before it, and those of every block before, a wave
// knows where its first slot of each key goes, and the second pass hands out the
// places.  A batch of up to kSortChunk slots is one launch of one block; more
// slots take a launch of the counts first.  Latency bound: 8 K slots in 64
// experts 9 us, 64 K 13 us (MI355X).
constexpr int kSortWaves = 16;
constexpr int kSortThreads = kSortWaves * 64;
constexpr int kSortChunk = 8192;
constexpr int kMaxExperts = 1024;

template <class I>
__device__ __forceinline__ int key_of(const I* ids, int64_t s, int E) {
    const I v = ids[s];
    return v >= 0 && v < I(E) ? int(v) : E;
}

// the lanes of the wave whose key equals this lane's, among the lanes of `live`
__device__ __forceinline__ uint64_t peers(int key, int bits, uint64_t live) {
    uint64_t m = live;
    for (int b = 0; b < bits; ++b) {
        const bool one = (key >> b) & 1;
        const uint64_t set = __builtin_amdgcn_ballot_w64(one);
        m &= one ? set : ~set;
    }
    return m;
}

// Counts of each key in each wave's run of the block's chunk, in LDS
// count[wave * (E + 1) + key] (cleared here).
template <class I>
__device__ __forceinline__ void count_keys(const I* ids, int64_t first, int64_t last, int per_wave,
                                           int E, int bits, int* count) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int i = threadIdx.x; i < kSortWaves * (E + 1); i += kSortThreads) count[i] = 0;
    __syncthreads();
    int* mine = count + wave * (E + 1);
    const int64_t lo = first + int64_t(wave) * per_wave, hi = min(lo + per_wave, last);
    for (int64_t s0 = lo; s0 < hi; s0 += 64) {
        const int64_t s = s0 + lane;
        const bool in = s < hi;
        const int key = in ? key_of(ids, s, E) : 0;
        const uint64_t m = peers(key, bits, __builtin_amdgcn_ballot_w64(in));
        if (in && __builtin_ctzll(m) == lane) mine[key] += __builtin_popcountll(m);
    }
    __syncthreads();
}

template <class I>
__global__ __launch_bounds__(kSortThreads) void moe_count_kernel(const I* __restrict__ ids,
                                                                 int* __restrict__ counts,
                                                                 int64_t S, int E, int bits) {
    __shared__ int count[kSortWaves * (kMaxExperts + 1)];
    const int64_t first = int64_t(blockIdx.x) * kSortChunk;
    count_keys(ids, first, min(first + kSortChunk, S), kSortChunk / kSortWaves, E, bits, count);
    for (int k = threadIdx.x; k <= E; k += kSortThreads) {
        int n = 0;
        for (int w = 0; w < kSortWaves; ++w) n += count[w * (E + 1) + k];
        counts[int64_t(blockIdx.x) * (E + 1) + k] = n;
    }
}

// counts: the keys' numbers in each of the nb chunks (unused where nb == 1)
template <class I>
__global__ __launch_bounds__(kSortThreads) void moe_sort_kernel(
    const I* __restrict__ ids, const int* __restrict__ counts, int* __restrict__ order,
    int* __restrict__ position, int* __restrict__ rows, int* __restrict__ offsets, int64_t S,
    int top, int E, int bits, int nb, int per_wave) {
    __shared__ int count[kSortWaves * (kMaxExperts + 1)];
    __shared__ int total[kSortThreads + 64];                // (E + 1 <= kSortThreads + 1)
    __shared__ int wave_sum[kSortWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t first = int64_t(blockIdx.x) * kSortChunk;
    const int64_t last = min(first + kSortChunk, S);
    count_keys(ids, first, last, per_wave, E, bits, count);
    // per key: its number in the blocks before (left in `before`) and in all
    int before = 0, all = 0;
    const int k = threadIdx.x;
    if (k < E) {
        if (nb == 1) {
            for (int w = 0; w < kSortWaves; ++w) all += count[w * (E + 1) + k];
        } else {
            for (int b = 0; b < nb; ++b) {
                const int n = counts[int64_t(b) * (E + 1) + k];
                if (b < int(blockIdx.x)) before += n;
                all += n;
            }
        }
    }
    // exclusive scan of the numbers over the keys 0 .. E - 1
    int incl = all;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int n = __shfl_up(incl, d);
        if (lane >= d) incl += n;
    }
    if (lane == 63) wave_sum[wave] = incl;
    __syncthreads();
    int base = incl - all;
    for (int w = 0; w < wave; ++w) base += wave_sum[w];
    if (k < E) total[k] = base + before;
    if (blockIdx.x == 0 && k < E) {
        offsets[k] = base;
        if (k == E - 1) offsets[E] = base + all;
    }
    // the slots without an expert follow all others, in slot order: those before
    // this block are its first slot less the slots with an expert before it
    if (k == 0) {
        int live = 0, live_before = 0;
        for (int w = 0; w < kSortWaves; ++w) live += wave_sum[w];
        if (nb > 1) {
            for (int b = 0; b < int(blockIdx.x); ++b) live_before += counts[int64_t(b) * (E + 1) + E];
        }
        total[E] = live + live_before;
    }
    __syncthreads();
    // each wave's first place of each key, in place of its count
    for (int kk = threadIdx.x; kk <= E; kk += kSortThreads) {
        int at = total[kk];
        for (int w = 0; w < kSortWaves; ++w) {
            const int n = count[w * (E + 1) + kk];
            count[w * (E + 1) + kk] = at;
            at += n;
        }
    }
    __syncthreads();
    int* mine = count + wave * (E + 1);
    const int64_t lo = first + int64_t(wave) * per_wave, hi = min(lo + per_wave, last);
    for (int64_t s0 = lo; s0 < hi; s0 += 64) {
        const int64_t s = s0 + lane;
        const bool in = s < hi;
        const int key = in ? key_of(ids, s, E) : 0;
        const uint64_t m = peers(key, bits, __builtin_amdgcn_ballot_w64(in));
        if (in) {
            const int at = mine[key] + __builtin_popcountll(m & ((uint64_t(1) << lane) - 1));
            order[at] = int(s);
            position[s] = at;
            rows[at] = int(s) / top;
        }
        // every lane has its place before the counter moves on (the wave's LDS
        // accesses are in order)
        __builtin_amdgcn_wave_barrier();
        if (in && __builtin_ctzll(m) == lane) mine[key] += __builtin_popcountll(m);
        __builtin_amdgcn_wave_barrier();
    }
}

template <class I>
hipError_t sort_launch(hipStream_t st, const I* ids, int* counts, int* order, int* position,
                       int* rows, int* offsets, int64_t S, int top, int E) {
    int bits = 1;
    while ((1 << bits) < E + 1) ++bits;
    const int nb = int((S + kSortChunk - 1) / kSortChunk);
    int per_wave = kSortChunk / kSortWaves;
    if (nb == 1) per_wave = int((S + kSortThreads - 1) / kSortThreads) * 64;
    if (nb > 1)
        hipLaunchKernelGGL((moe_count_kernel<I>), dim3(unsigned(nb)), dim3(kSortThreads), 0, st,
                           ids, counts, S, E, bits);
    hipLaunchKernelGGL((moe_sort_kernel<I>), dim3(unsigned(nb)), dim3(kSortThreads), 0, st, ids,
                       counts, order, position, rows, offsets, S, top, E, bits, nb, per_wave);
    return hipGetLastError();
}

// ------------------------------------------------------- rows out and back
// All four are bound by HBM: each row of either side is read or written once.
// They go by tokens, not by rows: a token's own row is read (or its sum kept in
// registers) once for all its slots, and the row of slot j is at position[t, j];
// positions are every row exactly once, so every row is written, zeros where no
// expert has it (position >= offsets[E]).  A wave takes 64 x 8 x U consecutive
// elements of one token; position values are clamped to the S rows that exist.
template <int T>
constexpr int kSize = T == kF32 ? 4 : 2;

struct Piece {
    int64_t t;
    int d;            // first element of this lane's first 8
};
// piece p of `pieces` a token; U chunks of 512 elements a piece
template <int U>
__device__ __forceinline__ bool piece_of(int64_t T, int pieces, Piece& p) {
    const int64_t w = int64_t(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
    p.t = w / pieces;
    p.d = int(w - p.t * pieces) * (512 * U) + int(threadIdx.x & 63) * 8;
    return p.t < T;
}

// A row's 8 elements at d, of which those past D are left alone (the vector form is
// taken for rows of whole, aligned 8s only)
template <int T, bool VEC>
__device__ __forceinline__ void load_row8(const char* row, int d, int D, float (&v)[8]) {
    if constexpr (VEC) {
        load8<T, true>(row + int64_t(d) * kSize<T>, v);
    } else if (d + 8 <= D) {
        load8<T, false>(row + int64_t(d) * kSize<T>, v);
    } else {
        for (int i = 0; i < 8; ++i) {
            v[i] = 0.f;
            if (d + i >= D) continue;
            if constexpr (T == kF32) v[i] = reinterpret_cast<const float*>(row)[d + i];
            else if constexpr (T == kBf16) v[i] = bf16_to_f32(reinterpret_cast<const uint16_t*>(row)[d + i]);
            else v[i] = float(reinterpret_cast<const _Float16*>(row)[d + i]);
        }
    }
}
template <int T, bool VEC>
__device__ __forceinline__ void store_row8(char* row, int d, int D, const float (&v)[8]) {
    if constexpr (VEC) {
        store8<T, true>(row + int64_t(d) * kSize<T>, v);
    } else if (d + 8 <= D) {
        store8<T, false>(row + int64_t(d) * kSize<T>, v);
    } else {
        for (int i = 0; i < 8; ++i) {
            if (d + i >= D) continue;
            if constexpr (T == kF32) reinterpret_cast<float*>(row)[d + i] = v[i];
            else if constexpr (T == kBf16) reinterpret_cast<uint16_t*>(row)[d + i] = uint16_t(f32_to_bf16_bits(v[i]));
            else reinterpret_cast<_Float16*>(row)[d + i] = _Float16(v[i]);
        }
    }
}

// out[position[t, j]] = x[t], or zeros (the element's bits pass through fp32
// unchanged: every conversion back is of a value of the type)
template <int T, bool VEC, int U>
__global__ __launch_bounds__(256) void moe_dispatch_kernel(const char* __restrict__ x, int64_t ldx,
                                                           const int* __restrict__ position,
                                                           const int* __restrict__ offsets,
                                                           char* __restrict__ out, int64_t tokens,
                                                           int top, int E, int D, int pieces) {
    Piece p;
    if (!piece_of<U>(tokens, pieces, p)) return;
    const int S1 = int(tokens * top - 1);
    const int live = offsets[E];
    float v[U][8];
    const char* src = x + p.t * ldx * kSize<T>;
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (p.d + 512 * u < D) load_row8<T, VEC>(src, p.d + 512 * u, D, v[u]);
    const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int j = 0; j < top; ++j) {
        const int at = min(max(position[p.t * top + j], 0), S1);
        char* dst = out + int64_t(at) * D * kSize<T>;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (p.d + 512 * u < D) {
                if (at < live) store_row8<T, VEC>(dst, p.d + 512 * u, D, v[u]);
                else store_row8<T, VEC>(dst, p.d + 512 * u, D, zero);
            }
    }
}

// out[t] = sum over the slots that an expert has, in slot order, of
// [weights[t, j] *] rows[position[t, j]], in fp32, rounded once
template <int T, int TO, bool VEC, int U, bool WEIGHTED>
__global__ __launch_bounds__(256) void moe_gather_kernel(const char* __restrict__ z, int64_t ldz,
                                                         const int* __restrict__ position,
                                                         const int* __restrict__ offsets,
                                                         const float* __restrict__ weights,
                                                         char* __restrict__ out, int64_t tokens,
                                                         int top, int E, int D, int pieces) {
    Piece p;
    if (!piece_of<U>(tokens, pieces, p)) return;
    const int live = min(offsets[E], int(tokens * top));
    float acc[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[u][i] = 0.f;
#pragma unroll 4
    for (int j = 0; j < top; ++j) {
        const int at = position[p.t * top + j];
        if (at < 0 || at >= live) continue;
        const float w = WEIGHTED ? weights[p.t * top + j] : 1.f;
        const char* src = z + int64_t(at) * ldz * kSize<T>;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (p.d + 512 * u < D) {
                float v[8];
                load_row8<T, VEC>(src, p.d + 512 * u, D, v);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    acc[u][i] = WEIGHTED ? __builtin_fmaf(w, v[i], acc[u][i]) : acc[u][i] + v[i];
            }
    }
    char* dst = out + p.t * D * kSize<TO>;
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (p.d + 512 * u < D) store_row8<TO, VEC>(dst, p.d + 512 * u, D, acc[u]);
}

__device__ __forceinline__ float lanes_sum(float x) {
    x += dpp<kDppXor1>(x);
    x += dpp<kDppXor2>(x);
    x += dpp<kDppXor7>(x);
    x += dpp<kDppXor15>(x);
    x += swz_xor<16>(x);
    x += __shfl_xor(x, 32);
    return x;
}

// the gradients of the weighted sum: dz[position[t, j]] = weights[t, j] * dy[t]
// (zeros where no expert has the row), dweights[t, j] = <dy[t], z[position[t, j]]>
// (0 there), one wave a token: dy's row is read from HBM once and from the cache
// for the slots after the first
template <int T, bool VEC>
__global__ __launch_bounds__(256) void moe_combine_grad_kernel(
    const char* __restrict__ dy, int64_t ldy, const char* __restrict__ z, int64_t ldz,
    const int* __restrict__ position, const int* __restrict__ offsets,
    const float* __restrict__ weights, char* __restrict__ dz, float* __restrict__ dweights,
    int64_t tokens, int top, int E, int D) {
    const int64_t t = int64_t(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
    if (t >= tokens) return;
    const int lane = threadIdx.x & 63;
    const int S = int(tokens * top);
    const int live = min(offsets[E], S);
    const char* g = dy + t * ldy * kSize<T>;
    for (int j = 0; j < top; ++j) {
        const int at = min(max(position[t * top + j], 0), S - 1);
        const bool has = at < live;
        const float w = has ? weights[t * top + j] : 0.f;
        const char* src = z + int64_t(at) * ldz * kSize<T>;
        char* dst = dz + int64_t(at) * D * kSize<T>;
        float dot = 0.f;
#pragma unroll 4
        for (int d = lane * 8; d < D; d += 512) {
            float a[8], b[8];
            if (has) {
                load_row8<T, VEC>(g, d, D, a);
                load_row8<T, VEC>(src, d, D, b);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                dot = has ? __builtin_fmaf(a[i], b[i], dot) : 0.f;
                a[i] = has ? w * a[i] : 0.f;
            }
            store_row8<T, VEC>(dst, d, D, a);
        }
        dot = lanes_sum(dot);
        if (lane == 0) dweights[t * top + j] = dot;
    }
}

// whether a row's elements come in whole, 16-byte aligned 8s
bool vec_rows(const void* p, int64_t ld, int type, int D) {
    const int size = type == kF32 ? 4 : 2;
    return D % 8 == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0 && (ld * size) % 16 == 0;
}

// calls f with the element type, the vector form and the chunks a wave takes:
// four once the pieces still give every CU eight waves
template <class F>
void by_form(int type, bool vec, int64_t tokens, int D, const F& f) {
    const int64_t pieces4 = tokens * ((D + 2047) / 2048);
    auto form = [&](auto T) {
        using One = std::integral_constant<int, 1>;
        using Four = std::integral_constant<int, 4>;
        if (vec) {
            if (pieces4 >= 2048) f(T, std::true_type{}, Four{});
            else f(T, std::true_type{}, One{});
        } else {
            f(T, std::false_type{}, One{});
        }
    };
    if (type == kBf16) form(std::integral_constant<int, kBf16>{});
    else if (type == kF16) form(std::integral_constant<int, kF16>{});
    else form(std::integral_constant<int, kF32>{});
}

}  // namespace

int64_t moe_sort_work_bytes(int64_t S, int E) {
    const int64_t nb = (S + kSortChunk - 1) / kSortChunk;
    return nb > 1 ? nb * (E + 1) * int64_t(sizeof(int)) : 0;
}

hipError_t moe_sort(hipStream_t st, const void* ids, bool wide, int* order, int* position,
                    int* rows, int* offsets, int64_t S, int top, int E, void* work) {
    int* counts = static_cast<int*>(work);
    if (wide)
        return sort_launch(st, static_cast<const int64_t*>(ids), counts, order, position, rows,
                           offsets, S, top, E);
    return sort_launch(st, static_cast<const int32_t*>(ids), counts, order, position, rows,
                       offsets, S, top, E);
}

hipError_t moe_dispatch(hipStream_t st, const void* x, int type, int64_t ldx, const int* position,
                        const int* offsets, void* out, int64_t tokens, int top, int E, int D) {
    by_form(type, vec_rows(x, ldx, type, D) && vec_rows(out, D, type, D), tokens, D,
            [&](auto T, auto V, auto U) {
        constexpr int t = decltype(T)::value, u = decltype(U)::value;
        const int pieces = (D + 512 * u - 1) / (512 * u);
        hipLaunchKernelGGL((moe_dispatch_kernel<t, decltype(V)::value, u>),
                           dim3(unsigned((tokens * pieces + 3) / 4)), dim3(256), 0, st,
                           static_cast<const char*>(x), ldx, position, offsets,
                           static_cast<char*>(out), tokens, top, E, D, pieces);
    });
    return hipGetLastError();
}

hipError_t moe_gather(hipStream_t st, const void* z, int type, int64_t ldz, const int* position,
                      const int* offsets, const float* weights, void* out, int out_type,
                      int64_t tokens, int top, int E, int D) {
    by_form(type, vec_rows(z, ldz, type, D) && vec_rows(out, D, out_type, D), tokens, D,
            [&](auto T, auto V, auto U) {
        constexpr int t = decltype(T)::value, u = decltype(U)::value;
        constexpr bool v = decltype(V)::value;
        const int pieces = (D + 512 * u - 1) / (512 * u);
        const dim3 grid(unsigned((tokens * pieces + 3) / 4));
        auto go = [&](auto TO, auto W) {
            hipLaunchKernelGGL((moe_gather_kernel<t, decltype(TO)::value, v, u, decltype(W)::value>),
                               grid, dim3(256), 0, st, static_cast<const char*>(z), ldz, position,
                               offsets, weights, static_cast<char*>(out), tokens, top, E, D, pieces);
        };
        if (weights) go(T, std::true_type{});
        else if (type == out_type) go(T, std::false_type{});
        else if constexpr (t == kF32) {        // the experts' gradients, fp32 rows of any type
            if (out_type == kBf16) go(std::integral_constant<int, kBf16>{}, std::false_type{});
            else go(std::integral_constant<int, kF16>{}, std::false_type{});
        }
    });
    return hipGetLastError();
}

hipError_t moe_combine_grad(hipStream_t st, const void* dy, int type, int64_t ldy, const void* z,
                            int64_t ldz, const int* position, const int* offsets,
                            const float* weights, void* dz, float* dweights, int64_t tokens,
                            int top, int E, int D) {
    const bool vec = vec_rows(dy, ldy, type, D) && vec_rows(z, ldz, type, D) && vec_rows(dz, D, type, D);
    const dim3 grid(unsigned((tokens + 3) / 4));
    auto go = [&](auto T, auto V) {
        hipLaunchKernelGGL((moe_combine_grad_kernel<decltype(T)::value, decltype(V)::value>), grid,
                           dim3(256), 0, st, static_cast<const char*>(dy), ldy,
                           static_cast<const char*>(z), ldz, position, offsets, weights,
                           static_cast<char*>(dz), dweights, tokens, top, E, D);
    };
    auto form = [&](auto T) {
        if (vec) go(T, std::true_type{});
        else go(T, std::false_type{});
    };
    if (type == kBf16) form(std::integral_constant<int, kBf16>{});
    else if (type == kF16) form(std::integral_constant<int, kF16>{});
    else form(std::integral_constant<int, kF32>{});
    return hipGetLastError();
}

}  // namespace xpuint8
