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
// A counting sort: a block of 16 waves takes 1024 KPL consecutive slots, a wave 64 KPL of
// them, a lane KPL, 64 apart, whose keys it reads once, all together.  The lanes of one
// key are found with one ballot per bit of the key (no atomics, so ranks do not depend
// on timing); the first of them adds their number to the wave's counter of that key.
// With the counters of every wave before it, and those of every block before, a wave
// knows where its first slot of each key goes, and a second pass over the same
// registers hands out the places.  Up to 8192 slots are one launch of one block; more
// take a launch of the counts first, in blocks of 2048 slots (8192 from 128 K on: each
// block reads the counts of all).  Bound by latency: the loads of the keys, some 200 cycles
// for each 64 of a wave, a store a slot.  32 slots 3.5 us, 64 K slots 4.6 + 9.7 us (27 with the
// keys read again from memory in the second pass).
constexpr int kSortWaves = 16;
constexpr int kSortThreads = kSortWaves * 64;
constexpr int kMaxExperts = 1024;

template <class I>
__device__ __forceinline__ int key_of(const I* ids, int64_t s, int E) {
    const I v = ids[s];
    return v >= 0 && v < I(E) ? int(v) : E;
}

// the lanes of the wave whose key equals this lane's, among those of `live`
__device__ __forceinline__ uint64_t peers(int key, int bits, uint64_t live) {
    uint64_t m = live;
    for (int b = 0; b < bits; ++b) {
        const bool one = (key >> b) & 1;
        const uint64_t set = __builtin_amdgcn_ballot_w64(one);
        m &= one ? set : ~set;
    }
    return m;
}

// This lane's keys (-1 past the end) and, in LDS count[wave * (E + 1) + key] (cleared
// here), the number of each key among the wave's.
template <int KPL, class I>
__device__ __forceinline__ void count_keys(const I* ids, int64_t S, int E, int bits,
                                           int (&key)[KPL], int* count) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t lo = (int64_t(blockIdx.x) * kSortWaves + wave) * (64 * KPL) + lane;
#pragma unroll
    for (int i = 0; i < KPL; ++i) key[i] = lo + 64 * i < S ? key_of(ids, lo + 64 * i, E) : -1;
    for (int i = threadIdx.x; i < kSortWaves * (E + 1); i += kSortThreads) count[i] = 0;
    __syncthreads();
    int* mine = count + wave * (E + 1);
#pragma unroll
    for (int i = 0; i < KPL; ++i) {
        const bool in = key[i] >= 0;
        const uint64_t m = peers(key[i], bits, __builtin_amdgcn_ballot_w64(in));
        if (in && __builtin_ctzll(m) == lane) mine[key[i]] += __builtin_popcountll(m);
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
}

template <int KPL, class I>
__global__ __launch_bounds__(kSortThreads) void moe_count_kernel(const I* __restrict__ ids,
                                                                 int* __restrict__ counts,
                                                                 int64_t S, int E, int bits) {
    __shared__ int count[kSortWaves * (kMaxExperts + 1)];
    int key[KPL];
    count_keys(ids, S, E, bits, key, count);
    for (int k = threadIdx.x; k <= E; k += kSortThreads) {
        int n = 0;
        for (int w = 0; w < kSortWaves; ++w) n += count[w * (E + 1) + k];
        counts[int64_t(blockIdx.x) * (E + 1) + k] = n;
    }
}

// counts: the keys' numbers in each block (unused where there is one block)
template <int KPL, class I>
__global__ __launch_bounds__(kSortThreads) void moe_sort_kernel(
    const I* __restrict__ ids, const int* __restrict__ counts, int* __restrict__ order,
    int* __restrict__ position, int* __restrict__ rows, int* __restrict__ offsets, int64_t S,
    int top, int E, int bits) {
    __shared__ int count[kSortWaves * (kMaxExperts + 1)];
    __shared__ int total[kMaxExperts + 1];
    __shared__ int wave_sum[kSortWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int nb = gridDim.x, k = threadIdx.x;
    // per key: its number in the blocks before and in all; of the slots without an
    // expert, which follow all others in slot order, the number before
    int before = 0, all = 0, loose = 0;
    if (nb > 1 && k <= E) {
#pragma unroll 8
        for (int b = 0; b < nb; ++b) {
            const int n = counts[int64_t(b) * (E + 1) + k];
            if (b < int(blockIdx.x)) before += n;
            all += n;
        }
    }
    if (nb > 1 && k == 0) {
#pragma unroll 8
        for (int b = 0; b < int(blockIdx.x); ++b) loose += counts[int64_t(b) * (E + 1) + E];
    }
    if (k >= E) before = all = 0;
    int key[KPL];
    count_keys(ids, S, E, bits, key, count);
    if (nb == 1 && k < E)
        for (int w = 0; w < kSortWaves; ++w) all += count[w * (E + 1) + k];
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
    if (k == 0) {
        int live = 0;
        for (int w = 0; w < kSortWaves; ++w) live += wave_sum[w];
        total[E] = live + loose;
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
    const int64_t lo = (int64_t(blockIdx.x) * kSortWaves + wave) * (64 * KPL) + lane;
#pragma unroll
    for (int i = 0; i < KPL; ++i) {
        const int s = int(lo) + 64 * i;
        const bool in = key[i] >= 0;
        const uint64_t m = peers(key[i], bits, __builtin_amdgcn_ballot_w64(in));
        if (in) {
            const int at = mine[key[i]] + __builtin_popcountll(m & ((uint64_t(1) << lane) - 1));
            order[at] = s;
            position[s] = at;
            rows[at] = s / top;
        }
        // every lane has its place before the counter moves on (the wave's LDS
        // accesses are in order)
        __builtin_amdgcn_wave_barrier();
        if (in && __builtin_ctzll(m) == lane) mine[key[i]] += __builtin_popcountll(m);
        __builtin_amdgcn_wave_barrier();
    }
}

// keys a lane, by the number of slots
int keys_per_lane(int64_t S) { return S <= 1024 ? 1 : S <= 2048 ? 2 : S <= 8192 ? 8 : S <= 131072 ? 2 : 8; }
int sort_blocks(int64_t S) {
    const int64_t chunk = 1024 * keys_per_lane(S);
    return int((S + chunk - 1) / chunk);
}

template <class I>
hipError_t sort_launch(hipStream_t st, const I* ids, int* counts, int* order, int* position,
                       int* rows, int* offsets, int64_t S, int top, int E) {
    int bits = 1;
    while ((1 << bits) < E + 1) ++bits;
    const int nb = sort_blocks(S);
    auto go = [&](auto K) {
        constexpr int kpl = decltype(K)::value;
        if (nb > 1)
            hipLaunchKernelGGL((moe_count_kernel<kpl, I>), dim3(unsigned(nb)), dim3(kSortThreads),
                               0, st, ids, counts, S, E, bits);
        hipLaunchKernelGGL((moe_sort_kernel<kpl, I>), dim3(unsigned(nb)), dim3(kSortThreads), 0,
                           st, ids, counts, order, position, rows, offsets, S, top, E, bits);
    };
    const int kpl = keys_per_lane(S);
    if (kpl == 1) go(std::integral_constant<int, 1>{});
    else if (kpl == 2) go(std::integral_constant<int, 2>{});
    else go(std::integral_constant<int, 8>{});
    return hipGetLastError();
}

// ------------------------------------------------------- rows out and back
// All four are bound by HBM: each row of either side is read or written once.
// They go by tokens, not by rows: a token's own row is read (or its sum kept in
// registers) once for all its slots, and the row of slot j is at position[t, j];
// positions are every row exactly once, so every row is written, zeros where no
// expert has it (position >= offsets[E]).  A wave takes 512 consecutive elements of one
// token (of 2048, four times as many: dispatch 60 against 55 us, the weighted sum 109 / 89);
// position values are clamped to the S rows that exist.  8190 tokens of 2048 bf16 in 8 slots:
// dispatch 55 us (5.5 TB/s), the sum 48 after reads, 89 after writes of as many bytes that are still
// on their way, its gradient 126 (4.6 TB/s).
template <int T>
constexpr int kSize = T == kF32 ? 4 : 2;

struct Piece {
    int64_t t;
    int d;            // first element of this lane's 8
};
// the wave's piece, of `pieces` a token; the launch starts at token t0
__device__ __forceinline__ bool piece_of(int64_t t0, int64_t T, int pieces, Piece& p) {
    const int64_t w = int64_t(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
    const int64_t t = w / pieces;
    p.t = t0 + t;
    p.d = int(w - t * pieces) * 512 + int(threadIdx.x & 63) * 8;
    return p.t < T;
}

// a row's 8 elements at d, of which those past D are left alone
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
template <int T, bool VEC>
__global__ __launch_bounds__(256) void moe_dispatch_kernel(const char* __restrict__ x, int64_t ldx,
                                                           const int* __restrict__ position,
                                                           const int* __restrict__ offsets,
                                                           char* __restrict__ out, int64_t t0,
                                                           int64_t tokens, int top, int E, int D,
                                                           int pieces) {
    Piece p;
    if (!piece_of(t0, tokens, pieces, p) || p.d >= D) return;
    const int S1 = int(tokens * top - 1);
    const int live = offsets[E];
    float v[8];
    load_row8<T, VEC>(x + p.t * ldx * kSize<T>, p.d, D, v);
    const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int j = 0; j < top; ++j) {
        const int at = min(max(position[p.t * top + j], 0), S1);
        char* dst = out + int64_t(at) * D * kSize<T>;
        if (at < live) store_row8<T, VEC>(dst, p.d, D, v);
        else store_row8<T, VEC>(dst, p.d, D, zero);
    }
}

// out[t] = sum over the slots that an expert has, in slot order, of
// [weights[t, j] *] rows[position[t, j]], in fp32, rounded once
template <int T, int TO, bool VEC, bool WEIGHTED>
__global__ __launch_bounds__(256) void moe_gather_kernel(const char* __restrict__ z, int64_t ldz,
                                                         const int* __restrict__ position,
                                                         const int* __restrict__ offsets,
                                                         const float* __restrict__ weights,
                                                         char* __restrict__ out, int64_t t0,
                                                         int64_t tokens, int top, int E, int D,
                                                         int pieces) {
    Piece p;
    if (!piece_of(t0, tokens, pieces, p) || p.d >= D) return;
    const int live = min(offsets[E], int(tokens * top));
    float acc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.f;
    // four rows are requested together (one after the other: 92 against 89 us); one that no
    // expert has gives way to row 0 and is not added
    for (int j0 = 0; j0 < top; j0 += 4) {
        float v[4][8], w[4];
        bool has[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int64_t slot = p.t * top + min(j0 + q, top - 1);
            const int at = position[slot];
            has[q] = j0 + q < top && at >= 0 && at < live;
            w[q] = WEIGHTED ? weights[slot] : 1.f;
            load_row8<T, VEC>(z + int64_t(has[q] ? at : 0) * ldz * kSize<T>, p.d, D, v[q]);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if (!has[q]) continue;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                acc[i] = WEIGHTED ? __builtin_fmaf(w[q], v[q][i], acc[i]) : acc[i] + v[q][i];
        }
    }
    store_row8<TO, VEC>(out + p.t * D * kSize<TO>, p.d, D, acc);
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
// (0 there), one wave a token, slot by slot.  dy's row is read again for each slot, mostly
// past the L2, through which z and dz stream meanwhile: 8190 tokens of 2048 bf16 in 8
// slots read 474 MB, where z's live rows and dy are 289
template <int T, bool VEC>
__global__ __launch_bounds__(256) void moe_combine_grad_kernel(
    const char* __restrict__ dy, int64_t ldy, const char* __restrict__ z, int64_t ldz,
    const int* __restrict__ position, const int* __restrict__ offsets,
    const float* __restrict__ weights, char* __restrict__ dz, float* __restrict__ dweights,
    int64_t t0, int64_t tokens, int top, int E, int D) {
    const int64_t t = t0 + int64_t(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
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

// calls f with the element type and the vector form
template <class F>
void by_form(int type, bool vec, const F& f) {
    auto form = [&](auto T) {
        if (vec) f(T, std::true_type{});
        else f(T, std::false_type{});
    };
    if (type == kBf16) form(std::integral_constant<int, kBf16>{});
    else if (type == kF16) form(std::integral_constant<int, kF16>{});
    else form(std::integral_constant<int, kF32>{});
}

}  // namespace

int64_t moe_sort_work_bytes(int64_t S, int E) {
    const int64_t nb = sort_blocks(S);
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
    const int pieces = (D + 511) / 512;
    by_form(type, vec_rows(x, ldx, type, D) && vec_rows(out, D, type, D), [&](auto T, auto V) {
        in_launches(tokens, 4 * kMaxBlocks / pieces, [&](int64_t t0, int64_t n) {
            hipLaunchKernelGGL((moe_dispatch_kernel<decltype(T)::value, decltype(V)::value>),
                               dim3(unsigned((n * pieces + 3) / 4)), dim3(256), 0, st,
                               static_cast<const char*>(x), ldx, position, offsets,
                               static_cast<char*>(out), t0, tokens, top, E, D, pieces);
        });
    });
    return hipGetLastError();
}

hipError_t moe_gather(hipStream_t st, const void* z, int type, int64_t ldz, const int* position,
                      const int* offsets, const float* weights, void* out, int out_type,
                      int64_t tokens, int top, int E, int D) {
    const int pieces = (D + 511) / 512;
    by_form(type, vec_rows(z, ldz, type, D) && vec_rows(out, D, out_type, D), [&](auto T, auto V) {
        constexpr int t = decltype(T)::value;
        constexpr bool v = decltype(V)::value;
        auto go = [&](auto TO, auto W) {
            in_launches(tokens, 4 * kMaxBlocks / pieces, [&](int64_t t0, int64_t n) {
                hipLaunchKernelGGL((moe_gather_kernel<t, decltype(TO)::value, v, decltype(W)::value>),
                                   dim3(unsigned((n * pieces + 3) / 4)), dim3(256), 0, st,
                                   static_cast<const char*>(z), ldz, position, offsets, weights,
                                   static_cast<char*>(out), t0, tokens, top, E, D, pieces);
            });
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
    by_form(type, vec, [&](auto T, auto V) {
        in_launches(tokens, 4 * kMaxBlocks, [&](int64_t t0, int64_t n) {
            hipLaunchKernelGGL((moe_combine_grad_kernel<decltype(T)::value, decltype(V)::value>),
                               dim3(unsigned((n + 3) / 4)), dim3(256), 0, st,
                               static_cast<const char*>(dy), ldy, static_cast<const char*>(z), ldz,
                               position, offsets, weights, static_cast<char*>(dz), dweights, t0,
                               tokens, top, E, D);
        });
    });
    return hipGetLastError();
}

}  // namespace xpuint8
