// Log-probabilities of given tokens, entropy and the most likely ids of rows of logits (tmw_token_logprobs), and the gradient.
//
// With M the largest logit of a row and S = sum e^(x - M): log p_i = (x_i - M) - ln S, and the entropy
// H = ln S - (1 / S) sum e^(x - M) (x - M).  The subtractions come first: ln S + M rounded together would cost what the logits
// have in front of their differences.  One pass: every thread keeps the largest of its logits, and S and the other sum under it.
// The gradient, for the gradients g of log p_t, h of H and a_j of the log-probability of the j-th likely id i_j:
//   dx_i = g [i = t] + sum_j a_j [i = i_j] - p_i (g + sum_j a_j + h (log p_i + H)).
// Both are bound by HBM: the logits once, and once more with their gradient on the way back (bf16, 4096 rows of 128000: 178 us, 5.9
// TB/s, with the exponentials at 73 % of their pipe; 319 us, 6.6 TB/s).
//
// The most likely ids, the lower one first among equals: if every warp knows r logits, of different threads, at or above a bound,
// and r times the warps is k, then the k best of the row are at or above the bound.  The pass leaves every thread's best, so the
// bound costs r maxima in each warp and the least of them all; then only the threads whose best reaches it look at their logits
// again (from L2).  What they find - some dozens - is ranked by counting what is ahead of each: (value, index) in 64 bits, so there
// are no equals, and the order of arrival does not matter.  Where it is more than fits (long runs of equal logits), every warp
// keeps a sorted list of 32 keys, one to a lane, and the lists are merged.
//
// A row goes to a CTA, or, where there are few, to a cluster of them that joins through distributed shared memory.
#include <cooperative_groups.h>
#include <float.h>
#include <math_constants.h>

#include "tc_ptx.cuh"
#include "tmw_common.cuh"

namespace tmw {
namespace {

constexpr long long kNoTarget = -100;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kMostTop = 32;

struct Logprobs {
    const void* logits;
    long long stride[2];
    const int64_t* targets;
    float *logprobs, *entropy, *lse, *top_logprobs;
    int64_t* top_ids;
    int tokens, vocab, top, rows;
    int* status;
};

__device__ __forceinline__ const char* row_of(const Logprobs& p, int row, int size) {
    const int b = row / p.tokens;
    return static_cast<const char*>(p.logits) + (b * p.stride[0] + (row - b * p.tokens) * p.stride[1]) * size;
}

// A row as whole 16-byte vectors: vector v holds the elements v * E - shift .. v * E - shift + E - 1, the first and the last one
// in part.
template <typename T>
struct RowView {
    static constexpr int E = 16 / (int)sizeof(T);
    const T* x;
    int shift, vocab, vectors;
    __device__ __forceinline__ RowView(const char* at, int vocab) : x(reinterpret_cast<const T*>(at)), vocab(vocab) {
        shift = (int)(reinterpret_cast<uintptr_t>(at) % 16 / sizeof(T));
        vectors = (vocab + shift + E - 1) / E;
    }
    __device__ __forceinline__ bool whole(int v) const { return v * E >= shift && (v + 1) * E - shift <= vocab; }
    __device__ __forceinline__ bool has(int v, int e) const { return v * E + e >= shift && v * E + e - shift < vocab; }
    // elements that are not the row's come as -inf
    __device__ __forceinline__ uint4 load(int v) const {
        uint4 raw;
        if (whole(v)) {
            raw = *reinterpret_cast<const uint4*>(x + (long long)v * E - shift);
        } else {
            T* part = reinterpret_cast<T*>(&raw);
#pragma unroll
            for (int e = 0; e < E; ++e) part[e] = has(v, e) ? x[v * E + e - shift] : from_f32<T>(-CUDART_INF_F);
        }
        return raw;
    }
};

template <typename T>
__device__ __forceinline__ void unpack(const uint4& raw, float (&f)[16 / sizeof(T)]);
template <>
__device__ __forceinline__ void unpack<float>(const uint4& raw, float (&f)[4]) {
    f[0] = __uint_as_float(raw.x); f[1] = __uint_as_float(raw.y); f[2] = __uint_as_float(raw.z); f[3] = __uint_as_float(raw.w);
}
template <>
__device__ __forceinline__ void unpack<__nv_bfloat16>(const uint4& raw, float (&f)[8]) {
    load8<__nv_bfloat16>(reinterpret_cast<const __nv_bfloat16*>(&raw), f);
}
template <>
__device__ __forceinline__ void unpack<__half>(const uint4& raw, float (&f)[8]) {
    load8<__half>(reinterpret_cast<const __half*>(&raw), f);
}

template <typename T>
__device__ __forceinline__ void pack(const float (&f)[16 / sizeof(T)], uint4& raw);
template <>
__device__ __forceinline__ void pack<float>(const float (&f)[4], uint4& raw) {
    raw = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}
template <>
__device__ __forceinline__ void pack<__nv_bfloat16>(const float (&f)[8], uint4& raw) {
    store8<__nv_bfloat16>(reinterpret_cast<__nv_bfloat16*>(&raw), f);
}
template <>
__device__ __forceinline__ void pack<__half>(const float (&f)[8], uint4& raw) { store8<__half>(reinterpret_cast<__half*>(&raw), f); }

// the largest of a vector's elements (NaN aside) - for 16-bit types two at a time
template <typename T>
__device__ __forceinline__ float largest(const uint4& raw);
template <>
__device__ __forceinline__ float largest<float>(const uint4& raw) {
    return fmaxf(fmaxf(__uint_as_float(raw.x), __uint_as_float(raw.y)), fmaxf(__uint_as_float(raw.z), __uint_as_float(raw.w)));
}
template <>
__device__ __forceinline__ float largest<__nv_bfloat16>(const uint4& raw) {
    const __nv_bfloat162* v = reinterpret_cast<const __nv_bfloat162*>(&raw);
    const __nv_bfloat162 m = __hmax2(__hmax2(v[0], v[1]), __hmax2(v[2], v[3]));
    return fmaxf(__bfloat162float(m.x), __bfloat162float(m.y));
}
template <>
__device__ __forceinline__ float largest<__half>(const uint4& raw) {
    const __half2* v = reinterpret_cast<const __half2*>(&raw);
    const __half2 m = __hmax2(__hmax2(v[0], v[1]), __hmax2(v[2], v[3]));
    return fmaxf(__half2float(m.x), __half2float(m.y));
}

// ---- ranking ------------------------------------------------------------------------------------------------------------------
// an order of unsigned numbers that is the values' (-0 is 0; 0: none), and back
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t bits = __float_as_uint(x + 0.0f);
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t order) {
    return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order);
}
// value above index, the lower index first
__device__ __forceinline__ uint64_t key_of(uint32_t order, uint32_t index) { return (uint64_t)order << 32 | (uint32_t)~index; }
__device__ __forceinline__ uint32_t index_of(uint64_t key) { return ~(uint32_t)key; }

// one step of a bitonic network over the lanes: the larger key of a pair to the lower lane (down), or to the upper one
__device__ __forceinline__ uint64_t exchange(uint64_t key, int apart, bool down) {
    const uint64_t other = __shfl_xor_sync(0xffffffffu, key, apart);
    const bool lower = (threadIdx.x & apart) == 0;
    return (lower == down) == (key > other) ? key : other;
}
// the largest key to lane 0
__device__ __forceinline__ uint64_t sorted(uint64_t key) {
#pragma unroll
    for (int size = 2; size <= 32; size *= 2)
#pragma unroll
        for (int apart = size / 2; apart > 0; apart /= 2) key = exchange(key, apart, (threadIdx.x & size & 31) == 0);
    return key;
}
// the 32 largest of two sorted lists
__device__ __forceinline__ uint64_t merged(uint64_t a, uint64_t b) {
    const uint64_t back = __shfl_sync(0xffffffffu, b, 31 - (threadIdx.x & 31));
    uint64_t key = a > back ? a : back;
#pragma unroll
    for (int apart = 16; apart > 0; apart /= 2) key = exchange(key, apart, true);
    return key;
}
// The 32 largest of n sorted lists (n a power of two, at most twice the CTA's warps), in the first one.  All threads.
__device__ __forceinline__ void merge_lists(uint64_t (*lists)[32], int n) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (; n > 1; n /= 2) {
        __syncthreads();
        uint64_t key = 0;
        if (warp < n / 2) key = merged(lists[warp][lane], lists[warp + n / 2][lane]);
        if (warp < n / 2) lists[warp][lane] = key;
    }
    __syncthreads();
}

// ---- forward --------------------------------------------------------------------------------------------------------------------
// of a part of a row: largest logit (at least -FLT_MAX), sum of e^(x - m), sum of e^(x - m) (x - m) log2(e)
struct Sums {
    float m, s, t;
};
// A logarithm below which a weight is zero (2^-150, flushed): the bound keeps infinity times zero out of the sums.
__device__ __forceinline__ float bounded(float d) { return fmaxf(d, -150.f); }
// the same under a larger maximum
__device__ __forceinline__ void raise(Sums& a, float m) {
    const float d = bounded((a.m - m) * kLog2e), w = ex2_ftz(d);
    a.t = w * fmaf(d, a.s, a.t);
    a.s *= w;
    a.m = m;
}
__device__ __forceinline__ float warp_max(float x) { return value_of(__reduce_max_sync(0xffffffffu, order_of(x))); }
// all lanes' together, on every lane
__device__ __forceinline__ Sums warp_sums(Sums a) {
    raise(a, warp_max(a.m));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
        a.t += __shfl_xor_sync(0xffffffffu, a.t, o);
    }
    return a;
}

constexpr float kSlack = 8.f;  // (each unit is one of 2^-23 on the entropy, where the sums are brought under the largest logit)
constexpr int kKeys = 256;  // that are ranked by counting

template <typename T, int W>
__global__ void __launch_bounds__(W * 32, 32 / W) logprobs_kernel(const __grid_constant__ Logprobs p, int ctas) {
    constexpr int THREADS = W * 32, E = RowView<T>::E, AHEAD = 4;
    __shared__ Sums sums[W];
    __shared__ uint32_t low[W];
    __shared__ Sums part;   // this CTA's
    __shared__ float rest;  // S without the largest logit's own 1
    __shared__ __align__(16) uint64_t keys[kKeys / 32][32];
    __shared__ uint64_t tops[kMostTop];  // the likely ids' keys in order
    __shared__ int found;
    __shared__ unsigned char chosen[W][32];
    __shared__ Sums whole_row;
    __shared__ float whole_rest;
    namespace cg = cooperative_groups;
    const int row = blockIdx.x / ctas, rank = blockIdx.x - row * ctas, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const RowView<T> x(row_of(p, row, sizeof(T)), p.vocab);
    const int per = (x.vectors + ctas - 1) / ctas, v_first = min(rank * per, x.vectors), v_end = min(v_first + per, x.vectors);
    long long y = kNoTarget;
    float picked = 0.f;
    if (tid == 0 && rank == 0) {
        y = p.targets[row];
        if (y >= 0 && y < p.vocab) picked = to_f32<T>(x.x[y]);
    }
    if (tid == 0) found = 0;
    if (tid < kMostTop) tops[tid] = 0;

    // best: this thread's largest logit.  Its sums stand under a base that follows only a logit more than kSlack above it: some
    // lane of a warp meets a new largest logit at most steps (3000 rows of 49999 with it followed each time: 89 us, 190 for 4096 of
    // 128000).
    float best = -CUDART_INF_F, base = -FLT_MAX, limit = -FLT_MAX;
    uint64_t s2 = ptx::pack2(0.f, 0.f), t2 = s2, base2 = ptx::pack2(FLT_MAX, FLT_MAX);
    const uint64_t log2e2 = ptx::pack2(kLog2e, kLog2e);
    auto take = [&](const uint4& raw) {
        const float top = largest<T>(raw);
        best = fmaxf(best, top);
        if (top > limit) {
            Sums a, b;
            a.m = b.m = base;
            ptx::unpack2(s2, a.s, b.s);
            ptx::unpack2(t2, a.t, b.t);
            base = fmaxf(top, base);
            limit = base + kSlack;
            raise(a, base);
            raise(b, base);
            s2 = ptx::pack2(a.s, b.s);
            t2 = ptx::pack2(a.t, b.t);
            base2 = ptx::pack2(-base, -base);
        }
        float f[E];
        unpack<T>(raw, f);
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            float da, db;
            ptx::unpack2(ptx::mul2(ptx::add2(ptx::pack2(f[e], f[e + 1]), base2), log2e2), da, db);
            const uint64_t w = ptx::pack2(ex2_ftz(da), ex2_ftz(db));  // (not of the bounded one: that would drop a NaN)
            s2 = ptx::add2(s2, w);
            t2 = ptx::fma2(w, ptx::pack2(bounded(da), bounded(db)), t2);
        }
    };
    int v = v_first + tid;
    const bool any = v < v_end;
    if (any && !x.whole(v)) {  // (the row's first vector, or its only one)
        take(x.load(v));
        v += THREADS;
    }
    // whole vectors, the next batch on its way under this one
    const int stop = v_end > v_first && !x.whole(v_end - 1) ? v_end - 1 : v_end;
    const uint4* at = reinterpret_cast<const uint4*>(x.x - x.shift) + v;
    uint4 now[AHEAD], next[AHEAD];
    auto fetch = [&](uint4 (&raw)[AHEAD]) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) raw[u] = at[u * THREADS];
        at += AHEAD * THREADS;
    };
    int batches = v < stop ? ((stop - v - 1) / THREADS + 1) / AHEAD : 0;
    v += batches * AHEAD * THREADS;
    if (batches > 0) fetch(now);
    for (; batches > 1; --batches) {
        fetch(next);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) take(now[u]);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) now[u] = next[u];
    }
    // the rest, fewer than a batch, under the last one
#pragma unroll
    for (int u = 0; u < AHEAD - 1; ++u)
        if (v + u * THREADS < v_end) next[u] = x.load(v + u * THREADS);
    if (batches > 0) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) take(now[u]);
    }
#pragma unroll
    for (int u = 0; u < AHEAD - 1; ++u)
        if (v + u * THREADS < v_end) take(next[u]);
    if (AHEAD > 1 && v + (AHEAD - 1) * THREADS < v_end) take(x.load(v + (AHEAD - 1) * THREADS));  // (the row's last, in part)
    float sa, sb, ta, tb;
    ptx::unpack2(s2, sa, sb);
    ptx::unpack2(t2, ta, tb);
    Sums mine{base, sa + sb, ta + tb};
    raise(mine, fmaxf(best, base));
    const Sums of_warp = warp_sums(mine);
    const uint32_t best_order = any ? order_of(best) : 0;
    if (lane == 0) sums[warp] = of_warp;
    // the r-th best of every warp whose threads all have logits (a warp alone: of as many as have some, if those are enough); with
    // less than one such warp, everything fits
    const int n_vectors = v_end - v_first, full = W == 1 ? (n_vectors >= p.top ? 1 : 0) : min(n_vectors, THREADS) / 32;
    if (p.top > 0 && warp < full) {
        uint32_t left = best_order, top = 0;
        for (int r = (p.top + full - 1) / full; r > 0; --r) {
            top = __reduce_max_sync(0xffffffffu, left);
            if (lane == __ffs(__ballot_sync(0xffffffffu, left == top)) - 1) left = 0;
        }
        if (lane == 0) low[warp] = top;
    }
    __syncthreads();
    if (warp == 0) {
        const Sums all = warp_sums(lane < W ? sums[lane] : Sums{-FLT_MAX, 0.f, 0.f});
        if (lane == 0) {
            part = all;
            rest = all.s - 1.f;
        }
    }

    if (p.top > 0) {
        uint32_t least = full > 0 ? 0xffffffffu : 0;
        for (int w = 0; w < full; ++w) least = min(least, low[w]);
        const float floor = least == 0 ? -CUDART_INF_F : value_of(least);
        const bool look = any && best >= floor;
        const uint32_t todo = __ballot_sync(0xffffffffu, look);
        const int looking = __popc(todo), rounds = (v_end - v_first + THREADS - 1) / THREADS;
        if (look) chosen[warp][__popc(todo & ((1u << lane) - 1))] = (unsigned char)lane;
        __syncwarp();
        for (int i = lane; i < looking * rounds; i += 32) {
            const int c = i / rounds, at = v_first + warp * 32 + chosen[warp][c] + (i - c * rounds) * THREADS;
            if (at >= v_end) continue;
            float f[E];
            unpack<T>(x.load(at), f);
            uint32_t hits = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) hits |= (f[e] >= floor ? 1u : 0u) << e;
            for (; hits != 0; hits &= hits - 1) {
                const int e = __ffs(hits) - 1;
                if (!x.has(at, e)) continue;
                const int n = atomicAdd(&found, 1);
                if (n < kKeys) keys[n / 32][n % 32] = key_of(order_of(to_f32<T>(x.x[at * E + e - x.shift])), (uint32_t)(at * E + e));
            }
        }
        __syncthreads();
        const int n = found;
        if (n <= kKeys) {
            for (int i = tid; i < n; i += THREADS) {
                const uint64_t key = keys[i / 32][i % 32];
                int ahead = 0;
#pragma unroll 4
                for (int j = 0; j < n; ++j) ahead += keys[j / 32][j % 32] > key;
                if (ahead < p.top) tops[ahead] = key;
            }
        } else {
            uint64_t top = 0;
            for (int i0 = 0; i0 < looking * rounds; i0 += 32) {
                const int i = i0 + lane, c = min(i / rounds, looking - 1);
                const int at = v_first + warp * 32 + chosen[warp][c] + (i - c * rounds) * THREADS;
                const bool there = i < looking * rounds && at < v_end;
                float f[E];
                if (there) unpack<T>(x.load(at), f);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const uint64_t key = there && x.has(at, e) ? key_of(order_of(f[e]), (uint32_t)(at * E + e)) : 0;
                    const uint64_t last = __shfl_sync(0xffffffffu, top, p.top - 1);
                    if (__any_sync(0xffffffffu, key > last)) top = merged(top, sorted(key > last ? key : 0));
                }
            }
            __syncthreads();
            keys[warp][lane] = top;
            merge_lists(keys, W);
            if (tid < p.top) tops[tid] = keys[0][tid];
        }
    }
    __syncthreads();

    // A row whose largest logit has nearly all of it: ln S = ln(1 + rest) is as exact as the rest is, and in fp32 a sum that holds the 1
    // would leave a rest of 2^-10 with 14 bits.  The one thread that has that logit leaves its sums to its warp, without it.
    if (part.s >= 1.f && part.s < 1.f + 1.f / 64) {
        const bool has_largest = any && best == part.m;
        Sums others = mine;
        raise(others, part.m);
        if (has_largest) others.s = others.t = 0.f;
        const uint32_t owner = __ballot_sync(0xffffffffu, has_largest);
        for (int at = v_first + warp * 32 + __ffs(owner) - 1 + lane * THREADS; owner != 0 && at < v_end; at += 32 * THREADS) {
            float f[E];
            unpack<T>(x.load(at), f);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float d = (f[e] - part.m) * kLog2e, w = f[e] < part.m ? ex2_ftz(d) : 0.f;
                others.s += w;
                others.t = fmaf(w, bounded(d), others.t);
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            others.s += __shfl_xor_sync(0xffffffffu, others.s, o);
            others.t += __shfl_xor_sync(0xffffffffu, others.t, o);
        }
        if (lane == 0) sums[warp] = others;
        __syncthreads();
        if (tid == 0) {
            rest = part.t = 0.f;
            for (int w = 0; w < W; ++w) {
                rest += sums[w].s;
                part.t += sums[w].t;
            }
        }
        __syncthreads();
    }

    if (ctas > 1) {  // the first CTA of the cluster takes the others' parts
        auto cluster = cg::this_cluster();
        cluster.sync();
        if (rank == 0) {
            if (warp == 0) {
                const Sums its = lane < ctas ? *cluster.map_shared_rank(&part, lane) : Sums{-FLT_MAX, 0.f, 0.f}, all = warp_sums(its);
                // the rest: of the first part with the largest logit, and all of the others
                const int owner = __ffs(__ballot_sync(0xffffffffu, its.m == all.m)) - 1;
                float others = its.s * ex2_ftz((its.m - all.m) * kLog2e);
                if (lane == owner) others = *cluster.map_shared_rank(&rest, lane);
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) others += __shfl_xor_sync(0xffffffffu, others, o);
                if (lane == 0) {
                    whole_row = all;
                    whole_rest = others;
                }
            }
            if (p.top > 0) {
                for (int c = warp; c < ctas; c += W) keys[c][lane] = cluster.map_shared_rank(tops, c)[lane];
                merge_lists(keys, ctas);
                if (tid < p.top) tops[tid] = keys[0][tid];
            }
        }
        cluster.sync();
        if (rank != 0) return;
    } else if (tid == 0) {
        whole_row = part;
        whole_rest = rest;
    }
    __syncthreads();

    const Sums all = whole_row;
    const bool fine = all.s > 0.f;  // (NaN: a NaN or +inf among the logits; 0: nothing but -inf)
    const float log_sum = log1pf(whole_rest);
    if (tid == 0) {
        float lp = CUDART_NAN_F;
        if (y == kNoTarget) lp = 0.f;
        else if (y < 0 || y >= p.vocab) atomicCAS(p.status, 0, (int)TMW_ERR_INVALID_ARGUMENT);
        else if (fine) lp = (picked - all.m) - log_sum;
        p.logprobs[row] = lp;
        p.entropy[row] = fine ? log_sum - kLn2 * (all.t / all.s) : CUDART_NAN_F;
        if (p.lse != nullptr) {
            p.lse[2LL * row] = fine ? all.m : CUDART_NAN_F;
            p.lse[2LL * row + 1] = fine ? log_sum : CUDART_NAN_F;
        }
    }
    if (tid < p.top) {
        const long long at = (long long)row * p.top + tid;
        const uint64_t key = tops[tid];
        p.top_ids[at] = fine ? (int64_t)(index_of(key) - (uint32_t)x.shift) : -1;
        p.top_logprobs[at] = fine ? (value_of((uint32_t)(key >> 32)) - all.m) - log_sum : CUDART_NAN_F;
    }
}

// ---- backward ---------------------------------------------------------------------------------------------------------------------
struct LogprobsBackward {
    Logprobs f;
    const float *d_logprobs, *d_entropy, *d_top;
    void* d_logits;
    long long stride[2];
};

// (us with 4, 8, 16 and 32 vectors to a thread, bf16: 4096 rows of 128000 without the entropy 361, 326, 325, 327, with it 322, 325, 326,
// 329; 4096 of 50264 135, 136, 133, 136; 4 of 128000 4.2, 5.3, 6.3, 8.4.  2048 of 32000 in fp32, and of 1000 and 8000, the same with all.)
constexpr int kBackThreads = 256, kBackVectors = 16;  // vectors of a thread

// VEC: whole vectors; else (logits and gradient begin at different places of their vectors) one element at a time.
// H: the entropy has a gradient.
template <typename T, bool VEC, bool H>
__global__ void __launch_bounds__(kBackThreads) logprobs_backward_kernel(const __grid_constant__ LogprobsBackward p) {
    constexpr int E = VEC ? RowView<T>::E : 1, AHEAD = 2;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 31;
    const RowView<T> x(row_of(p.f, row, sizeof(T)), p.f.vocab);
    const int b = row / p.f.tokens;
    T* d = static_cast<T*>(p.d_logits) + b * p.stride[0] + (row - b * p.f.tokens) * p.stride[1];
    const int shift = VEC ? x.shift : 0, n = VEC ? x.vectors : p.f.vocab;
    const int first = blockIdx.y * (kBackThreads * kBackVectors), end = min(first + kBackThreads * kBackVectors, n);

    // this thread's vectors, every kBackThreads-th one of the CTA's; the row's first and last may be there in part and go by
    // themselves
    const int count = first + tid < end ? (end - first - tid + kBackThreads - 1) / kBackThreads : 0;
    int from = 0, to = count;  // the whole ones
    if (VEC && count > 0) {
        if (!x.whole(first + tid)) from = 1;
        if (!x.whole(first + tid + (count - 1) * kBackThreads)) to = count - 1;
    }
    // the first logits are on their way while the row's numbers are, and then AHEAD vectors always
    const uint4* in = reinterpret_cast<const uint4*>(x.x - x.shift) + first + tid;
    uint4 raw[AHEAD];
    auto fetch = [&](int i) {
        if (VEC && i >= from && i < to) raw[i % AHEAD] = in[i * kBackThreads];
    };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) fetch(i);

    const float m = p.f.lse[2LL * row], log_sum = p.f.lse[2LL * row + 1];
    const long long y = p.f.targets[row];
    const float h = H ? p.d_entropy[row] : 0.f;
    float g = p.d_logprobs != nullptr && y != kNoTarget ? p.d_logprobs[row] : 0.f;
    if (y != kNoTarget && (y < 0 || y >= p.f.vocab)) g = CUDART_NAN_F;
    const int top = p.d_top != nullptr ? p.f.top : 0;
    float pulled = top > 0 && lane < top ? p.d_top[(long long)row * top + lane] : 0.f;
    bool none = true;  // nothing comes back to the row: nothing goes on, whatever its logits are
    if (top > 0) {
        none = __all_sync(0xffffffffu, pulled == 0.f);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) pulled += __shfl_xor_sync(0xffffffffu, pulled, o);
    }
    none = none && g == 0.f && h == 0.f;
    pulled += g;
    // dx_i = p_i (-pulled - h H - h log p_i)
    const float at_zero = H ? -fmaf(h, p.f.entropy[row], pulled) : -pulled;
    auto gradient = [&](float v) {
        const float lp = (v - m) - log_sum;
        return ex2_ftz(lp * kLog2e) * (H ? fmaf(-h, fmaxf(lp, -200.f), at_zero) : at_zero);  // (e^-200 is zero: infinity stays out)
    };
    const uint64_t m2 = ptx::pack2(-m, -m), log_sum2 = ptx::pack2(-log_sum, -log_sum), log2e2 = ptx::pack2(kLog2e, kLog2e),
                   h2 = ptx::pack2(-h, -h), zero2 = ptx::pack2(at_zero, at_zero);
    auto gradients = [&](float va, float vb, float& ra, float& rb) {
        const uint64_t lp = ptx::add2(ptx::add2(ptx::pack2(va, vb), m2), log_sum2);
        float ea, eb;
        ptx::unpack2(ptx::mul2(lp, log2e2), ea, eb);
        uint64_t c = zero2;
        if (H) {
            float la, lb;
            ptx::unpack2(lp, la, lb);
            c = ptx::fma2(h2, ptx::pack2(fmaxf(la, -200.f), fmaxf(lb, -200.f)), zero2);
        }
        ptx::unpack2(ptx::mul2(ptx::pack2(ex2_ftz(ea), ex2_ftz(eb)), c), ra, rb);
    };
    auto one = [&](int v, int e) {  // an element by itself
        const int i = v * E + e - shift;
        if (VEC && !x.has(v, e)) return;
        d[i] = from_f32<T>(none ? 0.f : gradient(to_f32<T>(x.x[i])));
    };
    if constexpr (VEC) {
        uint4* out = reinterpret_cast<uint4*>(d - shift) + first + tid;
#pragma unroll
        for (int i = 0; i < kBackVectors; ++i) {
            if (i >= to) break;
            const uint4 now = raw[i % AHEAD];
            if (i + AHEAD < kBackVectors) fetch(i + AHEAD);
            if (i < from) continue;
            float f[E];
            unpack<T>(now, f);
#pragma unroll
            for (int e = 0; e < E; e += 2) gradients(f[e], f[e + 1], f[e], f[e + 1]);
            uint4 result;
            pack<T>(f, result);
            out[i * kBackThreads] = none ? make_uint4(0, 0, 0, 0) : result;
        }
        if (from > 0) {
#pragma unroll
            for (int e = 0; e < E; ++e) one(first + tid, e);
        }
        if (to < count && count - 1 >= from) {
#pragma unroll
            for (int e = 0; e < E; ++e) one(first + tid + (count - 1) * kBackThreads, e);
        }
    } else {
        for (int i = 0; i < count; ++i) one(first + tid + i * kBackThreads, 0);
    }
    if (none) return;
    __syncthreads();  // over what the pass has written: the target and the likely ids, whose gradients are more
    if (tid >= 32) return;
    // With `more` its own incoming gradient and `others` the rest of the row's: more (1 - p) - p (others + h (log p + H)).  1 - p
    // comes from log p, and the others are added up without `more`: where an id has nearly all of its row, more - p (more + others) by
    // a subtraction would leave little of it (nothing from log p = -2e-8 on), and the forward has log p to 1e-5 of itself.
    auto of_one = [&](long long i, float more, float others) {
        const float lp = (to_f32<T>(x.x[i]) - m) - log_sum;
        if (H) others = fmaf(h, fmaxf(lp, -200.f) + p.f.entropy[row], others);
        return fmaf(-ex2_ftz(lp * kLog2e), others, -more * expm1f(lp));
    };
    long long id = tid < top ? p.f.top_ids[(long long)row * top + tid] : -1;
    float more = tid < top ? p.d_top[(long long)row * top + tid] : 0.f, others = 0.f;
    for (int l = 0; l < top; ++l) {
        const float its = __shfl_sync(0xffffffffu, more, l);
        if (l != lane) others += its;
    }
    const bool is_target = id == y && id >= 0;
    if (!__any_sync(0xffffffffu, is_target)) {  // a lane without a likely id takes the target; else the last one, in turn
        const bool spare = top < 32 ? tid == top : tid == 31;
        if (spare && top == 32 && y >= 0 && y < p.f.vocab && (y + shift) / E >= first && (y + shift) / E < end)
            d[y] = from_f32<T>(of_one(y, g, others + more));
        if (spare && top < 32) id = y, more = g;
        else others += g;
    } else if (is_target) {
        more += g;
    } else {
        others += g;
    }
    if (id < 0 || id >= p.f.vocab || (id + shift) / E < first || (id + shift) / E >= end) return;
    d[id] = from_f32<T>(of_one(id, more, others));
}

template <typename T, int W>
int launch_forward(const Logprobs& p, int ctas, cudaStream_t stream) {
    TMW_CUDA_TRY(launch_ex(logprobs_kernel<T, W>, dim3((unsigned)p.rows * ctas), dim3(W * 32), 0, stream, false, ctas, p, ctas));
    return TMW_OK;
}
template <typename T>
int launch_forward(const Logprobs& p, cudaStream_t stream) {
    // Few rows: eight warps each, and clusters while every thread of them has a vector or more.  With rows enough to keep kWarpsBusy
    // warps to an SM, a row has fewer warps - no barrier to wait at, more rows at once - unless a thread's part of it, or what the
    // likely ids make it read again, top / (32 warps) of the row, became long.  Measured, us, bf16:
    //                                     1 warp   2      4      8 warps
    //   16384 rows of 1000, no ids         21.5   28.5   43.1   76.9
    //   4096 rows of 8000, no ids          19.7   20.6   24.7   33.3
    //   3000 rows of 50000, no ids         67.6   66.2   61.2   64.6   (four here: kMostOfThread)
    //   4096 rows of 128000, no ids       178.4  173.2  168.8  171.0   (eight here)
    //   3000 rows of 49999, 5 ids, fp16           98.3   81.3   83.4   (four here: kMostAgain)
    // kMostAgain, us with 512 | 2048 | 8192: 4096 rows of 16000 with 5 ids 59.6 | 47.2 | 47.2, with 20 70 | 70 | 55; 4096 of 8000 with 20 54 | 39 |
    // 38; 4096 of 32000 with 10 88 | 88 | 78; 2048 of 50257 with 20 73 | 73 | 76; 2048 of 32000 with 5 in fp32 65 | 66 | 72: no one number is best for all.
    constexpr int kWarpsBusy = 20, kMostAgain = 2048, kMostOfThread = 64;
    const int vectors = (int)(((long long)p.vocab * sizeof(T) + 15) / 16);
    int warps = 8;
    while (warps > 1 && (vectors <= warps * 16 || ((long long)p.rows * (warps / 2) >= (long long)kWarpsBusy * sm_count() &&
                                                   vectors <= warps * 16 * kMostOfThread &&
                                                   (long long)p.top * vectors <= (long long)kMostAgain * (warps / 2) * (warps / 2))))
        warps /= 2;
    if (warps == 1) return launch_forward<T, 1>(p, 1, stream);
    if (warps == 2) return launch_forward<T, 2>(p, 1, stream);
    if (warps == 4) return launch_forward<T, 4>(p, 1, stream);
    int ctas = 1;
    while (ctas < 8 && (long long)p.rows * ctas * 2 <= 4LL * sm_count() && vectors / (ctas * 2) >= 256) ctas *= 2;
    return launch_forward<T, 8>(p, ctas, stream);
}

template <typename T>
int launch_backward(const LogprobsBackward& p, cudaStream_t stream) {
    constexpr int E = RowView<T>::E;
    const bool vec = (reinterpret_cast<uintptr_t>(p.f.logits) - reinterpret_cast<uintptr_t>(p.d_logits)) % 16 == 0 &&
                     (p.f.stride[0] - p.stride[0]) % E == 0 && (p.f.stride[1] - p.stride[1]) % E == 0;
    const long long n = vec ? ((long long)p.f.vocab + 2 * E - 2) / E : p.f.vocab;
    const dim3 grid((unsigned)p.f.rows, (unsigned)((n + kBackThreads * kBackVectors - 1) / (kBackThreads * kBackVectors)));
    const auto run = [&](auto kern) { kern<<<grid, kBackThreads, 0, stream>>>(p); };
    if (vec) p.d_entropy != nullptr ? run(logprobs_backward_kernel<T, true, true>) : run(logprobs_backward_kernel<T, true, false>);
    else p.d_entropy != nullptr ? run(logprobs_backward_kernel<T, false, true>) : run(logprobs_backward_kernel<T, false, false>);
    TMW_CUDA_TRY(cudaGetLastError());
    return TMW_OK;
}

int checked(const tmw_logprobs_desc* d, Logprobs& p) {
    if (d == nullptr) return TMW_ERR_INVALID_ARGUMENT;
    if (d->dtype != TMW_F32 && d->dtype != TMW_BF16 && d->dtype != TMW_F16) return TMW_ERR_UNSUPPORTED;
    if (d->batch < 0 || d->tokens < 0 || d->vocab <= 0 || d->top < 0 || d->top > d->vocab || d->stride[0] < 0 || d->stride[1] < 0)
        return TMW_ERR_INVALID_ARGUMENT;
    if (d->top > kMostTop) {
        set_error_text("tmw_token_logprobs: at most 32 alternatives");
        return TMW_ERR_TOO_LARGE;
    }
    // (the grids' limits)
    if ((int64_t)d->batch * d->tokens > 0x7fffffff / 8 || d->vocab > 1 << 26) return TMW_ERR_TOO_LARGE;
    if (d->batch == 0 || d->tokens == 0) return TMW_OK;
    if (d->logits == nullptr || d->targets == nullptr || d->entropy == nullptr || reinterpret_cast<uintptr_t>(d->logits) % dtype_size(d->dtype) != 0)
        return TMW_ERR_INVALID_ARGUMENT;
    p.logits = d->logits;
    p.stride[0] = d->stride[0];
    p.stride[1] = d->stride[1];
    p.targets = d->targets;
    p.logprobs = d->logprobs; p.entropy = d->entropy; p.lse = d->lse; p.top_logprobs = d->top_logprobs; p.top_ids = d->top_ids;
    p.tokens = d->tokens; p.vocab = d->vocab; p.top = d->top;
    p.rows = d->batch * d->tokens;
    return TMW_OK;
}

}  // namespace
}  // namespace tmw

extern "C" int tmw_token_logprobs(const tmw_logprobs_desc* d, void* stream) {
    using namespace tmw;
    Logprobs p = {};
    const int rc = checked(d, p);
    if (rc != TMW_OK || p.rows == 0) return rc;
    if (p.logprobs == nullptr || (p.top > 0 && (p.top_ids == nullptr || p.top_logprobs == nullptr))) return TMW_ERR_INVALID_ARGUMENT;
    p.status = device_status_word();
    if (p.status == nullptr) return TMW_ERR_CUDA;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (d->dtype == TMW_F32) return launch_forward<float>(p, s);
    return d->dtype == TMW_BF16 ? launch_forward<__nv_bfloat16>(p, s) : launch_forward<__half>(p, s);
}

extern "C" int tmw_token_logprobs_backward(const tmw_logprobs_desc* d, const float* d_logprobs, const float* d_entropy,
                                           const float* d_top, void* d_logits, const int64_t d_stride[2], void* stream) {
    using namespace tmw;
    LogprobsBackward p = {};
    const int rc = checked(d, p.f);
    if (rc != TMW_OK || p.f.rows == 0) return rc;
    if (p.f.lse == nullptr || d_logits == nullptr || d_logits == d->logits || d_stride == nullptr || d_stride[0] < 0 || d_stride[1] < 0 ||
        (d_stride[0] == 0 && d->batch > 1) || (d_stride[1] == 0 && d->tokens > 1) ||
        (d_top != nullptr && p.f.top > 0 && p.f.top_ids == nullptr) || reinterpret_cast<uintptr_t>(d_logits) % dtype_size(d->dtype) != 0)
        return TMW_ERR_INVALID_ARGUMENT;
    p.d_logprobs = d_logprobs;
    p.d_entropy = d_entropy;
    p.d_top = d_top;
    p.d_logits = d_logits;
    p.stride[0] = d_stride[0];
    p.stride[1] = d_stride[1];
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (d->dtype == TMW_F32) return launch_backward<float>(p, s);
    return d->dtype == TMW_BF16 ? launch_backward<__nv_bfloat16>(p, s) : launch_backward<__half>(p, s);
}
