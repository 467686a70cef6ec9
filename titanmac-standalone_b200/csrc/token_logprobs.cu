// Log-probabilities of given tokens, entropy and the most likely ids of rows of logits (tmw_token_logprobs), and the gradient.
//
// With M the largest logit of a row and S = sum e^(x - M): log p_i = (x_i - M) - ln S, and the entropy
// H = ln S - (1 / S) sum e^(x - M) (x - M).  The subtractions come first: ln S + M rounded together would cost what the logits
// have in front of their differences.  One pass: every thread keeps the largest of its logits, and S and the other sum under it.
// The gradient, for the gradients g of log p_t, h of H and a_j of the log-probability of the j-th likely id i_j:
//   dx_i = g [i = t] + sum_j a_j [i = i_j] - p_i (g + sum_j a_j + h (log p_i + H)).
// Both are bound by HBM: the logits once, and once more with their gradient on the way back.
//
// The most likely ids, the lower one first among equals: the k best of a row lie with the k threads whose own best are the k best
// of all threads' (any other thread's logits have k ahead of them).  So the threads' bests, of which the pass has kept value and
// vector, are ranked first, and then only those k threads' logits are looked at again (from L2).  Ranking is merging of sorted
// lists of 32, one key to a lane: (value, index) in 64 bits, so there are no equals and no order of arrival.
//
// A row goes to a CTA, or, where there are few, to a cluster of them that joins through distributed shared memory.
#include <cooperative_groups.h>
#include <float.h>
#include <math_constants.h>

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

// ---- ranking ------------------------------------------------------------------------------------------------------------------
// value in the high word, in an order that unsigned numbers have; the complement of the index in the low one; 0: none
__device__ __forceinline__ uint64_t key_of(float x, uint32_t index) {
    const uint32_t bits = __float_as_uint(x + 0.0f);  // (-0 is 0)
    const uint32_t order = bits & 0x80000000u ? ~bits : bits | 0x80000000u;
    return (uint64_t)order << 32 | (uint32_t)~index;
}
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
// The 32 largest of n lists in shared memory (n a power of two, at most the CTA's warps times two), in the first one.  All threads.
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
// (a difference of -inf weighs nothing: the bound keeps infinity times zero out)
__device__ __forceinline__ float bounded(float d) { return fmaxf(d, -1e30f); }
__device__ __forceinline__ Sums joined(const Sums& a, const Sums& b) {
    Sums r;
    r.m = fmaxf(a.m, b.m);
    const float da = (a.m - r.m) * kLog2e, db = (b.m - r.m) * kLog2e, wa = exp2f(da), wb = exp2f(db);
    r.s = wa * a.s + wb * b.s;
    r.t = wa * (a.t + bounded(da) * a.s) + wb * (b.t + bounded(db) * b.s);
    return r;
}

template <typename T, int W>
__global__ void __launch_bounds__(W * 32) logprobs_kernel(const __grid_constant__ Logprobs p, int ctas) {
    constexpr int THREADS = W * 32, E = RowView<T>::E, AHEAD = 4, LISTS = W > 8 ? W : 8;
    __shared__ Sums warp_sums[W];
    __shared__ Sums part;                // this CTA's
    __shared__ uint64_t lists[LISTS][32];
    __shared__ Sums whole_row;
    namespace cg = cooperative_groups;
    const int row = blockIdx.x / ctas, rank = blockIdx.x - row * ctas, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const RowView<T> x(row_of(p, row, sizeof(T)), p.vocab);
    const int per = (x.vectors + ctas - 1) / ctas, v_first = min(rank * per, x.vectors), v_end = min(v_first + per, x.vectors);

    // best: this thread's largest logit, best_at: the first vector that has it
    float best = -CUDART_INF_F, base = -FLT_MAX, s = 0.f, t = 0.f;
    int best_at = -1;
    for (int v0 = v_first + tid; v0 < v_end; v0 += THREADS * AHEAD) {
        uint4 raw[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
            if (v0 + u * THREADS < v_end) raw[u] = x.load(v0 + u * THREADS);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int v = v0 + u * THREADS;
            if (v >= v_end) break;
            float f[E];
            unpack<T>(raw[u], f);
            float top = f[0];
#pragma unroll
            for (int e = 1; e < E; ++e) top = fmaxf(top, f[e]);
            if (top > best || best_at < 0) {
                best = top;
                best_at = v;
                if (top > base) {
                    const float d = (base - top) * kLog2e, w = exp2f(d);
                    t = w * (t + bounded(d) * s);
                    s *= w;
                    base = top;
                }
            }
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float d = (f[e] - base) * kLog2e, w = ex2_ftz(d);
                s += w;
                t = fmaf(w, bounded(d), t);
            }
        }
    }
    Sums mine{base, s, t};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const Sums other{__shfl_xor_sync(0xffffffffu, mine.m, o), __shfl_xor_sync(0xffffffffu, mine.s, o),
                         __shfl_xor_sync(0xffffffffu, mine.t, o)};
        mine = lane & o ? joined(other, mine) : joined(mine, other);  // (the same order on both sides)
    }
    if (lane == 0) warp_sums[warp] = mine;
    __syncthreads();
    if (tid == 0) {
        Sums all = warp_sums[0];
        for (int w = 1; w < W; ++w) all = joined(all, warp_sums[w]);
        part = all;
    }

    if (p.top > 0) {
        // the threads whose best are among the k best: `least` and above
        lists[warp][lane] = sorted(best_at < 0 ? 0 : key_of(best, (uint32_t)best_at * E));
        merge_lists(lists, W);
        const uint64_t least = lists[0][p.top - 1];
        const bool look = best_at >= 0 && key_of(best, (uint32_t)best_at * E) >= least;
        // (the best's own place in its vector is not known: the vector's last one stands for it)
        const uint64_t floor = least == 0 ? 0 : least - (E - 1);
        __syncthreads();
        uint64_t top = 0;
        for (uint32_t todo = __ballot_sync(0xffffffffu, look); todo != 0; todo &= todo - 1) {
            const int from = v_first + warp * 32 + __ffs(todo) - 1;
            for (int v0 = from; v0 < v_end; v0 += 32 * THREADS) {
                const int v = v0 + lane * THREADS;
                float f[E];
                if (v < v_end) unpack<T>(x.load(v), f);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const uint64_t key = v < v_end && x.has(v, e) ? key_of(f[e], (uint32_t)(v * E + e)) : 0;
                    const uint64_t last = __shfl_sync(0xffffffffu, top, p.top - 1);
                    const bool in = key >= floor && key > last;
                    if (__any_sync(0xffffffffu, in)) top = merged(top, sorted(in ? key : 0));
                }
            }
        }
        lists[warp][lane] = top;
        merge_lists(lists, W);
    }
    __syncthreads();

    if (ctas > 1) {  // the first CTA of the cluster takes the others' parts
        auto cluster = cg::this_cluster();
        cluster.sync();
        if (rank == 0) {
            if (tid == 0) {
                Sums all = part;
                for (int c = 1; c < ctas; ++c) all = joined(all, *cluster.map_shared_rank(&part, c));
                whole_row = all;
            }
            uint64_t key = 0;
            if (p.top > 0 && warp < ctas) key = cluster.map_shared_rank(&lists[0][0], warp)[lane];
            __syncthreads();  // (list 0 is this CTA's own)
            if (p.top > 0) {
                if (warp < ctas) lists[warp][lane] = key;
                merge_lists(lists, ctas);
            }
        }
        cluster.sync();
        if (rank != 0) return;
    } else if (tid == 0) {
        whole_row = part;
    }
    __syncthreads();

    const Sums all = whole_row;
    const bool fine = all.s > 0.f;  // (NaN: a NaN or +inf among the logits; 0: nothing but -inf)
    const float log_sum = logf(all.s);
    if (tid == 0) {
        const long long y = p.targets[row];
        float lp = CUDART_NAN_F;
        if (y == kNoTarget) lp = 0.f;
        else if (y < 0 || y >= p.vocab) atomicCAS(p.status, 0, (int)TMW_ERR_INVALID_ARGUMENT);
        else if (fine) lp = (to_f32<T>(x.x[y]) - all.m) - log_sum;
        p.logprobs[row] = lp;
        p.entropy[row] = fine ? log_sum - kLn2 * (all.t / all.s) : CUDART_NAN_F;
        if (p.lse != nullptr) {
            p.lse[2LL * row] = fine ? all.m : CUDART_NAN_F;
            p.lse[2LL * row + 1] = fine ? log_sum : CUDART_NAN_F;
        }
    }
    if (tid < p.top) {
        const long long at = (long long)row * p.top + tid;
        const uint32_t i = index_of(lists[0][tid]) - (uint32_t)x.shift;
        p.top_ids[at] = fine ? (int64_t)i : -1;
        p.top_logprobs[at] = fine ? (to_f32<T>(x.x[i]) - all.m) - log_sum : CUDART_NAN_F;
    }
}

// ---- backward ---------------------------------------------------------------------------------------------------------------------
struct LogprobsBackward {
    Logprobs f;
    const float *d_logprobs, *d_entropy, *d_top;
    void* d_logits;
    long long stride[2];
};

constexpr int kBackThreads = 256, kBackVectors = 8;  // vectors of a thread

// VEC: whole vectors; else (logits and gradient begin at different places of their vectors) one element at a time
template <typename T, bool VEC>
__global__ void __launch_bounds__(kBackThreads) logprobs_backward_kernel(const __grid_constant__ LogprobsBackward p) {
    constexpr int E = VEC ? RowView<T>::E : 1;
    const int row = blockIdx.x, tid = threadIdx.x;
    const RowView<T> x(row_of(p.f, row, sizeof(T)), p.f.vocab);
    const int b = row / p.f.tokens;
    T* d = static_cast<T*>(p.d_logits) + b * p.stride[0] + (row - b * p.f.tokens) * p.stride[1];
    const float m = p.f.lse[2LL * row], log_sum = p.f.lse[2LL * row + 1], entropy = p.f.entropy[row];
    const long long y = p.f.targets[row];
    const float h = p.d_entropy != nullptr ? p.d_entropy[row] : 0.f;
    float g = p.d_logprobs != nullptr && y != kNoTarget ? p.d_logprobs[row] : 0.f;
    if (y != kNoTarget && (y < 0 || y >= p.f.vocab)) g = CUDART_NAN_F;
    float pulled = g;
    const int top = p.d_top != nullptr ? p.f.top : 0;
    for (int j = 0; j < top; ++j) pulled += p.d_top[(long long)row * top + j];
    const float at_zero = pulled + h * entropy;  // - dx_i / p_i = pulled + h (log p_i + H)
    // nothing comes back to the row: nothing goes on, whatever its logits are
    const bool none = g == 0.f && h == 0.f && pulled == 0.f;
    auto gradient = [&](float v) {
        if (none) return 0.f;
        const float lp = (v - m) - log_sum;
        return -exp2f(lp * kLog2e) * fmaf(h, fmaxf(lp, -200.f), at_zero);  // (e^-200 is zero: the bound keeps infinity out)
    };

    const int shift = VEC ? x.shift : 0, n = VEC ? x.vectors : p.f.vocab;
    const int first = blockIdx.y * (kBackThreads * kBackVectors), end = min(first + kBackThreads * kBackVectors, n);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        constexpr int AHEAD = kBackVectors / 2;
        uint4 raw[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int v = first + tid + (half * AHEAD + u) * kBackThreads;
            if (v >= end) continue;
            if (VEC) raw[u] = x.load(v);
            else *reinterpret_cast<T*>(&raw[u]) = x.x[v];
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int v = first + tid + (half * AHEAD + u) * kBackThreads;
            if (v >= end) continue;
            float f[E];
            if constexpr (VEC) unpack<T>(raw[u], f);
            else f[0] = to_f32<T>(*reinterpret_cast<T*>(&raw[u]));
            T out[E];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                float r = gradient(f[e]);
                if (v * E + e - shift == y) r += g;
                out[e] = from_f32<T>(r);
            }
            if (!VEC || x.whole(v)) {
                if constexpr (VEC) *reinterpret_cast<uint4*>(d + (long long)v * E - shift) = *reinterpret_cast<const uint4*>(out);
                else d[v] = out[0];
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (x.has(v, e)) d[v * E + e - shift] = out[e];
            }
        }
    }
    if (top == 0) return;
    __syncthreads();  // the likely ids' own gradients, over what the pass has written
    if (tid < top) {
        const long long id = p.f.top_ids[(long long)row * top + tid];
        if (id < 0 || (id + shift) / E < first || (id + shift) / E >= end) return;
        float r = gradient(to_f32<T>(x.x[id])) + p.d_top[(long long)row * top + tid];
        if (id == y) r += g;
        d[id] = from_f32<T>(r);
    }
}

template <typename T>
int launch_forward(const Logprobs& p, cudaStream_t stream) {
    // Eight warps to a row, four for short ones.  Few rows: clusters, while every thread of them has a vector or more.
    const int vectors = (int)(((long long)p.vocab * sizeof(T) + 15) / 16);
    const bool narrow = vectors <= 512;
    int ctas = 1;
    while (ctas < 8 && (long long)p.rows * ctas * 2 <= 4LL * sm_count() && vectors / (ctas * 2) >= 256) ctas *= 2;
    const dim3 grid((unsigned)p.rows * ctas);
    if (narrow) TMW_CUDA_TRY(launch_ex(logprobs_kernel<T, 4>, grid, dim3(128), 0, stream, false, ctas, p, ctas));
    else TMW_CUDA_TRY(launch_ex(logprobs_kernel<T, 8>, grid, dim3(256), 0, stream, false, ctas, p, ctas));
    return TMW_OK;
}

template <typename T>
int launch_backward(const LogprobsBackward& p, cudaStream_t stream) {
    constexpr int E = RowView<T>::E;
    const bool vec = (reinterpret_cast<uintptr_t>(p.f.logits) - reinterpret_cast<uintptr_t>(p.d_logits)) % 16 == 0 &&
                     (p.f.stride[0] - p.stride[0]) % E == 0 && (p.f.stride[1] - p.stride[1]) % E == 0;
    const long long n = vec ? ((long long)p.f.vocab + 2 * E - 2) / E : p.f.vocab;
    const dim3 grid((unsigned)p.f.rows, (unsigned)((n + kBackThreads * kBackVectors - 1) / (kBackThreads * kBackVectors)));
    if (vec) logprobs_backward_kernel<T, true><<<grid, kBackThreads, 0, stream>>>(p);
    else logprobs_backward_kernel<T, false><<<grid, kBackThreads, 0, stream>>>(p);
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
