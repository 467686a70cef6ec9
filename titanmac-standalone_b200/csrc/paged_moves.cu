// Tokens out of their pages and from place to place in them: tmw_paged_read, tmw_paged_keep.
//
// Both move bytes: bound by HBM, or for a few tokens by launch and latency (reading 21600 tokens of 16 heads of 128 from e4m3 in bf16,
// 250 MB, takes 48 us cold, 5.2 TB/s; one row after the other in a thread, eight numbers of it, 62).
#include "paged.cuh"

namespace tmw {
namespace {

constexpr int kThreads = 256;

struct PagedRead {
    PageMap map;
    const void *k_pages, *v_pages;
    const float *k_scales, *v_scales;
    void *k, *v;
    long long ks[3], vs[3];  // {batch, head, row}
    const int32_t *start, *counts;
    int rows;
    int* status;
};

// A CTA has kReadTokens tokens of a sequence, all heads of theirs; a thread sixteen bytes of a row of a page at a time, at the same
// place of every row it has, two rows under way.
constexpr int kReadTokens = 16, kReadAhead = 2;
template <typename T, typename P, bool WHOLE>
__global__ void __launch_bounds__(kThreads, 6) paged_read_kernel(const __grid_constant__ PagedRead p) {
    __shared__ long long place[kReadTokens];
    constexpr int kOne = 16 / sizeof(P);
    const int b = blockIdx.y, r0 = blockIdx.x * kReadTokens, tid = threadIdx.x;
    const int start = p.start[b];
    int count = p.counts != nullptr ? p.counts[b] : p.rows;
    if (start == -1) return;
    const bool nowhere = start < -1 || count < 0 || count > p.rows;
    if (count < 0 || count > p.rows) count = p.rows;
    const int tokens = min(kReadTokens, count - r0);
    if (tokens <= 0) return;
    if (tid < tokens) {
        const long long t = (long long)start + r0 + tid;
        const long long at = !nowhere && t < p.map.capacity ? p.map.row(b, (int)t) : -1;
        if (at < 0) atomicCAS(p.status, 0, (int)TMW_ERR_INVALID_ARGUMENT);
        place[tid] = at;
    }
    const int units = p.map.head_dim / kOne, slots = 2 * p.map.kv_heads, step = kThreads / units;
    const int step_r = step / slots, step_slot = step - step_r * slots;
    const int row = tid / units, d = (tid - row * units) * kOne;
    int r = row < step ? row / slots : tokens, slot = row % slots;  // (threads behind the last whole row have none)
    __syncthreads();
    while (r < tokens) {
        uint4 w[kReadAhead];
        float scale[kReadAhead];
        T* to[kReadAhead];  // NULL: no row
        bool there[kReadAhead];
#pragma unroll
        for (int i = 0; i < kReadAhead; ++i) {
            to[i] = nullptr;
            there[i] = false;
            if (r < tokens) {
                const bool value = slot >= p.map.kv_heads;
                const int head = value ? slot - p.map.kv_heads : slot;
                to[i] = value ? static_cast<T*>(p.v) + b * p.vs[0] + head * p.vs[1] + (r0 + r) * p.vs[2] + d
                              : static_cast<T*>(p.k) + b * p.ks[0] + head * p.ks[1] + (r0 + r) * p.ks[2] + d;
                there[i] = place[r] >= 0;
                if (there[i]) {
                    const long long at = place[r] + (long long)head * p.map.page.d;
                    w[i] = *reinterpret_cast<const uint4*>(static_cast<const P*>(value ? p.v_pages : p.k_pages) + at * p.map.head_dim + d);
                    if constexpr (sizeof(P) == 1) scale[i] = (value ? p.v_scales : p.k_scales)[at];
                }
                r += step_r;
                slot += step_slot;
                if (slot >= slots) slot -= slots, ++r;
            }
        }
#pragma unroll
        for (int i = 0; i < kReadAhead; ++i) {
            if (to[i] == nullptr) continue;
            alignas(16) T x[kOne];
            if (!there[i]) {
#pragma unroll
                for (int e = 0; e < kOne; ++e) x[e] = from_f32<T>(__int_as_float(0x7fffffff));
            } else if constexpr (sizeof(P) == 1) {
                const uint32_t codes[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint32_t two = codes[e / 2] >> e % 2 * 16;
                    float2 c;
                    if constexpr (std::is_same<P, E4m3>::value) c = __half22float2(from_e4m3(two));
                    else c = make_float2((float)(int8_t)two, (float)(int8_t)(two >> 8));
                    x[2 * e] = from_f32<T>(c.x * scale[i]);
                    x[2 * e + 1] = from_f32<T>(c.y * scale[i]);
                }
            } else {
                *reinterpret_cast<uint4*>(x) = w[i];
            }
            if constexpr (WHOLE) {
#pragma unroll
                for (int e = 0; e < (int)sizeof(x) / 16; ++e) reinterpret_cast<uint4*>(to[i])[e] = reinterpret_cast<const uint4*>(x)[e];
            } else {
#pragma unroll
                for (int e = 0; e < kOne; ++e) to[i][e] = x[e];
            }
        }
    }
}

template <typename T>
int launch_read(const PagedRead& p, int format, int batch, bool whole, cudaStream_t stream) {
    const dim3 grid((unsigned)((p.rows + kReadTokens - 1) / kReadTokens), (unsigned)batch);
    auto with = [&](auto page) {
        using P = decltype(page);
        if (whole) paged_read_kernel<T, P, true><<<grid, kThreads, 0, stream>>>(p);
        else paged_read_kernel<T, P, false><<<grid, kThreads, 0, stream>>>(p);
    };
    if (format == TMW_PAGES_INT8) with(int8_t{});
    else if (format == TMW_PAGES_E4M3) with(E4m3{});
    else with(T{});
    TMW_CUDA_TRY(cudaGetLastError());
    return TMW_OK;
}

constexpr int kMostKept = 64;
struct PagedKeep {
    PageMap map;
    unsigned char *k_pages, *v_pages;
    float *k_scales, *v_scales;  // NULL: none
    const int32_t *start, *kept, *counts;
    int rows, vectors, heads;  // vectors: of 16 bytes, in a row; heads: of a CTA
    int* status;
};

// A CTA has keys and values of some heads of a sequence, as many as its threads can have under way at once, or of one: every CTA looks the tokens'
// places up first, four loads one after the other, so that fewer CTAs are faster (256 sequences, 6 of 32 tokens, 10 heads of 64: keys and
// values of every head apart 18.3 us, so 5.8).  Tokens come from further back than they go to, in the order of both,
// so a batch of them is read, and when every thread has its part, written: no later token of its head has been written over by then.
constexpr int kKeepAhead = 4;
__global__ void __launch_bounds__(kThreads) paged_keep_kernel(const __grid_constant__ PagedKeep p) {
    __shared__ long long from[kMostKept], to[kMostKept];
    const int b = blockIdx.y, tid = threadIdx.x, head0 = blockIdx.x * p.heads, heads = min(p.heads, p.map.kv_heads - head0);
    const int start = p.start[b], count = p.counts[b];
    if (start == -1) return;
    bool bad = start < -1 || count < 0 || count > p.rows;
    if (!bad && tid < count) {
        const int32_t* kept = p.kept + (long long)b * p.rows;
        const int j = kept[tid];
        bad = j < tid || (tid > 0 && j <= kept[tid - 1]) || (long long)start + j >= p.map.capacity;
        if (!bad) {
            const long long source = p.map.row(b, start + j), target = p.map.row(b, start + tid);
            bad = source < 0 || target < 0;
            from[tid] = source;
            to[tid] = target;
        }
    }
    if (__syncthreads_or(bad)) {
        if (tid == 0) atomicCAS(p.status, 0, (int)TMW_ERR_INVALID_ARGUMENT);
        return;
    }
    // rows, in this order: [keys, values][head][token]
    const int rows = 2 * heads * count, n = rows * p.vectors;
    const auto row_at = [&](int row, int& t, bool& value) {  // (its head's first row of page 0)
        const int of = row / count;
        t = row - of * count;
        value = of >= heads;
        return (long long)(head0 + of - (value ? heads : 0)) * p.map.page.d;
    };
    float scale[kKeepAhead];  // (no more rows than that: several heads have so many vectors at most, one has 128 rows)
    if (p.k_scales != nullptr) {
#pragma unroll
        for (int a = 0; a < kKeepAhead; ++a) {
            const int row = a * kThreads + tid;
            if (row >= rows) continue;
            int t;
            bool value;
            const long long at = row_at(row, t, value);
            scale[a] = (value ? p.v_scales : p.k_scales)[at + from[t]];
        }
    }
    for (int i0 = 0; i0 < n; i0 += kThreads * kKeepAhead) {
        uint4 x[kKeepAhead], *target[kKeepAhead];
#pragma unroll
        for (int a = 0; a < kKeepAhead; ++a) {
            const int i = i0 + a * kThreads + tid, row = i / p.vectors;
            target[a] = nullptr;
            if (i >= n) continue;
            int t;
            bool value;
            const long long at = row_at(row, t, value);
            if (from[t] == to[t]) continue;
            uint4* pages = reinterpret_cast<uint4*>(value ? p.v_pages : p.k_pages) + (i - row * p.vectors);
            x[a] = pages[(at + from[t]) * p.vectors];
            target[a] = pages + (at + to[t]) * p.vectors;
        }
        __syncthreads();
#pragma unroll
        for (int a = 0; a < kKeepAhead; ++a)
            if (target[a] != nullptr) *target[a] = x[a];
    }
    if (p.k_scales != nullptr) {  // (read before the barrier)
#pragma unroll
        for (int a = 0; a < kKeepAhead; ++a) {
            const int row = a * kThreads + tid;
            if (row >= rows) continue;
            int t;
            bool value;
            const long long at = row_at(row, t, value);
            (value ? p.v_scales : p.k_scales)[at + to[t]] = scale[a];
        }
    }
}

}  // namespace
}  // namespace tmw

extern "C" int tmw_paged_read(const tmw_paged_read_desc* d, const tmw_page_scales* scales, void* stream) {
    using namespace tmw;
    if (d == nullptr) return TMW_ERR_INVALID_ARGUMENT;
    const bool used = d->at.batch > 0 && d->rows > 0;
    int rc = validate_pages(d->at, used);
    if (rc != TMW_OK) return rc;
    const tmw_page_scales s = scales != nullptr ? *scales : tmw_page_scales{};
    rc = validate_scales(d->at, s, used, false);
    if (rc != TMW_OK) return rc;
    if (d->rows < 0) return TMW_ERR_INVALID_ARGUMENT;
    if (!used) return TMW_OK;
    if (d->k == nullptr || d->v == nullptr || d->start == nullptr) return TMW_ERR_INVALID_ARGUMENT;
    const size_t size = dtype_size(d->at.dtype);
    const uintptr_t bits = reinterpret_cast<uintptr_t>(d->k) | reinterpret_cast<uintptr_t>(d->v);
    long long strides = 0;
    for (int i = 0; i < 3; ++i) {
        if (d->k_stride[i] < 0 || d->v_stride[i] < 0) return TMW_ERR_INVALID_ARGUMENT;
        strides |= d->k_stride[i] | d->v_stride[i];
    }
    if (bits % size != 0) return TMW_ERR_INVALID_ARGUMENT;
    if (d->k == d->v || !rows_apart(d->k_stride, {d->at.batch, d->at.kv_heads, d->rows}) ||
        !rows_apart(d->v_stride, {d->at.batch, d->at.kv_heads, d->rows})) {
        set_error_text("tmw_paged_read: every output must have a place of its own");
        return TMW_ERR_INVALID_ARGUMENT;
    }
    PagedRead p = {};
    p.map = PageMap(d->at);
    p.k_pages = d->at.k_pages; p.v_pages = d->at.v_pages;
    p.k_scales = s.k_scales; p.v_scales = s.v_scales;
    p.k = d->k; p.v = d->v;
    for (int i = 0; i < 3; ++i) {
        p.ks[i] = d->k_stride[i];
        p.vs[i] = d->v_stride[i];
    }
    p.start = d->start; p.counts = d->counts;
    p.rows = d->rows;
    p.status = device_status_word();
    if (p.status == nullptr) return TMW_ERR_CUDA;
    const bool whole = bits % 16 == 0 && strides % (16 / (long long)size) == 0;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (d->at.dtype == TMW_F32) return launch_read<float>(p, s.format, d->at.batch, whole, st);
    return d->at.dtype == TMW_BF16 ? launch_read<__nv_bfloat16>(p, s.format, d->at.batch, whole, st)
                                   : launch_read<__half>(p, s.format, d->at.batch, whole, st);
}

extern "C" int tmw_paged_keep(const tmw_paged_keep_desc* d, const tmw_page_scales* scales, void* stream) {
    using namespace tmw;
    if (d == nullptr) return TMW_ERR_INVALID_ARGUMENT;
    const bool used = d->at.batch > 0 && d->rows > 0;
    int rc = validate_pages(d->at, used);
    if (rc != TMW_OK) return rc;
    const tmw_page_scales s = scales != nullptr ? *scales : tmw_page_scales{};
    rc = validate_scales(d->at, s, used, false);
    if (rc != TMW_OK) return rc;
    if (d->rows < 0) return TMW_ERR_INVALID_ARGUMENT;
    if (d->rows > kMostKept) {
        set_error_text("tmw_paged_keep: at most 64 tokens of a sequence");
        return TMW_ERR_TOO_LARGE;
    }
    if (!used) return TMW_OK;
    if (d->start == nullptr || d->kept == nullptr || d->counts == nullptr) return TMW_ERR_INVALID_ARGUMENT;
    PagedKeep p = {};
    p.map = PageMap(d->at);
    p.k_pages = static_cast<unsigned char*>(d->at.k_pages); p.v_pages = static_cast<unsigned char*>(d->at.v_pages);
    if (s.format != TMW_PAGES_SAME) p.k_scales = s.k_scales, p.v_scales = s.v_scales;
    p.start = d->start; p.kept = d->kept; p.counts = d->counts;
    p.rows = d->rows;
    const int bytes = d->at.head_dim * (s.format == TMW_PAGES_SAME ? (int)dtype_size(d->at.dtype) : 1);
    p.vectors = bytes / 16;  // (head_dim is a multiple of 8, of 16 in 8 bits)
    p.status = device_status_word();
    if (p.status == nullptr) return TMW_ERR_CUDA;
    p.heads = max(1, min(d->at.kv_heads, kThreads * kKeepAhead / (2 * d->rows * p.vectors)));
    const dim3 grid((unsigned)((d->at.kv_heads + p.heads - 1) / p.heads), (unsigned)d->at.batch);
    paged_keep_kernel<<<grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
    TMW_CUDA_TRY(cudaGetLastError());
    return TMW_OK;
}
