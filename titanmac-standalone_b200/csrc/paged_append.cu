// New tokens into a paged cache (tmw_paged_append): keys, turned by their positions, and values to their slots, queries turned
// into a buffer of their own.
//
// A pair (a, b) of a head's numbers at token t turns by the angle x = t f: (a cos x - b sin x, b cos x + a sin x).  All heads of
// a token share their angles, so a CTA takes a few tokens of one sequence with every head of theirs: it computes the sines once
// into shared memory and looks the tokens' places up, then its threads go over the heads two 16-byte vectors at a time - the two
// that hold both ends of their pairs, the next two on their way under them (with four on their way half as many warps find room:
// 8 prompts, 453 MB in and out, 111 us against 80; nothing on its way 92).  Bound by HBM, 5.7 TB/s there; a decode step by its launch
// (64 tokens: 5.2 us).  t f goes through 64 bits: in fp32 the angle of token 100,000 would be off by 0.004.
#include "paged.cuh"

namespace tmw {
namespace {

struct PagedAppend {
    PageMap map;
    const void *k, *v, *q;
    void *k_pages, *v_pages, *q_out;
    long long ks[3], vs[3], qs[3], os[3];  // {batch, head, row}
    const int32_t *start, *counts;
    const float* inv_freq;
    int rows, heads, half;
    int step_r, step_slot, step_u;  // from a thread's pair of vectors to its next one: tokens, heads, pairs
    int* status;
};

constexpr int kAppendThreads = 256;
constexpr int kAppendTokens = 4;  // tokens of a CTA

template <typename T, int E>
struct alignas(sizeof(T) * E) Pack {
    T x[E];
};

// x c + y s, in one way for every layout: the same bits wherever a row begins
__device__ __forceinline__ float turned(float x, float y, float c, float s) { return fmaf(x, c, __fmul_rn(y, s)); }

// E: elements of a vector, 16 bytes or (rows at any address, pairs that fit no vector) one element
template <typename T, int E, bool INTERLEAVED>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const __grid_constant__ PagedAppend p) {
    using V = Pack<T, E>;
    extern __shared__ float2 turn[];  // [token][half] cosine and sine
    __shared__ long long place[kAppendTokens];
    const int b = blockIdx.y, r0 = blockIdx.x * kAppendTokens, tid = threadIdx.x;
    const int start = p.start[b];
    int count = p.counts != nullptr ? p.counts[b] : p.rows;
    if (start == -1) return;
    const bool nowhere = start < -1 || count < 0 || count > p.rows;  // every row that the sequence may have is NaN
    if (nowhere && (count < 0 || count > p.rows)) count = p.rows;
    const int tokens = min(kAppendTokens, count - r0);
    if (tokens <= 0) return;

    // A pair of vectors of a head of a token; a thread takes every kAppendThreads-th one of the CTA's.
    struct Item {
        int r, slot, u;  // token, head (queries, keys, values), pair of the head
    };
    const int units = p.map.head_dim / (2 * E), slots = p.heads + 2 * p.map.kv_heads;
    auto after = [&](Item w) {
        w.u += p.step_u;
        w.slot += p.step_slot;
        w.r += p.step_r;
        if (w.u >= units) w.u -= units, ++w.slot;
        if (w.slot >= slots) w.slot -= slots, ++w.r;
        return w;
    };
    // first elements of the two: rotated halves face each other, everything else lies side by side
    auto ends = [&](int u, int& ia, int& ib) {
        const bool facing = (!INTERLEAVED || E == 1) && u * E < p.half;
        if (INTERLEAVED && E == 1) ia = 2 * u, ib = 2 * u + 1;
        else if (facing) ia = u * E, ib = u * E + p.half;
        else ia = 2 * u * E, ib = ia + E;
    };
    const T *q = static_cast<const T*>(p.q) + b * p.qs[0] + r0 * p.qs[2], *k = static_cast<const T*>(p.k) + b * p.ks[0] + r0 * p.ks[2],
            *v = static_cast<const T*>(p.v) + b * p.vs[0] + r0 * p.vs[2];
    T* q_out = static_cast<T*>(p.q_out) + b * p.os[0] + r0 * p.os[2];
    auto load = [&](const Item& w, V& va, V& vb) {
        if (w.r >= tokens) return;
        int ia, ib;
        ends(w.u, ia, ib);
        const int of_kv = w.slot - p.heads;
        const T* from;
        if (of_kv < 0) from = q + w.slot * p.qs[1] + w.r * p.qs[2];
        else if (of_kv < p.map.kv_heads) from = k + of_kv * p.ks[1] + w.r * p.ks[2];
        else from = v + (of_kv - p.map.kv_heads) * p.vs[1] + w.r * p.vs[2];
        va = *reinterpret_cast<const V*>(from + ia);
        vb = *reinterpret_cast<const V*>(from + ib);
    };
    auto store = [&](const Item& w, V& va, V& vb) {
        int ia, ib;
        ends(w.u, ia, ib);
        const int of_kv = w.slot - p.heads;
        const bool query = of_kv < 0, value = of_kv >= p.map.kv_heads;
        const long long at = place[w.r];
        T* to;
        if (query) to = q_out + w.slot * p.os[1] + w.r * p.os[2];
        else if (at < 0) return;
        else if (value) to = static_cast<T*>(p.v_pages) + at + (of_kv - p.map.kv_heads) * p.map.head_step();
        else to = static_cast<T*>(p.k_pages) + at + of_kv * p.map.head_step();
        const float2* t = turn + w.r * p.half;
        if (query && at < 0) {
#pragma unroll
            for (int e = 0; e < E; ++e) va.x[e] = vb.x[e] = from_f32<T>(__int_as_float(0x7fffffff));
        } else if (!value && INTERLEAVED && E > 1) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                V& v = h ? vb : va;
                const int first = h ? ib : ia;
                if (first >= 2 * p.half) continue;
#pragma unroll
                for (int e = 0; e + 1 < E; e += 2) {
                    const float2 cs = t[(first + e) / 2];
                    const float x = to_f32<T>(v.x[e]), y = to_f32<T>(v.x[e + 1]);
                    v.x[e] = from_f32<T>(turned(x, y, cs.x, -cs.y));
                    v.x[e + 1] = from_f32<T>(turned(y, x, cs.x, cs.y));
                }
            }
        } else if (!value) {
            const int pair = INTERLEAVED ? ia / 2 : ia;
            if (pair < p.half && ib < 2 * p.half) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float2 cs = t[pair + e];
                    const float x = to_f32<T>(va.x[e]), y = to_f32<T>(vb.x[e]);
                    va.x[e] = from_f32<T>(turned(x, y, cs.x, -cs.y));
                    vb.x[e] = from_f32<T>(turned(y, x, cs.x, cs.y));
                }
            }
        }
        *reinterpret_cast<V*>(to + ia) = va;
        *reinterpret_cast<V*>(to + ib) = vb;
    };

    Item now;
    now.slot = tid / units;
    now.u = tid - now.slot * units;
    now.r = now.slot / slots;
    now.slot -= now.r * slots;
    V va, vb;
    load(now, va, vb);
    // under the first loads: the tokens' places, and their angles
    if (tid < tokens) {
        const long long t = (long long)start + r0 + tid;
        const long long at = !nowhere && t < p.map.capacity ? p.map.token(b, (int)t) : -1;
        if (at < 0) atomicCAS(p.status, 0, (int)TMW_ERR_INVALID_ARGUMENT);
        place[tid] = at;
    }
    for (int i = tid; i < tokens * p.half; i += kAppendThreads) {
        const int r = i / p.half;
        // turns instead of radians: the whole ones fall away exactly
        double x = (double)((long long)start + r0 + r) * (double)p.inv_freq[i - r * p.half] * 0.15915494309189533577;
        x -= rint(x);
        float s, c;
        sincospif(2.0f * (float)x, &s, &c);
        turn[i] = make_float2(c, s);
    }
    __syncthreads();
    while (now.r < tokens) {  // the next pair loads under this one
        const Item next = after(now);
        V na, nb;
        load(next, na, nb);
        store(now, va, vb);
        va = na;
        vb = nb;
        now = next;
    }
}

template <typename T, int E>
int launch_append(PagedAppend& p, bool interleaved, int batch, cudaStream_t stream) {
    const int units = p.map.head_dim / (2 * E), slots = p.heads + 2 * p.map.kv_heads;
    p.step_u = kAppendThreads % units;
    p.step_slot = kAppendThreads / units % slots;
    p.step_r = kAppendThreads / units / slots;
    const dim3 grid((unsigned)((p.rows + kAppendTokens - 1) / kAppendTokens), (unsigned)batch), block(kAppendThreads);
    const int smem = kAppendTokens * p.half * (int)sizeof(float2);
    if (interleaved) paged_append_kernel<T, E, true><<<grid, block, smem, stream>>>(p);
    else paged_append_kernel<T, E, false><<<grid, block, smem, stream>>>(p);
    TMW_CUDA_TRY(cudaGetLastError());
    return TMW_OK;
}

}  // namespace
}  // namespace tmw

extern "C" int tmw_paged_append(const tmw_paged_append_desc* d, void* stream) {
    using namespace tmw;
    if (d == nullptr) return TMW_ERR_INVALID_ARGUMENT;
    const bool used = d->at.batch > 0 && d->rows > 0;
    const int rc = validate_pages(d->at, used);
    if (rc != TMW_OK) return rc;
    if (d->rows < 0 || d->heads < 0 || d->rotated < 0 || d->rotated % 2 != 0 || d->rotated > d->at.head_dim)
        return TMW_ERR_INVALID_ARGUMENT;
    if (!used) return TMW_OK;
    if (d->k == nullptr || d->v == nullptr || d->start == nullptr || (d->rotated > 0 && d->inv_freq == nullptr) ||
        (d->heads > 0 && (d->q == nullptr || d->q_out == nullptr)))
        return TMW_ERR_INVALID_ARGUMENT;
    const size_t size = dtype_size(d->at.dtype);
    const int e = 16 / (int)size;
    uintptr_t bits = 0;     // of every address
    long long strides = 0;  // and stride
    auto add = [&](const void* x, const int64_t* s, bool with) {
        if (!with) return true;
        bits |= reinterpret_cast<uintptr_t>(x);
        for (int i = 0; i < 3; ++i) {
            if (s[i] < 0) return false;
            strides |= s[i];
        }
        return reinterpret_cast<uintptr_t>(x) % size == 0;
    };
    if (!add(d->k, d->k_stride, true) || !add(d->v, d->v_stride, true) || !add(d->q, d->q_stride, d->heads > 0) ||
        !add(d->q_out, d->q_out_stride, d->heads > 0))
        return TMW_ERR_INVALID_ARGUMENT;
    if (d->heads > 65535) return TMW_ERR_TOO_LARGE;
    if (d->heads > 0) {
        const int extents[3] = {d->at.batch, d->heads, d->rows};
        bool same = true;
        for (int i = 0; i < 3; ++i) same = same && (extents[i] == 1 || d->q_stride[i] == d->q_out_stride[i]);
        if ((d->q == d->q_out && !same) || !rows_apart(d->q_out_stride, {d->at.batch, d->heads, d->rows})) {
            set_error_text("tmw_paged_append: q_out must have places of its own, or be q with q's strides");
            return TMW_ERR_INVALID_ARGUMENT;
        }
    }

    PagedAppend p = {};
    p.map = PageMap(d->at);
    p.k = d->k; p.v = d->v; p.q = d->q;
    p.k_pages = d->at.k_pages; p.v_pages = d->at.v_pages; p.q_out = d->q_out;
    for (int i = 0; i < 3; ++i) {
        p.ks[i] = d->k_stride[i];
        p.vs[i] = d->v_stride[i];
        p.qs[i] = d->q_stride[i];
        p.os[i] = d->q_out_stride[i];
    }
    p.start = d->start; p.counts = d->counts; p.inv_freq = d->inv_freq;
    p.rows = d->rows; p.heads = d->heads; p.half = d->rotated / 2;
    p.status = device_status_word();
    if (p.status == nullptr) return TMW_ERR_CUDA;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    // Whole vectors where every row begins on 16 bytes and no pair is cut; single elements otherwise.
    const bool whole = bits % 16 == 0 && strides % e == 0 && d->at.head_dim % (2 * e) == 0 &&
                       (d->interleaved ? d->rotated : d->rotated / 2) % e == 0;
    const bool il = d->interleaved != 0;
    if (d->at.dtype == TMW_F32) return whole ? launch_append<float, 4>(p, il, d->at.batch, s) : launch_append<float, 1>(p, il, d->at.batch, s);
    if (d->at.dtype == TMW_BF16)
        return whole ? launch_append<__nv_bfloat16, 8>(p, il, d->at.batch, s) : launch_append<__nv_bfloat16, 1>(p, il, d->at.batch, s);
    return whole ? launch_append<__half, 8>(p, il, d->at.batch, s) : launch_append<__half, 1>(p, il, d->at.batch, s);
}
