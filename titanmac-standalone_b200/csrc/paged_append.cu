// New tokens into a paged cache (tmw_paged_append): keys, turned by their positions, and values to their slots, queries turned
// into a buffer of their own.
//
// A pair (a, b) of a head's numbers at token t turns by the angle x = t f: (a cos x - b sin x, b cos x + a sin x).  All heads of
// a token share their angles, so a CTA takes a few tokens of one sequence with every head of theirs: it computes the sines once
// into shared memory and looks the tokens' places up, then its threads go over the heads two 16-byte vectors at a time - the two
// that hold both ends of their pairs.  t f goes through 64 bits: in fp32 the angle of token 100,000 would be off by 0.004.
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
    FastDiv units, slots;  // vector pairs of a head; heads of a token, queries' first
    int* status;
};

constexpr int kAppendThreads = 256;
constexpr int kAppendTokens = 4;   // tokens of a CTA
constexpr int kAppendAhead = 2;    // vector pairs that a thread loads before it stores the first

template <typename T, int E>
struct alignas(sizeof(T) * E) Pack {
    T x[E];
};

// E: elements of a vector, 16 bytes or (rows at any address, pairs that fit no vector) one element
template <typename T, int E, bool INTERLEAVED>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const PagedAppend p) {
    extern __shared__ float2 turn[];  // [token][half] cosine and sine
    __shared__ long long place[kAppendTokens];
    const int b = blockIdx.y, r0 = blockIdx.x * kAppendTokens, tid = threadIdx.x;
    const int start = p.start[b];
    int count = p.counts != nullptr ? p.counts[b] : p.rows;
    if (start == -1) return;
    if (start < -1 || count < 0 || count > p.rows) {  // the sequence has no place: every row that it may have is NaN
        count = start < -1 && count >= 0 && count <= p.rows ? count : p.rows;
        if (tid < kAppendTokens) place[tid] = -1;
        if (tid == 0) atomicCAS(p.status, 0, (int)TMW_ERR_INVALID_ARGUMENT);
    } else if (tid < kAppendTokens && r0 + tid < count) {
        const long long t = (long long)start + r0 + tid;
        const long long at = t < p.map.capacity ? p.map.token(b, (int)t) : -1;
        if (at < 0) atomicCAS(p.status, 0, (int)TMW_ERR_INVALID_ARGUMENT);
        place[tid] = at;
    }
    const int tokens = min(kAppendTokens, count - r0);
    if (tokens <= 0) return;
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

    using V = Pack<T, E>;
    const int n = tokens * (int)(p.units.d * p.slots.d);
    for (int first = tid; first < n; first += kAppendThreads * kAppendAhead) {
        V va[kAppendAhead], vb[kAppendAhead];
        T* to[kAppendAhead];
        int ia[kAppendAhead], ib[kAppendAhead], row[kAppendAhead], kind[kAppendAhead];  // kind: 0 query, 1 key, 2 value
#pragma unroll
        for (int j = 0; j < kAppendAhead; ++j) {
            const int i = first + j * kAppendThreads;
            to[j] = nullptr;
            if (i >= n) continue;
            const int head = (int)p.units.div(i), u = i - head * (int)p.units.d;
            const int r = (int)p.slots.div(head);
            int slot = head - r * (int)p.slots.d;
            row[j] = r;
            // the pair of vectors: rotated halves face each other, everything else lies side by side
            const int facing = INTERLEAVED && E > 1 ? 0 : p.half / E;
            if (INTERLEAVED && E == 1) ia[j] = 2 * u, ib[j] = 2 * u + 1;
            else if (u < facing) ia[j] = u * E, ib[j] = u * E + p.half;
            else ia[j] = 2 * u * E, ib[j] = (2 * u + 1) * E;
            const T* from;
            const long long at = place[r];
            if (slot < p.heads) {
                kind[j] = 0;
                from = static_cast<const T*>(p.q) + b * p.qs[0] + slot * p.qs[1] + (r0 + r) * p.qs[2];
                to[j] = static_cast<T*>(p.q_out) + b * p.os[0] + slot * p.os[1] + (r0 + r) * p.os[2];
            } else {
                if (at < 0) continue;
                slot -= p.heads;
                const bool value = slot >= p.map.kv_heads;
                if (value) slot -= p.map.kv_heads;
                kind[j] = value ? 2 : 1;
                const long long* s = value ? p.vs : p.ks;
                from = static_cast<const T*>(value ? p.v : p.k) + b * s[0] + slot * s[1] + (r0 + r) * s[2];
                to[j] = static_cast<T*>(value ? p.v_pages : p.k_pages) + at + slot * p.map.head_step();
            }
            va[j] = *reinterpret_cast<const V*>(from + ia[j]);
            vb[j] = *reinterpret_cast<const V*>(from + ib[j]);
        }
#pragma unroll
        for (int j = 0; j < kAppendAhead; ++j) {
            if (to[j] == nullptr) continue;
            const float2* t = turn + row[j] * p.half;
            if (kind[j] == 0 && place[row[j]] < 0) {
#pragma unroll
                for (int e = 0; e < E; ++e) va[j].x[e] = vb[j].x[e] = from_f32<T>(__int_as_float(0x7fffffff));
            } else if (kind[j] != 2) {
                if (INTERLEAVED && E > 1) {
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        V& v = w ? vb[j] : va[j];
                        const int at = w ? ib[j] : ia[j];
                        if (at < 2 * p.half) {
#pragma unroll
                            for (int e = 0; e + 1 < E; e += 2) {
                                const float2 cs = t[(at + e) / 2];
                                const float x = to_f32<T>(v.x[e]), y = to_f32<T>(v.x[e + 1]);
                                v.x[e] = from_f32<T>(x * cs.x - y * cs.y);
                                v.x[e + 1] = from_f32<T>(y * cs.x + x * cs.y);
                            }
                        }
                    }
                } else if ((INTERLEAVED ? ia[j] / 2 : ia[j]) < p.half && ib[j] < 2 * p.half) {
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const float2 cs = t[(INTERLEAVED ? ia[j] / 2 : ia[j]) + e];
                        const float x = to_f32<T>(va[j].x[e]), y = to_f32<T>(vb[j].x[e]);
                        va[j].x[e] = from_f32<T>(x * cs.x - y * cs.y);
                        vb[j].x[e] = from_f32<T>(y * cs.x + x * cs.y);
                    }
                }
            }
            *reinterpret_cast<V*>(to[j] + ia[j]) = va[j];
            *reinterpret_cast<V*>(to[j] + ib[j]) = vb[j];
        }
    }
}

template <typename T, int E>
int launch_append(PagedAppend& p, bool interleaved, int batch, cudaStream_t stream) {
    p.units = FastDiv((uint32_t)(p.map.head_dim / (2 * E)));
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
    p.slots = FastDiv((uint32_t)(d->heads + 2 * d->at.kv_heads));
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
