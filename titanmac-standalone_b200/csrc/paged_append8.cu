// New tokens into pages of 8-bit numbers (tmw_paged_append_scaled): keys, turned by their positions, and values as codes with a scale
// for each row, queries turned into a buffer of their own.
//
// scale = max |x| / largest, code = the nearest one to x / scale.  A row's numbers are spread over up to sixteen lanes, sixteen each - eight
// pairs that turn together -, and its largest is found by shuffles, so a row is read once and written once.  The sines are
// computed once for a CTA's tokens, as in the append to wider pages.
//
// A byte read or written here costs more instructions than in the append to wider pages: 77 million for 21600 tokens of 16 heads of 128
// each of queries, keys and values, bf16 into e4m3, which take 93 us (80 % of what can be issued; their 415 MB alone 63 us).
#include "paged_append.cuh"

namespace tmw {
namespace {

constexpr int kThreads = 256;
constexpr int kTokens = 8;  // of a CTA

template <typename P>
constexpr float kLargest = 127.f;
template <>
constexpr float kLargest<E4m3> = 448.f;
constexpr float kLeastScale = 0x1p-100f;

// x / scale, but where that lies between two numbers one of them that is odd in its last place: no border between codes is, so the
// code nearest to it is the one nearest to the quotient, whatever a rounded quotient would have done (half a row's largest number,
// for one, lies on a border).  A quotient that is one number stays.
__device__ __forceinline__ float quotient(float x, float scale, float inverse) {
    float t = x * inverse;
    t = fmaf(fmaf(-t, scale, x), inverse, t);
    const float rest = fmaf(-t, scale, x);
    int bits = __float_as_int(t);
    if (rest != 0.f && t != 0.f && (bits & 1) == 0) bits += (__float_as_int(rest) ^ bits) >= 0 ? 1 : -1;
    return __int_as_float(bits);
}
template <typename P>
__device__ __forceinline__ uint32_t codes4(const float (&x)[4]);
template <>
__device__ __forceinline__ uint32_t codes4<int8_t>(const float (&x)[4]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(x[i] + 12582912.f);  // 1.5 2^23: a whole number in the lowest bits
    return __byte_perm(__byte_perm(w[0], w[1], 0x0040), __byte_perm(w[2], w[3], 0x0040), 0x5410);
}
template <>
__device__ __forceinline__ uint32_t codes4<E4m3>(const float (&x)[4]) {
    uint16_t a, b;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(a) : "f"(x[1]), "f"(x[0]));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(b) : "f"(x[3]), "f"(x[2]));
    return a | (uint32_t)b << 16;
}

template <typename T>
__device__ __forceinline__ void store8(T* to, const float* x) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            reinterpret_cast<float4*>(to)[i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same<T, __half>::value) {
                const __half2 two = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
                w[i] = reinterpret_cast<const uint32_t&>(two);
            } else {
                const __nv_bfloat162 two = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
                w[i] = reinterpret_cast<const uint32_t&>(two);
            }
        }
        *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// The codes of sixteen numbers.  Two quotients that enclose the right one, off by 2^-21 on either side (the reciprocal is off by 2^-23, its
// product with 1 -+ 2^-21 and the quotient are each rounded by 2^-24); where both become the same codes these are right, else a
// border is near and quotient() decides.  (Looking at every number's distance to a border instead: 111 us for 99, 21600
// tokens of 16 heads of 128 each of queries, keys and values.)
template <typename P>
__device__ __forceinline__ void codes16(const float (&x)[16], float scale, uint32_t (&codes)[4]) {
    float inverse;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(scale));  // (of 2^-100 to 2^122)
    const float below = inverse * (1.0f - 0x1p-21f), above = inverse * (1.0f + 0x1p-21f);
    uint32_t differ = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float lo[4], hi[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) lo[e] = x[4 * i + e] * below, hi[e] = x[4 * i + e] * above;
        codes[i] = codes4<P>(lo);
        differ |= codes[i] ^ codes4<P>(hi);
    }
    if (differ != 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float t[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) t[e] = quotient(x[4 * i + e], scale, inverse);
            codes[i] = codes4<P>(t);
        }
    }
}

// x cos + y sin, in one way for every layout
__device__ __forceinline__ float turned(float x, float y, float c, float s) { return fmaf(x, c, __fmul_rn(y, s)); }

// A row's lanes keep their place u in it from row to row; the next row's numbers are on their way while this one's are worked on, the
// first one's while the sines are computed.
//
// WHOLE: rows begin on 16 bytes and a lane's two runs of eight numbers are whole vectors; else they are read one by one.
template <typename T, typename P, bool INTERLEAVED, bool WHOLE>
__global__ void __launch_bounds__(kThreads, 4) paged_append8_kernel(const __grid_constant__ PagedAppend p) {
    extern __shared__ float4 turn[];  // cosine and sine of pair 8 u + e of token r: half e % 2 of [(r * 4 + e / 2) * eights + u]
    __shared__ long long place[kTokens];
    const int b = blockIdx.y, r0 = blockIdx.x * kTokens, tid = threadIdx.x;
    const int start = p.start[b];
    int count = p.counts != nullptr ? p.counts[b] : p.rows;
    if (start == -1) return;
    const bool nowhere = start < -1 || count < 0 || count > p.rows;
    if (count < 0 || count > p.rows) count = p.rows;
    const int tokens = min(kTokens, count - r0);
    if (tokens <= 0) return;

    const int units = p.map.head_dim / 16, eights = (p.half + 7) / 8;
    int lanes = 1;  // of a row; the first `units` have a part of it
    while (lanes < units) lanes *= 2;
    const int u = tid & (lanes - 1), slots = p.heads + 2 * p.map.kv_heads, step = kThreads / lanes;
    const int step_r = step / slots, step_slot = step - step_r * slots;
    // the lane's pairs 8 u .. are (ia + e, ib + e), or (ia + 2 e, ia + 2 e + 1) with ib = ia + 8
    const bool facing = !INTERLEAVED && 8 * u < p.half;
    const int ia = facing ? 8 * u : 16 * u, ib = facing ? ia + p.half : ia + 8;
    auto at_pair = [&](int e) {  // pair 8 u + e
        const int j = 8 * u + e;
        return !INTERLEAVED && j < p.half ? make_int2(j, j + p.half) : make_int2(2 * j, 2 * j + 1);
    };
    union Raw {
        uint4 w[16 * sizeof(T) / 16];
        T v[16];  // the lane's first eight numbers, then the others; read one by one: first numbers of its pairs, then second ones
        __device__ Raw() {}
    } raw;
    // (lanes without a part of a row have zeros for its largest number, and do nothing else)
#pragma unroll
    for (int i = 0; i < (int)sizeof(raw) / 16; ++i) raw.w[i] = make_uint4(0, 0, 0, 0);
    auto load = [&](int r, int slot) {
        const int of_kv = slot - p.heads;
        const T* from;
        if (of_kv < 0) from = static_cast<const T*>(p.q) + b * p.qs[0] + slot * p.qs[1] + (r0 + r) * p.qs[2];
        else if (of_kv < p.map.kv_heads) from = static_cast<const T*>(p.k) + b * p.ks[0] + of_kv * p.ks[1] + (r0 + r) * p.ks[2];
        else from = static_cast<const T*>(p.v) + b * p.vs[0] + (of_kv - p.map.kv_heads) * p.vs[1] + (r0 + r) * p.vs[2];
        if constexpr (WHOLE) {
            constexpr int kHalf = 8 * sizeof(T) / 16;
#pragma unroll
            for (int i = 0; i < kHalf; ++i) {
                raw.w[i] = reinterpret_cast<const uint4*>(from + ia)[i];
                raw.w[kHalf + i] = reinterpret_cast<const uint4*>(from + ib)[i];
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int2 at = at_pair(e);
                raw.v[e] = from[at.x];
                raw.v[8 + e] = from[at.y];
            }
        }
    };
    int r = tid / lanes / slots, slot = tid / lanes - r * slots;
    if (r < tokens && u < units) load(r, slot);

    if (tid < tokens) {
        const long long t = (long long)start + r0 + tid;
        const long long at = !nowhere && t < p.map.capacity ? p.map.row(b, (int)t) : -1;
        if (at < 0) atomicCAS(p.status, 0, (int)TMW_ERR_INVALID_ARGUMENT);
        place[tid] = at;
    }
    for (int i = tid; i < tokens * p.half; i += kThreads) {
        const int rr = i / p.half, j = i - rr * p.half;
        const long long t = p.positions != nullptr ? p.positions[(long long)b * p.rows + r0 + rr] : (long long)start + r0 + rr;
        // turns instead of radians: the whole ones fall away exactly
        double x = (double)t * (double)p.inv_freq[j] * 0.15915494309189533577;
        x -= rint(x);
        float s, c;
        sincospif(2.0f * (float)x, &s, &c);
        reinterpret_cast<float2*>(turn + (rr * 4 + j % 8 / 2) * eights + j / 8)[j % 2] = make_float2(c, s);
    }
    __syncthreads();

    for (int row = 0; row < tokens * slots; row += step) {  // (all lanes of a warp, for the shuffles)
        const bool mine = r < tokens && u < units;
        const int r_now = r, slot_now = slot, of_kv = slot - p.heads;
        const bool query = of_kv < 0, value = of_kv >= p.map.kv_heads;
        float x[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = to_f32<T>(raw.v[e]);
        r += step_r;
        slot += step_slot;
        if (slot >= slots) slot -= slots, ++r;
        if (r < tokens && u < units) load(r, slot);
        if (!value && mine) {
            const float4* t = turn + r_now * 4 * eights + u;
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                if (8 * u + (WHOLE && !INTERLEAVED ? 0 : e) >= p.half) continue;  // (whole: eight pairs or none)
                const float4 two = t[e / 2 * eights];
#pragma unroll
                for (int i = e; i < e + 2; ++i) {
                    const float cosine = i == e ? two.x : two.z, sine = i == e ? two.y : two.w;
                    float &a = WHOLE && INTERLEAVED ? x[2 * i] : x[i], &c = WHOLE && INTERLEAVED ? x[2 * i + 1] : x[8 + i];
                    const float first = a, second = c;
                    if (!(WHOLE && !INTERLEAVED) && 8 * u + i >= p.half) continue;
                    a = turned(first, second, cosine, -sine);
                    c = turned(second, first, cosine, sine);
                }
            }
        }
        const long long at = mine ? place[r_now] : -1;
        if (mine && query) {
            T* to = static_cast<T*>(p.q_out) + b * p.os[0] + slot_now * p.os[1] + (r0 + r_now) * p.os[2];
            if (at < 0) {
#pragma unroll
                for (int e = 0; e < 16; ++e) x[e] = __int_as_float(0x7fffffff);
            }
            if constexpr (WHOLE) {
                store8<T>(to + ia, x);
                store8<T>(to + ib, x + 8);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int2 where = at_pair(e);
                    to[where.x] = from_f32<T>(x[e]);
                    to[where.y] = from_f32<T>(x[8 + e]);
                }
            }
        }
        if (__all_sync(0xffffffffu, query || !mine)) continue;
        float top = 0.f, wrong = 0.f;  // the largest; NaN where an infinity or a NaN is
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            top = fmaxf(top, fabsf(x[e]));
            wrong = fmaf(x[e], 0.f, wrong);
        }
        if (wrong != 0.f) top = __int_as_float(0x7f800000);
        for (int d = 1; d < lanes; d *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        if (!mine || query || at < 0) continue;
        const bool finite = top < __int_as_float(0x7f800000);
        // top / largest, rounded once: a quotient, and what it leaves, divided by the nearest reciprocal (Markstein's correction)
        constexpr float kPart = 1.0f / kLargest<P>;
        float scale = top * kPart;
        scale = fmaxf(fmaf(fmaf(-scale, kLargest<P>, top), kPart, scale), kLeastScale);
        if (!finite) scale = __int_as_float(0x7fffffff);
        uint32_t codes[4] = {0, 0, 0, 0};
        if (finite) codes16<P>(x, scale, codes);
        const long long place_of = at + (long long)(value ? of_kv - p.map.kv_heads : of_kv) * p.map.page.d;
        if (u == 0) (value ? p.v_scales : p.k_scales)[place_of] = scale;
        uint8_t* to = static_cast<uint8_t*>(value ? p.v_pages : p.k_pages) + place_of * p.map.head_dim;
        if constexpr (WHOLE) {
            *reinterpret_cast<uint2*>(to + ia) = make_uint2(codes[0], codes[1]);
            *reinterpret_cast<uint2*>(to + ib) = make_uint2(codes[2], codes[3]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int2 where = at_pair(e);
                to[where.x] = (uint8_t)(codes[e / 4] >> e % 4 * 8);
                to[where.y] = (uint8_t)(codes[2 + e / 4] >> e % 4 * 8);
            }
        }
    }
}

template <typename T, typename P>
int launch(PagedAppend& p, const tmw_paged_append_desc& d, bool whole, cudaStream_t stream) {
    const dim3 grid((unsigned)((p.rows + kTokens - 1) / kTokens), (unsigned)d.at.batch), block(kThreads);
    const int smem = kTokens * 4 * ((p.half + 7) / 8) * (int)sizeof(float4);
    if (d.interleaved) {
        if (whole) paged_append8_kernel<T, P, true, true><<<grid, block, smem, stream>>>(p);
        else paged_append8_kernel<T, P, true, false><<<grid, block, smem, stream>>>(p);
    } else {
        if (whole) paged_append8_kernel<T, P, false, true><<<grid, block, smem, stream>>>(p);
        else paged_append8_kernel<T, P, false, false><<<grid, block, smem, stream>>>(p);
    }
    TMW_CUDA_TRY(cudaGetLastError());
    return TMW_OK;
}
template <typename T>
int launch(PagedAppend& p, const tmw_paged_append_desc& d, int format, bool whole, cudaStream_t stream) {
    return format == TMW_PAGES_INT8 ? launch<T, int8_t>(p, d, whole, stream) : launch<T, E4m3>(p, d, whole, stream);
}

}  // namespace
}  // namespace tmw

extern "C" int tmw_paged_append_scaled(const tmw_paged_append_desc* d, const tmw_page_scales* scales, const int32_t* positions,
                                       void* stream) {
    using namespace tmw;
    PagedAppend p;
    bool used = false;
    uintptr_t bits = 0;
    long long strides = 0;
    const int rc = append_arguments(d, scales, positions, p, used, bits, strides);
    if (rc != TMW_OK || !used) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (scales == nullptr || scales->format == TMW_PAGES_SAME) return append_same(p, *d, bits, strides, s);
    // Whole vectors where every row begins on 16 bytes and no pair is cut; single elements otherwise.
    const int e = 16 / (int)dtype_size(d->at.dtype);
    const bool whole = bits % 16 == 0 && strides % e == 0 && (d->interleaved || d->rotated / 2 % 8 == 0);
    if (d->at.dtype == TMW_F32) return launch<float>(p, *d, scales->format, whole, s);
    return d->at.dtype == TMW_BF16 ? launch<__nv_bfloat16>(p, *d, scales->format, whole, s) : launch<__half>(p, *d, scales->format, whole, s);
}
