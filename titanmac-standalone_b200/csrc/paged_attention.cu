// Attention of one new token per sequence over its paged keys (tmw_paged_attention).
//
// For every (sequence, key head) the query heads that read it see the persistent keys and the tokens lo .. pos of the sequence;
// with s_j = q k_j scale, o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m), m a running maximum: one pass, each key and value read
// once for all heads of the group.  A step does two to a few multiply-adds per number read: HBM bounds it, or, for a
// handful of keys, launch and latency.
//
// The lengths are on the device and may differ by any factor, so the host cannot cut the work up.  The keys of an item - a
// sequence and the heads of one key head, at most kMaxRows of them - come in tiles of 16, the tiles of all items in one line, and
// CTA c takes the tiles [c, c + 1) * per of it: every CTA the same number, whatever the lengths.  Its warps take every
// W-th tile, each with its own ring of tiles in shared memory (cp.async, no barrier in the loop) and its own maximum and
// sums, and join them where an item ends.  An item that lies in one CTA is stored at once; the parts of one that was cut go to
// scratch memory, and a second kernel, launched under the first, joins them in the order of the CTAs.
#include <math_constants.h>

#include <type_traits>

#include "paged.cuh"

namespace tmw {
namespace {

constexpr int kTile = 16;   // keys
constexpr int kMaxRows = 16;

struct PagedAttention {
    PageMap map;
    const void *q, *k_pages, *v_pages, *k_pers, *v_pers;
    void* o;
    long long qs[2], os[2];
    const int32_t* pos;
    int batch, np, window;
    int group;        // query heads of a key head
    int rows, parts;  // query heads of an item at most; items of a key head
    int items;        // of a sequence
    float scale;      // times log2(e)
    int row_bytes;
    bool q_pairs;  // queries can be read two at a time
    float* partial;  // [CTA][2][rows][head_dim]: of the item that a CTA begins with, of the one that it ends with
    float2* sums;    // [CTA][2][rows]: maximum, sum
    int4* joins;     // [CTA]: the item cut at the CTA's end that begins in it - sequence, item, last CTA, which of the two parts
    int* status;
};

// Tiles of sequence b's items; lo, pos: its first and last token seen (lo > pos: none).  0 with bad: no such position.
__device__ __forceinline__ int tiles_of(const PagedAttention& p, int b, int& lo, int& pos, bool& bad) {
    pos = __ldg(p.pos + b);
    bad = pos < -1 || pos >= p.map.capacity;
    lo = 0;
    if (bad) return 0;
    const int pers = (p.np + kTile - 1) / kTile;
    if (pos < 0) return pers;
    if (p.window >= 0 && pos > p.window) lo = pos - p.window;
    return pers + pos / kTile - lo / kTile + 1;
}

// A place in the line of tiles.
struct Cursor {
    int b, item;  // sequence, item of it
    int t, n;     // tile of the item, of so many
    int lo, pos;
    __device__ __forceinline__ void sequence(const PagedAttention& p) {
        bool bad;
        n = tiles_of(p, b, lo, pos, bad);
    }
    // k tiles on; not past the end of the line
    __device__ __forceinline__ void advance(const PagedAttention& p, int k) {
        t += k;
        while (t >= n) {
            t -= n;
            if (++item == p.items) {
                item = 0;
                do {
                    ++b;
                    sequence(p);
                } while (n == 0);
            }
        }
    }
};

// This CTA's part of the line, and the place where it begins.  Every thread of the CTA.
struct Share {
    long long first, end, per;
};
template <int W>
__device__ __forceinline__ Share find_share(const PagedAttention& p, Cursor& at) {
    __shared__ long long warp_sum[W];
    __shared__ long long found_before;
    __shared__ int found_b;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int lo, pos;
    bool bad;
    // tiles of all sequences
    long long sum = 0;
    for (int b = tid; b < p.batch; b += (W * 32)) sum += tiles_of(p, b, lo, pos, bad);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) warp_sum[warp] = sum;
    __syncthreads();
    long long total = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) total += warp_sum[w];
    total *= p.items;
    Share s;
    // (below a tile for every warp, a CTA more costs more to join than it saves)
    s.per = (total + gridDim.x - 1) / gridDim.x;
    if (s.per < W) s.per = W;
    s.first = s.per * blockIdx.x;
    s.end = s.first + s.per < total ? s.first + s.per : total;
    if (s.first >= s.end) return s;
    // the sequence that holds the first tile
    long long before = 0;
    for (int b0 = 0; b0 < p.batch; b0 += (W * 32)) {
        const int b = b0 + tid;
        const long long mine = b < p.batch ? (long long)tiles_of(p, b, lo, pos, bad) * p.items : 0;
        long long upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += x;
        }
        __syncthreads();
        if (lane == 31) warp_sum[warp] = upto;
        if (tid == 0) found_b = -1;
        __syncthreads();
        long long all = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            if (w < warp) upto += warp_sum[w];
            all += warp_sum[w];
        }
        upto += before;
        if (upto - mine <= s.first && s.first < upto) {
            found_b = b;
            found_before = upto - mine;
        }
        __syncthreads();
        if (found_b >= 0) break;
        before += all;
    }
    at.b = found_b;
    at.sequence(p);
    const long long inside = s.first - found_before;
    at.item = (int)(inside / at.n);
    at.t = (int)(inside - (long long)at.item * at.n);
    return s;
}

__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}

// A warp's ring: tiles of keys, as many of values, and what of them counts (bits 0-15: seen, 16-31: without a page).
struct Ring {
    unsigned char* tiles;
    uint32_t* marks;
};

// Tile `at` of keys and values into a stage of the ring.  Rows that do not count become zeros: whatever stands in a page behind a
// sequence's end, infinities and NaN among them, reaches no product.
template <typename T, typename Layout>
__device__ __forceinline__ void load_tile(const PagedAttention& p, const Ring& ring, const Layout& lay, const Cursor& at, int stage) {
    const int lane = threadIdx.x & 31, r = lane & (kTile - 1);
    const int head = at.item / p.parts;
    const int pers = (p.np + kTile - 1) / kTile;
    const unsigned char *k = static_cast<const unsigned char*>(p.k_pages), *v = static_cast<const unsigned char*>(p.v_pages);
    long long row = -1;
    bool seen;
    if (at.t < pers) {
        k = static_cast<const unsigned char*>(p.k_pers);
        v = static_cast<const unsigned char*>(p.v_pers);
        const int j = at.t * kTile + r;
        seen = j < p.np;
        if (seen) row = ((long long)head * p.np + j) * p.map.head_dim;
    } else {
        const int j = (at.lo / kTile + at.t - pers) * kTile + r;
        seen = j >= at.lo && j <= at.pos;
        if (seen) {
            row = p.map.token(at.b, j);
            if (row >= 0) row += head * p.map.head_step();
        }
    }
    const uint32_t bits = __ballot_sync(0xffffffffu, lane < kTile ? seen : row < 0 && seen);
    if (lane == 0) ring.marks[stage] = bits;
    const uint32_t to = (uint32_t)__cvta_generic_to_shared(ring.tiles) + stage * 2 * kTile * lay.pitch();
    const int chunks = lay.chunks(), n = kTile * chunks;
    for (int i0 = 0; i0 < n; i0 += 32) {
        const int i = min(i0 + lane, n - 1), rr = i / chunks, c = i - rr * chunks;
        const long long at_row = __shfl_sync(0xffffffffu, row, rr);
        if (i0 + lane >= n) continue;
        const bool there = at_row >= 0;
        const long long off = at_row * (long long)sizeof(T) + c * 16;
        const uint32_t dst = to + lay.offset(rr, c);
        copy16(dst, there ? static_cast<const void*>(k + off) : p.sums, there);  // (no byte is read where there is none)
        copy16(dst + kTile * lay.pitch(), there ? static_cast<const void*>(v + off) : p.sums, there);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
}

// ---- the core on CUDA cores: every type, head_dim a multiple of 8 --------------------------------------------------------
// Lane l has key l % 16 of a tile and one half of the head's dimensions of its scores; then the four dimensions from 4 l on (and
// from 128 + 4 l) of the outputs.  kRows query heads, their numbers as fp32 in shared memory.
template <typename T>
struct SimtLayout {
    int bytes;  // of a row; 16 more keep the rows of 8 lanes off each other's banks
    __host__ __device__ __forceinline__ int pitch() const { return bytes + 16; }
    __device__ __forceinline__ int chunks() const { return bytes / 16; }
    __device__ __forceinline__ int offset(int r, int c) const { return r * pitch() + c * 16; }
};

template <typename T>
__device__ __forceinline__ float4 load4(const unsigned char* at);
template <>
__device__ __forceinline__ float4 load4<float>(const unsigned char* at) { return *reinterpret_cast<const float4*>(at); }
template <>
__device__ __forceinline__ float4 load4<__nv_bfloat16>(const unsigned char* at) {
    const uint2 w = *reinterpret_cast<const uint2*>(at);
    return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                       __uint_as_float(w.y & 0xffff0000u));
}
template <>
__device__ __forceinline__ float4 load4<__half>(const unsigned char* at) {
    const uint2 w = *reinterpret_cast<const uint2*>(at);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
    return make_float4(a.x, a.y, b.x, b.y);
}

__device__ __forceinline__ void add_product(float4& acc, float w, const float4& x) {
    acc.x = fmaf(w, x.x, acc.x);
    acc.y = fmaf(w, x.y, acc.y);
    acc.z = fmaf(w, x.z, acc.z);
    acc.w = fmaf(w, x.w, acc.w);
}

constexpr int kSimtRows = 4;

template <typename T>
struct SimtCore {
    static constexpr int kRows = kSimtRows;
    using Layout = SimtLayout<T>;
    const PagedAttention& p;
    float* q;        // [kRows][head_dim], of the CTA's warp
    float* weights;  // [kTile][kRows]
    float m[kRows], l[kRows];
    float4 o[kRows][2];

    // shared memory of a warp besides its ring
    static __host__ __device__ int extra(int head_dim) { return (kRows * head_dim + kTile * kRows) * (int)sizeof(float); }

    __device__ SimtCore(const PagedAttention& p, unsigned char* mine) : p(p), q(reinterpret_cast<float*>(mine)) {
        weights = q + kRows * p.map.head_dim;
    }
    __device__ __forceinline__ void begin(int b, int first, int rows) {
        const int lane = threadIdx.x & 31, dim = p.map.head_dim;
        __syncwarp();
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const T* from = static_cast<const T*>(p.q) + b * p.qs[0] + (first + r) * p.qs[1];
            for (int i = lane; i < dim; i += 32) q[r * dim + i] = r < rows ? to_f32<T>(from[i]) : 0.f;
            m[r] = -CUDART_INF_F;
            l[r] = 0.f;
            o[r][0] = o[r][1] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        __syncwarp();
    }
    __device__ __forceinline__ void tile(const unsigned char* tile, uint32_t marks, const Layout& lay) {
        const int lane = threadIdx.x & 31, key = lane & (kTile - 1), dim = p.map.head_dim, half = dim / 2;
        const unsigned char* row = tile + key * lay.pitch();
        float s[kRows] = {};
        for (int i = (lane >> 4) * half; i < (lane >> 4) * half + half; i += 4) {
            const float4 k4 = load4<T>(row + i * sizeof(T));
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                const float4 q4 = *reinterpret_cast<const float4*>(q + r * dim + i);
                s[r] = fmaf(q4.x, k4.x, fmaf(q4.y, k4.y, fmaf(q4.z, k4.z, fmaf(q4.w, k4.w, s[r]))));
            }
        }
        const bool seen = marks >> key & 1, bad = marks >> (16 + key) & 1;
        float w[kRows];
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            float x = (s[r] + __shfl_xor_sync(0xffffffffu, s[r], 16)) * p.scale;
            x = bad ? CUDART_NAN_F : seen ? x : -CUDART_INF_F;
            float top = x;
#pragma unroll
            for (int d = 8; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            const float now = fmaxf(m[r], top), base = now == -CUDART_INF_F ? 0.f : now;
            const float keep = m[r] == -CUDART_INF_F ? 1.f : exp2f(m[r] - base);  // (nothing to keep, or NaN)
            m[r] = now;
            w[r] = seen ? exp2f(x - base) : 0.f;
            l[r] = l[r] * keep + w[r];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                o[r][h].x *= keep; o[r][h].y *= keep; o[r][h].z *= keep; o[r][h].w *= keep;
            }
        }
        if (lane < kTile) *reinterpret_cast<float4*>(weights + key * kRows) = make_float4(w[0], w[1], w[2], w[3]);
        __syncwarp();
        const unsigned char* values = tile + kTile * lay.pitch();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int i = h * 128 + lane * 4;
            if (i >= dim) break;
#pragma unroll 4
            for (int j = 0; j < kTile; ++j) {
                const float4 v4 = load4<T>(values + j * lay.pitch() + i * sizeof(T));
                const float4 w4 = *reinterpret_cast<const float4*>(weights + j * kRows);
                add_product(o[0][h], w4.x, v4);
                add_product(o[1][h], w4.y, v4);
                add_product(o[2][h], w4.z, v4);
                add_product(o[3][h], w4.w, v4);
            }
        }
        __syncwarp();
    }
    // this warp's part of the item: sums [rows], outputs [rows][head_dim]
    __device__ __forceinline__ void leave(float2* sums, float* out, int rows) {
        const int lane = threadIdx.x & 31, dim = p.map.head_dim;
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            float t = l[r];
#pragma unroll
            for (int d = 8; d > 0; d >>= 1) t += __shfl_xor_sync(0xffffffffu, t, d);
            if (r >= rows) continue;
            if (lane == 0) sums[r] = make_float2(m[r], t);
#pragma unroll
            for (int h = 0; h < 2; ++h)
                if (h * 128 + lane * 4 < dim) *reinterpret_cast<float4*>(out + r * dim + h * 128 + lane * 4) = o[r][h];
        }
    }
};

// ---- the core on tensor cores: 16-bit types, head_dim 32, 64, 96, 128 or 256 -------------------------------------------------
// mma.sync with the query heads as the sixteen rows of a tile (tcgen05's 64 or 128 would multiply a group of at most sixteen
// for nothing, and the step is bound by HBM long before): scores 16 x 16 keys, their exponentials straight from the accumulators
// to the operand of the second product.  The weights go in as two 16-bit numbers each, a value and what it lacks: one alone would
// put up to 2^-9 of itself on the output, the two 2^-16.  (The first is cut off and the second is never zero: both positive,
// they take an infinite value to infinity, as the weight itself would.)  In fp16 they are raised by 2^12, as far as the largest allows, so
// that those below 2^-14 of it keep their bits.  Up to eight heads: the tile's upper eight rows are zeros and have no registers.
template <int DH>
struct MmaLayout {
    int bytes;
    __host__ __device__ static constexpr int pitch() { return DH * 2; }
    __host__ __device__ static constexpr int chunks() { return DH / 8; }
    // a chunk's place in its row keeps eight rows' same chunk on different banks
    __device__ __forceinline__ static int offset(int r, int c) {
        const int turn = chunks() % 8 == 0 ? r & 7 : r >> 1 & 3;
        return r * pitch() + ((c ^ turn) << 4);
    }
};

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
// the same cut off instead of rounded
template <typename T>
__device__ __forceinline__ uint32_t cut2(float a, float b);
template <>
__device__ __forceinline__ uint32_t cut2<__nv_bfloat16>(float a, float b) {
    uint32_t w;
    asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(b), "f"(a));
    return w;
}
template <>
__device__ __forceinline__ uint32_t cut2<__half>(float a, float b) {
    uint32_t w;
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(b), "f"(a));
    return w;
}
// no number below the smallest that a product takes (2^-126, 2^-24)
template <typename T>
__device__ __forceinline__ uint32_t positive2(uint32_t w);
template <>
__device__ __forceinline__ uint32_t positive2<__nv_bfloat16>(uint32_t w) {
    const uint32_t least = 0x00800080u;
    const __nv_bfloat162 v = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&w), *reinterpret_cast<const __nv_bfloat162*>(&least));
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t positive2<__half>(uint32_t w) {
    const uint32_t least = 0x00010001u;
    const __half2 v = __hmax2(*reinterpret_cast<const __half2*>(&w), *reinterpret_cast<const __half2*>(&least));
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

template <typename T, int DH, bool WIDE>
struct MmaCore {
    static constexpr int kRows = kMaxRows;
    static constexpr int kHalves = WIDE ? 2 : 1;  // of the sixteen rows
    static constexpr float kRaise = std::is_same<T, __half>::value ? 12.f : 0.f;
    using Layout = MmaLayout<DH>;
    const PagedAttention& p;
    uint32_t q[DH / 16][2 * kHalves];  // a0, a2 (, a1, a3)
    float m[kHalves], l[kHalves];      // of rows lane / 4 and 8 + lane / 4; l: this lane's columns
    float o[DH / 8][2 * kHalves];

    static __host__ __device__ int extra(int) { return 0; }

    __device__ MmaCore(const PagedAttention& p, unsigned char*) : p(p) {}
    __device__ __forceinline__ void begin(int b, int first, int rows) {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
            const int r = h * 8 + lane / 4;
            const T* from = static_cast<const T*>(p.q) + b * p.qs[0] + (first + r) * p.qs[1] + lane % 4 * 2;
#pragma unroll
            for (int k = 0; k < DH / 16; ++k)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint32_t w = 0;
                    if (r < rows) {
                        const T* at = from + k * 16 + i * 8;
                        if (p.q_pairs) w = *reinterpret_cast<const uint32_t*>(at);
                        else w = *reinterpret_cast<const uint16_t*>(at) | (uint32_t)*reinterpret_cast<const uint16_t*>(at + 1) << 16;
                    }
                    q[k][h * 2 + i] = w;
                }
            m[h] = -CUDART_INF_F;
            l[h] = 0.f;
        }
#pragma unroll
        for (int j = 0; j < DH / 8; ++j)
#pragma unroll
            for (int i = 0; i < 2 * kHalves; ++i) o[j][i] = 0.f;
    }
    // c += a b, a the rows' two halves (the upper one zero where there is none)
    __device__ __forceinline__ static void product(float* c, const uint32_t (&a)[2 * kHalves], uint32_t b0, uint32_t b1) {
        float d[4] = {c[0], c[1], WIDE ? c[2] : 0.f, WIDE ? c[3] : 0.f};
        mma_16816<T>(d, a[0], WIDE ? a[2] : 0u, a[1], WIDE ? a[3] : 0u, b0, b1);
        c[0] = d[0];
        c[1] = d[1];
        if (WIDE) c[2] = d[2], c[3] = d[3];
    }
    __device__ __forceinline__ void tile(const unsigned char* tile, uint32_t marks, const Layout& lay) {
        const int lane = threadIdx.x & 31;
        const uint32_t keys = (uint32_t)__cvta_generic_to_shared(tile), values = keys + kTile * Layout::pitch();
        float s[2][2 * kHalves] = {};  // eight keys each
#pragma unroll
        for (int k = 0; k < DH / 16; ++k) {
            uint32_t b[4];
            ldmatrix4(b, keys + lay.offset((lane >> 4) * 8 + (lane & 7), k * 2 + (lane >> 3 & 1)));
            product(s[0], q[k], b[0], b[1]);
            product(s[1], q[k], b[2], b[3]);
        }
        uint32_t hi[2 * kHalves], lo[2 * kHalves];  // a0, a2 (, a1, a3) of the weights
        float keep[kHalves];
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
            float top = -CUDART_INF_F;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int key = j * 8 + lane % 4 * 2 + e;
                    float& x = s[j][h * 2 + e];
                    x = marks >> (16 + key) & 1 ? CUDART_NAN_F : marks >> key & 1 ? x * p.scale : -CUDART_INF_F;
                    top = fmaxf(top, x);
                }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float now = fmaxf(m[h], top), base = now == -CUDART_INF_F ? 0.f : now;
            keep[h] = m[h] == -CUDART_INF_F ? 1.f : ex2_ftz(m[h] - base);  // (nothing to keep, or NaN)
            m[h] = now;
            l[h] *= keep[h];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float w[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    w[e] = ex2_ftz(s[j][h * 2 + e] - base + kRaise);
                    l[h] += w[e];
                }
                hi[h * 2 + j] = cut2<T>(w[0], w[1]);
                const float2 there = unpack2<T>(hi[h * 2 + j]);
                lo[h * 2 + j] = positive2<T>(pack2<T>(w[0] - there.x, w[1] - there.y));
            }
        }
        if (__any_sync(0xffffffffu, keep[0] != 1.f || keep[kHalves - 1] != 1.f)) {
#pragma unroll
            for (int j = 0; j < DH / 8; ++j)
#pragma unroll
                for (int i = 0; i < 2 * kHalves; ++i) o[j][i] *= keep[i / 2];
        }
#pragma unroll
        for (int k = 0; k < DH / 16; ++k) {
            uint32_t b[4];
            ldmatrix4_trans(b, values + lay.offset((lane >> 3 & 1) * 8 + (lane & 7), k * 2 + (lane >> 4)));
            product(o[2 * k], hi, b[0], b[1]);
            product(o[2 * k + 1], hi, b[2], b[3]);
            product(o[2 * k], lo, b[0], b[1]);
            product(o[2 * k + 1], lo, b[2], b[3]);
        }
    }
    __device__ __forceinline__ void leave(float2* sums, float* out, int rows) {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
            const int r = h * 8 + lane / 4;
            float t = l[h];
            t += __shfl_xor_sync(0xffffffffu, t, 1);
            t += __shfl_xor_sync(0xffffffffu, t, 2);
            if (r >= rows) continue;
            if (lane % 4 == 0) sums[r] = make_float2(m[h], t);
#pragma unroll
            for (int j = 0; j < DH / 8; ++j)
                *reinterpret_cast<float2*>(out + r * DH + j * 8 + lane % 4 * 2) = make_float2(o[j][h * 2], o[j][h * 2 + 1]);
        }
    }
};

// ---- the line of tiles ------------------------------------------------------------------------------------------------------

// weight of a part whose maximum is m under the common one (base: that, or 0 where it is -inf): a part of hidden scores alone
// holds zeros, or NaN that has to stay
__device__ __forceinline__ float part_weight(float m, float base) { return m == -CUDART_INF_F ? 1.f : exp2f(m - base); }

// (the largest score's weight is 1 or more: no sum at all is that of scores of -inf)
__device__ __forceinline__ float quotient(float o, float l) { return l == 0.f ? CUDART_NAN_F : o / l; }

template <typename T, typename Core, int W, int S>
__global__ void __launch_bounds__(W * 32) paged_attention_kernel(const __grid_constant__ PagedAttention p) {
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ uint32_t marks[W][S];
    __shared__ float2 warp_sums[W][kMaxRows];
    pdl_trigger();
    const int tid = threadIdx.x, warp = tid >> 5, dim = p.map.head_dim;
    const typename Core::Layout lay{p.row_bytes};
    const int ring_bytes = S * 2 * kTile * lay.pitch(), extra = Core::extra(dim);
    unsigned char* mine = smem + warp * (ring_bytes + extra);
    const Ring ring{mine, marks[warp]};
    float* outs = reinterpret_cast<float*>(smem + W * (ring_bytes + extra));  // [warp][rows][head_dim]

    // sequences without a key to see, or without a place
    for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
        int lo, pos;
        bool bad;
        if (tiles_of(p, b, lo, pos, bad) > 0) continue;
        if (bad && tid == 0) atomicCAS(p.status, 0, (int)TMW_ERR_INVALID_ARGUMENT);
        const int heads = p.group * p.map.kv_heads;
        for (int i = tid; i < heads * dim; i += W * 32)
            static_cast<T*>(p.o)[b * p.os[0] + (i / dim) * p.os[1] + i % dim] = from_f32<T>(bad ? CUDART_NAN_F : 0.f);
    }
    if (tid == 0) p.joins[blockIdx.x] = make_int4(-1, 0, 0, 0);
    Cursor at;
    const Share share = find_share<W>(p, at);
    if (share.first >= share.end) return;

    Cursor ahead = at;  // the tile to load next
    long long load = share.first + warp;
    if (load < share.end) ahead.advance(p, warp);
    int stage_in = 0, stage_out = 0;
    auto fetch = [&]() {
        if (load < share.end) {
            load_tile<T>(p, ring, lay, ahead, stage_in);
            load += W;
            if (load < share.end) ahead.advance(p, W);
        } else {
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
        stage_in = stage_in + 1 == S ? 0 : stage_in + 1;
    };
#pragma unroll
    for (int s = 0; s < S - 1; ++s) fetch();

    Core core(p, mine + ring_bytes);
    long long u = share.first + warp, begin = share.first;
    bool bad_page = false;
    while (begin < share.end) {
        const long long item_end = begin + (at.n - at.t), end = item_end < share.end ? item_end : share.end;
        const int first = at.item % p.parts * p.rows, rows = min(p.rows, p.group - first);
        const int head = at.item / p.parts * p.group + first;
        core.begin(at.b, head, rows);
        for (; u < end; u += W) {
            asm volatile("cp.async.wait_group %0;" ::"n"(S - 2) : "memory");
            __syncwarp();
            fetch();
            const uint32_t mark = ring.marks[stage_out];
            bad_page |= mark >> 16 != 0;
            core.tile(ring.tiles + stage_out * 2 * kTile * lay.pitch(), mark, lay);
            stage_out = stage_out + 1 == S ? 0 : stage_out + 1;
        }
        // (a warp without a tile leaves a maximum of -inf and zeros)
        core.leave(warp_sums[warp], outs + warp * p.rows * dim, rows);
        __syncthreads();
        const bool whole = at.t == 0 && end == item_end;
        const int part = begin == share.first ? 0 : 1;
        const long long slot = (long long)blockIdx.x * 2 + part;
        for (int i = tid; i < rows * dim; i += W * 32) {
            const int r = i / dim;
            float m = warp_sums[0][r].x;
#pragma unroll
            for (int w = 1; w < W; ++w) m = fmaxf(m, warp_sums[w][r].x);
            const float base = m == -CUDART_INF_F ? 0.f : m;
            float l = 0.f, o = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const float x = part_weight(warp_sums[w][r].x, base);
                l = fmaf(x, warp_sums[w][r].y, l);
                o = fmaf(x, outs[w * p.rows * dim + i], o);
            }
            if (whole) {
                static_cast<T*>(p.o)[at.b * p.os[0] + (head + r) * p.os[1] + (i - r * dim)] = from_f32<T>(quotient(o, l));
            } else {
                p.partial[slot * p.rows * dim + i] = o;
                if (i == r * dim) p.sums[slot * p.rows + r] = make_float2(m, l);
            }
        }
        if (at.t == 0 && end < item_end && tid == 0)  // begins here, ends in another CTA
            p.joins[blockIdx.x] = make_int4(at.b, at.item, (int)((item_end - 1) / share.per), part);
        __syncthreads();
        if (item_end < share.end) at.advance(p, at.n - at.t);
        begin = end;
    }
    if (__any_sync(0xffffffffu, bad_page) && (tid & 31) == 0) atomicCAS(p.status, 0, (int)TMW_ERR_INVALID_ARGUMENT);
}

// The parts of an item that was cut: CTA (c, r) joins row r of the one that begins in CTA c.  Its warps take every
// kJoinWarps-th part each, a lane four dimensions.
constexpr int kJoinWarps = 8;
template <typename T>
__global__ void __launch_bounds__(kJoinWarps * 32) paged_join_kernel(const __grid_constant__ PagedAttention p) {
    __shared__ float warp_max[kJoinWarps], warp_sum[kJoinWarps];
    __shared__ float outs[kJoinWarps][256];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, dim = p.map.head_dim, r = blockIdx.y;
    pdl_wait();
    const int4 join = __ldcg(p.joins + blockIdx.x);
    if (join.x < 0) return;
    const int first = join.y % p.parts * p.rows;
    if (r >= min(p.rows, p.group - first)) return;
    const int n = join.z - (int)blockIdx.x + 1;
    auto slot = [&](int i) { return (2LL * (blockIdx.x + i) + (i == 0 ? join.w : 0)) * p.rows + r; };
    float m = -CUDART_INF_F;
    for (int i = tid; i < n; i += kJoinWarps * 32) m = fmaxf(m, __ldcg(p.sums + slot(i)).x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) warp_max[warp] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) m = fmaxf(m, warp_max[w]);
    const float base = m == -CUDART_INF_F ? 0.f : m;
    float l = 0.f;
    float4 o[2] = {};
#pragma unroll 4
    for (int i = warp; i < n; i += kJoinWarps) {
        const float2 ml = __ldcg(p.sums + slot(i));
        const float x = part_weight(ml.x, base);
        l = fmaf(x, ml.y, l);
        const float* from = p.partial + slot(i) * dim;
#pragma unroll
        for (int h = 0; h < 2; ++h)
            if (h * 128 + lane * 4 < dim) add_product(o[h], x, __ldcg(reinterpret_cast<const float4*>(from + h * 128 + lane * 4)));
    }
    if (lane == 0) warp_sum[warp] = l;
#pragma unroll
    for (int h = 0; h < 2; ++h)
        if (h * 128 + lane * 4 < dim) *reinterpret_cast<float4*>(&outs[warp][h * 128 + lane * 4]) = o[h];
    __syncthreads();
    if (tid >= dim) return;
    float sum = 0.f, out = 0.f;
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) {
        sum += warp_sum[w];
        out += outs[w][tid];
    }
    const int head = join.y / p.parts * p.group + first + r;
    static_cast<T*>(p.o)[join.x * p.os[0] + head * p.os[1] + tid] = from_f32<T>(quotient(out, sum));
}

// ---- host ---------------------------------------------------------------------------------------------------------------------

constexpr int kMostShared = 226 * 1024;  // of a CTA, beside what the kernel declares

struct Plan {
    int rows, parts, grid, smem;
    size_t sums_at, partial_at, bytes;
};

template <typename T, typename Core, int W, int S>
struct Kernel {
    static constexpr int kMostCtas = 4;  // to an SM
    static Plan plan(const tmw_paged_attention_desc& d, int row_bytes) {
        Plan n;
        const int group = d.heads / d.at.kv_heads;
        n.parts = (group + Core::kRows - 1) / Core::kRows;
        n.rows = (group + n.parts - 1) / n.parts;
        const int pitch = typename Core::Layout{row_bytes}.pitch();
        n.smem = W * (S * 2 * kTile * pitch + Core::extra(d.at.head_dim) + n.rows * d.at.head_dim * (int)sizeof(float));
        int ctas = 228 * 1024 / (n.smem + 2048);
        ctas = ctas < 1 ? 1 : ctas > kMostCtas ? kMostCtas : ctas;
        // no more CTAs than the longest sequences could have work for
        const long long capacity = (long long)d.at.columns * d.at.page_size;
        const long long keys = d.window >= 0 && d.window + 1LL < capacity ? d.window + 1LL : capacity;
        const long long tiles = ((d.n_persistent + kTile - 1) / kTile + keys / kTile + 2) * (long long)d.at.kv_heads * n.parts;
        const long long most = (tiles * d.at.batch + W - 1) / W;
        n.grid = (int)(most < (long long)ctas * sm_count() ? most : (long long)ctas * sm_count());
        n.sums_at = (size_t)n.grid * sizeof(int4);
        n.partial_at = (n.sums_at + (size_t)n.grid * 2 * n.rows * sizeof(float2) + 15) & ~(size_t)15;
        n.bytes = n.partial_at + (size_t)n.grid * 2 * n.rows * d.at.head_dim * sizeof(float);
        return n;
    }
    static int launch(PagedAttention& p, const Plan& n, unsigned char* scratch, cudaStream_t stream) {
        p.rows = n.rows;
        p.parts = n.parts;
        p.items = p.map.kv_heads * n.parts;
        p.joins = reinterpret_cast<int4*>(scratch);
        p.sums = reinterpret_cast<float2*>(scratch + n.sums_at);
        p.partial = reinterpret_cast<float*>(scratch + n.partial_at);
        auto kern = paged_attention_kernel<T, Core, W, S>;
        const int rc = allow_shared_memory(reinterpret_cast<const void*>(kern), n.smem);
        if (rc != TMW_OK) return rc;
        kern<<<n.grid, W * 32, n.smem, stream>>>(p);
        TMW_CUDA_TRY(cudaGetLastError());
        if (n.grid > 1)
            TMW_CUDA_TRY(launch_ex(paged_join_kernel<T>, dim3((unsigned)n.grid - 1, (unsigned)n.rows), dim3(kJoinWarps * 32), 0, stream, true,
                                   1, p));
        return TMW_OK;
    }
};

// four warps to a CTA, or two where the rings of four would not fit
template <typename T, typename F>
int with_simt(const tmw_paged_attention_desc& d, F&& use) {
    using Four = Kernel<T, SimtCore<T>, 4, 3>;
    if (Four::plan(d, d.at.head_dim * (int)sizeof(T)).smem <= kMostShared) return use(Four());
    return use(Kernel<T, SimtCore<T>, 2, 3>());
}

template <typename T, int DH, typename F>
int with_mma(const tmw_paged_attention_desc& d, F&& use) {
    if (d.heads / d.at.kv_heads <= 8) return use(Kernel<T, MmaCore<T, DH, false>, 4, 3>());
    return use(Kernel<T, MmaCore<T, DH, true>, (DH > 128 ? 2 : 4), 3>());
}
template <typename T, typename F>
int with_16_bits(const tmw_paged_attention_desc& d, F&& use) {
    switch (d.at.head_dim) {
        case 32: return with_mma<T, 32>(d, use);
        case 64: return with_mma<T, 64>(d, use);
        case 96: return with_mma<T, 96>(d, use);
        case 128: return with_mma<T, 128>(d, use);
        case 256: return with_mma<T, 256>(d, use);
        default: return with_simt<T>(d, use);
    }
}

// `use` with the Kernel that takes the call
template <typename F>
int with_kernel(const tmw_paged_attention_desc& d, F&& use) {
    if (d.at.dtype == TMW_F32) return with_simt<float>(d, use);
    return d.at.dtype == TMW_BF16 ? with_16_bits<__nv_bfloat16>(d, use) : with_16_bits<__half>(d, use);
}

int validate(const tmw_paged_attention_desc* d, bool& used) {
    if (d == nullptr) return TMW_ERR_INVALID_ARGUMENT;
    if (d->heads < 0 || d->n_persistent < 0 || d->window < -1 || !(d->scale >= 0.f)) return TMW_ERR_INVALID_ARGUMENT;
    used = d->at.batch > 0 && d->heads > 0;
    const int rc = validate_pages(d->at, used);
    if (rc != TMW_OK) return rc;
    if (d->heads % d->at.kv_heads != 0) {
        set_error_text("tmw_paged_attention: heads must be a multiple of kv_heads");
        return TMW_ERR_INVALID_ARGUMENT;
    }
    if (d->heads > 65535 || d->n_persistent > (1 << 24)) return TMW_ERR_TOO_LARGE;
    return TMW_OK;
}

}  // namespace
}  // namespace tmw

extern "C" size_t tmw_paged_attention_scratch_bytes(const tmw_paged_attention_desc* d) {
    using namespace tmw;
    bool used = false;
    if (validate(d, used) != TMW_OK || !used) return 0;
    size_t bytes = 0;
    with_kernel(*d, [&](auto kernel) {
        bytes = kernel.plan(*d, d->at.head_dim * (int)dtype_size(d->at.dtype)).bytes;
        return TMW_OK;
    });
    return bytes;
}

extern "C" int tmw_paged_attention(const tmw_paged_attention_desc* d, void* scratch, size_t scratch_bytes, void* stream) {
    using namespace tmw;
    bool used = false;
    const int rc = validate(d, used);
    if (rc != TMW_OK || !used) return rc;
    const size_t size = dtype_size(d->at.dtype);
    if (d->q == nullptr || d->o == nullptr || d->pos == nullptr || scratch == nullptr ||
        (d->n_persistent > 0 && (d->k_pers == nullptr || d->v_pers == nullptr)))
        return TMW_ERR_INVALID_ARGUMENT;
    for (int i = 0; i < 2; ++i)
        if (d->q_stride[i] < 0 || d->o_stride[i] < 0) return TMW_ERR_INVALID_ARGUMENT;
    const auto bits = [](const void* x) { return reinterpret_cast<uintptr_t>(x); };
    if ((bits(d->k_pers) | bits(d->v_pers) | bits(scratch)) % 16 != 0 || (bits(d->q) | bits(d->o)) % size != 0)
        return TMW_ERR_INVALID_ARGUMENT;

    PagedAttention p = {};
    p.map = PageMap(d->at);
    p.q = d->q; p.o = d->o;
    p.k_pages = d->at.k_pages; p.v_pages = d->at.v_pages;
    p.k_pers = d->k_pers; p.v_pers = d->v_pers;
    for (int i = 0; i < 2; ++i) {
        p.qs[i] = d->q_stride[i];
        p.os[i] = d->o_stride[i];
    }
    p.pos = d->pos;
    p.batch = d->at.batch; p.np = d->n_persistent; p.window = d->window;
    p.group = d->heads / d->at.kv_heads;
    p.scale = (d->scale > 0.f ? d->scale : 1.0f / sqrtf((float)d->at.head_dim)) * 1.4426950408889634f;
    p.row_bytes = d->at.head_dim * (int)size;
    p.q_pairs = bits(d->q) % 4 == 0 && (d->q_stride[0] | d->q_stride[1]) % 2 == 0;
    p.status = device_status_word();
    if (p.status == nullptr) return TMW_ERR_CUDA;
    return with_kernel(*d, [&](auto kernel) {
        const Plan n = kernel.plan(*d, p.row_bytes);
        if (scratch_bytes < n.bytes) {
            set_error_text("tmw_paged_attention: scratch smaller than tmw_paged_attention_scratch_bytes()");
            return (int)TMW_ERR_INVALID_ARGUMENT;
        }
        return kernel.launch(p, n, static_cast<unsigned char*>(scratch), static_cast<cudaStream_t>(stream));
    });
}
