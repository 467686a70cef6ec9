// Attention of one new token per sequence over its paged keys (tmw_paged_attention).
//
// For every (sequence, key head) the query heads that read it see the persistent keys and the tokens lo .. pos of the sequence;
// with s_j = q k_j scale, o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m), m a running maximum: one pass, each key and value read
// once for all heads of the group.  A step does two to a few multiply-adds per number read: HBM bounds it, or, for a
// handful of keys, launch and latency.
//
// The lengths are on the device and may differ by any factor, so the host cannot cut the work up.  The keys of an item - a
// sequence and the heads of one key head, at most kMaxRows of them - come in tiles of 32 or 16, the tiles of all items in one line, and
// every warp of the grid takes an equal piece of the line, whatever the lengths.  A warp has its own ring of tiles in shared
// memory (cp.async), its own running maximum and sums, and meets no barrier on its way: an item that lies in its piece is stored
// from its registers.  Of an item that was cut, the warps of a CTA join their parts through shared memory when all of them are
// done; what was cut between CTAs goes to scratch memory, and a second kernel, launched under the first, joins it in the order of
// the CTAs.
//
// bf16, 553,000 tokens of 12 sequences, 32 heads of 128 on 4: 191 us, 5.9 TB/s; 48 sequences of 1 to 16384 tokens, 32 heads on 8, fp16:
// 119 us, 5.7 TB/s.  (Warps of a CTA on neighbouring tiles, joined at every item's end: 192 and 202 when this took 187 and 118.)
#include <math_constants.h>

#include <type_traits>

#include "paged.cuh"

namespace tmw {
namespace {

constexpr int kMaxRows = 16;

struct PagedAttention {
    PageMap map;
    const void *q, *k_pages, *v_pages, *k_pers, *v_pers;
    void* o;
    long long qs[2], os[2];
    const int32_t* pos;
    int batch, np, window;
    int pers_tiles;         // of the persistent keys
    bool whole_runs;        // sixteen tokens from a multiple of sixteen on lie in one page
    bool q_pairs, o_pairs;  // queries can be read, outputs stored two at a time
    int group;              // query heads of a key head
    int rows, parts;        // query heads of an item at most; items of a key head
    int items;              // of a sequence
    float scale;            // times log2(e)
    int row_bytes;
    float* partial;  // [CTA][2][rows][head_dim]: of the item that a CTA begins in, of the one that begins in it
    float2* sums;    // [CTA][2][rows]: maximum, sum
    float* firsts;   // [CTA][warp][rows][head_dim]: what a warp has of the item that its piece begins in
    int4* joins;     // [CTA]: the item that begins in it and ends in another one - sequence (-1: none), item, last CTA
    int* status;
};

// Tiles, of KT keys, of sequence b's items; lo, pos: its first and last token seen (lo > pos: none).  0 with bad: no such position.
template <int KT>
__device__ __forceinline__ int tiles_of(const PagedAttention& p, int b, int& lo, int& pos, bool& bad) {
    pos = __ldg(p.pos + b);
    bad = pos < -1 || pos >= p.map.capacity;
    lo = 0;
    if (bad) return 0;
    if (pos < 0) return p.pers_tiles;
    if (p.window >= 0 && pos > p.window) lo = pos - p.window;
    return p.pers_tiles + pos / KT - lo / KT + 1;
}

// A place in the line.  An item takes kItemCost more units of it than it has tiles, ahead of them: loading the queries and
// storing the output hold a warp up for about that long, and pieces of equal length are to take equal time.
constexpr int kItemCost = 1;
template <int KT>
struct Cursor {
    int b, item;  // sequence, item of it
    int head;     // the item's key head
    int t, n;     // unit of the item; units of an item
    int lo, pos;
    __device__ __forceinline__ void sequence(const PagedAttention& p) {
        bool bad;
        n = tiles_of<KT>(p, b, lo, pos, bad);
        if (n > 0) n += kItemCost;
    }
    __device__ __forceinline__ int tile() const { return t - kItemCost; }
    // the next item's first unit; not past the end of the line
    __device__ __forceinline__ void next_item(const PagedAttention& p) {
        t = 0;
        if (++item < p.items) {
            head = p.parts == 1 ? item : item / p.parts;
            return;
        }
        item = head = 0;
        do {
            ++b;
            sequence(p);
        } while (n == 0);
    }
};

__device__ __forceinline__ long long scan(long long x) {  // sums up to each lane
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    return x;
}

// This warp's piece of the line: units [first, end), of pieces of `per` units, `warps` of which go to a CTA; and the place where it
// begins.
struct Share {
    long long first, end, per;
    int warps;
};
template <int KT>
__device__ __forceinline__ Share find_share(const PagedAttention& p, Cursor<KT>& at) {
    const int lane = threadIdx.x & 31;
    auto units = [&](int b) -> long long {
        if (b >= p.batch) return 0;
        int lo, pos;
        bool bad;
        const int n = tiles_of<KT>(p, b, lo, pos, bad);
        return n > 0 ? (long long)(n + kItemCost) * p.items : 0;
    };
    // each lane sums up a run of sequences
    const int run = (p.batch + 31) / 32;
    long long mine = 0;
#pragma unroll 8
    for (int i = 0; i < run; ++i) mine += units(lane * run + i);
    const long long upto = scan(mine), total = __shfl_sync(0xffffffffu, upto, 31);
    Share s;
    const int most = blockDim.x / 32, warp = threadIdx.x / 32;
    s.warps = most;
    s.per = (total + (long long)gridDim.x * most - 1) / ((long long)gridDim.x * most);
    if (s.per <= kItemCost) {  // a tile at least, and with less than that for every warp all SMs rather than all warps of some
        s.per = kItemCost + 1;
        s.warps = (int)((total + gridDim.x * s.per - 1) / (gridDim.x * s.per));
        s.warps = max(min(s.warps, most), 1);
    }
    s.first = s.per * (blockIdx.x * (long long)s.warps + warp);
    s.end = warp >= s.warps ? s.first : s.first + s.per < total ? s.first + s.per : total;
    if (s.first >= s.end) return s;
    // the run that holds the first unit, and the sequence in it
    const int owner = __ffs(__ballot_sync(0xffffffffu, upto > s.first)) - 1;
    long long before = __shfl_sync(0xffffffffu, upto - mine, owner);
    for (int i = 0;; i += 32) {
        const int b = owner * run + i + lane;
        const long long own = i + lane < run ? units(b) : 0, sum = scan(own) + before;
        const uint32_t there = __ballot_sync(0xffffffffu, sum > s.first);
        if (there != 0) {
            const int l = __ffs(there) - 1;
            at.b = owner * run + i + l;
            before = __shfl_sync(0xffffffffu, sum - own, l);
            break;
        }
        before = __shfl_sync(0xffffffffu, sum, 31);
    }
    at.sequence(p);
    const long long inside = s.first - before;
    at.item = (int)(inside / at.n);
    at.t = (int)(inside - (long long)at.item * at.n);
    at.head = at.item / p.parts;
    return s;
}

// 1 / l, what a sum of weights turns into (the largest score's weight is 1 or more: no sum at all is that of scores of -inf)
__device__ __forceinline__ float inverse(float l) { return l == 0.f ? CUDART_NAN_F : 1.0f / l; }

__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}

// A warp's ring: tiles of keys, as many of values, and which of their rows are seen and which have no page.
struct Ring {
    unsigned char* tiles;
    uint2* marks;
};

// Brings a warp's tiles into its ring, one after the other.  Rows that do not count become zeros: whatever stands in a page behind
// a sequence's end, infinities and NaN among them, reaches no product.  A lane looks its row's page up a tile ahead of the copies
// that need it.  Where pages are made of sixteens, so are the tiles' runs of memory; else every row is found by itself.
template <typename T, int KT, typename Layout>
struct Loader {
    const PagedAttention& p;
    const Ring& ring;
    const Layout& lay;
    Cursor<KT> at;
    int j0, first, last;  // of the tile: its first key; rows first .. last are seen
    int slot, page;       // of this lane's row

    __device__ __forceinline__ bool persistent() const { return at.tile() < p.pers_tiles; }
    __device__ __forceinline__ int row_of_lane() const { return threadIdx.x & (KT - 1) & 31; }
    __device__ __forceinline__ void look() {
        const bool pers = persistent();
        const int r = row_of_lane();
        j0 = (pers ? at.tile() : at.lo / KT + at.tile() - p.pers_tiles) * KT;
        first = pers ? 0 : max(at.lo - j0, 0);
        last = min(pers ? p.np - 1 - j0 : at.pos - j0, KT - 1);
        if (!pers && r >= first && r <= last) {
            const uint32_t column = p.map.page.div((uint32_t)(j0 + r));
            slot = j0 + r - (int)(column * p.map.page.d);
            page = __ldg(p.map.table + at.b * p.map.table_stride + column);
        }
    }
    __device__ __forceinline__ void issue(int stage) {
        const int lane = threadIdx.x & 31, r = row_of_lane();
        const bool pers = persistent(), mine = r >= first && r <= last;
        const unsigned char *k, *v;
        long long row = -1;  // where this lane's row is, in elements
        if (pers) {
            k = static_cast<const unsigned char*>(p.k_pers);
            v = static_cast<const unsigned char*>(p.v_pers);
            if (mine) row = ((long long)at.head * p.np + j0 + r) * p.map.head_dim;
        } else {
            k = static_cast<const unsigned char*>(p.k_pages);
            v = static_cast<const unsigned char*>(p.v_pages);
            if (mine && (uint32_t)page < (uint32_t)p.map.pages)
                row = (((long long)page * p.map.kv_heads + at.head) * p.map.page.d + slot) * p.map.head_dim;
        }
        const uint32_t seen = (2u << last) - (1u << first), lost = __ballot_sync(0xffffffffu, mine && row < 0) & (0xffffffffu >> (32 - KT));
        if (lane == 0) ring.marks[stage] = make_uint2(seen, lost);
        const uint32_t to = (uint32_t)__cvta_generic_to_shared(ring.tiles) + stage * 2 * KT * lay.pitch();
        const int chunks = lay.chunks();
        // a lane's chunks, every 32nd one: chunk c of row rr (by steps: chunks is not always a constant)
        struct Chunk {
            int rr, c;
        };
        const Chunk start{lane / chunks, lane % chunks};
        auto after = [&](Chunk x) {
            x.rr += 32 / chunks;
            x.c += 32 % chunks;
            if (x.c >= chunks) x.c -= chunks, ++x.rr;
            return x;
        };
        if (pers || p.whole_runs) {
#pragma unroll
            for (int h = 0; h < KT / 16; ++h) {
                const int from = min(max(first, h * 16), KT - 1);  // a row that has the run's page, if any has
                const long long off = (__shfl_sync(0xffffffffu, row, from) - (from - h * 16) * p.map.head_dim) * (long long)sizeof(T) + lane * 16;
                const unsigned char *kr = k + off, *vr = v + off;
                const int n = 16 * chunks;
                const uint32_t want = seen >> (h * 16) & 0xffffu & ~(lost >> (h * 16));
                Chunk x = start;
                if (want == 0xffffu) {
#pragma unroll
                    for (int i0 = 0; i0 < n; i0 += 32, x = after(x)) {
                        if (n % 32 != 0 && x.rr >= 16) break;
                        const uint32_t dst = to + lay.offset(h * 16 + x.rr, x.c);
                        copy16(dst, kr + i0 * 16, true);
                        copy16(dst + KT * lay.pitch(), vr + i0 * 16, true);
                    }
                } else {
#pragma unroll 4
                    for (int i0 = 0; i0 < n; i0 += 32, x = after(x)) {
                        if (n % 32 != 0 && x.rr >= 16) break;
                        const uint32_t dst = to + lay.offset(h * 16 + x.rr, x.c);
                        const bool there = want >> x.rr & 1;  // (no byte is read where not: any address will do)
                        copy16(dst, there ? static_cast<const void*>(kr + i0 * 16) : p.sums, there);
                        copy16(dst + KT * lay.pitch(), there ? static_cast<const void*>(vr + i0 * 16) : p.sums, there);
                    }
                }
            }
        } else {
            Chunk x = start;
            for (int i0 = 0; i0 < KT * chunks; i0 += 32, x = after(x)) {
                const long long at_row = __shfl_sync(0xffffffffu, row, x.rr & (KT - 1));
                if (x.rr >= KT) continue;
                const bool there = at_row >= 0;
                const long long off = at_row * (long long)sizeof(T) + x.c * 16;
                const uint32_t dst = to + lay.offset(x.rr, x.c);
                copy16(dst, there ? static_cast<const void*>(k + off) : p.sums, there);
                copy16(dst + KT * lay.pitch(), there ? static_cast<const void*>(v + off) : p.sums, there);
            }
        }
    }
};

// ---- the core on CUDA cores: every type, head_dim a multiple of 8 --------------------------------------------------------
// Lane l has key l % 16 of a tile and one half of the head's dimensions of its scores; then the four dimensions from 4 l on (and
// from 128 + 4 l, with QUADS 2) of the outputs.  kRows query heads, their numbers as fp32 in shared memory.
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

template <typename T, int ROWS, int QUADS>
struct SimtCore {
    static constexpr int kRows = ROWS, KT = 16;
    using Layout = SimtLayout<T>;
    const PagedAttention& p;
    float* q;        // [kRows][head_dim], of the CTA's warp
    float* weights;  // [KT][kRows]
    float m[kRows], l[kRows];
    float4 o[kRows][QUADS];

    // shared memory of a warp besides its ring
    static __host__ __device__ int extra(int head_dim) { return (kRows * head_dim + KT * kRows) * (int)sizeof(float); }

    __device__ SimtCore(const PagedAttention& p, unsigned char* mine) : p(p), q(reinterpret_cast<float*>(mine)) {
        weights = q + kRows * p.map.head_dim;
    }
    __device__ __forceinline__ void load_queries(int b, int first, int rows) {
        const int lane = threadIdx.x & 31, dim = p.map.head_dim;
        __syncwarp();
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const T* from = static_cast<const T*>(p.q) + b * p.qs[0] + (first + r) * p.qs[1];
            for (int i = lane; i < dim; i += 32) q[r * dim + i] = r < rows ? to_f32<T>(from[i]) : 0.f;
        }
        __syncwarp();
    }
    __device__ __forceinline__ void reset() {
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            m[r] = -CUDART_INF_F;
            l[r] = 0.f;
#pragma unroll
            for (int h = 0; h < QUADS; ++h) o[r][h] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
    }
    __device__ __forceinline__ void tile(const unsigned char* tile, uint2 marks, const Layout& lay) {
        const int lane = threadIdx.x & 31, key = lane & (KT - 1), dim = p.map.head_dim, half = dim / 2;
        const unsigned char* row = tile + key * lay.pitch();
        float s[kRows] = {};
#pragma unroll 4
        for (int i = (lane >> 4) * half; i < (lane >> 4) * half + half; i += 4) {
            const float4 k4 = load4<T>(row + i * sizeof(T));
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                const float4 q4 = *reinterpret_cast<const float4*>(q + r * dim + i);
                s[r] = fmaf(q4.x, k4.x, fmaf(q4.y, k4.y, fmaf(q4.z, k4.z, fmaf(q4.w, k4.w, s[r]))));
            }
        }
        const bool seen = marks.x >> key & 1, bad = marks.y >> key & 1;
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
            for (int h = 0; h < QUADS; ++h) {
                o[r][h].x *= keep; o[r][h].y *= keep; o[r][h].z *= keep; o[r][h].w *= keep;
            }
        }
        if (lane < KT) {
#pragma unroll
            for (int r = 0; r < kRows; ++r) weights[key * kRows + r] = w[r];
        }
        __syncwarp();
        const unsigned char* values = tile + KT * lay.pitch();
#pragma unroll
        for (int h = 0; h < QUADS; ++h) {
            const int i = h * 128 + lane * 4;
            if (i >= dim) break;
#pragma unroll
            for (int j = 0; j < KT; ++j) {
                const float4 v4 = load4<T>(values + j * lay.pitch() + i * sizeof(T));
                float wj[kRows];
#pragma unroll
                for (int r = 0; r < kRows; r += 4) {
                    if constexpr (kRows >= 4) *reinterpret_cast<float4*>(wj + r) = *reinterpret_cast<const float4*>(weights + j * kRows + r);
                    else wj[r] = weights[j * kRows + r];
                }
#pragma unroll
                for (int r = 0; r < kRows; ++r) add_product(o[r][h], wj[r], v4);
            }
        }
        __syncwarp();
    }
    // use(row, its maximum, its sum, first dimension, up to four numbers of the output), from every lane that has some
    template <typename F>
    __device__ __forceinline__ void results(int rows, F&& use) {
        const int lane = threadIdx.x & 31, dim = p.map.head_dim;
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            float t = l[r];
#pragma unroll
            for (int d = 8; d > 0; d >>= 1) t += __shfl_xor_sync(0xffffffffu, t, d);
            if (r >= rows) continue;
#pragma unroll
            for (int h = 0; h < QUADS; ++h) {
                const float x[4] = {o[r][h].x, o[r][h].y, o[r][h].z, o[r][h].w};
                if (h * 128 + lane * 4 < dim) use(r, m[r], t, h * 128 + lane * 4, x);
            }
        }
    }
    __device__ __forceinline__ void store(T* to, int rows) {
        results(rows, [&](int r, float, float sum, int d, const float (&x)[4]) {
            const float scale = inverse(sum);
            T* at = to + r * p.os[1] + d;
#pragma unroll
            for (int e = 0; e < 4; ++e) at[e] = from_f32<T>(x[e] * scale);
        });
    }
};

// ---- the core on tensor cores: 16-bit types, head_dim 16, 32, 64, 80, 96, 128, 192 or 256 -------------------------------------------------
// mma.sync with the keys, then the dimensions of the values, as the sixteen rows of a tile and eight query heads as its columns
// (tcgen05's 64 or 128 rows would wait for as many keys per step, and the step is bound by HBM long before the tensor cores): the
// scores are K Q^T, their exponentials, turned over eight by eight (movmatrix), are the operand of V^T W^T.  A weight goes in as several
// 16-bit numbers that add up to it: three in bf16, all 24 bits; two in fp16, 22 bits, what the exponential itself has.  One alone
// would put up to 2^-8 of itself on the output, two in bf16 2^-16, which shows where values cancel.  In fp16 they are raised by
// 2^12, as far as the largest allows, so that those below 2^-14 of it keep their bits.  The products cut their sums off instead of
// rounding them, so a tile's begin at zero and are added to the outputs by themselves (all in one chain, a warp's 900 tiles brought
// its part 2^-12 nearer to zero), one chain for each sixteen keys (one for all 32: 12.4 us for 700 tokens instead of 10.9).  Up to
// eight heads: the tile's upper eight rows are zeros and have no registers.
template <int DH>
struct MmaLayout {
    int bytes;
    static constexpr bool kTurned = DH / 8 % 4 == 0;
    __host__ __device__ static constexpr int pitch() { return DH * 2 + (kTurned ? 0 : 16); }
    __host__ __device__ static constexpr int chunks() { return DH / 8; }
    // eight rows' same chunk stands on different banks: by its place in the row, or by rows of an odd number of chunks
    __device__ __forceinline__ static int offset(int r, int c) {
        const int turn = !kTurned ? 0 : chunks() % 8 == 0 ? r & 7 : r >> 1 & 3;
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
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

// Two weights as so many 16-bit numbers each: a weight cut off, what that lacks, cut off too but for the last one.  Of a weight that
// is not zero none is below the smallest number that a product takes (2^-126; 2^-24 under the raise, 2^-36 of the largest weight), so
// that all of them take an infinite value to the same infinity; of one that is zero all are.
constexpr int kMostTerms = 3;
template <typename T>
constexpr int kTerms = std::is_same<T, __half>::value ? 2 : 3;
template <typename T>
__device__ __forceinline__ void split2(float a, float b, uint32_t (&terms)[kMostTerms]);
template <>
__device__ __forceinline__ void split2<__nv_bfloat16>(float a, float b, uint32_t (&terms)[kMostTerms]) {
    const auto as_pair = [](uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); };
    const auto bits = [](__nv_bfloat162 v) { return *reinterpret_cast<const uint32_t*>(&v); };
    terms[0] = cut2<__nv_bfloat16>(a, b);
    const __nv_bfloat162 least = __hmin2(as_pair(terms[0]), as_pair(0x00800080u));
    const float2 first = unpack2<__nv_bfloat16>(terms[0]);
    a -= first.x, b -= first.y;
    terms[1] = bits(__hmax2(as_pair(cut2<__nv_bfloat16>(a, b)), least));
    const float2 second = unpack2<__nv_bfloat16>(terms[1]);
    terms[2] = bits(__hmax2(as_pair(pack2<__nv_bfloat16>(a - second.x, b - second.y)), least));
}
template <>
__device__ __forceinline__ void split2<__half>(float a, float b, uint32_t (&terms)[kMostTerms]) {
    const auto as_pair = [](uint32_t w) { return *reinterpret_cast<const __half2*>(&w); };
    const auto bits = [](__half2 v) { return *reinterpret_cast<const uint32_t*>(&v); };
    // (whether a weight is zero, from its upper sixteen bits: those of a positive number are in order in every format)
    const __half2 least = __hmin2(as_pair(cut2<__nv_bfloat16>(a, b)), as_pair(0x00010001u));
    terms[0] = bits(__hmax2_nan(as_pair(cut2<__half>(a, b)), least));
    const float2 first = unpack2<__half>(terms[0]);
    terms[1] = bits(__hmax2(as_pair(pack2<__half>(a - first.x, b - first.y)), least));
}

// an 8 x 8 matrix of 16-bit numbers, two of a row to a lane, with rows and columns exchanged
__device__ __forceinline__ uint32_t turned(uint32_t w) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(w));
    return r;
}

// EIGHTS: of query heads; lane l has heads l % 4 * 2 and the next one of each eight
template <typename T, int DH, int EIGHTS>
struct MmaCore {
    static constexpr int kRows = kMaxRows, KT = DH > 128 ? 16 : 32;
    static constexpr float kRaise = std::is_same<T, __half>::value ? 12.f : 0.f;
    using Layout = MmaLayout<DH>;
    const PagedAttention& p;
    uint32_t q[EIGHTS][DH / 16][2];
    float m[EIGHTS][2], l[EIGHTS][2];  // l: of this lane's keys
    float o[EIGHTS][DH / 16][4];       // dimension 16 k + lane / 4 of both heads, 16 k + 8 + lane / 4 of both

    static __host__ __device__ int extra(int) { return 0; }

    __device__ MmaCore(const PagedAttention& p, unsigned char*) : p(p) {}
    __device__ __forceinline__ void load_queries(int b, int first, int rows) {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int h = 0; h < EIGHTS; ++h) {
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
                    q[h][k][i] = w;
                }
        }
    }
    __device__ __forceinline__ void reset() {
#pragma unroll
        for (int h = 0; h < EIGHTS; ++h) {
            m[h][0] = m[h][1] = -CUDART_INF_F;
            l[h][0] = l[h][1] = 0.f;
#pragma unroll
            for (int k = 0; k < DH / 16; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[h][k][i] = 0.f;
        }
    }
    __device__ __forceinline__ void tile(const unsigned char* tile, uint2 marks, const Layout& lay) {
        const int lane = threadIdx.x & 31;
        const uint32_t keys = (uint32_t)__cvta_generic_to_shared(tile), values = keys + KT * Layout::pitch();
        float s[EIGHTS][KT / 16][4];  // of each sixteen: keys lane / 4 and 8 + lane / 4, both heads each
#pragma unroll
        for (int h = 0; h < EIGHTS; ++h)
#pragma unroll
            for (int g = 0; g < KT / 16; ++g)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[h][g][i] = 0.f;
#pragma unroll
        for (int k = 0; k < DH / 16; ++k)
#pragma unroll
            for (int g = 0; g < KT / 16; ++g) {
                uint32_t a[4];
                ldmatrix4(a, keys + lay.offset(g * 16 + (lane & 15), k * 2 + (lane >> 4)));
#pragma unroll
                for (int h = 0; h < EIGHTS; ++h) mma_16816<T>(s[h][g], a[0], a[1], a[2], a[3], q[h][k][0], q[h][k][1]);
            }
        uint32_t weights[EIGHTS][KT / 16][2][kMostTerms];
        float keep[EIGHTS][2];
#pragma unroll
        for (int h = 0; h < EIGHTS; ++h) {
            float base[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float top = -CUDART_INF_F;
#pragma unroll
                for (int g = 0; g < KT / 16; ++g)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int key = g * 16 + i * 8 + lane / 4;
                        float& x = s[h][g][i * 2 + e];
                        x *= p.scale;
                        if (marks.x != 0xffffffffu >> (32 - KT) || marks.y != 0)
                            x = marks.y >> key & 1 ? CUDART_NAN_F : marks.x >> key & 1 ? x : -CUDART_INF_F;
                        top = fmaxf(top, x);
                    }
#pragma unroll
                for (int d = 4; d < 32; d *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                const float now = fmaxf(m[h][e], top);
                base[e] = now == -CUDART_INF_F ? 0.f : now;
                keep[h][e] = m[h][e] == -CUDART_INF_F ? 1.f : ex2_ftz(m[h][e] - base[e]);  // (nothing to keep, or NaN)
                m[h][e] = now;
                l[h][e] *= keep[h][e];
            }
#pragma unroll
            for (int g = 0; g < KT / 16; ++g)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float w[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        w[e] = ex2_ftz(s[h][g][i * 2 + e] - base[e] + kRaise);
                        l[h][e] += w[e];
                    }
                    split2<T>(w[0], w[1], weights[h][g][i]);
#pragma unroll
                    for (int t = 0; t < kTerms<T>; ++t) weights[h][g][i][t] = turned(weights[h][g][i][t]);
                }
        }
#pragma unroll
        for (int k = 0; k < DH / 16; ++k) {
            float sum[KT / 16][EIGHTS][4];  // of this tile
            uint32_t a[KT / 16][4];
#pragma unroll
            for (int g = 0; g < KT / 16; ++g) {
                ldmatrix4_trans(a[g], values + lay.offset(g * 16 + (lane >> 4) * 8 + (lane & 7), k * 2 + (lane >> 3 & 1)));
#pragma unroll
                for (int h = 0; h < EIGHTS; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) sum[g][h][i] = 0.f;
            }
#pragma unroll
            for (int t = 0; t < kTerms<T>; ++t)
#pragma unroll
                for (int g = 0; g < KT / 16; ++g)
#pragma unroll
                    for (int h = 0; h < EIGHTS; ++h)
                        mma_16816<T>(sum[g][h], a[g][0], a[g][1], a[g][2], a[g][3], weights[h][g][0][t], weights[h][g][1][t]);
#pragma unroll
            for (int h = 0; h < EIGHTS; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float x = sum[0][h][i];
#pragma unroll
                    for (int g = 1; g < KT / 16; ++g) x += sum[g][h][i];
                    o[h][k][i] = fmaf(o[h][k][i], keep[h][i & 1], x);
                }
        }
    }
    template <typename F>
    __device__ __forceinline__ void results(int rows, F&& use) {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int h = 0; h < EIGHTS; ++h)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = h * 8 + lane % 4 * 2 + e;
                float t = l[h][e];
#pragma unroll
                for (int d = 4; d < 32; d *= 2) t += __shfl_xor_sync(0xffffffffu, t, d);
                if (r >= rows) continue;
#pragma unroll
                for (int k = 0; k < DH / 16; ++k)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float x[1] = {o[h][k][i * 2 + e]};
                        use(r, m[h][e], t, k * 16 + i * 8 + lane / 4, x);
                    }
            }
    }
    // rounded, and turned over eight by eight so that a lane has two neighbouring dimensions of one head
    __device__ __forceinline__ void store(T* to, int rows) {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int h = 0; h < EIGHTS; ++h) {
            float scale[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float t = l[h][e];
#pragma unroll
                for (int d = 4; d < 32; d *= 2) t += __shfl_xor_sync(0xffffffffu, t, d);
                scale[e] = inverse(t);
            }
            const int r = h * 8 + lane / 4;
            T* at = to + r * p.os[1] + lane % 4 * 2;
#pragma unroll
            for (int k = 0; k < DH / 16; ++k)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t w = turned(pack2<T>(o[h][k][i * 2] * scale[0], o[h][k][i * 2 + 1] * scale[1]));
                    if (r >= rows) continue;
                    if (p.o_pairs) {
                        *reinterpret_cast<uint32_t*>(at + k * 16 + i * 8) = w;
                    } else {
                        reinterpret_cast<uint16_t*>(at)[k * 16 + i * 8] = (uint16_t)w;
                        reinterpret_cast<uint16_t*>(at)[k * 16 + i * 8 + 1] = (uint16_t)(w >> 16);
                    }
                }
        }
    }
};

// ---- the line of tiles ------------------------------------------------------------------------------------------------------

// weight of a part whose maximum is m under the common one (base: that, or 0 where it is -inf): a part of hidden scores alone
// holds zeros, or NaN that has to stay
__device__ __forceinline__ float part_weight(float m, float base) { return m == -CUDART_INF_F ? 1.f : exp2f(m - base); }

// A warp's part of an item that was cut: of the one that its piece begins in (0), of the one that begins in it (1).
struct Part {
    int there, b, item, starts, ends;
    long long item_end;
};

template <typename T, typename Core, int W, int S>  // up to W warps
__global__ void __launch_bounds__(W * 32) paged_attention_kernel(const __grid_constant__ PagedAttention p) {
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int KT = Core::KT;
    __shared__ uint2 marks[W][S];
    __shared__ Part parts[2 * W];
    pdl_trigger();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x / 32, dim = p.map.head_dim;
    const typename Core::Layout lay{p.row_bytes};
    const int ring_bytes = S * 2 * KT * lay.pitch(), extra = Core::extra(dim);
    unsigned char* mine = smem + warp * (ring_bytes + extra);
    const Ring ring{mine, marks[warp]};
    float2* part_sums = reinterpret_cast<float2*>(smem + warps * (ring_bytes + extra));  // [2 * warps][rows]
    // a warp's first part [rows][head_dim] goes through memory; its second one, made when all its tiles are done, where they were
    auto part_out = [&](int w, int which) {
        return which == 0 ? p.firsts + (blockIdx.x * warps + w) * (long long)p.rows * dim
                          : reinterpret_cast<float*>(smem + w * (ring_bytes + extra));
    };

    if (tid == 0) p.joins[blockIdx.x] = make_int4(-1, 0, 0, 0);
    if (lane < 2) parts[2 * warp + lane].there = 0;
    __syncwarp();

    Cursor<KT> at;
    const Share share = find_share<KT>(p, at);
    if (share.first < share.end) {
        Loader<T, KT, typename Core::Layout> ahead{p, ring, lay, at};  // of the tile to load next, unit `load` of the line
        long long load = share.first;
        int stage_in = 0, stage_out = 0;
        auto look = [&]() {
            if (load < share.end && ahead.at.t < kItemCost) {
                load += kItemCost - ahead.at.t;
                ahead.at.t = kItemCost;
            }
            if (load < share.end) ahead.look();
        };
        auto fetch = [&]() {
            if (load < share.end) {
                ahead.issue(stage_in);
                if (++load < share.end && ++ahead.at.t == ahead.at.n) ahead.at.next_item(p);
                look();
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            stage_in = stage_in + 1 == S ? 0 : stage_in + 1;
        };
        look();
#pragma unroll
        for (int s = 0; s < S - 1; ++s) fetch();

        Core core(p, mine + ring_bytes);
        auto queries = [&](const Cursor<KT>& c, int& head, int& rows) {  // the item's first head, and how many
            const int first = (c.item - c.head * p.parts) * p.rows;
            rows = min(p.rows, p.group - first);
            head = c.head * p.group + first;
            core.load_queries(c.b, head, rows);
        };
        long long begin = share.first;
        bool bad_page = false;
        int head, rows;
        queries(at, head, rows);
        while (begin < share.end) {
            const long long item_end = begin + (at.n - at.t), end = item_end < share.end ? item_end : share.end;
            const int tiles = (int)(end - begin) - max(kItemCost - at.t, 0);
            core.reset();
            for (int i = 0; i < tiles; ++i) {
                asm volatile("cp.async.wait_group %0;" ::"n"(S - 2) : "memory");
                __syncwarp();
                fetch();
                const uint2 mark = ring.marks[stage_out];
                bad_page |= mark.y != 0;
                core.tile(ring.tiles + stage_out * 2 * KT * lay.pitch(), mark, lay);
                stage_out = stage_out + 1 == S ? 0 : stage_out + 1;
            }
            const Cursor<KT> done = at;
            const int done_head = head, done_rows = rows;
            if (item_end < share.end) {  // the next item's queries load while this one's results are stored
                at.next_item(p);
                queries(at, head, rows);
            }
            begin = end;
            if (tiles <= 0) continue;
            const bool starts = done.t <= kItemCost, ends = end == item_end;
            if (starts && ends) {
                T* to = static_cast<T*>(p.o) + done.b * p.os[0] + done_head * p.os[1];
                core.store(to, done_rows);
            } else {
                const int which = starts ? 1 : 0;
                __syncwarp();
                float* to = part_out(warp, which);
                float2* sums = part_sums + (2 * warp + which) * p.rows;
                core.results(done_rows, [&](int r, float top, float sum, int d, const auto& x) {
                    constexpr int N = sizeof(x) / sizeof(float);
                    if (d == 0) sums[r] = make_float2(top, sum);
#pragma unroll
                    for (int e = 0; e < N; ++e) to[r * dim + d + e] = x[e];
                });
                if (lane == 0) parts[2 * warp + which] = {1, done.b, done.item, starts, ends, item_end};
            }
        }
        if (bad_page && lane == 0) atomicCAS(p.status, 0, (int)TMW_ERR_INVALID_ARGUMENT);
    }
    __syncthreads();

    // The CTA's parts of one item are neighbours: one that begins here, or that the CTA begins in, and those that go on with it.
    // Each item's numbers, four to a thread, begin with the thread behind the last one's.
    const uint32_t there = __ballot_sync(0xffffffffu, lane < 2 * warps && parts[lane].there);
    int turn = 0;
    for (uint32_t todo = there & (0xaaaaaaaau | 1u); todo != 0; todo &= todo - 1) {
        const int i = __ffs(todo) - 1;
        const uint32_t rest = todo & (todo - 1), members = there & ~((1u << i) - 1) & (rest != 0 ? (rest & (0u - rest)) - 1 : 0xffffffffu);
        const Part part = parts[i];
        const bool starts = part.starts, ends = parts[31 - __clz(members)].ends;
        const int first = part.item % p.parts * p.rows, rows = min(p.rows, p.group - first);
        const int head = part.item / p.parts * p.group + first;
        const long long slot = (blockIdx.x * 2 + (starts ? 1 : 0)) * (long long)p.rows;
        const int units = rows * dim / 4;
        int x = tid - turn;
        if (x < 0) x += blockDim.x;
        for (; x < units; x += blockDim.x) {
            const int r = x * 4 / dim;
            float m = -CUDART_INF_F, l = 0.f;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
            for (uint32_t j = members; j != 0; j &= j - 1) m = fmaxf(m, part_sums[(__ffs(j) - 1) * p.rows + r].x);
            const float base = m == -CUDART_INF_F ? 0.f : m;
#pragma unroll 4
            for (uint32_t j = members; j != 0; j &= j - 1) {
                const int at = __ffs(j) - 1;
                const float2 sum = part_sums[at * p.rows + r];
                const float w = part_weight(sum.x, base);
                l = fmaf(w, sum.y, l);
                add_product(o, w, reinterpret_cast<const float4*>(part_out(at >> 1, at & 1))[x]);
            }
            if (starts && ends) {
                T* to = static_cast<T*>(p.o) + part.b * p.os[0] + (head + r) * p.os[1] + (x * 4 - r * dim);
                const float scale = inverse(l);
                to[0] = from_f32<T>(o.x * scale);
                to[1] = from_f32<T>(o.y * scale);
                to[2] = from_f32<T>(o.z * scale);
                to[3] = from_f32<T>(o.w * scale);
            } else {
                reinterpret_cast<float4*>(p.partial + slot * dim)[x] = o;
                if (x * 4 == r * dim) p.sums[slot + r] = make_float2(m, l);
            }
        }
        turn = (turn + units) % blockDim.x;
        if (starts && !ends && tid == 0)
            p.joins[blockIdx.x] = make_int4(part.b, part.item, (int)((part.item_end - 1) / (share.per * share.warps)), 0);
    }

    // sequences without a key to see, or without a place
    for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
        int lo, pos;
        bool bad;
        if (tiles_of<KT>(p, b, lo, pos, bad) > 0) continue;
        if (bad && tid == 0) atomicCAS(p.status, 0, (int)TMW_ERR_INVALID_ARGUMENT);
        const int heads = p.group * p.map.kv_heads;
        for (int i = tid; i < heads * dim; i += blockDim.x)
            static_cast<T*>(p.o)[b * p.os[0] + (i / dim) * p.os[1] + i % dim] = from_f32<T>(bad ? CUDART_NAN_F : 0.f);
    }
}

// The parts of an item that was cut: CTA (c, .) joins 128 dimensions of a row of the one that begins in CTA c.  Its warps take every
// kJoinWarps-th part each, a lane four dimensions, kJoinAhead parts on their way at once.  The first two parts, mostly all there are,
// load before it is known whether there is an item (one sequence of 65536 tokens in 148 parts: 20.7 us the two kernels, with one part
// at a time 22.7; 700 tokens: 10.9, 12.4).
constexpr int kJoinWarps = 8, kJoinAhead = 6;
template <typename T>
__global__ void __launch_bounds__(kJoinWarps * 32) paged_join_kernel(const __grid_constant__ PagedAttention p) {
    __shared__ float2 warp_sums[kJoinWarps];
    __shared__ float4 outs[kJoinWarps][32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, dim = p.map.head_dim;
    const int r = blockIdx.y % p.rows, d = blockIdx.y / p.rows * 128 + lane * 4;
    auto slot = [&](int i) { return (2LL * (blockIdx.x + i) + (i == 0 ? 1 : 0)) * p.rows + r; };
    float2 ml[kJoinAhead];
    float4 part[kJoinAhead];
    auto load = [&](int i, float2& sums, float4& out) {
        sums = __ldcg(p.sums + slot(i));
        if (d < dim) out = __ldcg(reinterpret_cast<const float4*>(p.partial + slot(i) * dim + d));
    };
    pdl_wait();
    const int4 join = __ldcg(p.joins + blockIdx.x);
    if (warp < 2) load(warp, ml[0], part[0]);  // (there is a CTA behind this one: never past the scratch memory)
    if (join.x < 0) return;
    const int first = join.y % p.parts * p.rows;
    if (r >= min(p.rows, p.group - first)) return;
    const int n = join.z - (int)blockIdx.x + 1;
    float m = -CUDART_INF_F, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = warp; i0 < n; i0 += kJoinWarps * kJoinAhead) {
#pragma unroll
        for (int j = 0; j < kJoinAhead; ++j) {
            const int i = i0 + j * kJoinWarps;
            if (i >= 2 && i < n) load(i, ml[j], part[j]);
        }
#pragma unroll
        for (int j = 0; j < kJoinAhead; ++j) {
            if (i0 + j * kJoinWarps >= n) break;
            const float now = fmaxf(m, ml[j].x), base = now == -CUDART_INF_F ? 0.f : now, keep = part_weight(m, base),
                        w = part_weight(ml[j].x, base);
            m = now;
            l = fmaf(w, ml[j].y, l * keep);
            o.x *= keep; o.y *= keep; o.z *= keep; o.w *= keep;
            if (d < dim) add_product(o, w, part[j]);
        }
    }
    if (lane == 0) warp_sums[warp] = make_float2(m, l);
    outs[warp][lane] = o;
    __syncthreads();
    if (warp != 0 || d >= dim) return;
#pragma unroll
    for (int w = 1; w < kJoinWarps; ++w) m = fmaxf(m, warp_sums[w].x);
    const float base = m == -CUDART_INF_F ? 0.f : m;
    float sum = 0.f;
    float4 out = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) {
        const float x = part_weight(warp_sums[w].x, base);
        sum = fmaf(x, warp_sums[w].y, sum);
        add_product(out, x, outs[w][lane]);
    }
    const float scale = inverse(sum);
    T* to = static_cast<T*>(p.o) + join.x * p.os[0] + (join.y / p.parts * p.group + first + r) * p.os[1] + d;
    to[0] = from_f32<T>(out.x * scale);
    to[1] = from_f32<T>(out.y * scale);
    to[2] = from_f32<T>(out.z * scale);
    to[3] = from_f32<T>(out.w * scale);
}

// ---- host ---------------------------------------------------------------------------------------------------------------------

// Shared memory of a CTA, one to an SM: with much more, what is left of the SM's memory as L1 is too little for the copies on their
// way, and they come from L2 twice (32 heads on 4, 553,000 tokens, rings of three tiles in 226 KB: 231 us when this took 189).  Head
// size 64 has eleven warps here; with twelve its 256 windows of 512 take the same 68.5 us.
constexpr int kMostShared = 193 * 1024 + 512;

struct Plan {
    int rows, parts, warps, grid, smem;
    size_t sums_at, partial_at, firsts_at, bytes;
};

template <typename T, typename Core, int W, int S>
struct Kernel {
    static constexpr int KT = Core::KT;
    static Plan plan(const tmw_paged_attention_desc& d, int row_bytes) {
        Plan n;
        const int group = d.heads / d.at.kv_heads;
        n.parts = (group + Core::kRows - 1) / Core::kRows;
        n.rows = (group + n.parts - 1) / n.parts;
        const int warp = S * 2 * KT * typename Core::Layout{row_bytes}.pitch() + Core::extra(d.at.head_dim) + 2 * n.rows * (int)sizeof(float2);
        n.warps = kMostShared / warp < W ? kMostShared / warp : W;
        n.smem = n.warps * warp;
        // no more CTAs than the longest sequences could have work for
        const long long capacity = (long long)d.at.columns * d.at.page_size;
        const long long keys = d.window >= 0 && d.window + 1LL < capacity ? d.window + 1LL : capacity;
        const long long tiles = ((d.n_persistent + KT - 1) / KT + keys / KT + 2) * (long long)d.at.kv_heads * n.parts * d.at.batch;
        n.grid = (int)(tiles < sm_count() ? tiles : sm_count());
        const size_t out = (size_t)n.rows * d.at.head_dim * sizeof(float);
        n.sums_at = (size_t)n.grid * sizeof(int4);
        n.partial_at = (n.sums_at + (size_t)n.grid * 2 * n.rows * sizeof(float2) + 15) & ~(size_t)15;
        n.firsts_at = n.partial_at + n.grid * 2 * out;
        n.bytes = n.firsts_at + (size_t)n.grid * n.warps * out;
        return n;
    }
    static int launch(PagedAttention& p, const Plan& n, unsigned char* scratch, cudaStream_t stream) {
        p.rows = n.rows;
        p.parts = n.parts;
        p.items = p.map.kv_heads * n.parts;
        p.pers_tiles = (p.np + KT - 1) / KT;
        p.joins = reinterpret_cast<int4*>(scratch);
        p.sums = reinterpret_cast<float2*>(scratch + n.sums_at);
        p.partial = reinterpret_cast<float*>(scratch + n.partial_at);
        p.firsts = reinterpret_cast<float*>(scratch + n.firsts_at);
        auto kern = paged_attention_kernel<T, Core, W, S>;
        const int rc = allow_shared_memory(reinterpret_cast<const void*>(kern), n.smem);
        if (rc != TMW_OK) return rc;
        kern<<<n.grid, n.warps * 32, n.smem, stream>>>(p);
        TMW_CUDA_TRY(cudaGetLastError());
        if (n.grid > 1)
            TMW_CUDA_TRY(launch_ex(paged_join_kernel<T>, dim3((unsigned)n.grid - 1, (unsigned)(n.rows * ((p.map.head_dim + 127) / 128))),
                                   dim3(kJoinWarps * 32), 0, stream, true, 1, p));
        return TMW_OK;
    }
};

// as many query heads at once as a group has, up to four, or eight where a lane has four dimensions of each
template <typename T, typename F>
int with_simt(const tmw_paged_attention_desc& d, F&& use) {
    const int group = d.heads / d.at.kv_heads;
    if (d.at.head_dim > 128) return group == 1 ? use(Kernel<T, SimtCore<T, 1, 2>, 12, 2>()) : use(Kernel<T, SimtCore<T, 4, 2>, 12, 2>());
    if (group == 1) return use(Kernel<T, SimtCore<T, 1, 1>, 12, 2>());
    return group <= 4 ? use(Kernel<T, SimtCore<T, 4, 1>, 12, 2>()) : use(Kernel<T, SimtCore<T, 8, 1>, 12, 2>());
}
template <typename T, int DH, typename F>
int with_mma(const tmw_paged_attention_desc& d, F&& use) {
    constexpr int W = DH >= 128 ? 6 : DH > 64 ? 8 : 12;
    if (d.heads / d.at.kv_heads <= 8) return use(Kernel<T, MmaCore<T, DH, 1>, W, 2>());
    return use(Kernel<T, MmaCore<T, DH, 2>, W, 2>());
}
template <typename T, typename F>
int with_16_bits(const tmw_paged_attention_desc& d, F&& use) {
    switch (d.at.head_dim) {
        case 16: return with_mma<T, 16>(d, use);
        case 32: return with_mma<T, 32>(d, use);
        case 64: return with_mma<T, 64>(d, use);
        case 80: return with_mma<T, 80>(d, use);
        case 96: return with_mma<T, 96>(d, use);
        case 128: return with_mma<T, 128>(d, use);
        case 192: return with_mma<T, 192>(d, use);
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
    if (d->o == d->q) {
        set_error_text("tmw_paged_attention: o must not be q (other CTAs may still read it)");
        return TMW_ERR_INVALID_ARGUMENT;
    }
    if (d->q == nullptr || d->o == nullptr || d->pos == nullptr || scratch == nullptr ||
        (d->n_persistent > 0 && (d->k_pers == nullptr || d->v_pers == nullptr)))
        return TMW_ERR_INVALID_ARGUMENT;
    for (int i = 0; i < 2; ++i)
        if (d->q_stride[i] < 0 || d->o_stride[i] < 0) return TMW_ERR_INVALID_ARGUMENT;
    if (!rows_apart(d->o_stride, {d->at.batch, d->heads})) {
        set_error_text("tmw_paged_attention: every output must have a place of its own");
        return TMW_ERR_INVALID_ARGUMENT;
    }
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
    p.whole_runs = d->at.page_size % 16 == 0;
    p.group = d->heads / d->at.kv_heads;
    p.scale = (d->scale > 0.f ? d->scale : 1.0f / sqrtf((float)d->at.head_dim)) * 1.4426950408889634f;
    p.row_bytes = d->at.head_dim * (int)size;
    p.q_pairs = bits(d->q) % 4 == 0 && (d->q_stride[0] | d->q_stride[1]) % 2 == 0;
    p.o_pairs = bits(d->o) % 4 == 0 && (d->o_stride[0] | d->o_stride[1]) % 2 == 0;
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
