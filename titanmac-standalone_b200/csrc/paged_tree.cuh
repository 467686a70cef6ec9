// Attention of the drafted tokens of a tree over paged keys: the kernel on tensor cores (16-bit queries, head_dim 32, 64, 96, 128 or 256).
//
// For a key head the rows are the (node, query head) pairs that read it, up to 64 x 8 and more of them; a row sees the persistent keys,
// the cached tokens (from its own window's begin on) and the nodes of its word of bits.  Each key is read once for a block of up to 192
// rows: a worker of 1 to 12 warps, sixteen rows to a warp, shares a ring of tiles of 32 keys that the first of its warps has brought by
// TMA (pages made of eights; else by 16-byte copies), and the workers of all CTAs have equal pieces of the line of tiles, as in the
// attention of one token.  No barrier but the ring's own.
//
// S = Q K^T and O += P V by mma.sync with the rows as the sixteen of a tile: the scores' registers are the operand of the second
// product as they are.  (Here M is what bounds it: 2.25 cycles of the SM for each 16 x 8 x 16; which rows tcgen05's 128 take instead is
// said below, at tree_takes_tc.)  64 windows of 512, 16 nodes, 10 heads of 64, bf16, 86 MB: 39 us, a third of the issue slots: seven or eight tiles to a worker and eighteen to an
// item, so that every item is cut, and its parts go through memory twice.  A weight is two 16-bit numbers, as far as a tile's mask goes; only tiles that some row does not see in full, at the
// window's begin and among the nodes, run the body with the mask.
#pragma once

#include "paged_attention.cuh"

namespace tmw {
namespace {

// keys of a tile; what an item costs besides its tiles (2 | 4 | 7: 60 ragged sequences of up to 1000, 4 nodes, 32 heads on 4 of 128, codes,
// 42 | 44 | 46 us; equal pieces to a warp, as with windows, the same)
constexpr int kTreeKeys = 32, kTreeCost = 2;
constexpr int kMostSlots = 16, kMostTree = 212 * 1024;  // slots of a ring; bytes of rings and rows

// d = a b (+ d) in the type of P's products
template <typename M>
__device__ __forceinline__ void mma_from_zero(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_from_zero<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
template <>
__device__ __forceinline__ void mma_from_zero<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
template <typename M>
__device__ __forceinline__ void mma_onto_it(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_onto_it<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_onto_it<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Two weights as two 16-bit numbers each: cut off, and what that lacks.  Of a weight that is not zero neither is, so that both take an
// infinite value to the same infinity (see split2).  In bf16 these are 16 bits, where the attention of one token takes three numbers and 24:
// a third product for each is what bounds this kernel, and on tcgen05 three numbers of 64 weights do not fit over their scores' columns.
// 2^-16 of a weight is a 128th of an output's half step and shows where values cancel: of 64 windows' outputs 4 in 1000 are not the rounded
// exact ones (of one token's 2 in 10,000, of the formula's in fp32 4).
template <typename M>
__device__ __forceinline__ void split_in_two(float a, float b, uint32_t& first, uint32_t& second) {
    if constexpr (std::is_same<M, __half>::value) {
        uint32_t terms[kMostTerms];
        split2<__half>(a, b, terms);
        first = terms[0], second = terms[1];
    } else {
        const auto as_pair = [](uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); };
        first = cut2<__nv_bfloat16>(a, b);
        const __nv_bfloat162 least = __hmin2(as_pair(first), as_pair(0x00800080u));
        const float2 had = unpack2<__nv_bfloat16>(first);
        const __nv_bfloat162 rest = __hmax2(as_pair(pack2<__nv_bfloat16>(a - had.x, b - had.y)), least);
        second = *reinterpret_cast<const uint32_t*>(&rest);
    }
}
// One warp's sixteen rows of an item.  P: of keys and values; M: of the products, P itself or fp16 for codes of 8 bits.
template <typename P, int DH>
struct TreeCore {
    static constexpr bool k8 = kScaled<P>, kMayBeWild = !std::is_same<P, int8_t>::value;  // infinities and NaN among the values
    using M = std::conditional_t<k8, __half, P>;
    static constexpr int KT = kTreeKeys, kRowBytes = DH * (int)sizeof(P), kSteps = DH / 16;
    static constexpr float kRaise = std::is_same<M, __half>::value ? 12.f : 0.f;
    using Layout = BoxLayout<kRowBytes>;
    // What a warp has of its rows in shared memory (in registers the queries alone would be 32 of head_dim 128, next to 64 of
    // outputs): the queries, a row's sixteen bytes off the last one's banks, the first token that a row sees, the nodes that it sees.
    static constexpr int kQueryPitch = DH * 2 + 16, kQueries = 16 * kQueryPitch, kRowsBytes = kQueries + 16 * 16;
    const PagedAttention& p;
    unsigned char* mine;
    float q_scale[2];   // of rows lane / 4 and 8 + lane / 4
    float m[2], l[2];   // l: of this lane's keys
    float o[DH / 8][4]; // 16-bit pages: dimensions 8 n + 2 t and the next, of both rows; codes: see dim_of
    int start, lowest;  // tokens in front of the nodes, the last begin of a row's window

    __device__ __forceinline__ TreeCore(const PagedAttention& p, unsigned char* mine) : p(p), mine(mine) {}
    __device__ __forceinline__ uint64_t* nodes_of(int r) const { return reinterpret_cast<uint64_t*>(mine + kQueries + r * 16); }
    __device__ __forceinline__ int* low_of(int r) const { return reinterpret_cast<int*>(mine + kQueries + r * 16 + 8); }
    // 16-bit pages: the first of a lane's two neighbouring dimensions of tile n.  Codes: tiles 2 c and 2 c + 1 have the even and the odd
    // dimensions of the sixteen from 16 c on, a lane's four are neighbours.
    __device__ __forceinline__ static int dim_of(int n) { return (threadIdx.x & 3) * (k8 ? 4 : 2) + (k8 ? n / 2 * 16 : n * 8); }

    __device__ __forceinline__ void load_queries(const Rows& of, int count, int warp_rows) {
        const int lane = threadIdx.x & 31, t = lane & 3;
        start = __ldg(p.pos + of.b);
        lowest = 0;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int own = i * 8 + lane / 4, r = warp_rows + own;
            const bool there = r < of.n;
            const int node = (of.first + r) / p.group;
            const int low = there ? first_seen(p, of.b, start, node) : 0;
            lowest = max(lowest, low);
            if (t == 0) {
                *low_of(own) = low;
                *nodes_of(own) = there ? nodes_seen(p, of.b, count, node) : 0;
            }
            const uint16_t* from = static_cast<const uint16_t*>(p.q) + (there ? row_at<true>(p, p.qs, of, r) : 0);
            uint32_t w[kSteps][2];
            float top = 0.f;
#pragma unroll
            for (int k = 0; k < kSteps; ++k)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint16_t* at = from + k * 16 + (k8 ? t * 4 + h * 2 : t * 2 + h * 8);
                    w[k][h] = 0;
                    if (there) w[k][h] = p.q_pairs ? *reinterpret_cast<const uint32_t*>(at) : at[0] | (uint32_t)at[1] << 16;
                    if constexpr (k8) {
                        const float2 x = unpack2<__nv_bfloat16>(w[k][h]);
                        top = fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y)));
                    }
                }
            q_scale[i] = p.scale;
            if constexpr (k8) {  // bf16 as fp16 times a power of two of the row's own; then in the order of the codes
                if (p.bf16) {
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    const int e = max((__float_as_int(top) >> 23) - 127, -100);
                    const float up = __int_as_float((127 + 14 - e) << 23);
                    q_scale[i] *= __int_as_float((127 - 14 + e) << 23);
#pragma unroll
                    for (int k = 0; k < kSteps; ++k)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float2 x = unpack2<__nv_bfloat16>(w[k][h]);
                            w[k][h] = pack2<__half>(x.x * up, x.y * up);
                        }
                }
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                    const uint32_t a = w[k][0], b = w[k][1];
                    w[k][0] = __byte_perm(a, b, 0x5410);
                    w[k][1] = __byte_perm(a, b, 0x7632);
                }
            }
#pragma unroll
            for (int k = 0; k < kSteps; ++k)
#pragma unroll
                for (int h = 0; h < 2; ++h) *reinterpret_cast<uint32_t*>(mine + own * kQueryPitch + k * 32 + h * 16 + t * 4) = w[k][h];
        }
        for (int d = 4; d < 32; d *= 2) lowest = max(lowest, __shfl_xor_sync(0xffffffffu, lowest, d));
        __syncwarp();
    }
    __device__ __forceinline__ void reset() {
#pragma unroll
        for (int i = 0; i < 2; ++i) m[i] = -CUDART_INF_F, l[i] = 0.f;
#pragma unroll
        for (int n = 0; n < DH / 8; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[n][i] = 0.f;
    }
    // MASKED: some row may not see some key.
    template <bool MASKED>
    __device__ __forceinline__ void tile(const Ring& ring, int slot, uint2 marks, int place) {
        const int lane = threadIdx.x & 31, t = lane & 3;
        const uint32_t keys = (uint32_t)__cvta_generic_to_shared(ring.tiles) + slot * 2 * KT * kRowBytes, values = keys + KT * kRowBytes;
        const uint32_t query_at = (uint32_t)__cvta_generic_to_shared(mine) + (lane & 15) * kQueryPitch + (lane >> 4) * 16;
        float s[KT / 8][4];
        // of 16-bit rows: eight keys' first and second chunk of a step, then the next eight's; of codes two steps of eight keys, of the next eight
        const uint32_t key_at = Layout::offset((lane >> 4) * 8 + (lane & 7), lane >> 3 & 1);
        const auto chunk_at = [&](uint32_t at, int g, int c) {
            constexpr int in = Layout::kInBox;
            return (at ^ (c % in << 4)) + c / in * KT * Layout::kBoxBytes + g * 16 * Layout::kBoxBytes;
        };
#pragma unroll
        for (int c = 0; c < kRowBytes / 16; c += 2) {
            uint32_t q[k8 ? 2 : 1][4];
#pragma unroll
            for (int h = 0; h < (k8 ? 2 : 1); ++h) ldmatrix4(q[h], query_at + (k8 ? c + h : c / 2) * 32);
#pragma unroll
            for (int g = 0; g < KT / 16; ++g) {
                uint32_t b[4];
                ldmatrix4(b, keys + chunk_at(key_at, g, c));
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    if constexpr (k8) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            uint32_t even, odd;
                            to_pairs<P>(b[2 * n + h], even, odd);
                            if (c + h == 0) mma_from_zero<M>(s[2 * g + n], q[h], even, odd);
                            else mma_onto_it<M>(s[2 * g + n], q[h], even, odd);
                        }
                    } else {
                        if (c == 0) mma_from_zero<M>(s[2 * g + n], q[0], b[2 * n], b[2 * n + 1]);
                        else mma_onto_it<M>(s[2 * g + n], q[0], b[2 * n], b[2 * n + 1]);
                    }
                }
            }
        }
        // scores in powers of two; of codes with the values' scales in two parts (as in the attention of one token)
        float f[KT / 8][2], back[KT / 8][2];
#pragma unroll
        for (int n = 0; n < KT / 8; ++n) {
            if constexpr (k8) {
                const float* at = ring.scales + slot * 2 * KT + n * 8 + t * 2;
                const float2 ks = *reinterpret_cast<const float2*>(at), vs = *reinterpret_cast<const float2*>(at + KT);
#pragma unroll
                for (int a = 0; a < 2; ++a) {
                    const float v = a ? vs.y : vs.x, k = a ? ks.y : ks.x;
                    const int bits = __float_as_int(fmaxf(v, 0x1p-100f));
                    const float e = __int_as_float(0x4b000000 | (bits >> 23)) - (8388608.f + 127.f) + (v - v);  // (NaN stays that)
                    f[n][a] = __int_as_float((bits & 0x007fffff) | 0x3f800000);
                    back[n][a] = __int_as_float(0x7f000000 - min(bits & 0x7f800000, 0x7e800000));
#pragma unroll
                    for (int i = 0; i < 2; ++i) s[n][2 * i + a] = fmaf(s[n][2 * i + a] * k, q_scale[i], e);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) s[n][i] *= p.scale;
            }
        }
        if constexpr (MASKED) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                // the row's tile as a word of bits: nodes' from theirs, tokens' from its window's begin on
                uint32_t seen = marks.x;
                const uint64_t nodes = *nodes_of(i * 8 + lane / 4);
                const int low = *low_of(i * 8 + lane / 4);
                if (place >= 0) {
                    const int nodes_at = start - place;  // of node 0 in the tile
                    uint32_t of_nodes = 0;
                    if (nodes_at >= 0) of_nodes = nodes_at < 32 ? (uint32_t)(nodes << nodes_at) : 0u;
                    else of_nodes = -nodes_at < 64 ? (uint32_t)(nodes >> -nodes_at) : 0u;
                    const uint32_t tokens = nodes_at <= 0 ? 0u : nodes_at >= 32 ? 0xffffffffu : (1u << nodes_at) - 1;
                    const int first = low - place;
                    const uint32_t from = first <= 0 ? 0xffffffffu : first >= 32 ? 0u : 0xffffffffu << first;
                    seen &= (tokens & from) | (of_nodes & ~tokens);
                }
                const uint32_t bad = marks.y & seen;
#pragma unroll
                for (int n = 0; n < KT / 8; ++n)
#pragma unroll
                    for (int a = 0; a < 2; ++a) {
                        const int key = n * 8 + t * 2 + a;
                        float& x = s[n][2 * i + a];
                        x = bad >> key & 1 ? CUDART_NAN_F : seen >> key & 1 ? x : -CUDART_INF_F;
                    }
            }
        }
        float keep[2], base[2], top[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            top[i] = -CUDART_INF_F;
#pragma unroll
            for (int n = 0; n < KT / 8; ++n) top[i] = fmaxf(top[i], fmaxf(s[n][2 * i], s[n][2 * i + 1]));
        }
#pragma unroll
        for (int d = 1; d < 4; d *= 2)
#pragma unroll
            for (int i = 0; i < 2; ++i) top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], d));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float now = fmaxf(m[i], top[i]);
            base[i] = now == -CUDART_INF_F ? 0.f : now;
            keep[i] = m[i] == -CUDART_INF_F ? 1.f : ex2_ftz(m[i] - base[i]);  // (nothing to keep, or NaN)
            m[i] = now;
            l[i] *= keep[i];
            base[i] -= kRaise;
        }
        uint32_t w[2][KT / 16][4];  // first and second numbers of the weights, as operands
#pragma unroll
        for (int n = 0; n < KT / 8; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int a = 0; a < 2; ++a) {
                    float& x = s[n][2 * i + a];
                    x = ex2_ftz(x - base[i]);
                    if constexpr (k8) {
                        l[i] = fmaf(x, back[n][a], l[i]);
                        x *= f[n][a];
                    } else {
                        l[i] += x;
                    }
                }
                split_in_two<M>(s[n][2 * i], s[n][2 * i + 1], w[0][n / 2][n % 2 * 2 + i], w[1][n / 2][n % 2 * 2 + i]);
            }
        if constexpr (MASKED) {
            // rows that nobody sees may hold anything, and nothing times that need not be nothing (each warp makes them zero for itself: the
            // same zeros)
            const uint32_t want = marks.x & ~marks.y;
            if (want != 0xffffffffu) {
                if ((want >> lane & 1) == 0) {
#pragma unroll
                    for (int c = 0; c < kRowBytes / 16; ++c)
                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(values + Layout::offset(lane, c)), "r"(0) : "memory");
                }
                ptx::fence_proxy_async_smem();  // (before TMA writes there again)
                __syncwarp();
            }
            if constexpr (kMayBeWild) {
                if (has_wild(values)) {
                    add_by_numbers(values, s, keep);
                    return;
                }
            }
        }
        // of 16-bit rows: keys 0 - 7 and 8 - 15 of a step's eight dimensions, then of the next eight; of codes of sixteen dimensions
        const uint32_t value_at = Layout::offset((lane >> 3 & 1) * 8 + (lane & 7), lane >> 4);
#pragma unroll
        for (int c = 0; c < kRowBytes / 16; c += 2) {
            uint32_t b[KT / 16][4];
#pragma unroll
            for (int g = 0; g < KT / 16; ++g) ldmatrix4_trans(b[g], values + chunk_at(value_at, g, c));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if constexpr (k8) {
                    float even[4], odd[4];
#pragma unroll
                    for (int g = 0; g < KT / 16; ++g) {
                        uint32_t b0[2], b1[2];
                        to_pairs<P>(b[g][2 * h], b0[0], b0[1]);
                        to_pairs<P>(b[g][2 * h + 1], b1[0], b1[1]);
#pragma unroll
                        for (int n = 0; n < 2; ++n)
                            if (g + n == 0) {
                                mma_from_zero<M>(even, w[0][0], b0[0], b1[0]);
                                mma_from_zero<M>(odd, w[0][0], b0[1], b1[1]);
                            } else {
                                mma_onto_it<M>(even, w[n][g], b0[0], b1[0]);
                                mma_onto_it<M>(odd, w[n][g], b0[1], b1[1]);
                            }
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float &x = o[2 * (c + h)][i], &y = o[2 * (c + h) + 1][i];
                        x = fmaf(x, keep[i / 2], even[i]);
                        y = fmaf(y, keep[i / 2], odd[i]);
                    }
                } else {
                    float sum[4];
#pragma unroll
                    for (int g = 0; g < KT / 16; ++g) {
                        const uint32_t b0 = b[g][2 * h], b1 = b[g][2 * h + 1];
#pragma unroll
                        for (int n = 0; n < 2; ++n)
                            if (g + n == 0) mma_from_zero<M>(sum, w[0][0], b0, b1);
                            else mma_onto_it<M>(sum, w[n][g], b0, b1);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float& x = o[c + h][i];
                        x = fmaf(x, keep[i / 2], sum[i]);
                    }
                }
            }
        }
    }
    // Whether the values of a tile hold an infinity or a NaN (e4m3: codes that are no number, all seven bits): a row to a lane.
    __device__ __forceinline__ bool has_wild(uint32_t values) const {
        const int lane = threadIdx.x & 31;
        // carries the largest exponent, or all seven bits, into the sign
        constexpr uint32_t up = k8 ? 0x01010101u : std::is_same<M, __half>::value ? 0x04000400u : 0x00800080u;
        constexpr uint32_t signs = k8 ? 0x80808080u : 0x80008000u;
        uint32_t found = 0;
#pragma unroll 4
        for (int c = 0; c < kRowBytes / 16; ++c) {
            uint32_t v[4];
            asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                         : "r"(values + Layout::offset(lane, c))
                         : "memory");
#pragma unroll
            for (int i = 0; i < 4; ++i) found |= (v[i] & ~signs) + up;
        }
        return __any_sync(0xffffffffu, (found & signs) != 0);
    }
    // O += P V of a tile with such values: number by number, so that what a row does not see stays out of it.  s: the weights.
    __device__ __forceinline__ void add_by_numbers(uint32_t values, const float (&s)[KT / 8][4], const float (&keep)[2]) {
        const int lane = threadIdx.x & 31, t = lane & 3;
#pragma unroll
        for (int n = 0; n < DH / 8; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[n][i] *= keep[i / 2];
#pragma unroll 1
        for (int key = 0; key < KT; ++key) {
            float w[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float x = 0.f;
#pragma unroll
                for (int n = 0; n < KT / 8; ++n)
                    if (n == key / 8) x = key & 1 ? s[n][2 * i + 1] : s[n][2 * i];
                w[i] = __shfl_sync(0xffffffffu, x, (lane & ~3) + key % 8 / 2);
            }
#pragma unroll
            for (int c = 0; c < kRowBytes / 16; ++c) {
                uint32_t v;
                asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(values + Layout::offset(key, c) + t * 4) : "memory");
                float2 x, y = make_float2(0.f, 0.f);  // two neighbouring dimensions; codes: and the next two
                if constexpr (std::is_same<P, E4m3>::value) x = __half22float2(from_e4m3(v)), y = __half22float2(from_e4m3(v >> 16));
                else x = unpack2<M>(v);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (w[i] == 0.f) continue;
                    if constexpr (k8) {
                        o[2 * c][2 * i] = fmaf(w[i], x.x, o[2 * c][2 * i]);
                        o[2 * c + 1][2 * i] = fmaf(w[i], x.y, o[2 * c + 1][2 * i]);
                        o[2 * c][2 * i + 1] = fmaf(w[i], y.x, o[2 * c][2 * i + 1]);
                        o[2 * c + 1][2 * i + 1] = fmaf(w[i], y.y, o[2 * c + 1][2 * i + 1]);
                    } else {
                        o[c][2 * i] = fmaf(w[i], x.x, o[c][2 * i]);
                        o[c][2 * i + 1] = fmaf(w[i], x.y, o[c][2 * i + 1]);
                    }
                }
            }
        }
    }
    // use(row, its maximum, its sum, first dimension, two or four numbers of the output)
    template <typename F>
    __device__ __forceinline__ void results(const Rows& rows, int warp_rows, F&& use) {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float total = l[i];
            total += __shfl_xor_sync(0xffffffffu, total, 1);
            total += __shfl_xor_sync(0xffffffffu, total, 2);
            const int r = warp_rows + i * 8 + lane / 4;
            if (r >= rows.n) continue;
#pragma unroll
            for (int n = 0; n < DH / 8; n += k8 ? 2 : 1) {
                if constexpr (k8) {
                    const float x[4] = {o[n][2 * i], o[n + 1][2 * i], o[n][2 * i + 1], o[n + 1][2 * i + 1]};
                    use(r, m[i], total, dim_of(n), x);
                } else {
                    const float x[2] = {o[n][2 * i], o[n][2 * i + 1]};
                    use(r, m[i], total, dim_of(n), x);
                }
            }
        }
    }
    __device__ __forceinline__ void store(const Rows& rows, int warp_rows) {
        results(rows, warp_rows, [&](int r, float, float sum, int d, const auto& x) {
            constexpr int N = sizeof(x) / sizeof(float);
            const float scale = inverse_of<true>(p, rows, r, sum);
            Any16* at = static_cast<Any16*>(p.o) + row_at<true>(p, p.os, rows, r) + d;
#pragma unroll
            for (int e = 0; e < N; e += 2) {
                if (p.o_pairs) {
                    const uint32_t b = pack2<__nv_bfloat16>(x[e] * scale, x[e + 1] * scale), h = pack2<__half>(x[e] * scale, x[e + 1] * scale);
                    *reinterpret_cast<uint32_t*>(at + e) = p.bf16 ? b : h;
                } else {
                    put(p, at + e, x[e] * scale);
                    put(p, at + e + 1, x[e + 1] * scale);
                }
            }
        });
    }
};

// W warps at most, `team` of them to a worker.
template <typename P, int DH, int W, bool BULK>
__global__ void __launch_bounds__(W * 32, 1) paged_tree_kernel(const __grid_constant__ PagedAttentionBulk p, int team, int slots) {
    using Core = TreeCore<P, DH>;
    using Layout = typename Core::Layout;
    constexpr int KT = kTreeKeys, COST = kTreeCost, dim = DH;
    using Load = std::conditional_t<BULK, BulkLoader<P, KT, true, COST, Layout>, Loader<P, KT, true, COST, Layout>>;
    extern __shared__ __align__(16) unsigned char dynamic[];
    __shared__ uint2 marks[W][kMostSlots];
    __shared__ int places[W][kMostSlots];
    __shared__ alignas(8) uint64_t arrived[W][kMostSlots], left[W][kMostSlots];
    __shared__ Part parts[2 * W];
    __shared__ float2 part_sums[2 * W * 16];  // [2 * worker + part][rows]
    __shared__ int given_up;
    pdl_trigger();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, workers = blockDim.x / 32 / team;
    const int worker = warp / team, warp_rows = (warp - worker * team) * 16;
    const bool leads = warp_rows == 0;
    unsigned char* smem = dynamic + (1024 - (uint32_t)__cvta_generic_to_shared(dynamic)) % 1024;
    constexpr int kUnit = 2 * KT * Layout::pitch();
    const Layout lay{Layout::pitch()};
    const Ring ring{smem + worker * slots * kUnit, marks[worker], places[worker],
                    reinterpret_cast<float*>(smem + workers * slots * kUnit + worker * slots * 2 * KT * 4),
                    (uint32_t)__cvta_generic_to_shared(arrived[worker])};
    const uint32_t free = (uint32_t)__cvta_generic_to_shared(left[worker]);
    auto part_out = [&](int i) { return p.firsts + (blockIdx.x * 2LL * workers + i) * p.rows * dim; };

    if (tid == 0) p.joins[blockIdx.x] = make_int4(-1, 0, 0, 0), given_up = 0;
    if (leads) {
        if (lane < 2) parts[2 * worker + lane].there = 0;
        if (lane < slots) {
            ptx::mbar_init(ring.arrived + lane * 8, BULK ? 1 : 33);
            ptx::mbar_init(free + lane * 8, team);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        ptx::fence_proxy_async_smem();
    }
    __syncthreads();

    Cursor<KT, true, COST> at;
    const Share share = find_share<KT, true, COST>(p, at, worker, workers);
    if (share.first < share.end) {
        Load ahead{p, ring, lay, at};
        long long load = share.first;
        int slot_in = 0, slot_out = 0;
        uint32_t phase_in = 1, phase_out = 0;  // of a whole turn of the ring; a slot that nobody has used is free
        auto look = [&]() {
            if (load < share.end && ahead.at.t < COST) {
                load += COST - ahead.at.t;
                ahead.at.t = COST;
            }
            if (load < share.end) ahead.look();
        };
        auto fetch = [&]() {  // the leading warp alone
            if (load >= share.end) return;
            ptx::mbar_wait(free + slot_in * 8, phase_in, &given_up, p.status);
            __syncwarp();
            ahead.issue(slot_in);
            if constexpr (!BULK) {
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(ring.arrived + slot_in * 8) : "memory");
                if (lane == 0) ptx::mbar_arrive(ring.arrived + slot_in * 8);  // (the marks are written)
            }
            if (++slot_in == slots) slot_in = 0, phase_in ^= 1;
            if (++load < share.end && ++ahead.at.t == ahead.at.n) {
                ahead.at.next_item(p);
                if constexpr (BULK) ahead.planned = 1 << 30;
            }
            look();
        };
        if (leads) {
            look();
            // (some slots behind: the leading warp need not wait for the slowest one's last tile)
            for (int s = 0; s < slots - (slots > 4 ? slots / 4 + 1 : 1); ++s) fetch();
        }
        Core core(p, smem + workers * slots * (kUnit + 2 * KT * 4) + warp * Core::kRowsBytes);
        auto queries = [&](const Cursor<KT, true, COST>& c) {
            const Rows rows = rows_of<true>(p, c.b, c.head, c.item - c.head * c.parts(p), c.count);
            core.load_queries(rows, c.count, warp_rows);
            return rows;
        };
        long long begin = share.first;
        bool bad_page = false;
        Rows rows = queries(at);
        while (begin < share.end) {
            const long long item_end = begin + (at.n - at.t), end = item_end < share.end ? item_end : share.end;
            const int tiles = (int)(end - begin) - max(COST - at.t, 0);
            core.reset();
            for (int i = 0; i < tiles; ++i) {
                if (leads) fetch();
                ptx::mbar_wait(ring.arrived + slot_out * 8, phase_out, &given_up, p.status);
                __syncwarp();
                const uint2 mark = ring.marks[slot_out];
                const int place = ring.places[slot_out];
                bad_page |= mark.y != 0;
                if (rows.n > warp_rows) {
                    // seen in full by every row: a tile of the persistent keys, or of tokens behind every window's begin
                    const bool whole = mark.x == 0xffffffffu && mark.y == 0 && (place < 0 || (place + KT <= core.start && place >= core.lowest));
                    if (whole) core.template tile<false>(ring, slot_out, mark, place);
                    else core.template tile<true>(ring, slot_out, mark, place);
                }
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(free + slot_out * 8);
                if (++slot_out == slots) slot_out = 0, phase_out ^= 1;
            }
            const Cursor<KT, true, COST> done = at;
            const Rows done_rows = rows;
            if (tiles > 0) {
                const bool starts = done.t <= COST, ends = end == item_end;
                if (starts && ends) {
                    core.store(done_rows, warp_rows);
                } else {
                    const int which = 2 * worker + (starts ? 1 : 0);
                    float* to = part_out(which);
                    float2* sums = part_sums + which * team * 16;
                    core.results(done_rows, warp_rows, [&](int r, float top, float sum, int d, const auto& x) {
                        constexpr int N = sizeof(x) / sizeof(float);
                        if (d == 0) sums[r] = make_float2(top, sum);
                        if constexpr (N == 4) *reinterpret_cast<float4*>(to + r * dim + d) = make_float4(x[0], x[1], x[2], x[3]);
                        else *reinterpret_cast<float2*>(to + r * dim + d) = make_float2(x[0], x[1]);
                    });
                    if (leads && lane == 0) parts[which] = {1, done_rows, done.item, starts, ends, item_end};
                }
            }
            if (item_end < share.end) {
                at.next_item(p);
                rows = queries(at);
            }
            begin = end;
        }
        if (bad_page && leads && lane == 0) atomicCAS(p.status, 0, (int)TMW_ERR_INVALID_ARGUMENT);
    }
    __syncthreads();

    // The CTA's parts of one item are neighbours (see the attention of one token); its threads take four numbers of a row at a time.
    const uint32_t there = __ballot_sync(0xffffffffu, lane < 2 * workers && parts[lane].there);
    for (uint32_t todo = there & (0xaaaaaaaau | 1u); todo != 0; todo &= todo - 1) {
        const int i = __ffs(todo) - 1;
        const uint32_t rest = todo & (todo - 1), members = there & ~((1u << i) - 1) & (rest != 0 ? (rest & (0u - rest)) - 1 : 0xffffffffu);
        const Part part = parts[i];
        const bool starts = part.starts, ends = parts[31 - __clz(members)].ends;
        const Rows rows = part.rows;
        const long long where = (blockIdx.x * 2 + (starts ? 1 : 0)) * (long long)p.rows;
        for (int x = tid; x < rows.n * dim / 4; x += blockDim.x) {
            const int r = x * 4 / dim;
            float m = -CUDART_INF_F, l = 0.f;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
            for (uint32_t j = members; j != 0; j &= j - 1) m = fmaxf(m, part_sums[(__ffs(j) - 1) * team * 16 + r].x);
            const float base = m == -CUDART_INF_F ? 0.f : m;
            for (uint32_t j = members; j != 0; j &= j - 1) {
                const int of = __ffs(j) - 1;
                const float2 sum = part_sums[of * team * 16 + r];
                const float w = part_weight(sum.x, base);
                l = fmaf(w, sum.y, l);
                add_product(o, w, reinterpret_cast<const float4*>(part_out(of))[x]);
            }
            if (starts && ends) {
                Any16* to = static_cast<Any16*>(p.o) + row_at<true>(p, p.os, rows, r) + (x * 4 - r * dim);
                const float scale = inverse_of<true>(p, rows, r, l);
                put(p, to + 0, o.x * scale);
                put(p, to + 1, o.y * scale);
                put(p, to + 2, o.z * scale);
                put(p, to + 3, o.w * scale);
            } else {
                reinterpret_cast<float4*>(p.partial + where * dim)[x] = o;
                if (x * 4 == r * dim) p.sums[where + r] = make_float2(m, l);
            }
        }
        if (starts && !ends && tid == 0)
            p.joins[blockIdx.x] = make_int4(rows.b, part.item, (int)((part.item_end - 1) / (share.per * share.warps)), 0);
    }

    // sequences without a place
    for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
        int lo, pos, count;
        bool bad;
        if (tiles_of<KT, true>(p, b, lo, pos, count, bad) > 0 || !bad) continue;
        if (tid == 0) atomicCAS(p.status, 0, (int)TMW_ERR_INVALID_ARGUMENT);
        const int heads = p.group * p.map.kv_heads, n = count < 0 || count > p.nodes ? p.nodes : count;
        for (int i = tid; i < n * heads * dim; i += blockDim.x) {
            const int d = i % dim, row = i / dim, node = row / heads, h = row - node * heads;
            put(p, static_cast<Any16*>(p.o) + b * p.os[0] + h * p.os[1] + node * p.os[2] + d, CUDART_NAN_F);
        }
    }
}

// The parts of an item that was cut between CTAs, a warp to a row of the one that begins in CTA blockIdx.x.
constexpr int kTreeJoinWarps = 8, kTreeJoinAhead = 4;
template <int DH>
__global__ void __launch_bounds__(kTreeJoinWarps * 32) tree_join_kernel(const __grid_constant__ PagedAttention p) {
    const int lane = threadIdx.x & 31, r = blockIdx.y * kTreeJoinWarps + threadIdx.x / 32;
    constexpr int Q = (DH + 127) / 128;
    pdl_wait();
    const int4 join = __ldcg(p.joins + blockIdx.x);
    if (join.x < 0) return;
    const int count = p.counts != nullptr ? __ldg(p.counts + join.x) : p.nodes, parts = parts_of<true>(p, count);
    const Rows rows = rows_of<true>(p, join.x, join.y / parts, join.y % parts, count);
    if (r >= rows.n) return;
    const int n = join.z - (int)blockIdx.x + 1;
    auto slot = [&](int i) { return (2LL * (blockIdx.x + i) + (i == 0 ? 1 : 0)) * p.rows + r; };
    float m = -CUDART_INF_F, l = 0.f;
    float4 o[Q];
#pragma unroll
    for (int h = 0; h < Q; ++h) o[h] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = 0; i0 < n; i0 += kTreeJoinAhead) {
        float2 sums[kTreeJoinAhead];
        float4 part[kTreeJoinAhead][Q];
#pragma unroll
        for (int j = 0; j < kTreeJoinAhead; ++j) {
            if (i0 + j >= n) continue;
            sums[j] = __ldcg(p.sums + slot(i0 + j));
#pragma unroll
            for (int h = 0; h < Q; ++h)
                if (h * 128 + lane * 4 < DH) part[j][h] = __ldcg(reinterpret_cast<const float4*>(p.partial + slot(i0 + j) * DH + h * 128 + lane * 4));
        }
#pragma unroll
        for (int j = 0; j < kTreeJoinAhead; ++j) {
            if (i0 + j >= n) continue;
            const float now = fmaxf(m, sums[j].x), base = now == -CUDART_INF_F ? 0.f : now, keep = part_weight(m, base),
                        w = part_weight(sums[j].x, base);
            m = now;
            l = fmaf(w, sums[j].y, l * keep);
#pragma unroll
            for (int h = 0; h < Q; ++h)
                if (h * 128 + lane * 4 < DH) {
                    o[h].x *= keep; o[h].y *= keep; o[h].z *= keep; o[h].w *= keep;
                    add_product(o[h], w, part[j][h]);
                }
        }
    }
    const float scale = inverse_of<true>(p, rows, r, l);
    Any16* to = static_cast<Any16*>(p.o) + row_at<true>(p, p.os, rows, r);
#pragma unroll
    for (int h = 0; h < Q; ++h) {
        const int d = h * 128 + lane * 4;
        if (d >= DH) continue;
        put(p, to + d, o[h].x * scale);
        put(p, to + d + 1, o[h].y * scale);
        put(p, to + d + 2, o[h].z * scale);
        put(p, to + d + 3, o[h].w * scale);
    }
}

// What a tree's description adds to the arguments of one token's.
inline int tree_arguments(const tmw_paged_attention_desc& one, const tmw_page_scales& s, const tmw_paged_tree_desc& d, const void* scratch,
                          PagedAttention& p) {
    const int bad = arguments(one, s, scratch, p);
    if (bad != TMW_OK) return bad;
    p.qs[2] = d.q_stride[2];
    p.os[2] = d.o_stride[2];
    p.q_pairs = p.q_pairs && d.q_stride[2] % 2 == 0;
    p.o_pairs = p.o_pairs && d.o_stride[2] % 2 == 0;
    p.q_wide = p.q_wide && d.q_stride[2] % 8 == 0;  // (used with 16-bit numbers)
    p.o_wide = p.o_wide && d.o_stride[2] % 8 == 0;
    p.counts = d.counts; p.positions = d.positions;
    p.seen = d.seen;
    p.nodes = d.nodes;
    return TMW_OK;
}

// ---- host ---------------------------------------------------------------------------------------------------------------------

// A kernel and how it is launched, for a call over pages that come by TMA (BULK) or not.
template <typename P, int DH, bool BULK>
struct TreeKernel {
    static constexpr int W = DH > 128 ? 8 : 12;  // (sixteen rows of 256 outputs have 128 registers)
    struct Plan {
        int rows, team, slots, workers, grid, smem;
        size_t sums_at, partial_at, firsts_at, bytes;
    };
    static Plan plan(const tmw_paged_attention_desc& d, int nodes) {
        Plan n;
        const int all = d.heads / d.at.kv_heads * nodes, teams = (all + 15) / 16;
        const int parts = (teams + W - 1) / W;
        n.rows = (all + parts - 1) / parts;
        n.team = (n.rows + 15) / 16;
        constexpr int unit = 2 * kTreeKeys * (DH * (int)sizeof(P) + 4);
        const int rows = n.team * TreeCore<P, DH>::kRowsBytes;  // of a worker
        n.workers = W / n.team;
        while (n.workers > 1 && n.workers * (rows + 2 * unit) > kMostTree) --n.workers;
        n.slots = (kMostTree / n.workers - rows) / unit;
        if (n.slots > kMostSlots) n.slots = kMostSlots;
        n.smem = 1024 + n.workers * (n.slots * unit + rows);
        const long long capacity = (long long)d.at.columns * d.at.page_size;
        const long long keys = d.window >= 0 && d.window + (long long)nodes < capacity ? d.window + (long long)nodes : capacity;
        const long long tiles = ((d.n_persistent + 31) / 32 + keys / 32 + 2) * (long long)d.at.kv_heads * parts * d.at.batch;
        n.grid = (int)(tiles < sm_count() ? tiles : sm_count());
        const size_t out = (size_t)n.rows * DH * sizeof(float);
        n.sums_at = (size_t)n.grid * sizeof(int4);
        n.partial_at = (n.sums_at + (size_t)n.grid * 2 * n.rows * sizeof(float2) + 15) & ~(size_t)15;
        n.firsts_at = n.partial_at + n.grid * 2 * out;
        n.bytes = n.firsts_at + (size_t)n.grid * n.workers * 2 * out;
        return n;
    }
    static int launch(const tmw_paged_attention_desc& d, PagedAttentionBulk& p, const Plan& n, unsigned char* scratch, cudaStream_t stream) {
        if (BULK && !make_maps<typename TreeCore<P, DH>::Layout>(d, p)) return TMW_ERR_CUDA;
        p.rows = n.rows;
        p.pers_tiles = (p.np + kTreeKeys - 1) / kTreeKeys;
        p.joins = reinterpret_cast<int4*>(scratch);
        p.sums = reinterpret_cast<float2*>(scratch + n.sums_at);
        p.partial = reinterpret_cast<float*>(scratch + n.partial_at);
        p.firsts = reinterpret_cast<float*>(scratch + n.firsts_at);
        auto kern = paged_tree_kernel<P, DH, W, BULK>;
        const int rc = allow_shared_memory(reinterpret_cast<const void*>(kern), n.smem);
        if (rc != TMW_OK) return rc;
        kern<<<n.grid, n.workers * n.team * 32, n.smem, stream>>>(p, n.team, n.slots);
        TMW_CUDA_TRY(cudaGetLastError());
        if (n.grid > 1)
            TMW_CUDA_TRY(launch_ex(tree_join_kernel<DH>, dim3((unsigned)n.grid - 1, (unsigned)((n.rows + kTreeJoinWarps - 1) / kTreeJoinWarps)),
                                   dim3(kTreeJoinWarps * 32), 0, stream, true, 1, static_cast<const PagedAttention&>(p)));
        return TMW_OK;
    }
};

// `use` with the kernel for pages of P; false: head_dim is none of its
template <typename P, typename F>
bool with_tree_kernel(const tmw_paged_attention_desc& d, const tmw_page_scales& s, F&& use) {
    const bool bulk = can_bulk(d, s);
    const auto of = [&](auto dh) {
        constexpr int DH = decltype(dh)::value;
        if (bulk) use(TreeKernel<P, DH, true>());
        else use(TreeKernel<P, DH, false>());
        return true;
    };
    switch (d.at.head_dim) {
        case 32: return of(std::integral_constant<int, 32>());
        case 64: return of(std::integral_constant<int, 64>());
        case 96: return of(std::integral_constant<int, 96>());
        case 128: return of(std::integral_constant<int, 128>());
        case 256: return of(std::integral_constant<int, 256>());
    }
    return false;
}

template <typename P>
bool tree_scratch_of(const tmw_paged_attention_desc& d, const tmw_page_scales& s, int nodes, size_t& bytes) {
    return with_tree_kernel<P>(d, s, [&](auto kernel) { bytes = kernel.plan(d, nodes).bytes; });
}
template <typename P>
bool tree_launch_of(const tmw_paged_attention_desc& d, const tmw_page_scales& s, PagedAttentionBulk& p, void* scratch, size_t scratch_bytes,
                    cudaStream_t stream, int& status) {
    return with_tree_kernel<P>(d, s, [&](auto kernel) {
        const auto n = kernel.plan(d, p.nodes);
        status = TMW_ERR_INVALID_ARGUMENT;
        if (scratch_bytes < n.bytes) set_error_text("tmw_paged_tree_attention: scratch smaller than tmw_paged_tree_attention_scratch_bytes()");
        else status = kernel.launch(d, p, n, static_cast<unsigned char*>(scratch), stream);
    });
}

}  // namespace

// Whether the kernel on tensor cores takes a call over such pages, and if so how much scratch it needs, and the call itself: in a file of
// their own for each type of the pages.
#define TMW_TREE_OF(name)                                                                                                              \
    bool tree_scratch_##name(const tmw_paged_attention_desc& d, const tmw_page_scales& s, int nodes, size_t& bytes);                   \
    bool tree_launch_##name(const tmw_paged_attention_desc& d, const tmw_page_scales& s, const tmw_paged_tree_desc& tree, void* scratch, \
                            size_t scratch_bytes, cudaStream_t stream, int& status);
TMW_TREE_OF(bf16)
TMW_TREE_OF(f16)
TMW_TREE_OF(int8)
TMW_TREE_OF(e4m3)
TMW_TREE_OF(tc)
#undef TMW_TREE_OF

// Which calls tcgen05 takes: pages that come by TMA, head_dim 64 or 128, and so many rows to a key head that mma.sync's work outweighs the longer
// hand-overs here.  One border for all lengths, that of long sequences: windows of a few hundred keys, with fewer tiles to a worker, would want a
// later one (up to a fifth: 16-bit heads of 64 up to some 48 rows, of 128 up to 24).  us, tcgen05 | mma.sync:
//   16-bit pages, heads of 128: 16 sequences of up to 16384, 32 heads on 8: 8 rows 115 | 134, 16 rows 116 | 161, 32 rows 118 | 175;
//     64 windows of 512 of 10 heads: 8 rows 87 | 70, 16 rows 90 | 85, 33 rows 94 | 100
//   16-bit pages, heads of 64: the same sequences: 32 rows 108 | 99, 48 rows 108 | 121; 32 sequences of 10 heads, 20 rows 346 | 298,
//     33 rows 349 | 365; the windows: 33 rows 76 | 64, 64 rows 82 | 88
//   codes, 6 of up to 65536, 32 heads on 4: of 128: 32 rows 202 | 164, 40 rows 207 | 215; of 64: 48 rows 166 | 148, 56 rows 168 | 216
inline bool tree_takes_tc(const tmw_paged_attention_desc& d, const tmw_page_scales& s, int nodes) {
    const bool codes = s.format != TMW_PAGES_SAME, wide = d.at.head_dim == 128;
    const int few = codes ? (wide ? 32 : 48) : (wide ? 8 : 32);
    return d.at.dtype != TMW_F32 && (d.at.head_dim == 64 || wide) && can_bulk(d, s) && d.heads / d.at.kv_heads * nodes > few;
}

}  // namespace tmw
