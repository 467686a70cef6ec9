// Attention of one new token per sequence over pages in 8 bits: the core on tensor cores, and which kernel takes a call.
#pragma once

#include "paged_attention.cuh"

namespace tmw {
namespace {

// ---- the core on tensor cores: 16-bit queries, head_dim 32, 64, 96, 128 or 256 ---------------------------------------------------
// As the core for pages of 16 bits (the keys, then the dimensions of the values, are the rows of the products, eight query heads
// their columns), with every code turned into the fp16 number that it is between shared memory and the product:
//
// ldmatrix brings a lane four neighbouring codes of a key; the even and the odd ones, as pairs, are two registers of an operand
// whose dimensions are in another order than memory's, and the queries are laid out in that order.  Transposed it brings a lane two codes of one key
// and the same two of the next: the even ones, again, are a pair of keys for one dimension.  So no code ever moves between
// lanes.  Queries in bf16 go in as fp16 times a power of two of each head's own: what their largest number leaves no bits for is 2^-38 of it.
//
// A key's scale multiplies its score.  A value's, 2^e f with 1 <= f < 2, must not meet the 16-bit weights as it is, since scales may differ by
// far more than these hold: x_j = s_j + e_j takes the score's place under the running maximum, u_j = 2^(x_j - m) f_j are the weights of the
// codes, and u_j / scale_j = 2^(x_j - m) 2^-e_j those that are summed up for the denominator; both with one exponential and no
// logarithm, and a token whose values are small counts as much in the sum as any other.  That ends where 2^(x_j - m) is no fp32 number any
// more, 2^-126: with scales 2^114 apart for a token whose weight is 2^-24 of the largest (2^112 in the tcgen05 form, whose weights are
// raised by two less).
//
// HEADS: of an item at most, 1, 2, 4, 8 or 16.  With fewer than eight the columns hold them several times over, and each of the 8 / HEADS
// copies deals with its own share of the tile's keys: its weights are zero in the rows of the others', its running maximum
// is its own, and the copies are added up when the item ends.  So a lane has KT HEADS / 32 exponentials to a tile instead of KT / 4
// (256 windows of 512, 10 heads of 64: 127 us with one copy, 86 with eight; by TMA then 56).
//
// A warp's chain of copies, products and exponentials bounds it, at 51 to 66 % of the issue slots: 256 windows of 512 of 10 heads of 64,
// int8, 180 MB, 56 us; 48 sequences of up to 16384, 32 heads on 8 of 128, e4m3 under fp16, 350 MB, 77 us; 12 of up to 65536, 32
// heads on 4 of 128, int8, 583 MB, 129 us.
//
// d = a b + c for one 16 x 8 x 16 tile, and d += a b (not volatile: in whichever order the results are needed)
__device__ __forceinline__ void mma_more(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_onto(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, float c0,
                                         float c1, float c2, float c3) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

template <typename P, int DH, int HEADS, bool BULK>
struct Mma8Core {
    static constexpr int kRows = HEADS, KT = 32, kChunks = DH / 16;
    static constexpr int EIGHTS = HEADS > 8 ? 2 : 1, kCopies = HEADS < 8 ? 8 / HEADS : 1;
    static constexpr int kKeys = kCopies == 1 ? 4 : kCopies == 2 ? 2 : 1;  // of a lane
    static constexpr int kOfLane = HEADS == 1 ? 1 : 2;                     // heads of each eight
    static constexpr int kTerms8 = HEADS == 1 ? 1 : 2;  // products of a weight with the values
    static constexpr float kRaise = 12.f;  // as far as fp16 allows: a weight is at most 2^13
    using Layout = BoxLayout<DH>;
    static constexpr int kItemCost = 2;
    using Load = std::conditional_t<BULK, BulkLoader<P, KT, false, kItemCost, Layout>, Loader<P, KT, false, kItemCost, Layout>>;
    using Args = std::conditional_t<BULK, PagedAttentionBulk, PagedAttention>;
    const PagedAttention& p;
    uint32_t q[EIGHTS][kChunks][2];
    float q_scale[EIGHTS][2];
    float m[EIGHTS][2], l[EIGHTS][2];  // l: of this lane's keys
    float o[EIGHTS][kChunks][4];       // dimension 16 k + 2 (lane / 4) of both heads, the next dimension of both

    static __host__ __device__ int extra(int) { return 0; }

    __device__ Mma8Core(const PagedAttention& p, unsigned char*) : p(p) {}
    __device__ __forceinline__ void load_queries(const Rows& of, int) {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int h = 0; h < EIGHTS; ++h) {
            const int r = h * 8 + lane / 4 % HEADS;
            const uint16_t* from = static_cast<const uint16_t*>(p.q) + row_at<false>(p, p.qs, of, r) + lane % 4 * 4;
            uint32_t raw[kChunks][2];
            float top = 0.f;
#pragma unroll
            for (int k = 0; k < kChunks; ++k)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint32_t w = 0;
                    if (r < of.n) {
                        const uint16_t* at = from + k * 16 + i * 2;
                        w = p.q_pairs ? *reinterpret_cast<const uint32_t*>(at) : at[0] | (uint32_t)at[1] << 16;
                    }
                    raw[k][i] = w;
                    const float2 x = unpack2<__nv_bfloat16>(w);
                    top = fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y)));
                }
            float scale = p.scale;
            if (p.bf16) {
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                // the largest number becomes one from 2^14 on; an infinite one stays infinite
                const int e = max((__float_as_int(top) >> 23) - 127, -100);
                const float up = __int_as_float((127 + 14 - e) << 23);
                scale *= __int_as_float((127 - 14 + e) << 23);
#pragma unroll
                for (int k = 0; k < kChunks; ++k)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float2 x = unpack2<__nv_bfloat16>(raw[k][i]);
                        raw[k][i] = pack2<__half>(x.x * up, x.y * up);
                    }
            }
#pragma unroll
            for (int k = 0; k < kChunks; ++k) {  // numbers 4 t and 4 t + 2, then 4 t + 1 and 4 t + 3
                q[h][k][0] = __byte_perm(raw[k][0], raw[k][1], 0x5410);
                q[h][k][1] = __byte_perm(raw[k][0], raw[k][1], 0x7632);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) q_scale[h][e] = __shfl_sync(0xffffffffu, scale, (lane % 4 * 2 + e) * 4);
        }
    }
    __device__ __forceinline__ void reset() {
#pragma unroll
        for (int h = 0; h < EIGHTS; ++h) {
            m[h][0] = m[h][1] = -CUDART_INF_F;
            l[h][0] = l[h][1] = 0.f;
#pragma unroll
            for (int k = 0; k < kChunks; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[h][k][i] = 0.f;
        }
    }
    __device__ __forceinline__ void tile(const Ring& ring, int stage, uint2 marks, const Layout& lay) {
        const int lane = threadIdx.x & 31;
        const uint32_t keys = (uint32_t)__cvta_generic_to_shared(ring.tiles + stage * 2 * KT * Layout::pitch()), values = keys + KT * Layout::pitch();
        const float* scales = ring.scales + stage * 2 * KT + lane / 4;
        // of the lane's row and the first chunk of two, turned: two chunks further on is another number in the same bits, or the next box
        const uint32_t lane_at = Layout::offset(lane & 15, lane >> 4);
        const auto chunk_at = [&](int g, int k) {
            constexpr int in = Layout::kInBox;
            return (lane_at ^ (k % in << 4)) + k / in * KT * Layout::kBoxBytes + g * 16 * Layout::kBoxBytes;
        };
        float s[EIGHTS][KT / 16][4];  // of each sixteen: keys lane / 4 and 8 + lane / 4, both heads each
#pragma unroll
        for (int k = 0; k < kChunks; k += 2)
#pragma unroll
            for (int g = 0; g < KT / 16; ++g) {
                uint32_t a[4];
                ldmatrix4(a, keys + chunk_at(g, k));
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t even[2], odd[2];
                    to_pairs<P>(a[2 * c], even[0], odd[0]);
                    to_pairs<P>(a[2 * c + 1], even[1], odd[1]);
#pragma unroll
                    for (int h = 0; h < EIGHTS; ++h) {
                        const uint32_t(&b)[2] = q[h][k + c];
                        if (k + c == 0) mma_onto(s[h][g], even[0], even[1], odd[0], odd[1], b[0], b[1], 0.f, 0.f, 0.f, 0.f);
                        else mma_more(s[h][g], even[0], even[1], odd[0], odd[1], b[0], b[1]);
                    }
                }
            }
        // this lane's keys, with the values' scales in their two parts
        const int t = lane % 4;
        const auto key_of = [&](int j) { return kCopies == 1 ? j * 8 : kCopies == 2 ? (t >> 1) * 16 + j * 8 : t * 8; };
        float e[kKeys], f[kKeys], back[kKeys], ks[kKeys];
#pragma unroll
        for (int j = 0; j < kKeys; ++j) {
            ks[j] = scales[key_of(j)];
            const float vs = scales[KT + key_of(j)];
            const int bits = __float_as_int(fmaxf(vs, 0x1p-100f));
            e[j] = __int_as_float(0x4b000000 | (bits >> 23)) - (8388608.f + 127.f) + (vs - vs);  // (NaN stays that)
            f[j] = __int_as_float((bits & 0x007fffff) | 0x3f800000);
            back[j] = __int_as_float(0x7f000000 - min(bits & 0x7f800000, 0x7e800000));  // (finite under keys that are not seen)
        }
        // all heads side by side: their chains of shuffles and exponentials overlap
        uint32_t weights[EIGHTS][KT / 16][2][kTerms8];
        float keep[EIGHTS][2], base[EIGHTS][2], top[EIGHTS][2], w[EIGHTS][kKeys][2];
#pragma unroll
        for (int h = 0; h < EIGHTS; ++h)
#pragma unroll
            for (int a = 0; a < kOfLane; ++a) {
                top[h][a] = -CUDART_INF_F;
#pragma unroll
                for (int j = 0; j < kKeys; ++j) {
                    float x;
                    if constexpr (kCopies == 1) x = s[h][j / 2][j % 2 * 2 + a];
                    else if constexpr (kCopies == 2) x = t < 2 ? s[h][0][j * 2 + a] : s[h][1][j * 2 + a];
                    else x = t < 2 ? (t == 0 ? s[h][0][a] : s[h][0][2 + a]) : (t == 2 ? s[h][1][a] : s[h][1][2 + a]);
                    w[h][j][a] = fmaf(x * ks[j], q_scale[h][a], e[j]);
                }
            }
        if (marks.x != 0xffffffffu || marks.y != 0) {
#pragma unroll
            for (int j = 0; j < kKeys; ++j) {
                const int key = key_of(j) + lane / 4;
                const bool seen = marks.x >> key & 1, bad = marks.y >> key & 1;
#pragma unroll
                for (int h = 0; h < EIGHTS; ++h)
#pragma unroll
                    for (int a = 0; a < kOfLane; ++a) w[h][j][a] = bad ? CUDART_NAN_F : seen ? w[h][j][a] : -CUDART_INF_F;
            }
        }
#pragma unroll
        for (int h = 0; h < EIGHTS; ++h)
#pragma unroll
            for (int a = 0; a < kOfLane; ++a)
#pragma unroll
                for (int j = 0; j < kKeys; ++j) top[h][a] = fmaxf(top[h][a], w[h][j][a]);
#pragma unroll
        for (int d = 4; d < 32; d *= 2)
#pragma unroll
            for (int h = 0; h < EIGHTS; ++h)
#pragma unroll
                for (int a = 0; a < kOfLane; ++a) top[h][a] = fmaxf(top[h][a], __shfl_xor_sync(0xffffffffu, top[h][a], d));
#pragma unroll
        for (int h = 0; h < EIGHTS; ++h)
#pragma unroll
            for (int a = 0; a < kOfLane; ++a) {
                const float now = fmaxf(m[h][a], top[h][a]);
                base[h][a] = now == -CUDART_INF_F ? 0.f : now;
                keep[h][a] = m[h][a] == -CUDART_INF_F ? 1.f : ex2_ftz(m[h][a] - base[h][a]);  // (nothing to keep, or NaN)
                m[h][a] = now;
                l[h][a] *= keep[h][a];
                base[h][a] -= kRaise;
            }
#pragma unroll
        for (int h = 0; h < EIGHTS; ++h) {
#pragma unroll
            for (int j = 0; j < kKeys; ++j)
#pragma unroll
                for (int a = 0; a < kOfLane; ++a) {
                    const float x = ex2_ftz(w[h][j][a] - base[h][a]);
                    l[h][a] = fmaf(x, back[j], l[h][a]);
                    w[h][j][a] = x * f[j];
                }
            if (kOfLane == 1) keep[h][1] = keep[h][0];
            // weights as two numbers each, 22 bits: two registers, or (one head) its two columns
            uint32_t parts[kKeys][kTerms8];
#pragma unroll
            for (int j = 0; j < kKeys; ++j) {
                if constexpr (kOfLane == 1) {
                    const float first = __half2float(__float2half_rz(w[h][j][0]));
                    parts[j][0] = pack2<__half>(first, w[h][j][0] - first);
                } else {
                    parts[j][0] = cut2<__half>(w[h][j][0], w[h][j][1]);
                    const float2 had = unpack2<__half>(parts[j][0]);
                    parts[j][1] = pack2<__half>(w[h][j][0] - had.x, w[h][j][1] - had.y);
                }
            }
#pragma unroll
            for (int g = 0; g < KT / 16; ++g)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int n = 0; n < kTerms8; ++n) {
                        uint32_t x;
                        if constexpr (kCopies == 1) x = parts[g * 2 + i][n];
                        else if constexpr (kCopies == 2) x = (t >> 1) == g ? parts[i][n] : 0;
                        else x = t == g * 2 + i ? parts[0][n] : 0;
                        weights[h][g][i][n] = turned(x);
                    }
        }
        if constexpr (BULK && std::is_same<P, E4m3>::value) {
            // rows that are not seen may hold codes that are no number, and nothing times these is no number either
            const uint32_t want = marks.x & ~marks.y;
            if (want != 0xffffffffu) {
                if ((want >> lane & 1) == 0) {
#pragma unroll
                    for (int c = 0; c < kChunks; ++c)
                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(values + lay.offset(lane, c)), "r"(0) : "memory");
                }
                ptx::fence_proxy_async_smem();  // (before TMA writes there again)
                __syncwarp();
            }
        }
#pragma unroll
        for (int k = 0; k < kChunks; k += 2) {
            uint32_t a[KT / 16][4];
#pragma unroll
            for (int g = 0; g < KT / 16; ++g) ldmatrix4_trans(a[g], values + chunk_at(g, k));
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float sum[EIGHTS][KT / 16][4];  // of this tile, one chain of products for each sixteen keys
#pragma unroll
                for (int g = 0; g < KT / 16; ++g) {
                    uint32_t even[2], odd[2];
                    to_pairs<P>(a[g][2 * c], even[0], odd[0]);
                    to_pairs<P>(a[g][2 * c + 1], even[1], odd[1]);
#pragma unroll
                    for (int h = 0; h < EIGHTS; ++h)
#pragma unroll
                        for (int n = 0; n < kTerms8; ++n) {
                            const uint32_t b0 = weights[h][g][0][n], b1 = weights[h][g][1][n];
                            if (n == 0) mma_onto(sum[h][g], even[0], odd[0], even[1], odd[1], b0, b1, 0.f, 0.f, 0.f, 0.f);
                            else mma_more(sum[h][g], even[0], odd[0], even[1], odd[1], b0, b1);
                        }
                }
#pragma unroll
                for (int h = 0; h < EIGHTS; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float x = sum[h][0][i];
#pragma unroll
                        for (int g = 1; g < KT / 16; ++g) x += sum[h][g][i];
                        o[h][k + c][i] = fmaf(o[h][k + c][i], keep[h][i & 1], x);
                    }
            }
        }
    }
    // use(row, its maximum, its sum, first dimension, two numbers of the output), from every lane that has some
    template <typename F>
    __device__ __forceinline__ void results(const Rows& rows, F&& use) {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int h = 0; h < EIGHTS; ++h)
#pragma unroll
            for (int a = 0; a < kOfLane; ++a) {
                float total = l[h][a], top = m[h][a];
#pragma unroll
                for (int d = 4; d < 32; d *= 2) total += __shfl_xor_sync(0xffffffffu, total, d);
                float weight = 1.f;
                if constexpr (kCopies > 1) {  // copies of a head lie HEADS columns apart, two columns to a lane
#pragma unroll
                    for (int d = HEADS < 4 ? 1 : 2; d < 4; d *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                    weight = part_weight(m[h][a], top == -CUDART_INF_F ? 0.f : top);
                    total *= weight;
#pragma unroll
                    for (int d = HEADS < 4 ? 1 : 2; d < 4; d *= 2) total += __shfl_xor_sync(0xffffffffu, total, d);
                }
                const int r = h * 8 + lane % 4 * 2 + a;
#pragma unroll
                for (int k = 0; k < kChunks; ++k) {
                    float x[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        x[i] = kOfLane == 1 ? o[h][k][2 * i] + o[h][k][2 * i + 1] : o[h][k][2 * i + a];
                        if constexpr (kCopies > 1) {
                            x[i] *= weight;
#pragma unroll
                            for (int d = HEADS < 4 ? 1 : 2; d < 4; d *= 2) x[i] += __shfl_xor_sync(0xffffffffu, x[i], d);
                        }
                    }
                    if (r < rows.n && r < HEADS && (HEADS > 1 || a == 0)) use(r, top, total, k * 16 + lane / 4 * 2, x);
                }
            }
    }
    __device__ __forceinline__ void store(const Rows& rows) {
        results(rows, [&](int r, float, float sum, int d, const float (&x)[2]) {
            const float scale = inverse(sum);
            Any16* at = static_cast<Any16*>(p.o) + row_at<false>(p, p.os, rows, r) + d;
            if (p.o_pairs) {
                const uint32_t b = pack2<__nv_bfloat16>(x[0] * scale, x[1] * scale), h = pack2<__half>(x[0] * scale, x[1] * scale);
                *reinterpret_cast<uint32_t*>(at) = p.bf16 ? b : h;
            } else {
                put(p, at, x[0] * scale);
                put(p, at + 1, x[1] * scale);
            }
        });
    }
};

// Pages made of eights or sixteens come by TMA, with as many heads as a group has, the next power of two of them; others by copies of sixteen bytes, with
// eight or sixteen heads.
template <typename P, int DH, typename F>
int with_mma(const tmw_paged_attention_desc& d, bool bulk, F&& use) {
    constexpr int W = DH > 128 ? 6 : DH > 64 ? 12 : 16;
    const int group = d.heads / d.at.kv_heads;
    if (!bulk) {
        if (group <= 8) return use(Kernel<Any16, P, false, Mma8Core<P, DH, 8, false>, W, 2>());
        return use(Kernel<Any16, P, false, Mma8Core<P, DH, 16, false>, (DH > 64 ? W : 12), 2>());
    }
    if (group == 1) return use(Kernel<Any16, P, false, Mma8Core<P, DH, 1, true>, W, 2>());
    if (group == 2) return use(Kernel<Any16, P, false, Mma8Core<P, DH, 2, true>, W, 2>());
    if (group <= 4) return use(Kernel<Any16, P, false, Mma8Core<P, DH, 4, true>, W, 2>());
    if (group <= 8) return use(Kernel<Any16, P, false, Mma8Core<P, DH, 8, true>, W, 2>());
    return use(Kernel<Any16, P, false, Mma8Core<P, DH, 16, true>, (DH > 64 ? W : 12), 2>());
}
// `use` with the Kernel that takes the call
template <typename P, typename F>
int with_kernel(const tmw_paged_attention_desc& d, const tmw_page_scales& s, F&& use) {
    const bool bulk = can_bulk(d, s);
    if (d.at.dtype != TMW_F32) {
        switch (d.at.head_dim) {
            case 32: return with_mma<P, 32>(d, bulk, use);
            case 64: return with_mma<P, 64>(d, bulk, use);
            case 96: return with_mma<P, 96>(d, bulk, use);
            case 128: return with_mma<P, 128>(d, bulk, use);
            case 256: return with_mma<P, 256>(d, bulk, use);
        }
        return with_simt<Any16, P, false>(d, 1, use);
    }
    return with_simt<float, P, false>(d, 1, use);
}

template <typename P>
size_t scratch_bytes_of(const tmw_paged_attention_desc& d, const tmw_page_scales& s) {
    size_t bytes = 0;
    with_kernel<P>(d, s, [&](auto kernel) {
        bytes = kernel.plan(d, d.at.head_dim, 1).bytes;
        return TMW_OK;
    });
    return bytes;
}

template <typename P>
int launch_of(const tmw_paged_attention_desc& d, const tmw_page_scales& s, void* scratch, size_t scratch_bytes, cudaStream_t stream) {
    PagedAttentionBulk p;
    const int bad = arguments(d, s, scratch, p);
    if (bad != TMW_OK) return bad;
    return with_kernel<P>(d, s, [&](auto kernel) {
        using K = decltype(kernel);
        const Plan n = kernel.plan(d, p.row_bytes, 1);
        if (scratch_bytes < n.bytes) {
            set_error_text("tmw_paged_attention_scaled: scratch smaller than tmw_paged_attention_scaled_scratch_bytes()");
            return (int)TMW_ERR_INVALID_ARGUMENT;
        }
        if constexpr (K::CoreOf::Load::kBulk) {
            if (!make_maps<typename K::CoreOf::Layout>(d, p)) return (int)TMW_ERR_CUDA;
        }
        return kernel.launch(p, n, static_cast<unsigned char*>(scratch), stream);
    });
}

}  // namespace

// one for each form of the pages, in files of their own
size_t paged_attention_int8_scratch(const tmw_paged_attention_desc& d, const tmw_page_scales& s);
size_t paged_attention_e4m3_scratch(const tmw_paged_attention_desc& d, const tmw_page_scales& s);
int paged_attention_int8(const tmw_paged_attention_desc& d, const tmw_page_scales& s, void* scratch, size_t scratch_bytes, cudaStream_t stream);
int paged_attention_e4m3(const tmw_paged_attention_desc& d, const tmw_page_scales& s, void* scratch, size_t scratch_bytes, cudaStream_t stream);

}  // namespace tmw
