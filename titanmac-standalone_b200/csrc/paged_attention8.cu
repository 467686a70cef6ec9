// Attention of one new token per sequence over pages in 8 bits (tmw_paged_attention_scaled): which kernel takes a call.
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
// any factor: x_j = s_j + e_j takes the score's place under the running maximum, u_j = 2^(x_j - m) f_j are the weights of the
// codes, and u_j / scale_j = 2^(x_j - m) 2^-e_j those that are summed up for the denominator; both with one exponential and no
// logarithm, and a token whose values are small counts as much in the sum as any other.
//
// HEADS: of an item at most, 1, 2, 4, 8 or 16.  With fewer than eight the columns hold them several times over, and each of the 8 / HEADS
// copies deals with its own share of the tile's keys: its weights are zero in the rows of the others', its running maximum
// is its own, and the copies are added up when the item ends.  So a lane has KT HEADS / 32 exponentials to a tile instead of KT / 4.
template <int DH>
struct Mma8Layout {
    int bytes;
    static constexpr int kChunks = DH / 16;
    static constexpr bool kTurned = (kChunks & (kChunks - 1)) == 0;
    __host__ __device__ static constexpr int pitch() { return DH + (kTurned ? 0 : 16); }
    __host__ __device__ static constexpr int chunks() { return kChunks; }
    // eight rows' same chunk stands on different banks: by its place in the row, or by rows of an odd number of chunks
    __device__ __forceinline__ static int offset(int r, int c) {
        const int turn = !kTurned ? 0 : kChunks >= 8 ? r & 7 : kChunks == 4 ? r >> 1 & 3 : r >> 2 & 1;
        return r * pitch() + ((c ^ turn) << 4);
    }
};

// Four codes as fp16 numbers, two to a register: the first and third, the second and fourth.
template <typename P>
__device__ __forceinline__ void to_pairs(uint32_t w, uint32_t& even, uint32_t& odd);
template <>
__device__ __forceinline__ void to_pairs<int8_t>(uint32_t w, uint32_t& even, uint32_t& odd) {
    w ^= 0x80808080u;  // 0 .. 255 under the exponent of 1024, less 1024 + 128
    const uint32_t bias = 0x64806480u;
    const auto less = [&](uint32_t x) {
        const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&bias));
        return *reinterpret_cast<const uint32_t*>(&d);
    };
    even = less(__byte_perm(w, 0x64646464u, 0x4240));
    odd = less(__byte_perm(w, 0x64646464u, 0x4341));
}
template <>
__device__ __forceinline__ void to_pairs<E4m3>(uint32_t w, uint32_t& even, uint32_t& odd) {
    w = __byte_perm(w, w, 0x3120);
    const __half2 a = from_e4m3(w), b = from_e4m3(w >> 16);
    even = *reinterpret_cast<const uint32_t*>(&a);
    odd = *reinterpret_cast<const uint32_t*>(&b);
}

template <typename T, typename P, int DH, int HEADS>
struct Mma8Core {
    static constexpr int kRows = HEADS, KT = 32, kChunks = DH / 16;
    static constexpr int EIGHTS = HEADS > 8 ? 2 : 1, kCopies = HEADS < 8 ? 8 / HEADS : 1;
    static constexpr int kKeys = kCopies == 1 ? 4 : kCopies == 2 ? 2 : 1;  // of a lane
    static constexpr int kOfLane = HEADS == 1 ? 1 : 2;                     // heads of each eight
    static constexpr int kTerms8 = HEADS == 1 ? 1 : 2;  // products of a weight with the values
    static constexpr float kRaise = 12.f;  // as far as fp16 allows: a weight is at most 2^13
    using Layout = Mma8Layout<DH>;
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
            const T* from = static_cast<const T*>(p.q) + row_at<false>(p, p.qs, of, r) + lane % 4 * 4;
            uint32_t raw[kChunks][2];
            float top = 0.f;
#pragma unroll
            for (int k = 0; k < kChunks; ++k)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint32_t w = 0;
                    if (r < of.n) {
                        const T* at = from + k * 16 + i * 2;
                        if (p.q_pairs) w = *reinterpret_cast<const uint32_t*>(at);
                        else w = *reinterpret_cast<const uint16_t*>(at) | (uint32_t)*reinterpret_cast<const uint16_t*>(at + 1) << 16;
                    }
                    raw[k][i] = w;
                    const float2 x = unpack2<T>(w);
                    top = fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y)));
                }
            float scale = p.scale;
            if constexpr (std::is_same<T, __nv_bfloat16>::value) {
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
                        const float2 x = unpack2<T>(raw[k][i]);
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
        float s[EIGHTS][KT / 16][4];  // of each sixteen: keys lane / 4 and 8 + lane / 4, both heads each
#pragma unroll
        for (int h = 0; h < EIGHTS; ++h)
#pragma unroll
            for (int g = 0; g < KT / 16; ++g)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[h][g][i] = 0.f;
#pragma unroll
        for (int k = 0; k < kChunks; k += 2)
#pragma unroll
            for (int g = 0; g < KT / 16; ++g) {
                uint32_t a[4];
                ldmatrix4(a, keys + lay.offset(g * 16 + (lane & 15), k + (lane >> 4)));
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t even[2], odd[2];
                    to_pairs<P>(a[2 * c], even[0], odd[0]);
                    to_pairs<P>(a[2 * c + 1], even[1], odd[1]);
#pragma unroll
                    for (int h = 0; h < EIGHTS; ++h) mma_16816<__half>(s[h][g], even[0], even[1], odd[0], odd[1], q[h][k + c][0], q[h][k + c][1]);
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
            back[j] = __int_as_float(0x7f000000 - (bits & 0x7f800000));
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
                    x = fmaf(x * ks[j], q_scale[h][a], e[j]);
                    if (marks.x != 0xffffffffu || marks.y != 0) {
                        const int key = key_of(j) + lane / 4;
                        x = marks.y >> key & 1 ? CUDART_NAN_F : marks.x >> key & 1 ? x : -CUDART_INF_F;
                    }
                    w[h][j][a] = x;
                    top[h][a] = fmaxf(top[h][a], x);
                }
            }
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
#pragma unroll
        for (int k = 0; k < kChunks; k += 2) {
            uint32_t a[KT / 16][4];
#pragma unroll
            for (int g = 0; g < KT / 16; ++g) ldmatrix4_trans(a[g], values + lay.offset(g * 16 + (lane & 15), k + (lane >> 4)));
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float sum[KT / 16][EIGHTS][4];  // of this tile
#pragma unroll
                for (int g = 0; g < KT / 16; ++g) {
                    uint32_t even[2], odd[2];
                    to_pairs<P>(a[g][2 * c], even[0], odd[0]);
                    to_pairs<P>(a[g][2 * c + 1], even[1], odd[1]);
#pragma unroll
                    for (int h = 0; h < EIGHTS; ++h) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) sum[g][h][i] = 0.f;
#pragma unroll
                        for (int n = 0; n < kTerms8; ++n)
                            mma_16816<__half>(sum[g][h], even[0], odd[0], even[1], odd[1], weights[h][g][0][n], weights[h][g][1][n]);
                    }
                }
#pragma unroll
                for (int h = 0; h < EIGHTS; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float x = sum[0][h][i];
#pragma unroll
                        for (int g = 1; g < KT / 16; ++g) x += sum[g][h][i];
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
            T* at = static_cast<T*>(p.o) + row_at<false>(p, p.os, rows, r) + d;
            if (p.o_pairs) {
                *reinterpret_cast<uint32_t*>(at) = pack2<T>(x[0] * scale, x[1] * scale);
            } else {
                at[0] = from_f32<T>(x[0] * scale);
                at[1] = from_f32<T>(x[1] * scale);
            }
        });
    }
};

// as many heads as a group has, the next power of two of them
template <typename T, typename P, int DH, typename F>
int with_mma(const tmw_paged_attention_desc& d, F&& use) {
    constexpr int W = DH > 128 ? 6 : DH > 64 ? 12 : 16;
    const int group = d.heads / d.at.kv_heads;
    if (group == 1) return use(Kernel<T, P, false, Mma8Core<T, P, DH, 1>, W, 2>());
    if (group == 2) return use(Kernel<T, P, false, Mma8Core<T, P, DH, 2>, W, 2>());
    if (group <= 4) return use(Kernel<T, P, false, Mma8Core<T, P, DH, 4>, W, 2>());
    if (group <= 8) return use(Kernel<T, P, false, Mma8Core<T, P, DH, 8>, W, 2>());
    return use(Kernel<T, P, false, Mma8Core<T, P, DH, 16>, (DH > 64 ? W : 12), 2>());
}
template <typename T, typename P, typename F>
int with_16_bits(const tmw_paged_attention_desc& d, F&& use) {
    if constexpr (sizeof(T) == 2) {
        switch (d.at.head_dim) {
            case 32: return with_mma<T, P, 32>(d, use);
            case 64: return with_mma<T, P, 64>(d, use);
            case 96: return with_mma<T, P, 96>(d, use);
            case 128: return with_mma<T, P, 128>(d, use);
            case 256: return with_mma<T, P, 256>(d, use);
        }
    }
    return with_simt<T, P, false>(d, 1, use);
}
template <typename T, typename F>
int with_pages(const tmw_paged_attention_desc& d, const tmw_page_scales& s, F&& use) {
    return s.format == TMW_PAGES_INT8 ? with_16_bits<T, int8_t>(d, use) : with_16_bits<T, E4m3>(d, use);
}
// `use` with the Kernel that takes the call
template <typename F>
int with_kernel(const tmw_paged_attention_desc& d, const tmw_page_scales& s, F&& use) {
    if (d.at.dtype == TMW_F32) return with_pages<float>(d, s, use);
    return d.at.dtype == TMW_BF16 ? with_pages<__nv_bfloat16>(d, s, use) : with_pages<__half>(d, s, use);
}

int validate(const tmw_paged_attention_desc* d, const tmw_page_scales* s, bool& used) {
    const int rc = validate(d, used);
    if (rc != TMW_OK) return rc;
    if (s == nullptr || s->format == TMW_PAGES_SAME) return TMW_ERR_INVALID_ARGUMENT;
    return validate_scales(d->at, *s, false, false);
}

}  // namespace
}  // namespace tmw

extern "C" size_t tmw_paged_attention_scaled_scratch_bytes(const tmw_paged_attention_desc* d, const tmw_page_scales* s) {
    using namespace tmw;
    bool used = false;
    if (validate(d, s, used) != TMW_OK || !used) return 0;
    size_t bytes = 0;
    with_kernel(*d, *s, [&](auto kernel) {
        bytes = kernel.plan(*d, d->at.head_dim, 1).bytes;
        return TMW_OK;
    });
    return bytes;
}

extern "C" int tmw_paged_attention_scaled(const tmw_paged_attention_desc* d, const tmw_page_scales* s, void* scratch, size_t scratch_bytes,
                                          void* stream) {
    using namespace tmw;
    bool used = false;
    const int rc = validate(d, s, used);
    if (rc != TMW_OK || !used) return rc;
    PagedAttention p;
    const int bad = arguments(*d, *s, scratch, p);
    if (bad != TMW_OK) return bad;
    return with_kernel(*d, *s, [&](auto kernel) {
        const Plan n = kernel.plan(*d, p.row_bytes, 1);
        if (scratch_bytes < n.bytes) {
            set_error_text("tmw_paged_attention_scaled: scratch smaller than tmw_paged_attention_scaled_scratch_bytes()");
            return (int)TMW_ERR_INVALID_ARGUMENT;
        }
        return kernel.launch(p, n, static_cast<unsigned char*>(scratch), static_cast<cudaStream_t>(stream));
    });
}
