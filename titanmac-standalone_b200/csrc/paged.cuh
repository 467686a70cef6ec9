// What the kernels over paged keys and values share (internal): where a token lives.
#pragma once

#include <initializer_list>

#include "tmw_common.cuh"

namespace tmw {

// n / d for 0 <= n < 2^31 by a product: with 2^s the first power of two at or above d and m = floor(2^32 (2^s - d) / d) + 1,
// n / d = (high word of m n, plus n) >> s (Granlund and Montgomery, "Division by invariant integers using multiplication", 1994).
struct FastDiv {
    uint32_t m, s, d;
    FastDiv() = default;
    explicit FastDiv(uint32_t div) : d(div) {
        s = 0;
        while ((1ull << s) < div) ++s;
        m = (uint32_t)(((1ull << 32) * ((1ull << s) - div)) / div + 1);
    }
    __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(m, n) + n) >> s; }
};

struct PageMap {
    const int32_t* table;
    long long table_stride;
    int columns, pages, kv_heads, head_dim;
    long long capacity;  // tokens that a row of the table has room for
    FastDiv page;

    PageMap() = default;
    explicit PageMap(const tmw_pages& p)
        : table(p.page_table), table_stride(p.table_stride), columns(p.columns), pages(p.pages), kv_heads(p.kv_heads),
          head_dim(p.head_dim), capacity((long long)p.columns * p.page_size), page((uint32_t)p.page_size) {}

    // Offset, in elements, of token t (0 <= t < capacity) of sequence b under head 0; -1: its page is not one of the pool.
    __device__ __forceinline__ long long token(int b, int t) const {
        const uint32_t column = page.div((uint32_t)t);
        const int at = __ldg(table + b * table_stride + column);
        if ((uint32_t)at >= (uint32_t)pages) return -1;
        return ((long long)at * kv_heads * page.d + (t - column * page.d)) * head_dim;
    }
    // the same counted in rows
    __device__ __forceinline__ long long row(int b, int t) const {
        const uint32_t column = page.div((uint32_t)t);
        const int at = __ldg(table + b * table_stride + column);
        if ((uint32_t)at >= (uint32_t)pages) return -1;
        return (long long)at * kv_heads * page.d + (t - column * page.d);
    }
    // from one head's rows to the next one's
    __device__ __forceinline__ long long head_step() const { return (long long)page.d * head_dim; }
};

// Pages in 8 bits: a code of four exponent and three fraction bits.
struct E4m3 {
    uint8_t bits;
};
__device__ __forceinline__ __half2 from_e4m3(uint32_t two) {  // the lower two codes
    uint32_t w;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(w) : "h"((uint16_t)two));
    return *reinterpret_cast<const __half2*>(&w);
}

// TMW_OK, or what is wrong with the description (the pointers only where there is something to do)
inline int validate_pages(const tmw_pages& p, bool used) {
    if (p.dtype != TMW_F32 && p.dtype != TMW_BF16 && p.dtype != TMW_F16) return TMW_ERR_UNSUPPORTED;
    if (p.batch < 0 || p.kv_heads <= 0 || p.head_dim <= 0 || p.page_size <= 0 || p.pages < 0 || p.columns < 0 || p.table_stride < 0)
        return TMW_ERR_INVALID_ARGUMENT;
    if (p.head_dim % 8 != 0 || p.head_dim > 256) {
        set_error_text("paged cache: head_dim must be a multiple of 8, at most 256");
        return TMW_ERR_UNSUPPORTED;
    }
    if ((long long)p.columns * p.page_size > 0x7fffffffLL || p.batch > 65535 || p.kv_heads > 65535) return TMW_ERR_TOO_LARGE;
    if (!used) return TMW_OK;
    if (p.columns > 0 && p.page_table == nullptr) return TMW_ERR_INVALID_ARGUMENT;
    if (p.pages > 0 && (p.k_pages == nullptr || p.v_pages == nullptr)) return TMW_ERR_INVALID_ARGUMENT;
    if ((reinterpret_cast<uintptr_t>(p.k_pages) | reinterpret_cast<uintptr_t>(p.v_pages)) & 15u) return TMW_ERR_INVALID_ARGUMENT;
    return TMW_OK;
}

// The same of the scales, with as many pointers as a call needs.
inline int validate_scales(const tmw_pages& p, const tmw_page_scales& s, bool used, bool persistent) {
    if (s.format != TMW_PAGES_SAME && s.format != TMW_PAGES_INT8 && s.format != TMW_PAGES_E4M3) return TMW_ERR_UNSUPPORTED;
    if (s.format == TMW_PAGES_SAME) return TMW_OK;
    if (p.head_dim % 16 != 0) {
        set_error_text("paged cache: head_dim must be a multiple of 16 with pages in 8 bits");
        return TMW_ERR_UNSUPPORTED;
    }
    if (!used) return TMW_OK;
    if (p.pages > 0 && (s.k_scales == nullptr || s.v_scales == nullptr)) return TMW_ERR_INVALID_ARGUMENT;
    if (persistent && (s.k_pers_scales == nullptr || s.v_pers_scales == nullptr)) return TMW_ERR_INVALID_ARGUMENT;
    const auto bits = [](const float* x) { return reinterpret_cast<uintptr_t>(x); };
    if ((bits(s.k_scales) | bits(s.v_scales) | bits(s.k_pers_scales) | bits(s.v_pers_scales)) % 4 != 0) return TMW_ERR_INVALID_ARGUMENT;
    return TMW_OK;
}

// Whether an output's strides bring its rows to places of their own, as far as a stride of 0 tells.
inline bool rows_apart(const int64_t* strides, std::initializer_list<int> extents) {
    for (int n : extents)
        if (*strides++ == 0 && n > 1) return false;
    return true;
}

}  // namespace tmw
