// What the appends to pages of either form share (internal): their arguments, checked.
#pragma once

#include "paged.cuh"

namespace tmw {

struct PagedAppend {
    PageMap map;
    const void *k, *v, *q;
    void *k_pages, *v_pages, *q_out;
    long long ks[3], vs[3], qs[3], os[3];  // {batch, head, row}
    const int32_t *start, *counts, *positions;
    const float* inv_freq;
    int rows, heads, half;
    int step_r, step_slot, step_u;  // from a thread's pair of vectors to its next one: tokens, heads, pairs
    float *k_scales, *v_scales;         // of pages in 8 bits
    int* status;
};

// The arguments of a description; used: there is something to do; bits, strides: of every address and stride of k, v, q and q_out.
inline int append_arguments(const tmw_paged_append_desc* d, const tmw_page_scales* scales, const int32_t* positions, PagedAppend& p,
                            bool& used, uintptr_t& bits, long long& strides) {
    if (d == nullptr) return TMW_ERR_INVALID_ARGUMENT;
    used = d->at.batch > 0 && d->rows > 0;
    int rc = validate_pages(d->at, used);
    if (rc != TMW_OK) return rc;
    if (scales != nullptr && (rc = validate_scales(d->at, *scales, used, false)) != TMW_OK) return rc;
    if (d->rows < 0 || d->heads < 0 || d->rotated < 0 || d->rotated % 2 != 0 || d->rotated > d->at.head_dim)
        return TMW_ERR_INVALID_ARGUMENT;
    if (!used) return TMW_OK;
    if (d->k == nullptr || d->v == nullptr || d->start == nullptr || (d->rotated > 0 && d->inv_freq == nullptr) ||
        (d->heads > 0 && (d->q == nullptr || d->q_out == nullptr)))
        return TMW_ERR_INVALID_ARGUMENT;
    const size_t size = dtype_size(d->at.dtype);
    bits = 0;
    strides = 0;
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

    p = {};
    p.map = PageMap(d->at);
    p.k = d->k; p.v = d->v; p.q = d->q;
    p.k_pages = d->at.k_pages; p.v_pages = d->at.v_pages; p.q_out = d->q_out;
    for (int i = 0; i < 3; ++i) {
        p.ks[i] = d->k_stride[i];
        p.vs[i] = d->v_stride[i];
        p.qs[i] = d->q_stride[i];
        p.os[i] = d->q_out_stride[i];
    }
    p.start = d->start; p.counts = d->counts; p.positions = positions; p.inv_freq = d->inv_freq;
    p.rows = d->rows; p.heads = d->heads; p.half = d->rotated / 2;
    p.status = device_status_word();
    if (scales != nullptr) p.k_scales = scales->k_scales, p.v_scales = scales->v_scales;
    return p.status == nullptr ? TMW_ERR_CUDA : TMW_OK;
}

// the append to pages of the model's type
int append_same(PagedAppend& p, const tmw_paged_append_desc& d, uintptr_t bits, long long strides, cudaStream_t stream);

}  // namespace tmw
