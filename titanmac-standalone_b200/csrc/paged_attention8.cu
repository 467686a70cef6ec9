// Attention of one new token per sequence over pages in 8 bits (tmw_paged_attention_scaled): which kernel takes a call.
#include "paged_attention.cuh"

namespace tmw {
namespace {

template <typename T, typename F>
int with_pages(const tmw_paged_attention_desc& d, const tmw_page_scales& s, F&& use) {
    return s.format == TMW_PAGES_INT8 ? with_simt<T, int8_t, false>(d, 1, use) : with_simt<T, E4m3, false>(d, 1, use);
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
