// Attention of one new token per sequence over pages of int8 codes.
#include "paged_attention8.cuh"

namespace tmw {
namespace {

inline int validate(const tmw_paged_attention_desc* d, const tmw_page_scales* s, bool& used) {
    const int rc = validate(d, used);
    if (rc != TMW_OK) return rc;
    if (s == nullptr || s->format == TMW_PAGES_SAME) return TMW_ERR_INVALID_ARGUMENT;
    return validate_scales(d->at, *s, false, false);
}

}  // namespace

size_t paged_attention_int8_scratch(const tmw_paged_attention_desc& d, const tmw_page_scales& s) { return scratch_bytes_of<int8_t>(d, s); }
int paged_attention_int8(const tmw_paged_attention_desc& d, const tmw_page_scales& s, void* scratch, size_t scratch_bytes, cudaStream_t stream) {
    return launch_of<int8_t>(d, s, scratch, scratch_bytes, stream);
}

}  // namespace tmw

extern "C" size_t tmw_paged_attention_scaled_scratch_bytes(const tmw_paged_attention_desc* d, const tmw_page_scales* s) {
    using namespace tmw;
    bool used = false;
    if (validate(d, s, used) != TMW_OK || !used) return 0;
    return s->format == TMW_PAGES_INT8 ? paged_attention_int8_scratch(*d, *s) : paged_attention_e4m3_scratch(*d, *s);
}

extern "C" int tmw_paged_attention_scaled(const tmw_paged_attention_desc* d, const tmw_page_scales* s, void* scratch, size_t scratch_bytes,
                                          void* stream) {
    using namespace tmw;
    bool used = false;
    const int rc = validate(d, s, used);
    if (rc != TMW_OK || !used) return rc;
    const auto run = s->format == TMW_PAGES_INT8 ? paged_attention_int8 : paged_attention_e4m3;
    return run(*d, *s, scratch, scratch_bytes, static_cast<cudaStream_t>(stream));
}
