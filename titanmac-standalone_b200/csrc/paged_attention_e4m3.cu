// Attention of one new token per sequence over pages of e4m3 codes.
#include "paged_attention8.cuh"

namespace tmw {

size_t paged_attention_e4m3_scratch(const tmw_paged_attention_desc& d, const tmw_page_scales& s) { return scratch_bytes_of<E4m3>(d, s); }
int paged_attention_e4m3(const tmw_paged_attention_desc& d, const tmw_page_scales& s, void* scratch, size_t scratch_bytes, cudaStream_t stream) {
    return launch_of<E4m3>(d, s, scratch, scratch_bytes, stream);
}

}  // namespace tmw
