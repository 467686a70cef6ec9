// Attention of one new token per sequence over pages of the model's type (tmw_paged_attention): which kernel takes a call.
#include "paged_attention.cuh"

namespace tmw {
namespace {

template <typename T, int DH, typename F>
int with_mma(const tmw_paged_attention_desc& d, F&& use) {
    constexpr int W = DH >= 128 ? 6 : DH > 64 ? 8 : 12;
    if (d.heads / d.at.kv_heads <= 8) return use(Kernel<T, T, false, MmaCore<T, DH, 1>, W, 2>());
    return use(Kernel<T, T, false, MmaCore<T, DH, 2>, W, 2>());
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
        default: return with_simt<T, T, false>(d, 1, use);
    }
}

// `use` with the Kernel that takes the call
template <typename F>
int with_kernel(const tmw_paged_attention_desc& d, F&& use) {
    if (d.at.dtype == TMW_F32) return with_simt<float, float, false>(d, 1, use);
    return d.at.dtype == TMW_BF16 ? with_16_bits<__nv_bfloat16>(d, use) : with_16_bits<__half>(d, use);
}

}  // namespace
}  // namespace tmw

extern "C" size_t tmw_paged_attention_scratch_bytes(const tmw_paged_attention_desc* d) {
    using namespace tmw;
    bool used = false;
    if (validate(d, used) != TMW_OK || !used) return 0;
    size_t bytes = 0;
    with_kernel(*d, [&](auto kernel) {
        bytes = kernel.plan(*d, d->at.head_dim * (int)dtype_size(d->at.dtype), 1).bytes;
        return TMW_OK;
    });
    return bytes;
}

extern "C" int tmw_paged_attention(const tmw_paged_attention_desc* d, void* scratch, size_t scratch_bytes, void* stream) {
    using namespace tmw;
    bool used = false;
    const int rc = validate(d, used);
    if (rc != TMW_OK || !used) return rc;
    PagedAttention p;
    const int bad = arguments(*d, tmw_page_scales{}, scratch, p);
    if (bad != TMW_OK) return bad;
    return with_kernel(*d, [&](auto kernel) {
        const Plan n = kernel.plan(*d, p.row_bytes, 1);
        if (scratch_bytes < n.bytes) {
            set_error_text("tmw_paged_attention: scratch smaller than tmw_paged_attention_scratch_bytes()");
            return (int)TMW_ERR_INVALID_ARGUMENT;
        }
        return kernel.launch(p, n, static_cast<unsigned char*>(scratch), static_cast<cudaStream_t>(stream));
    });
}
