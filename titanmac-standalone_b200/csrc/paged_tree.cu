// Attention of the drafted tokens of a tree over paged keys (tmw_paged_tree_attention).
#include "paged_tree.cuh"

namespace tmw {
namespace {

constexpr int kMostNodes = 64;  // bits of a word

// what the kernels over paged keys share, as they are asked for one new token
tmw_paged_attention_desc shared_part(const tmw_paged_tree_desc& d) {
    tmw_paged_attention_desc one = {};
    one.at = d.at;
    one.heads = d.heads; one.n_persistent = d.n_persistent; one.window = d.window;
    one.scale = d.scale;
    one.q = d.q; one.k_pers = d.k_pers; one.v_pers = d.v_pers;
    one.o = d.o;
    for (int i = 0; i < 2; ++i) {
        one.q_stride[i] = d.q_stride[i];
        one.o_stride[i] = d.o_stride[i];
    }
    one.pos = d.start;
    return one;
}

// what the kernel on tensor cores does not take: fp32, head sizes that it is not built for
template <typename T, typename F>
int with_pages(const tmw_paged_attention_desc& d, const tmw_page_scales& s, int nodes, F&& use) {
    if (s.format == TMW_PAGES_INT8) return with_simt<T, int8_t, true>(d, nodes, use);
    if (s.format == TMW_PAGES_E4M3) return with_simt<T, E4m3, true>(d, nodes, use);
    if constexpr (std::is_same<T, Any16>::value) {
        return d.at.dtype == TMW_BF16 ? with_simt<T, __nv_bfloat16, true>(d, nodes, use) : with_simt<T, __half, true>(d, nodes, use);
    } else {
        return with_simt<T, T, true>(d, nodes, use);
    }
}
// `use` with the Kernel that takes the call
template <typename F>
int with_kernel(const tmw_paged_attention_desc& d, const tmw_page_scales& s, int nodes, F&& use) {
    return d.at.dtype == TMW_F32 ? with_pages<float>(d, s, nodes, use) : with_pages<Any16>(d, s, nodes, use);
}

int validate(const tmw_paged_tree_desc* d, const tmw_page_scales& s, bool& used) {
    if (d == nullptr || d->nodes < 0) return TMW_ERR_INVALID_ARGUMENT;
    tmw_paged_attention_desc one = shared_part(*d);
    if (d->nodes == 0) one.at.batch = min(one.at.batch, 0);  // nothing to do
    const int rc = validate(&one, used);
    if (rc != TMW_OK) return rc;
    if (d->nodes > kMostNodes) {
        set_error_text("tmw_paged_tree_attention: at most 64 nodes");
        return TMW_ERR_TOO_LARGE;
    }
    return validate_scales(d->at, s, false, false);
}

int row_bytes(const tmw_paged_tree_desc& d, const tmw_page_scales& s) {
    return d.at.head_dim * (s.format == TMW_PAGES_SAME ? (int)dtype_size(d.at.dtype) : 1);
}

}  // namespace
}  // namespace tmw

extern "C" size_t tmw_paged_tree_attention_scratch_bytes(const tmw_paged_tree_desc* d, const tmw_page_scales* scales) {
    using namespace tmw;
    const tmw_page_scales s = scales != nullptr ? *scales : tmw_page_scales{};
    bool used = false;
    if (validate(d, s, used) != TMW_OK || !used) return 0;
    const tmw_paged_attention_desc one = shared_part(*d);
    size_t bytes = 0;
    if (d->at.dtype != TMW_F32) {
        if (tree_scratch_tc(one, s, d->nodes, bytes)) return bytes;
        const auto of = s.format == TMW_PAGES_INT8   ? tree_scratch_int8
                        : s.format == TMW_PAGES_E4M3 ? tree_scratch_e4m3
                        : d->at.dtype == TMW_BF16    ? tree_scratch_bf16
                                                     : tree_scratch_f16;
        if (of(one, s, d->nodes, bytes)) return bytes;
    }
    with_kernel(one, s, d->nodes, [&](auto kernel) {
        bytes = kernel.plan(one, row_bytes(*d, s), d->nodes).bytes;
        return TMW_OK;
    });
    return bytes;
}

extern "C" int tmw_paged_tree_attention(const tmw_paged_tree_desc* d, const tmw_page_scales* scales, void* scratch, size_t scratch_bytes,
                                        void* stream) {
    using namespace tmw;
    const tmw_page_scales s = scales != nullptr ? *scales : tmw_page_scales{};
    bool used = false;
    const int rc = validate(d, s, used);
    if (rc != TMW_OK || !used) return rc;
    if (d->seen == nullptr || (d->window >= 0 && d->positions == nullptr) || d->q_stride[2] < 0 || d->o_stride[2] < 0 ||
        reinterpret_cast<uintptr_t>(d->seen) % 8 != 0)
        return TMW_ERR_INVALID_ARGUMENT;
    if (!rows_apart(d->o_stride, {d->at.batch, d->heads, d->nodes})) {
        set_error_text("tmw_paged_tree_attention: every output must have a place of its own");
        return TMW_ERR_INVALID_ARGUMENT;
    }
    const tmw_paged_attention_desc one = shared_part(*d);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (d->at.dtype != TMW_F32) {
        const auto run = s.format == TMW_PAGES_INT8   ? tree_launch_int8
                         : s.format == TMW_PAGES_E4M3 ? tree_launch_e4m3
                         : d->at.dtype == TMW_BF16    ? tree_launch_bf16
                                                      : tree_launch_f16;
        int status = TMW_OK;
        if (tree_launch_tc(one, s, *d, scratch, scratch_bytes, st, status)) return status;
        if (run(one, s, *d, scratch, scratch_bytes, st, status)) return status;
    }
    PagedAttention p;
    const int bad = tree_arguments(one, s, *d, scratch, p);
    if (bad != TMW_OK) return bad;
    return with_kernel(one, s, d->nodes, [&](auto kernel) {
        const Plan n = kernel.plan(one, p.row_bytes, d->nodes);
        if (scratch_bytes < n.bytes) {
            set_error_text("tmw_paged_tree_attention: scratch smaller than tmw_paged_tree_attention_scratch_bytes()");
            return (int)TMW_ERR_INVALID_ARGUMENT;
        }
        return kernel.launch(p, n, static_cast<unsigned char*>(scratch), st);
    });
}
