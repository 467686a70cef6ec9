// Attention of a tree's drafted tokens over pages of int8 codes.
#include "paged_tree.cuh"

namespace tmw {

bool tree_scratch_int8(const tmw_paged_attention_desc& d, const tmw_page_scales& s, int nodes, size_t& bytes) {
    return tree_scratch_of<int8_t>(d, s, nodes, bytes);
}
bool tree_launch_int8(const tmw_paged_attention_desc& d, const tmw_page_scales& s, const tmw_paged_tree_desc& tree, void* scratch,
                        size_t scratch_bytes, cudaStream_t stream, int& status) {
    PagedAttentionBulk p;
    status = tree_arguments(d, s, tree, scratch, p);
    return status != TMW_OK || tree_launch_of<int8_t>(d, s, p, scratch, scratch_bytes, stream, status);
}

}  // namespace tmw
