// attn_umma_tree.cu — attn_umma.cuh's kernels for the nodes of trees.
#include "attn_umma.cuh"

namespace warp {

int attn_umma_tree(const WideLaunch &l, const warp_kv_pages *c, AttnKind kind) {
    return kind == kAttnTree ? l.typed<kAttnTree>(c) : l.typed<kAttnTreeRuns>(c);
}

}  // namespace warp
