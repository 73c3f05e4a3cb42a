// attn_umma.cu — the host side of attn_umma.cuh's kernels.
#include "attn_umma.cuh"

namespace warp {

static CUresult (*encode_fn())(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *,
                               const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                               const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                               CUtensorMapL2promotion, CUtensorMapFloatOOBfill) {
    static const auto fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault,
                                             &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            p = nullptr;
        }
        return (decltype(encode_fn()))p;
    }();
    return fn;
}

// The pages as a tensor (dim, slot, head, page), boxes of 64 columns by a page's
// keys (a tile's at most).
static int page_map(CUtensorMap *m, const warp_kv_pages *c, void *ptr, int64_t page, int64_t slot,
                    int64_t head) {
    const auto fn = encode_fn();
    if (!fn) {
        set_error("warp_paged_attention: the driver has no cuTensorMapEncodeTiled");
        return WARP_E_CUDA;
    }
    const cuuint64_t row = (cuuint64_t)c->head_dim * 2;
    const cuuint64_t dims[4] = {(cuuint64_t)c->head_dim, (cuuint64_t)c->page_size,
                                (cuuint64_t)c->kv_heads, (cuuint64_t)c->pages};
    // the stride of an axis of one entry may be given as 0
    const cuuint64_t strides[3] = {slot ? (cuuint64_t)slot * 2 : row,
                                   head ? (cuuint64_t)head * 2 : row,
                                   page ? (cuuint64_t)page * 2 : row};
    const int keys = attn_wide(c->head_dim);
    const cuuint32_t box[4] = {64, (cuuint32_t)(c->page_size < keys ? c->page_size : keys), 1, 1};
    const cuuint32_t ones[4] = {1, 1, 1, 1};
    const CUresult r = fn(m, c->type == WARP_T_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                   : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                          4, ptr, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_error("warp_paged_attention: the pages' layout does not make a tensor map (%d)", (int)r);
        return WARP_E_ARG;
    }
    return WARP_OK;
}

int attn_umma(const AttnArgs &a, const warp_kv_pages *c, AttnKind kind, bool first,
              cudaStream_t st) {
    CUtensorMap km, vm;
    int rc = page_map(&km, c, c->k, c->k_page, c->k_slot, c->k_head);
    if (!rc) rc = page_map(&vm, c, c->v, c->v_page, c->v_slot, c->v_head);
    if (rc) return rc;
    const bool packed = kind == kAttnPacked;
    const int64_t rows = (int64_t)(packed ? a.tokens : a.max_q) * a.group;
    const unsigned pairs = (unsigned)((rows + 2 * kRows - 1) / (2 * kRows));
    const dim3 grid = kind == kAttnTreeRuns
                          ? dim3(a.runs)
                          : dim3(pairs * (packed ? a.prefix_parts : a.wide_parts), a.kv_heads,
                                 packed ? 1 : a.batch);
    const WideLaunch l = {a, km, vm, grid, first, st};
    return packed              ? l.typed<kAttnPacked>(c)
           : kind == kAttnOwn ? l.typed<kAttnOwn>(c)
                              : attn_umma_tree(l, c, kind);
}

}  // namespace warp
