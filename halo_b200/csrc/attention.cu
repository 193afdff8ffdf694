// ATTENTION over the paged 8-bit cache: which kernels a call runs.
#include <cuda.h>

#include "attention_rows.cuh"

namespace halo_cuda {
namespace attn {

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                   CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

int pool_map(const Cache& c, const uint8_t* pool, uint32_t box_rows, CUtensorMap* out) {
    static EncodeTiledFn encode = nullptr;
    if (encode == nullptr) {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult qres;
        HC_CUDA(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &qres));
        if (fn == nullptr || qres != cudaDriverEntryPointSuccess) return fail(HALO_CUDA_E_BACKEND, "cuTensorMapEncodeTiled is not available");
        encode = reinterpret_cast<EncodeTiledFn>(fn);
    }
    const bool narrow = c.head_dim == 64;
    const cuuint64_t dims[3] = {c.head_dim, uint64_t{c.n_kv} * c.page_tokens, c.n_pages};
    const cuuint64_t strides[2] = {c.head_dim, c.page_stride};
    const cuuint32_t box[3] = {narrow ? 64u : 128u, box_rows, 1}, elem[3] = {1, 1, 1};
    const CUresult r = encode(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<uint8_t*>(pool), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              narrow ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(HALO_CUDA_E_KERNEL, "ATTENTION: cannot describe the cache to the copy engine (CUresult %d)", static_cast<int>(r));
    return 0;
}

int launch_attention(HaloCudaCtx* ctx, const AttentionCall& c, cudaStream_t s) {
    if (c.cache.n_pages == 0 || c.cache.max_pages == 0) return fail(HALO_CUDA_E_UNSUPPORTED, "ATTENTION: a cache without pages");
    auto run = [&](uint32_t min_rows, uint32_t max_rows) {
        Work w{};
        w.window = static_cast<int32_t>(std::min(c.window, 0x7FFFFFFFu));
        w.min_rows = min_rows;
        w.max_rows = max_rows;
        return c.cache.head_dim == 64 ? launch_kernel<64>(ctx, c, w, s) : c.cache.head_dim == 128 ? launch_kernel<128>(ctx, c, w, s) : launch_kernel<256>(ctx, c, w, s);
    };
    // Sequences of few rows among others run in a launch of their own.
    const uint32_t most = c.rows.max_tokens * c.group, few = few_rows(c);
    const bool ragged = c.rows.n_tokens < uint64_t{c.cache.n_seq} * c.rows.max_tokens;
    if (most <= few || !ragged) return run(1, most);
    if (int rc = run(1, few)) return rc;
    return run(few + 1, most);
}

}  // namespace attn
}  // namespace halo_cuda
