// Which kernel a launch takes.  Internal.
#pragma once
#include "attention_tiles.cuh"

namespace halo_cuda {
namespace attn {

/// Sequences of up to few_rows packed rows: the row kernel, 16 rows at a time, each fetching the keys again (from L2).
template <int D>
int launch_kernel(HaloCudaCtx* ctx, const AttentionCall& c, const Work& w, cudaStream_t s) {
    return with_type(c.type, [&](auto t) {
        using T = decltype(t);
        if (w.max_rows <= few_rows(c)) return launch_rows_kernel<T, D, 4, 64, D == 256 ? 1 : 3>(ctx, c, w, s);
        return launch_tiles_kernel<T, D>(ctx, c, w, s);
    });
}

}  // namespace attn
}  // namespace halo_cuda
