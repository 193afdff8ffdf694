// Which of the row kernels a launch takes.  Internal.
#pragma once
#include "attention_tiles.cuh"

namespace halo_cuda {
namespace attn {

template <int D>
int launch_rows(HaloCudaCtx* ctx, const AttentionCall& c, const Work& w, cudaStream_t s) {
    return with_type(c.type, [&](auto t) {
        using T = decltype(t);
        if (w.max_rows <= 16) return launch_rows_kernel<T, D, 4, 64, D == 256 ? 1 : 3>(ctx, c, w, s);
        return launch_tiles_kernel<T, D>(ctx, c, w, s);
    });
}

}  // namespace attn
}  // namespace halo_cuda
