// The kernels of attention_rows.cuh for heads of 256 elements.
#include "attention_rows_launch.cuh"

namespace halo_cuda {
namespace attn {
template int launch_rows<256>(HaloCudaCtx*, const AttentionCall&, const Work&, cudaStream_t);
}
}  // namespace halo_cuda
