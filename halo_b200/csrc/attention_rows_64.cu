// The kernels of attention_rows.cuh for heads of 64 elements.
#include "attention_rows_launch.cuh"

namespace halo_cuda {
namespace attn {
template int launch_rows<64>(HaloCudaCtx*, const AttentionCall&, const Work&, cudaStream_t);
}
}  // namespace halo_cuda
