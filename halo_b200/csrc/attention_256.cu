// The attention kernels for heads of 256 elements.
#include "attention_launch.cuh"

namespace halo_cuda {
namespace attn {
template int launch_kernel<256>(HaloCudaCtx*, const AttentionCall&, const Work&, cudaStream_t);
}
}  // namespace halo_cuda
