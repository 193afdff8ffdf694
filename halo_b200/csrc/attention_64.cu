// The attention kernels for heads of 64 elements.
#include "attention_launch.cuh"

namespace halo_cuda {
namespace attn {
template int launch_kernel<64>(HaloCudaCtx*, const AttentionCall&, const Work&, cudaStream_t);
}
}  // namespace halo_cuda
