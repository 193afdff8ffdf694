// The validated call of PARTIAL_ROPE.  Not part of the ABI.
#pragma once
#include "attention.h"

namespace halo_cuda {
namespace attn {

struct RopeCall {
    uint32_t type, interleaved;
    const int32_t* positions;
    Heads q, k, q_out, k_out;
    uint32_t n_tokens, n_q, n_kv, head_dim;
    const HaloCudaRopeFreqs* freqs;
};
int launch_rope(const RopeCall& c, cudaStream_t s);

}  // namespace attn
}  // namespace halo_cuda
