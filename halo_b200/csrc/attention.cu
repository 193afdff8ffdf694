// ATTENTION over the paged 8-bit cache: a warp for every (row, query head), a cached token at a time.
//
//   x_t = scale * q . K[t], m = max x, o = sum exp(x_t - m) V[t] / sum exp(x_t - m), kept as a running maximum, sum and weighted row.
#include <cuda_fp8.h>

#include "attention.h"

namespace halo_cuda {
namespace attn {
namespace {

__device__ __forceinline__ float code(uint32_t byte) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte), __NV_E4M3)));
}

template <class T, int D>
__global__ void __launch_bounds__(128) attention_kernel(const AttentionCall c) {
    constexpr int E = D / 32;
    const uint32_t lane = threadIdx.x % 32, h = blockIdx.y * 4 + threadIdx.x / 32, seq = blockIdx.z;
    if (h >= c.n_q) return;
    const Seq s = sequence(c.rows, c.cache, seq);
    for (uint32_t j = blockIdx.x; j < s.count; j += gridDim.x) {
        const int32_t pos = s.length - static_cast<int32_t>(s.count) + static_cast<int32_t>(j);
        const int32_t hi = c.causal ? min(pos + 1, s.length) : s.length;
        const int32_t lo = c.window != 0 ? static_cast<int32_t>(max(int64_t{0}, int64_t{pos} + 1 - c.window)) : 0;
        const T* q = reinterpret_cast<const T*>(c.q.p + uint64_t{s.row0 + j} * c.q.token_stride + uint64_t{h} * c.q.head_stride);
        float x[E], o[E] = {}, m = -INFINITY, l = 0;
        for (int e = 0; e < E; ++e) x[e] = to_f32(q[lane * E + e]) * c.scale;
        for (int32_t t = lo; t < hi; ++t) {
            const int32_t page = page_of(c.cache, seq, t >> c.cache.page_shift);
            if (static_cast<uint32_t>(page) >= c.cache.n_pages) {
                if (lane == 0 && c.status != nullptr) atomicOr(c.status, 8u);  // kStatusBadIndex
                continue;
            }
            const uint32_t kvh = h / c.group;
            const uint64_t at = page * c.cache.page_stride + (uint64_t{kvh} * c.cache.page_tokens + (t & (c.cache.page_tokens - 1))) * D + lane * E;
            const uint64_t sc = page * c.cache.scale_stride + kvh;
            float dot = 0;
            for (int e = 0; e < E; ++e) dot += x[e] * code(c.cache.k[at + e]);
            for (int d = 16; d != 0; d >>= 1) dot += __shfl_xor_sync(0xFFFFFFFFu, dot, d);
            dot *= exp2_int(scale_byte(c.cache.k_scale[sc]) - 127);
            const float next = fmaxf(m, dot), old = m == -INFINITY ? 0 : expf(m - next), p = expf(dot - next);
            const float pv = p * exp2_int(scale_byte(c.cache.v_scale[sc]) - 127);
            l = l * old + p;
            for (int e = 0; e < E; ++e) o[e] = o[e] * old + pv * code(c.cache.v[at + e]);
            m = next;
        }
        T* out = reinterpret_cast<T*>(c.out.p + uint64_t{s.row0 + j} * c.out.token_stride + uint64_t{h} * c.out.head_stride);
        for (int e = 0; e < E; ++e) out[lane * E + e] = from_f32<T>(hi > lo && l != 0 ? o[e] / l : 0.0f);
    }
}

}  // namespace

int launch_attention(HaloCudaCtx*, const AttentionCall& c, cudaStream_t s) {
    const dim3 grid(std::min(c.rows.max_tokens, 65535u), (c.n_q + 3) / 4, c.cache.n_seq);
    return with_type(c.type, [&](auto t) {
        using T = decltype(t);
        if (c.cache.head_dim == 64) attention_kernel<T, 64><<<grid, 128, 0, s>>>(c);
        else if (c.cache.head_dim == 128) attention_kernel<T, 128><<<grid, 128, 0, s>>>(c);
        else attention_kernel<T, 256><<<grid, 128, 0, s>>>(c);
        HC_CUDA(cudaGetLastError());
        return 0;
    });
}

}  // namespace attn
}  // namespace halo_cuda
