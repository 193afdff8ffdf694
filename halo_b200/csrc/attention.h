// What the attention layer's translation units share: validated calls and the rows of a call as the kernels see them.  Not part of the ABI.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "halo_cuda_attention.h"
#include "internal.h"

namespace halo_cuda {
namespace attn {

/// Rows of heads with their strides resolved.  `vec`: base and strides are multiples of 16 bytes.
struct Heads {
    uint8_t* p;
    uint64_t token_stride, head_stride;
    uint32_t vec;
};

/// A validated cache; strides resolved, bytes.
struct Cache {
    uint8_t *k, *v;
    uint8_t *k_scale, *v_scale;
    const int32_t* table;
    uint64_t page_stride, scale_stride, table_stride;
    uint32_t n_pages, n_kv, head_dim, page_tokens, page_shift, max_pages, n_seq;
};

struct Rows {
    const int32_t* start;
    const int32_t* length;
    uint32_t n_tokens, max_tokens;
};

struct AttentionCall {
    uint32_t type, n_q, group;  // group: query heads of a kv head
    Cache cache;
    Rows rows;
    Heads q, out;
    uint32_t causal, window;
    float scale;
    uint32_t* status;
};

struct WriteCall {
    uint32_t type;
    Cache cache;
    Rows rows;
    Heads k, v;
    uint32_t* status;
};

/// For addresses that come with the launch, in kernels that are resident while the one in front still writes: the compiler may move __ldg in front of
/// griddepcontrol.wait, but not what passes through a volatile asm behind it.  (Page numbers, pages, scales and rows: their addresses depend on what is read so.
/// Plain loads would do as well; prompts 217 -> 225 us.)
template <class T>
__device__ __forceinline__ T load(const T* p) {
    asm volatile("" : "+l"(p));
    return __ldg(p);
}

/// Sequence i's rows and length, whatever the device arrays hold: [row0, row0 + count) lies inside the operands, length inside the table's row.
struct Seq {
    uint32_t row0, count;
    int32_t length;
};
__device__ __forceinline__ Seq sequence(const Rows& r, const Cache& c, uint32_t i) {
    Seq s;
    if (r.start == nullptr) {
        s.row0 = i * r.max_tokens;
        s.count = r.max_tokens;
    } else {
        const int32_t n = static_cast<int32_t>(r.n_tokens);
        const int32_t lo = min(max(load(r.start + i), 0), n), hi = min(max(load(r.start + i + 1), lo), n);
        s.row0 = static_cast<uint32_t>(lo);
        s.count = min(static_cast<uint32_t>(hi - lo), r.max_tokens);
    }
    s.length = min(max(load(r.length + i), 0), static_cast<int32_t>(c.max_pages << c.page_shift));
    return s;
}
__device__ __forceinline__ int32_t page_of(const Cache& c, uint32_t seq, uint32_t index) {
    return __ldg(reinterpret_cast<const int32_t*>(reinterpret_cast<const uint8_t*>(c.table) + seq * c.table_stride) + index);
}
/// 2^(b - 127) as a float's exponent field, with b held to what the cache allows.
__device__ __forceinline__ int32_t scale_byte(uint32_t b) { return min(max(static_cast<int32_t>(b), HALO_CUDA_KV_SCALE_MIN), HALO_CUDA_KV_SCALE_MAX); }
__device__ __forceinline__ float exp2_int(int32_t e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127

template <class T>
__device__ __forceinline__ float to_f32(T v) {
    if constexpr (sizeof(T) == 4) return v;
    else return static_cast<float>(v);
}
template <class T>
__device__ __forceinline__ T from_f32(float v) {
    if constexpr (sizeof(T) == 4) return v;
    else if constexpr (std::is_same_v<T, __half>) return __float2half_rn(v);
    else return __float2bfloat16_rn(v);
}

int launch_kv_write(HaloCudaCtx* ctx, const WriteCall& c, cudaStream_t s);
int launch_attention(HaloCudaCtx* ctx, const AttentionCall& c, cudaStream_t s);

/// f(T{}) with T the element type of an activation type id that validation has let through.
template <class F>
int with_type(uint32_t type, F&& f) {
    switch (type) {
        case HALO_CUDA_T_F32: return f(float{});
        case HALO_CUDA_T_F16: return f(__half{});
        default: return f(__nv_bfloat16{});
    }
}

}  // namespace attn
}  // namespace halo_cuda
