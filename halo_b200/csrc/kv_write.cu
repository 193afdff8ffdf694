// KV_WRITE: rows of keys and values -> e4m3 codes in the cache's pages, one power-of-two scale for every (page, kv head).
//
//   s = 2^e, e the smallest integer with max |x| <= 448 * 2^e over the new rows of a page that are finite, and not below the page's scale where
//   earlier tokens of the sequence stay in it;  code = e4m3(x / s);  kept codes become e4m3(code * s_old / s).
//
// Powers of two, because a page is written a token at a time: dividing by one is exact, so is rounding a kept code again unless it falls below the
// smallest normal code, and the bytes do not depend on how the arithmetic is done.  An e4m3 code loses nothing by a scale that is up to
// twice as large as need be, unless it is one of the smallest.
//
// One block for every (sequence, page it touches, kv head, K or V): the page's scale needs the maximum over all of its new rows.  A thread holds
// 16 elements of up to four rows in registers between the maximum and the codes, so every row is read once, and stores 16 codes at a time.
// What bounds it: for prompts HBM (size + 1 bytes an element) and the latency of read, maximum, write in one block (five prompts, 91 MB, 27.5 us, 3.3 TB/s; 22 us
// where the rows are in L2 from the call before); the launch and two dependent reads (table, rows) for single tokens.
#include <cuda_fp8.h>

#include "attention.h"

namespace halo_cuda {
namespace attn {
namespace {

constexpr uint32_t kUnit = 16;  // elements of a thread's unit: one 16-byte store of codes

/// A thread's unit as it lies in memory: 16-bit elements stay packed until they are needed, for the sake of registers.
template <class T>
struct Raw {
    uint32_t word[kUnit * sizeof(T) / 4];
    __device__ __forceinline__ void load(const uint8_t* p, bool vec) {
        if (vec) {
#pragma unroll
            for (uint32_t i = 0; i < kUnit * sizeof(T) / 16; ++i) {
                const uint4 w = __ldg(reinterpret_cast<const uint4*>(p) + i);
                word[4 * i] = w.x, word[4 * i + 1] = w.y, word[4 * i + 2] = w.z, word[4 * i + 3] = w.w;
            }
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (uint32_t i = 0; i < kUnit; ++i) word[i] = reinterpret_cast<const uint32_t*>(p)[i];
        } else {
#pragma unroll
            for (uint32_t i = 0; i < kUnit / 2; ++i) word[i] = reinterpret_cast<const uint16_t*>(p)[2 * i] | static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[2 * i + 1]) << 16;
        }
    }
    __device__ __forceinline__ float operator[](uint32_t j) const {
        T v;
        if constexpr (sizeof(T) == 4) {
            v = __uint_as_float(word[j]);
        } else {
            const uint16_t h = static_cast<uint16_t>(j % 2 != 0 ? word[j / 2] >> 16 : word[j / 2] & 0xFFFFu);
            __builtin_memcpy(&v, &h, 2);
        }
        return to_f32(v);
    }
};
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
}
__device__ __forceinline__ float code(uint32_t byte) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte), __NV_E4M3)));
}

template <class T, uint32_t UNITS>
__global__ void __launch_bounds__(512) kv_write_kernel(const WriteCall c) {
    __shared__ float warp_max[16];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const Cache& kv = c.cache;
    const uint32_t seq = blockIdx.z, head = blockIdx.y >> 1;
    const bool is_v = blockIdx.y & 1;
    const Seq s = sequence(c.rows, kv, seq);
    const int32_t first = s.length - static_cast<int32_t>(s.count);  // position of the first row
    if (s.count == 0 || s.length <= 0) return;
    const uint32_t index = (static_cast<uint32_t>(max(first, 0)) >> kv.page_shift) + blockIdx.x;
    const int32_t page0 = static_cast<int32_t>(index << kv.page_shift);  // position of the page's slot 0
    if (page0 >= s.length) return;
    const int32_t page = page_of(kv, seq, index);
    if (static_cast<uint32_t>(page) >= kv.n_pages) {
        if (threadIdx.x == 0 && c.status != nullptr) atomicOr(c.status, 8u);  // kStatusBadIndex
        return;
    }
    const uint32_t slot0 = static_cast<uint32_t>(max(first, page0) - page0);
    const uint32_t slot1 = static_cast<uint32_t>(min(s.length - page0, static_cast<int32_t>(kv.page_tokens)));
    const uint32_t row_units = kv.head_dim / kUnit, units = (slot1 - slot0) * row_units;
    const Heads& in = is_v ? c.v : c.k;
    const uint8_t* src = in.p + (s.row0 + static_cast<uint32_t>(page0 + static_cast<int32_t>(slot0) - first)) * in.token_stride + head * in.head_stride;
    uint8_t* dst = (is_v ? kv.v : kv.k) + page * kv.page_stride + uint64_t{head} * kv.page_tokens * kv.head_dim;
    uint8_t* scale = (is_v ? kv.v_scale : kv.k_scale) + page * kv.scale_stride + head;

    Raw<T> x[UNITS];
    float top = 0;
#pragma unroll
    for (uint32_t i = 0; i < UNITS; ++i) {
        const uint32_t u = threadIdx.x + i * blockDim.x;
        if (u >= units) break;
        const uint32_t row = u / row_units, at = u - row * row_units;
        x[i].load(src + row * in.token_stride + at * kUnit * sizeof(T), in.vec != 0);
    }
#pragma unroll
    for (uint32_t i = 0; i < UNITS; ++i) {
        if (threadIdx.x + i * blockDim.x >= units) break;
#pragma unroll
        for (uint32_t j = 0; j < kUnit; ++j) {
            const float m = fabsf(x[i][j]);
            top = fmaxf(top, m < INFINITY ? m : 0.0f);  // neither infinities nor NaN
        }
    }
#pragma unroll
    for (uint32_t d = 16; d != 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
    if (threadIdx.x % 32 == 0) warp_max[threadIdx.x / 32] = top;
    const int32_t old = scale_byte(*scale);
    __syncthreads();
    top = warp_max[0];
    for (uint32_t w = 1; w < blockDim.x / 32; ++w) top = fmaxf(top, warp_max[w]);
    // top = m * 2^e with 1 <= m < 2; it fits 448 = 1.75 * 2^8 under 2^(e - 8) where m <= 1.75, else under 2^(e - 7)
    const uint32_t bits = __float_as_uint(top);
    int32_t b = static_cast<int32_t>(bits >> 23) - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    b = scale_byte(static_cast<uint32_t>(max(b, 0)));
    if (slot0 != 0 && old >= b) b = old;
    if (threadIdx.x == 0) *scale = static_cast<uint8_t>(b);
    const float inv = exp2_int(127 - b);
#pragma unroll
    for (uint32_t i = 0; i < UNITS; ++i) {
        const uint32_t u = threadIdx.x + i * blockDim.x;
        if (u >= units) break;
        uint4 w;
        uint32_t* p = &w.x;
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) p[j] = codes4(x[i][4 * j] * inv, x[i][4 * j + 1] * inv, x[i][4 * j + 2] * inv, x[i][4 * j + 3] * inv);
        reinterpret_cast<uint4*>(dst + uint64_t{slot0} * kv.head_dim)[u] = w;
    }
    if (slot0 == 0 || old >= b) return;
    const float shrink = exp2_int(old - b);  // old - b >= -120
    for (uint32_t u = threadIdx.x; u < slot0 * row_units; u += blockDim.x) {
        uint4 w = reinterpret_cast<const uint4*>(dst)[u];
        uint32_t* p = &w.x;
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j)
            p[j] = codes4(code(p[j] & 255u) * shrink, code(p[j] >> 8 & 255u) * shrink, code(p[j] >> 16 & 255u) * shrink, code(p[j] >> 24) * shrink);
        reinterpret_cast<uint4*>(dst)[u] = w;
    }
}

template <class T, uint32_t UNITS>
int launch(const WriteCall& c, uint32_t threads, cudaStream_t s) {
    const uint32_t touched = (c.rows.max_tokens + c.cache.page_tokens - 2) / c.cache.page_tokens + 1;  // pages that max_tokens rows reach at most
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(std::min(touched, c.cache.max_pages), c.cache.n_kv * 2, c.cache.n_seq);
    cfg.blockDim = dim3(threads);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    HC_CUDA(cudaLaunchKernelEx(&cfg, kv_write_kernel<T, UNITS>, c));
    return 0;
}

}  // namespace

int launch_kv_write(HaloCudaCtx*, const WriteCall& c, cudaStream_t s) {
    if (c.cache.n_seq > 65535u || c.cache.n_kv > 32767u) return fail(HALO_CUDA_E_UNSUPPORTED, "KV_WRITE: %u sequences, %u kv heads", c.cache.n_seq, c.cache.n_kv);
    return with_type(c.type, [&](auto t) {
        using T = decltype(t);
        // A page's rows at most, or all that a sequence brings: up to four units a thread (five prompts in pages of 512 units: blocks of 512 threads 29.4 us, of
        // 256 22.8, of 128 22.2, back to back on the same rows), and blocks of 512 threads where 128 would not do.
        const uint32_t units = std::min(c.cache.page_tokens, c.rows.max_tokens) * (c.cache.head_dim / kUnit);  // <= 2048
        const uint32_t threads = std::min((units + 31u) / 32u * 32u, units > 512u ? 512u : 128u);
        const uint32_t per = (units + threads - 1) / threads;
        if (per <= 1) return launch<T, 1>(c, threads, s);
        return per <= 2 ? launch<T, 2>(c, threads, s) : launch<T, 4>(c, threads, s);
    });
}

}  // namespace attn
}  // namespace halo_cuda
