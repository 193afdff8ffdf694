// PARTIAL_ROPE: y = magnitude * R(position * f_j) x for every pair j of the first 2 * n_pairs elements of every head.
//
// The phase is kept in units of 2^-64 of a turn: position * turns[j] modulo 2^64 drops whole turns without rounding, so the phase of position
// 2^31 is as exact as that of position 1 (an fp32 product would be off by a tenth of a radian at a million).  Its leading 32 bits go through
// sincospif, whose argument is then in [-1, 1).
//
// What bounds it: HBM, 2 * size bytes an element.  A block takes a few tokens and a share of their heads: it computes the tokens' cosines and
// sines once into shared memory, then every thread has four units in flight, a unit being the 16-byte vectors of both halves of 16 / size
// pairs (one vector where pairs are adjacent), or a vector to copy.
#include "rope.h"

namespace halo_cuda {
namespace attn {
namespace {

constexpr uint32_t kThreads = 256, kUnroll = 4, kMaxTokens = 4;

struct RopeArgs {
    const int32_t* positions;
    Heads q, k, q_out, k_out;
    uint32_t n_tokens, n_q, heads, dim;     // heads: n_q + n_kv
    uint32_t tokens_per_block, heads_per_block;
    uint32_t pairs, turn_units, units;      // units of a row: those that turn, then those that copy
    uint32_t q_copies, k_copies;            // out of place: elements behind the pairs are copied
    float magnitude;
    uint64_t turns[HALO_CUDA_ROPE_MAX_PAIRS];
};

template <class T, int N>
struct alignas(sizeof(T) * N) Vec {
    T v[N];
};

/// V: elements of an access, 16 bytes or (misaligned operands, odd numbers of pairs) one.  A turning unit is V pairs of the half layout, V / 2 adjacent
/// pairs, or one pair.
template <class T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads) rope_kernel(const __grid_constant__ RopeArgs a) {
    __shared__ float2 spin[kMaxTokens * HALO_CUDA_ROPE_MAX_PAIRS];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const uint32_t t0 = blockIdx.x * a.tokens_per_block, nt = min(a.tokens_per_block, a.n_tokens - t0);
    const uint32_t h0 = blockIdx.y * a.heads_per_block, nh = min(a.heads_per_block, a.heads - h0);
    for (uint32_t i = threadIdx.x; i < nt * a.pairs; i += kThreads) {
        const uint32_t t = i / a.pairs, j = i - t * a.pairs;
        const uint64_t phase = static_cast<uint64_t>(static_cast<int64_t>(__ldg(a.positions + t0 + t))) * a.turns[j];
        float s, c;
        sincospif(static_cast<float>(static_cast<int32_t>(phase >> 32)) * 0x1p-31f, &s, &c);
        spin[i] = make_float2(c * a.magnitude, s * a.magnitude);
    }
    __syncthreads();
    using Word = Vec<T, V>;
    const uint32_t total = nt * nh * a.units;
    for (uint32_t base = threadIdx.x; base < total; base += kThreads * kUnroll) {
        Word x[kUnroll], z[kUnroll];
        Word *px[kUnroll], *pz[kUnroll];  // where the results go
        uint32_t pair[kUnroll];           // index of the unit's first pair in `spin`; ~0: copy; ~1: nothing
#pragma unroll
        for (uint32_t r = 0; r < kUnroll; ++r) {
            const uint32_t i = base + r * kThreads;
            pair[r] = ~1u;
            if (i >= total) continue;
            const uint32_t row = i / a.units, u = i - row * a.units, t = row / nh, h = h0 + row - t * nh;
            const bool is_q = h < a.n_q;
            const Heads &in = is_q ? a.q : a.k, &out = is_q ? a.q_out : a.k_out;
            const uint32_t hh = is_q ? h : h - a.n_q;
            const uint8_t* src = in.p + uint64_t{t0 + t} * in.token_stride + uint64_t{hh} * in.head_stride;
            uint8_t* dst = out.p + uint64_t{t0 + t} * out.token_stride + uint64_t{hh} * out.head_stride;
            if (u < a.turn_units) {
                constexpr uint32_t kPairs = INTERLEAVED ? (V > 1 ? V / 2 : 1) : V;
                const uint32_t first = INTERLEAVED ? u * 2 * kPairs : u * V, second = INTERLEAVED ? first + 1 : first + a.pairs;
                pair[r] = t * a.pairs + u * kPairs;
                x[r] = *reinterpret_cast<const Word*>(src + first * sizeof(T));
                px[r] = reinterpret_cast<Word*>(dst + first * sizeof(T));
                if (!INTERLEAVED || V == 1) {
                    z[r] = *reinterpret_cast<const Word*>(src + second * sizeof(T));
                    pz[r] = reinterpret_cast<Word*>(dst + second * sizeof(T));
                }
            } else if (is_q ? a.q_copies : a.k_copies) {
                const uint32_t at = 2 * a.pairs + (u - a.turn_units) * V;
                pair[r] = ~0u;
                x[r] = *reinterpret_cast<const Word*>(src + at * sizeof(T));
                px[r] = reinterpret_cast<Word*>(dst + at * sizeof(T));
            }
        }
#pragma unroll
        for (uint32_t r = 0; r < kUnroll; ++r) {
            if (pair[r] == ~1u) continue;
            if (pair[r] == ~0u) {
                *px[r] = x[r];
                continue;
            }
            if constexpr (INTERLEAVED && V > 1) {
#pragma unroll
                for (int j = 0; j < V / 2; ++j) {
                    const float2 cs = spin[pair[r] + j];
                    const float p = to_f32(x[r].v[2 * j]), q = to_f32(x[r].v[2 * j + 1]);
                    x[r].v[2 * j] = from_f32<T>(p * cs.x - q * cs.y);
                    x[r].v[2 * j + 1] = from_f32<T>(q * cs.x + p * cs.y);
                }
                *px[r] = x[r];
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float2 cs = spin[pair[r] + j];
                    const float p = to_f32(x[r].v[j]), q = to_f32(z[r].v[j]);
                    x[r].v[j] = from_f32<T>(p * cs.x - q * cs.y);
                    z[r].v[j] = from_f32<T>(q * cs.x + p * cs.y);
                }
                *px[r] = x[r];
                *pz[r] = z[r];
            }
        }
    }
}

template <class T, int V, bool INTERLEAVED>
int launch(RopeArgs a, cudaStream_t s) {
    const bool copies = a.q_copies || a.k_copies;
    a.turn_units = INTERLEAVED ? a.pairs * 2 / (V > 1 ? V : 2) : a.pairs / V;
    a.units = a.turn_units + (copies ? (a.dim - 2 * a.pairs) / V : 0);
    // One pass of the loop a block where there is enough for it: first whole tokens, then shares of one token's heads.
    const uint32_t room = kThreads * kUnroll, per_token = a.heads * a.units;
    a.tokens_per_block = per_token == 0 ? 1 : std::min(std::max(room / per_token, 1u), kMaxTokens);
    a.heads_per_block = a.tokens_per_block > 1 ? a.heads : std::min(a.heads, std::max(room / a.units, 1u));
    const uint32_t shares = (a.heads + a.heads_per_block - 1) / a.heads_per_block;  // <= 131070
    a.heads_per_block = (a.heads + shares - 1) / shares;
    if (shares > 65535u) a.heads_per_block = (a.heads + 65534u) / 65535u;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((a.n_tokens + a.tokens_per_block - 1) / a.tokens_per_block, (a.heads + a.heads_per_block - 1) / a.heads_per_block);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    HC_CUDA(cudaLaunchKernelEx(&cfg, rope_kernel<T, V, INTERLEAVED>, a));
    return 0;
}

}  // namespace

int launch_rope(const RopeCall& c, cudaStream_t s) {
    RopeArgs a{};
    a.positions = c.positions;
    a.q = c.q, a.k = c.k, a.q_out = c.q_out, a.k_out = c.k_out;
    a.n_tokens = c.n_tokens, a.n_q = c.n_q, a.heads = c.n_q + c.n_kv, a.dim = c.head_dim;
    a.pairs = c.freqs->n_pairs;
    a.magnitude = c.freqs->magnitude;
    for (uint32_t j = 0; j < a.pairs; ++j) a.turns[j] = c.freqs->turns[j];
    const bool rest = c.head_dim > 2 * a.pairs;
    a.q_copies = rest && c.n_q != 0 && c.q.p != c.q_out.p;
    a.k_copies = rest && c.n_kv != 0 && c.k.p != c.k_out.p;
    return with_type(c.type, [&](auto t) {
        using T = decltype(t);
        constexpr uint32_t V = 16 / sizeof(T);
        auto vec = [&](const Heads& h, uint32_t n) { return n == 0 || h.vec != 0; };
        const bool wide = vec(c.q, c.n_q) && vec(c.q_out, c.n_q) && vec(c.k, c.n_kv) && vec(c.k_out, c.n_kv) && c.head_dim % V == 0 &&
                          (c.interleaved ? 2 * a.pairs : a.pairs) % V == 0;
        if (c.interleaved) return wide ? launch<T, V, true>(a, s) : launch<T, 1, true>(a, s);
        return wide ? launch<T, V, false>(a, s) : launch<T, 1, false>(a, s);
    });
}

}  // namespace attn
}  // namespace halo_cuda
