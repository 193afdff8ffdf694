// PARTIAL_ROPE: y = magnitude * R(position * f_j) x for every pair j of the first 2 * n_pairs elements of every head.
//
// The phase is kept in units of 2^-64 of a turn: position * turns[j] modulo 2^64 drops whole turns without rounding, so the phase of position
// 2^31 is as exact as that of position 1 (an fp32 product would be off by a tenth of a radian at a million).  Its leading 32 bits go through
// sincospif, whose argument is then in [-1, 1).
//
// What bounds it: HBM, 2 * size bytes an element (8192 tokens of 40 heads of 128 in bf16, 168 MB, 33.4 us, 5.0 TB/s); for few tokens the launch.  A block takes a few tokens and a share of their heads: it computes the tokens' cosines and
// sines into shared memory while its first loads are under way; a thread has two units in flight, a unit being the 16-byte vectors of both halves of 16 / size
// pairs (one vector where pairs are adjacent), or a vector to copy.
#include "rope.h"

namespace halo_cuda {
namespace attn {
namespace {

constexpr uint32_t kThreads = 256, kUnroll = 2, kMaxTokens = 4;

struct RopeArgs {
    const int32_t* positions;
    Heads q, k, q_out, k_out;
    uint32_t n_tokens, n_q, heads, dim;     // heads: n_q + n_kv
    uint32_t tokens_per_block, heads_per_block;  // (of a warp, in rope_warp_kernel)
    uint32_t shares;                             // of a token's heads, in rope_warp_kernel
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
__global__ void __launch_bounds__(kThreads, 4) rope_kernel(const __grid_constant__ RopeArgs a) {
    constexpr int kPairs = INTERLEAVED ? (V > 1 ? V / 2 : 1) : V;  // of a unit
    using Factors = Vec<float, kPairs>;
    __shared__ alignas(16) float cosine[kMaxTokens * HALO_CUDA_ROPE_MAX_PAIRS], sine[kMaxTokens * HALO_CUDA_ROPE_MAX_PAIRS];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const uint32_t t0 = blockIdx.x * a.tokens_per_block, nt = min(a.tokens_per_block, a.n_tokens - t0);
    const uint32_t h0 = blockIdx.y * a.heads_per_block, nh = min(a.heads_per_block, a.heads - h0);
    using Word = Vec<T, V>;
    const uint32_t total = nt * nh * a.units;
    for (uint32_t base = threadIdx.x, turn = 0; turn == 0 || base - threadIdx.x < total; base += kThreads * kUnroll, ++turn) {
        Word x[kUnroll], z[kUnroll];
        Word *px[kUnroll], *pz[kUnroll];  // where the results go
        uint32_t pair[kUnroll];           // index of the unit's first pair in the factors; ~0: copy; ~1: nothing
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
        if (turn == 0) {  // behind the first loads, which are under way meanwhile
            for (uint32_t i = threadIdx.x; i < nt * a.pairs; i += kThreads) {
                const uint32_t t = i / a.pairs, j = i - t * a.pairs;
                const uint64_t phase = static_cast<uint64_t>(static_cast<int64_t>(attn::load(a.positions + t0 + t))) * a.turns[j];
                float s, c;
                sincospif(static_cast<float>(static_cast<int32_t>(phase >> 32)) * 0x1p-31f, &s, &c);
                cosine[i] = c * a.magnitude, sine[i] = s * a.magnitude;
            }
            __syncthreads();
        }
#pragma unroll
        for (uint32_t r = 0; r < kUnroll; ++r) {
            if (pair[r] == ~1u) continue;
            if (pair[r] == ~0u) {
                *px[r] = x[r];
                continue;
            }
            const Factors c = *reinterpret_cast<const Factors*>(cosine + pair[r]), s = *reinterpret_cast<const Factors*>(sine + pair[r]);
            if constexpr (INTERLEAVED && V > 1) {
#pragma unroll
                for (int j = 0; j < kPairs; ++j) {
                    const float p = to_f32(x[r].v[2 * j]), q = to_f32(x[r].v[2 * j + 1]);
                    x[r].v[2 * j] = from_f32<T>(p * c.v[j] - q * s.v[j]);
                    x[r].v[2 * j + 1] = from_f32<T>(q * c.v[j] + p * s.v[j]);
                }
                *px[r] = x[r];
            } else {
#pragma unroll
                for (int j = 0; j < kPairs; ++j) {
                    const float p = to_f32(x[r].v[j]), q = to_f32(z[r].v[j]);
                    x[r].v[j] = from_f32<T>(p * c.v[j] - q * s.v[j]);
                    z[r].v[j] = from_f32<T>(q * c.v[j] + p * s.v[j]);
                }
                *px[r] = x[r];
                *pz[r] = z[r];
            }
        }
    }
}

/// Wide operands whose heads have a power of two of turning units, at most 32: a warp for a share of one token's heads, a lane for one unit of every
/// 32 / units-th of them, so that its factors stay in registers.  Lanes that share a unit share out its sines and cosines; nothing is waited for but loads.
template <class T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads, 4) rope_warp_kernel(const __grid_constant__ RopeArgs a) {
    constexpr int kPairs = INTERLEAVED ? V / 2 : V;
    using Word = Vec<T, V>;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const uint32_t lane = threadIdx.x % 32, item = blockIdx.x * (kThreads / 32) + threadIdx.x / 32;
    const uint32_t t = item / a.shares, share = item - t * a.shares;
    if (t >= a.n_tokens) return;
    const uint32_t h0 = share * a.heads_per_block, h1 = min(h0 + a.heads_per_block, a.heads);
    const uint32_t units = a.turn_units, u = lane & (units - 1), sub = lane / units, step = 32 / units;
    auto row = [&](uint32_t h, bool to) {
        const bool is_q = h < a.n_q;
        const Heads& x = to ? (is_q ? a.q_out : a.k_out) : (is_q ? a.q : a.k);
        return x.p + uint64_t{t} * x.token_stride + uint64_t{is_q ? h : h - a.n_q} * x.head_stride;
    };
    const uint32_t first = INTERLEAVED ? u * 2 * kPairs : u * V, second = first + a.pairs;
    Word x, z;
    auto load = [&](uint32_t h, Word& x, Word& z) {
        if (h >= h1) return;
        const uint8_t* src = row(h, false);
        x = *reinterpret_cast<const Word*>(src + first * sizeof(T));
        if constexpr (!INTERLEAVED) z = *reinterpret_cast<const Word*>(src + second * sizeof(T));
    };
    load(h0 + sub, x, z);
    const uint64_t position = static_cast<uint64_t>(static_cast<int64_t>(attn::load(a.positions + t)));
    float c[kPairs], s[kPairs];
    // pair p of the unit is made by the unit's lane p % step
#pragma unroll
    for (int m = 0; m < kPairs; ++m) {
        if (m * step >= kPairs) break;
        const uint64_t phase = position * a.turns[u * kPairs + min(sub + m * step, static_cast<uint32_t>(kPairs - 1))];
        sincospif(static_cast<float>(static_cast<int32_t>(phase >> 32)) * 0x1p-31f, &s[m], &c[m]);
    }
    float cosine[kPairs], sine[kPairs];
#pragma unroll
    for (uint32_t p = 0; p < kPairs; ++p) {
        const uint32_t from = u + units * (p & (step - 1)), m = p / step;
        float cm = c[0], sm = s[0];
#pragma unroll
        for (uint32_t k = 1; k < kPairs; ++k)
            if (m == k) cm = c[k], sm = s[k];
        cosine[p] = __shfl_sync(0xFFFFFFFFu, cm, from) * a.magnitude;
        sine[p] = __shfl_sync(0xFFFFFFFFu, sm, from) * a.magnitude;
    }
    // the next head under way while one is turned (two heads at a time, each pair waited for: 39 us for 8192 tokens of 40 heads of 128 in bf16, so 34)
    for (uint32_t h = h0 + sub; h < h1; h += step) {
        Word next_x, next_z;
        load(h + step, next_x, next_z);
        uint8_t* dst = row(h, true);
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
            T &e0 = x.v[INTERLEAVED ? 2 * j : j], &e1 = INTERLEAVED ? x.v[2 * j + 1] : z.v[j];
            const float p = to_f32(e0), q = to_f32(e1);
            e0 = from_f32<T>(p * cosine[j] - q * sine[j]);
            e1 = from_f32<T>(q * cosine[j] + p * sine[j]);
        }
        *reinterpret_cast<Word*>(dst + first * sizeof(T)) = x;
        if constexpr (!INTERLEAVED) *reinterpret_cast<Word*>(dst + second * sizeof(T)) = z;
        x = next_x;
        if constexpr (!INTERLEAVED) z = next_z;
    }
    const uint32_t copies = a.units - a.turn_units;
    for (uint32_t i = lane; i < (h1 - h0) * copies; i += 32) {
        const uint32_t h = h0 + i / copies, at = 2 * a.pairs + i % copies * V;
        if (h < a.n_q ? a.q_copies : a.k_copies) *reinterpret_cast<Word*>(row(h, true) + at * sizeof(T)) = *reinterpret_cast<const Word*>(row(h, false) + at * sizeof(T));
    }
}

template <class T, int V, bool INTERLEAVED>
int launch(RopeArgs a, cudaStream_t s) {
    const bool copies = a.q_copies || a.k_copies;
    a.turn_units = INTERLEAVED ? a.pairs * 2 / (V > 1 ? V : 2) : a.pairs / V;
    a.units = a.turn_units + (copies ? (a.dim - 2 * a.pairs) / V : 0);
    cudaLaunchConfig_t cfg{};
    cfg.blockDim = dim3(kThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if constexpr (V > 1) {
        if (a.turn_units <= 32 && (a.turn_units & (a.turn_units - 1)) == 0) {
            // A token's heads to one warp, for its factors' sake, unless that leaves the device without warps; at least one step of heads each.
            constexpr uint32_t kWarps = 148 * 16;
            const uint32_t step = 32 / a.turn_units, most = (a.heads + step - 1) / step;
            a.shares = std::min(most, (kWarps + a.n_tokens - 1) / a.n_tokens);
            a.heads_per_block = (a.heads + a.shares - 1) / a.shares;
            a.shares = (a.heads + a.heads_per_block - 1) / a.heads_per_block;
            const uint64_t blocks = (uint64_t{a.n_tokens} * a.shares + kThreads / 32 - 1) / (kThreads / 32);
            if (uint64_t{a.n_tokens} * a.shares <= 0x7FFFFFFFu) {
                cfg.gridDim = dim3(static_cast<uint32_t>(blocks));
                HC_CUDA(cudaLaunchKernelEx(&cfg, rope_warp_kernel<T, V, INTERLEAVED>, a));
                return 0;
            }
        }
    }
    // One pass of the loop a block where there is enough for it: first whole tokens, then shares of one token's heads.
    const uint32_t room = kThreads * kUnroll, per_token = a.heads * a.units;
    a.tokens_per_block = per_token == 0 ? 1 : std::min(std::max(room / per_token, 1u), kMaxTokens);
    a.heads_per_block = a.tokens_per_block > 1 ? a.heads : std::min(a.heads, std::max(room / a.units, 1u));
    const uint32_t shares = (a.heads + a.heads_per_block - 1) / a.heads_per_block;  // <= 131070
    a.heads_per_block = (a.heads + shares - 1) / shares;
    if (shares > 65535u) a.heads_per_block = (a.heads + 65534u) / 65535u;
    cfg.gridDim = dim3((a.n_tokens + a.tokens_per_block - 1) / a.tokens_per_block, (a.heads + a.heads_per_block - 1) / a.heads_per_block);
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
