// ATTENTION for few rows to a sequence (decoded tokens, drafts): warp-level fp16 tensor-core products over the cache's codes, converted in registers.
//
//   x_t = q . k_t * (s_K(t) * scale * log2 e) + log2 s_V(t),   m = max x_t,   p_t = 2^(x_t - m + 14)
//   o = sum p_t code(v_t),   l = sum p_t / s_V(t),   out = o / l
//
// The scale of a value's page rides in its token's exponent, so that o needs no rescaling between pages and p_t, at most 2^14, is an fp16 number with
// 11 bits down to 2^-28 of the largest.  e4m3 codes are exact in fp16.  A row of q is multiplied by the power of two that puts its largest magnitude
// into [2^14, 2^15) and rounded to fp16: exact for fp16 and bf16 operands (but for elements below 2^-28 of the row's largest);
// fp32 operands are taken as two fp16 terms, and so are their p_t.  Accumulators, maxima and sums are fp32.
//
// A CTA has 16 packed rows (attention_work.cuh).  Its warps share the keys of a tile, each with a running maximum, sum and accumulators of its own
// that are joined at the end of a segment, so no warp waits for another inside the walk.  Heads of 256 elements would take 128 registers of accumulators a
// thread: there two warps share the same keys, each makes half of the scores and all of the weights, and has half of the dims.  A producer warp
// brings the tiles' codes by TMA, a box for each page, into a ring, and with them the scales of every 16 tokens (a page is at least 16).
//
// What bounds it: HBM while the walk lasts where a sequence is long (131071 tokens of 8 heads of 128 in bf16, 268 MB, take 64 us, 4.2 TB/s; four times the
// tokens take 193, so that the further ones come at 6.3 TB/s and 20 us are fixed: the launch 8, search, first tile, joins).  Many sequences of all lengths come at
// 5.0 TB/s (48 of 156 - 7697, pages of 16, 200 MB in 56 us; twice and four times as many 95 and 193): the ends of units.  A byte of the cache costs a warp
// half a conversion, and a sixteenth of a 16 x 8 x 16 product for 16 rows.  Heads of 256 with fp32 operands, four products for one, are bound by the dependent
// steps of eight warps an SM (a third of the issue slots used): 12 sequences of 2156 - 4688 with 24 rows each 68 us, further ones at 1.7 TB/s.
#pragma once
#include <cuda.h>

#include "attention_work.cuh"

namespace halo_cuda {
namespace attn {

struct GroupScale {
    float k, log_v, inv_v;  // s_K * scale * log2 e; log2 s_V, -inf for tokens of no page; 1 / s_V
    uint32_t gap;           // a visible key of the tile has no page (the prompts kernel)
};

/// TS: warps, or pairs of them, that share a tile's keys.  TILE: keys of a tile.  CPS: CTAs that share an SM.
template <int D, int TS, int TILE, int CPS, int TERMS>
struct RowsShape {
    static constexpr uint32_t kTile = TILE, kGroups = TILE / 16;  // groups of 16 tokens, each inside one page
    static_assert(TILE % 64 == 0 && TILE % (16 * TS) == 0 && kGroups <= 32);
    static constexpr int kSplit = D == 256 ? 2 : 1;               // warps that share the dims of the same keys
    static constexpr int kWarps = TS * kSplit, kThreads = (kWarps + 1) * 32, kRows = 16;
    static constexpr uint32_t kHalfTile = kTile * D;  // K or V of a tile
    static constexpr uint32_t kStage = 2 * kHalfTile;
    static constexpr uint32_t kQ = (D / 16) * TERMS * 512;
    static constexpr uint32_t kJoinRow = D + D / 8 + (D == 256 ? 16 : 0);  // floats of a row of the warps' joined rows
    static constexpr uint32_t kJoin = 16 * kJoinRow * 4;
    static constexpr uint32_t kFixed = 1024 + kQ + kJoin;  // alignment, q, the warps' joined rows
    // an SM's 228 KiB, less 1 KiB a CTA for the system and what is declared in the kernel (up to 8 KiB with pairs of warps, else 3)
    static constexpr uint32_t kStagesRoom = (228 / CPS * 1024 - (kSplit == 2 ? 9216 : 4096) - kFixed) / kStage;
    static constexpr int kStages = kStagesRoom > 6 ? 6 : kStagesRoom;
    static constexpr uint32_t kSmem = kFixed + kStages * kStage;
    static_assert(kStages >= 2);
    // The tensor cores cut a sum off where they add a product to it, always towards zero, by up to an ulp (fp32 operands, a chain of 8192 products: 4e-4 too
    // small).  After so many tiles a thread's rows and sums are added up in fp32 outside: 64 products of 16 keys for fp32 operands (262144 positions: 1.5e-6
    // off), 512 for 16-bit ones (2^-15 in the mean, a sixteenth of fp16's half step).  A chain begun anew with every tile and added up in registers cost
    // more: 32 sequences of 3000 - 9000 tokens, 24 rows of 256, fp32: 109 us with no settling, 115 so, 129.
    static constexpr int32_t kSettle = (TERMS == 2 ? 64 : 512) / (TERMS * (TILE / TS / 16));
    static constexpr uint32_t kPieces = D / 8 / kSplit;  // float4 of a thread's part of the rows
    static constexpr uint64_t kSettledBytes = uint64_t{kWarps} * 32 * (kPieces + 1) * 16;
};

__device__ __forceinline__ uint32_t swizzled(uint32_t row, uint32_t chunk, int dim) {  // of a tile's half: 128-byte rows, or 64-byte rows of 64 elements
    return dim == 64 ? row * 64 + ((chunk ^ (row >> 1 & 3)) << 4) : row * 128 + ((chunk ^ (row & 7)) << 4);
}
__device__ __forceinline__ uint4 lds128(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t at) {
    uint2 v;
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at));
    return v;
}
/// Two codes -> two fp16.
__device__ __forceinline__ uint32_t widen(uint16_t codes) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(codes));
    return h;
}
__device__ __forceinline__ uint32_t widen_lo(uint32_t w) { return widen(static_cast<uint16_t>(w & 0xFFFFu)); }
__device__ __forceinline__ uint32_t widen_hi(uint32_t w) { return widen(static_cast<uint16_t>(w >> 16)); }
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
/// What two-term rounding leaves behind the first term.
__device__ __forceinline__ uint32_t half2_rest(float a, float b, uint32_t first) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&first));
    return half2_bits(a - f.x, b - f.y);
}
/// Bit 7 of every byte of four that is a NaN code, 0x7F or 0xFF.
__device__ __forceinline__ uint32_t nan_bits(uint32_t w) { return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u; }
/// Zeroes the NaN codes of four, or with `keep` of all ones leaves them; true if there were any.
__device__ __forceinline__ bool drop_nan(uint32_t& w, uint32_t keep = 0) {
    const uint32_t hit = nan_bits(w);
    if (hit == 0) return false;
    w &= ~((hit >> 7) * 255u) | keep;
    return true;
}

/// Writes NaN over the results of rows that see a token whose value is NaN there: the walk left those codes out in tiles that some rows do not see
/// whole, since a product with weight zero would have spread them to these.  Only those tiles are looked at, a handful at the edges of what a unit's rows see (every
/// token of 60000, one after the other, took 300 to 9000 us).  Called by whole warps that share the segment's codes of dims [first_dim, first_dim + dims), 16
/// bytes to a thread at a time; `at(row, d)` is the result's address.
template <class At>
__device__ void spread_nan(const AttentionCall& c, const Work& w, const Unit& u, const Segment& g, uint32_t first_row, uint32_t end_row, uint32_t first_dim, uint32_t dims,
                           uint32_t thread, uint32_t threads, At&& at) {
    const uint32_t r0 = u.row0(w), lane = threadIdx.x % 32, chunks = dims / 16;
    const int32_t tile_keys = static_cast<int32_t>(w.tile), page_tokens = static_cast<int32_t>(c.cache.page_tokens);
    const int32_t all_lo = first_key(u.s, w.window, (r0 + u.rows(w) - 1) / c.group), all_hi = end_key(u.s, c.causal, r0 / c.group);
    for (int32_t base = g.lo; base < g.hi; base += 32) {
        const int32_t tile = base + static_cast<int32_t>(lane), t = tile * tile_keys;
        const bool look = tile < g.hi && (t < all_lo || t + tile_keys > all_hi);
        for (uint32_t left = __ballot_sync(0xFFFFFFFFu, look); left != 0; left &= left - 1) {
            const int32_t first = (base + __ffs(left) - 1) * tile_keys;
            for (int32_t t0 = first; t0 < min(first + tile_keys, u.s.length); t0 += 16) {
                const int32_t page = page_of(c.cache, u.seq, t0 >> c.cache.page_shift);
                if (static_cast<uint32_t>(page) >= c.cache.n_pages) continue;
                const uint8_t* v = c.cache.v + page * c.cache.page_stride + (uint64_t{u.head} * c.cache.page_tokens + (t0 & (page_tokens - 1))) * c.cache.head_dim + first_dim;
                for (uint32_t i = thread; i < dims; i += threads) {  // 16 tokens of `chunks` pieces each
                    const int32_t key = t0 + static_cast<int32_t>(i / chunks);
                    const uint4 codes = *reinterpret_cast<const uint4*>(v + i / chunks * c.cache.head_dim + i % chunks * 16);
                    if (key >= u.s.length) continue;
#pragma unroll
                    for (uint32_t n = 0; n < 4; ++n) {
                        for (uint32_t hit = nan_bits(n == 0 ? codes.x : n == 1 ? codes.y : n == 2 ? codes.z : codes.w); hit != 0; hit &= hit - 1) {
                            const uint32_t d = first_dim + i % chunks * 16 + n * 4 + (__ffs(hit) - 1) / 8;
                            for (uint32_t r = first_row; r < end_row; ++r) {
                                const uint32_t j = (r0 + r) / c.group;
                                if (key >= first_key(u.s, w.window, j) && key < end_key(u.s, c.causal, j)) at(r, d);
                            }
                        }
                    }
                }
            }
        }
    }
}

template <class T, int D, int SHARES, int AHEAD, class Slot, class Weight, class Add, class Put>
__device__ __forceinline__ void join_few(uint32_t pieces, uint32_t thread, uint32_t threads, const Work& w, Slot& slot, Weight& weight, Add& add, Put& put, const float2* row_ml) {
#pragma unroll 1
    for (uint32_t i = thread; i < pieces; i += AHEAD * threads) {
        float f[AHEAD][SHARES];
        float4 x[AHEAD][SHARES];
#pragma unroll
        for (uint32_t h = 0; h < AHEAD; ++h)
#pragma unroll
            for (uint32_t k = 0; k < SHARES; ++k) {
                const uint32_t at = min(i + h * threads, pieces - 1), r = at / (D / 4);
                f[h][k] = __ldcg(slot(k) + w.rows * D + 2 * r);
                x[h][k] = __ldcg(reinterpret_cast<const float4*>(slot(k) + at * 4));
            }
#pragma unroll
        for (uint32_t h = 0; h < AHEAD; ++h) {
            const uint32_t at = i + h * threads;
            if (at >= pieces) break;
            const uint32_t r = at / (D / 4);
            float4 o = make_float4(0, 0, 0, 0);
#pragma unroll
            for (uint32_t k = 0; k < SHARES; ++k) add(o, weight(k, f[h][k], row_ml[r].x), x[h][k]);
            put(r, at % (D / 4) * 4, o);
        }
    }
}

/// Joins the shares of a unit in CTA order and stores its rows.  All `warps` of the caller, from warp0 on, take part; `row_ml` has room for every row's
/// (maximum, 1 / sum).  FEW, AHEAD: up to FEW shares, loads of AHEAD pieces of a row are under way together (a caller whose walk has the registers to
/// spare: 4 pieces, 8 of up to two shares, for 7 prompts of 360 - 1570 tokens 10 us of 250).
template <class T, int D, int AHEAD>
__device__ __forceinline__ void join_partials(const AttentionCall& c, const Work& w, const Walk& walk, uint32_t c0, uint32_t shares, uint32_t warp0, uint32_t warps, float2* row_ml) {
    const uint32_t thread = threadIdx.x - warp0 * 32, threads = warps * 32, lane = thread % 32, rows = walk.rows;
    auto slot = [&](uint32_t k) { return partial_slot(w, D, c0 + min(k, shares - 1), k == 0); };
    // Without a maximum a share's sum and row are zero, or NaN: they count as they are.
    if (shares <= 4) {
#pragma unroll 1
        for (uint32_t r = thread; r < rows; r += threads) {
            float2 ml[4];
            float m = -INFINITY, l = 0;
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) ml[k] = __ldcg(reinterpret_cast<const float2*>(slot(k) + w.rows * D + 2 * r));
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) m = fmaxf(m, ml[k].x);
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k)
                if (k < shares) l += ml[k].x == -INFINITY ? ml[k].y : exp2_approx(ml[k].x - m) * ml[k].y;
            row_ml[r] = make_float2(m, l != 0 ? 1.0f / l : 0.0f);
        }
    } else {  // a warp to four rows, a lane to every 32nd share
#pragma unroll 1
        for (uint32_t r0 = thread / 32 * 4; r0 < rows; r0 += warps * 4) {
            float m[4], l[4] = {};
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) m[i] = -INFINITY;
#pragma unroll 1
            for (uint32_t k = lane; k < shares; k += 32) {
                float2 ml[4];
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) ml[i] = __ldcg(reinterpret_cast<const float2*>(slot(k) + w.rows * D + 2 * min(r0 + i, rows - 1)));
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    const float top = fmaxf(m[i], ml[i].x);
                    l[i] = (m[i] == -INFINITY ? l[i] : exp2_approx(m[i] - top) * l[i]) + (ml[i].x == -INFINITY ? ml[i].y : exp2_approx(ml[i].x - top) * ml[i].y);
                    m[i] = top;
                }
            }
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                float top = m[i];
#pragma unroll
                for (uint32_t d = 16; d != 0; d /= 2) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
                l[i] = m[i] == -INFINITY ? l[i] : exp2_approx(m[i] - top) * l[i];
#pragma unroll
                for (uint32_t d = 16; d != 0; d /= 2) l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], d);
                if (lane == 0 && r0 + i < rows) row_ml[r0 + i] = make_float2(top, l[i] != 0 ? 1.0f / l[i] : 0.0f);
            }
        }
    }
    bar_sync(1, threads);
    // a share of weight zero adds nothing, but a NaN in it is one of a token that the row sees; behind the last share: the last again, with weight zero
    auto weight = [&](uint32_t k, float of, float m) { return k >= shares ? 0.0f : of == -INFINITY ? 1.0f : exp2_approx(of - m); };
    auto add = [&](float4& o, float by, const float4& x) { o.x += by * x.x, o.y += by * x.y, o.z += by * x.z, o.w += by * x.w; };
    auto put = [&](uint32_t r, uint32_t d, const float4& o) {
        const float inv = row_ml[r].y;
        T* out = reinterpret_cast<T*>(walk.at(c, w, c.out, r)) + d;
        out[0] = from_f32<T>(o.x * inv), out[1] = from_f32<T>(o.y * inv), out[2] = from_f32<T>(o.z * inv), out[3] = from_f32<T>(o.w * inv);
    };
    const uint32_t pieces = rows * (D / 4);
    if (AHEAD > 2 && shares <= 2) join_few<T, D, 2, 2 * AHEAD>(pieces, thread, threads, w, slot, weight, add, put, row_ml);
    else if (shares <= 4) {
        join_few<T, D, 4, AHEAD>(pieces, thread, threads, w, slot, weight, add, put, row_ml);
    } else {  // of a piece's next ten shares
        constexpr uint32_t kAhead = 10;
#pragma unroll 1
        for (uint32_t i = thread; i < pieces; i += threads) {
            const uint32_t r = i / (D / 4);
            const float m = row_ml[r].x;
            float4 o = make_float4(0, 0, 0, 0);
#pragma unroll 1
            for (uint32_t k0 = 0; k0 < shares; k0 += kAhead) {
                float f[kAhead];
                float4 x[kAhead];
#pragma unroll
                for (uint32_t k = 0; k < kAhead; ++k) {
                    f[k] = __ldcg(slot(k0 + k) + w.rows * D + 2 * r);
                    x[k] = __ldcg(reinterpret_cast<const float4*>(slot(k0 + k) + i * 4));
                }
#pragma unroll
                for (uint32_t k = 0; k < kAhead; ++k) add(o, weight(k0 + k, f[k], m), x[k]);
            }
            put(r, i % (D / 4) * 4, o);
        }
    }
}

template <class T, int D, int TS, int TILE, int CPS>
__global__ void __launch_bounds__(RowsShape<D, TS, TILE, CPS, sizeof(T) == 4 ? 2 : 1>::kThreads, CPS)
    rows_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const __grid_constant__ AttentionCall c,
                const __grid_constant__ Work w) {
    constexpr int TERMS = sizeof(T) == 4 ? 2 : 1;
    using S = RowsShape<D, TS, TILE, CPS, TERMS>;
    constexpr int kParts = D > 128 ? D / 128 : 1, kPartDim = D / kParts;  // 128-byte columns of a tile
    constexpr int kOwn = kParts / S::kSplit, NO = TILE / TS / 8 / S::kSplit;  // parts, and blocks of 8 tokens' scores, of a warp
    constexpr int kChunk = kPartDim / 8;    // dims of a lane group in a part: 16, or 8
    constexpr uint32_t kTile = S::kTile, kGroups = S::kGroups;
    constexpr int NT = TILE / TS / 8;                                        // blocks of 8 tokens of a warp
    constexpr bool kKeepQ = TERMS == 1 && D <= 64;                        // a row group's q in registers
    extern __shared__ uint8_t raw_smem[];
    __shared__ PlanSmem plan;
    __shared__ uint64_t bars[2 * S::kStages];
    __shared__ GroupScale scales[S::kStages][kGroups];
    __shared__ uint32_t partly[S::kStages];  // a page of the stage's tile is missing
    __shared__ float2 row_ml[TS][16];
    __shared__ float4 told[S::kSplit == 2 ? 2 : 1][TS][S::kSplit][NO][32];  // scores that a pair's warps tell each other, of a tile and the next
    __shared__ float q_unscale[S::kRows];
    __shared__ uint32_t nan_seen, is_last;
    __shared__ Walk walk;
    __shared__ float2 joined_ml[S::kRows];

    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const uint32_t smem = (smem_u32(raw_smem) + 1023u) & ~1023u;
    const uint32_t ring = smem, q_at = smem + S::kStages * S::kStage;
    float* join = reinterpret_cast<float*>(raw_smem + (smem - smem_u32(raw_smem)) + S::kStages * S::kStage + S::kQ);
    const uint32_t full = smem_u32(bars), empty = full + 8 * S::kStages;
    if (threadIdx.x == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&k_map) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&v_map) : "memory");
        for (int i = 0; i < S::kStages; ++i) {
            mbar_init(full + 8 * i, 1);
            mbar_init(empty + 8 * i, S::kWarps);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        nan_seen = 0;
    }
    {
        Range range;
        if (!find_range(c, w, plan, &range)) return;  // (its barriers order the initialisation above)
        if (threadIdx.x == 0) {
            walk.range = range;
            walk.u = range.unit;
            walk.enter(c, w, range.unit_begin);
        }
    }
    __syncthreads();
    uint32_t stage = 0, parity = 0;
    bool alive = true;  // no wait has run out
    auto advance = [&] {
        if (++stage == S::kStages) stage = 0, parity ^= 1;
    };

    if (warp == S::kWarps) {
        // ---- producer --------------------------------------------------------------------------------------------------------------
        const uint32_t page_rows = min(c.cache.page_tokens, 64u);
        const float scale = c.scale * 1.4426950408889634f;
        uint32_t issued = 0;
        const Range range = walk.range;
        Unit u = range.unit;
        uint64_t unit_begin = range.unit_begin;
        __syncthreads();  // the consumers move `walk` on from here
        for (;;) {
            const Segment g = segment(range, u, unit_begin);
            const int32_t first = first_key(u.s, w.window, u.row0(w) / c.group), end = end_key(u.s, c.causal, (u.row0(w) + u.rows(w) - 1) / c.group);
            // a lane knows the page and the scale bytes of one group of 16 tokens, for as many tiles as 32 lanes cover; the next lot is on its way
            constexpr int32_t kLot = 32 / kGroups;
            int32_t page_next = -1;
            uint32_t k_next = 0, v_next = 0;
            auto fetch = [&](int32_t tile) {
                const int32_t t = tile * static_cast<int32_t>(kTile) + static_cast<int32_t>(lane) * 16;
                page_next = -1;
                if (lane < kLot * kGroups && t < end && t + 16 > first && tile + static_cast<int32_t>(lane / kGroups) < g.hi) {
                    const int32_t p = page_of(c.cache, u.seq, t >> c.cache.page_shift);
                    if (static_cast<uint32_t>(p) < c.cache.n_pages) {
                        page_next = p;
                        const uint64_t at = p * c.cache.scale_stride + u.head;
                        k_next = __ldg(c.cache.k_scale + at);
                        v_next = __ldg(c.cache.v_scale + at);
                    } else {
                        page_next = -2;  // a visible token's page is not there
                    }
                }
            };
            fetch(g.lo);
            for (int32_t base = g.lo; base < g.hi; base += kLot) {
                const int32_t page = page_next;
                const uint32_t k_byte = k_next, v_byte = v_next;
                if (base + kLot < g.hi) fetch(base + kLot);
                if (page == -2 && c.status != nullptr) atomicOr(c.status, 8u);  // kStatusBadIndex
                const uint32_t present = __ballot_sync(0xFFFFFFFFu, page >= 0);
                for (int32_t tile = base; tile < min(base + kLot, g.hi); ++tile) {
                    if (alive) alive = __all_sync(0xFFFFFFFFu, mbar_wait(empty + 8 * stage, parity ^ 1));
                    if (!alive) break;
                    const uint32_t in_tile = (tile - base) * kGroups, here = present >> in_tile & static_cast<uint32_t>((uint64_t{1} << kGroups) - 1);
                    const uint32_t step = page_rows / 16;  // groups of a box
                    // a box is issued by the lane that knows its page: the first of its groups that is there
                    const uint32_t box = (lane - in_tile) / step, of = lane >= in_tile && lane < in_tile + kGroups ? here >> (box * step) & ((1u << step) - 1) : 0;
                    const bool issues = of != 0 && lane == in_tile + box * step + __ffs(of) - 1;
                    const uint32_t bytes = __popc(__ballot_sync(0xFFFFFFFFu, issues)) * page_rows * D * 2;
                    if (issues) {
                        const int32_t t = tile * static_cast<int32_t>(kTile) + static_cast<int32_t>(box * page_rows);
                        const int32_t y = static_cast<int32_t>(u.head * c.cache.page_tokens) + (t & static_cast<int32_t>(c.cache.page_tokens - 1));
                        const uint32_t dst = ring + stage * S::kStage + box * page_rows * kPartDim;
#pragma unroll
                        for (int part = 0; part < kParts; ++part) {
                            tma_3d(dst + part * kTile * kPartDim, &k_map, part * 128, y, page, full + 8 * stage);
                            tma_3d(dst + S::kHalfTile + part * kTile * kPartDim, &v_map, part * 128, y, page, full + 8 * stage);
                        }
                    }
                    // The scales, whose bytes arrive while the copies run; the arrival that completes the barrier's phase comes behind them.
                    if (lane >= in_tile && lane < in_tile + kGroups) {
                        GroupScale& s = scales[stage][lane - in_tile];
                        const int32_t v = scale_byte(v_byte) - 127;
                        s.k = page >= 0 ? exp2_int(scale_byte(k_byte) - 127) * scale : 0.0f;
                        s.log_v = page >= 0 ? static_cast<float>(v) : -INFINITY;
                        s.inv_v = page >= 0 ? exp2_int(-v) : 0.0f;
                    }
                    if (lane == 0) partly[stage] = here != static_cast<uint32_t>((uint64_t{1} << kGroups) - 1);
                    __syncwarp();
                    if (elect_one()) mbar_expect(full + 8 * stage, bytes);
                    ++issued;
                    advance();
                }
                if (!alive) break;
            }
            unit_begin = g.unit_end;
            if (!alive || !range.reaches(unit_begin) || !next_unit(c, w, u)) break;
        }
        if (!alive) {
            if (lane == 0) report_lost(w.error_word);
            // nothing may land in this CTA's shared memory once it is gone
            for (uint32_t i = 0; i < min(issued, static_cast<uint32_t>(S::kStages)); ++i) {
                stage = stage == 0 ? S::kStages - 1 : stage - 1;
                if (stage == S::kStages - 1) parity ^= 1;
                mbar_wait(full + 8 * stage, parity);
            }
        }
        __syncthreads();
        return;
    }

    // ---- consumers -------------------------------------------------------------------------------------------------------------------
    constexpr uint32_t kConsumers = S::kWarps * 32;
    const uint32_t ds = warp % S::kSplit, ts = warp / S::kSplit, g8 = lane / 4, t4 = lane % 4;
    const uint32_t my_q = q_at + lane * 16;
    auto tau = [](uint32_t n) { return n ^ ((n & 1) << 2); };  // token of column n of a block of 8: spreads a quarter warp's reads over the banks
    __syncthreads();
    do {
        // q: a warp takes a row at a time, scales it and stores its fp16 terms in the order of the products' operands
        const Unit& u = walk.u;
        const uint32_t rows = walk.rows;
        constexpr int E = D / 32, kEach = (S::kRows + S::kWarps - 1) / S::kWarps, kBatch = kEach < 4 ? kEach : 4;  // rows of a warp whose loads are under way together
        for (uint32_t first = warp; first < rows; first += S::kWarps * kBatch) {
            T raw[kBatch][E];
#pragma unroll
            for (int n = 0; n < kBatch; ++n) {
                const uint32_t r = min(first + n * S::kWarps, rows - 1);
                const T* q = reinterpret_cast<const T*>(walk.at(c, w, c.q, r)) + lane * E;
                if (c.q.vec) {
                    constexpr int kBytes = E * sizeof(T) < 16 ? E * sizeof(T) : 16, kPer = kBytes / sizeof(T);
                    using Word = std::conditional_t<kBytes == 16, uint4, std::conditional_t<kBytes == 8, uint2, uint32_t>>;
#pragma unroll
                    for (int e = 0; e < E; e += kPer) {
                        const Word v = __ldg(reinterpret_cast<const Word*>(q + e));
                        __builtin_memcpy(&raw[n][e], &v, kBytes);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < E; ++e) raw[n][e] = q[e];
                }
            }
#pragma unroll
            for (int n = 0; n < kBatch; ++n) {
                const uint32_t r = first + n * S::kWarps;
                if (r >= S::kRows) break;
                float x[E], top = 0;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    x[e] = r < rows ? to_f32(raw[n][e]) : 0.0f;
                    top = fmaxf(top, fabsf(x[e]) < INFINITY ? fabsf(x[e]) : 0.0f);
                }
#pragma unroll
                for (int d = 16; d != 0; d /= 2) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
                const int32_t exponent = max(static_cast<int32_t>(__float_as_uint(top) >> 23) - 127, -100);
                const float by = exp2_int(14 - exponent);
                if (lane == 0) q_unscale[r] = exp2_int(exponent - 14);
#pragma unroll
                for (int e = 0; e < E; e += 2) {
                    // dim 64 a + 16 t + 4 s + 2 p + {0, 1}: k step 4 a + s, lane t of a quad, register 2 p (+ 1 for the rows 8 and up)
                    const uint32_t d = lane * E + e, step = d / 64 * 4 + d % 16 / 4, t = d % 64 / 16, p = d % 4 / 2;
                    const uint32_t at = q_at + step * TERMS * 512 + (r % 8 * 4 + t) * 16 + (2 * p + r / 8 % 2) * 4;
                    const float a = x[e] * by, b = x[e + 1] * by;
                    const uint32_t hi = half2_bits(a, b);
                    asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(hi) : "memory");
                    if constexpr (TERMS == 2) asm volatile("st.shared.b32 [%0], %1;" ::"r"(at + 512), "r"(half2_rest(a, b, hi)) : "memory");
                }
            }
        }
        bar_sync(1, kConsumers);
        uint4 q_reg[kKeepQ ? D / 16 : 1];
        if constexpr (kKeepQ) {
#pragma unroll
            for (int s = 0; s < D / 16; ++s) q_reg[s] = lds128(my_q + s * 512);
        }
        // this lane's rows of the accumulators: g8 and g8 + 8 of the group
        int32_t lo[2], hi[2];
        float qs[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t r = g8 + 8 * i, j = walk.token(w, min(r, rows - 1));
            lo[i] = first_key(u.s, w.window, j);
            hi[i] = end_key(u.s, c.causal, j);
            qs[i] = q_unscale[r];
        }
        // tiles that every row sees whole, and what any row sees
        const uint32_t first_token = walk.token0, last_token = walk.token(w, rows - 1);
        const int32_t all_lo = first_key(u.s, w.window, last_token), all_hi = end_key(u.s, c.causal, first_token);
        const int32_t any_lo = first_key(u.s, w.window, first_token), any_hi = end_key(u.s, c.causal, last_token);

        float o[kOwn][kChunk][4];
#pragma unroll
        for (int a = 0; a < kOwn; ++a)
#pragma unroll
            for (int b = 0; b < kChunk; ++b) o[a][b][0] = o[a][b][1] = o[a][b][2] = o[a][b][3] = 0;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0, 0};
        // Adds the rows and sums to what lies outside, and begins them anew; behind the last tile the other way round.
        auto settle = [&](bool first, bool last) __attribute__((always_inline)) {
            // Outside: this thread's rows, the threads of a piece side by side, and behind them (maximum that they refer to, sum) of either row.
            float4* outside = reinterpret_cast<float4*>(w.settled) + blockIdx.x * (kConsumers * (S::kPieces + 1)) + threadIdx.x;
            float4 ml = make_float4(-INFINITY, 0, -INFINITY, 0);
            if (!first) ml = outside[S::kPieces * kConsumers];
            // without a maximum what lies outside is zero, or NaN
            const float f[2] = {ml.x == -INFINITY ? 1.0f : exp2_approx(ml.x - m[0]), ml.z == -INFINITY ? 1.0f : exp2_approx(ml.z - m[1])};
            l[0] = fmaf(ml.y, f[0], l[0]), l[1] = fmaf(ml.w, f[1], l[1]);
#pragma unroll
            for (int a = 0; a < kOwn; ++a)
#pragma unroll
                for (int b = 0; b < kChunk; ++b) {
                    float4* at = outside + (a * kChunk + b) * kConsumers;
                    float (&v)[4] = o[a][b];
                    if (!first) {
                        const float4 x = *at;
                        v[0] = fmaf(x.x, f[0], v[0]), v[1] = fmaf(x.y, f[0], v[1]), v[2] = fmaf(x.z, f[1], v[2]), v[3] = fmaf(x.w, f[1], v[3]);
                    }
                    if (!last) {
                        *at = make_float4(v[0], v[1], v[2], v[3]);
                        v[0] = v[1] = v[2] = v[3] = 0;
                    }
                }
            if (!last) {
                outside[S::kPieces * kConsumers] = make_float4(m[0], l[0], m[1], l[1]);
                l[0] = l[1] = 0;
            }
        };

        const uint32_t tok = ts * (NT * 8);  // this warp's first token of a tile
        auto scores = [&](uint32_t st, float (&x)[NO][4]) {  // q . k of this warp's tokens of a stage's tile
            const uint32_t k_at = ring + st * S::kStage, first = tok + ds * (NO * 8);
            constexpr int kChains = NO == 1 ? 2 : 1;  // sums of every other step, where one block of tokens would be one chain of products
            float y[kChains][NO][4];
#pragma unroll
            for (int h = 0; h < kChains; ++h)
#pragma unroll
                for (int n = 0; n < NO; ++n) y[h][n][0] = y[h][n][1] = y[h][n][2] = y[h][n][3] = 0;
#pragma unroll
            for (int a = 0; a < D / 64; ++a) {
                uint4 kw[NO];
#pragma unroll
                for (int n = 0; n < NO; ++n)
                    kw[n] = lds128(k_at + (D > 64 ? a / 2 * kTile * 128 : 0) + swizzled(first + 8 * n + tau(g8), (D > 64 ? a % 2 * 4 : 0) + t4, D));
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    uint4 q[TERMS];
                    if constexpr (kKeepQ) q[0] = q_reg[a * 4 + s];
                    else {
#pragma unroll
                        for (int term = 0; term < TERMS; ++term) q[term] = lds128(my_q + ((a * 4 + s) * TERMS + term) * 512);
                    }
#pragma unroll
                    for (int n = 0; n < NO; ++n) {
                        const uint32_t word = s == 0 ? kw[n].x : s == 1 ? kw[n].y : s == 2 ? kw[n].z : kw[n].w;
                        const uint32_t b0 = widen_lo(word), b1 = widen_hi(word);
#pragma unroll
                        for (int term = 0; term < TERMS; ++term) mma16816(y[s % kChains][n], q[term].x, q[term].y, q[term].z, q[term].w, b0, b1);
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < NO; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) x[n][e] = kChains == 2 ? y[0][n][e] + y[kChains - 1][n][e] : y[0][n][e];
        };
        auto tell = [&](int32_t tile, const float (&x)[NO][4]) {
            if constexpr (S::kSplit == 2) {
#pragma unroll
                for (int n = 0; n < NO; ++n) told[tile & 1][ts][ds][n][lane] = make_float4(x[n][0], x[n][1], x[n][2], x[n][3]);
            }
        };
        // the weights of a tile's scores, and what they add to the sums and rows.  MASKED: some row does not see some token of the tile, because it is at the edge of
        // what the rows see, or has no page.
        auto weigh = [&](const bool MASKED, int32_t t0, float (&x)[NT][4]) __attribute__((always_inline)) {
            const uint32_t v_at = ring + stage * S::kStage + S::kHalfTile;
            // a tile that all rows see spreads the NaN codes of those of its pages that are there to all of them, rightly
            const uint32_t keep = t0 < all_lo || t0 + static_cast<int32_t>(kTile) > all_hi ? 0u : ~0u;
            float top[2] = {-INFINITY, -INFINITY}, inv[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const GroupScale s = scales[stage][(tok + 8 * n) / 16];
                inv[n] = s.inv_v;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float by = s.k * qs[i];
                    x[n][2 * i] = fmaf(x[n][2 * i], by, s.log_v);
                    x[n][2 * i + 1] = fmaf(x[n][2 * i + 1], by, s.log_v);
                }
                if (MASKED) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int32_t t = t0 + static_cast<int32_t>(tok + 8 * n + tau(2 * t4 + e % 2));
                        if (t < lo[e / 2] || t >= hi[e / 2] || s.log_v == -INFINITY) x[n][e] = -INFINITY;
                    }
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) top[i] = fmaxf(top[i], fmaxf(x[n][2 * i], x[n][2 * i + 1]));
            }
            bool grows = false;
            float fade[2], base[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                top[i] = fmaxf(top[i], __shfl_xor_sync(0xFFFFFFFFu, top[i], 1));
                top[i] = fmaxf(top[i], __shfl_xor_sync(0xFFFFFFFFu, top[i], 2));
                const float next = fmaxf(m[i], top[i]);
                grows |= next > m[i];
                fade[i] = m[i] == -INFINITY ? 1.0f : exp2_approx(m[i] - next);  // without a maximum sum and row are zero, or NaN
                m[i] = next;
                base[i] = next == -INFINITY ? 0.0f : next - 14.0f;
            }
            if (__any_sync(0xFFFFFFFFu, grows)) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    l[i] *= fade[i];
#pragma unroll
                    for (int a = 0; a < kOwn; ++a)
#pragma unroll
                        for (int b = 0; b < kChunk; ++b) o[a][b][2 * i] *= fade[i], o[a][b][2 * i + 1] *= fade[i];
                }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[n][e] = exp2_approx(x[n][e] - base[e / 2]);
                l[0] = fmaf(x[n][0] + x[n][1], inv[n], l[0]);
                l[1] = fmaf(x[n][2] + x[n][3], inv[n], l[1]);
            }
            bool nan = false;
#pragma unroll
            for (int s = 0; s < NT / 2; ++s) {
                uint32_t p[TERMS][4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float a = x[2 * s + i / 2][i % 2 * 2], b = x[2 * s + i / 2][i % 2 * 2 + 1];
                    p[0][i] = half2_bits(a, b);
                    if constexpr (TERMS == 2) p[1][i] = half2_rest(a, b, p[0][i]);
                }
                uint32_t row[4];  // the tokens of b0's and b1's halves
#pragma unroll
                for (int i = 0; i < 4; ++i) row[i] = tok + 16 * s + 8 * (i / 2) + tau(2 * t4 + i % 2);
#pragma unroll
                for (int a = 0; a < kOwn; ++a) {
                    uint32_t vw[4][kChunk / 4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if constexpr (D > 64) {
                            const uint4 v = lds128(v_at + (ds * kOwn + a) * kTile * 128 + swizzled(row[i], g8, D));
                            vw[i][0] = v.x, vw[i][1] = v.y, vw[i][2] = v.z, vw[i][3] = v.w;
                        } else {
                            const uint2 v = lds64(v_at + swizzled(row[i], g8 / 2, D) + g8 % 2 * 8);
                            vw[i][0] = v.x, vw[i][1] = v.y;
                        }
                    }
                    if (MASKED) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int32_t t = t0 + static_cast<int32_t>(row[i]);
                            const bool held = t >= any_lo && t < any_hi && scales[stage][row[i] / 16].log_v != -INFINITY;
#pragma unroll
                            for (int b = 0; b < kChunk / 4; ++b) {
                                if (!held) vw[i][b] = 0;
                                nan |= drop_nan(vw[i][b], keep);
                            }
                        }
                    }
#pragma unroll
                    for (int b = 0; b < kChunk / 4; ++b) {
                        const uint32_t l0 = __byte_perm(vw[0][b], vw[1][b], 0x5140), h0 = __byte_perm(vw[0][b], vw[1][b], 0x7362);
                        const uint32_t l1 = __byte_perm(vw[2][b], vw[3][b], 0x5140), h1 = __byte_perm(vw[2][b], vw[3][b], 0x7362);
                        const uint32_t b0[4] = {widen_lo(l0), widen_hi(l0), widen_lo(h0), widen_hi(h0)};
                        const uint32_t b1[4] = {widen_lo(l1), widen_hi(l1), widen_lo(h1), widen_hi(h1)};
#pragma unroll
                        for (int d = 0; d < 4; ++d)
#pragma unroll
                            for (int term = 0; term < TERMS; ++term) mma16816(o[a][4 * b + d], p[term][0], p[term][1], p[term][2], p[term][3], b0[d], b1[d]);
                    }
                }
            }
            if (nan) nan_seen = 1;
        };
        // The next tile's scores are issued in front of this tile's weights: two independent chains for a warp that has few neighbours.  Behind the last
        // tile they are those of whatever the next stage holds, and unused.
        if (alive) alive = __all_sync(0xFFFFFFFFu, mbar_wait(full + 8 * stage, parity));
        float mine[NO][4];
        scores(stage, mine);
        tell(walk.g.lo, mine);
        const int32_t last = walk.g.hi;
        for (int32_t tile = walk.g.lo;;) {
            const int32_t until = min(last, tile + S::kSettle);
            for (; tile < until; ++tile) {
                const bool wraps = stage + 1 == S::kStages;
                const uint32_t next = wraps ? 0 : stage + 1;
                if (alive && tile + 1 < last) alive = __all_sync(0xFFFFFFFFu, mbar_wait(full + 8 * next, parity ^ (wraps ? 1 : 0)));
                const int32_t t0 = tile * static_cast<int32_t>(kTile);
                const bool masked = t0 < all_lo || t0 + static_cast<int32_t>(kTile) > all_hi || partly[stage] != 0;
                float x[NT][4];
                if constexpr (S::kSplit == 2) {  // what is told of the next tile goes beside this one's: one barrier a tile
                    bar_sync(2 + ts, 64);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const float4 v = told[tile & 1][ts][n / NO][n % NO][lane];
                        x[n][0] = v.x, x[n][1] = v.y, x[n][2] = v.z, x[n][3] = v.w;
                    }
                } else {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[n][e] = mine[n][e];
                }
                scores(next, mine);
                tell(tile + 1, mine);
                weigh(masked, t0, x);  // a tile that all rows see spreads its NaN codes to all of them, rightly
                __syncwarp();
                if (lane == 0) mbar_arrive(empty + 8 * stage);
                advance();
            }
            if (tile == last) break;
            settle(tile - walk.g.lo == S::kSettle, false);
        }
        if (last - walk.g.lo > S::kSettle) settle(false, true);

        // ---- the segment's rows: joined over the group's warps, then stored or left in scratch ---------------------------------------------------
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], 1);
            l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], 2);
        }
        const Segment& g = walk.g;
        float* slot = g.whole() ? nullptr : partial_slot(w, D, blockIdx.x, g.from_start);
        auto out_at = [&](uint32_t r) {
            return reinterpret_cast<T*>(walk.at(c, w, c.out, r));
        };
        if (t4 == 0 && ds == 0) row_ml[ts][g8] = make_float2(m[0], l[0]), row_ml[ts][g8 + 8] = make_float2(m[1], l[1]);
        bar_sync(1, kConsumers);
        float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0, 0}, f[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int k = 0; k < TS; ++k) top[i] = fmaxf(top[i], row_ml[k][g8 + 8 * i].x);
#pragma unroll
            for (int k = 0; k < TS; ++k) {
                const float2 ml = row_ml[k][g8 + 8 * i];
                sum[i] += ml.x == -INFINITY ? ml.y : exp2_approx(ml.x - top[i]) * ml.y;
            }
            f[i] = m[i] == -INFINITY ? 1.0f : exp2_approx(m[i] - top[i]);
        }
        // Dim d of a row lies at d + d / 32 * 4: the lanes of a 16-byte store spread over the banks.
        float* into = join + g8 * S::kJoinRow + t4 * (2 * kChunk) + t4 * (2 * kChunk) / 32 * 4;
#pragma unroll 1
        for (int k = 0; k < TS; ++k) {
            if (ts == static_cast<uint32_t>(k)) {
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int a = 0; a < kOwn; ++a)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
#pragma unroll
                            for (int b = 0; b < kChunk; b += 4) {
                                float4* to = reinterpret_cast<float4*>(into + 8 * i * S::kJoinRow + (ds * kOwn + a) * (kPartDim / 32 * 36) + e * kChunk + b);
                                float4 v = make_float4(o[a][b][2 * i + e] * f[i], o[a][b + 1][2 * i + e] * f[i], o[a][b + 2][2 * i + e] * f[i], o[a][b + 3][2 * i + e] * f[i]);
                                if (k != 0) {
                                    const float4 x = *to;
                                    v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
                                }
                                *to = v;
                            }
            }
            bar_sync(1, kConsumers);
        }
        if (warp == 0 && t4 == 0) row_ml[0][g8] = make_float2(top[0], sum[0]), row_ml[0][g8 + 8] = make_float2(top[1], sum[1]);
        bar_sync(1, kConsumers);
        for (uint32_t r = warp; r < walk.rows; r += S::kWarps) {
            const float2 ml = row_ml[0][r];
            const float inv = ml.y != 0 ? 1.0f / ml.y : 0.0f;
            T* out = out_at(r);
#pragma unroll
            for (int e = 0; e < D / 32; ++e) {
                const uint32_t d = e * 32 + lane;
                const float v = join[r * S::kJoinRow + e * 36 + lane];
                if (slot == nullptr) out[d] = from_f32<T>(v * inv);
                else slot[r * D + d] = v;
            }
            if (slot != nullptr && lane == 0) *reinterpret_cast<float2*>(slot + w.rows * D + 2 * r) = ml;
        }
        bar_sync(1, kConsumers);
        if (nan_seen != 0) {
            spread_nan(c, w, walk.u, walk.g, 0, walk.u.rows(w), 0, D, threadIdx.x, kConsumers, [&](uint32_t r, uint32_t d) {
                if (slot == nullptr) out_at(r)[d] = from_f32<T>(NAN);
                else slot[r * D + d] = NAN;
            });
            bar_sync(1, kConsumers);
            if (threadIdx.x == 0) nan_seen = 0;
        }
        if (slot != nullptr) {
            const Range& range = walk.range;
            const uint32_t c0 = owner(g.unit_begin, range.total, range.ctas), shares = owner(g.unit_end - 1, range.total, range.ctas) - c0 + 1;
            __threadfence();
            bar_sync(1, kConsumers);
            if (threadIdx.x == 0) {
                const bool last = atomicAdd(w.counters + c0, 1u) == shares - 1;
                if (last) w.counters[c0] = 0;
                is_last = last;
            }
            bar_sync(1, kConsumers);
            if (is_last != 0) {
                __threadfence();
                join_partials<T, D, 2>(c, w, walk, c0, shares, 0, S::kWarps, joined_ml);
            }
        }
        bar_sync(1, kConsumers);  // nobody reads q, the joined rows or `walk` any more
        if (threadIdx.x == 0) walk.advance(c, w);
        bar_sync(1, kConsumers);
    } while (walk.more != 0);
    if (!alive && lane == 0) report_lost(w.error_word);
    __syncthreads();
}

/// The cache's pool as {dim, rows of all heads of a page, pages}, a box of one page's rows of one head.
int pool_map(const Cache& c, const uint8_t* pool, uint32_t box_rows, CUtensorMap* out);

template <class T, int D, int TS, int TILE, int CPS>
int launch_rows_kernel(HaloCudaCtx* ctx, const AttentionCall& c, Work w, cudaStream_t s) {
    using S = RowsShape<D, TS, TILE, CPS, sizeof(T) == 4 ? 2 : 1>;
    w.rows = S::kRows;
    w.tile = S::kTile;
    w.pad = 4;  // 48 decoding sequences of 156 - 7697 tokens 65.6 us, with 2 or 6 67.6; drafts of 12 sequences 73.9, 74.7 with 2, 73.7 with 6
    w.group = c.group;
    w.group_inverse = static_cast<uint32_t>((0xFFFFFFFFull + c.group) / c.group);
    w.row_tiles = (w.max_rows + S::kRows - 1) / S::kRows;
    w.lanes = 1;
    while (w.lanes < 32 && w.lanes < w.row_tiles) w.lanes *= 2;
    CUtensorMap k_map, v_map;
    const uint32_t box = std::min(c.cache.page_tokens, 64u);
    if (int rc = pool_map(c.cache, c.cache.k, box, &k_map)) return rc;
    if (int rc = pool_map(c.cache, c.cache.v, box, &v_map)) return rc;
    const uint32_t ctas = CPS * static_cast<uint32_t>(ctx->prop.multiProcessorCount);
    void* p = nullptr;
    if (int rc = workspace(ctx, 5, ctas * sizeof(uint32_t), s, &p, true)) return rc;
    w.counters = static_cast<uint32_t*>(p);
    const uint64_t partials = partial_bytes(S::kRows, D, ctas);
    if (int rc = workspace(ctx, 6, partials + ctas * S::kSettledBytes, s, &p)) return rc;
    w.partials = static_cast<float*>(p);
    w.settled = w.partials + partials / 4;
    w.error_word = ctx->error_word_dev;
    auto kernel = rows_kernel<T, D, TS, TILE, CPS>;
    if (int rc = allow_dynamic_smem(ctx, reinterpret_cast<const void*>(kernel), S::kSmem)) return rc;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(S::kThreads);
    cfg.dynamicSmemBytes = S::kSmem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    HC_CUDA(cudaLaunchKernelEx(&cfg, kernel, k_map, v_map, c, w));
    return 0;
}

/// One of the kernels by operand type and rows; instantiated for each head size in a file of its own.
template <int D>
int launch_kernel(HaloCudaCtx* ctx, const AttentionCall& c, const Work& w, cudaStream_t s);

/// Up to how many packed rows of a sequence the row kernel takes.  12 sequences of 2156 - 4688 tokens, row kernel / tcgen05 kernel, us: heads of 256, 24
/// rows: fp32 68 / 82, bf16 57 / 52; 48 rows: 93 / 94, 77 / 61.  Heads of 128, 32 rows: fp32 62 / 72; 48 rows: 83 / 75, bf16 64 / 82; 64 rows: bf16 80 / 83; 96
/// rows: 110 / 86.  Heads of 64, 48 rows: fp32 53 / 57; 64 rows: 65 / 58, bf16 56 / 58; 96 rows: 77 / 60.  One rule between calls that want another: a
/// single sequence of 1037 tokens is better off here with more rows (heads of 256, 48 rows: bf16 21 / 33, fp32 23 / 44), 48 sequences of 6000 there
/// with fewer (heads of 256, 24 rows, bf16: 272 / 187; heads of 128, 48 rows, fp32: 462 / 347).
inline uint32_t few_rows(const AttentionCall& c) { return c.cache.head_dim == 256 ? 32 : c.type == HALO_CUDA_T_F32 ? 48 : 64; }

}  // namespace attn
}  // namespace halo_cuda
