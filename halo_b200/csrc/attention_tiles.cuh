// ATTENTION for many rows to a sequence (prompts, chunks of prompts): tcgen05 products with fp16 operands, the cache's codes converted to fp16 once
// for 256 packed rows (128 for heads of 256 elements, and for fp32 operands, whose q and weights are two fp16 terms each).
//
//   x_t = q . k_t * (s_K(t) * scale * log2 e) + log2 s_V(t),   p_t = 2^(x_t - r + 6),   o = sum p_t code(v_t),   l = sum p_t / s_V(t),   out = o / l
//
// as in attention_rows.cuh; r is a reference that follows the running maximum lazily: the accumulators are rescaled only when a row's maximum
// passes r by 8, so p_t is at most 2^14 and keeps 11 bits down to 2^-20 of the reference.
//
// Packed rows are the M side (a TMEM lane each), keys the N side of S = Q K^T, dims the N side of O = P V.  A CTA (one an SM) holds NS tiles of
// 128 rows: two, each with scores, weights and accumulators of its own (128 + D columns), or one (D = 256, and fp32 operands) with two score
// buffers.  A step is (tile of 128 keys, or of 64 for fp32 rows of 256 elements; row tile) and takes score buffer step % 2: while the softmax of one step
// runs, the tensor cores run the other's products.  The weights overwrite the scores in TMEM as fp16 and are the A operand of P V from there.
// Warps:
//   0       tcgen05.mma issue
//   1-3     q -> fp16 in shared memory, of the next segment while the last one's last weights are made (and TMEM's allocation)
//   4-7     conversion (4-11 where D is 256): each warp makes one part of K or V of every tile in a ring of eight 16 KiB slots (a K slot: 128 keys x
//           64 dims; a V slot: 8192 / D keys x all dims, the N operand with dims contiguous); keys that no row of the CTA sees, missing pages and,
//           in tiles at the edge of what some row sees, NaN codes of values become zeros (spread_nan puts the latter back)
//   last 8  softmax, a thread to a row and a tile's keys, or to half of them where NS is 1; also the epilogue, and the joining of shares
// Work is dealt as in attention_work.cuh, so a causal prompt's long and short rows and a short chunk behind a long context fill the device alike.
//
// What bounds it.  For D = 128 256 rows x 128 keys are 2100 clocks of products, and as many of exponentials (16 a clock).  Prompts of 364 - 1568 tokens (76.6
// GFLOP, 720 units) take 209 us, 370 TFLOP/s: the two row tiles' chains of scores, maximum, weights and products overlap only in part, and a unit's ends
// (q, first scores, last rows) cost as much as two or three tiles.  Code size counts as much as instructions: the warps of an SM run five different loops,
// and unrolled ones waited for instructions more than for anything else.  2048 tokens behind 28000 with D = 256 (1459 GFLOP) take 1611 us, 906 TFLOP/s,
// with inputs that change (1480 back to back on the same ones): a little over half of what the tensor cores do; the conversion of the codes, once for 128 rows,
// holds it up.
#pragma once
#include "attention_rows.cuh"

namespace halo_cuda {
namespace attn {

/// TERMS: fp16 terms of q and of the weights (1: 16-bit operands, 2: fp32 operands).
template <int D, int TERMS>
struct TilesShape {
    static constexpr int kStreams = D == 256 || TERMS == 2 ? 1 : 2, kRows = 128 * kStreams, kSlots = 8;
    static constexpr int kTile = D == 256 && TERMS == 2 ? 64 : 128;  // keys: both terms of q leave room for half
    static constexpr int kParts = D / 64;                  // slots of a tile of K, and of V
    static constexpr int kVTokens = kTile * 64 / D;        // keys of a V slot
    static constexpr uint32_t kSlot = kTile * 128, kQ = kRows * D * 2 * TERMS;
    static constexpr uint32_t kSmem = 1024 + kQ + kSlots * kSlot;
    static constexpr uint32_t kBuffer = kTile;             // columns of a score buffer, which the terms of the weights (kTile / 2 columns each) overwrite
    static constexpr uint32_t kO = 256;                    // first accumulator column
    // The tensor cores cut sums off instead of rounding them, always towards zero.  After so many tiles a row's products, and its sum of weights, are added up
    // in fp32 outside: 64 products of 16 keys for fp32 operands (8 tiles of 64 keys, 4 of 128; 262144 positions to a block: 1e-5 off), 1024 for 16-bit ones
    // (128 tiles; 4 million positions to a block: 7e-3 too small without, within fp16's half step with it, for 2 % of short prompts' time).
    static constexpr int32_t kSettle = (TERMS == 2 ? 64 : 1024) / (kTile / 16 * TERMS);
    static constexpr int kHalves = 2 / kStreams;           // softmax warpgroups that share a row tile's keys
    static constexpr int kKeys = kTile / kHalves;          // of a tile that one of them has
    /// Column of a score buffer that the weights of a tile's 16 keys from 16 * i on begin at: a warpgroup's lie where its scores were.
    static constexpr uint32_t weights_at(uint32_t term, uint32_t i) {
        return TERMS == 2 ? term * (kTile / 2) + i * 8 : i / (kKeys / 16) * kKeys + i % (kKeys / 16) * 8;
    }
    static constexpr int kConvWarps = D == 256 ? 8 : 4, kSoftWarp = 4 + kConvWarps, kSoftWarps = 8, kThreads = (kSoftWarp + kSoftWarps) * 32;
    // Slot number i of a CTA (the parts of K of its first tile, those of V, those of K of the second, ...) has place i % kSlots.  A place's user waits for
    // its last use by the parity of that use, so all of a place's uses are to be one warp's: 2 * kParts * kEvery of convert_slots divides kSlots.
    static_assert(kSlots % kConvWarps == 0);
    static constexpr uint32_t kAccesses = kSlot / 1024;    // 16-byte pieces of a slot that a conversion thread makes
    static constexpr uint32_t kAhead = 8;                  // that it has under way (all 16 of D = 256: 1672 -> 2147 us for 2048 tokens behind 28000)
    // What a thread has at launch; the warpgroups hand each other what they leave.
    static constexpr int kLaunchRegs = kThreads == 512 ? 128 : 96;
    static constexpr int kIdleRegs = kStreams == 1 ? 80 : 72, kConvRegs = D == 256 ? 80 : 88, kSoftRegs = D == 256 ? 120 : kStreams == 1 ? 168 : 176;
    static_assert(kIdleRegs + kConvRegs * (kConvWarps / 4) + 2 * kSoftRegs <= kLaunchRegs * (kThreads / 128));
};

__device__ __forceinline__ uint64_t desc_k(uint32_t addr) {  // K-major, 128-byte rows and swizzle: atoms of 8 rows, 1024 bytes apart
    return static_cast<uint64_t>((addr & 0x3FFFFu) >> 4) | (uint64_t{1} << 16) | (uint64_t{64} << 32) | (uint64_t{1} << 46) | (uint64_t{2} << 61);
}
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr, uint32_t block) {  // N-major: atoms of 64 elements x 8 keys, 1024 bytes apart along the keys, `block` along N
    return static_cast<uint64_t>((addr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(block >> 4) << 16) | (uint64_t{64} << 32) | (uint64_t{1} << 46) | (uint64_t{2} << 61);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add)
                 : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(add)
                 : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

#define HALO_R8(v, i) "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3]), "=r"(v[i + 4]), "=r"(v[i + 5]), "=r"(v[i + 6]), "=r"(v[i + 7])
#define HALO_W8(v, i) "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3]), "r"(v[i + 4]), "r"(v[i + 5]), "r"(v[i + 6]), "r"(v[i + 7])
/// 32 columns of this warp's lanes.
__device__ __forceinline__ void tmem_ld32(uint32_t at, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : HALO_R8(v, 0), HALO_R8(v, 8), HALO_R8(v, 16), HALO_R8(v, 24)
        : "r"(at)
        : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t at, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::HALO_W8(v, 0),
        HALO_W8(v, 8), HALO_W8(v, 16), HALO_W8(v, 24), "r"(at)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::HALO_W8(v, 0), HALO_W8(v, 8), "r"(at)
                 : "memory");
}
#undef HALO_R8
#undef HALO_W8
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ void unpair(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ void sts128(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

/// Where a conversion warp's loads are: in shared memory, so that the pieces under way have the registers.
struct Cursor {
    Unit u;
    Segment g;
};

/// The slots of one part of K or V, of every `every`-th tile from `turn` on, over a CTA's whole range, by one warp: 16-byte pieces straight from the
/// pages to registers, kAhead of the slot's 16 accesses under way in front of the one that is converted.  The warp of K's part 0 publishes the tile's scales
/// with its slot.
template <int D, int TERMS, bool IS_V>
__device__ __forceinline__ void convert_slots(const AttentionCall& c, const Work& w, const Range& range, Cursor& cursor, uint32_t part, uint32_t turn, uint32_t every, uint32_t ring,
                                              uint32_t full, uint32_t empty, GroupScale (*scales)[8], uint32_t* nan_tiles, bool& alive) {
    using S = TilesShape<D, TERMS>;
    constexpr uint32_t kBlocks = IS_V ? S::kParts : 1;                   // 64-dim blocks of a slot's rows
    constexpr int32_t kTile = S::kTile;
    constexpr uint32_t kRows = IS_V ? S::kVTokens : kTile, kStep = 8 / kBlocks;  // rows of a slot; of one access of the warp
    constexpr uint32_t kAccesses = S::kAccesses, kAhead = S::kAhead;
    constexpr uint32_t kPerGroup = 16 / kStep;                           // accesses of 16 rows
    const uint32_t lane = threadIdx.x % 32;
    // a quarter warp has four pieces of two rows: its eight 16-byte stores lie in different banks
    const uint32_t lane_row = lane / 8 / kBlocks * 2 + lane / 4 % 2, block = lane / 8 % kBlocks;
    const uint32_t from = lane_row * D + (IS_V ? block * 64 : part * 64) + lane % 4 * 16;             // of a group's first row
    const uint32_t to = block * (kRows * 128) + lane_row * 128 + ((lane % 4 * 2 ^ (lane_row & 7)) << 4);  // second half: the same ^ 16
    // the tile that is loaded: of the CTA's tiles number `count`, keys from t0 on; lane i knows page and scale bytes of its i-th 16 keys, and those of
    // this warp's next tile
    int32_t tile, last, any_lo, any_hi, all_lo, all_hi, page = -1;
    int32_t entry = -1;                 // of the page table, for this warp's next tile; not looked at before that tile's turn
    uint32_t k_byte = 0, v_byte = 0, count = 0;
    uint64_t group_at = 0;              // lane i: where its keys' codes begin in the pool
    bool plain = false, whole = false;  // every key is there and seen by some row; every key that is there is seen by all rows
    const uint8_t* pool = nullptr;
    auto fetch = [&](int32_t of) {
        const int32_t t = of * kTile + static_cast<int32_t>(lane) * 16;
        entry = -1;
        if (lane < kTile / 16 && of < last && t < any_hi && t + 16 > any_lo) {
            entry = page_of(c.cache, cursor.u.seq, t >> c.cache.page_shift);
        }
    };
    auto take = [&] {  // the fetched tile becomes the one that is loaded
        const int32_t t0 = tile * kTile, t = t0 + static_cast<int32_t>(lane) * 16;
        const bool wanted = lane < kTile / 16 && t < any_hi && t + 16 > any_lo;
        page = !wanted ? -1 : static_cast<uint32_t>(entry) < c.cache.n_pages ? entry : -2;  // -2: a visible key's page is not there
        if (!IS_V && part == 0 && page >= 0) {
            const uint64_t at = page * c.cache.scale_stride + cursor.u.head;
            k_byte = __ldg(c.cache.k_scale + at);
            v_byte = __ldg(c.cache.v_scale + at);
        }
        plain = t0 >= any_lo && t0 + kTile <= any_hi && __all_sync(0xFFFFFFFFu, page >= 0 || lane >= kTile / 16);
        whole = t0 >= all_lo && t0 + kTile <= all_hi;
        group_at = static_cast<uint32_t>(max(page, 0)) * c.cache.page_stride + ((static_cast<uint32_t>(t0) + lane * 16) & (c.cache.page_tokens - 1)) * D;
        fetch(tile + static_cast<int32_t>(every));
    };
    /// Enters the cursor's segment at its tile number `skip`, or a later one's at what is left of it; false at the end of the range.
    auto enter = [&](uint32_t skip) -> bool {
        for (;;) {
            const uint32_t n = static_cast<uint32_t>(cursor.g.hi - cursor.g.lo);
            if (skip < n) break;
            skip -= n, count += n;
            const uint64_t begin = cursor.g.unit_end;
            bool more = range.reaches(begin);
            if (more) {
                Unit u = cursor.u;
                more = next_unit(c, w, u);
                const Segment g = segment(range, u, begin);
                __syncwarp();
                if (lane == 0) cursor.u = u, cursor.g = g;
                __syncwarp();
            }
            if (!more) return false;
        }
        const Unit& u = cursor.u;
        const uint32_t first = u.row0(w) / c.group, final = (u.row0(w) + u.rows(w) - 1) / c.group;
        any_lo = first_key(u.s, w.window, first), any_hi = end_key(u.s, c.causal, final);
        all_lo = first_key(u.s, w.window, final), all_hi = end_key(u.s, c.causal, first);
        tile = cursor.g.lo + static_cast<int32_t>(skip), last = cursor.g.hi, count += skip;
        pool = (IS_V ? c.cache.v : c.cache.k) + (uint64_t{u.head} << c.cache.page_shift) * D + from;
        fetch(tile);
        take();
        return true;
    };
    auto advance = [&]() -> bool {  // to this warp's next tile
        if (tile + static_cast<int32_t>(every) < last) {
            tile += static_cast<int32_t>(every), count += every;
            take();
            return true;
        }
        const uint32_t done = static_cast<uint32_t>(tile - cursor.g.lo);
        count -= done;
        return enter(done + every);
    };
    uint4 x[kAhead];
    constexpr uint32_t kLot = kAhead / 2;  // accesses that are converted, and asked for, together
    auto load = [&](uint32_t lot, uint32_t p) __attribute__((always_inline)) {  // accesses lot * kLot .. of the tile that is loaded; lot % 2 == p
        constexpr uint32_t kFirst = IS_V ? kRows / 16 : 0;  // groups of a part of V
        if (plain) {
            constexpr uint32_t kSpan = kLot > kPerGroup ? kLot / kPerGroup : 1, kIn = kLot / kSpan;  // groups of a lot; accesses of each
#pragma unroll
            for (uint32_t n = 0; n < kSpan; ++n) {
                const uint32_t i0 = lot * kLot + n * kIn;
                const uint8_t* src = pool + __shfl_sync(0xFFFFFFFFu, group_at, i0 / kPerGroup + part * kFirst);
#pragma unroll
                for (uint32_t j = 0; j < kIn; ++j) x[p * kLot + n * kIn + j] = __ldg(reinterpret_cast<const uint4*>(src + (i0 + j) % kPerGroup * kStep * D));
            }
        } else {
#pragma unroll
            for (uint32_t j = 0; j < kLot; ++j) x[p * kLot + j] = make_uint4(0, 0, 0, 0);
#pragma unroll 1
            for (uint32_t g = lot * kLot / kPerGroup; g <= (lot * kLot + kLot - 1) / kPerGroup; ++g) {
                const uint32_t group = g + (IS_V ? part * (kRows / 16) : 0);
                const uint8_t* from_group = pool + __shfl_sync(0xFFFFFFFFu, group_at, group);
                const bool there = __shfl_sync(0xFFFFFFFFu, page, group) >= 0;
#pragma unroll
                for (uint32_t j = 0; j < kLot; ++j) {
                    const uint32_t i = lot * kLot + j, k = i % kPerGroup * kStep;
                    const int32_t t = tile * kTile + static_cast<int32_t>(group * 16 + k + lane_row);
                    if (i / kPerGroup == g && there && t >= any_lo && t < any_hi) x[p * kLot + j] = __ldg(reinterpret_cast<const uint4*>(from_group + k * D));
                }
            }
        }
    };
    if (!enter(turn)) return;
    load(0, 0);
    load(1, 1);
    const float scale = fabsf(c.scale) * 1.4426950408889634f;  // its sign is q's
    for (bool more = true; more;) {
        const uint32_t number = (2 * count + (IS_V ? 1 : 0)) * S::kParts + part, at = number % S::kSlots, slot = ring + at * S::kSlot;
        const bool check = IS_V && !whole;
        if (alive) alive = __all_sync(0xFFFFFFFFu, mbar_wait(empty + 8 * at, (number / S::kSlots & 1) ^ 1));
        const bool gap = !IS_V && part == 0 && __any_sync(0xFFFFFFFFu, page == -2);
        if (!IS_V && part == 0 && lane < kTile / 16) {
            GroupScale& s = scales[count % 8][lane];
            s.gap = gap;
            const int32_t v = scale_byte(v_byte) - 127;
            s.k = page >= 0 ? exp2_int(scale_byte(k_byte) - 127) * scale : 0.0f;
            s.log_v = page >= 0 ? static_cast<float>(v) : -INFINITY;
            s.inv_v = page >= 0 ? exp2_int(-v) : 0.0f;
            if (page == -2 && c.status != nullptr) atomicOr(c.status, 8u);  // kStatusBadIndex
        }
        // two lots' worth of code for all: unrolled, the warps waited for instructions (2048 tokens behind 28000, heads of 256: 1520 us, so 1440)
#pragma unroll 1
        for (uint32_t o = 0; o < kAccesses / kAhead; ++o) {
            const bool last_ones = o + 1 == kAccesses / kAhead;  // behind them the next tile is loaded
#pragma unroll
            for (uint32_t p = 0; p < 2; ++p) {
                const uint32_t lot = 2 * o + p;
                if (check) {  // a weight of zero would spread a NaN to rows that do not see it
                    bool nan = false;
#pragma unroll
                    for (uint32_t j = 0; j < kLot; ++j) {
                        uint4& v = x[p * kLot + j];
                        nan |= drop_nan(v.x) | drop_nan(v.y) | drop_nan(v.z) | drop_nan(v.w);
                    }
                    if (nan) atomicMax(nan_tiles, count + 1);  // (of the next tile where that is loaded already)
                }
#pragma unroll
                for (uint32_t j = 0; j < kLot; ++j) {
                    const uint32_t row = (lot * kLot + j) * kStep, to_row = (slot + to + row * 128) ^ ((row & 7) << 4);
                    const uint4 v = x[p * kLot + j];
                    sts128(to_row, widen_lo(v.x), widen_hi(v.x), widen_lo(v.y), widen_hi(v.y));
                    sts128(to_row ^ 16, widen_lo(v.z), widen_hi(v.z), widen_lo(v.w), widen_hi(v.w));
                }
                if (p == 0 && last_ones) more = advance();
                if (!last_ones || more) load(last_ones ? p : lot + 2, p);
            }
        }
        proxy_fence();
        __syncwarp();
        if (lane == 0) mbar_arrive(full + 8 * at);
    }
}

template <class T, int D>
__global__ void __launch_bounds__(TilesShape<D, sizeof(T) == 4 ? 2 : 1>::kThreads, 1) tiles_kernel(const __grid_constant__ AttentionCall c, const __grid_constant__ Work w) {
    constexpr int TERMS = sizeof(T) == 4 ? 2 : 1;
    using S = TilesShape<D, TERMS>;
    constexpr int kTile = S::kTile;
    constexpr int kStreams = S::kStreams, kParts = S::kParts, kSlots = S::kSlots, kScaleTiles = 8;
    extern __shared__ uint8_t raw_smem[];
    __shared__ PlanSmem plan;
    __shared__ uint64_t bars[2 * kSlots + 3 * 2 + 3];
    __shared__ GroupScale scales[kScaleTiles][8];  // a tile's stay until the slots' ring has gone round behind it: at most six tiles ahead are written
    __shared__ float q_unscale[2][S::kRows];  // of a segment and the next
    __shared__ float2 joined_ml[S::kRows];
    __shared__ float shared_top[2][S::kHalves][128];  // of a tile and the next: the maxima that a row tile's warpgroups tell each other
    __shared__ uint32_t nan_tiles, is_last, tmem_word;  // nan_tiles: of the CTA's tiles, how many the last one with a NaN code left out is in
    __shared__ uint32_t moved;                          // counted up by the softmax warps as they go on
    __shared__ Cursor cursors[S::kConvWarps];
    __shared__ Walk walks[2];  // the segment at hand and the next one, in turn

    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const uint32_t q_at = (smem_u32(raw_smem) + 1023u) & ~1023u, ring = q_at + S::kQ;
    const uint32_t full = smem_u32(bars), empty = full + 8 * kSlots, s_full = empty + 8 * kSlots, p_ready = s_full + 16, pv_done = p_ready + 16, q_ready = pv_done + 16, q_free = q_ready + 8, idle = q_free + 8;
    if (threadIdx.x == 0) {
        for (int i = 0; i < kSlots; ++i) {
            mbar_init(full + 8 * i, 1);
            mbar_init(empty + 8 * i, 1);
        }
        mbar_init(q_ready, 3);
        mbar_init(q_free, 1);
        mbar_init(idle, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(s_full + 8 * i, 1);
            mbar_init(p_ready + 8 * i, 4 * S::kHalves);
            mbar_init(pv_done + 8 * i, 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        nan_tiles = 0;
        moved = 0;
    }
    {
        Range range;
        if (!find_range(c, w, plan, &range)) return;
        if (threadIdx.x == 0) {
            walks[0].range = range;
            walks[0].u = range.unit;
            walks[0].enter(c, w, range.unit_begin);
            for (Cursor& x : cursors) x = Cursor{range.unit, walks[0].g};
        }
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_word)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tmem_before();
    __syncthreads();
    tmem_after();
    const uint32_t tmem = tmem_word;
    bool alive = true;  // no wait has run out; behind one nothing is waited for and the results are void (the context is lost)
    auto wait = [&](uint32_t bar, uint32_t parity) {
        if (alive) alive = __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity));
    };
    const Range range = walks[0].range;
    __syncthreads();  // `walks` belong to the softmax warps from here

    if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::kIdleRegs));
    if (warp == 0) {
        // ---- products --------------------------------------------------------------------------------------------------------------------
        constexpr uint32_t kScores = (1u << 4) | (static_cast<uint32_t>(kTile) / 8 << 17) | (128u / 16 << 24), kRowsOut = (1u << 4) | (1u << 16) | (static_cast<uint32_t>(D) / 8 << 17) | (128u / 16 << 24);
        // What the issue needs is in uniform registers: the slots' places follow from the tile's number alone, and nothing but elect_one() guards it.
        Unit u = range.unit;
        uint64_t unit_begin = range.unit_begin;
        uint32_t count = 0, segments = 0, uses[2] = {0, 0};  // tiles; segments; waits for the weights in either score buffer
        constexpr uint32_t kRounds = kSlots / (2 * kParts);  // tiles that fill the ring
        const uint64_t q_desc = desc_k(q_at), k_desc = desc_k(ring), v_desc = desc_mn(ring, S::kVTokens * 128);
        constexpr uint32_t kSlotDesc = S::kSlot / 16, kSteps = S::kVTokens / 16;
        auto scores = [&](uint32_t tile, uint32_t s, uint32_t buffer) {  // tile: its number in the CTA
            const uint32_t place = __shfl_sync(0xFFFFFFFFu, tile % kRounds * (2 * kParts), 0), parity = tile / kRounds & 1;
            // the small terms first: sums are cut off at the size they have by then
#pragma unroll
            for (uint32_t i = 0; i < TERMS * kParts; ++i) {
                const uint32_t term = TERMS - 1 - i / kParts, part = i % kParts;
                if (s == 0 && i < kParts) wait(full + 8 * (place + part), parity);
                tmem_after();
                if (elect_one()) {
                    const uint64_t a = q_desc + ((term + s) * kParts + part) * 1024u, b = k_desc + (place + part) * kSlotDesc;
#pragma unroll
                    for (uint32_t k = 0; k < 4; ++k) mma_ss(tmem + buffer * S::kBuffer, a + k * 2, b + k * 2, kScores, i + k != 0);
                    if (term == 0 && s == kStreams - 1) mma_commit(empty + 8 * (place + part));
                    if (i == TERMS * kParts - 1) mma_commit(s_full + 8 * buffer);
                }
            }
        };
        auto rows = [&](uint32_t tile, uint32_t s, uint32_t buffer, bool add) {
            const uint32_t place = __shfl_sync(0xFFFFFFFFu, tile % kRounds * (2 * kParts) + kParts, 0), parity = tile / kRounds & 1;
            wait(p_ready + 8 * buffer, (buffer == 0 ? uses[0]++ : uses[1]++) & 1);
            const uint32_t first = __shfl_sync(0xFFFFFFFFu, add ? 1u : 0u, 0);
#pragma unroll
            for (uint32_t part = 0; part < kParts; ++part) {
                if (s == 0) wait(full + 8 * (place + part), parity);
                tmem_after();
                if (elect_one()) {
                    const uint64_t v = v_desc + (place + part) * kSlotDesc;
#pragma unroll
                    for (uint32_t term = 0; term < TERMS; ++term)
#pragma unroll
                        for (uint32_t k = 0; k < kSteps; ++k)
                            mma_ts(tmem + S::kO + s * D, tmem + buffer * S::kBuffer + S::weights_at(term, part * kSteps + k), v + k * 128, kRowsOut,
                                   part + term + k != 0 ? 1u : first);
                    if (s == kStreams - 1) mma_commit(empty + 8 * (place + part));
                    if (part == kParts - 1) mma_commit(pv_done + 8 * buffer);
                }
            }
        };
        // Behind the segment's last scores the next one's q may be written, while the last weights are still to come.  Not before weights of this segment
        // were there, though: all softmax warps are past their look at q_ready then, and it can go on by a phase.
        auto release_q = [&] {
            if (elect_one()) mma_commit(q_free);
        };
        for (;;) {
            const Segment g = segment(range, u, unit_begin);
            const uint32_t n = static_cast<uint32_t>(g.hi - g.lo);
            wait(q_ready, segments & 1);
#pragma unroll
            for (uint32_t s = 0; s < kStreams; ++s) scores(count, s, s);
            if (kStreams == 1 && n > 1) scores(count + 1, 0, 1);
            for (uint32_t t = 0; t < n; ++t) {
                if constexpr (kStreams == 2) {
#pragma unroll
                    for (uint32_t s = 0; s < kStreams; ++s) {
                        rows(count + t, s, s, t % S::kSettle != 0);
                        if (t + 1 < n) scores(count + t + 1, s, s);
                        if (s == kStreams - 1 && t + 2 == n) release_q();
                    }
                } else {
                    const uint32_t buffer = __shfl_sync(0xFFFFFFFFu, t & 1, 0);
                    rows(count + t, 0, buffer, t % S::kSettle != 0);
                    if (t + 2 < n) scores(count + t + 2, 0, buffer);
                    if (t + 3 == n) release_q();
                }
            }
            count += n;
            ++segments;
            if (n < 4 - kStreams) release_q();
            unit_begin = g.unit_end;
            if (!range.reaches(unit_begin) || !next_unit(c, w, u)) break;
        }
        if (!alive) {  // products may still be under way: TMEM and shared memory are given back when they are done
            if (elect_one()) mma_commit(idle);
            mbar_wait(idle, 0);
        }
    } else if (warp < 4) {
        // ---- q: eight lanes to a row.  The operand's bits take as much room as the fp16 terms that they become: all rows are copied to where their terms
        // go, so that their latency shows once, and converted in place, every lane what it has copied. ------------------------------------------------------
        constexpr uint32_t kPieces = D / 64, kWords = 4 * TERMS, kStride = 12;  // pieces of 8 elements of a lane, 64 elements apart; rows of the three warps
        const uint32_t l8 = lane % 8, first = (warp - 1) * 4 + lane / 8;
        Unit u = range.unit;
        uint64_t unit_begin = range.unit_begin;
        for (uint32_t segments = 0;; ++segments) {
            const Segment g = segment(range, u, unit_begin);
            const uint32_t rows = u.rows(w), r0 = u.row0(w), token0 = r0 / c.group, behind = r0 - token0 * c.group;
            const uint8_t* base = c.q.p + uint64_t{u.s.row0 + token0} * c.q.token_stride + uint64_t{u.head} * c.group * c.q.head_stride + l8 * (8 * sizeof(T));
            auto source = [&](uint32_t row) {
                const uint32_t p = behind + row, t = w.group == 1 ? p : __umulhi(p, w.group_inverse);
                return base + t * c.q.token_stride + (p - t * w.group) * c.q.head_stride;
            };
            auto place = [&](uint32_t row) {  // 64-element blocks of [128 rows][128 bytes]; a second term's are behind the first's
                return q_at + row / 128 * (kParts * 16384) + row % 128 * 128 + ((l8 ^ (row & 7)) << 4);
            };
            for (uint32_t row = first; row < rows; row += kStride) {
                const uint8_t* q = source(row);
#pragma unroll
                for (uint32_t k = 0; k < kPieces; ++k) asm volatile("prefetch.global.L2 [%0];" ::"l"(q + k * (64 * sizeof(T))));
            }
            // The segment before has its last scores, and the softmax is not behind it.  That is as far away as the segment is long: on contexts of some tens of
            // millions of positions a wait for one step would run out.  (The products' and conversion's waits are for a step, and looked at `moved` 2 - 4 % slower.)
            if (segments != 0 && alive) alive = __all_sync(0xFFFFFFFFu, mbar_wait(q_free, (segments - 1) & 1, &moved));
#pragma unroll 1
            for (uint32_t row = first; row < rows; row += kStride) {
                const uint8_t* q = source(row);
                const uint32_t to = place(row);
                if (c.q.vec) {
#pragma unroll
                    for (uint32_t k = 0; k < kPieces * TERMS; ++k)
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + (k / TERMS + k % TERMS * kParts) * 16384), "l"(q + k / TERMS * (64 * sizeof(T)) + k % TERMS * 16) : "memory");
                } else {
#pragma unroll 1
                    for (uint32_t k = 0; k < kPieces * TERMS; ++k) {
                        const uint8_t* from = q + k / TERMS * (64 * sizeof(T)) + k % TERMS * 16;
                        uint32_t x[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if constexpr (TERMS == 2) x[e] = reinterpret_cast<const uint32_t*>(from)[e];
                            else x[e] = reinterpret_cast<const uint16_t*>(from)[2 * e] | static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(from)[2 * e + 1]) << 16;
                        }
                        sts128(to + (k / TERMS + k % TERMS * kParts) * 16384, x[0], x[1], x[2], x[3]);
                    }
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll 2
            for (uint32_t row = first; row - first % 4 < rows; row += kStride) {  // all of a warp's rows or none
                const uint32_t at = place(min(row, static_cast<uint32_t>(S::kRows) - 1));
                uint32_t word[kPieces * kWords];
#pragma unroll
                for (uint32_t k = 0; k < kPieces * TERMS; ++k) {
                    const uint4 v = lds128(at + (k / TERMS + k % TERMS * kParts) * 16384);
                    word[4 * k] = v.x, word[4 * k + 1] = v.y, word[4 * k + 2] = v.z, word[4 * k + 3] = v.w;
                }
                // the largest finite magnitude: as integers the magnitudes of every type have their order, infinities and NaN above
                uint32_t top = 0;
                if constexpr (TERMS == 2) {
#pragma unroll
                    for (uint32_t k = 0; k < kPieces * kWords; ++k) {
                        const uint32_t m = word[k] & 0x7FFFFFFFu;
                        top = max(top, m < 0x7F800000u ? m : 0u);
                    }
                } else {
                    constexpr uint32_t kInf = std::is_same_v<T, __half> ? 0x7C00u : 0x7F80u;
                    uint32_t top2 = 0;
#pragma unroll
                    for (uint32_t k = 0; k < kPieces * kWords; ++k) top2 = __vmaxu2(top2, word[k] & 0x7FFF7FFFu);
                    top = max(top2 & 0xFFFFu, top2 >> 16);
                    if (top >= kInf) {  // leave them out
                        top = 0;
#pragma unroll
                        for (uint32_t k = 0; k < kPieces * kWords; ++k) {
                            const uint32_t lo = word[k] & 0x7FFFu, hi = word[k] >> 16 & 0x7FFFu;
                            top = max(top, max(lo < kInf ? lo : 0u, hi < kInf ? hi : 0u));
                        }
                    }
                }
#pragma unroll
                for (int d = 4; d != 0; d /= 2) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
                int32_t exponent;
                if constexpr (TERMS == 2) {
                    exponent = static_cast<int32_t>(top >> 23) - 127;
                } else {
                    const uint16_t top16 = static_cast<uint16_t>(top);
                    T largest;
                    __builtin_memcpy(&largest, &top16, 2);
                    exponent = static_cast<int32_t>(__float_as_uint(to_f32(largest)) >> 23) - 127;
                }
                if (row >= rows) continue;
                exponent = max(exponent, -100);
                const float by = c.scale < 0 ? -exp2_int(14 - exponent) : exp2_int(14 - exponent);
                if (l8 == 0) q_unscale[segments & 1][row] = exp2_int(exponent - 14);
#pragma unroll
                for (uint32_t k = 0; k < kPieces; ++k) {
                    uint32_t h[4], rest[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float p, q;
                        if constexpr (TERMS == 2) {
                            p = __uint_as_float(word[8 * k + 2 * e]) * by, q = __uint_as_float(word[8 * k + 2 * e + 1]) * by;
                        } else {
                            T x2[2];
                            __builtin_memcpy(x2, &word[4 * k + e], 4);
                            p = to_f32(x2[0]) * by, q = to_f32(x2[1]) * by;
                        }
                        h[e] = half2_bits(p, q);
                        if constexpr (TERMS == 2) rest[e] = half2_rest(p, q, h[e]);
                    }
                    sts128(at + k * 16384, h[0], h[1], h[2], h[3]);
                    if constexpr (TERMS == 2) sts128(at + (k + kParts) * 16384, rest[0], rest[1], rest[2], rest[3]);
                }
            }
            proxy_fence();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_ready);
            unit_begin = g.unit_end;
            if (!range.reaches(unit_begin) || !next_unit(c, w, u)) break;
        }
    } else if (warp >= 4 && warp < S::kSoftWarp) {
        // ---- conversion ------------------------------------------------------------------------------------------------------------------
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::kConvRegs));
        // A warp makes one slot of every tile: its part of K, or of V (of every other tile where a tile has two slots).
        constexpr uint32_t kEvery = S::kConvWarps / (2 * kParts);
        const uint32_t role = (warp - 4) % (2 * kParts), turn = (warp - 4) / (2 * kParts), part = role % kParts;
        const bool is_v = role >= kParts;
        if (is_v) convert_slots<D, TERMS, true>(c, w, range, cursors[warp - 4], part, turn, kEvery, ring, full, empty, scales, &nan_tiles, alive);
        else convert_slots<D, TERMS, false>(c, w, range, cursors[warp - 4], part, turn, kEvery, ring, full, empty, scales, &nan_tiles, alive);
    } else if (warp >= S::kSoftWarp) {
        // ---- softmax ---------------------------------------------------------------------------------------------------------------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::kSoftRegs));
        constexpr uint32_t kSoft = S::kSoftWarps * 32;
        const uint32_t group = (warp - S::kSoftWarp) / 4, stream = kStreams == 2 ? group : 0, half = kStreams == 2 ? 0 : group;
        const uint32_t quarter = warp % 4, r = stream * 128 + quarter * 32 + lane;  // this thread's row of the unit
        const uint32_t lanes = quarter * 32 << 16, o_at = tmem + lanes + S::kO + stream * D;
        uint32_t uses[2] = {0, 0}, tiles = 0;
        const bool leader = threadIdx.x == S::kSoftWarp * 32;
        for (uint32_t segments = 0;; ++segments) {
            // The warps' way from segment to segment, and so the barriers that they meet at, follows from the lengths alone: also when a wait has run out.
            const Walk& walk = walks[segments & 1];
            if (leader) {
                Walk& next = walks[(segments & 1) ^ 1];
                next = walk;
                next.advance(c, w);
            }
            wait(q_ready, segments & 1);
            const float qs = q_unscale[segments & 1][r];
            const uint32_t j = walk.token(w, min(r, walk.rows - 1));
            const int32_t lo = first_key(walk.u.s, w.window, j), hi = end_key(walk.u.s, c.causal, j);
            // keys that every row of this row tile sees (a tile without rows: of its last row's; nothing of it is kept)
            const int32_t all_lo = first_key(walk.u.s, w.window, walk.token(w, min(stream * 128 + 127, walk.rows - 1)));
            const int32_t all_hi = end_key(walk.u.s, c.causal, walk.token(w, min(stream * 128, walk.rows - 1)));
            const int32_t last_tile = walk.g.hi;
            float ref = -INFINITY, l = 0;
            // This thread's part of the row as far as it is added up outside, four dims at a time, the rows of a warp side by side; (reference, sum of weights) of it.
            constexpr uint32_t kOutside = S::kRows * D / 4;
            auto outside = [&] { return reinterpret_cast<float4*>(w.settled) + blockIdx.x * kOutside + r; };
            auto outside_l = [&] {
                return reinterpret_cast<float2*>(reinterpret_cast<float4*>(w.settled) + gridDim.x * kOutside) + blockIdx.x * kSoft + threadIdx.x - S::kSoftWarp * 32;
            };
            auto fade_outside = [&](float2 of) { return of.x == -INFINITY ? 1.0f : exp2_approx(of.x - ref); };  // without a reference: zero, or NaN
            auto settle = [&](bool first) {  // the accumulators and l go outside; the next products begin anew
                const float2 of = first ? make_float2(-INFINITY, 0) : *outside_l();
                const float fade = fade_outside(of);
#pragma unroll 1
                for (uint32_t d = half * (D / S::kHalves); d < (half + 1) * (D / S::kHalves); d += 32) {
                    uint32_t o[32];
                    tmem_ld32(o_at + d, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        float4* at = outside() + (d + e) / 4 * S::kRows;
                        float4 v = make_float4(0, 0, 0, 0);
                        if (!first) v = *at;
                        v.x = fmaf(v.x, fade, __uint_as_float(o[e])), v.y = fmaf(v.y, fade, __uint_as_float(o[e + 1]));
                        v.z = fmaf(v.z, fade, __uint_as_float(o[e + 2])), v.w = fmaf(v.w, fade, __uint_as_float(o[e + 3]));
                        *at = v;
                    }
                }
                *outside_l() = make_float2(ref, fmaf(of.y, fade, l));
                l = 0;
            };
            const bool any_row = stream * 128 + quarter * 32 < walk.rows;
            uint32_t prev_bar = 0, prev_parity = 0;
            uint32_t b = kStreams == 2 ? stream : 0;
            for (int32_t tile = walk.g.lo;;) {
                const int32_t until = TERMS == 2 ? last_tile : min(last_tile, tile + S::kSettle);
                for (; tile < until; ++tile) {
                    const uint32_t use = b == 0 ? uses[0]++ : uses[1]++, s_at = tmem + lanes + b * S::kBuffer;
                    wait(s_full + 8 * b, use & 1);
                    tmem_after();
                    if (!any_row) {  // nothing of this warp's rows is kept
                        tmem_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(p_ready + 8 * b);
                        prev_bar = pv_done + 8 * b, prev_parity = use & 1;
                        if (kStreams == 1) b ^= 1;
                        ++tiles;
                        continue;
                    }
                    const GroupScale* sc = scales[tiles % kScaleTiles] + half * (S::kKeys / 16);
                    const int32_t t0 = tile * kTile;
                    const bool masked = t0 < all_lo || t0 + kTile > all_hi;
                    const uint32_t from = static_cast<uint32_t>(t0 - lo) + half * S::kKeys, seen = static_cast<uint32_t>(max(hi - lo, 0));  // key e of this thread's: from + e < seen
                    constexpr int kChunks = S::kKeys / 32;
                    // The scores are read again for the weights, 32 at a time: a loop's worth of code for both passes, and of registers.  (Unrolled over 128 keys the
                    // warps waited for instructions: prompts of 360 - 1570 tokens 245 us, with 64 keys 232, with 32 215.)  Two terms of the weights take
                    // the room of scores that are still to be read: there the scores are held.
                    constexpr bool kHold = TERMS == 2;
                    constexpr int kUnrolled = kHold ? kChunks : 1;
                    uint32_t x[kHold ? kChunks : 1][32];
                    auto mask = [&](int q, uint32_t (&v)[32]) __attribute__((always_inline)) {
                        const uint32_t at = from + static_cast<uint32_t>(32 * q);
                        if (__all_sync(0xFFFFFFFFu, at < seen && seen - at >= 32u)) return;  // every row of the warp sees these keys
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (at + static_cast<uint32_t>(e) >= seen) v[e] = 0xFF800000u;  // -inf
                    };
                    if (sc->gap != 0) {  // keys that are not there are zeros: times a NaN or an infinity of q they would count
#pragma unroll 1
                        for (int i = 0; i < S::kKeys / 16; ++i) {
                            if (sc[i].log_v != -INFINITY) continue;
                            uint32_t none[16];
#pragma unroll
                            for (int e = 0; e < 16; ++e) none[e] = 0xFF800000u;
                            tmem_st16(s_at + half * S::kKeys + 16 * i, none);
                        }
                        tmem_wait_st();
                    }
                    if (kHold) {
#pragma unroll
                        for (int q = 0; q < kChunks; ++q) tmem_ld32(s_at + half * S::kKeys + 32 * q, x[kHold ? q : 0]);
                        tmem_wait_ld();
                    }
                    // Missing keys are zeros with log_v = -inf; the factor of a group's scores is not negative: the largest score is the largest exponent.
                    float top = -INFINITY;
#pragma unroll kUnrolled
                    for (int q = 0; q < kChunks; ++q) {
                        uint32_t (&v)[32] = x[kHold ? q : 0];
                        if (!kHold) {
                            tmem_ld32(s_at + half * S::kKeys + 32 * q, v);
                            tmem_wait_ld();
                        }
                        if (masked) mask(q, v);
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const GroupScale s = sc[2 * q + i];
                            float m = fmaxf(__uint_as_float(v[16 * i]), __uint_as_float(v[16 * i + 1]));
#pragma unroll
                            for (int e = 2; e < 16; e += 2) m = fmaxf(fmaxf(m, __uint_as_float(v[16 * i + e])), __uint_as_float(v[16 * i + e + 1]));
                            top = fmaxf(top, m == -INFINITY ? m : fmaf(m, s.k * qs, s.log_v));
                        }
                    }
                    if constexpr (S::kHalves == 2) {  // the warp that has the other keys of these rows; both have read their scores behind this
                        shared_top[tiles & 1][half][r] = top;
                        bar_sync(2 + quarter, 64);
                        top = fmaxf(top, shared_top[tiles & 1][half ^ 1][r]);
                    }
                    const float next = fmaxf(ref, top);
                    const bool first = ref == -INFINITY, grows = !first && next > ref + 8.0f;
                    if (__any_sync(0xFFFFFFFFu, grows)) {
                        // the products into the accumulators so far have to be done; a row without a reference has accumulators of zero, or NaN
                        const float fade = grows ? exp2_approx(ref - next) : 1.0f;
                        wait(prev_bar, prev_parity);
                        tmem_after();
#pragma unroll 1
                        for (int d = half * (D / S::kHalves); d < static_cast<int>(half + 1) * (D / S::kHalves); d += 32) {
                            uint32_t o[32];
                            tmem_ld32(o_at + d, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * fade);
                            tmem_st32(o_at + d, o);
                        }
                        tmem_wait_st();
                        l *= fade;
                    }
                    if (first || grows) ref = next;
                    if constexpr (TERMS == 2) {
                        const int32_t t = tile - walk.g.lo;
                        if (t != 0 && t % S::kSettle == 0) {  // (behind this tile's maximum, which need not wait)
                            wait(prev_bar, prev_parity);
                            tmem_after();
                            settle(t == S::kSettle);
                        }
                    }
                    const float base = ref == -INFINITY ? 0.0f : ref - 6.0f;
#pragma unroll kUnrolled
                    for (int q = 0; q < kChunks; ++q) {
                        uint32_t weights[16], rest[16];
                        uint32_t (&v)[32] = x[kHold ? q : 0];
                        if (!kHold) {
                            tmem_ld32(s_at + half * S::kKeys + 32 * q, v);
                            tmem_wait_ld();
                            if (masked) mask(q, v);
                        }
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const GroupScale s = sc[2 * q + i];
                            // an unseen key's score of -inf times a factor of zero would be NaN; the factor is zero where every score counts for nothing
                            const float by = fmaxf(s.k * qs, 0x1p-126f), add = s.log_v - base;
                            const uint64_t by2 = pair(by, by), add2 = pair(add, add);
                            uint64_t sum = 0;
#pragma unroll
                            for (int e = 0; e < 16; e += 2) {
                                float y0, y1;
                                unpair(fma_pair(pair(__uint_as_float(v[16 * i + e]), __uint_as_float(v[16 * i + e + 1])), by2, add2), y0, y1);
                                y0 = exp2_approx(y0), y1 = exp2_approx(y1);
                                sum = add_pair(sum, pair(y0, y1));
                                weights[8 * i + e / 2] = half2_bits(y0, y1);
                                if constexpr (TERMS == 2) rest[8 * i + e / 2] = half2_rest(y0, y1, weights[8 * i + e / 2]);
                            }
                            float s0, s1;
                            unpair(sum, s0, s1);
                            l = fmaf(s0 + s1, s.inv_v, l);
                        }
                        tmem_st16(s_at + half * (TERMS == 2 ? S::kKeys / 2 : S::kKeys) + 16 * q, weights);  // over scores that have been read
                        if constexpr (TERMS == 2) tmem_st16(s_at + kTile / 2 + half * (S::kKeys / 2) + 16 * q, rest);
                    }
                    tmem_wait_st();
                    tmem_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(p_ready + 8 * b);
                    prev_bar = pv_done + 8 * b, prev_parity = use & 1;
                    if (kStreams == 1) b ^= 1;
                    ++tiles;
                    if (leader) *static_cast<volatile uint32_t*>(&moved) = moved + 1;
                }
                if (__builtin_expect(tile == last_tile, 1)) break;
                if (any_row) {
                    wait(prev_bar, prev_parity);
                    tmem_after();
                    settle(tile - walk.g.lo == S::kSettle);
                }
            }
            wait(prev_bar, prev_parity);
            tmem_after();
            // ---- the segment's rows ------------------------------------------------------------------------------------------------------
            const bool keep = r < walk.rows;
            float fade = 0;
            if (__builtin_expect(any_row && last_tile - walk.g.lo > S::kSettle, 0)) {
                const float2 of = *outside_l();
                fade = fade_outside(of);
                l = fmaf(of.y, fade, l);
            }
            if constexpr (S::kHalves == 2) {
                shared_top[tiles & 1][half][r] = l;
                bar_sync(2 + quarter, 64);
                l += shared_top[tiles & 1][half ^ 1][r];
                bar_sync(2 + quarter, 64);  // read, before the next segment's first tile writes there
            }
            float* slot = walk.g.whole() ? nullptr : partial_slot(w, D, blockIdx.x, walk.g.from_start) + r * D;
            auto out_at = [&](uint32_t row) {
                return reinterpret_cast<T*>(walk.at(c, w, c.out, row));
            };
            T* out = out_at(min(r, walk.rows - 1));
            const float inv = l != 0 ? 1.0f / l : 0.0f;
#pragma unroll 1
            for (int d = half * (D / S::kHalves); d < static_cast<int>(half + 1) * (D / S::kHalves); d += 32) {
                uint32_t o[32];
                tmem_ld32(o_at + d, o);
                tmem_wait_ld();
                if (__builtin_expect(any_row && last_tile - walk.g.lo > S::kSettle, 0)) {
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        const float4 v = outside()[(d + e) / 4 * S::kRows];
                        o[e] = __float_as_uint(fmaf(v.x, fade, __uint_as_float(o[e]))), o[e + 1] = __float_as_uint(fmaf(v.y, fade, __uint_as_float(o[e + 1])));
                        o[e + 2] = __float_as_uint(fmaf(v.z, fade, __uint_as_float(o[e + 2]))), o[e + 3] = __float_as_uint(fmaf(v.w, fade, __uint_as_float(o[e + 3])));
                    }
                }
                if (!keep) continue;
                if (slot != nullptr) {
#pragma unroll
                    for (int e = 0; e < 32; e += 4) *reinterpret_cast<uint4*>(slot + d + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                } else {
                    T y[32];
#pragma unroll
                    for (int e = 0; e < 32; ++e) y[e] = from_f32<T>(__uint_as_float(o[e]) * inv);
                    constexpr int kPer = 16 / sizeof(T);
                    if (c.out.vec) {
#pragma unroll
                        for (int e = 0; e < 32; e += kPer) {
                            uint4 v;
                            __builtin_memcpy(&v, &y[e], 16);
                            *reinterpret_cast<uint4*>(out + d + e) = v;
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) out[d + e] = y[e];
                    }
                }
            }
            if (keep && half == 0 && slot != nullptr) {
                float* ml = partial_slot(w, D, blockIdx.x, walk.g.from_start) + w.rows * D + 2 * r;
                *reinterpret_cast<float2*>(ml) = make_float2(ref, l);
            }
            tmem_before();
            // every warp for what it stored; the conversion is ahead, and what it saw may belong to a segment to come
            if (any_row && __any_sync(0xFFFFFFFFu, *static_cast<volatile uint32_t*>(&nan_tiles) > tiles - static_cast<uint32_t>(last_tile - walk.g.lo))) {
                __syncwarp();
                const uint32_t top = stream * 128 + quarter * 32, dims = D / S::kHalves;
                spread_nan(c, w, walk.u, walk.g, top, min(top + 32, walk.rows), half * dims, dims, lane, 32, [&](uint32_t row, uint32_t d) {
                    if (walk.g.whole()) out_at(row)[d] = from_f32<T>(NAN);
                    else partial_slot(w, D, blockIdx.x, walk.g.from_start)[row * D + d] = NAN;
                });
            }
            if (!walk.g.whole()) {
                const uint32_t c0 = owner(walk.g.unit_begin, range.total, range.ctas), shares = owner(walk.g.unit_end - 1, range.total, range.ctas) - c0 + 1;
                __threadfence();
                bar_sync(1, kSoft);
                if (leader) {
                    const bool last = atomicAdd(w.counters + c0, 1u) == shares - 1;
                    if (last) w.counters[c0] = 0;
                    is_last = last;
                }
                bar_sync(1, kSoft);
                if (is_last != 0) {
                    __threadfence();
                    join_partials<T, D, 4>(c, w, walk, c0, shares, S::kSoftWarp, S::kSoftWarps, joined_ml);
                }
            }
            bar_sync(1, kSoft);  // nobody reads `walk`, `is_last` or `joined_ml` any more; the next walk is there
            if (walks[(segments & 1) ^ 1].more == 0) break;
        }
    }
    if (!alive && lane == 0) report_lost(w.error_word);
    tmem_before();
    __syncthreads();
    if (warp == 1) {
        tmem_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

template <class T, int D>
int launch_tiles_kernel(HaloCudaCtx* ctx, const AttentionCall& c, Work w, cudaStream_t s) {
    using S = TilesShape<D, sizeof(T) == 4 ? 2 : 1>;
    w.rows = S::kRows;
    w.tile = S::kTile;
    w.pad = 3;  // prompts of 364 - 1568 tokens 245 us with 2 or 3, 309 with 1, and 1 % more with 5 than with 3
    w.group = c.group;
    w.group_inverse = static_cast<uint32_t>((0xFFFFFFFFull + c.group) / c.group);
    w.row_tiles = (w.max_rows + S::kRows - 1) / S::kRows;
    w.lanes = 1;
    while (w.lanes < 32 && w.lanes < w.row_tiles) w.lanes *= 2;
    const uint32_t ctas = static_cast<uint32_t>(ctx->prop.multiProcessorCount);
    void* p = nullptr;
    if (int rc = workspace(ctx, 5, ctas * sizeof(uint32_t), s, &p, true)) return rc;
    w.counters = static_cast<uint32_t*>(p);
    const uint64_t partials = partial_bytes(S::kRows, D, ctas);
    if (int rc = workspace(ctx, 6, partials + uint64_t{ctas} * (S::kRows * D * 4 + S::kSoftWarps * 32 * 8), s, &p)) return rc;
    w.partials = static_cast<float*>(p);
    w.settled = w.partials + partials / 4;
    w.error_word = ctx->error_word_dev;
    auto kernel = tiles_kernel<T, D>;
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
    HC_CUDA(cudaLaunchKernelEx(&cfg, kernel, c, w));
    return 0;
}

}  // namespace attn
}  // namespace halo_cuda
