// How a call's work is dealt to a persistent grid.  Internal.
//
// A unit is (sequence, tile of packed rows, kv head): the packed rows of a sequence under one kv head are its (token, query head of the group)
// pairs, token-major, so that a group's heads share every key and value that is fetched.  A unit walks the key tiles that any of its rows sees.  The key tiles
// of all units, one unit after the other and `pad` positions without a tile in front of each (what a unit costs besides its tiles), are cut into gridDim.x
// equal ranges: the CTAs' work is alike whatever the lengths, and only the units at the ends of a range are shared with other CTAs.  An end among
// the positions without a tile counts as the unit's beginning.  Every CTA finds its range by itself from the lengths on the device, so that a captured
// call follows them.
//
// A shared unit's CTAs store (maximum, sum, weighted row) per row in scratch; the last one to arrive (a counter in scratch, left at zero) joins them in
// CTA order, so the result does not depend on who was last.
#pragma once
#include "attention.h"

namespace halo_cuda {
namespace attn {

struct Work {  // what every kernel of a call is told besides the call
    uint32_t rows, tile;          // packed rows of a unit, keys of a tile
    uint32_t pad;                 // what a unit costs besides its tiles, in tiles
    uint32_t group, group_inverse;  // query heads of a kv head; ceil(2^32 / group)
    uint32_t row_tiles;           // of the longest sequence at most
    uint32_t lanes;               // of a warp that look at one sequence when the tiles are counted: a power of two
    int32_t window;               // 0: none
    uint32_t* counters;           // one for each CTA
    float* partials;              // two slots for each CTA
    float* settled;               // what a CTA has taken out of the tensor cores of the segment at hand, 16-byte aligned
    uint32_t* error_word;
    uint32_t min_rows, max_rows;  // packed rows of the sequences that this launch answers for
};

/// The tiles of keys [lo, hi) that rows [r0, r1] of a sequence see between them; at least one, so that every row is answered.
struct Span {
    int32_t lo, hi;
    __device__ __forceinline__ uint32_t tiles() const { return static_cast<uint32_t>(hi - lo); }
};
/// First and last + 1 key that the row of token j sees.
__device__ __forceinline__ int32_t first_key(const Seq& s, int32_t window, uint32_t j) {
    return window == 0 ? 0 : static_cast<int32_t>(max(int64_t{0}, int64_t{s.length} - s.count + j + 1 - window));
}
__device__ __forceinline__ int32_t end_key(const Seq& s, uint32_t causal, uint32_t j) {
    return causal ? max(0, min(s.length, s.length - static_cast<int32_t>(s.count) + static_cast<int32_t>(j) + 1)) : s.length;
}
__device__ __forceinline__ Span span_of(const AttentionCall& c, const Work& w, const Seq& s, uint32_t r0, uint32_t r1) {
    const int32_t lo = first_key(s, w.window, r0 / c.group), hi = end_key(s, c.causal, r1 / c.group), tile = static_cast<int32_t>(w.tile);
    Span x;
    x.lo = lo / tile;
    x.hi = max((hi + tile - 1) / tile, x.lo + 1);
    return x;
}

struct Unit {
    Seq s;
    uint32_t seq, row_tile, head, packed;  // packed: rows of the sequence under one kv head
    Span span;
    __device__ __forceinline__ uint32_t row0(const Work& w) const { return row_tile * w.rows; }
    __device__ __forceinline__ uint32_t rows(const Work& w) const { return min(w.rows, packed - row_tile * w.rows); }
};

__device__ __forceinline__ uint32_t packed_rows(const AttentionCall& c, const Work& w, const Seq& s) {
    const uint32_t n = s.count * c.group;
    return n >= w.min_rows && n <= w.max_rows ? n : 0;
}
__device__ __forceinline__ void set_row_tile(const AttentionCall& c, const Work& w, Unit& u, uint32_t row_tile) {
    u.row_tile = row_tile;
    const uint32_t r0 = row_tile * w.rows;
    u.span = span_of(c, w, u.s, r0, min(r0 + w.rows, u.packed) - 1);
}
/// The unit behind u, past sequences without rows here; false at the end.
__device__ __forceinline__ bool next_unit(const AttentionCall& c, const Work& w, Unit& u) {
    if (++u.head < c.cache.n_kv) return true;
    u.head = 0;
    if ((u.row_tile + 1) * w.rows < u.packed) {
        set_row_tile(c, w, u, u.row_tile + 1);
        return true;
    }
    while (++u.seq < c.cache.n_seq) {
        u.s = sequence(c.rows, c.cache, u.seq);
        u.packed = packed_rows(c, w, u.s);
        if (u.packed != 0) {
            set_row_tile(c, w, u, 0);
            return true;
        }
    }
    return false;
}

/// Quotients of 64-bit numbers that are small as a rule: a 64-bit division is a hundred dependent instructions.
__device__ __forceinline__ uint64_t quotient(uint64_t a, uint64_t b) {
    return a >> 32 == 0 && b >> 32 == 0 ? static_cast<uint32_t>(a) / static_cast<uint32_t>(b) : a / b;
}
/// The CTA that has position x of `total` (range b of n is [total * b / n, total * (b + 1) / n)).
__device__ __forceinline__ uint32_t owner(uint64_t x, uint64_t total, uint32_t n) { return static_cast<uint32_t>(quotient((x + 1) * n - 1, total)); }

struct Range {
    uint64_t begin, end, total;  // this CTA's positions
    uint32_t ctas, pad;          // CTAs that have a range
    uint64_t unit_begin;         // position that the first unit begins at
    Unit unit;                   // of position `begin`
    __device__ __forceinline__ bool reaches(uint64_t unit) const { return end > unit + pad; }  // a tile of the unit that begins at this position
};

struct PlanSmem {
    uint64_t warp_sum[32];
    uint64_t before;  // tiles in front of the sequence that was found
    uint32_t seq;
};

/// The CTA's positions out of `total`; false if it has none.
__device__ __forceinline__ bool cut_range(const Work& w, uint64_t total, Range* out) {
    out->total = total;
    if (total == 0) return false;
    const uint32_t ctas = static_cast<uint32_t>(min(uint64_t{gridDim.x}, total));
    if (blockIdx.x >= ctas) return false;
    out->ctas = ctas;
    out->pad = w.pad;
    out->begin = quotient(total * blockIdx.x, ctas);
    out->end = quotient(total * (blockIdx.x + 1), ctas);
    return true;
}

/// find_range where no sequence has more than one row tile: every warp for itself, a lane to a sequence, without a barrier.
__device__ inline bool find_range_by_warps(const AttentionCall& c, const Work& w, Range* out) {
    const uint32_t lane = threadIdx.x % 32, n_seq = c.cache.n_seq;
    uint64_t total = 0, n = 0, upto = 0;
    auto count = [&](uint32_t i) {  // this lane's sequence's positions, and the sum up to it
        n = 0;
        if (i < n_seq) {
            const Seq s = sequence(c.rows, c.cache, i);
            const uint32_t packed = packed_rows(c, w, s);
            if (packed != 0) n = uint64_t{span_of(c, w, s, 0, packed - 1).tiles() + w.pad} * c.cache.n_kv;
        }
        upto = n;
        for (uint32_t d = 1; d < 32; d *= 2) {
            const uint64_t y = __shfl_up_sync(0xFFFFFFFFu, upto, d);
            if (lane >= d) upto += y;
        }
    };
    for (uint32_t base = 0; base < n_seq; base += 32) {
        count(base + lane);
        total += __shfl_sync(0xFFFFFFFFu, upto, 31);
    }
    if (!cut_range(w, total, out)) return false;
    uint64_t before = 0;
    for (uint32_t base = 0; base < n_seq; base += 32) {
        if (n_seq > 32) count(base + lane);
        const uint32_t hit = __ballot_sync(0xFFFFFFFFu, out->begin < before + upto);
        if (hit != 0) {
            const uint32_t l = __ffs(hit) - 1;
            before += __shfl_sync(0xFFFFFFFFu, upto - n, l);
            Unit& u = out->unit;
            u.seq = base + l;
            u.s = sequence(c.rows, c.cache, u.seq);
            u.packed = packed_rows(c, w, u.s);
            set_row_tile(c, w, u, 0);
            const uint64_t at = out->begin - before, length = u.span.tiles() + w.pad;
            u.head = static_cast<uint32_t>(quotient(at, length));
            out->unit_begin = before + u.head * length;
            break;
        }
        before += __shfl_sync(0xFFFFFFFFu, upto, 31);
    }
    return out->reaches(out->unit_begin);
}

/// All threads of the CTA (a multiple of a warp).  `lanes` lanes share a sequence; a pass over the sequences sums their tiles, another finds
/// the one that this CTA's range begins in (one pass does both where the CTA sees all sequences at once).
__device__ inline bool find_range(const AttentionCall& c, const Work& w, PlanSmem& sm, Range* out) {
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = blockDim.x / 32;
    const uint32_t per_pass = blockDim.x / w.lanes, sub = threadIdx.x % w.lanes, n_seq = c.cache.n_seq;
    if (w.row_tiles == 1) return find_range_by_warps(c, w, out);
    auto tiles_of = [&](uint32_t i) {  // all lanes of the group get the sum
        uint64_t n = 0;
        if (i < n_seq) {
            const Seq s = sequence(c.rows, c.cache, i);
            const uint32_t packed = packed_rows(c, w, s);
            for (uint32_t r0 = sub * w.rows; r0 < packed; r0 += w.lanes * w.rows) n += span_of(c, w, s, r0, min(r0 + w.rows, packed) - 1).tiles() + w.pad;
        }
        for (uint32_t d = w.lanes / 2; d != 0; d /= 2) n += __shfl_xor_sync(0xFFFFFFFFu, n, d);
        return n * c.cache.n_kv;
    };
    // inclusive sum over the groups of the CTA; *all is the CTA's
    auto scan = [&](uint64_t n, uint64_t* all) {
        uint64_t x = sub == 0 ? n : 0;
        for (uint32_t d = 1; d < 32; d *= 2) {
            const uint64_t y = __shfl_up_sync(0xFFFFFFFFu, x, d);
            if (lane >= d) x += y;
        }
        __syncthreads();
        if (lane == 31) sm.warp_sum[warp] = x;
        __syncthreads();
        uint64_t sum = 0;
        for (uint32_t i = 0; i < warps; ++i) {
            if (i == warp) x += sum;
            sum += sm.warp_sum[i];
        }
        *all = sum;
        return x;
    };
    uint64_t total = 0, n = 0, upto = 0;
    for (uint32_t base = 0; base < n_seq; base += per_pass) {
        uint64_t all;
        n = tiles_of(base + threadIdx.x / w.lanes);
        upto = scan(n, &all);
        total += all;
    }
    if (!cut_range(w, total, out)) return false;
    uint64_t before = 0;
    for (uint32_t base = 0; base < n_seq; base += per_pass) {
        uint64_t all = total;
        if (n_seq > per_pass) {
            n = tiles_of(base + threadIdx.x / w.lanes);
            upto = scan(n, &all);
        }
        if (sub == 0 && out->begin >= before + upto - n && out->begin < before + upto) {
            sm.before = before + upto - n;
            sm.seq = base + threadIdx.x / w.lanes;
        }
        before += all;
        if (out->begin < before) break;
    }
    __syncthreads();
    Unit& u = out->unit;
    u.seq = sm.seq;
    u.s = sequence(c.rows, c.cache, u.seq);
    u.packed = packed_rows(c, w, u.s);
    // within the sequence: the tiles of 32 row tiles at a time, every warp for itself
    uint64_t at = out->begin - sm.before, front = 0;
    const uint32_t row_tiles = (u.packed + w.rows - 1) / w.rows;
    uint32_t row_tile = 0;
    for (uint32_t base = 0; base < row_tiles; base += 32) {
        const uint32_t r = base + lane;
        uint64_t x = 0;
        if (r < row_tiles) x = uint64_t{span_of(c, w, u.s, r * w.rows, min((r + 1) * w.rows, u.packed) - 1).tiles() + w.pad} * c.cache.n_kv;
        const uint64_t mine = x;
        for (uint32_t d = 1; d < 32; d *= 2) {
            const uint64_t y = __shfl_up_sync(0xFFFFFFFFu, x, d);
            if (lane >= d) x += y;
        }
        const uint32_t hit = __ballot_sync(0xFFFFFFFFu, at < front + x);
        if (hit != 0) {
            const uint32_t l = __ffs(hit) - 1;
            row_tile = base + l;
            front += __shfl_sync(0xFFFFFFFFu, x - mine, l);
            break;
        }
        front += __shfl_sync(0xFFFFFFFFu, x, 31);
    }
    set_row_tile(c, w, u, row_tile);
    at -= front;
    u.head = static_cast<uint32_t>(quotient(at, u.span.tiles() + w.pad));
    out->unit_begin = out->begin - (at - uint64_t{u.head} * (u.span.tiles() + w.pad));
    return out->reaches(out->unit_begin);
}

/// A stretch of a unit's tiles that one CTA walks.
struct Segment {
    int32_t lo, hi;            // tiles of keys
    uint64_t unit_begin, unit_end;  // positions of the unit's tiles
    bool from_start, to_end;
    __device__ __forceinline__ bool whole() const { return from_start && to_end; }
};
__device__ __forceinline__ Segment segment(const Range& r, const Unit& u, uint64_t unit_begin) {
    Segment g;
    const uint64_t first = unit_begin + r.pad;  // position of the unit's first tile
    g.unit_begin = first;
    g.unit_end = first + u.span.tiles();
    g.from_start = first >= r.begin;
    g.to_end = g.unit_end <= r.end;
    g.lo = u.span.lo + (g.from_start ? 0 : static_cast<int32_t>(r.begin - first));
    g.hi = g.to_end ? u.span.hi : u.span.lo + static_cast<int32_t>(r.end - first);
    return g;
}

/// Where a CTA's consumers are: in shared memory, so that the walk over the tiles has the registers.
struct Walk {
    Range range;
    Unit u;
    Segment g;
    uint32_t rows, r0;        // of the unit
    uint32_t token0, behind;  // row 0's token, and which of the token's heads it is
    uint32_t more;
    __device__ void enter(const AttentionCall& c, const Work& w, uint64_t unit_begin) {
        g = segment(range, u, unit_begin);
        rows = u.rows(w), r0 = u.row0(w);
        token0 = r0 / c.group, behind = r0 - token0 * c.group;
        more = 1;
    }
    __device__ void advance(const AttentionCall& c, const Work& w) {
        more = range.reaches(g.unit_end) && next_unit(c, w, u);
        if (more) enter(c, w, g.unit_end);
    }
    /// The token of row r < 256 of the unit (group_inverse = ceil(2^32 / group): exact while (group + 256) * group < 2^32).
    __device__ __forceinline__ uint32_t token(const Work& w, uint32_t r) const { return token0 + (w.group == 1 ? r : __umulhi(behind + r, w.group_inverse)); }
    /// Where row r's head begins.
    __device__ __forceinline__ uint8_t* at(const AttentionCall& c, const Work& w, const Heads& x, uint32_t r) const {
        const uint32_t t = token(w, r), h = r0 + r - t * w.group + u.head * w.group;
        return x.p + uint64_t{u.s.row0 + t} * x.token_stride + uint64_t{h} * x.head_stride;
    }
};

/// Where a CTA's share of a unit that it has not alone lies: [row][dim] weighted rows, then (maximum, sum) of every row.
__device__ __forceinline__ float* partial_slot(const Work& w, uint32_t dim, uint32_t cta, bool from_start) {
    return w.partials + uint64_t{2 * cta + (from_start ? 1u : 0u)} * w.rows * (dim + 2);
}
inline uint64_t partial_bytes(uint32_t rows, uint32_t dim, uint32_t ctas) { return uint64_t{2} * ctas * rows * (dim + 2) * 4; }

// ---- barriers and copies ---------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count)); }
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
constexpr uint32_t kWaitSpins = 1u << 18;  // of a try_wait that sleeps in hardware: seconds
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity) {  // for what one step of another warp brings
    for (uint32_t i = 0; i < kWaitSpins; ++i) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(bar), "r"(parity)
            : "memory");
        if (ok) return true;
    }
    return false;
}
/// For what more than a step may come in front of (a segment takes as long as its context): given up once `moved`, which the warps waited for count up as they
/// go on, has stood still for as long as a step may take.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, const volatile uint32_t* moved) {
    uint32_t before = ~0u;
    while (!mbar_wait(bar, parity)) {
        const uint32_t now = *moved;
        if (now == before) return false;
        before = now;
    }
    return true;
}
/// A wait has run out: the host finds the context lost at its next synchronisation.  A context without pinned host memory has no word for it.
__device__ __forceinline__ void report_lost(uint32_t* error_word) {
    if (error_word != nullptr) atomicOr(error_word, 1u);
}
__device__ __forceinline__ void tma_3d(uint32_t dst, const void* map, int32_t x, int32_t y, int32_t z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(map),
                 "r"(x), "r"(y), "r"(z), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void bar_sync(uint32_t id, uint32_t threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

}  // namespace attn
}  // namespace halo_cuda
