// Entry points of halo_cuda_attention.h: validation (before the context is looked at, so that a malformed call is told apart without a device) and
// the host arithmetic of the rotary frequencies.
#include <cmath>
#include <cstring>

#include "attention.h"
#include "rope.h"

namespace halo_cuda {
namespace attn {
namespace {

using u64 = unsigned long long;

uint32_t type_size(uint32_t type) {
    switch (type) {
        case HALO_CUDA_T_F32: return 4;
        case HALO_CUDA_T_F16:
        case HALO_CUDA_T_BF16: return 2;
        default: return 0;
    }
}

/// A block of device memory an operand lies in, as repeating rows: `n` of them `pitch` apart, of which `row` bytes belong to it.
struct Span {
    const char* name;
    uintptr_t p;
    uint64_t n, pitch, row;  // row <= pitch unless n == 1
    uint64_t bytes() const { return n == 0 || row == 0 ? 0 : (n - 1) * pitch + row; }
};

/// Whether two operands share a byte.  Operands that are columns of the same rows (a fused q|k|v product) do not, although their ranges interleave.
bool overlap(const Span& a, const Span& b) {
    if (a.bytes() == 0 || b.bytes() == 0 || a.p >= b.p + b.bytes() || b.p >= a.p + a.bytes()) return false;
    if (a.pitch != b.pitch || a.n == 1 || b.n == 1) return true;
    const uint64_t d = a.p <= b.p ? (b.p - a.p) % a.pitch : (a.pitch - (a.p - b.p) % a.pitch) % a.pitch;  // b's rows begin d behind a's
    return d < a.row || d + b.row > a.pitch;
}

int no_overlap(const Span& a, const Span& b, const char* op) {
    return overlap(a, b) ? fail(HALO_CUDA_E_KERNEL, "%s: output %s overlaps operand %s", op, a.name, b.name) : 0;
}

/// Resolves and checks rows of heads; *span is what they occupy.
int take_heads(const HaloCudaHeads& h, const char* op, const char* name, uint32_t n_tokens, uint32_t n_heads, uint32_t head_dim, uint32_t size, Heads* out, Span* span) {
    const uint64_t head = uint64_t{head_dim} * size;
    out->p = static_cast<uint8_t*>(h.p);
    out->head_stride = h.head_stride != 0 ? h.head_stride : head;
    if (n_heads > 1 && out->head_stride < head) return fail(HALO_CUDA_E_KERNEL, "%s: operand %s head stride %llu < head bytes %llu", op, name, (u64)out->head_stride, (u64)head);
    if (n_heads > 1 && out->head_stride > (UINT64_MAX >> 1) / n_heads) return fail(HALO_CUDA_E_KERNEL, "%s: operand %s size overflows", op, name);
    const uint64_t row = n_heads == 0 ? 0 : (n_heads - 1) * out->head_stride + head;
    out->token_stride = h.token_stride != 0 ? h.token_stride : n_heads * out->head_stride;
    if (n_tokens > 1 && out->token_stride < row)
        return fail(HALO_CUDA_E_KERNEL, "%s: operand %s token stride %llu < row bytes %llu", op, name, (u64)out->token_stride, (u64)row);
    if (n_tokens > 1 && out->token_stride > (UINT64_MAX >> 1) / n_tokens) return fail(HALO_CUDA_E_KERNEL, "%s: operand %s size overflows", op, name);
    const uintptr_t p = reinterpret_cast<uintptr_t>(h.p);
    *span = Span{name, p, n_tokens, out->token_stride, row};
    if (span->bytes() != 0 && h.p == nullptr) return fail(HALO_CUDA_E_KERNEL, "%s: operand %s is empty", op, name);
    if (p > UINTPTR_MAX - span->bytes()) return fail(HALO_CUDA_E_KERNEL, "%s: operand %s size overflows", op, name);
    if (p % size != 0 || out->head_stride % size != 0 || out->token_stride % size != 0)
        return fail(HALO_CUDA_E_KERNEL, "%s: operand %s is not %u-byte aligned", op, name, size);
    out->vec = p % 16 == 0 && out->head_stride % 16 == 0 && out->token_stride % 16 == 0;
    return 0;
}

struct CacheSpans {
    Span k, v, k_scale, v_scale, table;
};

int take_cache(const HaloCudaKvCache& c, const char* op, Cache* out, CacheSpans* spans) {
    if (c.type != HALO_CUDA_KV_E4M3) return fail(HALO_CUDA_E_UNSUPPORTED, "%s: no cache of type id %u", op, c.type);
    if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256) return fail(HALO_CUDA_E_UNSUPPORTED, "%s: heads of %u elements (64, 128 or 256)", op, c.head_dim);
    if (c.page_tokens != 16 && c.page_tokens != 32 && c.page_tokens != 64 && c.page_tokens != 128)
        return fail(HALO_CUDA_E_UNSUPPORTED, "%s: pages of %u tokens (16, 32, 64 or 128)", op, c.page_tokens);
    if (c.n_kv == 0 || c.n_kv > 65535u) return fail(HALO_CUDA_E_KERNEL, "%s: %u kv heads", op, c.n_kv);
    if (c.n_pages > 0x7FFFFFFFu) return fail(HALO_CUDA_E_KERNEL, "%s: %u pages", op, c.n_pages);
    if (c.n_seq > 0x7FFFFFFFu) return fail(HALO_CUDA_E_KERNEL, "%s: %u sequences", op, c.n_seq);
    if (uint64_t{c.max_pages} * c.page_tokens > (1ull << 30)) return fail(HALO_CUDA_E_KERNEL, "%s: sequences of %u pages of %u tokens", op, c.max_pages, c.page_tokens);
    const uint64_t page = uint64_t{c.n_kv} * c.page_tokens * c.head_dim;
    *out = Cache{static_cast<uint8_t*>(c.k), static_cast<uint8_t*>(c.v), c.k_scale, c.v_scale, c.table, c.page_stride != 0 ? c.page_stride : page,
                 c.scale_stride != 0 ? c.scale_stride : c.n_kv, c.table_stride != 0 ? c.table_stride : uint64_t{c.max_pages} * 4,
                 c.n_pages, c.n_kv, c.head_dim, c.page_tokens, static_cast<uint32_t>(__builtin_ctz(c.page_tokens)), c.max_pages, c.n_seq};
    if (c.n_pages > 1 && out->page_stride < page) return fail(HALO_CUDA_E_KERNEL, "%s: page stride %llu < page bytes %llu", op, (u64)out->page_stride, (u64)page);
    if (out->page_stride >= (1ull << 40)) return fail(HALO_CUDA_E_KERNEL, "%s: page stride %llu", op, (u64)out->page_stride);  // what the copy engine takes
    if (c.n_pages > 1 && out->scale_stride < c.n_kv) return fail(HALO_CUDA_E_KERNEL, "%s: scale stride %llu < %u heads", op, (u64)out->scale_stride, c.n_kv);
    if (out->scale_stride >= (1ull << 32)) return fail(HALO_CUDA_E_KERNEL, "%s: scale stride %llu", op, (u64)out->scale_stride);
    if (c.n_seq > 1 && out->table_stride < uint64_t{c.max_pages} * 4) return fail(HALO_CUDA_E_KERNEL, "%s: table stride %llu < row bytes", op, (u64)out->table_stride);
    if (out->table_stride >= (1ull << 32)) return fail(HALO_CUDA_E_KERNEL, "%s: table stride %llu", op, (u64)out->table_stride);
    auto at = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
    if (at(c.k) % 16 != 0 || at(c.v) % 16 != 0 || out->page_stride % 16 != 0) return fail(HALO_CUDA_E_KERNEL, "%s: the cache's pages are not 16-byte aligned", op);
    if (at(c.table) % 4 != 0 || out->table_stride % 4 != 0) return fail(HALO_CUDA_E_KERNEL, "%s: the page table is not 4-byte aligned", op);
    if (c.n_pages != 0 && (c.k == nullptr || c.v == nullptr || c.k_scale == nullptr || c.v_scale == nullptr))
        return fail(HALO_CUDA_E_KERNEL, "%s: a pool or its scales are missing", op);
    if (c.n_seq != 0 && c.max_pages != 0 && c.table == nullptr) return fail(HALO_CUDA_E_KERNEL, "%s: the page table is missing", op);
    *spans = CacheSpans{{"k cache", at(c.k), c.n_pages, out->page_stride, page},
                        {"v cache", at(c.v), c.n_pages, out->page_stride, page},
                        {"k scales", at(c.k_scale), c.n_pages, out->scale_stride, c.n_kv},
                        {"v scales", at(c.v_scale), c.n_pages, out->scale_stride, c.n_kv},
                        {"page table", at(c.table), c.n_seq, out->table_stride, uint64_t{c.max_pages} * 4}};
    return 0;
}

int take_rows(const HaloCudaKvRows& r, const char* op, uint32_t n_seq, Rows* out) {
    *out = Rows{r.start, r.length, r.n_tokens, r.max_tokens};
    if (n_seq == 0 || r.n_tokens == 0 || r.max_tokens == 0) return 0;
    if (r.n_tokens > 0x7FFFFFFFu || r.max_tokens > 0x7FFFFFFFu) return fail(HALO_CUDA_E_KERNEL, "%s: %u rows, %u of one sequence", op, r.n_tokens, r.max_tokens);
    if (r.length == nullptr) return fail(HALO_CUDA_E_KERNEL, "%s: the sequences' lengths are missing", op);
    if (reinterpret_cast<uintptr_t>(r.length) % 4 != 0 || reinterpret_cast<uintptr_t>(r.start) % 4 != 0)
        return fail(HALO_CUDA_E_KERNEL, "%s: starts / lengths are not 4-byte aligned", op);
    if (r.start == nullptr && uint64_t{n_seq} * r.max_tokens != r.n_tokens)
        return fail(HALO_CUDA_E_KERNEL, "%s: %u rows are not %u for each of %u sequences", op, r.n_tokens, r.max_tokens, n_seq);
    return 0;
}

/// The arrays that tell whose the rows are; an output that covered one of them would change the call under way.
int keeps_control(const Span& out, const Rows& r, uint32_t n_seq, const uint32_t* status, const char* op) {
    const Span control[3] = {{"start", reinterpret_cast<uintptr_t>(r.start), 1, 0, r.start != nullptr ? (uint64_t{n_seq} + 1) * 4 : 0},
                             {"length", reinterpret_cast<uintptr_t>(r.length), 1, 0, uint64_t{n_seq} * 4},
                             {"status", reinterpret_cast<uintptr_t>(status), 1, 0, status != nullptr ? 4u : 0u}};
    for (const Span& c : control)
        if (int rc = no_overlap(out, c, op)) return rc;
    return 0;
}

int take_write(const HaloCudaKvWrite* a, WriteCall* c) {
    constexpr const char* op = "KV_WRITE";
    if (a == nullptr) return fail(HALO_CUDA_E_API, "%s: null argument struct", op);
    const uint32_t size = type_size(a->type);
    if (size == 0) return fail(HALO_CUDA_E_UNSUPPORTED, "%s: no activations of type id %u", op, a->type);
    CacheSpans cs;
    Span k, v;
    c->type = a->type;
    c->status = a->status;
    if (int rc = take_cache(a->cache, op, &c->cache, &cs)) return rc;
    if (int rc = take_rows(a->rows, op, a->cache.n_seq, &c->rows)) return rc;
    if (int rc = take_heads(a->k, op, "k", a->rows.n_tokens, a->cache.n_kv, a->cache.head_dim, size, &c->k, &k)) return rc;
    if (int rc = take_heads(a->v, op, "v", a->rows.n_tokens, a->cache.n_kv, a->cache.head_dim, size, &c->v, &v)) return rc;
    if (reinterpret_cast<uintptr_t>(a->status) % 4 != 0) return fail(HALO_CUDA_E_KERNEL, "%s: status is not 4-byte aligned", op);
    const Span outs[4] = {cs.k, cs.v, cs.k_scale, cs.v_scale};
    for (int i = 0; i < 4; ++i) {
        const Span& o = outs[i];
        for (const Span* in : {&k, &v, &cs.table})
            if (int rc = no_overlap(o, *in, op)) return rc;
        for (int j = i + 1; j < 4; ++j)
            if (int rc = no_overlap(o, outs[j], op)) return rc;
        if (int rc = keeps_control(o, c->rows, a->cache.n_seq, a->status, op)) return rc;
    }
    return 0;
}

int take_attention(const HaloCudaAttention* a, AttentionCall* c) {
    constexpr const char* op = "ATTENTION";
    if (a == nullptr) return fail(HALO_CUDA_E_API, "%s: null argument struct", op);
    const uint32_t size = type_size(a->type);
    if (size == 0) return fail(HALO_CUDA_E_UNSUPPORTED, "%s: no activations of type id %u", op, a->type);
    CacheSpans cs;
    Span q, out;
    if (int rc = take_cache(a->cache, op, &c->cache, &cs)) return rc;
    if (int rc = take_rows(a->rows, op, a->cache.n_seq, &c->rows)) return rc;
    // A block steps past sequences without rows one by one, and its warps wait 1.3 s for one another: tens of millions would be too many.
    if (a->cache.n_seq > (1u << 20)) return fail(HALO_CUDA_E_UNSUPPORTED, "%s: %u sequences", op, a->cache.n_seq);
    if (a->n_q == 0 || a->n_q > 32768u || a->n_q % a->cache.n_kv != 0) return fail(HALO_CUDA_E_KERNEL, "%s: %u query heads over %u kv heads", op, a->n_q, a->cache.n_kv);
    if (a->causal > 1) return fail(HALO_CUDA_E_API, "%s: causal is 0 or 1", op);
    if (a->window != 0 && a->causal == 0) return fail(HALO_CUDA_E_UNSUPPORTED, "%s: a window without a causal mask", op);
    if (!std::isfinite(a->scale)) return fail(HALO_CUDA_E_KERNEL, "%s: scale is not finite", op);
    c->type = a->type;
    c->n_q = a->n_q;
    c->group = a->n_q / a->cache.n_kv;
    c->causal = a->causal;
    c->window = a->window;
    c->scale = a->scale;
    c->status = a->status;
    if (uint64_t{c->group} * a->rows.max_tokens > 0x7FFFFFFFu) return fail(HALO_CUDA_E_KERNEL, "%s: %u rows of %u heads for one kv head", op, a->rows.max_tokens, c->group);
    if (int rc = take_heads(a->q, op, "q", a->rows.n_tokens, a->n_q, a->cache.head_dim, size, &c->q, &q)) return rc;
    if (int rc = take_heads(a->out, op, "out", a->rows.n_tokens, a->n_q, a->cache.head_dim, size, &c->out, &out)) return rc;
    if (reinterpret_cast<uintptr_t>(a->status) % 4 != 0) return fail(HALO_CUDA_E_KERNEL, "%s: status is not 4-byte aligned", op);
    for (const Span* in : {&q, &cs.k, &cs.v, &cs.k_scale, &cs.v_scale, &cs.table})
        if (int rc = no_overlap(out, *in, op)) return rc;
    return keeps_control(out, c->rows, a->cache.n_seq, a->status, op);
}

int take_rope(const HaloCudaRope* a, RopeCall* c) {
    constexpr const char* op = "PARTIAL_ROPE";
    if (a == nullptr) return fail(HALO_CUDA_E_API, "%s: null argument struct", op);
    const uint32_t size = type_size(a->type);
    if (size == 0) return fail(HALO_CUDA_E_UNSUPPORTED, "%s: no activations of type id %u", op, a->type);
    if (a->freqs == nullptr) return fail(HALO_CUDA_E_API, "%s: no frequencies", op);
    if (a->interleaved > 1) return fail(HALO_CUDA_E_API, "%s: interleaved is 0 or 1", op);
    const uint32_t pairs = a->freqs->n_pairs;
    if (pairs == 0 || pairs > HALO_CUDA_ROPE_MAX_PAIRS) return fail(HALO_CUDA_E_KERNEL, "%s: %u pairs", op, pairs);
    if (a->head_dim < 2 * pairs || a->head_dim > 1024) return fail(HALO_CUDA_E_KERNEL, "%s: %u pairs of heads of %u elements", op, pairs, a->head_dim);
    if (a->n_tokens > 0x7FFFFFFFu || a->n_q > 65535u || a->n_kv > 65535u) return fail(HALO_CUDA_E_KERNEL, "%s: %u rows of %u + %u heads", op, a->n_tokens, a->n_q, a->n_kv);
    if (!std::isfinite(a->freqs->magnitude)) return fail(HALO_CUDA_E_KERNEL, "%s: magnitude is not finite", op);
    *c = RopeCall{a->type, a->interleaved, a->positions, {}, {}, {}, {}, a->n_tokens, a->n_q, a->n_kv, a->head_dim};
    c->freqs = a->freqs;
    Span in[2], out[2];
    if (int rc = take_heads(a->q, op, "q", a->n_tokens, a->n_q, a->head_dim, size, &c->q, &in[0])) return rc;
    if (int rc = take_heads(a->q_out, op, "q_out", a->n_tokens, a->n_q, a->head_dim, size, &c->q_out, &out[0])) return rc;
    if (int rc = take_heads(a->k, op, "k", a->n_tokens, a->n_kv, a->head_dim, size, &c->k, &in[1])) return rc;
    if (int rc = take_heads(a->k_out, op, "k_out", a->n_tokens, a->n_kv, a->head_dim, size, &c->k_out, &out[1])) return rc;
    if (a->n_tokens != 0 && a->positions == nullptr) return fail(HALO_CUDA_E_KERNEL, "%s: operand positions is empty", op);
    if (reinterpret_cast<uintptr_t>(a->positions) % 4 != 0) return fail(HALO_CUDA_E_KERNEL, "%s: positions is not 4-byte aligned", op);
    const Span pos{"positions", reinterpret_cast<uintptr_t>(a->positions), 1, 0, uint64_t{a->n_tokens} * 4};
    const Heads* heads[2][2] = {{&c->q, &c->q_out}, {&c->k, &c->k_out}};
    for (int i = 0; i < 2; ++i) {
        const Heads &x = *heads[i][0], &y = *heads[i][1];
        const bool in_place = x.p == y.p && x.token_stride == y.token_stride && x.head_stride == y.head_stride;
        if (!in_place)
            if (int rc = no_overlap(out[i], in[i], op)) return rc;
        if (int rc = no_overlap(out[i], in[1 - i], op)) return rc;
        if (int rc = no_overlap(out[i], pos, op)) return rc;
    }
    return no_overlap(out[0], out[1], op);
}

int take_freqs(uint32_t rot_dim, double base, const HaloCudaRopeScaling* s, HaloCudaRopeFreqs* out) {
    constexpr const char* op = "PARTIAL_ROPE";
    if (out == nullptr) return fail(HALO_CUDA_E_API, "%s: null frequencies", op);
    if (rot_dim == 0 || rot_dim % 2 != 0 || rot_dim > 2 * HALO_CUDA_ROPE_MAX_PAIRS) return fail(HALO_CUDA_E_KERNEL, "%s: %u rotated elements", op, rot_dim);
    if (!(base > 0) || !std::isfinite(base)) return fail(HALO_CUDA_E_KERNEL, "%s: base %g", op, base);
    const uint32_t kind = s != nullptr ? s->kind : HALO_CUDA_ROPE_NONE;
    if (kind > HALO_CUDA_ROPE_FACTORS) return fail(HALO_CUDA_E_UNSUPPORTED, "%s: no scaling of kind %u", op, kind);
    const bool limits = kind == HALO_CUDA_ROPE_RAMP || kind == HALO_CUDA_ROPE_BANDS;
    if (kind >= HALO_CUDA_ROPE_LINEAR && kind <= HALO_CUDA_ROPE_BANDS && (!(s->factor > 0) || !std::isfinite(s->factor)))
        return fail(HALO_CUDA_E_KERNEL, "%s: factor %g", op, s->factor);
    if (kind == HALO_CUDA_ROPE_RAMP && (s->factor < 1 || base <= 1)) return fail(HALO_CUDA_E_KERNEL, "%s: factor %g, base %g", op, s->factor, base);
    if (kind == HALO_CUDA_ROPE_BASE && rot_dim == 2) return fail(HALO_CUDA_E_KERNEL, "%s: one pair has no base to scale", op);
    if (limits && (!(s->original_context > 0) || !std::isfinite(s->original_context) || !(s->slow > 0) || !(s->fast > s->slow) || !std::isfinite(s->fast)))
        return fail(HALO_CUDA_E_KERNEL, "%s: original context %g, limits %g and %g", op, s->original_context, s->fast, s->slow);
    if (kind == HALO_CUDA_ROPE_FACTORS && s->pair_factors == nullptr) return fail(HALO_CUDA_E_API, "%s: no pair factors", op);
    if (s != nullptr && !(s->magnitude >= 0 && std::isfinite(s->magnitude))) return fail(HALO_CUDA_E_KERNEL, "%s: magnitude %g", op, s->magnitude);

    constexpr long double kTurn = 6.283185307179586476925286766559005768L;
    HaloCudaRopeFreqs f{};
    f.n_pairs = rot_dim / 2;
    long double magnitude = kind == HALO_CUDA_ROPE_RAMP ? 0.1L * std::log(static_cast<long double>(s->factor)) + 1 : 1;
    if (s != nullptr && s->magnitude != 0) magnitude = s->magnitude;
    f.magnitude = static_cast<float>(magnitude);
    long double b = base;
    if (kind == HALO_CUDA_ROPE_BASE) b *= std::pow(static_cast<long double>(s->factor), static_cast<long double>(rot_dim) / (rot_dim - 2));
    long double lo = 0, hi = 0;  // RAMP: the pairs that turn `fast` and `slow` times over the original context
    if (kind == HALO_CUDA_ROPE_RAMP) {
        auto pair_of = [&](double turns) { return rot_dim * std::log(s->original_context / (turns * kTurn)) / (2 * std::log(static_cast<long double>(base))); };
        lo = std::fmax(std::floor(pair_of(s->fast)), 0.0L);
        hi = std::fmin(std::ceil(pair_of(s->slow)), rot_dim - 1.0L);
    }
    for (uint32_t j = 0; j < f.n_pairs; ++j) {
        long double w = std::pow(b, -2.0L * j / rot_dim);
        if (kind == HALO_CUDA_ROPE_LINEAR) w /= s->factor;
        if (kind == HALO_CUDA_ROPE_FACTORS) {
            if (!(s->pair_factors[j] > 0) || !std::isfinite(s->pair_factors[j])) return fail(HALO_CUDA_E_KERNEL, "%s: pair factor %g", op, s->pair_factors[j]);
            w /= s->pair_factors[j];
        }
        if (limits) {
            long double slowed = kind == HALO_CUDA_ROPE_RAMP ? (j - lo) / std::fmax(hi - lo, 0.001L)
                                                             : 1 - (s->original_context * w / kTurn - s->slow) / (static_cast<long double>(s->fast) - s->slow);
            slowed = std::fmin(std::fmax(slowed, 0.0L), 1.0L);
            w = w / s->factor * slowed + w * (1 - slowed);
        }
        const long double turns = w / kTurn;
        const long double part = std::ldexp(turns - std::floor(turns), 64);  // whole turns do not show
        f.turns[j] = !std::isfinite(part) ? 0 : part >= 18446744073709551615.0L ? UINT64_MAX : static_cast<uint64_t>(part);
    }
    *out = f;
    return 0;
}

/// A C entry lets no exception out: the context's tables may grow in the call.
template <class F>
int guarded(F&& f) {
    try {
        return f();
    } catch (const std::bad_alloc&) {
        return fail(HALO_CUDA_E_MEMORY, "out of host memory");
    } catch (...) {
        return fail(HALO_CUDA_E_BACKEND, "unexpected exception");
    }
}

}  // namespace
}  // namespace attn
}  // namespace halo_cuda

using namespace halo_cuda;

extern "C" {

int halo_cuda_rope_freqs(uint32_t rot_dim, double base, const HaloCudaRopeScaling* scaling, HaloCudaRopeFreqs* freqs) {
    return attn::take_freqs(rot_dim, base, scaling, freqs);
}

int halo_cuda_rope(HaloCudaCtx* ctx, const HaloCudaRope* args, HaloCudaStream stream) {
    return attn::guarded([&] {
        attn::RopeCall c{};
        if (int rc = attn::take_rope(args, &c)) return rc;
        if (int rc = enter(ctx)) return rc;
        if (c.n_tokens == 0 || c.n_q + c.n_kv == 0) return 0;
        return attn::launch_rope(c, static_cast<cudaStream_t>(stream));
    });
}

int halo_cuda_kv_write(HaloCudaCtx* ctx, const HaloCudaKvWrite* args, HaloCudaStream stream) {
    return attn::guarded([&] {
        attn::WriteCall c{};
        if (int rc = attn::take_write(args, &c)) return rc;
        if (int rc = enter(ctx)) return rc;
        if (c.cache.n_seq == 0 || c.rows.n_tokens == 0 || c.rows.max_tokens == 0 || c.cache.max_pages == 0) return 0;
        return attn::launch_kv_write(ctx, c, static_cast<cudaStream_t>(stream));
    });
}

int halo_cuda_attention(HaloCudaCtx* ctx, const HaloCudaAttention* args, HaloCudaStream stream) {
    return attn::guarded([&] {
        attn::AttentionCall c{};
        if (int rc = attn::take_attention(args, &c)) return rc;
        if (int rc = enter(ctx)) return rc;
        if (c.cache.n_seq == 0 || c.rows.n_tokens == 0 || c.rows.max_tokens == 0) return 0;
        return attn::launch_attention(ctx, c, static_cast<cudaStream_t>(stream));
    });
}

}  // extern "C"
