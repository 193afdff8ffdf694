/*
 * halo_cuda_attention.h -- the attention layer's operators between the matmuls of halo_cuda.h: rotary positions, the write of keys and
 * values into a paged cache held in 8 bits, and the attention that reads the cache.
 *
 * Same contract as halo_cuda.h: every entry point returns 0 or a negative status, validates on the host before anything is enqueued, and
 * enqueues on the given stream.  What lies in device memory (positions, lengths, page numbers) is read by the kernels when they run, so a
 * captured call may be replayed over new contents; values there that are out of range are handled as said below and never reach past an
 * operand.  Counterparts in the reference's interface: Backend::partial_rope, kv_write and attention; its cache holds floats and its CPU
 * operators are serial, so the layouts here are this library's own.
 */
#ifndef HALO_CUDA_ATTENTION_H
#define HALO_CUDA_ATTENTION_H

#include "halo_cuda.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Types of activations besides HALO_CUDA_T_F32: ggml ids, like the weight types. */
#define HALO_CUDA_T_F16 1
#define HALO_CUDA_T_BF16 30

/* Rows of heads: element d of head h of token t lies at p + t * token_stride + h * head_stride + d * size.  Strides in bytes; 0 = dense (a
 * head's elements, then the next head, then the next token).  p and the strides are multiples of the element's size. */
typedef struct HaloCudaHeads {
    void* p;
    uint64_t token_stride, head_stride;
} HaloCudaHeads;

/* ---- rotary positions --------------------------------------------------------------------------------------------------
 * Pair j of a head's first rot_dim elements is turned by position * f_j radians and multiplied by `magnitude`.  f_j = base^(-2j / rot_dim),
 * stretched for contexts longer than a model was trained on in one of these ways: */
#define HALO_CUDA_ROPE_NONE 0
#define HALO_CUDA_ROPE_LINEAR 1  /* f_j / factor */
#define HALO_CUDA_ROPE_BASE 2    /* base * factor^(rot_dim / (rot_dim - 2)): the slowest pair slows by `factor`, the fastest keeps its pace */
#define HALO_CUDA_ROPE_RAMP 3    /* pairs that turn more than `fast` times over original_context keep f_j, those below `slow` turns get f_j / factor,
                                    linear in j between the two (rounded outwards); magnitude = 0.1 ln(factor) + 1 */
#define HALO_CUDA_ROPE_BANDS 4   /* the same two limits (`fast`, `slow`), linear in the number of turns between them; magnitude 1 */
#define HALO_CUDA_ROPE_FACTORS 5 /* f_j / pair_factors[j] */
typedef struct HaloCudaRopeScaling {
    uint32_t kind, reserved;
    double factor;              /* > 0 (RAMP: >= 1) */
    double original_context;    /* RAMP, BANDS: tokens */
    double fast, slow;          /* RAMP, BANDS: fast > slow > 0 */
    double magnitude;           /* 0 = what the kind says */
    const double* pair_factors; /* FACTORS: rot_dim / 2 of them, each > 0 */
} HaloCudaRopeScaling;

/* What a model's host makes once: turns[j] = f_j / 2 pi in units of 2^-64 of a turn.  position * turns[j] modulo 2^64 is then the phase,
 * reduced exactly for every 32-bit position; cosine and sine are taken of its leading 32 bits. */
#define HALO_CUDA_ROPE_MAX_PAIRS 128
typedef struct HaloCudaRopeFreqs {
    uint32_t n_pairs;
    float magnitude;
    uint64_t turns[HALO_CUDA_ROPE_MAX_PAIRS];
} HaloCudaRopeFreqs;
/* Host arithmetic, no device needed.  rot_dim: even, 2 to 256; base > 0; scaling null = HALO_CUDA_ROPE_NONE. */
int halo_cuda_rope_freqs(uint32_t rot_dim, double base, const HaloCudaRopeScaling* scaling, HaloCudaRopeFreqs* freqs);

/* Turns q's and k's heads (k.p null with n_kv 0: q alone).  Pair j is elements (j, j + n_pairs), or (2j, 2j + 1) with interleaved = 1.
 * Products and sums in fp32, rounded once.  q_out / k_out: equal to q / k (in place: elements behind rot_dim are not touched), or memory that
 * overlaps neither input (elements behind rot_dim are copied).  positions: n_tokens int32 (device), any value, negative ones turn backwards.
 * head_dim: at least 2 * n_pairs, at most 1024.  n_tokens == 0 is a no-op. */
typedef struct HaloCudaRope {
    uint32_t type; /* of q and k: HALO_CUDA_T_F32, _F16, _BF16 */
    uint32_t interleaved;
    const HaloCudaRopeFreqs* freqs; /* host memory, read by the call */
    const int32_t* positions;
    HaloCudaHeads q, k, q_out, k_out;
    uint32_t n_tokens, n_q, n_kv, head_dim;
} HaloCudaRope;
int halo_cuda_rope(HaloCudaCtx* ctx, const HaloCudaRope* args, HaloCudaStream stream);

/* ---- the cache -----------------------------------------------------------------------------------------------------------
 * Two pools of pages.  A page of one kv head is page_tokens rows of head_dim e4m3 codes, dense; its n_kv heads follow one another; pages are
 * page_stride bytes apart (0 = dense), so that the pages of several layers can share one block.  Every (page, head) of either pool has one
 * byte b in k_scale / v_scale (at page * scale_stride + head): an element stands for code * 2^(b - 127), b being between 87 and 207 (2^-40 to
 * 2^80; the operators read a byte beyond as the nearer of the two).  Token t of sequence i is slot t % page_tokens of page
 * table[i][t / page_tokens]. */
#define HALO_CUDA_KV_E4M3 1
#define HALO_CUDA_KV_SCALE_MIN 87
#define HALO_CUDA_KV_SCALE_MAX 207
typedef struct HaloCudaKvCache {
    void* k; /* 16-byte aligned, like page_stride */
    void* v;
    uint8_t* k_scale;
    uint8_t* v_scale;
    const int32_t* table;                           /* n_seq rows of max_pages page numbers (device) */
    uint64_t page_stride, scale_stride, table_stride; /* bytes; 0 = dense: n_kv * page_tokens * head_dim, n_kv, max_pages * 4 */
    uint32_t type;        /* HALO_CUDA_KV_E4M3 */
    uint32_t n_pages;     /* in the pools; below 2^31 */
    uint32_t n_kv;
    uint32_t head_dim;    /* 64, 128 or 256 */
    uint32_t page_tokens; /* 16, 32, 64 or 128 */
    uint32_t max_pages;   /* of one sequence; max_pages * page_tokens at most 2^30 */
    uint32_t n_seq, reserved; /* n_seq below 2^31 */
} HaloCudaKvCache;

/* Whose the token rows of a call are: sequence i has rows start[i] .. start[i + 1] - 1 of the operands (device, n_seq + 1 values, never
 * falling, at most n_tokens; null: max_tokens rows each, n_tokens = n_seq * max_tokens), and they are its LAST tokens: the last one is at position
 * length[i] - 1 (device, n_seq values, each 0 to max_pages * page_tokens).  A sequence with fewer tokens than rows has rows at negative
 * positions.  max_tokens: no sequence has more rows (rows beyond are left out).  Rows behind the last sequence's are left as they were. */
typedef struct HaloCudaKvRows {
    const int32_t* start;
    const int32_t* length;
    uint32_t n_tokens, max_tokens;
} HaloCudaKvRows;

/* Writes k's and v's rows into their slots.  The scale of a touched (page, head) is the smallest power of two (2^-40 at least, 2^80 at most) under which
 * the largest finite magnitude of its new rows is at most 448, or the scale it had if that is larger and slots in front of the new rows hold
 * the sequence's earlier tokens: those are then rounded again to the new scale.  Codes are rounded to nearest, ties to even; infinities become
 * +-448, a NaN stays one.  Slots behind the new rows keep their bytes (and no meaning).  Rows at negative positions are skipped.  A page
 * number outside [0, n_pages) sets bit 8 (kStatusBadIndex) of *status (device word, optional) and nothing is written for it.  At most 65535
 * sequences and 32767 kv heads.  Two sequences of one call must not write into the same page, nor one sequence through two columns of
 * its row: a forked page is copied first (halo_cuda_memcpy_d2d_async of its codes and scale bytes). */
typedef struct HaloCudaKvWrite {
    uint32_t type, reserved; /* of k and v: HALO_CUDA_T_F32, _F16, _BF16 */
    HaloCudaKvCache cache;
    HaloCudaKvRows rows;
    HaloCudaHeads k, v; /* n_tokens x n_kv x head_dim */
    uint32_t* status;
} HaloCudaKvWrite;
int halo_cuda_kv_write(HaloCudaCtx* ctx, const HaloCudaKvWrite* args, HaloCudaStream stream);

/* out[row][h] = sum_t w_t V[t], w = softmax over the tokens t that the row sees of scale * q[row][h] . K[t], with K and V of kv head
 * h / (n_q / n_kv) of the row's sequence.  A row at position p sees tokens t < length; causal = 1: of those t <= p; window > 0 (causal only): of
 * those t > p - window.  A row that sees none gets zeros.  What a row does not see has no influence on it, whatever it holds.  Tokens of a page whose
 * number is outside [0, n_pages) are left out and set bit 8 of *status (device word, optional).  A row whose q holds a NaN or an infinity gets NaN, or
 * zeros where it sees none or all of its scores are minus infinity; no other row is touched by it.
 * Type F32 computes to fp32 accuracy (both factors of the products in two fp16 terms, 22 bits); F16 and BF16 take q exactly (but for elements below
 * 2^-28 of their row's largest) and round the weights to 11 bits.  Softmax and sums are fp32; the tensor cores cut a sum off where they add 16 keys to it,
 * so one is taken out and added up, rounded, after at most 64 (F32) or 1024 (F16, BF16) such steps: what is lost of it is below 2^-17 or 2^-13, however
 * long the context.  Weights (times their values' scale) below 2^-20 of the row's largest are rounded to multiples of 2^-30 of it, for all types.  The
 * order of the sums goes with the shape and the lengths of the whole call, and the same call gives the same bits.
 * The cache has at least one page, the table a column, and at most 2^20 sequences.  Uses context scratch, whose size goes with the operands' shapes alone: run a call once
 * before capturing it. */
typedef struct HaloCudaAttention {
    uint32_t type, n_q; /* of q and out; n_q: a multiple of n_kv, at most 32768 */
    HaloCudaKvCache cache;
    HaloCudaKvRows rows;
    HaloCudaHeads q, out; /* n_tokens x n_q x head_dim; out overlaps neither q nor the cache */
    uint32_t causal, window;
    float scale; /* finite */
    uint32_t reserved;
    uint32_t* status;
} HaloCudaAttention;
int halo_cuda_attention(HaloCudaCtx* ctx, const HaloCudaAttention* args, HaloCudaStream stream);

#ifdef __cplusplus
}
#endif
#endif /* HALO_CUDA_ATTENTION_H */
