/* trlm_serve.h -- operators for serving many sequences at once (additive: the
 * reference's generate.c recomputes one window per token and has none).
 *
 * Four operators on device buffers, beside trlm_gemm (trlm_ext.h):
 *   trlm_kv_append     rotary positions of new queries and keys, keys and
 *                      values written into a paged cache (fp32, bf16, 8 bits);
 *   trlm_kv_read       cached rows back as fp32;
 *   trlm_attn_paged    causal attention of new tokens over their sequences'
 *                      cached tokens;
 *   trlm_logits_rules  penalties for repeated tokens, biases and grammar masks;
 * and gpu_paged_*, a decoder over a trainer's parameters whose sequences have
 * lengths of their own, built on them.
 *
 * Every operator queues its kernels on the stream of the calling thread's
 * current context and returns; nothing is allocated or copied, so a call may
 * be captured into a HIP graph.  Lengths, pages and tokens are read on the
 * device when the kernels run: a captured call follows what its buffers hold
 * at each replay.  0: queued.  -1: refused, with a message on stderr and
 * nothing launched (an argument out of range, a null or unaligned buffer, a
 * workspace too small, another device current than the handle's).  What is
 * only known on the device is kept safe there: lengths and row ranges are
 * clamped, a page outside the pool holds no tokens, an id outside the
 * vocabulary is passed over. */
#ifndef TRLM_SERVE_H
#define TRLM_SERVE_H

#include "trlm_ext.h"

#ifdef __cplusplus
extern "C" {
#endif

/* The operators' kernels in one context. */
typedef struct TrlmServe TrlmServe;
TrlmServe* trlm_serve_create(HipCtx* ctx);
void trlm_serve_destroy(TrlmServe* e);

/* How a cache holds its numbers.  TRLM_KV_I8: for every token and head a
 * scale s = amax / 127 (fp32, kept in [2^-126, 8454659 * 2^98]) and the
 * integers rint(x / s), the quotient rounded to fp32, ties to even; a row
 * with a number that is not finite has the scale NaN, so it reads as NaN. */
enum { TRLM_KV_F32 = 0, TRLM_KV_BF16 = 1, TRLM_KV_I8 = 2 };

/* One layer's cache: a pool of pages.  Token t of a sequence is row
 * t % page_size of the sequence's page t / page_size; a page holds
 * [kv_heads][page_size][head_dim] numbers of k and as many of v. */
typedef struct TrlmKvCache {
    hipDeviceptr_t k, v;               /* [num_pages][kv_heads][page_size][head_dim], 16-byte aligned */
    hipDeviceptr_t k_scale, v_scale;   /* f32 [num_pages][kv_heads][page_size], 16-byte aligned; TRLM_KV_I8 only */
    u32 type;                          /* TRLM_KV_* */
    u32 num_pages;
    u32 page_size;                     /* a power of two, 16 .. 65536 */
    u32 kv_heads;                      /* 1 .. 1024 */
    u32 head_dim;                      /* 16, 32, 64 or 128 */
} TrlmKvCache;

/* The sequences of a call, their new tokens' rows stacked: sequence i's are
 * the rows q_start[i] .. q_start[i + 1] - 1 of the row buffers (none, or one
 * token, or many), the last of its kv_len[i] tokens in order: row r is the
 * token at position kv_len[i] - (q_start[i + 1] - r).  Rows from q_start[n]
 * on are left alone.  Sequences may share pages (a common prefix); tokens of
 * one append go to places of their own. */
#define TRLM_SERVE_MAX_SEQS 4096u
typedef struct TrlmKvSeqs {
    u32 n;                    /* sequences, 0 .. TRLM_SERVE_MAX_SEQS */
    u32 rows;                 /* rows of the row buffers (q_start[n] <= rows), below 2^24 */
    hipDeviceptr_t q_start;   /* i32 [n + 1], ascending */
    hipDeviceptr_t kv_len;    /* i32 [n], the new tokens among them */
    hipDeviceptr_t pages;     /* i32 [n][max_pages] */
    u32 max_pages;            /* max_pages * page_size <= 2^30 */
    u32 max_q;                /* bounds of this call's (or, captured, of every replay's) new tokens of one */
    u32 max_kv;               /* sequence and tokens of one sequence; trlm_attn_paged takes no more */
} TrlmKvSeqs;

/* The new tokens' rows: head h at columns h * head_dim of q, k and v, row
 * strides in floats (16-byte aligned rows).  The first rot_dim numbers of
 * every head of q and k are turned as pairs by the angles of the token's
 * position: (2i, 2i + 1), or with rot_half (i, i + rot_dim / 2); angle tables
 * [max_pos][rot_dim / 2] (any scaling for long contexts is in them).  Products
 * and differences are formed in 64 bits and rounded once.  A token at or past
 * max_pos, or whose position has no page, is passed over. */
typedef struct TrlmKvRows {
    hipDeviceptr_t q, k, v;   /* q may be NULL (heads 0): keys and values only */
    u32 ldq, ldk, ldv;
    hipDeviceptr_t q_out;     /* rotated queries; q itself, or rows apart from q, k and v */
    u32 ldqo;
    u32 heads;                /* query heads, up to 1024 */
    hipDeviceptr_t cos_t, sin_t;
    u32 max_pos;
    u32 rot_dim;              /* 0 (no rotation), or a multiple of 8 up to head_dim */
    u32 rot_half;
} TrlmKvRows;

i32 trlm_kv_append(TrlmServe* e, const TrlmKvCache* c, const TrlmKvSeqs* s, const TrlmKvRows* r);

/* The cached k and v of the call's rows as fp32 rows of kv_heads * head_dim
 * numbers, ld floats apart: what trlm_kv_append wrote for the same sequences
 * (with q_start ranges as long as kv_len: the whole sequences).  A token
 * without a page reads as zeros. */
i32 trlm_kv_read(TrlmServe* e, const TrlmKvCache* c, const TrlmKvSeqs* s, hipDeviceptr_t k_out, hipDeviceptr_t v_out,
                 u32 ld);

/* out row r, head h = sum over the tokens t <= position of r of softmax(scale
 * <q_r, k_t>) v_t, query head h reading cached head h / (heads / kv_heads).
 * q and out: fp32 rows (rows * heads below 2^31), heads side by side, strides
 * in floats; out may not overlap q.  Accuracy as of fp32 products and sums, for every cache type.  A
 * row without tokens to see (kv_len 0, no pages) is zeros.  A number that is
 * not finite makes the outputs that see it NaN (an infinite key whose score
 * is -infinity may also count as if it were not there) and no others: tokens after a row's
 * own, and whatever a page holds behind its sequence, do not count.
 * ws: trlm_attn_paged_workspace bytes (0: none needed), 16-byte aligned;
 * calls that may overlap in time need workspaces apart, and so do captured
 * graphs that may run together. */
i32 trlm_attn_paged(TrlmServe* e, const TrlmKvCache* c, const TrlmKvSeqs* s, hipDeviceptr_t q, u32 ldq, u32 heads,
                    f32 scale, hipDeviceptr_t out, u32 ldo, hipDeviceptr_t ws, u64 ws_bytes);
u64 trlm_attn_paged_workspace(const TrlmKvCache* c, const TrlmKvSeqs* s, u32 heads);

/* out[r][t] = the rules of row r on logits[r][t], in this order:
 *   t among history[r][0 .. hist_len[r]):             x = x > 0 ? x / repetition[r] : x * repetition[r]
 *   c > 0 times among history[r][gen_start[r] ..):     x = x - (frequency[r] * c + presence[r])
 *   t in bias_ids[r][0 .. n_bias[r]):                  x = x + bias[r][its last place]
 *   mask[r]'s bit t (bit t % 32 of word t / 32) zero:  x = -infinity
 * Each part may be left out: history NULL (then no penalties), repetition,
 * frequency or presence NULL (1, 0, 0), gen_start NULL (0), bias_ids NULL,
 * mask NULL.  A row whose mask leaves nothing is -infinity throughout.  out
 * may be logits itself (the same address and stride), otherwise apart from it. */
typedef struct TrlmLogitsRules {
    hipDeviceptr_t logits, out;   /* f32 [rows][ld], [rows][ld_out] */
    u32 rows, vocab, ld, ld_out;
    hipDeviceptr_t history;       /* u32 [rows][ld_hist] token ids */
    hipDeviceptr_t hist_len;      /* i32 [rows] */
    hipDeviceptr_t gen_start;     /* i32 [rows] */
    u32 ld_hist;
    hipDeviceptr_t repetition, frequency, presence;   /* f32 [rows] */
    hipDeviceptr_t bias_ids;      /* u32 [rows][ld_bias] */
    hipDeviceptr_t bias;          /* f32 [rows][ld_bias] */
    hipDeviceptr_t n_bias;        /* i32 [rows] */
    u32 ld_bias;
    hipDeviceptr_t mask;          /* u32 [rows][ld_mask], ld_mask >= ceil(vocab / 32) */
    u32 ld_mask;
} TrlmLogitsRules;

i32 trlm_logits_rules(TrlmServe* e, const TrlmLogitsRules* r);

/* ---- decoding many sequences of their own lengths ----
 * A decoder over the trainer's resident parameters, on its stream, with one
 * paged cache a layer.  Sequences are slots 0 .. max_seqs - 1; a slot is empty
 * until gpu_paged_extend gives it tokens and again after gpu_paged_release.
 * head_dim is one of the operators'; num_pages x page_size at most 2^36.
 * Where a call returns i32: 0, or -1 with a message on stderr and nothing
 * changed (a slot, token or length out of range, a slot twice in a call, no
 * pages left).  Creation with sizes out of range ends the process, as the
 * trainer's does. */
typedef struct TrlmPagedDecoder TrlmPagedDecoder;
TrlmPagedDecoder* gpu_paged_create(GpuTrainer* g, u32 max_seqs, u32 max_ctx, u32 num_pages, u32 page_size, u32 kv_type);
void gpu_paged_destroy(TrlmPagedDecoder* d);
/* lens[i] new tokens (at least one) of slot seqs[i], i < n, their ids one after
 * the other: prompts, chunks of them and single tokens in one call.  Leaves the
 * logits of every slot's last token as rows 0 .. n - 1. */
i32 gpu_paged_extend(TrlmPagedDecoder* d, u32 n, const u32* seqs, const u32* lens, const u32* ids);
void gpu_paged_release(TrlmPagedDecoder* d, u32 seq);
u32 gpu_paged_length(const TrlmPagedDecoder* d, u32 seq);   /* 0 for an empty slot or none */
u32 gpu_paged_free_pages(const TrlmPagedDecoder* d);
/* On the rows of the last extend: the logits [n][V]; rules on them (a slot's
 * history is its tokens, those after its first extend count as generated, a released
 * slot has none; each
 * pointer may be NULL; host arrays of n entries or rows); the first maximum of
 * each row (0 where a mask left nothing); sample_next (generate.c:57-73) per
 * row, as gpu_decoder_sample (the last token where a mask left nothing). */
typedef struct TrlmTokenRules {
    const f32 *repetition, *frequency, *presence;   /* [n] */
    const u32* bias_ids;                            /* [n][ld_bias] */
    const f32* bias;                                /* [n][ld_bias] */
    const u32* n_bias;                              /* [n], up to ld_bias */
    u32 ld_bias;
    const u32* mask;                                /* [n][ceil(V / 32)] */
} TrlmTokenRules;
void gpu_paged_logits(TrlmPagedDecoder* d, f32* host_logits);
i32 gpu_paged_rules(TrlmPagedDecoder* d, const TrlmTokenRules* r);
void gpu_paged_greedy(TrlmPagedDecoder* d, u32* out_ids);
void gpu_paged_sample(TrlmPagedDecoder* d, PCGState* rngs, f32 temperature, u32* out_ids);
/* The cached rows of a slot in one layer, k and v [length][d_model]. */
i32 gpu_paged_read(TrlmPagedDecoder* d, u32 seq, u32 layer, f32* k, f32* v);

#ifdef __cplusplus
}
#endif

#endif /* TRLM_SERVE_H */
