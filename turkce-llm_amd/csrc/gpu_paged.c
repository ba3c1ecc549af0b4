/* gpu_paged.c -- decoding sequences of their own lengths over a paged cache
 * (trlm_serve.h), on a GpuTrainer's resident parameters.
 *
 * gpu_decode.c keeps one contiguous cache for a batch whose sequences share a
 * length.  Here every sequence holds pages of its own from one pool, and a call
 * takes any mix of prompts, chunks of prompts and single tokens as stacked
 * rows: embedding, then per layer RMSNorm, the QKV product, trlm_kv_append
 * (rotation in place, keys and values into the cache), trlm_attn_paged, the
 * output product with the residual, RMSNorm, the gate/up product, SwiGLU and
 * the down product with the residual; the final norm and the tied head run on
 * every sequence's last row.  The products are the prefill's: an engine that is
 * not kept to fp32.
 *
 * Six layers of d_model 384, V 31769, all sequences past 256 tokens, one token
 * each with its greedy pick (host calls included): 1 sequence 350 us, 16
 * sequences 381, 64 sequences 447 with a bf16 cache (fp32 490, int8 442); the
 * fixed batch of gpu_decode.c, whose step is fused for equal lengths, 268, 293
 * and 308.  Both wait on launches and small products, not on the cache.
 */
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#include <unistd.h>

#include "trlm_serve.h"
#include "gpu_internal.h"

#define F4 ((u64)sizeof(f32))
#define SAMPLE_THREADS 1024u   /* threads per workgroup of the sampling kernels (as in decode.hip) */
#define SAMPLE_CHUNKS 8u       /* k_sample_exp workgroups per row */
#define LAYER_BUFS 10u         /* row buffers of a pass */

typedef struct Slot {
    u32 len, first;   /* tokens held; of them, those of the first extend */
    u32 pages;        /* pages held */
} Slot;

struct TrlmPagedDecoder {
    GpuTrainer* g;
    TrlmGemm* gemm;
    TrlmServe* serve;
    u32 max_seqs, max_ctx, per;          /* per: pages of a full sequence */
    TrlmKvCache* layer;                  /* [L] */
    hipDeviceptr_t cos_t, sin_t;         /* [max_ctx][hd / 2] */
    /* host: slots, their tokens and pages, the pages of nobody */
    Slot* slot;
    u32* tokens;                         /* [max_seqs][max_ctx] */
    i32* table;                          /* [max_seqs][per] */
    i32* free_page;
    u32 num_pages, num_free;
    /* the last extend's rows */
    u32 n;
    u32* rows;                           /* [max_seqs] their slots */
    /* the call's sequences, one upload: q_start [n + 1], kv_len [n], last rows [n], pages [n][width], tokens [R] */
    u32* call;
    hipDeviceptr_t call_dev;
    u64 call_words;
    hipDeviceptr_t buf[LAYER_BUFS];      /* x, x2, n, rinv, qkv, att, gu, h, nf, rf */
    u64 cap_rows;
    hipDeviceptr_t ws;
    u64 ws_bytes;
    hipDeviceptr_t logits, out_ids, e, prefix, u;
    hipFunction_t k_sample_exp, k_sample;
};

static void paged_fatal(const char* msg) {
    fprintf(stderr, "[HIP ERROR] gpu_paged: %s\n", msg);
    fflush(stderr);
    _exit(1);
}

static i32 refuse(const char* op, const char* why) {
    fprintf(stderr, "%s: refused, nothing changed: %s\n", op, why);
    fflush(stderr);
    return -1;
}

static void* host_mem(u64 n, u64 size) {
    void* p = calloc(n ? n : 1, size);
    if (!p) paged_fatal("out of host memory");
    return p;
}

static hipDeviceptr_t fl(u64 floats) { return hip_alloc(floats * F4); }
static hipDeviceptr_t at(hipDeviceptr_t base, u64 floats) { return (hipDeviceptr_t)((char*)base + floats * F4); }
static u32 cdiv(u64 a, u64 b) { return (u32)((a + b - 1) / b); }

TrlmPagedDecoder* gpu_paged_create(GpuTrainer* g, u32 max_seqs, u32 max_ctx, u32 num_pages, u32 page_size, u32 kv_type) {
    if (!max_seqs || max_seqs > TRLM_SERVE_MAX_SEQS || !max_ctx || max_ctx > (1u << 24) || !num_pages ||
        num_pages > (1u << 30))
        paged_fatal("max_seqs, max_ctx and num_pages must be positive (and up to 4096, 2^24 and 2^30)");
    if (page_size < 16 || page_size > 65536 || (page_size & (page_size - 1)))
        paged_fatal("page_size must be a power of two, 16 to 65536");
    if ((u64)num_pages * page_size > (1ull << 36)) paged_fatal("more than 2^36 positions");
    if (g->hd != 16 && g->hd != 32 && g->hd != 64 && g->hd != 128) paged_fatal("head_dim must be 16, 32, 64 or 128");
    if (kv_type > TRLM_KV_I8) paged_fatal("unknown cache type");
    trlm_bind(g);
    TrlmPagedDecoder* d = (TrlmPagedDecoder*)host_mem(1, sizeof(*d));
    d->g = g;
    d->max_seqs = max_seqs;
    d->max_ctx = max_ctx;
    d->per = cdiv(max_ctx, page_size);
    d->num_pages = d->num_free = num_pages;
    d->slot = (Slot*)host_mem(max_seqs, sizeof(Slot));
    d->tokens = (u32*)host_mem((u64)max_seqs * max_ctx, sizeof(u32));
    d->table = (i32*)host_mem((u64)max_seqs * d->per, sizeof(i32));
    d->free_page = (i32*)host_mem(num_pages, sizeof(i32));
    d->rows = (u32*)host_mem(max_seqs, sizeof(u32));
    for (u32 i = 0; i < num_pages; i++) d->free_page[i] = (i32)(num_pages - 1 - i);   /* page 0 is taken first */

    const u64 numbers = (u64)num_pages * g->H * page_size * g->hd, scales = (u64)num_pages * g->H * page_size;
    const u64 bytes = numbers * (kv_type == TRLM_KV_F32 ? 4 : kv_type == TRLM_KV_BF16 ? 2 : 1);
    d->layer = (TrlmKvCache*)host_mem(g->L, sizeof(TrlmKvCache));
    for (u32 l = 0; l < g->L; l++) {
        TrlmKvCache* c = &d->layer[l];
        c->k = hip_alloc(bytes);
        c->v = hip_alloc(bytes);
        if (kv_type == TRLM_KV_I8) {
            c->k_scale = fl(scales);
            c->v_scale = fl(scales);
        }
        c->type = kv_type;
        c->num_pages = num_pages;
        c->page_size = page_size;
        c->kv_heads = g->H;
        c->head_dim = g->hd;
    }

    /* RoPE tables for every position, built on the host as the reference
     * builds them (model/rope.c) */
    Tensor ct, st;
    memset(&ct, 0, sizeof(ct));
    ct.ndim = 2;
    ct.shape[0] = max_ctx;
    ct.shape[1] = g->hd / 2;
    ct.strides[0] = (i64)(g->hd / 2);
    ct.strides[1] = 1;
    ct.numel = (u64)max_ctx * (g->hd / 2);
    st = ct;
    ct.data = (f32*)host_mem(ct.numel, F4);
    st.data = (f32*)host_mem(st.numel, F4);
    rope_build_tables(&ct, &st, max_ctx, g->hd, 10000.0f);
    d->cos_t = fl(ct.numel);
    d->sin_t = fl(st.numel);
    hip_h2d(d->cos_t, ct.data, ct.numel * F4);
    hip_h2d(d->sin_t, st.data, st.numel * F4);
    free(ct.data);
    free(st.data);

    const u64 S = max_seqs;
    d->logits = fl(S * g->ldv);
    hip_memset_zero(d->logits, S * g->ldv * F4);
    d->out_ids = hip_alloc(S * sizeof(u32));
    d->e = fl(S * g->ldv);
    d->prefix = hip_alloc(S * g->V * sizeof(f64));
    d->u = hip_alloc(S * sizeof(f64));
    d->k_sample_exp = hip_get_kernel(&g->hip, "k_sample_exp");
    d->k_sample = hip_get_kernel(&g->hip, "k_sample_rows");
    d->gemm = trlm_gemm_create(&g->hip);
    d->serve = trlm_serve_create(&g->hip);
    hip_sync();
    return d;
}

static void free_rows(TrlmPagedDecoder* d) {
    for (u32 i = 0; i < LAYER_BUFS; i++)
        if (d->buf[i]) { hip_free(d->buf[i]); d->buf[i] = NULL; }
    d->cap_rows = 0;
}

void gpu_paged_destroy(TrlmPagedDecoder* d) {
    if (!d) return;
    trlm_bind(d->g);
    hip_sync();
    free_rows(d);
    for (u32 l = 0; l < d->g->L; l++) {
        hip_free(d->layer[l].k);
        hip_free(d->layer[l].v);
        if (d->layer[l].k_scale) hip_free(d->layer[l].k_scale);
        if (d->layer[l].v_scale) hip_free(d->layer[l].v_scale);
    }
    if (d->ws) hip_free(d->ws);
    if (d->call_dev) hip_free(d->call_dev);
    free(d->call);
    hipDeviceptr_t bufs[] = { d->cos_t, d->sin_t, d->logits, d->out_ids, d->e, d->prefix, d->u };
    for (u32 i = 0; i < sizeof(bufs) / sizeof(bufs[0]); i++) hip_free(bufs[i]);
    trlm_gemm_destroy(d->gemm);
    trlm_serve_destroy(d->serve);
    free(d->layer);
    free(d->slot);
    free(d->tokens);
    free(d->table);
    free(d->free_page);
    free(d->rows);
    free(d);
}

u32 gpu_paged_length(const TrlmPagedDecoder* d, u32 seq) { return seq < d->max_seqs ? d->slot[seq].len : 0; }
u32 gpu_paged_free_pages(const TrlmPagedDecoder* d) { return d->num_free; }

void gpu_paged_release(TrlmPagedDecoder* d, u32 seq) {
    if (seq >= d->max_seqs) return;
    Slot* s = &d->slot[seq];
    while (s->pages) d->free_page[d->num_free++] = d->table[(u64)seq * d->per + --s->pages];
    s->len = s->first = 0;
}

static void want_rows(TrlmPagedDecoder* d, u64 R) {
    if (R <= d->cap_rows) return;
    const GpuTrainer* g = d->g;
    free_rows(d);
    const u64 width[LAYER_BUFS] = { g->D, g->D, g->D, 1, 3ull * g->D, g->D, 2ull * g->F, g->F, 0, 0 };
    for (u32 i = 0; i < 8; i++) d->buf[i] = fl(R * width[i]);
    d->buf[8] = fl((u64)d->max_seqs * g->D);      /* the last rows, and their norm */
    d->buf[9] = fl((u64)d->max_seqs * g->D + d->max_seqs);
    d->cap_rows = R;
}

static void want_call(TrlmPagedDecoder* d, u64 words) {
    if (words <= d->call_words) return;
    if (d->call_dev) hip_free(d->call_dev);
    free(d->call);
    d->call = (u32*)host_mem(words, sizeof(u32));
    d->call_dev = hip_alloc(words * sizeof(u32));
    d->call_words = words;
}

/* The queued pass over R rows. */
static void run_rows(TrlmPagedDecoder* d, u32 n, u32 R, u32 max_q, u32 max_kv, u32 width) {
    hipDeviceptr_t kv_len = at(d->call_dev, n + 1ull), last = at(kv_len, n), pages = at(last, n),
                   ids = at(pages, (u64)n * width);
    GpuTrainer pf = *d->g;                        /* the same parameters and kernels, the prefill's products */
    pf.gemm = d->gemm;
    const i32 D = (i32)pf.D, F = (i32)pf.F, M = (i32)R;
    const u32 H = pf.H;
    hipDeviceptr_t x = d->buf[0], x2 = d->buf[1], nr = d->buf[2], rinv = d->buf[3], qkv = d->buf[4], att = d->buf[5],
                   gu = d->buf[6], h = d->buf[7];
    TrlmKvSeqs s;
    memset(&s, 0, sizeof(s));
    s.n = n;
    s.rows = R;
    s.q_start = d->call_dev;
    s.kv_len = kv_len;
    s.pages = pages;
    s.max_pages = width;
    s.max_q = max_q;
    s.max_kv = max_kv;
    TrlmKvRows r;
    memset(&r, 0, sizeof(r));
    r.q = r.q_out = qkv;
    r.k = at(qkv, (u64)D);
    r.v = at(qkv, 2ull * D);
    r.ldq = r.ldk = r.ldv = r.ldqo = 3u * (u32)D;
    r.heads = H;
    r.cos_t = d->cos_t;
    r.sin_t = d->sin_t;
    r.max_pos = d->max_ctx;
    r.rot_dim = pf.hd;
    const u64 need = trlm_attn_paged_workspace(&d->layer[0], &s, H);
    if (need > d->ws_bytes) {
        if (d->ws) hip_free(d->ws);
        d->ws = hip_alloc(need);
        d->ws_bytes = need;
    }
    const f32 scale = 1.0f / m_sqrtf((f32)pf.hd);   /* attention.c:78 */
    trlm_embed_rows(&pf, ids, x, R);
    for (u32 l = 0; l < pf.L; l++) {
#define PP(k) trlm_param_ptr(&pf, trlm_pidx(l, k))
        trlm_rmsnorm_rows(&pf, x, PP(PK_ATTN_NORM), nr, rinv, R);
        trlm_gemm_rows(&pf, GEMM_NN, nr, PP(PK_WQKV), qkv, M, 3 * D, D, D, 3 * D, 3 * D, PP(PK_BQKV), NULL);
        if (trlm_kv_append(d->serve, &d->layer[l], &s, &r) ||
            trlm_attn_paged(d->serve, &d->layer[l], &s, qkv, 3u * (u32)D, H, scale, att, (u32)D, d->ws, d->ws_bytes))
            paged_fatal("an operator refused the decoder's own buffers");
        trlm_gemm_rows(&pf, GEMM_NN, att, PP(PK_WO), x2, M, D, D, D, D, D, PP(PK_BO), x);
        trlm_rmsnorm_rows(&pf, x2, PP(PK_FFN_NORM), nr, rinv, R);
        trlm_gemm_rows(&pf, GEMM_NN, nr, PP(PK_WGU), gu, M, 2 * F, D, D, 2 * F, 2 * F, PP(PK_BGU), NULL);
        trlm_swiglu_rows(&pf, gu, h, R);
        trlm_gemm_rows(&pf, GEMM_NN, h, PP(PK_WDOWN), x, M, D, F, F, D, D, PP(PK_BDOWN), x2);
#undef PP
    }
    /* every sequence's last row (the embedding kernel takes rows by index) */
    hipDeviceptr_t rows = d->buf[8], nf = d->buf[9];
    i32 ni = (i32)n, Di = D;
    void* args[] = { &x, &last, &rows, &ni, &Di };
    hip_launch(pf.k.embed_fwd, cdiv((u64)n * pf.D / (pf.D % 4 == 0 ? 4 : 1), 256), 1, 1, 256, 1, 1, 0, args);
    trlm_rmsnorm_rows(&pf, rows, trlm_param_ptr(&pf, trlm_pidx(pf.L, 0)), nf, at(nf, (u64)d->max_seqs * pf.D), n);
    trlm_gemm_rows(&pf, GEMM_NT, nf, trlm_param_ptr(&pf, 0), d->logits, ni, (i32)pf.V, D, D, D, (i32)pf.ldv, NULL, NULL);
}

i32 gpu_paged_extend(TrlmPagedDecoder* d, u32 n, const u32* seqs, const u32* lens, const u32* ids) {
    static const char* op = "gpu_paged_extend";
    if (!n || n > d->max_seqs) return refuse(op, "the number of sequences must be 1 to max_seqs");
    if (!seqs || !lens || !ids) return refuse(op, "no sequences, lengths or tokens");
    u64 R = 0, want = 0;
    u32 max_q = 0, max_kv = 0;
    const u32 page = d->layer[0].page_size;
    u8* seen = (u8*)host_mem(d->max_seqs, 1);
    const char* why = NULL;
    for (u32 i = 0; i < n && !why; i++) {
        if (seqs[i] >= d->max_seqs) why = "a slot out of range";
        else if (seen[seqs[i]]) why = "a slot twice in one call";
        else if (!lens[i]) why = "a sequence without new tokens";
        else if (lens[i] > d->max_ctx - d->slot[seqs[i]].len) why = "a sequence longer than max_ctx";
        if (why) break;
        const Slot* s = &d->slot[seqs[i]];
        seen[seqs[i]] = 1;
        R += lens[i];
        want += cdiv(s->len + lens[i], page) - s->pages;
        if (lens[i] > max_q) max_q = lens[i];
        if (s->len + lens[i] > max_kv) max_kv = s->len + lens[i];
    }
    free(seen);
    if (!why && (R >= (1u << 24) || R * d->g->H >= (1ull << 31) || (u64)n * d->g->H >= (1u << 22)))
        why = "more rows or sequences than one call of the operators takes";
    for (u64 r = 0; r < R && !why; r++)
        if (ids[r] >= d->g->V) why = "a token outside the vocabulary";
    if (!why && want > d->num_free) why = "no pages left";
    if (why) return refuse(op, why);

    trlm_bind(d->g);
    want_rows(d, R);
    const u32 width = cdiv(max_kv, page);
    want_call(d, 3ull * n + 1 + (u64)n * width + R);
    u32 *q_start = d->call, *kv_len = q_start + n + 1, *last = kv_len + n, *pages = last + n;
    memcpy(pages + (u64)n * width, ids, R * sizeof(u32));
    q_start[0] = 0;
    for (u32 i = 0; i < n; i++) {
        const u32 q = seqs[i];
        Slot* s = &d->slot[q];
        memcpy(d->tokens + (u64)q * d->max_ctx + s->len, ids + q_start[i], (u64)lens[i] * sizeof(u32));
        if (!s->len) s->first = lens[i];
        s->len += lens[i];
        i32* t = d->table + (u64)q * d->per;
        while (s->pages < cdiv(s->len, page)) t[s->pages++] = d->free_page[--d->num_free];
        q_start[i + 1] = q_start[i] + lens[i];
        kv_len[i] = s->len;
        last[i] = q_start[i + 1] - 1;
        for (u32 p = 0; p < width; p++) pages[(u64)i * width + p] = p < s->pages ? (u32)t[p] : ~0u;
        d->rows[i] = q;
    }
    d->n = n;
    hip_h2d(d->call_dev, d->call, (3ull * n + 1 + (u64)n * width + R) * sizeof(u32));
    run_rows(d, n, (u32)R, max_q, max_kv, width);
    return 0;
}

void gpu_paged_logits(TrlmPagedDecoder* d, f32* host_logits) {
    trlm_bind(d->g);
    if (d->n) hip_d2h_rows(host_logits, d->logits, (u64)d->g->ldv * F4, (u64)d->g->V * F4, d->n);
}

/* A copy on the device for one call, NULL for NULL. */
static hipDeviceptr_t up(const void* host, u64 bytes) {
    if (!host || !bytes) return NULL;
    hipDeviceptr_t p = hip_alloc(bytes);
    hip_h2d(p, host, bytes);
    return p;
}

i32 gpu_paged_rules(TrlmPagedDecoder* d, const TrlmTokenRules* r) {
    static const char* op = "gpu_paged_rules";
    if (!r) return refuse(op, "no rules");
    if (!d->n) return refuse(op, "no logits: extend comes first");
    if (r->bias_ids && (!r->bias || !r->n_bias || !r->ld_bias || r->ld_bias > (1u << 24)))
        return refuse(op, "biases need their values, counts and ld_bias, up to 2^24");
    const u64 n = d->n;
    for (u64 i = 0; r->bias_ids && i < n; i++)
        if (r->n_bias[i] > r->ld_bias) return refuse(op, "more biases than ld_bias");
    trlm_bind(d->g);
    u32 longest = 1;
    for (u64 i = 0; i < n; i++)
        if (d->slot[d->rows[i]].len > longest) longest = d->slot[d->rows[i]].len;
    const int history = r->repetition || r->frequency || r->presence;
    u32* tokens = (u32*)host_mem(history ? n * longest : 1, sizeof(u32));
    i32* len = (i32*)host_mem(n, sizeof(i32));
    i32* gen = (i32*)host_mem(n, sizeof(i32));
    for (u64 i = 0; history && i < n; i++) {
        const Slot* s = &d->slot[d->rows[i]];
        memcpy(tokens + i * longest, d->tokens + (u64)d->rows[i] * d->max_ctx, (u64)s->len * sizeof(u32));
        len[i] = (i32)s->len;
        gen[i] = (i32)s->first;
    }
    const u64 words = (d->g->V + 31) / 32;
    TrlmLogitsRules o;
    memset(&o, 0, sizeof(o));
    o.logits = o.out = d->logits;
    o.rows = (u32)n;
    o.vocab = d->g->V;
    o.ld = o.ld_out = d->g->ldv;
    if (history) {
        o.history = up(tokens, n * longest * sizeof(u32));
        o.hist_len = up(len, n * sizeof(i32));
        o.gen_start = up(gen, n * sizeof(i32));
        o.ld_hist = longest;
        o.repetition = up(r->repetition, n * F4);
        o.frequency = up(r->frequency, n * F4);
        o.presence = up(r->presence, n * F4);
    }
    if (r->bias_ids) {
        o.bias_ids = up(r->bias_ids, n * r->ld_bias * sizeof(u32));
        o.bias = up(r->bias, n * r->ld_bias * F4);
        o.n_bias = up(r->n_bias, n * sizeof(u32));
        o.ld_bias = r->ld_bias;
    }
    o.mask = up(r->mask, n * words * sizeof(u32));
    o.ld_mask = (u32)words;
    const i32 rc = trlm_logits_rules(d->serve, &o);
    hipDeviceptr_t used[] = { o.history, o.hist_len, o.gen_start, o.repetition, o.frequency, o.presence, o.bias_ids,
                              o.bias, o.n_bias, o.mask };
    for (u32 i = 0; i < sizeof(used) / sizeof(used[0]); i++)
        if (used[i]) hip_free(used[i]);           /* waits for the stream */
    free(tokens);
    free(len);
    free(gen);
    return rc;
}

void gpu_paged_greedy(TrlmPagedDecoder* d, u32* out_ids) {
    if (!d->n) return;
    trlm_bind(d->g);
    trlm_argmax_rows(d->g, d->logits, (i32)d->g->ldv, d->n, d->out_ids);
    hip_d2h(out_ids, d->out_ids, (u64)d->n * sizeof(u32));
}

void gpu_paged_sample(TrlmPagedDecoder* d, PCGState* rngs, f32 temperature, u32* out_ids) {
    if (!d->n) return;
    trlm_bind(d->g);
    f64* u = (f64*)host_mem(d->n, sizeof(f64));
    for (u32 i = 0; i < d->n; i++) u[i] = (f64)pcg_next_u32(&rngs[i]) * (1.0 / 4294967296.0);   /* pcg_uniform */
    hip_h2d(d->u, u, (u64)d->n * sizeof(f64));
    free(u);
    hipDeviceptr_t lg = d->logits, e = d->e, pr = d->prefix, ud = d->u, out = d->out_ids;
    i32 ld = (i32)d->g->ldv, V = (i32)d->g->V, seq = 0;
    void* a1[] = { &lg, &ld, &V, &temperature, &e };
    hip_launch(d->k_sample_exp, d->n, SAMPLE_CHUNKS, 1, SAMPLE_THREADS, 1, 1, 0, a1);
    void* a2[] = { &V, &ld, &ud, &e, &pr, &out, &seq };
    hip_launch(d->k_sample, d->n, 1, 1, SAMPLE_THREADS, 1, 1, 0, a2);
    hip_d2h(out_ids, d->out_ids, (u64)d->n * sizeof(u32));
}

i32 gpu_paged_read(TrlmPagedDecoder* d, u32 seq, u32 layer, f32* k, f32* v) {
    static const char* op = "gpu_paged_read";
    if (seq >= d->max_seqs || layer >= d->g->L) return refuse(op, "a slot or layer out of range");
    const Slot* s = &d->slot[seq];
    if (!s->len) return 0;
    if (!k || !v) return refuse(op, "no place for k or v");
    trlm_bind(d->g);
    const u64 D = d->g->D, n = s->len;
    const i32 q_start[2] = { 0, (i32)n }, len = (i32)n;
    hipDeviceptr_t kd = fl(n * D), vd = fl(n * D);
    hipDeviceptr_t qs = up(q_start, sizeof(q_start)), kl = up(&len, sizeof(len));
    hipDeviceptr_t pg = up(d->table + (u64)seq * d->per, (u64)s->pages * sizeof(i32));
    TrlmKvSeqs q;
    memset(&q, 0, sizeof(q));
    q.n = 1;
    q.rows = (u32)n;
    q.q_start = qs;
    q.kv_len = kl;
    q.pages = pg;
    q.max_pages = s->pages;
    q.max_q = q.max_kv = (u32)n;
    if (trlm_kv_read(d->serve, &d->layer[layer], &q, kd, vd, (u32)D))
        paged_fatal("an operator refused the decoder's own buffers");
    hip_d2h(k, kd, n * D * F4);
    hip_d2h(v, vd, n * D * F4);
    hipDeviceptr_t used[] = { kd, vd, qs, kl, pg };
    for (u32 i = 0; i < sizeof(used) / sizeof(used[0]); i++) hip_free(used[i]);
    return 0;
}
