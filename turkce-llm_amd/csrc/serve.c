/* serve.c -- host side of the serving operators (trlm_serve.h): argument
 * checks, launch shapes, the split of long contexts. */
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#include <unistd.h>

#include "trlm_serve.h"
#include "gpu_internal.h"
#include "kernel_params.h"

#define NHD 4
#define NTYPE 3
static const u32 HDS[NHD] = { 16, 32, 64, 128 };
static const char* const TYPE_NAMES[NTYPE] = { "f32", "bf16", "i8" };

struct TrlmServe {
    HipCtx* ctx;
    i32 device;
    /* looked up on first use of a head width and type */
    hipFunction_t append[NHD][NTYPE][2], read[NHD][NTYPE][2], few[NHD][NTYPE], tile[NHD][NTYPE][2], join[NHD][2];
    hipFunction_t rules[2][2];   /* [narrow, wide][aligned, not] */
};

TrlmServe* trlm_serve_create(HipCtx* ctx) {
    TrlmServe* e = (TrlmServe*)calloc(1, sizeof(TrlmServe));
    if (!e) {
        fprintf(stderr, "[HIP ERROR] trlm_serve_create: out of host memory\n");
        fflush(stderr);
        _exit(1);
    }
    e->ctx = ctx;
    e->device = ctx->device;
    return e;
}

void trlm_serve_destroy(TrlmServe* e) { free(e); }

static i32 refuse(const char* op, const char* why) {
    fprintf(stderr, "%s: refused, nothing launched: %s\n", op, why);
    fflush(stderr);
    return -1;
}

static int unaligned(hipDeviceptr_t p, u64 to) { return !p || ((u64)(uintptr_t)p & (to - 1)) != 0; }
static u64 cdiv64(u64 a, u64 b) { return (a + b - 1) / b; }

static i32 hd_index(u32 hd) {
    for (i32 i = 0; i < NHD; i++)
        if (HDS[i] == hd) return i;
    return -1;
}

static hipFunction_t kernel(TrlmServe* e, hipFunction_t* slot, const char* name) {
    if (!*slot) *slot = hip_get_kernel(e->ctx, name);
    return *slot;
}

static hipFunction_t kernel_hd(TrlmServe* e, hipFunction_t* slot, const char* stem, i32 hd, i32 type) {
    if (!*slot) {
        char name[64];
        if (type < 0) snprintf(name, sizeof(name), "%s_hd%u", stem, HDS[hd]);
        else snprintf(name, sizeof(name), "%s_hd%u_%s", stem, HDS[hd], TYPE_NAMES[type]);
        *slot = hip_get_kernel(e->ctx, name);
    }
    return *slot;
}

/* NULL, or why the handle cannot be used on this thread. */
static const char* handle_fault(const TrlmServe* e) {
    if (!e) return "no handle";
    int cur = -1;
    if (hipGetDevice(&cur) != hipSuccess || cur != e->device) return "the handle belongs to another device than the current one";
    return NULL;
}

/* NULL, or what is wrong with a cache and a call's sequences. */
static const char* cache_fault(const TrlmKvCache* c, const TrlmKvSeqs* s) {
    if (!c || !s) return "no cache or no sequences";
    if (c->type > TRLM_KV_I8) return "unknown cache type";
    if (hd_index(c->head_dim) < 0) return "head_dim must be 16, 32, 64 or 128";
    if (c->kv_heads < 1 || c->kv_heads > 1024) return "kv_heads must be 1 to 1024";
    if (c->page_size < 16 || c->page_size > 65536 || (c->page_size & (c->page_size - 1)))
        return "page_size must be a power of two, 16 to 65536";
    if (c->num_pages < 1 || c->num_pages > 0x7fffffffu) return "num_pages must be 1 to 2^31 - 1";
    if (unaligned(c->k, 16) || unaligned(c->v, 16)) return "k and v must be 16-byte aligned device buffers";
    if (c->type == TRLM_KV_I8 && (unaligned(c->k_scale, 16) || unaligned(c->v_scale, 16)))
        return "an 8-bit cache needs 16-byte aligned k_scale and v_scale";
    if (s->n > TRLM_SERVE_MAX_SEQS) return "more than 4096 sequences";
    if (s->rows >= (1u << 24)) return "rows must be below 2^24";
    if (s->max_pages < 1 || (u64)s->max_pages * c->page_size > (1ull << 30))
        return "max_pages * page_size must be 1 to 2^30";
    if (unaligned(s->q_start, 4) || unaligned(s->kv_len, 4) || unaligned(s->pages, 4))
        return "q_start, kv_len and pages must be 4-byte aligned device buffers";
    return NULL;
}

static u32 shift_of(u32 x) {
    u32 s = 0;
    while ((1u << s) < x) s++;
    return s;
}

static PagedKv paged_kv(const TrlmKvCache* c, const TrlmKvSeqs* s) {
    PagedKv p;
    memset(&p, 0, sizeof(p));
    p.k = c->k; p.v = c->v;
    p.ks = (float*)c->k_scale; p.vs = (float*)c->v_scale;
    p.q_start = (const int*)s->q_start; p.kv_len = (const int*)s->kv_len; p.pages = (const int*)s->pages;
    p.n = (int)s->n; p.rows = (int)s->rows;
    p.num_pages = (int)c->num_pages; p.page_shift = (int)shift_of(c->page_size);
    p.max_pages = (int)s->max_pages; p.kv_heads = (int)c->kv_heads;
    return p;
}

/* A 256-thread workgroup of the append and read kernels moves 1024 / head_dim
 * rows of one head, or of four heads where that still leaves at least four
 * workgroups for each of the 256 compute units: the rows' places and angles are
 * then found once for four heads. */
static int four_heads(u64 rows, u32 hd, u32 heads) { return cdiv64(rows, 1024 / hd) * cdiv64(heads, 4) >= 1024; }

i32 trlm_kv_append(TrlmServe* e, const TrlmKvCache* c, const TrlmKvSeqs* s, const TrlmKvRows* r) {
    static const char* op = "trlm_kv_append";
    const char* why = handle_fault(e);
    if (!why) why = cache_fault(c, s);
    if (why) return refuse(op, why);
    if (!r) return refuse(op, "no rows");
    const u32 hd = c->head_dim;
    if (unaligned(r->k, 16) || unaligned(r->v, 16) || (r->ldk | r->ldv) % 4)
        return refuse(op, "k and v rows must be 16-byte aligned");
    if (r->ldk < c->kv_heads * hd || r->ldv < c->kv_heads * hd || (r->ldk | r->ldv) > 0x7fffffffu)
        return refuse(op, "ldk and ldv must hold a row");
    if (!r->q != !r->heads || !r->q != !r->q_out) return refuse(op, "q, q_out and heads go together");
    if (r->heads > 1024) return refuse(op, "more than 1024 heads");
    if (r->heads && (unaligned(r->q, 16) || unaligned(r->q_out, 16) || (r->ldq | r->ldqo) % 4))
        return refuse(op, "q and q_out rows must be 16-byte aligned");
    if (r->heads && (r->ldq < r->heads * hd || r->ldqo < r->heads * hd || (r->ldq | r->ldqo) > 0x7fffffffu))
        return refuse(op, "ldq and ldqo must hold a row");
    if (r->q_out && r->q_out == r->q && r->ldqo != r->ldq) return refuse(op, "rows turned in place keep their stride");
    if (r->rot_dim % 8 || r->rot_dim > hd) return refuse(op, "rot_dim must be a multiple of 8 up to head_dim");
    if (r->rot_dim && (unaligned(r->cos_t, 16) || unaligned(r->sin_t, 16) || r->max_pos < 1 || r->max_pos > 0x7fffffffu))
        return refuse(op, "a rotation needs 16-byte aligned tables and max_pos");
    if (!s->n || !s->rows) return 0;
    KvAppendParams p;
    memset(&p, 0, sizeof(p));
    p.kv = paged_kv(c, s);
    p.q = (const float*)r->q; p.k = (const float*)r->k; p.v = (const float*)r->v; p.q_out = (float*)r->q_out;
    p.cos_t = (const float*)r->cos_t; p.sin_t = (const float*)r->sin_t;
    p.ldq = (int)r->ldq; p.ldk = (int)r->ldk; p.ldv = (int)r->ldv; p.ldqo = (int)r->ldqo;
    p.heads = (int)r->heads;
    p.max_pos = (int)r->max_pos; p.rot = (int)r->rot_dim; p.rot_half = r->rot_half != 0;
    const i32 i = hd_index(hd);
    const u32 heads = r->heads + 2 * c->kv_heads;
    const int four = four_heads(s->rows, hd, heads);
    void* args[] = { &p };
    hip_launch(kernel_hd(e, &e->append[i][c->type][four], four ? "k_kv_append4" : "k_kv_append", i, (i32)c->type),
               (u32)cdiv64(s->rows, 1024 / hd), (u32)cdiv64(heads, four ? 4 : 1), 1, 256, 1, 1, 0, args);
    return 0;
}

i32 trlm_kv_read(TrlmServe* e, const TrlmKvCache* c, const TrlmKvSeqs* s, hipDeviceptr_t k_out, hipDeviceptr_t v_out,
                 u32 ld) {
    static const char* op = "trlm_kv_read";
    const char* why = handle_fault(e);
    if (!why) why = cache_fault(c, s);
    if (why) return refuse(op, why);
    const u32 hd = c->head_dim;
    if (unaligned(k_out, 16) || unaligned(v_out, 16) || ld % 4) return refuse(op, "output rows must be 16-byte aligned");
    if (ld < c->kv_heads * hd || ld > 0x7fffffffu) return refuse(op, "ld must hold a row");
    if (!s->n || !s->rows) return 0;
    KvReadParams p;
    memset(&p, 0, sizeof(p));
    p.kv = paged_kv(c, s);
    p.k_out = (float*)k_out; p.v_out = (float*)v_out;
    p.ld = (int)ld;
    const i32 i = hd_index(hd);
    const u32 heads = 2 * c->kv_heads;
    const int four = four_heads(s->rows, hd, heads);
    void* args[] = { &p };
    hip_launch(kernel_hd(e, &e->read[i][c->type][four], four ? "k_kv_read4" : "k_kv_read", i, (i32)c->type),
               (u32)cdiv64(s->rows, 1024 / hd), (u32)cdiv64(heads, four ? 4 : 1), 1, 256, 1, 1, 0, args);
    return 0;
}

/* ---------------- attention ---------------- */

#define FEW_TILE 16u      /* rows of a k_paged_attn_few workgroup */
#define FEW_KEYS 128u     /* keys its four waves take at a time: splits are multiples of it */
/* Workgroups of that kernel wanted.  Measured at 512 / 768 / 1024: 8 tokens over
 * 16000 in bf16 69 / 57 / 72 us, 32 over 8192 in 8 bits 97 / 73 / 95, 64 over 1024
 * in fp32 33.1 / 32.9 / 32.8. */
#define FEW_GROUPS 768u
/* Contexts up to which one workgroup takes all keys, two turns of its waves, and
 * saves the join: one token over 200 7.7 us against 9.3; over 500 12.4 against
 * 10.6. */
#define FEW_WHOLE 256u
/* A wave joins a row where the splits are more than 8, or the rows (tokens x
 * heads) too few for a workgroup to take several: one token 9.6 us against 11.5,
 * 1920 rows 13.9 against 15.7; 49152 rows of two splits 29 us against 9. */
#define JOIN_SPLITS 8u
#define JOIN_ROWS 16384u
/* Rows (tokens x group) of a sequence up to which that kernel, which reads the
 * keys once for every 16 rows, is the faster.  Measured, few against many rows'
 * kernel: 24 sequences of 40 rows over 2000 tokens 15.8 / 34 us, 16 of 64 rows
 * over 4000 70 / 147 us; of 128 rows 175 / 121 us. */
#define FEW_MAX 64u
#define TILE_ROWS 256u    /* rows of a k_paged_attn_tile workgroup: its registers fill a compute unit */
#define TILE_KEYS 64u     /* keys of its stages */
/* The kernel that looks its tile up (and spills registers at head_dim 128, 15%)
 * is taken where the tiles that a call's rows make up are less than half of all
 * sequences' at their longest.  Measured, with and without: a prompt of 2048
 * beside 64 single tokens over 1000 94 / 204 us; 8 prompts of 90 to 2000 (28 of
 * 64 tiles) 66 / 93; 64 of 70 to 300 (110 of 128) 57 / 56. */
#define MIXED_MIN 2u
#define CUS 256u
#define MAX_SPLITS 256u

typedef struct AttnPlan {
    u32 few_tiles, tiles;             /* row tiles of a sequence in each kernel (0: not launched) */
    u32 few_splits, tile_splits, chunk_few, chunk_tile, splits;
    u64 few_groups, tile_groups;
    int few_apart;
    int mixed;                        /* tile_groups: what the rows make up, not the longest's for each */
} AttnPlan;

static u32 max_kv_of(const TrlmKvCache* c, const TrlmKvSeqs* s) {
    const u64 held = (u64)s->max_pages * c->page_size;
    return s->max_kv > held ? (u32)held : s->max_kv;
}

/* Splits of kv keys, in multiples of `unit`, so that `groups` row tiles make
 * at least `wanted` workgroups; returns their number. */
static u32 split_keys(u32 kv, u64 groups, u32 wanted, u32 unit, u32* chunk) {
    u64 want = cdiv64(wanted, groups);
    if (want > MAX_SPLITS) want = MAX_SPLITS;
    *chunk = (u32)(cdiv64(cdiv64(kv, want), unit) * unit);
    return (u32)cdiv64(kv, *chunk);
}

/* Splits for row tiles that take a compute unit each.  The time of s splits in
 * keys: rounds of 256 workgroups, each as long as its keys and about 128 more
 * for its start; the join about 64.  Where the new tokens are most of the
 * context the workgroups have all lengths up to a split's and are taken longest
 * first, so that the units share the sum.  Otherwise sequences that are shorter
 * than the longest leave units idle in large splits: among several sequences the
 * most splits within a tenth of the least time are taken.  (Measured, splits and
 * us: 8 x 1024 prompts 2 50.8, 4 56.5; 2048 tokens over 16384 1 1120, 2 1154,
 * 4 1198; 512 over 8192 16 46.1, 32 59.7; 4096 from empty 1 390, 2 296, 4 349;
 * 16 ragged sequences of 32 over 4000 2 170, 4 121.) */
static u32 split_tiles(u32 kv, u32 max_q, u64 groups, u32 n, u32* chunk) {
    u64 best = 0;
    u32 best_s = 1;
    if (max_q > kv) max_q = kv;       /* more new tokens than kept ones: the first see nothing */
    *chunk = (u32)(cdiv64(kv, TILE_KEYS) * TILE_KEYS);
    for (u32 s = 1; s <= MAX_SPLITS && (s == 1 || s * groups <= 4 * CUS); s++) {
        const u32 c = (u32)(cdiv64(cdiv64(kv, s), TILE_KEYS) * TILE_KEYS);
        if (cdiv64(kv, c) != s) continue;
        const u64 wgs = groups * s;
        const int uniform = 2ull * max_q < kv;
        u64 t;
        if (uniform) {
            t = cdiv64(wgs, CUS) * (c + 128);
        } else {
            const u64 share = wgs * c / CUS * (2ull * kv - max_q) / (2ull * kv);
            t = (share > c ? share : c) + 128 * cdiv64(wgs, CUS);
        }
        t += s > 1 ? 64 : 0;
        if (!best || t < best || (uniform && n > 1 && 10 * t <= 11 * best)) {
            if (!best || t < best) best = t;
            best_s = s;
            *chunk = c;
        }
    }
    return best_s;
}

/* A call's launch shape, from what the host knows of it alone, so that a
 * captured call keeps it. */
static AttnPlan attn_plan(const TrlmKvCache* c, const TrlmKvSeqs* s, u32 heads) {
    AttnPlan p;
    memset(&p, 0, sizeof(p));
    const u32 group = heads / c->kv_heads, max_q = s->max_q < s->rows ? s->max_q : s->rows;
    const u32 kv = max_kv_of(c, s) ? max_kv_of(c, s) : 1;
    const u64 most = (u64)max_q * group, seq_heads = (u64)s->n * c->kv_heads;
    p.few_tiles = (u32)cdiv64(most < FEW_MAX ? most : FEW_MAX, FEW_TILE);
    p.few_groups = seq_heads * p.few_tiles;
    /* rest: of the rows, what one sequence at its longest leaves; busy: the row tiles that may have work.  Where
     * they are at most half of the grid, as in calls that mix long and short sequences, the others are kept apart
     * and the splits planned without them (16 sequences of 1 .. 8 tokens, nearly all tiles busy: 38 us, apart 44). */
    const u64 rest = ((u64)s->rows - max_q) * group, few_all = (u64)s->n * p.few_tiles;
    u64 busy = s->n + rest / FEW_TILE;
    p.few_apart = most > FEW_MAX || 2 * busy <= few_all;
    if (!p.few_apart || busy > few_all) busy = few_all;
    p.few_splits = split_keys(kv, busy * c->kv_heads, FEW_GROUPS, FEW_KEYS, &p.chunk_few);
    if (kv <= FEW_WHOLE) {
        p.few_splits = 1;
        p.chunk_few = (u32)(cdiv64(kv, FEW_KEYS) * FEW_KEYS);
    }
    p.chunk_tile = p.chunk_few;
    if (most > FEW_MAX) {
        p.tiles = (u32)cdiv64(most, TILE_ROWS);
        const u64 all = (u64)s->n * p.tiles;
        u64 t = p.tiles + (s->n - 1 < rest / FEW_MAX ? s->n - 1 : rest / FEW_MAX) + rest / TILE_ROWS;
        if (t > all) t = all;
        p.mixed = t * MIXED_MIN < all;
        if (!p.mixed) t = all;
        p.tile_groups = t * c->kv_heads;
        p.tile_splits = split_tiles(kv, max_q, t * c->kv_heads, s->n, &p.chunk_tile);
        /* one sequence, or as many rows as all sequences at their longest: none is short, or should one be
         * (max_q and rows are bounds), the tile kernel takes it too */
        if (s->n == 1 || (u64)s->n * max_q <= s->rows) p.few_splits = 0;
    }
    p.splits = p.tile_splits > p.few_splits ? p.tile_splits : p.few_splits;
    return p;
}

static u64 attn_ws(const TrlmKvCache* c, const TrlmKvSeqs* s, u32 heads, const AttnPlan* p) {
    return p->splits > 1 ? (u64)s->rows * heads * p->splits * (c->head_dim + 2) * sizeof(f32) : 0;
}

u64 trlm_attn_paged_workspace(const TrlmKvCache* c, const TrlmKvSeqs* s, u32 heads) {
    if (cache_fault(c, s) || !heads || heads > 1024 || heads % c->kv_heads || !s->n || !s->rows || !s->max_q) return 0;
    const AttnPlan p = attn_plan(c, s, heads);
    return attn_ws(c, s, heads, &p);
}

i32 trlm_attn_paged(TrlmServe* e, const TrlmKvCache* c, const TrlmKvSeqs* s, hipDeviceptr_t q, u32 ldq, u32 heads,
                    f32 scale, hipDeviceptr_t out, u32 ldo, hipDeviceptr_t ws, u64 ws_bytes) {
    static const char* op = "trlm_attn_paged";
    const char* why = handle_fault(e);
    if (!why) why = cache_fault(c, s);
    if (why) return refuse(op, why);
    const u32 hd = c->head_dim;
    if (!heads || heads > 1024 || heads % c->kv_heads) return refuse(op, "heads must be a multiple of kv_heads, up to 1024");
    if (unaligned(q, 16) || unaligned(out, 16) || (ldq | ldo) % 4) return refuse(op, "q and out rows must be 16-byte aligned");
    if (ldq < heads * hd || ldo < heads * hd || (ldq | ldo) > 0x7fffffffu) return refuse(op, "ldq and ldo must hold a row");
    if (!s->n || !s->rows || !s->max_q) return 0;
    if ((u64)s->rows * heads > 0x7fffffffull) return refuse(op, "rows * heads must be below 2^31");
    const AttnPlan pl = attn_plan(c, s, heads);
    const u64 need = attn_ws(c, s, heads, &pl);
    if (need && (unaligned(ws, 16) || ws_bytes < need)) return refuse(op, "the workspace is too small or not 16-byte aligned");
    const int many = pl.splits > JOIN_SPLITS || (u64)s->rows * heads < JOIN_ROWS;
    const u64 join_groups = pl.splits > 1 ? cdiv64((u64)s->rows * heads, many ? 4 : 1024 / hd) : 0;
    if (pl.few_groups * 256 > 0xffffffffull || pl.tile_groups * 512 > 0xffffffffull || join_groups * 256 > 0xffffffffull)
        return refuse(op, "more work than one launch holds (2^32 threads)");
    PagedAttnParams p;
    memset(&p, 0, sizeof(p));
    p.kv = paged_kv(c, s);
    p.q = (const float*)q; p.out = (float*)out;
    p.part_o = (float*)ws;
    p.part_ml = need ? (float*)ws + (u64)s->rows * heads * pl.splits * hd : NULL;
    p.ldq = (int)ldq; p.ldo = (int)ldo; p.heads = (int)heads;
    p.max_q = (int)(s->max_q < s->rows ? s->max_q : s->rows);
    p.max_kv = (int)max_kv_of(c, s);
    p.few_rows = pl.few_splits ? (int)FEW_MAX : 0;
    p.few_apart = pl.few_apart;
    p.splits = (int)pl.splits; p.chunk_few = (int)pl.chunk_few; p.chunk_tile = (int)pl.chunk_tile;
    p.scale = scale;
    const i32 i = hd_index(hd);
    void* args[] = { &p };
    if (pl.tiles)
        hip_launch(kernel_hd(e, &e->tile[i][c->type][pl.mixed], pl.mixed ? "k_paged_attn_mixed" : "k_paged_attn_tile", i,
                             (i32)c->type), (u32)pl.tile_groups,
                   pl.tile_splits, 1, 512, 1, 1, 0, args);
    if (pl.few_splits)
        hip_launch(kernel_hd(e, &e->few[i][c->type], "k_paged_attn_few", i, (i32)c->type), (u32)pl.few_groups,
                   pl.few_splits, 1, 256, 1, 1, 0, args);
    if (pl.splits > 1)
        hip_launch(kernel_hd(e, &e->join[i][many], many ? "k_paged_attn_join_long" : "k_paged_attn_join", i, -1),
                   (u32)join_groups, 1, 1, 256, 1, 1, 0, args);
    return 0;
}

/* ---------------- rules on logits ---------------- */

/* Tokens a workgroup takes of its row: 1024; or 4096, so that a history is read
 * by fewer of them, where that leaves 16 workgroups for each of the 256 compute
 * units.  Measured, wide against narrow: 64 rows of 31769 tokens and 1024 of
 * history 7.7 / 6.6 us, 64 of 131072 and 2048 16.8 / 15.9, 256 of them 56.5 / 61.1;
 * without a history 50.9 / 46.2. */
#define RULES_WIDE 4096u
#define RULES_NARROW 1024u
#define RULES_WIDE_MIN 4096u

i32 trlm_logits_rules(TrlmServe* e, const TrlmLogitsRules* r) {
    static const char* op = "trlm_logits_rules";
    const char* why = handle_fault(e);
    if (why) return refuse(op, why);
    if (!r) return refuse(op, "no rules");
    if (unaligned(r->logits, 4) || unaligned(r->out, 4)) return refuse(op, "logits and out must be device buffers");
    if (r->vocab < 1 || r->vocab > (1u << 30) || r->ld < r->vocab || r->ld_out < r->vocab)
        return refuse(op, "vocab must be 1 to 2^30 and ld, ld_out at least vocab");
    if (r->rows > 65535) return refuse(op, "more than 65535 rows");
    if (r->out == r->logits && r->ld != r->ld_out) return refuse(op, "rules in place keep the rows' stride");
    if (r->history && (unaligned(r->history, 4) || unaligned(r->hist_len, 4) || !r->ld_hist || r->ld_hist > (1u << 30)))
        return refuse(op, "a history needs its lengths and ld_hist, 1 to 2^30");
    if (r->bias_ids && (unaligned(r->bias_ids, 4) || unaligned(r->bias, 4) || unaligned(r->n_bias, 4) || !r->ld_bias ||
                        r->ld_bias > (1u << 30)))
        return refuse(op, "biases need their ids, values, counts and ld_bias, 1 to 2^30");
    if (r->mask && (unaligned(r->mask, 4) || r->ld_mask < (r->vocab + 31) / 32))
        return refuse(op, "ld_mask must be at least ceil(vocab / 32)");
    if (!r->rows) return 0;
    RulesParams p;
    memset(&p, 0, sizeof(p));
    p.logits = (const float*)r->logits; p.out = (float*)r->out;
    p.history = (const unsigned*)r->history; p.hist_len = (const int*)r->hist_len; p.gen_start = (const int*)r->gen_start;
    p.repetition = (const float*)r->repetition; p.frequency = (const float*)r->frequency;
    p.presence = (const float*)r->presence;
    p.bias_ids = (const unsigned*)r->bias_ids; p.bias = (const float*)r->bias; p.n_bias = (const int*)r->n_bias;
    p.mask = (const unsigned*)r->mask;
    p.ld = r->ld; p.ld_out = r->ld_out; p.ld_hist = r->ld_hist; p.ld_bias = r->ld_bias; p.ld_mask = r->ld_mask;
    p.vocab = (int)r->vocab;
    const int u = unaligned(r->logits, 16) || unaligned(r->out, 16) || (r->ld | r->ld_out) % 4;
    const int wide = r->history && cdiv64(r->vocab, RULES_WIDE) * r->rows >= RULES_WIDE_MIN;
    static const char* const NAMES[2][2] = { { "k_logits_rules_1024", "k_logits_rules_1024_u" },
                                             { "k_logits_rules_4096", "k_logits_rules_4096_u" } };
    void* args[] = { &p };
    hip_launch(kernel(e, &e->rules[wide][u], NAMES[wide][u]), (u32)cdiv64(r->vocab, wide ? RULES_WIDE : RULES_NARROW),
               r->rows, 1, 256, 1, 1, 0, args);
    return 0;
}
