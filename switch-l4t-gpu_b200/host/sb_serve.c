/* sb_serve.c -- host entry points for a batch of requests that share a
 * prompt: page plan, rotary positions with the cache write, attention over
 * the shared prefix and each request's own pages, log probabilities and
 * their gradient.  Each validates its arguments, picks the launch shape and
 * issues its launches on the caller's stream; nothing is allocated, scratch
 * comes from the caller. */
#include <math.h>
#include <string.h>

#include "sb_internal.h"

#define CEIL_DIV(a, b) (((a) + (b)-1) / (b))
#define DP(p) ((CUdeviceptr)(uintptr_t)(p))
#define ALIGNED(p, n) ((((uintptr_t)(p)) & ((n)-1)) == 0)

static int type_size(int type) { return type == SB_F32 ? 4 : 2; }
static int type_ok(int type) { return type == SB_F32 || type == SB_F16 || type == SB_BF16; }
/* kernels of a family stand in the order f32, f16, bf16 */
#define BY_TYPE(f, type) ((sb_fn_id)((f) + (type)))

/* ---------------------------------------------------------------- page plan */
int sb_kv_plan(const int *cache_len, const int *new_len, int B, int page, const int *free_pages, int n_free, int *table,
               int table_stride, int width, int64_t *slots, int *pos, int *req, int T, int *cu_q, int *kv_len, int *used,
               void *stream) {
    SB_ARG(B >= 1 && B <= SB_PLAN_MAX_B, "kv_plan: B must be 1..16384");
    SB_ARG(cache_len && new_len && table && cu_q && kv_len && used, "kv_plan: null pointer");
    SB_ARG(page >= 1 && n_free >= 0 && (free_pages || n_free == 0), "kv_plan: bad page size or free list");
    SB_ARG(width >= 1 && table_stride >= width, "kv_plan: table_stride must be at least the width");
    SB_ARG(kv_len != cache_len && kv_len != new_len && cu_q != cache_len && cu_q != new_len, "kv_plan: outputs over the input lengths");
    SB_ARG(T >= 0 && T <= 0x7ffffff0 && ((slots && pos && req) || T == 0), "kv_plan: bad token arrays");
    sb_ctx *c = sb_ctx_get();
    if (!c) return SB_ERR_STATE;
    CUdeviceptr cl = DP(cache_len), nl = DP(new_len), fp = DP(free_pages), tb = DP(table), sl = DP(slots), po = DP(pos),
                rq = DP(req), cq = DP(cu_q), kl = DP(kv_len), us = DP(used);
    void *args[] = {&cl, &nl, &B, &page, &fp, &n_free, &tb, &table_stride, &width, &sl, &po, &rq, &T, &cq, &kl, &us};
    /* a decode step of up to 128 requests is one small CTA (its barriers are
     * cheaper); else enough CTAs for four tokens a thread and a warp a
     * request, two per SM at most */
    const int threads = B <= 128 && T <= 512 ? 128 : 512;
    long g = CEIL_DIV((long)T, 4L * threads), gb = CEIL_DIV(B, threads / 32);
    if (gb > g && threads == 512) g = gb;
    if (g > 2L * c->sms) g = 2L * c->sms;
    return sb_launch(c, F_KV_PLAN, (unsigned)(g < 1 ? 1 : g), 1, (unsigned)threads, (unsigned)(2 * (B + 1) * 4), (CUstream)stream, args, 0);
}

/* ---------------------------------------------------------------- rotary */
int sb_rotary_plan_init(sb_rotary_plan *r, int dim, int layout, double theta, int scaling, double factor, int orig_ctx) {
    SB_ARG(r, "rotary_plan_init: null pointer");
    SB_ARG(dim >= 2 && dim <= SB_ROTARY_MAX_DIM && dim % 2 == 0, "rotary_plan_init: dim must be even, 2..256");
    SB_ARG(layout == SB_ROPE_HALF || layout == SB_ROPE_PAIRS, "rotary_plan_init: unknown layout");
    SB_ARG(isfinite(theta) && theta > 1.0, "rotary_plan_init: theta must be above 1");
    SB_ARG(scaling >= SB_ROPE_PLAIN && scaling <= SB_ROPE_BANDS, "rotary_plan_init: unknown scaling");
    SB_ARG(scaling == SB_ROPE_PLAIN || (isfinite(factor) && factor >= 1.0), "rotary_plan_init: factor must be at least 1");
    SB_ARG(scaling < SB_ROPE_YARN || orig_ctx >= 1, "rotary_plan_init: this scaling needs the trained context");
    SB_ARG(scaling != SB_ROPE_NTK || dim > 2, "rotary_plan_init: this scaling needs dim > 2");
    const double pi2 = 6.283185307179586476925286766559;
    /* frequencies in long double (64-bit mantissa): a double's half unit is 2^-25 turns at a position of 2^31 */
    const long double pi2l = 6.283185307179586476925286766559L;
    long double base = theta;
    double lo = 0, hi = 0;
    if (scaling == SB_ROPE_NTK) base *= powl(factor, dim / (dim - 2.0L));
    if (scaling == SB_ROPE_YARN) { /* pairs that turn 32 times and once over the trained context */
        lo = floor(dim * log(orig_ctx / (32.0 * pi2)) / (2.0 * log(theta)));
        hi = ceil(dim * log(orig_ctx / pi2) / (2.0 * log(theta)));
        if (lo < 0) lo = 0;
        if (hi > dim - 1) hi = dim - 1;
    }
    memset(r, 0, sizeof *r);
    r->dim = dim;
    r->layout = layout;
    r->mscale = 1.0f;
    if (scaling == SB_ROPE_YARN) r->mscale = (float)(0.1 * log(factor) + 1.0);
    for (int i = 0; i < dim / 2; i++) {
        long double f = powl(base, -2.0L * i / dim);
        if (scaling == SB_ROPE_LINEAR) f /= factor;
        if (scaling == SB_ROPE_YARN) {
            long double ramp = (i - lo) / (hi > lo ? hi - lo : 0.001L);
            ramp = ramp < 0 ? 0 : ramp > 1 ? 1 : ramp;
            f = f / factor * ramp + f * (1 - ramp);
        }
        if (scaling == SB_ROPE_BANDS) { /* turns over the trained context: 1 and fewer stretched, 4 and more kept */
            long double s = (orig_ctx * f / pi2l - 1) / 3;
            s = s < 0 ? 0 : s > 1 ? 1 : s;
            f = f / factor * (1 - s) + f * s;
        }
        r->turn[i] = (uint64_t)(f / pi2l * 18446744073709551616.0L + 0.5L); /* turns per position in units of 2^-64 */
    }
    return 0;
}

/* mirrors RotParams in csrc/serve_rotary.cuh */
struct rot_params {
    CUdeviceptr src[3], dst[3];
    int64_t st[3], sh[3], dt, dh, page_stride, pos_stride, head_stride;
    CUdeviceptr pos, slots;
    int64_t n_slots;
    int T, heads[3], HD, dim, layout, inverse, page, tokens_per_cta;
    float mscale;
    uint64_t turn[SB_ROTARY_MAX_DIM / 2];
};
static int rotary_launch(struct rot_params *p, const sb_rotary_plan *r, int type, int vec, void *stream) {
    sb_ctx *c = sb_ctx_get();
    if (!c) return SB_ERR_STATE;
    if (p->T == 0) return 0;
    p->dim = r->dim;
    p->layout = r->layout;
    p->mscale = r->mscale;
    memcpy(p->turn, r->turn, sizeof p->turn);
    const int V = vec ? 16 / type_size(type) : 1;
    const long H = p->heads[0] + p->heads[1] + p->heads[2], units = H * (p->HD / (2 * V));
    /* tokens per CTA: up to 4 while that leaves two CTAs per SM (8: more idle at
     * the end, 4099 tokens of 14 heads of 64 in FP32 6.7 against 6.0 us); a
     * single token's heads are spread over several CTAs when they exceed one pass */
    int tok = 4;
    while (tok > 1 && (CEIL_DIV(p->T, tok) < 2L * c->sms || tok * units > 8 * 256)) tok >>= 1;
    p->tokens_per_cta = tok;
    long gy = 1;
    const long gx = CEIL_DIV(p->T, tok);
    if (gx < 2L * c->sms) gy = CEIL_DIV(tok * units, 256);
    if (gy > 64) gy = 64;
    void *args[] = {p};
    return sb_launch(c, vec ? BY_TYPE(F_ROTARY_F32, type) : BY_TYPE(F_ROTARY_F32_ANY, type), (unsigned)gx, (unsigned)gy, 256, 0,
                     (CUstream)stream, args, 0);
}
static int rotary_args(const sb_rotary_plan *r, int type, int T, int HD) {
    SB_ARG(r && r->dim >= 2 && r->dim <= SB_ROTARY_MAX_DIM && r->dim % 2 == 0, "rotary: plan not initialised");
    SB_ARG(r->layout == SB_ROPE_HALF || r->layout == SB_ROPE_PAIRS, "rotary: plan not initialised");
    SB_ARG(type_ok(type), "rotary: unknown element type");
    SB_ARG(T >= 0 && HD >= r->dim && HD % 2 == 0, "rotary: need an even head size of at least the rotated part");
    return 0;
}
/* all vectors of a row family start on 16 bytes */
static int vec_ok(int type, const void *p, int64_t a, int64_t b, int64_t c) {
    const int64_t V = 16 / type_size(type);
    return ALIGNED(p, 16) && a % V == 0 && b % V == 0 && c % V == 0;
}

int sb_rotary(const void *x, int64_t x_tok, int64_t x_head, void *y, int64_t y_tok, int64_t y_head, int type, int T, int H,
              int HD, const int *pos, const sb_rotary_plan *r, int inverse, void *stream) {
    int rc = rotary_args(r, type, T, HD);
    if (rc) return rc;
    SB_ARG(H >= 1 && ((x && y && pos) || T == 0), "rotary: null pointer");
    SB_ARG(ALIGNED(x, type_size(type)) && ALIGNED(y, type_size(type)), "rotary: misaligned rows");
    SB_ARG(x != y || ((T <= 1 || x_tok == y_tok) && (H == 1 || x_head == y_head)), "rotary: in place needs one set of strides");
    struct rot_params p;
    memset(&p, 0, sizeof p);
    p.src[0] = DP(x);
    p.dst[0] = DP(y);
    p.st[0] = x_tok;
    p.sh[0] = x_head;
    p.dt = y_tok;
    p.dh = y_head;
    p.pos = DP(pos);
    p.T = T;
    p.heads[0] = H;
    p.HD = HD;
    p.page = 1;
    p.inverse = inverse != 0;
    const int V = 16 / type_size(type);
    const int vec = vec_ok(type, x, x_tok, x_head, 0) && vec_ok(type, y, y_tok, y_head, 0) && r->dim % (2 * V) == 0 && HD % (2 * V) == 0;
    return rotary_launch(&p, r, type, vec, stream);
}

static int pages_args(const sb_kv_pages *kv) {
    SB_ARG(kv && kv->k && kv->v, "pages: null pointer");
    SB_ARG(type_ok(kv->type), "pages: unknown element type");
    SB_ARG(kv->n_pages >= 1 && kv->page >= 1 && kv->NKV >= 1 && kv->HD >= 1, "pages: bad sizes");
    SB_ARG(kv->page_stride >= 0 && kv->pos_stride >= 0 && kv->head_stride >= 0, "pages: negative strides");
    return 0;
}

int sb_rotary_kv(const void *q, int64_t q_tok, int64_t q_head, void *q_out, int64_t qo_tok, int64_t qo_head, const void *k,
                 int64_t k_tok, int64_t k_head, const void *v, int64_t v_tok, int64_t v_head, int T, int NH, const int *pos,
                 const int64_t *slots, const sb_rotary_plan *r, const sb_kv_pages *kv, void *stream) {
    int rc = pages_args(kv);
    if (!rc) rc = rotary_args(r, kv->type, T, kv->HD);
    if (rc) return rc;
    SB_ARG(NH >= 1 && ((q && q_out && k && v && pos && slots) || T == 0), "rotary_kv: null pointer");
    const int e = type_size(kv->type);
    SB_ARG(ALIGNED(q, e) && ALIGNED(q_out, e) && ALIGNED(k, e) && ALIGNED(v, e) && ALIGNED(kv->k, e) && ALIGNED(kv->v, e),
           "rotary_kv: misaligned rows");
    SB_ARG(q != q_out || ((T <= 1 || q_tok == qo_tok) && (NH == 1 || q_head == qo_head)), "rotary_kv: in place needs one set of strides");
    struct rot_params p;
    memset(&p, 0, sizeof p);
    p.src[0] = DP(q);
    p.src[1] = DP(k);
    p.src[2] = DP(v);
    p.dst[0] = DP(q_out);
    p.dst[1] = DP(kv->k);
    p.dst[2] = DP(kv->v);
    p.st[0] = q_tok;
    p.sh[0] = q_head;
    p.st[1] = k_tok;
    p.sh[1] = k_head;
    p.st[2] = v_tok;
    p.sh[2] = v_head;
    p.dt = qo_tok;
    p.dh = qo_head;
    p.page_stride = kv->page_stride;
    p.pos_stride = kv->pos_stride;
    p.head_stride = kv->head_stride;
    p.pos = DP(pos);
    p.slots = DP(slots);
    p.n_slots = (int64_t)kv->n_pages * kv->page;
    p.T = T;
    p.heads[0] = NH;
    p.heads[1] = p.heads[2] = kv->NKV;
    p.HD = kv->HD;
    p.page = kv->page;
    const int V = 16 / e;
    const int vec = vec_ok(kv->type, q, q_tok, q_head, 0) && vec_ok(kv->type, q_out, qo_tok, qo_head, 0) &&
                    vec_ok(kv->type, k, k_tok, k_head, 0) && vec_ok(kv->type, v, v_tok, v_head, 0) &&
                    vec_ok(kv->type, kv->k, kv->page_stride, kv->pos_stride, kv->head_stride) && ALIGNED(kv->v, 16) &&
                    r->dim % (2 * V) == 0 && kv->HD % (2 * V) == 0;
    return rotary_launch(&p, r, kv->type, vec, stream);
}

/* ---------------------------------------------------------------- attention */
/* mirrors AttnParams in csrc/serve_attn.cuh */
struct attn_pages {
    CUdeviceptr k, v;
    int64_t page_stride, pos_stride, head_stride;
    int n_pages, page, shift;
};
struct attn_params {
    CUdeviceptr q, out, lse, cu_q, ptable, table, kv_len, ws_o, ws_ml, ws_n;
    int64_t q_row, q_head, o_row, o_head;
    struct attn_pages pre, suf;
    int T, B, NH, NKV, G, HD, P, max_kv, table_stride;
    int chunk1, S1, tiles1, chunk2, S2, tiles2, items1, deep;
    float scale_log2;
    unsigned call;
    int test_skip;
};
/* a number for every call (a kernel that gives up stops its own call only), and the test hook */
static unsigned attn_calls;
static int attn_test_skip;
int sb_attn_set_test_skip(int tile) {
    SB_ARG(tile >= -1 && tile < 1 << 30, "tile must be >= -1");
    __atomic_store_n(&attn_test_skip, tile + 1, __ATOMIC_RELAXED);
    return 0;
}
/* Shared memory of the kernels with a ring a warp: 8 KB (16-bit types: K and V
 * tiles of 16 keys, one each for heads of 128, two for 64; four and six CTAs an SM)
 * or 16 KB (FP32, and long items of heads of 128: two each, three CTAs).  256
 * requests in BF16, 32 / 8 heads of 128, up to 40 keys: 17.7 and 22.8 us; 250:
 * 30 and 35; 500: 49 and 49; 1000: 88 and 86; 24 / 3 heads of 96, up to 500:
 * 18.4 and 22; 1000: 81 and 43; 2000: 158 and 83 */
#define SB_ATTN_SHALLOW 32768u
#define SB_ATTN_DEEP 65536u
#define SB_ATTN_DEEP_TILES 8
/* one of the two launches: kernel, row tiles, key ranges, items */
struct attn_part {
    sb_fn_id f;
    unsigned smem, threads;
    int f32, wide, rows, step, tiles, S, chunk;
    long grid;
};

/* The kernel for `rows` query rows of a key head.  FP32: row tiles of 1, 2,
 * 4, 8 or 16, the smallest that holds them (unused rows cost FMAs).  16-bit
 * types: a tile of 8 or 16 rows (the four warps split the keys) while it holds
 * all rows; beyond that the prefix goes to the tcgen05 kernel's 256 rows, most
 * of them empty at first (20 rows behind 300 keys, 32/8 heads of 128: 12.5
 * against 15.1 us for 64-row tiles of mma.sync; 100 behind 16000: 27.6 against
 * 49.5), and own rows, each with its own limit, to 64-row tiles (which leaves
 * a prompt's own rows at 0.12 of the tensor peak: four of 2048 rows, 32 / 8
 * heads of 128, in BF16 348 us). */
static void attn_kernel(int type, int HD, long rows, int prefix, struct attn_part *a) {
    const int wide = HD > 64, second = type == SB_BF16;
    a->threads = 128;
    a->smem = SB_ATTN_DEEP;
    a->f32 = type == SB_F32;
    a->wide = wide;
    if (type == SB_F32) {
        int i = 0;
        while (i < 4 && (1 << i) < rows) i++;
        a->f = (sb_fn_id)(F_ATTN_F32_64_R1 + 5 * wide + i);
        a->rows = 1 << i;
        a->step = wide ? 32 : 64;
    } else if (prefix && rows > 16) {
        a->f = (sb_fn_id)(F_ATTN_TC_F16_64 + 2 * second + wide);
        a->smem = 1024 + (wide ? 6 * 32768 : 10 * 16384);
        a->threads = 512;
        a->rows = 256;
        a->step = 128;
    } else {
        const int big = rows > 16;
        a->f = rows <= 8 ? (sb_fn_id)(F_ATTN_F16_64_R8 + 2 * second + wide)
                         : big ? (sb_fn_id)(F_ATTN_F16_64_R64 + 2 * second + wide)
                               : (sb_fn_id)(F_ATTN_F16_64_R16 + 2 * second + wide);
        a->smem = big ? 2 * 64 * 2 * (wide ? 2 * 128 : 3 * 64) : SB_ATTN_SHALLOW;
        a->rows = rows <= 8 ? 8 : big ? 64 : 16;
        a->step = 64;
    }
    a->tiles = (int)CEIL_DIV(rows, a->rows);
}
/* Key ranges of `keys` keys for `units` independent (head, row tile) pairs,
 * the count with the least cost in tile times: an item of n tiles of keys
 * takes about n + SB_ATTN_ITEM of them (its queries, its part to write), and
 * every part of `bytes` is written and read again by the join (a tile takes
 * 0.5 us, 2 us on the tcgen05 kernel; parts move at about 4 MB / us).  Items
 * of one length run in rounds on `sms` SMs; `ragged` ones (requests are shorter
 * than the longest: half its length) fill in for one another, and the longest
 * is left at the end.  In FP32 half the items, in rounds, choose better (48
 * requests of 12 heads of 64, up to 777 own keys: 25.1 us, by total and longest
 * item 28; 16 of up to 2000 behind 1000: 38.9 and 41.7; 30 of 32 / 8 heads of
 * 128, up to 3000: 100 and 108; 200 of up to 1000: 294 and 297).  `alone`: one
 * range would need no join. */
static void attn_split(sb_ctx *c, struct attn_part *a, int keys, long units, long bytes, long sms, int ragged, int alone) {
    const long tiles = CEIL_DIV(keys, a->step), move = a->threads == 512 ? 8L << 20 : 2L << 20;
    for (;;) {
        const long cap = sms * sb_occupancy_of(c, a->f, (int)a->threads, a->smem);
        long best = 0, best_cost = 0;
        for (long S = 1; S <= SB_ATTN_MAX_SPLITS && S <= tiles; S++) {
            const long n = CEIL_DIV(tiles, S), parts = CEIL_DIV(tiles, n), items = units * parts;
            const long run = ragged && !a->f32 ? 8 * units * (tiles + (parts + 1) * SB_ATTN_ITEM) / cap + 16 * (n + SB_ATTN_ITEM)
                                               : 16 * CEIL_DIV(items, ragged ? 2 * cap : cap) * (n + SB_ATTN_ITEM);
            const long cost = run + 2 * parts + 16 * parts * bytes / move + (alone && parts > 1 ? 16 * SB_ATTN_ITEM : 0);
            if (!best || cost < best_cost) {
                best = n;
                best_cost = cost;
            }
            if (items > 32 * cap) break;
        }
        a->chunk = (int)(best * a->step);
        a->S = (int)CEIL_DIV((long)keys, a->chunk);
        a->grid = units * a->S;
        if (a->smem != SB_ATTN_SHALLOW || !a->wide || best <= SB_ATTN_DEEP_TILES) return;
        a->smem = SB_ATTN_DEEP;
    }
}
static int attn_parts(sb_ctx *c, int type, int T, int B, int NH, int NKV, int HD, int max_q, int P, int max_kv,
                      struct attn_part *pre, struct attn_part *own) {
    const long G = NH / NKV, bytes = (long)T * NH * HD * 8;
    memset(pre, 0, sizeof *pre);
    memset(own, 0, sizeof *own);
    if (max_kv > 0) {
        attn_kernel(type, HD, max_q * G, 0, own);
        attn_split(c, own, max_kv, (long)own->tiles * NKV * B, bytes, c->sms, 1, P == 0);
    }
    if (P > 0) {
        attn_kernel(type, HD, T * G, 1, pre);
        const long units = (long)pre->tiles * NKV;
        long sms = c->sms;
        if (max_kv > 0 && pre->threads == 512) {
            /* The tcgen05 kernel fills an SM, so it gets the share of the SMs
             * that it has in the work, in units of 0.2 us of one SM, and the
             * own items run beside it on the others (a tile of either kernel's
             * 2 and 1.2 us; half the longest length).  256 requests behind
             * 16000 tokens, 32 / 8 heads of 128, in BF16: 103 to 110 us, all
             * SMs to one after the other 126; 32 requests of up to 33 rows
             * behind 4001, 14 / 2 heads of 64: 32 and 37 */
            const long mine = units * CEIL_DIV(P, pre->step) * 10;
            const long others = own->grid * (own->chunk / own->step + 2 * SB_ATTN_ITEM) * 3 / sb_occupancy_of(c, own->f, 128, own->smem);
            sms = sms * mine / (mine + others);
            if (sms < 1) sms = 1;
        }
        attn_split(c, pre, P, units, bytes, sms, 0, max_kv == 0);
    }
    if (P > 0 && max_kv > 0 && pre->f != own->f && pre->threads == 128 && pre->rows > own->rows &&
        pre->grid + own->grid <= (long)c->sms * sb_occupancy_of(c, pre->f, 128, pre->smem)) {
        /* a call that does not fill the card is bound by its launches: the
         * requests' rows go through the prefix' kernel too, in one launch (4
         * requests behind 300 tokens in FP32: 13.6 us instead of 15.2) */
        const int tiles = (int)CEIL_DIV(max_q * G, pre->rows);
        own->f = pre->f;
        own->smem = pre->smem;
        own->rows = pre->rows;
        own->tiles = tiles;
        attn_split(c, own, max_kv, (long)tiles * NKV * B, bytes, c->sms, 1, 0);
    }
    if (pre->f == own->f) pre->smem = own->smem = pre->smem > own->smem ? pre->smem : own->smem; /* one launch */
    SB_ARG(pre->grid + own->grid < 0x7fffffffL, "attn_prefix: too many rows for one launch");
    return 0;
}
static size_t attn_ws_bytes(int T, int NH, int HD, const struct attn_part *pre, const struct attn_part *own) {
    const size_t rows = (size_t)T * NH, S = (size_t)pre->S + own->S;
    if (S <= 1) return 0;
    return rows * S * HD * 4 + rows * S * 8 + (size_t)T * 4;
}
static int attn_args(int type, int T, int B, int NH, int NKV, int HD, int max_q, int P, int max_kv) {
    SB_ARG(type_ok(type), "attn_prefix: unknown element type");
    SB_ARG(T >= 0 && B >= 0 && NH >= 1 && NKV >= 1 && NH % NKV == 0, "attn_prefix: need T, B >= 0 and NH % NKV == 0");
    SB_ARG(HD >= 8 && HD <= 128 && HD % 8 == 0, "attn_prefix: the head size must be a multiple of 8, at most 128");
    SB_ARG(max_q >= 1 && P >= 0 && max_kv >= 0 && P <= (1 << 30) && max_kv <= (1 << 30), "attn_prefix: bad lengths");
    SB_ARG((int64_t)T * (NH / NKV) < (1 << 30) && (int64_t)max_q * (NH / NKV) < (1 << 30), "attn_prefix: too many rows");
    return 0;
}

int sb_attn_prefix_ws(int type, int T, int B, int NH, int NKV, int HD, int max_q, int prefix_len, int max_kv, size_t *bytes) {
    SB_ARG(bytes, "null pointer");
    int rc = attn_args(type, T, B, NH, NKV, HD, max_q, prefix_len, max_kv);
    if (rc) return rc;
    *bytes = 0;
    if (T == 0 || B == 0) return 0;
    sb_ctx *c = sb_ctx_get();
    if (!c) return SB_ERR_STATE;
    struct attn_part pre, own;
    rc = attn_parts(c, type, T, B, NH, NKV, HD, max_q, prefix_len, max_kv, &pre, &own);
    if (rc) return rc;
    *bytes = attn_ws_bytes(T, NH, HD, &pre, &own);
    return 0;
}

static int pages_for_attn(const sb_kv_pages *kv, struct attn_pages *p) {
    const int e = type_size(kv->type);
    SB_ARG(vec_ok(kv->type, kv->k, kv->page_stride, kv->pos_stride, kv->head_stride) && ALIGNED(kv->v, 16) && e,
           "attn_prefix: pages need 16-byte aligned rows");
    p->k = DP(kv->k);
    p->v = DP(kv->v);
    p->page_stride = kv->page_stride;
    p->pos_stride = kv->pos_stride;
    p->head_stride = kv->head_stride;
    p->n_pages = kv->n_pages;
    p->page = kv->page;
    p->shift = -1;
    for (int i = 0; i < 31; i++)
        if (kv->page == 1 << i) p->shift = i;
    return 0;
}

/* Tensor maps of K and V pages, {HD, heads, positions, pages} with boxes of 128
 * bytes of one head x `box` positions, 128-byte swizzle; what is past HD reads
 * as zero.  Returns the box: pages, or parts of `most` positions of one (a
 * smaller page must divide it, and hold eight positions: the swizzle's
 * period); 0 where pages of this size, or strides that a map cannot hold, go
 * through the kernels' own copies (256 requests behind 16000 in BF16: 107 us
 * with pages of 16, 32, 64 or 128, 147 with 24 or 48, 154 with 96; 32 of up to
 * 33 rows behind 4001 in FP16: 32.4 and 35.8). */
static int encode_pages(CUtensorMap *tk, CUtensorMap *tv, const sb_kv_pages *kv, int most) {
    const int e = type_size(kv->type), box = kv->page % most == 0 ? most : most % kv->page == 0 && kv->page >= 8 ? kv->page : 0;
    const cuuint64_t dims[4] = {(cuuint64_t)kv->HD, (cuuint64_t)kv->NKV, (cuuint64_t)kv->page, (cuuint64_t)kv->n_pages};
    const cuuint64_t strides[3] = {(cuuint64_t)kv->head_stride * e, (cuuint64_t)kv->pos_stride * e, (cuuint64_t)kv->page_stride * e};
    const cuuint32_t size[4] = {(cuuint32_t)(128 / e), 1, (cuuint32_t)box, 1}, estr[4] = {1, 1, 1, 1};
    const CUtensorMapDataType type = e == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16;
    for (int i = 0; box && i < 2; i++)
        if (cuTensorMapEncodeTiled(i ? tv : tk, type, 4, i ? kv->v : kv->k, dims, strides, size, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return 0;
    return box;
}
/* positions of a box: what one warp of the kernel loads at a time */
static int attn_box(const struct attn_part *a, int type, int HD) { return a->threads == 512 ? 64 : type == SB_F32 && HD > 64 ? 8 : 16; }

int sb_attn_prefix(const void *q, int64_t q_row, int64_t q_head, void *out, int64_t o_row, int64_t o_head, float *lse, int T,
                   int NH, const int *cu_q, int B, int max_q, const sb_kv_pages *prefix, const int *prefix_table,
                   int prefix_len, const sb_kv_pages *kv, const int *table, int table_stride, const int *kv_len, int max_kv,
                   float scale, void *ws, size_t ws_bytes, void *stream) {
    const sb_kv_pages *any = prefix_len > 0 || (max_kv <= 0 && !kv) ? prefix : kv;
    int rc = pages_args(any);
    if (!rc && prefix_len > 0 && max_kv > 0) rc = pages_args(kv);
    if (!rc) rc = attn_args(any->type, T, B, NH, any->NKV, any->HD, max_q, prefix_len, max_kv);
    if (rc) return rc;
    SB_ARG(isfinite(scale * 1.4426950408889634f), "attn_prefix: scale must be finite");
    SB_ARG(cu_q || (T == B && max_q == 1), "attn_prefix: without cu_q there is one row a request (T == B, max_q == 1)");
    if (T == 0 || B == 0) return 0;
    SB_ARG(q && out && ALIGNED(lse, 4), "attn_prefix: null or misaligned pointer");
    SB_ARG(vec_ok(any->type, q, q_row, q_head, 0) && vec_ok(any->type, out, o_row, o_head, 0),
           "attn_prefix: query and output rows must be 16-byte aligned");
    struct attn_params p;
    memset(&p, 0, sizeof p);
    if (prefix_len > 0) {
        SB_ARG(prefix_table || prefix_len <= (int64_t)prefix->n_pages * prefix->page, "attn_prefix: the prefix exceeds its pages");
        if ((rc = pages_for_attn(prefix, &p.pre))) return rc;
    }
    if (max_kv > 0) {
        SB_ARG(table && kv_len, "attn_prefix: null table or lengths");
        SB_ARG(kv->type == any->type && kv->NKV == any->NKV && kv->HD == any->HD,
               "attn_prefix: prefix and own pages must have one type, head count and head size");
        SB_ARG(table_stride >= CEIL_DIV((int64_t)max_kv, kv->page), "attn_prefix: the table is narrower than max_kv positions");
        if ((rc = pages_for_attn(kv, &p.suf))) return rc;
    }
    sb_ctx *c = sb_ctx_get();
    if (!c) return SB_ERR_STATE;
    const int type = any->type, NKV = any->NKV, HD = any->HD;
    struct attn_part pre, own;
    rc = attn_parts(c, type, T, B, NH, NKV, HD, max_q, prefix_len, max_kv, &pre, &own);
    if (rc) return rc;
    const size_t need = attn_ws_bytes(T, NH, HD, &pre, &own);
    SB_ARG(ws_bytes >= need && (ws || need == 0) && ALIGNED(ws, 32), "attn_prefix: workspace too small (sb_attn_prefix_ws) or misaligned");
    const size_t parts = (size_t)T * NH * (pre.S + own.S);
    p.q = DP(q);
    p.out = DP(out);
    p.lse = DP(lse);
    p.cu_q = DP(cu_q);
    p.ptable = DP(prefix_table);
    p.table = DP(table);
    p.kv_len = DP(kv_len);
    if (need) {
        p.ws_o = DP(ws);
        p.ws_ml = p.ws_o + parts * HD * 4;
        p.ws_n = p.ws_ml + parts * 8;
    }
    p.q_row = q_row;
    p.q_head = q_head;
    p.o_row = o_row;
    p.o_head = o_head;
    p.T = T;
    p.B = B;
    p.NH = NH;
    p.NKV = NKV;
    p.G = NH / NKV;
    p.HD = HD;
    p.P = prefix_len;
    p.max_kv = max_kv;
    p.table_stride = table_stride;
    p.chunk1 = pre.chunk;
    p.S1 = pre.S;
    p.tiles1 = pre.tiles;
    p.chunk2 = own.chunk;
    p.S2 = own.S;
    p.tiles2 = own.tiles;
    p.scale_log2 = scale * 1.4426950408889634f;
    do p.call = __atomic_add_fetch(&attn_calls, 1, __ATOMIC_RELAXED);
    while (p.call == 0);
    p.test_skip = __atomic_load_n(&attn_test_skip, __ATOMIC_RELAXED);
    CUtensorMap tk, tv;
    int box = 0;
    memset(&tk, 0, sizeof tk);
    memset(&tv, 0, sizeof tv);
    void *args[] = {&p, &tk, &tv, &box};
    /* Two maps cost a microsecond of the host: not for a call that is over in a
     * few, nor for a launch whose two parts have pools of their own.  The
     * tcgen05 kernel's own copies take longer than that. */
    /* Order.  tcgen05 items that the own items would keep waiting go first: each
     * takes an SM, the own items those left.  Otherwise own items first, the
     * smaller kernel: prefix items start where SMs have room (48 requests
     * behind 1000 tokens in FP32: 38.2 us, the prefix first 45.4), and the join
     * does not wait for a third launch in line (6 requests behind 1819, 20 / 4
     * heads of 80, in FP16: 13.4 and 15.2) */
    const int apart = own.S && own.f != pre.f, tc = pre.threads == 512;
    const int prefix_first = tc && pre.grid + (own.grid < c->sms ? own.grid : c->sms) > c->sms;
    for (int i = 0; i < 2; i++) {
        const int of_prefix = (i == 0) == prefix_first, second = i == 1 && pre.S && apart;
        if (of_prefix ? !pre.S : !apart) continue;
        if (of_prefix) {
            const long grid = pre.grid + (apart ? 0 : own.grid);
            p.items1 = (int)pre.grid;
            p.deep = pre.smem == SB_ATTN_DEEP;
            box = 0;
            if (grid == pre.grid && (tc || grid * pre.chunk >= SB_ATTN_TMA_KEYS)) box = encode_pages(&tk, &tv, prefix, attn_box(&pre, type, HD));
            rc = sb_launch(c, pre.f, (unsigned)grid, 1, pre.threads, pre.smem, (CUstream)stream, args, second);
        } else {
            p.items1 = box = 0;
            p.deep = own.smem == SB_ATTN_DEEP;
            if (own.grid * (long)own.chunk >= SB_ATTN_TMA_KEYS) box = encode_pages(&tk, &tv, kv, attn_box(&own, type, HD));
            rc = sb_launch(c, own.f, (unsigned)own.grid, 1, own.threads, own.smem, (CUstream)stream, args, second);
        }
        if (rc) return rc;
    }
    if (pre.S + own.S == 1) return 0;
    long g = CEIL_DIV((long)T * NH, 4);
    if (g > 16L * c->sms) g = 16L * c->sms;
    void *join_args[] = {&p, (void *)&type};
    return sb_launch(c, F_ATTN_JOIN, (unsigned)g, 1, 128, 0, (CUstream)stream, join_args, 1);
}

/* ---------------------------------------------------------------- log probabilities */
/* mirrors LpParams / LpGradParams in csrc/score_kernels.cu */
struct lp_params {
    CUdeviceptr x;
    int64_t stride;
    int R, V, S, k;
    float c, inv_temp;
    CUdeviceptr tok, logp, entropy, lse, rank, top_ids, top_logp, part, keys;
};
struct lp_grad_params {
    CUdeviceptr x, dx;
    int64_t stride, dstride;
    int R, V, S;
    float c, inv_temp;
    CUdeviceptr tok, lse, entropy, g_logp, g_entropy;
};
/* parts of a row: one where the rows fill the SMs (no join, and the bound of
 * the alternatives is renewed less often), else enough for `waves` CTAs per
 * SM, 4 KB of logits each at least */
static int lp_parts(sb_ctx *c, int R, int V, int type, long waves) {
    long S = R >= 4L * c->sms ? 1 : CEIL_DIV(waves * c->sms, (long)R), most = (long)V * type_size(type) / 4096;
    if (S > most) S = most;
    if (S > SB_LOGPROBS_MAX_PARTS) S = SB_LOGPROBS_MAX_PARTS;
    return (int)(S < 1 ? 1 : S);
}
static int lp_args(int type, int R, int V, int top_k) {
    SB_ARG(type_ok(type), "logprobs: unknown element type");
    SB_ARG(R >= 0 && V >= 1 && V <= (1 << 30), "logprobs: bad sizes");
    SB_ARG(top_k >= 0 && top_k <= 64 && top_k <= V, "logprobs: top_k must be 0..64 and at most V");
    return 0;
}
static size_t lp_ws_bytes(int R, int S, int k) { return S > 1 ? (size_t)R * S * (16 + 8 * (size_t)k) : 0; }

int sb_logprobs_ws(int type, int R, int V, int top_k, size_t *bytes) {
    SB_ARG(bytes, "null pointer");
    int rc = lp_args(type, R, V, top_k);
    if (rc) return rc;
    *bytes = 0;
    if (R == 0) return 0;
    sb_ctx *c = sb_ctx_get();
    if (!c) return SB_ERR_STATE;
    /* fewer rows are cut into more parts, so the most is needed by some number below R */
    for (int r = R < 4 * c->sms ? R : 4 * c->sms; r > 0; r--) {
        const size_t need = lp_ws_bytes(r, lp_parts(c, r, V, type, 8), top_k);
        if (need > *bytes) *bytes = need;
    }
    return 0;
}

int sb_logprobs(const void *logits, int64_t row_stride, int type, int R, int V, float temperature, const int *tokens,
                float *logp, float *entropy, float *lse, int *rank, int top_k, int *top_ids, float *top_logp, void *ws,
                size_t ws_bytes, void *stream) {
    int rc = lp_args(type, R, V, top_k);
    if (rc) return rc;
    SB_ARG(isfinite(temperature) && temperature >= 1e-8f, "logprobs: temperature must be at least 1e-8");
    SB_ARG(tokens || (!logp && !rank), "logprobs: logp and rank need tokens");
    SB_ARG(top_k == 0 || top_ids || top_logp, "logprobs: top_k without an output");
    if (R == 0) return 0;
    SB_ARG(logits && ALIGNED(logits, type_size(type)) && (row_stride >= V || R == 1), "logprobs: bad logits or row stride");
    sb_ctx *c = sb_ctx_get();
    if (!c) return SB_ERR_STATE;
    struct lp_params p;
    memset(&p, 0, sizeof p);
    p.S = lp_parts(c, R, V, type, 8);
    const size_t need = lp_ws_bytes(R, p.S, top_k);
    SB_ARG(ws_bytes >= need && (ws || need == 0) && ALIGNED(ws, 16), "logprobs: workspace too small (sb_logprobs_ws) or misaligned");
    p.x = DP(logits);
    p.stride = row_stride;
    p.R = R;
    p.V = V;
    p.k = top_k;
    p.c = 1.4426950408889634f / temperature;
    p.inv_temp = 1.0f / temperature;
    p.tok = DP(tokens);
    p.logp = DP(logp);
    p.entropy = DP(entropy);
    p.lse = DP(lse);
    p.rank = DP(rank);
    p.top_ids = DP(top_ids);
    p.top_logp = DP(top_logp);
    p.part = DP(ws);
    p.keys = p.part + (size_t)R * p.S * 16;
    SB_ARG((int64_t)R * p.S < 0x7fffffffL, "logprobs: too many rows");
    void *args[] = {&p};
    rc = sb_launch(c, top_k ? BY_TYPE(F_LOGPROBS_TOP_F32, type) : BY_TYPE(F_LOGPROBS_F32, type), (unsigned)(R * p.S), 1, SB_LOGPROBS_THREADS, 0,
                   (CUstream)stream, args, 0);
    if (rc || p.S == 1) return rc;
    void *jargs[] = {&p, &type};
    return sb_launch(c, F_LOGPROBS_JOIN, (unsigned)R, 1, SB_LOGPROBS_THREADS, 0, (CUstream)stream, jargs, 1);
}

int sb_logprobs_grad(const void *logits, int64_t row_stride, int type, int R, int V, float temperature, const int *tokens,
                     const float *lse, const float *entropy, const float *g_logp, const float *g_entropy, void *grad,
                     int64_t grad_stride, void *stream) {
    int rc = lp_args(type, R, V, 0);
    if (rc) return rc;
    SB_ARG(isfinite(temperature) && temperature >= 1e-8f, "logprobs_grad: temperature must be at least 1e-8");
    SB_ARG(tokens || !g_logp, "logprobs_grad: g_logp needs tokens");
    if (R == 0) return 0;
    SB_ARG(logits && grad && lse && (entropy || !g_entropy), "logprobs_grad: null pointer");
    SB_ARG(ALIGNED(logits, type_size(type)) && ALIGNED(grad, type_size(type)), "logprobs_grad: misaligned rows");
    SB_ARG(R == 1 || (row_stride >= V && grad_stride >= V), "logprobs_grad: bad row stride");
    SB_ARG(logits != grad || R == 1 || row_stride == grad_stride, "logprobs_grad: in place needs one row stride");
    sb_ctx *c = sb_ctx_get();
    if (!c) return SB_ERR_STATE;
    struct lp_grad_params p;
    memset(&p, 0, sizeof p);
    p.x = DP(logits);
    p.dx = DP(grad);
    p.stride = row_stride;
    p.dstride = grad_stride;
    p.R = R;
    p.V = V;
    /* the gradient has nothing to join: 16 CTAs per SM even out the last wave */
    long S = CEIL_DIV(16L * c->sms, (long)R), most = CEIL_DIV((long)V * type_size(type), 16384);
    p.S = (int)(S < most ? S : most);
    p.c = 1.4426950408889634f / temperature;
    p.inv_temp = 1.0f / temperature;
    p.tok = DP(tokens);
    p.lse = DP(lse);
    p.entropy = DP(entropy);
    p.g_logp = DP(g_logp);
    p.g_entropy = DP(g_entropy);
    SB_ARG((int64_t)R * p.S < 0x7fffffffL, "logprobs_grad: too many rows");
    void *args[] = {&p};
    return sb_launch(c, BY_TYPE(F_LOGPROBS_GRAD_F32, type), (unsigned)(R * p.S), 1, SB_LOGPROBS_THREADS, 0, (CUstream)stream, args, 0);
}
