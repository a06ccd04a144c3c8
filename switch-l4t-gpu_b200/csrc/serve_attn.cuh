// serve_attn.cuh -- attention of a batch over a shared prefix and each
// request's own pages (attn_prefix).
//
// Row r of request b sees every position of the prefix and the first
// len - n + i + 1 of the request's own (row i of its n).  With s_j = scale
// q.k_j the result is sum_j e^(s_j - m) v_j / sum_j e^(s_j - m): sums over
// disjoint sets of keys join by their maxima, so the work is cut into items
// (row tile, key head, key range) that leave (m, l, o) and attn_join adds
// them.  The point of the cut: the prefix is read once for ALL rows of a key
// head (T x G rows stacked into tiles), not once a request; a request's own
// keys meet only its own rows.
//
// One item runs one of these bodies; each streams K and V tiles through a
// ring in shared memory, positions going through the block table, looked up a
// tile ahead.  Whole pages come by TMA boxes in the first and the last two, a
// position without a page, or past the range, is filled with zeros and masked,
// so nothing of it is read:
//   attn_mmaw_body f16 / bf16, mma.sync m16n8k16, up to 8 or 16 rows (the head
//                  group of a decode step) against long own pages: memory-bound
//   attn_mma_body  64-row tiles, a warp 16 rows (own pages of requests with
//                  more rows)
//   attn_f32_body  FP32 on the CUDA cores: 1..16-row tiles, a lane a key
//   attn_tc_body   the prefix for more than 16 rows (serve_attn_tc.cuh)
// Scores, maxima, sums and outputs are FP32; the softmax weights are rounded
// to the value type for the second tensor-core product (half a step, like
// the values they multiply).
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>

#include "sb_common.cuh"

#define SB_AP_THREADS 128
// stages of the K / V ring: two of 32 KB for 128 values leave room for three CTAs on an SM
#define SB_AP_ST(HDP) ((HDP) == 128 ? 2 : 3)
#define SB_AP_RING 4  // offsets of the tiles in flight

__device__ int tc_err;        // nonzero after a wait timed out
__device__ unsigned tc_call;  // the last call in which one did: its other waits need not run out too

struct AttnPages {  // strides in elements
    const void *k, *v;
    long long page_stride, pos_stride, head_stride;
    int n_pages, page, shift;  // shift: log2 of the page, -1 where it is no power of two
};
// parameter block, mirrored by the host (host/sb_serve.c)
struct AttnParams {
    const void *q;
    void *out;
    float *lse;
    const int *cu_q, *ptable, *table, *kv_len;
    float *ws_o;
    float2 *ws_ml;
    int *ws_n;
    long long q_row, q_head, o_row, o_head;
    AttnPages pre, suf;
    int T, B, NH, NKV, G, HD, P, max_kv, table_stride;
    int chunk1, S1, tiles1, chunk2, S2, tiles2;  // key ranges and row tiles of the items
    int items1;                                  // prefix items in this launch; own items follow them
    int deep;                                    // 16-bit types, heads of 128: rings of two tiles instead of one
    float scale_log2;
    unsigned call;   // this call's number, not 0
    int test_skip;   // test hook: 0, or 1 + the tile of every item before which the loaders of keys stop
};

struct AttnItem {
    AttnPages pg;
    const int *table;
    int k0, k1, kvh, slot;
    int f0, F;       // first row of the tile, rows (query row x head of the group) there are
    int row0;        // query row of f = 0
    int vis0;        // positions that f sees: clamp(vis0 + f / G, 0, vis1)  (prefix: vis0 = vis1 = P, step 0)
    int vis1, step;
    bool one;        // F <= G: every f is of query row 0
};

SB_DEV int ap_rows(const AttnParams &P) { return P.cu_q ? min(max(P.cu_q[P.B], 0), P.T) : P.T; }
SB_DEV int ap_row(const AttnItem &it, int f, int G) { return it.one ? 0 : f / G; }
SB_DEV int ap_vis(const AttnItem &it, int f, int G) { return min(max(it.vis0 + it.step * ap_row(it, f, G), 0), it.vis1); }
SB_DEV int ap_page(const AttnPages &pg, int p) { return pg.shift >= 0 ? p >> pg.shift : p / pg.page; }

// Item `idx` of the prefix (row tiles fastest: neighbours read the same keys)
SB_DEV bool ap_prefix_item(const AttnParams &P, int idx, int MT, AttnItem &it) {
    const int rest = P.tiles1 > 1 ? idx / P.tiles1 : idx, tile = idx - rest * P.tiles1;
    it.kvh = rest % P.NKV;
    it.slot = rest / P.NKV;
    it.pg = P.pre;
    it.table = P.ptable;
    it.k0 = it.slot * P.chunk1;
    it.k1 = min(it.k0 + P.chunk1, P.P);
    it.F = ap_rows(P) * P.G;
    it.f0 = tile * MT;
    it.row0 = 0;
    it.vis0 = it.vis1 = P.P;
    it.step = 0;
    it.one = it.F <= P.G;
    return it.f0 < it.F;
}
// Request of item `idx`, its key head and key range; row tiles are looped by the caller
SB_DEV bool ap_own_item(const AttnParams &P, int idx, int MT, AttnItem &it, int &tile) {
    int rest = P.S2 > 1 ? idx / P.S2 : idx;
    const int s = idx - rest * P.S2;
    const int pair = P.tiles2 > 1 ? rest / P.tiles2 : rest;
    tile = rest - pair * P.tiles2;
    const int b = P.NKV > 1 ? pair / P.NKV : pair;
    it.kvh = pair - b * P.NKV;
    int q0 = b, q1 = b + 1, n = 1;  // rows that are there, and all of the request's: their limits go by these
    if (P.cu_q) {
        q0 = min(max(P.cu_q[b], 0), P.T);
        q1 = max(P.cu_q[b + 1], q0);
        n = q1 - q0;
        q1 = min(q1, P.T);
    }
    const int len = min(max(P.kv_len[b], 0), P.max_kv);
    it.slot = P.S1 + s;
    it.pg = P.suf;
    it.table = P.table + (long long)b * P.table_stride;
    it.k0 = s * P.chunk2;
    it.k1 = min(it.k0 + P.chunk2, len);
    it.F = (q1 - q0) * P.G;
    it.row0 = q0;
    it.vis0 = len - n + 1;
    it.vis1 = len;
    it.step = 1;
    it.one = it.F <= P.G;
    const int used = P.S2 > 1 ? max(1, (len + P.chunk2 - 1) / P.chunk2) : 1;
    if (s == 0 && it.kvh == 0 && P.ws_n)
        for (int r = q0 + tile * (int)blockDim.x + (int)threadIdx.x; r < q1; r += P.tiles2 * (int)blockDim.x) P.ws_n[r] = used;
    return s < used;
}

SB_DEV float ap_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
SB_DEV unsigned ap_smem(const void *p) { return (unsigned)__cvta_generic_to_shared(p); }
SB_DEV void ap_cp16(unsigned dst, const void *src, bool ok) {  // 16 bytes, or zeros (nothing is read)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
SB_DEV void ap_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> SB_DEV void ap_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// ---- barriers.  Every wait is bounded: after two seconds it sets tc_err
// (sb_tc_error reads and clears it) and tc_call, and the caller stops.  The
// call's results are NaN where that happened; another call's are not touched.
SB_DEV void ap_bar_init(uint64_t *b, unsigned count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(ap_smem(b)), "r"(count) : "memory");
}
SB_DEV void ap_arrive(uint64_t *b) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(ap_smem(b)) : "memory"); }
SB_DEV void ap_expect(uint64_t *b, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(ap_smem(b)), "r"(bytes) : "memory");
}
SB_DEV bool ap_bar_try(uint64_t *b, unsigned ph) {
    unsigned done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done)
                 : "r"(ap_smem(b)), "r"(ph)
                 : "memory");
    return done;
}
SB_DEV unsigned long long ap_now() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}
// false after WAIT_NS, or once a wait of this call has given up (call 0: only after WAIT_NS)
SB_DEV bool ap_bar_wait(uint64_t *b, unsigned ph, unsigned call) {
    constexpr unsigned long long WAIT_NS = 2000000000ull;
    if (ap_bar_try(b, ph)) return true;
    unsigned long long t0 = 0;
#pragma unroll 1
    for (int spin = 0; spin < (1 << 26); spin++) {
        if (ap_bar_try(b, ph)) return true;
        if ((spin & 1023) == 1023) {
            if (call && *(volatile unsigned *)&tc_call == call) return false;
            const unsigned long long t = ap_now();
            if (t0 == 0) t0 = t;
            else if (t - t0 > WAIT_NS) break;
        }
    }
    atomicExch(&tc_err, 1);
    if (call) {
        atomicExch(&tc_call, call);
        __threadfence();
    }
    return false;
}
SB_DEV void ap_fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// box {128 bytes of values, one head, rows of a page, one page}
SB_DEV void ap_tma(unsigned dst, const CUtensorMap *tm, int d, int head, int row, int page, uint64_t *b) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(tm), "r"(d), "r"(head), "r"(row), "r"(page), "r"(ap_smem(b))
        : "memory");
}
// a warp's ring: K and V tiles that have landed (32 arrivals and the bytes), and which keys of a tile are there
struct ApBars {
    uint64_t full[2][2];
    unsigned valid[2];
};

// element offset of position p in the pages (without the head) with the lowest
// bit set (offsets are multiples of 16 bytes), 0 where it has none
SB_DEV long long ap_offset(const AttnItem &it, int p) {
    if (p >= it.k1) return 0;
    const int j = ap_page(it.pg, p);
    const int pg = it.table ? it.table[j] : j;
    if (pg < 0 || pg >= it.pg.n_pages) return 0;
    return (pg * it.pg.page_stride + (p - j * it.pg.page) * it.pg.pos_stride) | 1;
}
// A thread's share of the copies of a K and a V tile of KT positions, rows of
// HDP values of E bytes: its 16-byte chunk of every STEP-th row, swizzled by
// the row's low three bits.  Places that are not
// there are filled with zeros, nothing of them is read.
template <int KT, int HDP, int E> struct ApCopy {
    static constexpr int C = HDP * E / 16, STEP = SB_AP_THREADS / C, N = KT / STEP;
    const char *k;
    long long to_v;
    unsigned dst;
    int row;
    bool in;
    SB_DEV ApCopy(const AttnItem &it, int HD) {
        static_assert(STEP % 8 == 0 || STEP == 4, "rows of a thread share their low three bits, or differ in the third");
        const int c = threadIdx.x % C;
        row = threadIdx.x / C;
        k = static_cast<const char *>(it.pg.k) + it.kvh * it.pg.head_stride * E + c * 16;
        to_v = static_cast<const char *>(it.pg.v) - static_cast<const char *>(it.pg.k);
        dst = row * (HDP * E) + ((c ^ (row & 7)) << 4);
        in = c * 16 < HD * E;
    }
    SB_DEV void copy(unsigned kd, unsigned vd, const long long *off) const {
#pragma unroll
        for (int j = 0; j < N; j++) {
            const long long o = off[row + j * STEP];
            const bool ok = (o & 1) && in;
            const char *p = k + (o & ~1ll) * E;
            const unsigned at = (dst ^ ((j * STEP & 4) << 4)) + j * STEP * HDP * E;  // chunk ^ 4 where the row's third bit is set
            ap_cp16(kd + at, p, ok);
            ap_cp16(vd + at, p + to_v, ok);
        }
    }
};

// The keys of one warp: KW positions of every KT, K and V tiles in a ring of st
// (1 or 2) each.  The block never meets: a tile of K is asked for as soon as the warp
// has its scores, one of V as soon as it has its outputs, so nearly 2 st tiles
// are always in flight.  A tile is rows of 128 bytes in column blocks, 16-byte
// chunks xor-ed by the row's low three bits (ldmatrix, or eight lanes on eight
// keys, touch all banks).  Whole pages come by TMA boxes, one lane a box:
// copies by the lanes (tiles that end inside a page or miss one, other page
// sizes, calls too small to encode a map for) cost a third of all
// instructions of a decode tile.  Where a box may follow into the place of a
// tile that the lanes copied, that tile has a gap: its reader orders the two by
// a proxy fence before it gives the place up.
template <int KW, int HDP, int E> struct ApRing {
    static constexpr int SUB = HDP * E / 128, BLOCK = KW * 128, TILE = SUB * BLOCK, KT = KW * (SB_AP_THREADS / 32);
    static constexpr int C = HDP * E / 16, STEP = 32 / C, N = KW / STEP;
    const AttnParams &P;
    const AttnItem &it;
    const CUtensorMap *tm[2];
    ApBars *bars;
    unsigned sm;
    int st, first, box, HD, seq;  // seq: tiles that went through the ring before this item, -1 after giving up
    int pg, in_pg, row, sub;  // this lane's box of the tile looked up last
    bool mine;
    SB_DEV ApRing(const AttnParams &prm, const AttnItem &item, int stages, unsigned char *ring, ApBars *b, int seq0, const CUtensorMap *k,
                  const CUtensorMap *v, int bx)
        : P(prm), it(item), bars(b + (threadIdx.x >> 5)), st(stages), box(min(bx, KW)), HD(prm.HD), seq(seq0) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, pieces = box ? KW / box : 1;
        tm[0] = k;
        tm[1] = v;
        sm = ap_smem(ring) + warp * (2 * st * TILE);
        first = it.k0 + warp * KW;
        sub = lane / pieces;
        row = lane % pieces * box;
        mine = box && sub < SUB;
    }
    SB_DEV int tiles(int k1) const { return k1 > first && seq >= 0 ? (k1 - first + KT - 1) / KT : 0; }
    SB_DEV int slot(int t) const { return (seq + t) & (st - 1); }
    SB_DEV unsigned phase(int t) const { return (unsigned)((seq + t) >> (st - 1)) & 1u; }  // of st = 1 or 2
    SB_DEV unsigned tile(int which, int t) const { return sm + (which * st + slot(t)) * TILE; }
    SB_DEV void look(int t) {  // a tile ahead of its use
        const int p = first + t * KT + row;
        pg = -1;
        if (mine && p - row + KW <= it.k1) {
            const int j = ap_page(it.pg, p);
            pg = it.table ? it.table[j] : j;
            in_pg = p - j * it.pg.page;
        }
    }
    SB_DEV void copy(int which, int t) {  // tile t, looked up
        if (which == 0 && t + 1 == P.test_skip) return;
        const int lane = threadIdx.x & 31, n = slot(t);
        const unsigned dst = tile(which, t);
        uint64_t *bar = &bars->full[which][n];
        if (__all_sync(SB_FULL, box && (!mine || (pg >= 0 && pg < it.pg.n_pages)))) {
            if (lane == 0) {
                if (which == 0) bars->valid[n] = ~0u;
                ap_expect(bar, TILE);
            } else {
                ap_arrive(bar);
            }
            __syncwarp();
            if (mine) ap_tma(dst + sub * BLOCK + row * 128, tm[which], sub * (128 / E), it.kvh, in_pg, pg, bar);
            return;
        }
        const long long off = ap_offset(it, first + t * KT + lane % KW);
        const unsigned valid = __ballot_sync(SB_FULL, off & 1);
        if (which == 0 && lane == 0) bars->valid[n] = valid;
        const int c = lane % C, r0 = lane / C;
        const char *base = static_cast<const char *>(which ? it.pg.v : it.pg.k) + it.kvh * it.pg.head_stride * E + c * 16;
        ap_fence_async();  // the ring's place may have been written by TMA, or will be
#pragma unroll
        for (int j = 0; j < N; j++) {
            const int r = r0 + j * STEP;
            const long long o = __shfl_sync(SB_FULL, off, r);
            ap_cp16(dst + (c >> 3) * BLOCK + r * 128 + (((c & 7) ^ (r & 7)) << 4), base + (o & ~1ll) * E, (o & 1) && c * 16 < HD * E);
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(ap_smem(bar)) : "memory");
    }
    SB_DEV bool wait(int which, int t) const {
        return __all_sync(SB_FULL, ap_bar_wait(&bars->full[which][slot(t)], phase(t), P.call));
    }
    SB_DEV void drain(int t, int nt, int at_v) {  // given up at tile t, its K or V: what was asked for still has to land
        for (int u = t + at_v; u < min(t + st + at_v, nt); u++) ap_bar_wait(&bars->full[0][slot(u)], phase(u), 0);
        for (int u = t; u < min(t + st, nt); u++) ap_bar_wait(&bars->full[1][slot(u)], phase(u), 0);
        __syncwarp();
    }
    SB_DEV unsigned valid(int t) const { return bars->valid[slot(t)]; }
};

// what a finished row leaves: the output itself where the item is the only one, else its part
SB_DEV void ap_row_stats(const AttnParams &P, const AttnItem &it, int f, float m, float l) {
    const int qr = ap_row(it, f, P.G), row = it.row0 + qr, head = it.kvh * P.G + f - qr * P.G;
    if (P.S1 + P.S2 == 1) {
        if (P.lse) P.lse[(long long)row * P.NH + head] = l > 0.f ? (m + log2f(l)) * 0.6931471805599453f : (l == 0.f ? -INFINITY : l);
    } else {
        P.ws_ml[((long long)it.slot * P.T + row) * P.NH + head] = make_float2(m, l);
    }
}
template <typename T> SB_DEV void ap_store2(T *p, float a, float b);
template <> SB_DEV void ap_store2<float>(float *p, float a, float b) { *reinterpret_cast<float2 *>(p) = make_float2(a, b); }
template <> SB_DEV void ap_store2<__half>(__half *p, float a, float b) { *reinterpret_cast<__half2 *>(p) = __floats2half2_rn(a, b); }
template <> SB_DEV void ap_store2<__nv_bfloat16>(__nv_bfloat16 *p, float a, float b) {
    *reinterpret_cast<__nv_bfloat162 *>(p) = __floats2bfloat162_rn(a, b);
}
// two neighbouring values (d even) of row f; a row that sees nothing gives zeros
template <typename T>
SB_DEV void ap_row_out(const AttnParams &P, const AttnItem &it, int f, int d, float a, float b, float l) {
    if (d >= P.HD) return;
    const int qr = ap_row(it, f, P.G), row = it.row0 + qr, head = it.kvh * P.G + f - qr * P.G;
    if (P.S1 + P.S2 == 1) {
        const float w = l == 0.f ? 0.f : 1.f / l;
        ap_store2<T>(static_cast<T *>(P.out) + row * P.o_row + head * P.o_head + d, a * w, b * w);
    } else if (l != 0.f) {  // the join skips parts without weight
        ap_store2<float>(P.ws_o + (((long long)it.slot * P.T + row) * P.NH + head) * P.HD + d, a, b);
    }
}

template <typename T> SB_DEV const T *ap_query(const AttnParams &P, const AttnItem &it, int f) {
    const int qr = ap_row(it, f, P.G);
    return static_cast<const T *>(P.q) + (long long)(it.row0 + qr) * P.q_row + (it.kvh * P.G + f - qr * P.G) * P.q_head;
}
template <typename T> SB_DEV void ap_store4(T *p, float a, float b, float c, float d) {
    ap_store2<T>(p, a, b);
    ap_store2<T>(p + 2, c, d);
}
template <> SB_DEV void ap_store4<float>(float *p, float a, float b, float c, float d) { *reinterpret_cast<float4 *>(p) = make_float4(a, b, c, d); }
// The warps of a block join: o [warps][R][HDP], (m, l) [warps][R]; four values a thread.
template <typename T, int HDP, int R>
SB_DEV void ap_block_join(const AttnParams &P, const AttnItem &it, const float *o, const float (*ms)[R], const float (*ls)[R]) {
    constexpr int NW = SB_AP_THREADS / 32;
    for (int i = threadIdx.x; i < R * HDP / 4; i += SB_AP_THREADS) {
        const int r = i / (HDP / 4), d = (i % (HDP / 4)) * 4, f = it.f0 + r;
        if (f >= it.F) break;
        if (d >= P.HD) continue;
        float M = ms[0][r], L = 0.f;
#pragma unroll
        for (int w = 1; w < NW; w++) M = fmaxf(M, ms[w][r]);
        const float base = M == -INFINITY ? 0.f : M;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float e = ap_exp2(ms[w][r] - base);
            const float4 x = *reinterpret_cast<const float4 *>(o + (w * R + r) * HDP + d);
            L = fmaf(e, ls[w][r], L);
            a.x = fmaf(e, x.x, a.x);
            a.y = fmaf(e, x.y, a.y);
            a.z = fmaf(e, x.z, a.z);
            a.w = fmaf(e, x.w, a.w);
        }
        const int qr = ap_row(it, f, P.G), row = it.row0 + qr, head = it.kvh * P.G + f - qr * P.G;
        if (d == 0) ap_row_stats(P, it, f, M, L);
        if (P.S1 + P.S2 == 1) {
            const float w = L == 0.f ? 0.f : 1.f / L;
            ap_store4<T>(static_cast<T *>(P.out) + row * P.o_row + head * P.o_head + d, a.x * w, a.y * w, a.z * w, a.w * w);
        } else if (L != 0.f) {
            ap_store4<float>(P.ws_o + (((long long)it.slot * P.T + row) * P.NH + head) * P.HD + d, a.x, a.y, a.z, a.w);
        }
    }
}

// ---------------------------------------------------------------- f16 / bf16
template <typename T> SB_DEV void ap_mma(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1);
template <> SB_DEV void ap_mma<__half>(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> SB_DEV void ap_mma<__nv_bfloat16>(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T> SB_DEV unsigned ap_pack(float a, float b);
template <> SB_DEV unsigned ap_pack<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const unsigned *>(&h);
}
template <> SB_DEV unsigned ap_pack<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const unsigned *>(&h);
}
SB_DEV void ap_ldsm(unsigned (&r)[4], unsigned addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
SB_DEV void ap_ldsm_t(unsigned (&r)[4], unsigned addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}

// 64-row tiles, a warp 16 rows against all keys.  HDP: head size padded to 64
// or 128.  Shared memory: SB_AP_ST x 2 x 64 x HDP x 2 bytes, rows of 128 / 256
// bytes with their 16-byte chunks xor-ed by the row's low three bits (ldmatrix
// reads eight rows of one chunk without a conflict).
template <typename T, int HDP>
SB_DEV void attn_mma_body(const AttnParams &P, const AttnItem &it, unsigned char *sm, long long (*off_s)[64]) {
    constexpr int KT = 64, NT = KT / 8, KS = HDP / 16, ST = SB_AP_ST(HDP);
    constexpr int TILE = KT * HDP * 2, STAGE = 2 * TILE, RING = SB_AP_RING;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q4 = lane & 3;
    const int fw = it.f0 + warp * 16;  // this warp's first row
    const ApCopy<KT, HDP, 2> copier(it, P.HD);

    // query fragments from global memory: rows fw + g and fw + g + 8
    unsigned qa[KS][4];
    int vis[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int f = fw + g + 8 * h;
        vis[h] = f < it.F ? ap_vis(it, f, P.G) : 0;
        const T *qp = ap_query<T>(P, it, f);
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int d = k * 16 + e * 8 + q4 * 2;
                qa[k][h + 2 * e] = f < it.F && d < P.HD ? *reinterpret_cast<const unsigned *>(qp + d) : 0u;
            }
    }
    // keys that some row of the tile sees end here
    const int flast = min(it.f0 + 64, it.F) - 1;
    const int k1 = min(it.k1, ap_vis(it, flast, P.G));
    const int nt = k1 > it.k0 ? (k1 - it.k0 + KT - 1) / KT : 0;

    auto load = [&](int t) {
        if (t < nt) {
            const unsigned kd = ap_smem(sm) + (t % ST) * STAGE;
            copier.copy(kd, kd + TILE, off_s[t % RING]);
        }
        ap_commit();
    };
    float o[HDP / 8][4];
#pragma unroll
    for (int i = 0; i < HDP / 8; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    __syncthreads();  // the ring and the offsets of an earlier item are no longer read
    for (int t = 0; t < ST; t++)
        if (tid < KT) off_s[t][tid] = ap_offset(it, it.k0 + t * KT + tid);
    __syncthreads();
    for (int t = 0; t < ST - 1; t++) load(t);
    for (int t = 0; t < nt; t++) {
        ap_wait<ST - 2>();
        __syncthreads();  // tile t is there for all; tile t - 1 and its offsets are read
        load(t + ST - 1);
        long long next = 0;
        if (tid < KT) next = ap_offset(it, it.k0 + (t + ST) * KT + tid);
        const unsigned kt = ap_smem(sm) + (t % ST) * STAGE, vt = kt + TILE;
        const long long *off = off_s[t % RING];
        const int key0 = it.k0 + t * KT;
        float s[NT][4];
#pragma unroll
        for (int i = 0; i < NT; i++) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
        const int mid = lane >> 3, r8 = lane & 7;
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
            for (int n = 0; n < NT / 2; n++) {
                const int r = n * 16 + r8 + (mid >> 1) * 8, c = k * 2 + (mid & 1);
                unsigned b[4];
                ap_ldsm(b, kt + r * (HDP * 2) + ((c ^ (r & 7)) << 4));
                ap_mma<T>(s[2 * n], qa[k], b[0], b[1]);
                ap_mma<T>(s[2 * n + 1], qa[k], b[2], b[3]);
            }
        // scores in log2 units; masked where the row does not see the key or the key has no page
        float mx[2] = {m[0], m[1]};
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int j = n * 8 + q4 * 2 + (e & 1);
                const bool seen = key0 + j < vis[e >> 1] && (off[j] & 1);
                s[n][e] = seen ? s[n][e] * P.scale_log2 : -INFINITY;
                mx[e >> 1] = fmaxf(mx[e >> 1], s[n][e]);
            }
        float base[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            mx[h] = fmaxf(mx[h], __shfl_xor_sync(SB_FULL, mx[h], 1));
            mx[h] = fmaxf(mx[h], __shfl_xor_sync(SB_FULL, mx[h], 2));
            base[h] = mx[h] == -INFINITY ? 0.f : mx[h];
            const float a = ap_exp2(m[h] - base[h]);
            m[h] = mx[h];
            l[h] *= a;
#pragma unroll
            for (int i = 0; i < HDP / 8; i++) {
                o[i][2 * h] *= a;
                o[i][2 * h + 1] *= a;
            }
        }
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                s[n][e] = ap_exp2(s[n][e] - base[e >> 1]);
                l[e >> 1] += s[n][e];
            }
#pragma unroll
        for (int n = 0; n < NT / 2; n++) {
            const unsigned a[4] = {ap_pack<T>(s[2 * n][0], s[2 * n][1]), ap_pack<T>(s[2 * n][2], s[2 * n][3]),
                                   ap_pack<T>(s[2 * n + 1][0], s[2 * n + 1][1]), ap_pack<T>(s[2 * n + 1][2], s[2 * n + 1][3])};
#pragma unroll
            for (int i = 0; i < HDP / 16; i++) {
                const int r = n * 16 + r8 + (mid & 1) * 8, c = i * 2 + (mid >> 1);
                unsigned b[4];
                ap_ldsm_t(b, vt + r * (HDP * 2) + ((c ^ (r & 7)) << 4));
                ap_mma<T>(o[2 * i], a, b[0], b[1]);
                ap_mma<T>(o[2 * i + 1], a, b[2], b[3]);
            }
        }
        if (tid < KT) off_s[(t + ST) % RING][tid] = next;
    }
    ap_wait<0>();
#pragma unroll
    for (int h = 0; h < 2; h++) {
        l[h] += __shfl_xor_sync(SB_FULL, l[h], 1);
        l[h] += __shfl_xor_sync(SB_FULL, l[h], 2);
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int f = fw + g + 8 * h;
        if (f >= it.F) continue;
        if (q4 == 0) ap_row_stats(P, it, f, m[h], l[h]);
#pragma unroll
        for (int i = 0; i < HDP / 8; i++) ap_row_out<T>(P, it, f, i * 8 + q4 * 2, o[i][2 * h], o[i][2 * h + 1], l[h]);
    }
}

// Up to 8 NB rows, a warp a quarter of the keys of every 64, the products with
// the keys along m: S^T = K Q^T (rows along n = 8) and O^T = V^T P^T.  Nothing
// is spent on rows that are not there (a group of 4 or 7 heads filled a
// quarter or half of a 16-row tile), and the outputs take half the registers.
// P^T turns from accumulator into operand by movmatrix.  Like the tcgen05
// kernel it rescales only when a row's maximum has grown by more than 2^8; a
// tile without that costs one vote.
SB_DEV unsigned ap_movmatrix(unsigned a) {
    unsigned d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
template <typename T, int HDP, int NB>
SB_DEV void attn_mmaw_body(const AttnParams &P, const AttnItem &it, unsigned char *sm, ApBars *bars, int &seq, const CUtensorMap *tm_k,
                           const CUtensorMap *tm_v, int box) {
    constexpr int NW = SB_AP_THREADS / 32, KS = HDP / 16, KT = 16 * NW;
    const int st = HDP == 128 && !P.deep ? 1 : 2;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q4 = lane & 3;
    ApRing<16, HDP, 2> ring(P, it, st, sm, bars, seq, tm_k, tm_v, box);
    unsigned qb[NB][KS][2];  // rows f0 + 8 b + g
    int vis[NB][2];          // of rows f0 + 8 b + 2 q4, + 1
#pragma unroll
    for (int b = 0; b < NB; b++) {
        const int f = it.f0 + b * 8 + g;
        const T *qp = ap_query<T>(P, it, f);
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int d = k * 16 + e * 8 + q4 * 2;
                qb[b][k][e] = f < it.F && d < P.HD ? *reinterpret_cast<const unsigned *>(qp + d) : 0u;
            }
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int fh = it.f0 + b * 8 + 2 * q4 + h;
            vis[b][h] = fh < it.F ? ap_vis(it, fh, P.G) : 0;
        }
    }
    const int flast = min(it.f0 + 8 * NB, it.F) - 1, first = ring.first;
    const int nt = ring.tiles(min(it.k1, ap_vis(it, flast, P.G)));  // this warp's tiles: 16 keys of every KT
    float o[NB][KS][4], m[NB][2], l[NB][2];
#pragma unroll
    for (int b = 0; b < NB; b++) {
#pragma unroll
        for (int i = 0; i < KS; i++) o[b][i][0] = o[b][i][1] = o[b][i][2] = o[b][i][3] = 0.f;
        m[b][0] = m[b][1] = -INFINITY;
        l[b][0] = l[b][1] = 0.f;
    }
    ap_fence_async();
    __syncthreads();  // an earlier item's join has been read
    for (int t = 0; t < st; t++) {
        ring.look(t);
        if (t < nt) {
            ring.copy(0, t);
            ring.copy(1, t);
        }
    }
    ring.look(st);
    bool ok = seq >= 0;
    int t = 0, at_v = 0;
    for (; t < nt; t++) {
        const unsigned kt = ring.tile(0, t), vt = ring.tile(1, t);
        const int key = first + t * KT + g;
        if (!(ok = ring.wait(0, t))) break;
        const unsigned valid = ring.valid(t);
        const bool there0 = valid >> g & 1, there1 = valid >> (g + 8) & 1, gaps = valid != ~0u;
        if (gaps) ap_fence_async();
        float s[NB][4];
#pragma unroll
        for (int b = 0; b < NB; b++) s[b][0] = s[b][1] = s[b][2] = s[b][3] = 0.f;
#pragma unroll
        for (int k = 0; k < KS; k++) {
            const int r = lane & 15, c = 2 * k + (lane >> 4);
            unsigned a[4];
            ap_ldsm(a, kt + (c >> 3) * 2048 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
#pragma unroll
            for (int b = 0; b < NB; b++) ap_mma<T>(s[b], a, qb[b][k][0], qb[b][k][1]);
        }
        __syncwarp();
        if (t + st < nt) ring.copy(0, t + st);
        bool grown = false;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int e = 0; e < 4; e++) {  // key g + 8 (e >> 1), row 2 q4 + (e & 1)
                const bool seen = ((e >> 1) ? there1 : there0) && key + 8 * (e >> 1) < vis[b][e & 1];
                s[b][e] = seen ? s[b][e] * P.scale_log2 : -INFINITY;
                grown |= s[b][e] > m[b][e & 1] + 8.f;
            }
        if (__any_sync(SB_FULL, grown)) {
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    float mx = fmaxf(s[b][h], s[b][2 + h]);
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(SB_FULL, mx, x));
                    const float to = fmaxf(m[b][h], mx), a = to == m[b][h] ? 1.f : ap_exp2(m[b][h] - to);
                    m[b][h] = to;
                    l[b][h] *= a;
#pragma unroll
                    for (int i = 0; i < KS; i++) {
                        o[b][i][h] *= a;
                        o[b][i][2 + h] *= a;
                    }
                }
        }
        unsigned p[NB][2];
#pragma unroll
        for (int b = 0; b < NB; b++) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                s[b][e] = ap_exp2(s[b][e] - (m[b][e & 1] == -INFINITY ? 0.f : m[b][e & 1]));
                l[b][e & 1] += s[b][e];
            }
            p[b][0] = ap_movmatrix(ap_pack<T>(s[b][0], s[b][1]));
            p[b][1] = ap_movmatrix(ap_pack<T>(s[b][2], s[b][3]));
        }
        if (!(ok = ring.wait(1, t))) {
            at_v = 1;
            break;
        }
        if (gaps) ap_fence_async();
#pragma unroll
        for (int i = 0; i < KS; i++) {
            const int mid = lane >> 3, r = (mid >> 1) * 8 + (lane & 7), c = 2 * i + (mid & 1);
            unsigned a[4];
            ap_ldsm_t(a, vt + (c >> 3) * 2048 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
#pragma unroll
            for (int b = 0; b < NB; b++) ap_mma<T>(o[b][i], a, p[b][0], p[b][1]);
        }
        __syncwarp();
        if (t + st < nt) {
            ring.copy(1, t + st);
            ring.look(t + st + 1);
        }
    }
    if (ok) seq += nt;
    if (!ok) {  // given up (tc_err), here or in an item before: nothing that passes for a result
        ring.drain(t, nt, at_v);
        seq = -1;
#pragma unroll
        for (int b = 0; b < NB; b++) l[b][0] = l[b][1] = __int_as_float(0x7fc00000);
    }
    float *ow = reinterpret_cast<float *>(sm);  // [NW][8 NB rows][HDP]
    __shared__ float ms[NW][8 * NB], ls[NW][8 * NB];
    __syncthreads();
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int r = b * 8 + 2 * q4 + h;
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) l[b][h] += __shfl_xor_sync(SB_FULL, l[b][h], x);
            if (g == 0) {
                ms[warp][r] = m[b][h];
                ls[warp][r] = l[b][h];
            }
#pragma unroll
            for (int i = 0; i < KS; i++) {
                ow[(warp * 8 * NB + r) * HDP + i * 16 + g] = o[b][i][h];
                ow[(warp * 8 * NB + r) * HDP + i * 16 + g + 8] = o[b][i][2 + h];
            }
        }
    __syncthreads();
    ap_block_join<T, HDP, 8 * NB>(P, it, ow, ms, ls);
}

// ---------------------------------------------------------------- FP32
// MT rows, a warp a quarter of the keys of every KT from the scores to the
// outputs (the block meets only for the join).  Scores: a lane takes a key and
// 32 of its dimensions; K chunks are xor-swizzled so that eight lanes reading
// eight keys touch all banks, query values are broadcast (the DQ parts of a
// row 36 floats apart, on banks of their own).  Outputs: a lane owns HDP / 32
// dimensions of all rows, the weights come as pairs from shared memory for
// two-wide FMAs.  Rows rescale when their maximum has grown by more than 2^8,
// as in the other kernels.
// Bound: HBM up to eight rows, the shared-memory and FMA pipes beyond.  HBM
// gives an SM 23 bytes a cycle (6.55 TB/s, 148 SMs, 1.9 GHz); at MT rows of 64
// the FMA pipe takes MT cycles a key (128 MT products, 128 a cycle) of 512
// bytes, 64 bytes a cycle at 8 rows and 32 at 16, where the reads of queries
// and weights from shared memory take as long again.  FFMA and not the
// tensor pipe: its FP32 sums are not IEEE-rounded and drift by 1e-5 over some
// thousand keys.
template <int HDP, int MT>
SB_DEV void attn_f32_body(const AttnParams &P, const AttnItem &it, unsigned char *sm, ApBars *bars, int &seq, const CUtensorMap *tm_k,
                          const CUtensorMap *tm_v, int box) {
    constexpr int NW = SB_AP_THREADS / 32, KW = HDP == 64 ? 16 : 8, KT = KW * NW, DQ = 32 / KW, DP = HDP / 64;  // keys a warp, parts of a key, pairs of a lane
    constexpr int st = 2, BLOCK = KW * 128;
    __shared__ __align__(16) float q_s[MT][DQ][36];
    __shared__ __align__(16) float2 p_s[NW][KW][MT < 2 ? 2 : MT];
    __shared__ float m_s[NW][MT], l_s[NW][MT];
    __shared__ int vis_s[MT];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, key = lane % KW, dq = lane / KW;
    ApRing<KW, HDP, 4> ring(P, it, st, sm, bars, seq, tm_k, tm_v, box);
    __syncthreads();  // an earlier item's shared memory is no longer read
    for (int i = tid; i < MT * HDP / 4; i += SB_AP_THREADS) {
        const int r = i / (HDP / 4), d = i % (HDP / 4) * 4, f = it.f0 + r;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (f < it.F && d < P.HD) v = *reinterpret_cast<const float4 *>(ap_query<float>(P, it, f) + d);
        *reinterpret_cast<float4 *>(&q_s[r][d / 32][d % 32]) = make_float4(v.x * P.scale_log2, v.y * P.scale_log2, v.z * P.scale_log2, v.w * P.scale_log2);
    }
    if (tid < MT) vis_s[tid] = it.f0 + tid < it.F ? ap_vis(it, it.f0 + tid, P.G) : 0;
    const int flast = min(it.f0 + MT, it.F) - 1;
    const int k1 = min(it.k1, ap_vis(it, flast, P.G)), vmin = ap_vis(it, it.f0, P.G);  // rows in order see more and more
    const int first = ring.first, nt = ring.tiles(k1);  // this warp's KW keys of every KT
    ap_fence_async();
    __syncthreads();
    for (int t = 0; t < st; t++) {
        ring.look(t);
        if (t < nt) {
            ring.copy(0, t);
            ring.copy(1, t);
        }
    }
    ring.look(st);
    bool ok = seq >= 0;
    unsigned long long o[MT][DP];
    float m[MT], l[MT];
#pragma unroll
    for (int r = 0; r < MT; r++) {
        m[r] = -INFINITY;
        l[r] = 0.f;
#pragma unroll
        for (int e = 0; e < DP; e++) o[r][e] = 0ull;
    }
    int t = 0, at_v = 0;
    for (; t < nt; t++) {
        const unsigned char *kt = sm + (ring.tile(0, t) - ap_smem(sm)), *vt = sm + (ring.tile(1, t) - ap_smem(sm));
        if (!(ok = ring.wait(0, t))) break;
        const unsigned valid = ring.valid(t);
        const bool there = valid >> key & 1, gaps = valid != ~0u;
        if (gaps) ap_fence_async();
        unsigned long long acc[MT];
#pragma unroll
        for (int r = 0; r < MT; r++) acc[r] = 0ull;
#pragma unroll
        for (int c = 0; c < 8; c++) {
            const ulonglong2 k2 = *reinterpret_cast<const ulonglong2 *>(kt + dq * BLOCK + key * 128 + ((c ^ (key & 7)) << 4));
#pragma unroll
            for (int r = 0; r < MT; r++) {
                const ulonglong2 q2 = *reinterpret_cast<const ulonglong2 *>(&q_s[r][dq][c * 4]);
                acc[r] = ffma2(q2.x, k2.x, acc[r]);
                acc[r] = ffma2(q2.y, k2.y, acc[r]);
            }
        }
        __syncwarp();
        if (t + st < nt) ring.copy(0, t + st);
        float s[MT];
        bool grown = false;
        const int at = first + t * KT + key;
        const bool all = there && at < vmin;
#pragma unroll
        for (int r = 0; r < MT; r++) {
            s[r] = f2_sum(acc[r]);
#pragma unroll
            for (int x = KW; x < 32; x <<= 1) s[r] += __shfl_xor_sync(SB_FULL, s[r], x);
            if (!all && !(there && at < vis_s[r])) s[r] = -INFINITY;
            grown |= s[r] > m[r] + 8.f;
        }
        if (__any_sync(SB_FULL, grown)) {
#pragma unroll
            for (int r = 0; r < MT; r++) {
                const float to = fmaxf(m[r], warp_max(s[r])), a = to == m[r] ? 1.f : ap_exp2(m[r] - to);
                m[r] = to;
                l[r] *= a;
#pragma unroll
                for (int e = 0; e < DP; e++) o[r][e] = ffma2(o[r][e], f2_pack(a, a), 0ull);
            }
        }
#pragma unroll
        for (int r = 0; r < MT; r++) {
            s[r] = ap_exp2(s[r] - (m[r] == -INFINITY ? 0.f : m[r]));
            l[r] += s[r];
            if (r % DQ == dq) p_s[warp][key][r] = make_float2(s[r], s[r]);
        }
        __syncwarp();
        if (!(ok = ring.wait(1, t))) {
            at_v = 1;
            break;
        }
        if (gaps) ap_fence_async();
#pragma unroll
        for (int k = 0; k < KW; k++) {
            unsigned long long v[DP];
            if constexpr (DP == 1) {
                const int at = ((((lane >> 1) & 7) ^ (k & 7)) << 4) + (lane & 1) * 8;
                v[0] = *reinterpret_cast<const unsigned long long *>(vt + (lane >> 4) * BLOCK + k * 128 + at);
            } else {
                const ulonglong2 w = *reinterpret_cast<const ulonglong2 *>(vt + (lane >> 3) * BLOCK + k * 128 + (((lane & 7) ^ (k & 7)) << 4));
                v[0] = w.x;
                v[DP - 1] = w.y;
            }
            if constexpr (MT == 1) {
                const unsigned long long p = *reinterpret_cast<const unsigned long long *>(&p_s[warp][k][0]);
#pragma unroll
                for (int e = 0; e < DP; e++) o[0][e] = ffma2(p, v[e], o[0][e]);
            } else {
#pragma unroll
                for (int r = 0; r < MT; r += 2) {
                    const ulonglong2 p = *reinterpret_cast<const ulonglong2 *>(&p_s[warp][k][r]);
#pragma unroll
                    for (int e = 0; e < DP; e++) {
                        o[r][e] = ffma2(p.x, v[e], o[r][e]);
                        o[r + (MT > 1)][e] = ffma2(p.y, v[e], o[r + (MT > 1)][e]);
                    }
                }
            }
        }
        __syncwarp();  // values and weights are read
        if (t + st < nt) {
            ring.copy(1, t + st);
            ring.look(t + st + 1);
        }
    }
    if (ok) seq += nt;
    if (!ok) {  // given up (tc_err), here or in an item before: nothing that passes for a result
        ring.drain(t, nt, at_v);
        seq = -1;
#pragma unroll
        for (int r = 0; r < MT; r++) l[r] = __int_as_float(0x7fc00000);
    }
    __syncthreads();
    float *red = reinterpret_cast<float *>(sm);  // [NW][MT][HDP] floats: 32 KB at most, in the ring
#pragma unroll
    for (int r = 0; r < MT; r++) {
        const float sum = warp_sum(l[r]) * (1.f / DQ);  // every key is held by DQ lanes
        if (lane == 0) {
            m_s[warp][r] = m[r];
            l_s[warp][r] = sum;
        }
#pragma unroll
        for (int e = 0; e < DP; e++) *reinterpret_cast<unsigned long long *>(red + (warp * MT + r) * HDP + lane * (2 * DP) + 2 * e) = o[r][e];
    }
    __syncthreads();
    ap_block_join<float, HDP, MT>(P, it, red, m_s, l_s);
}

// A CTA an item: the prefix items of the launch, then own ones (either may be
// none; row tiles of a request beyond the grid's are looped).  Each launch lets
// the next start early and does not end before the one before it, so that the
// join, which waits for the last, has all of them behind it.  The CTA that is
// started last waits for that; when every CTA did, the first of the second
// launch held their SMs until the first launch was over.
#define SB_AP_KERNEL(name, CTAS, MT, SHARED, CALL)                                                                   \
    extern "C" __global__ void __launch_bounds__(SB_AP_THREADS, CTAS)                                                  \
        name(const __grid_constant__ AttnParams P, const __grid_constant__ CUtensorMap tm_k,                           \
             const __grid_constant__ CUtensorMap tm_v, int box) {                                                      \
        extern __shared__ __align__(1024) unsigned char ap_sm[];                                                       \
        SHARED;                                                                                                        \
        pdl_launch_dependents();                                                                                       \
        AttnItem it;                                                                                                   \
        const int item = (int)blockIdx.x - P.items1;                                                                   \
        it.f0 = 0;                                                                                                     \
        if (item < 0) {                                                                                                \
            if (!ap_prefix_item(P, blockIdx.x, MT, it)) it.F = 0;                                                      \
        } else {                                                                                                       \
            int tile;                                                                                                  \
            if (ap_own_item(P, item, MT, it, tile)) it.f0 = tile * MT;                                                 \
            else it.F = 0;                                                                                             \
        }                                                                                                              \
        for (const int step = item < 0 ? 1 << 30 : P.tiles2 * MT; it.f0 < it.F; it.f0 += step) CALL;                   \
        if (blockIdx.x == gridDim.x - 1) pdl_wait();                                                                   \
    }
// the four warps' barriers; a warp counts its own tiles
#define SB_AP_WARPS                                                                                                    \
    __shared__ ApBars bars[SB_AP_THREADS / 32];                                                                        \
    int seq = 0;                                                                                                       \
    if ((threadIdx.x & 31) < 4) ap_bar_init(&bars[threadIdx.x >> 5].full[0][0] + (threadIdx.x & 3), 32);               \
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");                                                 \
    __syncwarp()
#define SB_AP_MMAW(name, T, HDP, NB, CTAS) \
    SB_AP_KERNEL(name, CTAS, 8 * NB, SB_AP_WARPS, (attn_mmaw_body<T, HDP, NB>(P, it, ap_sm, bars, seq, &tm_k, &tm_v, box)))
#define SB_AP_MMA(name, T, HDP) \
    SB_AP_KERNEL(name, (HDP == 128 ? 2 : 3), 64, __shared__ long long off_s[SB_AP_RING][64], (attn_mma_body<T, HDP>(P, it, ap_sm, off_s)))
// (16 rows of heads of 128 need 250 registers: 24 rows behind 1194 keys, 16 heads on one: 27.5 us, with three CTAs and
// 168 registers 31.8)
#define SB_AP_F32(name, HDP, MT) \
    SB_AP_KERNEL(name, (MT * HDP == 2048 ? 2 : 3), MT, SB_AP_WARPS, (attn_f32_body<HDP, MT>(P, it, ap_sm, bars, seq, &tm_k, &tm_v, box)))
SB_AP_MMAW(attn_f16_64_r8, __half, 64, 1, 6)
SB_AP_MMAW(attn_f16_128_r8, __half, 128, 1, 4)
SB_AP_MMAW(attn_bf16_64_r8, __nv_bfloat16, 64, 1, 6)
SB_AP_MMAW(attn_bf16_128_r8, __nv_bfloat16, 128, 1, 4)
SB_AP_MMAW(attn_f16_64_r16, __half, 64, 2, 4)
SB_AP_MMAW(attn_f16_128_r16, __half, 128, 2, 3)
SB_AP_MMAW(attn_bf16_64_r16, __nv_bfloat16, 64, 2, 4)
SB_AP_MMAW(attn_bf16_128_r16, __nv_bfloat16, 128, 2, 3)
SB_AP_MMA(attn_f16_64_r64, __half, 64)
SB_AP_MMA(attn_f16_128_r64, __half, 128)
SB_AP_MMA(attn_bf16_64_r64, __nv_bfloat16, 64)
SB_AP_MMA(attn_bf16_128_r64, __nv_bfloat16, 128)
SB_AP_F32(attn_f32_64_r1, 64, 1)
SB_AP_F32(attn_f32_64_r2, 64, 2)
SB_AP_F32(attn_f32_64_r4, 64, 4)
SB_AP_F32(attn_f32_64_r8, 64, 8)
SB_AP_F32(attn_f32_64_r16, 64, 16)
SB_AP_F32(attn_f32_128_r1, 128, 1)
SB_AP_F32(attn_f32_128_r2, 128, 2)
SB_AP_F32(attn_f32_128_r4, 128, 4)
SB_AP_F32(attn_f32_128_r8, 128, 8)
SB_AP_F32(attn_f32_128_r16, 128, 16)

// ---------------------------------------------------------------- join
// A warp a (row, head): parts of the prefix, then those of the request's own
// keys that are in use, 32 at a time, a lane's weight each; then four values a
// lane, where head sizes up to 64, 32, ... let 2, 4, ... groups of lanes take
// parts side by side.  A part without weight may not have been written and
// does not count.  Bound by latency: the row count, the row's own parts and
// the parts' maxima and sums are read at once, then the parts themselves.
// type: 0 f32, 1 f16, 2 bf16.
extern "C" __global__ void __launch_bounds__(128) attn_join(const __grid_constant__ AttnParams P, int type) {
    const int lane = threadIdx.x & 31;
    const int width = P.HD > 64 ? 32 : P.HD > 32 ? 16 : P.HD > 16 ? 8 : 4, groups = 32 / width, d = (lane & (width - 1)) * 4;
    const long long TH = (long long)P.T * P.NH;
    pdl_wait();
    const long long rows = (long long)ap_rows(P) * P.NH;
    for (long long i = (long long)blockIdx.x * 4 + (threadIdx.x >> 5); i < TH; i += (long long)gridDim.x * 4) {
        const int row = TH >> 32 ? (int)(i / P.NH) : (int)((unsigned)i / (unsigned)P.NH), head = (int)(i - (long long)row * P.NH);
        const int most = P.S1 + P.S2, own = P.S2 ? min(max(P.ws_n[row], 0), P.S2) : 0;  // a row of no request has no count
        float M = -INFINITY, L = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        float2 ml = lane < most ? P.ws_ml[lane * TH + i] : make_float2(0.f, 0.f);
        if (i >= rows) return;  // rows behind the last request have no parts and stay as they were
        for (int base = 0; base < P.S1 + own; base += 32) {
            const int n = min(P.S1 + own - base, 32);
            if (base && lane < n) ml = P.ws_ml[(base + lane) * TH + i];
            const bool some = lane < n && ml.y != 0.f;
            const float top = fmaxf(M, warp_max(some ? ml.x : -INFINITY));
            if (base && M != -INFINITY) {
                const float f = ap_exp2(M - top);
                L *= f;
                acc = make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f);
            }
            M = top;
            const float weight = some ? ap_exp2(ml.x - M) : 0.f;
            if (some) L = fmaf(weight, ml.y, L);
#pragma unroll 4
            for (int s = 0; s < n; s += groups) {
                const int mine = s + lane / width;
                const float w = __shfl_sync(SB_FULL, weight, mine);
                float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
                if (w != 0.f && d < P.HD) o = *reinterpret_cast<const float4 *>(P.ws_o + ((base + mine) * TH + i) * P.HD + d);
                acc.x = fmaf(w, o.x, acc.x);
                acc.y = fmaf(w, o.y, acc.y);
                acc.z = fmaf(w, o.z, acc.z);
                acc.w = fmaf(w, o.w, acc.w);
            }
        }
        L = warp_sum(L);
        for (int o = width; o < 32; o <<= 1) {
            acc.x += __shfl_xor_sync(SB_FULL, acc.x, o);
            acc.y += __shfl_xor_sync(SB_FULL, acc.y, o);
            acc.z += __shfl_xor_sync(SB_FULL, acc.z, o);
            acc.w += __shfl_xor_sync(SB_FULL, acc.w, o);
        }
        const float inv = L == 0.f ? 0.f : 1.f / L;
        const long long at = row * P.o_row + head * P.o_head + d;
        if (lane < width && d < P.HD) {
            const float a = acc.x * inv, b = acc.y * inv, e = acc.z * inv, f = acc.w * inv;
            if (type == 0) *reinterpret_cast<float4 *>(static_cast<float *>(P.out) + at) = make_float4(a, b, e, f);
            else if (type == 1)
                *reinterpret_cast<uint2 *>(static_cast<__half *>(P.out) + at) = make_uint2(ap_pack<__half>(a, b), ap_pack<__half>(e, f));
            else
                *reinterpret_cast<uint2 *>(static_cast<__nv_bfloat16 *>(P.out) + at) =
                    make_uint2(ap_pack<__nv_bfloat16>(a, b), ap_pack<__nv_bfloat16>(e, f));
        }
        if (P.lse && lane == 0) P.lse[i] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
    }
}
