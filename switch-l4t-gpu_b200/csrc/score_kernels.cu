// score_kernels.cu -- the "score" module image (sm_100a cubin): log
// probabilities of given tokens with entropy, rank and the best
// alternatives, from one pass over the logits, and their gradient.  No
// counterpart in the reference, which samples one token a step.
//
// With c = log2(e) / temperature and m the maximum of a row,
//   s = sum 2^(c (x - m)),  t = sum 2^(c (x - m)) c (x - m)
//   lse = m / temperature + ln2 log2 s,  logp = ln2 (c (x_tok - m) - log2 s)
//   entropy = ln2 (log2 s - t / s)
// and a change of m turns (s, t) into f s, f (t + s d), f = 2^d: a thread
// keeps (m, s, t) of its values and looks at m once per four vectors.
// c (x - m) is one fma with the rounded product c m, the same in every term,
// so that its rounding cancels: while |c m| < 2^24 it is a factor of at most
// 2^(1/2) on s.  From 2^31 on that factor would pass FP32 (a thread that meets
// masks of -1e10 alone, a temperature of 1e-8), so larger maxima take the
// difference x - m first, a vector at a time (2048 x 151936 bf16, half of it
// masks of -1e9: 150 us, of -1e4: 120; unrolled over the tile it would be 144
// and 137).  Values whose product could overflow (masks of the type's lowest
// value, -inf) take a guarded form, chosen by the tile's minimum.  Sums are FP32.
//
// Bound: HBM (one read of the logits).  For 16-bit logits the 16 exponentials
// per SM and cycle are close behind, and issue slots too: about eight
// instructions a value, with maxima, minima and rank compares on packed pairs.
//
// The k best without a second pass.  A key is the value's order-preserving
// bits above the complemented id, so a larger key is a better candidate and
// equal values go to the lower id (-0 counts as +0); masked choices (-inf) are
// not listed.  On the way every thread leaves the maximum of each of its cells
// (a few tiles) in shared memory.  The k-th best of the threads' (or thread
// groups') maxima bounds the k-th best value from below: k holders each have a
// value at least that good.  So only cells that reach it -- 1.2 to 1.4 k of
// them -- are looked into again, a thread a vector, and what reaches it there
// is ranked by counting.  (Collecting candidates on the way, against a bound
// renewed tile by tile, cost three times as much: each hit stalls a warp, each
// renewal the block.)  Where too many reach it (equal or rising logits), the
// part's k best are taken by k passes instead.
#include <cfloat>
#include <cuda_bf16.h>

#include "sb_common.cuh"

#define LP_THREADS 128
#define LP_U 4        // vectors of a thread per tile
#define LP_LIST 512   // keys, and cells
#define LP_CELLS 32    // cells of a thread
#define LP_KMAX 64
#define LP_LN2 0.6931471805599453f
#define LP_L2E 1.4426950408889634f
#define LP_L2E_LO 1.925963033500e-08f  // log2 e less its FP32 value

// parameter block, mirrored by the host (host/sb_serve.c)
struct LpParams {
    const void *x;
    long long stride;  // elements
    int R, V, S, k;    // S parts per row, one CTA each
    float c, inv_temp;  // log2(e) / temperature
    const int *tok;
    float *logp, *entropy, *lse;
    int *rank, *top_ids;
    float *top_logp;
    float4 *part;                // [R][S]: m, s, t, rank count (bits)
    unsigned long long *keys;    // [R][S][k]
};

SB_DEV float lp_f(float v) { return v; }
SB_DEV float lp_f(__half v) { return __half2float(v); }
SB_DEV float lp_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> SB_DEV T lp_to(float v);
template <> SB_DEV float lp_to<float>(float v) { return v; }
template <> SB_DEV __half lp_to<__half>(float v) { return __float2half_rn(v); }
template <> SB_DEV __nv_bfloat16 lp_to<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
SB_DEV float lp_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
SB_DEV float lp_max_nan(float a, float b) {  // a NaN stays
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
SB_DEV unsigned long long lp_key(float v, int id) {
    const unsigned u = __float_as_uint(v == 0.f ? 0.f : v);
    return ((unsigned long long)((u & 0x80000000u) ? ~u : (u | 0x80000000u)) << 32) | (unsigned)~id;
}
SB_DEV float lp_key_value(unsigned long long k) {
    const unsigned u = (unsigned)(k >> 32);
    return __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u);
}
SB_DEV int lp_key_id(unsigned long long k) { return (int)~(unsigned)k; }

// sixteen bytes of a row: maximum and minimum (a NaN loses), values, and how
// many reach a bound (counted in the type itself: exact for the 16 of a tile)
template <typename T> struct LpVec;
template <> struct LpVec<float> {
    static constexpr int N = 4;
    static constexpr unsigned NEG_INF = 0xff800000u;
    using Count = int;
    using Bound = float;
    static SB_DEV float max(const uint4 &r) {
        return fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)), fmaxf(__uint_as_float(r.z), __uint_as_float(r.w)));
    }
    static SB_DEV float min(const uint4 &r) {
        return fminf(fminf(__uint_as_float(r.x), __uint_as_float(r.y)), fminf(__uint_as_float(r.z), __uint_as_float(r.w)));
    }
    static SB_DEV float max(const uint4 (&r)[LP_U]) { return fmaxf(fmaxf(max(r[0]), max(r[1])), fmaxf(max(r[2]), max(r[3]))); }
    static SB_DEV float min(const uint4 (&r)[LP_U]) { return fminf(fminf(min(r[0]), min(r[1])), fminf(min(r[2]), min(r[3]))); }
    static SB_DEV void values(const uint4 &r, float (&v)[4]) {
        v[0] = __uint_as_float(r.x);
        v[1] = __uint_as_float(r.y);
        v[2] = __uint_as_float(r.z);
        v[3] = __uint_as_float(r.w);
    }
    static SB_DEV uint4 packed(const float (&v)[4]) {
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
    static SB_DEV Bound bound(float v) { return v; }
    static SB_DEV Bound above(float v) {  // the next value up
        const unsigned u = __float_as_uint(v);
        return __uint_as_float(v == 0.f ? 1u : u & 0x80000000u ? u - 1 : u + 1);
    }
    static SB_DEV Count zero() { return 0; }
    static SB_DEV void count(const uint4 &r, Bound b, Count &n) {
        n += __uint_as_float(r.x) >= b;
        n += __uint_as_float(r.y) >= b;
        n += __uint_as_float(r.z) >= b;
        n += __uint_as_float(r.w) >= b;
    }
    static SB_DEV int total(Count n) { return n; }
};
template <typename T, typename T2> struct LpVec16 {
    static constexpr int N = 8;
    using Count = T2;
    using Bound = T2;
    static SB_DEV T2 pair(unsigned u) { return *reinterpret_cast<const T2 *>(&u); }
    static SB_DEV T2 max2(const uint4 &r) { return __hmax2(__hmax2(pair(r.x), pair(r.y)), __hmax2(pair(r.z), pair(r.w))); }
    static SB_DEV T2 min2(const uint4 &r) { return __hmin2(__hmin2(pair(r.x), pair(r.y)), __hmin2(pair(r.z), pair(r.w))); }
    static SB_DEV float max(const uint4 &r) {
        const T2 m = max2(r);
        return fmaxf(lp_f(m.x), lp_f(m.y));
    }
    static SB_DEV float max(const uint4 (&r)[LP_U]) {
        const T2 m = __hmax2(__hmax2(max2(r[0]), max2(r[1])), __hmax2(max2(r[2]), max2(r[3])));
        return fmaxf(lp_f(m.x), lp_f(m.y));
    }
    static SB_DEV float min(const uint4 (&r)[LP_U]) {
        const T2 m = __hmin2(__hmin2(min2(r[0]), min2(r[1])), __hmin2(min2(r[2]), min2(r[3])));
        return fminf(lp_f(m.x), lp_f(m.y));
    }
    static SB_DEV void values(const uint4 &r, float (&v)[8]) {
        const unsigned w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[2 * i] = lp_f(pair(w[i]).x);
            v[2 * i + 1] = lp_f(pair(w[i]).y);
        }
    }
    static SB_DEV unsigned pack(float a, float b) {
        if constexpr (__is_same(T, __half)) {
            const __half2 h = __floats2half2_rn(a, b);
            return *reinterpret_cast<const unsigned *>(&h);
        } else {
            const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
            return *reinterpret_cast<const unsigned *>(&h);
        }
    }
    static SB_DEV uint4 packed(const float (&v)[8]) { return make_uint4(pack(v[0], v[1]), pack(v[2], v[3]), pack(v[4], v[5]), pack(v[6], v[7])); }
    static SB_DEV Bound both(unsigned short b) { return pair(b * 0x10001u); }
    static SB_DEV unsigned short bits(float v) {  // v is a value of the type
        if constexpr (__is_same(T, __half)) return __half_as_ushort(__float2half_rn(v));
        else return __bfloat16_as_ushort(__float2bfloat16_rn(v));
    }
    static SB_DEV Bound bound(float v) { return both(bits(v)); }
    static SB_DEV Bound above(float v) {
        const unsigned short u = bits(v);
        return both(v == 0.f ? 1 : u & 0x8000 ? u - 1 : u + 1);
    }
    static SB_DEV Count zero() { return pair(0u); }
    static SB_DEV void count(const uint4 &r, Bound b, Count &n) {
        n = __hadd2(n, __hge2(pair(r.x), b));
        n = __hadd2(n, __hge2(pair(r.y), b));
        n = __hadd2(n, __hge2(pair(r.z), b));
        n = __hadd2(n, __hge2(pair(r.w), b));
    }
    static SB_DEV int total(Count n) { return (int)(lp_f(n.x) + lp_f(n.y)); }
};
template <> struct LpVec<__half> : LpVec16<__half, __half2> { static constexpr unsigned NEG_INF = 0xfc00fc00u; };
template <> struct LpVec<__nv_bfloat16> : LpVec16<__nv_bfloat16, __nv_bfloat162> { static constexpr unsigned NEG_INF = 0xff80ff80u; };

// value e of a vector, e not known at compile time (an indexed register array would live in memory)
template <typename T>
SB_DEV float lp_at(const uint4 &r, int e) {
    const int w = sizeof(T) == 4 ? e : e >> 1;
    const unsigned u = w & 2 ? (w & 1 ? r.w : r.z) : (w & 1 ? r.y : r.x);
    if constexpr (sizeof(T) == 4) return __uint_as_float(u);
    const unsigned short h = (unsigned short)(e & 1 ? u >> 16 : u);
    return lp_f(*reinterpret_cast<const T *>(&h));
}
// vector j of a row, counted from the 16-byte boundary at or below its start;
// values outside the row are -inf
template <typename T>
SB_DEV uint4 lp_load(const T *x, int lead, int V, int j) {
    constexpr int N = LpVec<T>::N;
    const int e0 = j * N - lead;
    if (e0 >= 0 && e0 + N <= V) return ld_stream_u4(x + e0);
    uint4 r = make_uint4(LpVec<T>::NEG_INF, LpVec<T>::NEG_INF, LpVec<T>::NEG_INF, LpVec<T>::NEG_INF);
    T *h = reinterpret_cast<T *>(&r);
#pragma unroll
    for (int e = 0; e < N; e++)
        if (e0 + e >= 0 && e0 + e < V) h[e] = x[e0 + e];
    return r;
}

// (m, s, t) of a set of values; m in logits, s and t as at the top
struct LpSum { float m, s, t; };
SB_DEV bool lp_sane(float cm) { return fabsf(cm) < 16777216.f; }  // of a product c m: rounded by at most 1/2
SB_DEV unsigned long long lp_add2(unsigned long long a, unsigned long long b) {  // two FP32 sums in one instruction
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
SB_DEV unsigned long long lp_mul2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// c (a - b) between two maxima that sums are held against: of the rounded products where they are
SB_DEV float lp_gap(float a, float b, float c) {
    const float ca = __fmul_rn(a, c), cb = __fmul_rn(b, c);
    const bool sa = lp_sane(ca), sb = lp_sane(cb);
    if (sa && sb) return ca - cb;
    return (a - b) * c + ((sb ? fmaf(b, c, -cb) : 0.f) - (sa ? fmaf(a, c, -ca) : 0.f));
}
SB_DEV void lp_raise(LpSum &a, float m, float c) {  // m >= a.m
    if (a.s != 0.f) {
        const float d = lp_max_nan(lp_gap(a.m, m, c), -200.f), f = lp_exp2(d);
        a.t = f * fmaf(a.s, d, a.t);
        a.s *= f;
    }
    a.m = m;
}
// all threads' sums and counts: the common maximum first, then plain sums.
// lp_s: [3][warps]; a barrier must stand before its next use.
struct LpShared { float m[LP_THREADS / 32], s[LP_THREADS / 32], t[LP_THREADS / 32]; int n[LP_THREADS / 32]; };
SB_DEV void lp_block(LpSum &a, int &above, float c, LpShared &sh) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float m = warp_max(a.m);
    if (lane == 0) sh.m[warp] = m;
    __syncthreads();
    m = sh.m[0];
#pragma unroll
    for (int w = 1; w < LP_THREADS / 32; w++) m = fmaxf(m, sh.m[w]);
    lp_raise(a, m, c);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        a.s += __shfl_xor_sync(SB_FULL, a.s, o);
        a.t += __shfl_xor_sync(SB_FULL, a.t, o);
    }
    above = __reduce_add_sync(SB_FULL, above);
    if (lane == 0) {
        sh.s[warp] = a.s;
        sh.t[warp] = a.t;
        sh.n[warp] = above;
    }
    __syncthreads();
    a = {m, 0.f, 0.f};
    above = 0;
#pragma unroll
    for (int w = 0; w < LP_THREADS / 32; w++) {
        a.s += sh.s[w];
        a.t += sh.t[w];
        above += sh.n[w];
    }
}

// ln2 (c (x - m) - l2) of a value against finished sums
SB_DEV float lp_logp(float x, float m, float l2, float c) {
    const float cm = __fmul_rn(m, c);
    return ((lp_sane(cm) ? fmaf(x, c, -cm) : (x - m) * c) - l2) * LP_LN2;
}
// a row of masked choices has m = -inf and s = 0
SB_DEV float lp_lse(LpSum a, float l2, float c, float inv_temp) {
    const float cm = __fmul_rn(a.m, c);
    return a.m == -INFINITY && a.s == 0.f ? -INFINITY : lp_sane(cm) ? (cm + l2) * LP_LN2 : fmaf(l2, LP_LN2, a.m * inv_temp);
}
// results of a row from its joined sums
SB_DEV void lp_finish(const LpParams &P, int r, LpSum a, int above, float xt, bool given) {
    const bool none = a.m == -INFINITY && a.s == 0.f;
    const float l2 = log2f(a.s);
    if (P.lse) P.lse[r] = lp_lse(a, l2, P.c, P.inv_temp);
    if (P.entropy) P.entropy[r] = none ? 0.f : (l2 - a.t / a.s) * LP_LN2;
    if (P.logp) P.logp[r] = !given ? 0.f : none ? -INFINITY : lp_logp(xt, a.m, l2, P.c);
    if (P.rank) P.rank[r] = given ? above : -1;
}
SB_DEV void lp_top(const LpParams &P, int r, int i, unsigned long long key, float m, float l2) {
    if (P.top_ids) P.top_ids[(long long)r * P.k + i] = key ? lp_key_id(key) : -1;
    if (P.top_logp) P.top_logp[(long long)r * P.k + i] = key ? lp_logp(lp_key_value(key), m, l2, P.c) : -INFINITY;
}
// the first k of n keys in a list, ranked by counting, as emit(rank, key)
template <typename F>
SB_DEV void lp_rank(const unsigned long long *list, int n, int k, F emit) {
    for (int i = threadIdx.x; i < n; i += LP_THREADS) {
        const unsigned long long me = list[i];
        int r = 0;
        for (int j = 0; j < n; j++) r += list[j] > me;
        if (r < k) emit(r, me);
    }
}

// CTA = part s of row r: vectors [n s / S, n (s + 1) / S) of the row
template <typename T, bool TOP>
SB_DEV void logprobs_body(const LpParams &P) {
    using Vec = LpVec<T>;
    constexpr int N = Vec::N, TILE = LP_THREADS * LP_U;
    __shared__ LpShared sum_s;
    __shared__ unsigned long long list[TOP ? LP_LIST : 1];
    __shared__ T cell_s[TOP ? LP_CELLS : 1][LP_THREADS];
    __shared__ __align__(16) float best_s[TOP ? LP_THREADS : 4];
    __shared__ unsigned short hit_s[TOP ? LP_LIST : 1];
    __shared__ int n_s, hits_s;
    __shared__ float thr_s;
    const int tid = threadIdx.x;
    const int r = blockIdx.x / P.S, part = blockIdx.x % P.S;
    pdl_launch_dependents();
    const T *x = static_cast<const T *>(P.x) + r * P.stride;
    const int lead = (int)(((uintptr_t)x & 15) / sizeof(T));  // places of the first vector that are not the row's
    const int nv = (int)(((long long)lead + P.V + N - 1) / N);
    const int v0 = P.S == 1 ? 0 : (int)((long long)nv * part / P.S), v1 = P.S == 1 ? nv : (int)((long long)nv * (part + 1) / P.S);
    const int whole1 = min((int)(((long long)lead + P.V) / N), v1);  // vectors that end inside the row
    const int tok = P.tok ? P.tok[r] : -1;
    const bool given = tok >= 0 && tok < P.V, count = P.rank && given;
    const float xt = given ? lp_f(x[tok]) : 0.f, c = P.c;
    const int jt = given ? (tok + lead) / N : -1;  // the token's vector
    // ids before the token's vector count when equal, later ones do not; equal ids inside it, and
    // masked ones where the token is masked itself, are added behind the loop
    const typename Vec::Bound more = Vec::above(xt), at_least = xt == -INFINITY ? more : Vec::bound(xt);

    LpSum a = {-INFINITY, 0.f, 0.f};
    int above = 0;
    float best = -INFINITY, cell_best = -INFINITY;
    const int tiles = (v1 - v0 + TILE - 1) / TILE, per_cell = (tiles + LP_CELLS - 1) / LP_CELLS;  // tiles of a cell
    int tile = 0, cell = 0, cell_end = per_cell;
    if (TOP && tid == 0) {
        n_s = hits_s = 0;
        thr_s = -FLT_MAX;
    }

    // A whole tile's loads are issued a tile ahead: twice the bytes in flight (10 us of 338 for 2048 x 151936 bf16
    // with the gradient; 1056 x 50257 FP32 with 5 alternatives 46 against 72 us).  16-bit types with alternatives
    // have more CTAs per SM instead, which overlap the part behind the loop better (36 against 37 us).
    uint4 raw[LP_U], ahead[LP_U];
    bool loaded = false;
    for (int b = v0; b < v1; b += TILE, tile++) {
        if (loaded) {
#pragma unroll
            for (int u = 0; u < LP_U; u++) raw[u] = ahead[u];
        } else {
#pragma unroll
            for (int u = 0; u < LP_U; u++) {
                const int j = b + u * LP_THREADS + tid;
                raw[u] = make_uint4(Vec::NEG_INF, Vec::NEG_INF, Vec::NEG_INF, Vec::NEG_INF);
                if (j < v1) raw[u] = lp_load(x, lead, P.V, j);
            }
        }
        loaded = (!TOP || sizeof(T) == 4) && b + 2 * TILE <= whole1;
        if (loaded) {
#pragma unroll
            for (int u = 0; u < LP_U; u++) ahead[u] = ld_stream_u4(x + ((b + TILE + u * LP_THREADS + tid) * N - lead));
        }
        const float mx = Vec::max(raw), mn = Vec::min(raw);
        best = fmaxf(best, mx);
        if (best > a.m) lp_raise(a, best, c);
        const float mc = __fmul_rn(a.m, c);
        const bool sane = lp_sane(mc);
        if (sane) {
            const unsigned long long c2 = f2_pack(c, c), mc2 = f2_pack(-mc, -mc);
            unsigned long long s2 = 0ull, t2 = 0ull;
            if (mn > -1e30f) {
#pragma unroll
                for (int u = 0; u < LP_U; u++) {
                    float v[N];
                    Vec::values(raw[u], v);
#pragma unroll
                    for (int e = 0; e < N; e += 2) {
                        const unsigned long long d2 = ffma2(f2_pack(v[e], v[e + 1]), c2, mc2);
                        float d0, d1;
                        f2_unpack(d2, d0, d1);
                        const unsigned long long w2 = f2_pack(lp_exp2(d0), lp_exp2(d1));
                        s2 = lp_add2(s2, w2);
                        t2 = ffma2(w2, d2, t2);
                    }
                }
            } else {  // masked or absent values among them: a product of -inf becomes a power of two that is 0
#pragma unroll
                for (int u = 0; u < LP_U; u++) {
                    float v[N];
                    Vec::values(raw[u], v);
#pragma unroll
                    for (int e = 0; e < N; e += 2) {
                        const float d0 = lp_max_nan(fmaf(v[e], c, -mc), -200.f), d1 = lp_max_nan(fmaf(v[e + 1], c, -mc), -200.f);
                        const unsigned long long w2 = f2_pack(lp_exp2(d0), lp_exp2(d1));
                        s2 = lp_add2(s2, w2);
                        t2 = ffma2(w2, f2_pack(d0, d1), t2);
                    }
                }
            }
            a.s += f2_sum(s2);
            a.t += f2_sum(t2);
        } else if (a.m == -INFINITY) {  // masked choices only so far: no weight, but a NaN among them stays
            float sum = 0.f;
#pragma unroll
            for (int u = 0; u < LP_U; u++) {
                float v[N];
                Vec::values(raw[u], v);
#pragma unroll
                for (int e = 0; e < N; e++) sum += v[e];
            }
            if (sum != sum) a.s = sum;
        } else {  // a large maximum: differences first
#pragma unroll 1
            for (int u = 0; u < LP_U; u++) {  // a vector at a time, the tile turned round
                float v[N];
                Vec::values(raw[0], v);
#pragma unroll
                for (int e = 0; e < N; e++) {
                    const float d = lp_max_nan((v[e] - a.m) * c, -200.f), w = lp_exp2(d);
                    a.s += w;
                    a.t = fmaf(w, d, a.t);
                }
                const uint4 first = raw[0];
#pragma unroll
                for (int i = 0; i + 1 < LP_U; i++) raw[i] = raw[i + 1];
                raw[LP_U - 1] = first;
            }
        }
        if (count) {
            typename Vec::Count n = Vec::zero();
#pragma unroll
            for (int u = 0; u < LP_U; u++) Vec::count(raw[u], b + u * LP_THREADS + tid < jt ? at_least : more, n);
            above += Vec::total(n);
        }
        if constexpr (TOP) {
            cell_best = fmaxf(cell_best, mx);
            if (tile + 1 == cell_end || b + TILE >= v1) {
                cell_s[cell++][tid] = lp_to<T>(cell_best);  // exact: a value of the type
                cell_best = -INFINITY;
                cell_end += per_cell;
            }
        }
    }
    if (count) {
        if (tid < N && jt >= v0 && jt < v1) {
            const int id = jt * N - lead + tid;
            above += id >= 0 && id < tok && lp_f(x[id]) == xt;
        }
        if (xt == -INFINITY)
            for (int id = max(v0 * N - lead, 0) + tid; id < min(v1, jt) * N - lead; id += LP_THREADS) above += lp_f(x[id]) == xt;
    }
    lp_block(a, above, c, sum_s);
    if (tid == 0) {
        if (P.S == 1) lp_finish(P, r, a, above, xt, given);
        else P.part[(long long)r * P.S + part] = make_float4(a.m, a.s, a.t, __int_as_float(above));
    }
    if constexpr (TOP) {
        // group maxima, one per 1, 2 or 4 threads: 2 to 4 times k of them leave 1.2 to 1.4 k cells
        const int per = P.k > 24 ? 1 : P.k > 8 ? 2 : 4, groups = LP_THREADS / per;
        float g = best;
        for (int o = 1; o < per; o <<= 1) g = fmaxf(g, __shfl_xor_sync(SB_FULL, g, o));
        if (tid % per == 0) best_s[tid / per] = g;
        __syncthreads();
        if (tid < groups) {
            g = best_s[tid];
            int rk = 0;
            for (int i = 0; i < groups; i += 4) {
                const float4 o = *reinterpret_cast<const float4 *>(best_s + i);
                rk += (o.x > g || (o.x == g && i < tid)) + (o.y > g || (o.y == g && i + 1 < tid)) +
                      (o.z > g || (o.z == g && i + 2 < tid)) + (o.w > g || (o.w == g && i + 3 < tid));
            }
            if (rk == P.k - 1 && g > thr_s) thr_s = g;
        }
        __syncthreads();
        const float thr = thr_s;  // at least the lowest finite value
        if (best >= thr)
            for (int i = 0; i < cell; i++)
                if (lp_f(cell_s[i][tid]) >= thr) {
                    const int at = atomicAdd(&hits_s, 1);
                    if (at < LP_LIST) hit_s[at] = (unsigned short)(i * LP_THREADS + tid);
                }
        __syncthreads();
        const int hits = hits_s, vecs = per_cell * LP_U;  // vectors of a cell
        if (hits <= LP_LIST)
            for (int i = tid; i < hits * vecs; i += LP_THREADS) {
                const int h = i / vecs, u = i - h * vecs, at = hit_s[h];
                const int j = v0 + ((at / LP_THREADS) * vecs + u) * LP_THREADS + at % LP_THREADS;
                if (j >= v1) continue;
                const uint4 w = lp_load(x, lead, P.V, j);
                if (Vec::max(w) < thr) continue;
                float v[N];
                Vec::values(w, v);
#pragma unroll
                for (int e = 0; e < N; e++)
                    if (v[e] >= thr) {
                        const int slot = atomicAdd(&n_s, 1);
                        if (slot < LP_LIST) list[slot] = lp_key(v[e], j * N - lead + e);
                    }
            }
        __syncthreads();
        int n = n_s;
        if (hits > LP_LIST || n > LP_LIST) {  // k passes: the best key below the last one
            unsigned long long last = ~0ull;
            for (n = 0; n < P.k; n++) {
                unsigned long long top = 0ull;
                for (int j = v0 + tid; j < v1; j += LP_THREADS) {
                    const uint4 w = lp_load(x, lead, P.V, j);
                    if (Vec::max(w) < thr) continue;
#pragma unroll 1
                    for (int e = 0; e < N; e++) {
                        const float y = lp_at<T>(w, e);
                        const unsigned long long key = y >= thr ? lp_key(y, j * N - lead + e) : 0ull;
                        if (key < last && key > top) top = key;
                    }
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    const unsigned long long other = __shfl_xor_sync(SB_FULL, top, o);
                    top = other > top ? other : top;
                }
                __syncthreads();
                if ((tid & 31) == 0) list[LP_KMAX + (tid >> 5)] = top;
                __syncthreads();
                for (int w = 0; w < LP_THREADS / 32; w++) top = list[LP_KMAX + w] > top ? list[LP_KMAX + w] : top;
                if (top == 0ull) break;
                if (tid == 0) list[n] = top;
                last = top;
            }
            __syncthreads();
        }
        const float l2 = log2f(a.s);
        unsigned long long *out = P.keys + ((long long)r * P.S + part) * P.k;
        lp_rank(list, n, P.k, [&](int i, unsigned long long key) {
            if (P.S == 1) lp_top(P, r, i, key, a.m, l2);
            else out[i] = key;
        });
        for (int i = n + tid; i < P.k; i += LP_THREADS) {
            if (P.S == 1) lp_top(P, r, i, 0ull, a.m, l2);
            else out[i] = 0ull;
        }
    }
}
#define LP_KERNEL(name, T, TOP, CTAS) \
    extern "C" __global__ void __launch_bounds__(LP_THREADS, CTAS) name(const __grid_constant__ LpParams P) { logprobs_body<T, TOP>(P); }
LP_KERNEL(logprobs_f32, float, false, 8)
LP_KERNEL(logprobs_f16, __half, false, 8)
LP_KERNEL(logprobs_bf16, __nv_bfloat16, false, 8)
LP_KERNEL(logprobs_top_f32, float, true, 8)
LP_KERNEL(logprobs_top_f16, __half, true, 10)
LP_KERNEL(logprobs_top_bf16, __nv_bfloat16, true, 10)

// A CTA a row: the parts' sums, and the k best of their S sorted lists.  With
// S >= k the k-th best list head bounds the k-th best key from below, so at
// most k lists matter; with fewer lists the worst of their entries at depth
// ceil(k / S) does.  What reaches the bound (at most max(k, S) k <= 4096 keys,
// in general some more than k) is ranked by counting.
// type: 0 f32, 1 f16, 2 bf16.
extern "C" __global__ void __launch_bounds__(LP_THREADS) logprobs_join(const __grid_constant__ LpParams P, int type) {
    __shared__ LpShared sum_s;
    __shared__ unsigned long long list[LP_KMAX * LP_KMAX], head_s[LP_THREADS];
    __shared__ unsigned long long bound_s;
    __shared__ int n_s, lists_n, lists_s[LP_THREADS];
    const int tid = threadIdx.x, r = blockIdx.x;
    const int tok = P.tok ? P.tok[r] : -1;
    const bool given = tok >= 0 && tok < P.V;
    float xt = 0.f;
    if (given) {
        const long long at = r * P.stride + tok;
        xt = type == 0 ? static_cast<const float *>(P.x)[at]
                       : type == 1 ? lp_f(static_cast<const __half *>(P.x)[at]) : lp_f(static_cast<const __nv_bfloat16 *>(P.x)[at]);
    }
    pdl_wait();
    // S <= LP_THREADS: a part a thread
    LpSum a = {-INFINITY, 0.f, 0.f};
    int above = 0;
    const int depth = P.S >= P.k ? 1 : (P.k + P.S - 1) / P.S;
    unsigned long long head = 0ull;
    const unsigned long long *keys = P.keys + (long long)r * P.S * P.k;
    if (tid < P.S) {
        const float4 p = P.part[(long long)r * P.S + tid];
        if (P.k) head = keys[(long long)tid * P.k + depth - 1];
        a = {p.x, p.y, p.z};
        above = __float_as_int(p.w);
    }
    head_s[tid] = head;
    if (tid == 0) {
        n_s = lists_n = 0;
        bound_s = 0ull;
    }
    lp_block(a, above, P.c, sum_s);
    if (tid == 0) lp_finish(P, r, a, above, xt, given);
    if (P.k == 0) return;
    const float l2 = log2f(a.s);
    if (tid < P.S) {
        int rk = 0;
        for (int j = 0; j < P.S; j++) rk += head_s[j] > head || (head_s[j] == head && j < tid);
        if (rk == (P.S >= P.k ? P.k : P.S) - 1) bound_s = head;
    }
    __syncthreads();
    const unsigned long long bound = bound_s;
    // the lists that matter, then their keys, a thread a key
    const bool matters = tid < P.S && (depth > 1 || (head && head >= bound));
    if (matters) lists_s[atomicAdd(&lists_n, 1)] = tid;
    __syncthreads();
    const int total = lists_n * P.k;
#pragma unroll 4
    for (int i = tid; i < total; i += LP_THREADS) {
        const int h = i / P.k;
        const unsigned long long key = keys[(long long)lists_s[h] * P.k + i - h * P.k];
        if (key && key >= bound) list[atomicAdd(&n_s, 1)] = key;
    }
    __syncthreads();
    const int n = n_s;
    lp_rank(list, n, P.k, [&](int i, unsigned long long key) { lp_top(P, r, i, key, a.m, l2); });
    for (int i = n + tid; i < P.k; i += LP_THREADS) lp_top(P, r, i, 0ull, a.m, l2);
}

// ---------------------------------------------------------------- gradient
// d logits[v] = (g_logp (1[v = tok] - p_v) - g_entropy p_v (ln p_v + H)) / temperature,
// p_v = e^(x_v - lse).  Bound: HBM, one read and one write.  lse log2(e) is
// held as two floats: its rounding alone would be 1e-6 of every p.  What lse
// lost when it was rounded to FP32 is half a step, |lse| 2^-24 of every p.
// Below LP_FAR that is at most 2^-17 (16-bit types 2^-15); a row beyond (a
// common offset of the logits, a tiny temperature, nothing but the type's
// lowest value, -inf) is the work of one CTA, which takes its maximum and sum
// again as the forward pass does, before anything of it is written (grad may
// be the logits): 2048 x 151936 bf16 offset by 1e4 357 us instead of 205, 300 x
// 50257 FP32 67 instead of 22, one row of 151936 109 instead of 3.5.  An lse
// that is not the row's own is used as given.
struct LpGradParams {
    const void *x;
    void *dx;
    long long stride, dstride;
    int R, V, S;
    float c, inv_temp;
    const int *tok;
    const float *lse, *entropy, *g_logp, *g_entropy;
};
template <typename T> constexpr float LP_FAR = sizeof(T) == 4 ? 256.f : 1024.f;
// dx = -p (a0 + a1 log2 p) / temperature with log2 p = d - lo: 2^-lo goes into the factors
struct LpFactors { float lo, gl, b0, b1; };
SB_DEV LpFactors lp_factors(const LpGradParams &P, int r, bool given, float lo) {
    const float gl = given && P.g_logp ? P.g_logp[r] * P.inv_temp : 0.f, ge = P.g_entropy ? P.g_entropy[r] * P.inv_temp : 0.f;
    const float a1 = ge * LP_LN2, a0 = gl + ge * (P.g_entropy ? P.entropy[r] : 0.f), f = lp_exp2(-lo);
    return {lo, gl, -(a0 - a1 * lo) * f, -a1 * f};
}
// one value at d, any range
SB_DEV float lp_grad1(float d, const LpFactors &F, bool token) {
    d = lp_max_nan(d, -200.f);
    const float g = lp_exp2(d) * fmaf(F.b1, d, F.b0);
    return token ? g + F.gl : g;
}
// vector j of a row, and its gradient
template <typename T> SB_DEV uint4 lp_load_again(const T *x, int lead, int V, int j) {  // not as constant memory
    const int e0 = j * LpVec<T>::N - lead;
    return e0 >= 0 && e0 + LpVec<T>::N <= V ? *reinterpret_cast<const uint4 *>(x + e0) : lp_load(x, lead, V, j);
}
template <typename T> SB_DEV void lp_store(T *dx, bool same, int lead, int V, int j, const float (&v)[LpVec<T>::N]) {
    constexpr int N = LpVec<T>::N;
    const int e0 = j * N - lead;
    if (same && e0 >= 0 && e0 + N <= V) *reinterpret_cast<uint4 *>(dx + e0) = LpVec<T>::packed(v);
    else
#pragma unroll
        for (int e = 0; e < N; e++)
            if (e0 + e >= 0 && e0 + e < V) dx[e0 + e] = lp_to<T>(v[e]);
}
// A row whose lse is far from 0, by one CTA.  Not inlined: its code and registers are not those of the kernel below.
template <typename T>
__device__ __noinline__ void logprobs_grad_far(const LpGradParams &P, int r) {
    using Vec = LpVec<T>;
    constexpr int N = Vec::N, STEP = LP_THREADS * LP_U;
    __shared__ LpShared sum_s;
    const T *x = static_cast<const T *>(P.x) + r * P.stride;
    T *dx = static_cast<T *>(P.dx) + r * P.dstride;
    const int lead = (int)(((uintptr_t)x & 15) / sizeof(T)), nv = (int)(((long long)lead + P.V + N - 1) / N);
    const bool same = (((uintptr_t)x ^ (uintptr_t)dx) & 15) == 0;
    const float c = P.c, lse = P.lse[r];
    uint4 raw[LP_U];
    LpSum a = {-INFINITY, 0.f, 0.f};
    for (int b = threadIdx.x; b < nv; b += STEP) {
#pragma unroll
        for (int u = 0; u < LP_U; u++) {
            raw[u] = make_uint4(Vec::NEG_INF, Vec::NEG_INF, Vec::NEG_INF, Vec::NEG_INF);
            if (b + u * LP_THREADS < nv) raw[u] = lp_load_again(x, lead, P.V, b + u * LP_THREADS);
        }
        const float mx = Vec::max(raw);
        if (mx > a.m) lp_raise(a, mx, c);
        if (a.m == -INFINITY) continue;
        const float mc = __fmul_rn(a.m, c);
        const bool sane = lp_sane(mc);
        const float off = sane ? 0.f : a.m, base = sane ? -mc : 0.f;
#pragma unroll
        for (int u = 0; u < LP_U; u++) {
            float v[N];
            Vec::values(raw[u], v);
#pragma unroll
            for (int e = 0; e < N; e++) a.s += lp_exp2(fmaf(v[e] - off, c, base));
        }
        a.t = 0.f;
    }
    int count = 0;
    lp_block(a, count, c, sum_s);
    // p = 2^(d - lo), d = (x k - off) c1 - hi
    const float l2 = log2f(a.s), own = lp_lse(a, l2, c, P.inv_temp);
    float k = 1.f, off = 0.f, c1 = c, hi = 0.f, lo = 0.f;
    bool none = lse == -INFINITY;
    if (own == lse || fabsf(own - lse) <= fabsf(lse) * 4.76837158e-7f) {  // 2^-21: both are rounded, on either side
        none = a.m == -INFINITY;
        const float cm = __fmul_rn(a.m, c);
        if (lp_sane(cm)) hi = cm;
        else off = a.m;
        lo = none ? 0.f : l2;
    } else if (fabsf(lse) < 1e30f) {  // of more than this row
        hi = lse * LP_L2E;
        lo = fmaf(lse, LP_L2E, -hi) + lse * LP_L2E_LO;
    } else {
        k = P.inv_temp;
        off = lse;
        c1 = LP_L2E;
    }
    const int tok = P.tok ? P.tok[r] : -1;
    const LpFactors F = lp_factors(P, r, tok >= 0 && tok < P.V, lo);
    for (int b = threadIdx.x; b < nv; b += STEP) {
#pragma unroll
        for (int u = 0; u < LP_U; u++)
            if (b + u * LP_THREADS < nv) raw[u] = lp_load_again(x, lead, P.V, b + u * LP_THREADS);
#pragma unroll
        for (int u = 0; u < LP_U; u++) {
            const int j = b + u * LP_THREADS;
            if (j >= nv) break;
            float v[N];
            Vec::values(raw[u], v);
#pragma unroll
            for (int e = 0; e < N; e++) v[e] = none ? 0.f : lp_grad1(fmaf(fmaf(v[e], k, -off), c1, -hi), F, j * N - lead + e == tok);
            lp_store(dx, same, lead, P.V, j, v);
        }
    }
}
template <typename T>
SB_DEV void logprobs_grad_body(const LpGradParams &P) {
    using Vec = LpVec<T>;
    constexpr int N = Vec::N, TILE = LP_THREADS * LP_U;
    const int r = blockIdx.x / P.S, part = blockIdx.x % P.S, tid = threadIdx.x;
    const T *x = static_cast<const T *>(P.x) + r * P.stride;
    T *dx = static_cast<T *>(P.dx) + r * P.dstride;
    const int lead = (int)(((uintptr_t)x & 15) / sizeof(T));
    const bool same = (((uintptr_t)x ^ (uintptr_t)dx) & 15) == 0;  // else the vectors of dx would straddle
    const int nv = (int)(((long long)lead + P.V + N - 1) / N);
    const int v0 = (int)((long long)nv * part / P.S), v1 = (int)((long long)nv * (part + 1) / P.S);
    const int whole0 = lead ? 1 : 0, whole1 = min((int)(((long long)lead + P.V) / N), v1);
    const int tok = P.tok ? P.tok[r] : -1;
    const bool given = tok >= 0 && tok < P.V;
    const int jt = given ? (tok + lead) / N : -1;
    const float lse = P.lse[r];
    if (fabsf(lse) >= LP_FAR<T>) {  // not a NaN: that makes a row of them
        if (part == 0) logprobs_grad_far<T>(P, r);
        return;
    }
    const float hi = lse * LP_L2E;
    const LpFactors F = lp_factors(P, r, given, fmaf(lse, LP_L2E, -hi) + lse * LP_L2E_LO);
    auto grad = [&](float v, int id) { return lp_grad1(fmaf(v, P.c, -hi), F, id == tok); };
    // values above this need no such limit: |b1 d| stays below 1e37 (a power of two of 0 times an infinity is NaN)
    const float least = fmaxf(-1e30f, (hi - 1e37f / fmaxf(fabsf(F.b1), 1.f)) / P.c);
    const unsigned long long c2 = f2_pack(P.c, P.c), hi2 = f2_pack(-hi, -hi), b12 = f2_pack(F.b1, F.b1), b02 = f2_pack(F.b0, F.b0);
    for (int b = v0; b < v1; b += TILE) {
        uint4 raw[LP_U];
        const bool whole = same && b >= whole0 && b + TILE <= whole1;
        if (whole) {
#pragma unroll
            for (int u = 0; u < LP_U; u++) raw[u] = *reinterpret_cast<const uint4 *>(x + ((b + u * LP_THREADS + tid) * N - lead));
            if (Vec::min(raw) > least) {
#pragma unroll
                for (int u = 0; u < LP_U; u++) {
                    const int j = b + u * LP_THREADS + tid;
                    float v[N];
                    Vec::values(raw[u], v);
                    if (j == jt) continue;  // written below
#pragma unroll
                    for (int e = 0; e < N; e += 2) {
                        const unsigned long long d2 = ffma2(f2_pack(v[e], v[e + 1]), c2, hi2);
                        float d0, d1;
                        f2_unpack(d2, d0, d1);
                        const unsigned long long g2 = lp_mul2(f2_pack(lp_exp2(d0), lp_exp2(d1)), ffma2(b12, d2, b02));
                        f2_unpack(g2, v[e], v[e + 1]);
                    }
                    *reinterpret_cast<uint4 *>(dx + (j * N - lead)) = Vec::packed(v);
                }
                if (jt >= b && jt < b + TILE && (jt - b) % LP_THREADS == tid) {
#pragma unroll
                    for (int u = 0; u < LP_U; u++) {
                        const int j = b + u * LP_THREADS + tid;
                        float v[N];
                        Vec::values(raw[u], v);
                        if (j != jt) continue;
#pragma unroll
                        for (int e = 0; e < N; e++) v[e] = grad(v[e], j * N - lead + e);
                        *reinterpret_cast<uint4 *>(dx + (j * N - lead)) = Vec::packed(v);
                    }
                }
                continue;
            }
        }
#pragma unroll
        for (int u = 0; u < LP_U; u++) {
            const int j = b + u * LP_THREADS + tid, e0 = j * N - lead;
            if (j >= v1) break;
            if (same && e0 >= 0 && e0 + N <= P.V) {
                if (!whole) raw[u] = *reinterpret_cast<const uint4 *>(x + e0);
                float v[N];
                Vec::values(raw[u], v);
#pragma unroll
                for (int e = 0; e < N; e++) v[e] = grad(v[e], e0 + e);
                *reinterpret_cast<uint4 *>(dx + e0) = Vec::packed(v);
            } else {
                for (int e = 0; e < N; e++)
                    if (e0 + e >= 0 && e0 + e < P.V) dx[e0 + e] = lp_to<T>(grad(lp_f(x[e0 + e]), e0 + e));
            }
        }
    }
}
#define LP_GRAD(name, T) \
    extern "C" __global__ void __launch_bounds__(LP_THREADS) name(const __grid_constant__ LpGradParams P) { logprobs_grad_body<T>(P); }
LP_GRAD(logprobs_grad_f32, float)
LP_GRAD(logprobs_grad_f16, __half)
LP_GRAD(logprobs_grad_bf16, __nv_bfloat16)
