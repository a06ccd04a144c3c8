// serve_attn_tc.cuh -- the shared prefix of attn_prefix on the tcgen05 tensor
// cores (f16 / bf16): many query rows of a key head against a range of keys.
//
// Item = (key head, 256 stacked query rows, key range), one CTA of 16 warps:
//   warps 0-3, 4-7    softmax of row tile A / B (128 rows each, a thread a row)
//   warps 8-9, 10-11  loaders of K and V: tiles of 128 keys, two (HD 128) or
//                     four (HD 64) stages with the 128-byte swizzle; whole
//                     pages by TMA boxes, tiles that end inside a page, miss
//                     one, or have pages of other sizes by cp.async
//   warp 12           issues the tcgen05.mma of both products
// S = Q K^T (128 x 128, FP32) and P V run on the tensor pipe with S, P and O
// in tensor memory: the softmax threads read S, write P as 16-bit pairs over
// it (the A operand of the second product), and O stays there until the end.
// While one tile's softmax runs, the pipe works on the other tile: PV(t) and
// S(t + 1) of a tile are issued together as soon as its weights are there.
//
// The running maximum is lazy: O is rescaled only when a row's maximum has
// grown by more than 2^8 since the last time (weights up to 256 are as exact
// as weights up to 1 in floating point), which leaves a few rescales a row.
//
// Bound: 16 exponentials per SM and cycle (1024 cycles for a tile of 128 x
// 128), against 512 (HD 64) or 1024 (HD 128) cycles of the tensor pipe.
//
// Every wait is bounded; after a timeout tc_err is set, the roles stop, what
// was issued drains, and the tensor memory is freed.
#pragma once
#include <cuda.h>

#include "serve_attn.cuh"

#define ATC_POLY 4

namespace atc {
constexpr int THREADS = 512, BM = 128, KT = 128;
template <int HDP> struct Cfg {
    static constexpr int ST = HDP == 128 ? 2 : 4, SUB = HDP / 64, TILE = KT * HDP * 2;
    static constexpr int SMEM = 1024 + (2 * ST + 2) * TILE;
};
// the same for a converged warp, one answer for all lanes
SB_DEV bool warp_wait(uint64_t *mb, unsigned ph, unsigned call) { return __all_sync(SB_FULL, ap_bar_wait(mb, ph, call)); }
SB_DEV void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
SB_DEV void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// 128-byte swizzled operand: rows (K-major: query rows or keys; MN-major: keys)
// of 128 bytes, 8-row atoms 1024 bytes apart, 64-value column blocks 16 KB apart
SB_DEV uint64_t desc(unsigned addr) {
    return (uint64_t)((addr >> 4) & 0x3fffu) | ((uint64_t)(16384 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// f32 accumulator, M = 128; B K-major (keys as rows) or MN-major (values along N)
template <typename T> SB_DEV uint32_t idesc(int n, bool b_mn) {
    constexpr uint32_t fmt = __is_same(T, __half) ? 0u : 1u;
    return (1u << 4) | (fmt << 7) | (fmt << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
}
SB_DEV void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b),
        "r"(id), "r"(acc)
        : "memory");
}
SB_DEV void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b),
        "r"(id), "r"(acc)
        : "memory");
}
SB_DEV void commit(uint64_t *mb) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(ap_smem(mb)) : "memory");
}
#define ATC_R32(r) \
    "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), \
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), \
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), \
        "=r"(r[31])
// 32 columns of this warp's 32 lanes; wait_ld before the registers are read
SB_DEV void ld32(uint32_t addr, unsigned (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,"
        "%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : ATC_R32(r)
        : "r"(addr));
}
#define ATC_W32(r) \
    "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), \
        "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), \
        "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29])
// waits for every load of this thread; r's values are used behind it only
SB_DEV void wait_ld(unsigned (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : ATC_W32(r)::"memory");
    asm volatile("" : "+r"(r[30]), "+r"(r[31])::"memory");
}
SB_DEV void ld16(uint32_t addr, unsigned (&r)[16]) {  // and waits
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr)
        : "memory");
}
SB_DEV void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
SB_DEV void st16(uint32_t addr, const unsigned (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr), "r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
SB_DEV float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
SB_DEV unsigned long long add2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// Two powers of two on the FMA pipe, x <= 8: 2^x = 2^n 2^f, n = x rounded,
// |f| <= 1/2, 2^f as 1 + f q(f), q cubic with the least largest relative error
// (2.8e-6, 0.01 of a half step of the weights' type); n goes into the
// exponent.  At x <= -127 it is exactly 0.
SB_DEV void exp2_pair(unsigned long long x2, float &p0, float &p1) {
    float x0, x1;
    f2_unpack(x2, x0, x1);
    const unsigned long long x = f2_pack(fmaxf(x0, -127.f), fmaxf(x1, -127.f));
    constexpr float R = 12582912.f;  // 1.5 x 2^23: adding it rounds to a whole number in the low bits
    const unsigned long long t = add2(x, f2_pack(R, R)), f = add2(x, ffma2(t, f2_pack(-1.f, -1.f), f2_pack(R, R)));
    unsigned long long q = ffma2(f, f2_pack(0.009582852944731712f, 0.009582852944731712f), f2_pack(0.055906426161527634f, 0.055906426161527634f));
    q = ffma2(f, q, f2_pack(0.24024099111557007f, 0.24024099111557007f));
    q = ffma2(f, q, f2_pack(0.6931241750717163f, 0.6931241750717163f));
    q = ffma2(f, q, f2_pack(1.f, 1.f));
    float q0, q1, t0, t1;
    f2_unpack(q, q0, q1);
    f2_unpack(t, t0, t1);
    p0 = __uint_as_float(__float_as_uint(q0) + (__float_as_uint(t0) << 23));
    p1 = __uint_as_float(__float_as_uint(q1) + (__float_as_uint(t1) << 23));
}
// weights 2^(sc s - b) of 128 scores as 16-bit pairs over the scores' columns;
// returns their sum (two halves).  Every fourth pair leaves the exponential unit to the others.
template <typename T> SB_DEV unsigned long long weights(const unsigned (&r)[4][32], float sc, float b, uint32_t at) {
    const unsigned long long sc2 = f2_pack(sc, sc), b2 = f2_pack(-b, -b);
    unsigned long long sum[2] = {0ull, 0ull};
#pragma unroll
    for (int c = 0; c < 4; c++) {
        unsigned w[16];
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const unsigned long long x = ffma2(f2_pack(__uint_as_float(r[c][2 * i]), __uint_as_float(r[c][2 * i + 1])), sc2, b2);
            float p0, p1;
            if (i % ATC_POLY == ATC_POLY - 1) {
                exp2_pair(x, p0, p1);
            } else {
                f2_unpack(x, p0, p1);
                p0 = ap_exp2(p0);
                p1 = ap_exp2(p1);
            }
            sum[i & 1] = add2(sum[i & 1], f2_pack(p0, p1));
            w[i] = ap_pack<T>(p0, p1);
        }
        st16(at + c * 16, w);
    }
    return add2(sum[0], sum[1]);
}
}  // namespace atc

#define ATC_MORE asm volatile("setmaxnreg.inc.sync.aligned.u32 200;")
#define ATC_FEWER asm volatile("setmaxnreg.dec.sync.aligned.u32 56;")

template <typename T, int HDP>
SB_DEV void attn_tc_body(const AttnParams &P, const CUtensorMap *tm_k, const CUtensorMap *tm_v, int box) {
    using namespace atc;
    using C = Cfg<HDP>;
    constexpr int ST = C::ST, TILE = C::TILE;
    extern __shared__ unsigned char tc_sm_raw[];
    __shared__ uint64_t kfull[ST], kempty[ST], vfull[ST], vempty[ST], sfull[2], pfull[2], qfull, ofull;
    __shared__ uint32_t tmem_s;
    __shared__ __align__(16) uint32_t valid_s[2 * ST][4];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_launch_dependents();
    AttnItem it;
    if (!ap_prefix_item(P, blockIdx.x, 2 * BM, it)) return;
    const unsigned sm = (ap_smem(tc_sm_raw) + 1023u) & ~1023u;
    const unsigned vst = sm, kst = sm + ST * TILE, qst = sm + 2 * ST * TILE;  // stages of V and K, both query tiles
    const int nt = (it.k1 - it.k0 + KT - 1) / KT;
    const int nx = it.f0 + BM < it.F ? 2 : 1;  // row tiles with rows

    if (tid == 0) {
        for (int s = 0; s < ST; s++) {
            ap_bar_init(&kfull[s], 2);
            ap_bar_init(&vfull[s], 2);
            ap_bar_init(&kempty[s], 1);
            ap_bar_init(&vempty[s], 1);
        }
        for (int x = 0; x < 2; x++) {
            ap_bar_init(&sfull[x], 1);
            ap_bar_init(&pfull[x], 4);
        }
        ap_bar_init(&ofull, 1);
        ap_bar_init(&qfull, 4 * nx);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (tid == 32 * 8 && box) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(tm_k) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(tm_v) : "memory");
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(ap_smem(&tmem_s)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_s;
    // 512 threads x 128 registers = 256 x 200 + 256 x 56 (inside each role: the compiler goes by it)
    if (warp >= 8 && warp < 12) {
        ATC_FEWER;
        // ---- loaders: warps 8, 9 the keys, warps 10, 11 the values; each 64 positions of a tile.  A tile is
        // waited for right after its copies are issued: its stage came free a whole tile time before it is needed
        const bool is_k = warp < 10;
        const int p0 = (warp & 1) * 64;
        const T *base = static_cast<const T *>(is_k ? it.pg.k : it.pg.v) + it.kvh * it.pg.head_stride;
        const CUtensorMap *tm = is_k ? tm_k : tm_v;
        uint64_t *full = is_k ? kfull : vfull, *empty = is_k ? kempty : vempty;
        constexpr int CH = HDP / 8, RPI = 32 / CH;  // chunks of a row, rows an instruction
        const int c = lane % CH, rsub = lane / CH;
        const bool cok = c * 8 < P.HD;
        const T *col = base + c * 8;
        // TMA: lane i takes rows [box i, box i + box) of these 64 in column block i / pieces
        const int pieces = box ? 64 / box : 1, sub = lane / pieces, row = lane % pieces * box;
        const bool mine = box && sub < C::SUB;
        bool ok = true, any_tma = false;
        int t = 0, next = -1, in_next = 0;
        auto look = [&](int t) {  // a tile ahead of its use
            const int p = it.k0 + t * KT + p0;
            next = -1;
            if (mine && p + 64 <= it.k1) {
                const int j = ap_page(it.pg, p + row);
                next = it.table ? it.table[j] : j;
                in_next = p + row - j * it.pg.page;
            }
        };
        look(0);
        for (; t < nt; t++) {
            const int s = t % ST, key = it.k0 + t * KT + p0, page = next, in_page = in_next;
            look(t + 1);
            const bool by_tma = __all_sync(SB_FULL, box && (!mine || (page >= 0 && page < it.pg.n_pages)));
            if (t >= ST) ok = warp_wait(&empty[s], (unsigned)((t / ST) - 1) & 1u, P.call);
            if (is_k && t + 1 == P.test_skip) ok = false;
            if (!ok) break;
            const unsigned stage = (is_k ? kst : vst) + s * TILE;
            if (by_tma) {
                any_tma = true;
                if (lane == 0) {
                    if (is_k) *reinterpret_cast<uint2 *>(&valid_s[t % (2 * ST)][(warp & 1) * 2]) = make_uint2(~0u, ~0u);
                    ap_expect(&full[s], 64 * HDP * 2);
                }
                __syncwarp();
                if (mine) ap_tma(stage + sub * 16384 + (p0 + row) * 128, tm, sub * 64, it.kvh, in_page, page, &full[s]);
                continue;
            }
#pragma unroll 1
            for (int h = 0; h < 2; h++) {
                const long long off = ap_offset(it, key + h * 32 + lane);
                if (is_k) {
                    const unsigned valid = __ballot_sync(SB_FULL, off & 1);
                    if (lane == 0) valid_s[t % (2 * ST)][(warp & 1) * 2 + h] = valid;
                }
#pragma unroll 4
                for (int i = 0; i < CH; i++) {
                    const int r = i * RPI + rsub;
                    const long long o = __shfl_sync(SB_FULL, off, r);
                    const bool there = (o & 1) && cok;
                    ap_cp16(stage + (c >> 3) * 16384 + (p0 + h * 32 + r) * 128 + (((c & 7) ^ (r & 7)) << 4), col + (o & ~1ll), there);
                }
            }
            ap_commit();
            ap_wait<0>();
            ap_fence_async();
            __syncwarp();
            if (lane == 0) ap_arrive(&full[s]);
        }
        ap_wait<0>();
        if (!ok && any_tma)  // given up: the copies that were issued still have to land
            for (int i = t > ST ? t - ST : 0; i < t; i++) ap_bar_wait(&full[i % ST], (i / ST) & 1, 0);
    } else if (warp >= 12) {
        ATC_FEWER;
        if (tid == 12 * 32) {
            // ---- issuer.  One for both tiles: it keeps their phases apart (with an issuer each they fell into step,
            // both in their softmax, then both on the tensor pipe)
            const uint32_t id_s = idesc<T>(KT, false), id_o = idesc<T>(HDP, true);
            const uint64_t qd = desc(qst), kd = desc(kst), vd = desc(vst);
            auto scores = [&](int x, int s) {
                const uint64_t qs = qd + x * (TILE >> 4), ks = kd + s * (TILE >> 4);
#pragma unroll
                for (int k = 0; k < HDP / 16; k++) {
                    const uint32_t in = (k >> 2) * 1024 + 2 * (k & 3);
                    mma_ss(tmem + x * 128, qs + in, ks + in, id_s, k > 0);
                }
                commit(&sfull[x]);
            };
            bool ok = nt > 0 && ap_bar_wait(&qfull, 0, P.call) && ap_bar_wait(&kfull[0], 0, P.call);
            if (ok) {
                fence_after();
                for (int x = 0; x < nx; x++) scores(x, 0);
                commit(&kempty[0]);
            }
            int s = 0;
            unsigned ph = 0;
            for (int t = 0; t < nt && ok; t++) {
                const int s1 = s + 1 == ST ? 0 : s + 1;
                const unsigned ph1 = s1 ? ph : ph ^ 1;
                const bool more = t + 1 < nt;
                ok = ap_bar_wait(&vfull[s], ph, P.call) && (!more || ap_bar_wait(&kfull[s1], ph1, P.call));
#pragma unroll 1
                for (int x = 0; x < nx && ok; x++) {
                    ok = ap_bar_wait(&pfull[x], t & 1, P.call);
                    if (!ok) break;
                    fence_after();
                    const uint64_t vs = vd + s * (TILE >> 4);
#pragma unroll
                    for (int k = 0; k < KT / 16; k++)
                        mma_ts(tmem + 256 + x * 128, tmem + x * 128 + k * 8, vs + k * 128, id_o, t > 0 || k > 0);
                    if (more) scores(x, s1);
                }
                commit(&vempty[s]);
                if (more) commit(&kempty[s1]);
                s = s1;
                ph = ph1;
            }
            commit(&ofull);  // when everything issued above has completed, also after giving up
        }
        __syncwarp();
    } else if ((warp >> 2) < nx) {
        ATC_MORE;
        // ---- softmax and epilogue: a thread a row
        const int x = warp >> 2, f = it.f0 + tid;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, s_at = tmem + lanes + x * 128, o_at = tmem + lanes + 256 + x * 128;
        const float sc = fmaxf(fabsf(P.scale_log2), 1e-30f);  // 0 times a masked score would be NaN
        {  // this warp's 32 query rows, neighbouring lanes on one row, zeros behind the last.  A short loop: code that
           // runs once costs six cycles an instruction to fetch
            constexpr int CH = HDP / 8, RPI = 32 / CH;
            const int c = lane % CH, qr = f / P.G;
            const long long at = f < it.F ? ((long long)(it.row0 + qr) * P.q_row + (it.kvh * P.G + f - qr * P.G) * P.q_head) | 1 : 0;
            const T *col = static_cast<const T *>(P.q) + c * 8;
            const unsigned dst = qst + x * TILE + (c >> 3) * 16384 + (warp & 3) * 4096;
#pragma unroll 1
            for (int i = 0; i < CH; i++) {
                const int r = i * RPI + lane / CH;
                const long long o = __shfl_sync(SB_FULL, at, r);
                ap_cp16(dst + r * 128 + (((c & 7) ^ (r & 7)) << 4), col + (o & ~1ll), (o & 1) && c * 8 < P.HD);
            }
            ap_commit();
            ap_wait<0>();
            __syncwarp();
            if (P.scale_log2 < 0.f) {  // maxima are taken of the scores: a negative scale turns the queries round
#pragma unroll 1
                for (int i = 0; i < HDP / 2; i++) {  // this lane's row: 32 x 4 bytes of each column block
                    const unsigned a = qst + x * TILE + (i >> 5) * 16384 + (warp & 3) * 4096 + lane * 128 + (i & 31) * 4;
                    unsigned v;
                    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
                    asm volatile("st.shared.b32 [%0], %1;" ::"r"(a), "r"(v ^ 0x80008000u) : "memory");
                }
            }
            ap_fence_async();
            __syncwarp();
            if (lane == 0) ap_arrive(&qfull);
        }
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        for (int t = 0; t < nt && ok; t++) {
            ok = warp_wait(&sfull[x], t & 1, P.call);
            if (!ok) break;
            fence_after();
            const uint4 valid = *reinterpret_cast<const uint4 *>(valid_s[t % (2 * ST)]);
            unsigned r[4][32];
#pragma unroll
            for (int c = 0; c < 4; c++) ld32(s_at + c * 32, r[c]);
#pragma unroll
            for (int c = 0; c < 4; c++) wait_ld(r[c]);
            if ((valid.x & valid.y & valid.z & valid.w) != 0xffffffffu) {  // the end of the range, or a page that is not there
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const unsigned bits = c == 0 ? valid.x : c == 1 ? valid.y : c == 2 ? valid.z : valid.w;
#pragma unroll
                    for (int i = 0; i < 32; i++)
                        if (!(bits >> i & 1)) r[c][i] = 0xff800000u;
                }
            }
            float mx4[4];
#pragma unroll
            for (int c = 0; c < 4; c++) {
                mx4[c] = max_nan(__uint_as_float(r[c][0]), __uint_as_float(r[c][1]));
#pragma unroll
                for (int i = 2; i < 32; i += 2) mx4[c] = max_nan(max_nan(mx4[c], __uint_as_float(r[c][i])), __uint_as_float(r[c][i + 1]));
            }
            const float mx = max_nan(max_nan(mx4[0], mx4[1]), max_nan(mx4[2], mx4[3])) * sc;
            if (t == 0) m = mx;
            // the weights are taken against the maximum so far, beside the search for the new one; where that has
            // grown too far (or a NaN turns up) they are taken again.  sc s - m is one fma with a rounded m: from 2^24 on
            // that is off by 1/2 and more, as the FP32 scores are, and from 2^31 on it passes FP32 as a power of two.
            // There the scores are rounded first, as m was
            unsigned long long l2;
            float by = sc;
            for (;;) {
                l2 = weights<T>(r, by, m == -INFINITY ? 0.f : m, s_at);
                if (!__any_sync(SB_FULL, mx > m + 8.f || (fabsf(mx) >= 16777216.f && by != 1.f) || (mx != mx && m == m))) break;
                if (by != 1.f && __any_sync(SB_FULL, fabsf(mx) >= 16777216.f)) {
#pragma unroll
                    for (int c = 0; c < 4; c++)
#pragma unroll
                        for (int i = 0; i < 32; i++) r[c][i] = __float_as_uint(__fmul_rn(__uint_as_float(r[c][i]), sc));
                    by = 1.f;
                }
                const float to = max_nan(m, mx), a = m == to ? 1.f : ap_exp2(m - to);
                m = to;
                l *= a;
                wait_st();
#pragma unroll 1
                for (int c = 0; c < HDP / 16; c++) {  // S(t) is complete, so PV(t - 1) is
                    unsigned w[16];
                    ld16(o_at + c * 16, w);
#pragma unroll
                    for (int i = 0; i < 16; i++) w[i] = __float_as_uint(__uint_as_float(w[i]) * a);
                    st16(o_at + c * 16, w);
                }
            }
            l += f2_sum(l2);
            wait_st();
            fence_before();
            __syncwarp();
            if (lane == 0) ap_arrive(&pfull[x]);
        }
        if (m == INFINITY) l = __int_as_float(0x7fc00000);  // an infinite score: NaN, as its softmax
        ok = __all_sync(SB_FULL, ap_bar_wait(&ofull, 0, 0) && ok && *(volatile unsigned *)&tc_call != P.call);
        fence_after();
        if (!ok) l = __int_as_float(0x7fc00000);  // given up: nothing that passes for a result
        const bool live = f < it.F;
        if (live) ap_row_stats(P, it, f, m, l);
        const int qrow = it.row0 + f / P.G, head = it.kvh * P.G + f % P.G;
        const bool whole = P.S1 + P.S2 == 1;  // the result itself, else this range's part of it
        const float inv = whole ? (l == 0.f ? 0.f : 1.f / l) : 1.f;
        float *po = P.ws_o + (((long long)it.slot * P.T + qrow) * P.NH + head) * P.HD;
        T *out = static_cast<T *>(P.out) + qrow * P.o_row + head * P.o_head;
#pragma unroll 1
        for (int c = 0; c < HDP / 32; c++) {
            unsigned r[32];
            ld32(o_at + c * 32, r);
            wait_ld(r);
            if (!live) continue;
#pragma unroll
            for (int i = 0; i < 32; i += 8) {  // 32-byte stores (a lane a row: full sectors)
                if (c * 32 + i >= P.HD) break;
                if (whole) {
                    unsigned w[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) w[e] = ap_pack<T>(__uint_as_float(r[i + 2 * e]) * inv, __uint_as_float(r[i + 2 * e + 1]) * inv);
                    *reinterpret_cast<uint4 *>(out + c * 32 + i) = make_uint4(w[0], w[1], w[2], w[3]);
                } else if (l != 0.f) {
                    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(po + c * 32 + i), "r"(r[i]), "r"(r[i + 1]),
                                 "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])
                                 : "memory");
                }
            }
        }
    }
    fence_before();
    __syncthreads();
    if (warp == 12) {
        fence_after();
        ap_bar_wait(&ofull, 0, 0);
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}
#define ATC_KERNEL(name, T, HDP)                                                                                                     \
    extern "C" __global__ void __launch_bounds__(atc::THREADS, 1)                                                                       \
        name(const __grid_constant__ AttnParams P, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,  \
             int box) {                                                                                                                 \
        attn_tc_body<T, HDP>(P, &tm_k, &tm_v, box);                                                                                     \
        if (blockIdx.x == gridDim.x - 1) pdl_wait();                                                                                    \
    }
ATC_KERNEL(attn_tc_f16_64, __half, 64)
ATC_KERNEL(attn_tc_f16_128, __half, 128)
ATC_KERNEL(attn_tc_bf16_64, __nv_bfloat16, 64)
ATC_KERNEL(attn_tc_bf16_128, __nv_bfloat16, 128)
