// score_kernels.cu -- the "score" module image (sm_100a cubin): log
// probabilities of given tokens with entropy, rank and the best
// alternatives, from one pass over the logits, and their gradient.  No
// counterpart in the reference, which samples one token a step.
//
// With y = x log2(e) / temperature of a row and m its maximum,
//   s = sum 2^(y - m),  t = sum 2^(y - m) (y - m)
//   lse = ln2 (m + log2 s),  logp = ln2 (y_tok - m - log2 s)
//   entropy = ln2 (log2 s - t / s)
// and a change of m turns (s, t) into f s, f (t + s (m - m')), f = 2^(m - m'):
// a thread keeps (m, s, t) of its values and looks at m once per vector.
// y - m is one fma with m's own rounded product, so the rounding of m is the
// same in every term and cancels.  Sums are FP32.
//
// Bound: HBM (one read of the logits); for 16-bit logits the 16 exponentials
// per SM and cycle are close behind (5.5 against 4.2 us for 10^7 values).
//
// The k best in the same pass.  A key is the value's order-preserving bits
// above the complemented id, so a larger key is a better candidate and equal
// values go to the lower id (-0 counts as +0); masked choices (-inf) are not
// listed.  The k-th best of the
// threads' (or thread groups') maxima so far is a lower bound of the k-th
// best value: k holders each have a value at least that good.  Only values
// that reach it go to a list in shared memory -- about k per doubling of the
// values seen, as the bound is renewed after tiles 0, 1, 3, 7, ...  A list
// that would overflow (rising or equal logits) is cut to its k best first.
#include <cfloat>
#include <cuda_bf16.h>

#include "sb_common.cuh"

#define LP_THREADS 256
#define LP_U 4        // vectors of a thread per tile
#define LP_LIST 1024  // keys
#define LP_KMAX 64
#define LP_LN2 0.6931471805599453f

// parameter block, mirrored by the host (host/sb_serve.c)
struct LpParams {
    const void *x;
    long long stride;  // elements
    int R, V, S, k;    // S parts per row, one CTA each
    float c;           // log2(e) / temperature
    const int *tok;
    float *logp, *entropy, *lse;
    int *rank, *top_ids;
    float *top_logp;
    float4 *part;                // [R][S]: m, s, t, rank count (bits)
    unsigned long long *keys;    // [R][S][k]
};

template <typename T> struct LpVec { static constexpr int N = 16 / sizeof(T); };
SB_DEV float lp_f(float v) { return v; }
SB_DEV float lp_f(__half v) { return __half2float(v); }
SB_DEV float lp_f(__nv_bfloat16 v) { return __bfloat162float(v); }
SB_DEV float lp_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
SB_DEV float lp_max_nan(float a, float b) {  // a NaN stays: the row's results become NaN
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
// y - m; -inf logits (and m = -inf) become a power of two that is 0
SB_DEV float lp_diff(float x, float c, float mc) { return fmaxf(fmaf(x, c, -mc), -200.f); }
SB_DEV unsigned long long lp_key(float v, int id) {
    const unsigned u = __float_as_uint(v == 0.f ? 0.f : v);
    return ((unsigned long long)((u & 0x80000000u) ? ~u : (u | 0x80000000u)) << 32) | (unsigned)~id;
}
SB_DEV float lp_key_value(unsigned long long k) {
    const unsigned u = (unsigned)(k >> 32);
    return __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u);
}
SB_DEV int lp_key_id(unsigned long long k) { return (int)~(unsigned)k; }

struct LpSum { float m, s, t; };
SB_DEV void lp_raise(LpSum &a, float m) {  // m >= a.m
    if (a.s != 0.f) {
        const float d = fmaxf(a.m - m, -200.f), f = lp_exp2(d);
        a.t = f * fmaf(a.s, d, a.t);
        a.s *= f;
    }
    a.m = m;
}
SB_DEV LpSum lp_join(LpSum a, LpSum b) {
    const float m = lp_max_nan(a.m, b.m);
    lp_raise(a, m);
    lp_raise(b, m);
    return {m, a.s + b.s, a.t + b.t};
}
SB_DEV LpSum lp_warp(LpSum a) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const LpSum b = {__shfl_xor_sync(SB_FULL, a.m, o), __shfl_xor_sync(SB_FULL, a.s, o), __shfl_xor_sync(SB_FULL, a.t, o)};
        a = lp_join(a, b);
    }
    return a;
}

// the first k of n keys in a list, ranked by counting, as emit(rank, key)
template <int THREADS, typename F>
SB_DEV void lp_rank(const unsigned long long *list, int n, int k, F emit) {
    for (int i = threadIdx.x; i < n; i += THREADS) {
        const unsigned long long me = list[i];
        int r = 0;
        for (int j = 0; j < n; j++) r += list[j] > me;
        if (r < k) emit(r, me);
    }
}
// the list cut to its k best (in any case to at most k); returns how many
template <int THREADS>
SB_DEV int lp_cut(unsigned long long *list, int n, int k) {
    unsigned long long mine[(LP_LIST + THREADS - 1) / THREADS];
    int rank[(LP_LIST + THREADS - 1) / THREADS];
#pragma unroll
    for (int q = 0; q < (LP_LIST + THREADS - 1) / THREADS; q++) {
        const int i = threadIdx.x + q * THREADS;
        mine[q] = i < n ? list[i] : 0ull;
        rank[q] = 0;
        if (i < n)
            for (int j = 0; j < n; j++) rank[q] += list[j] > mine[q];
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < (LP_LIST + THREADS - 1) / THREADS; q++)
        if ((int)threadIdx.x + q * THREADS < n && rank[q] < k) list[rank[q]] = mine[q];
    __syncthreads();
    return min(n, k);
}

// results of a row from its joined sums
SB_DEV void lp_finish(const LpParams &P, int r, LpSum a, int above, float xt, bool given) {
    const bool none = a.m == -INFINITY;  // every choice is masked
    const float l2 = log2f(a.s);
    if (P.lse) P.lse[r] = none ? -INFINITY : (a.m + l2) * LP_LN2;
    if (P.entropy) P.entropy[r] = none ? 0.f : (l2 - a.t / a.s) * LP_LN2;
    if (P.logp) P.logp[r] = !given ? 0.f : none ? -INFINITY : (fmaf(xt, P.c, -a.m) - l2) * LP_LN2;
    if (P.rank) P.rank[r] = given ? above : -1;
}
SB_DEV void lp_top(const LpParams &P, int r, int i, unsigned long long key, float m, float l2) {
    const bool ok = key != 0ull;
    if (P.top_ids) P.top_ids[(long long)r * P.k + i] = ok ? lp_key_id(key) : -1;
    if (P.top_logp)
        P.top_logp[(long long)r * P.k + i] = !ok || m == -INFINITY ? -INFINITY : (fmaf(lp_key_value(key), P.c, -m) - l2) * LP_LN2;
}

// CTA = part s of row r: vectors [n s / S, n (s + 1) / S) of the row, counted
// from the 16-byte boundary at or below its start (the partial first and
// last vectors are read value by value).
template <typename T, bool TOP>
SB_DEV void logprobs_body(const LpParams &P) {
    constexpr int N = LpVec<T>::N;
    __shared__ LpSum sum_s[LP_THREADS / 32];
    __shared__ int cnt_s[LP_THREADS / 32];
    __shared__ unsigned long long list[TOP ? LP_LIST : 1];
    __shared__ __align__(16) float best_s[TOP ? LP_THREADS : 4];
    __shared__ int n_s;
    __shared__ float thr_s;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int r = blockIdx.x / P.S, part = blockIdx.x % P.S;
    pdl_launch_dependents();
    const T *x = static_cast<const T *>(P.x) + r * P.stride;
    const int lead = (int)(((uintptr_t)x & 15) / sizeof(T));  // values of the first vector that are not the row's
    const T *x0 = x - lead;
    const int nv = (int)(((long long)lead + P.V + N - 1) / N);
    const int v0 = (int)((long long)nv * part / P.S), v1 = (int)((long long)nv * (part + 1) / P.S);
    const int tok = P.tok ? P.tok[r] : -1;
    const bool given = tok >= 0 && tok < P.V;
    const float xt = given ? lp_f(x[tok]) : 0.f;
    const bool count = P.rank && given;

    LpSum a = {-INFINITY, 0.f, 0.f};
    float best = -INFINITY;  // this thread's best raw value
    int above = 0;
    float thr = -FLT_MAX;  // masked choices (-inf) are never listed
    unsigned long long cut = 0ull;  // keys at or below it are out
    if (TOP && tid == 0) n_s = 0;
    const int groups = P.k > 24 ? LP_THREADS : LP_THREADS / 4;
    int renew = 0, tile = 0, held = 0;  // held: keys in the list

    // the k-th best group maximum bounds the k-th best value from below
    auto raise_bound = [&]() {
        float g = best;
        if (groups != LP_THREADS) {
            g = fmaxf(g, __shfl_xor_sync(SB_FULL, g, 1));
            g = fmaxf(g, __shfl_xor_sync(SB_FULL, g, 2));
        }
        const bool lead_lane = groups == LP_THREADS || (tid & 3) == 0;
        const int gi = groups == LP_THREADS ? tid : tid >> 2;
        if (lead_lane) best_s[gi] = g;
        if (tid == 0) thr_s = -FLT_MAX;
        __syncthreads();
        if (lead_lane) {
            int rk = 0;
            for (int i = 0; i < groups; i += 4) {
                const float4 o = *reinterpret_cast<const float4 *>(best_s + i);
                rk += (o.x > g || (o.x == g && i < gi)) + (o.y > g || (o.y == g && i + 1 < gi)) +
                      (o.z > g || (o.z == g && i + 2 < gi)) + (o.w > g || (o.w == g && i + 3 < gi));
            }
            if (rk == P.k - 1) thr_s = g;
        }
        __syncthreads();
        thr = fmaxf(thr, thr_s);
    };

    for (int b = v0; b < v1; b += LP_THREADS * LP_U, tile++) {
        float v[LP_U][N];
        uint4 raw[LP_U];
#pragma unroll
        for (int u = 0; u < LP_U; u++) {
            const int j = b + u * LP_THREADS + tid;
            const int e0 = j * N - lead;
            if (j < v1 && e0 >= 0 && e0 + N <= P.V) raw[u] = ld_stream_u4(x0 + (long long)j * N);
        }
        float mx = -INFINITY;
#pragma unroll
        for (int u = 0; u < LP_U; u++) {
            const int j = b + u * LP_THREADS + tid;
            const int e0 = j * N - lead;
            if (j < v1 && e0 >= 0 && e0 + N <= P.V) {
                const T *h = reinterpret_cast<const T *>(&raw[u]);
#pragma unroll
                for (int e = 0; e < N; e++) v[u][e] = lp_f(h[e]);
            } else {
#pragma unroll
                for (int e = 0; e < N; e++) v[u][e] = j < v1 && e0 + e >= 0 && e0 + e < P.V ? lp_f(x[e0 + e]) : -INFINITY;
            }
#pragma unroll
            for (int e = 0; e < N; e++) mx = lp_max_nan(mx, v[u][e]);
        }
        best = lp_max_nan(best, mx);
        if (best * P.c > a.m || best != best) lp_raise(a, best * P.c);
#pragma unroll
        for (int u = 0; u < LP_U; u++)
#pragma unroll
            for (int e = 0; e < N; e++) {
                const float d = lp_diff(v[u][e], P.c, a.m), w = lp_exp2(d);
                a.s += w;
                a.t = fmaf(w, d, a.t);
            }
        if (count) {
#pragma unroll
            for (int u = 0; u < LP_U; u++) {
                const int j = b + u * LP_THREADS + tid, e0 = j * N - lead;
#pragma unroll
                for (int e = 0; e < N; e++)
                    above += v[u][e] > xt || (v[u][e] == xt && e0 + e < tok && e0 + e >= 0 && j < v1);
            }
        }
        if constexpr (TOP) {
            if (tile == renew) {
                renew = 2 * renew + 1;
                raise_bound();
            }
            int pass = 0;
            if (mx >= thr) {
#pragma unroll
                for (int u = 0; u < LP_U; u++) {
                    const int j = b + u * LP_THREADS + tid, e0 = j * N - lead;
#pragma unroll
                    for (int e = 0; e < N; e++)
                        pass += v[u][e] >= thr && j < v1 && e0 + e >= 0 && e0 + e < P.V && lp_key(v[u][e], e0 + e) > cut;
                }
            }
            if (__syncthreads_or(pass)) {
                int at = pass ? atomicAdd(&n_s, pass) : 0;
                __syncthreads();
                const int n = n_s;
                if (n <= LP_LIST) {
                    held = n;
                    if (pass) {
#pragma unroll
                        for (int u = 0; u < LP_U; u++) {
                            const int j = b + u * LP_THREADS + tid, e0 = j * N - lead;
#pragma unroll
                            for (int e = 0; e < N; e++) {
                                const unsigned long long key = lp_key(v[u][e], e0 + e);
                                if (v[u][e] >= thr && j < v1 && e0 + e >= 0 && e0 + e < P.V && key > cut) list[at++] = key;
                            }
                        }
                    }
                    __syncthreads();
                } else {  // too many at once: value by value, the list cut to its k best whenever 256 more might not fit
                    int have = held;
                    __syncthreads();  // n_s is read
#pragma unroll 1
                    for (int u = 0; u < LP_U; u++)
#pragma unroll 1
                        for (int e = 0; e < N; e++) {
                            if (have + LP_THREADS > LP_LIST) {
                                have = lp_cut<LP_THREADS>(list, have, P.k);
                                if (have == P.k) cut = max(cut, list[P.k - 1]);
                            }
                            if (tid == 0) n_s = have;
                            __syncthreads();
                            const int j = b + u * LP_THREADS + tid, id = j * N - lead + e;
                            if (j < v1 && id >= 0 && id < P.V) {
                                const float w = lp_f(x[id]);
                                const unsigned long long key = lp_key(w, id);
                                if (w >= thr && key > cut) list[atomicAdd(&n_s, 1)] = key;
                            }
                            __syncthreads();
                            have = n_s;
                            __syncthreads();
                        }
                    held = have;
                }
            }
        }
    }
    // join over the block
    a = lp_warp(a);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) above += __shfl_xor_sync(SB_FULL, above, o);
    if (lane == 0) {
        sum_s[warp] = a;
        cnt_s[warp] = above;
    }
    __syncthreads();
    a = sum_s[0];
    above = cnt_s[0];
#pragma unroll
    for (int w = 1; w < LP_THREADS / 32; w++) {
        a = lp_join(a, sum_s[w]);
        above += cnt_s[w];
    }
    if (tid == 0) {
        if (P.S == 1) lp_finish(P, r, a, above, xt, given);
        else P.part[(long long)r * P.S + part] = make_float4(a.m, a.s, a.t, __int_as_float(above));
    }
    if constexpr (TOP) {
        // what the final bound leaves of the list, ranked
        raise_bound();
        unsigned long long mine[LP_LIST / LP_THREADS];
#pragma unroll
        for (int q = 0; q < LP_LIST / LP_THREADS; q++) {
            const int i = tid + q * LP_THREADS;
            mine[q] = i < held ? list[i] : 0ull;
        }
        __syncthreads();
        if (tid == 0) n_s = 0;
        __syncthreads();
#pragma unroll
        for (int q = 0; q < LP_LIST / LP_THREADS; q++)
            if (mine[q] && lp_key_value(mine[q]) >= thr) list[atomicAdd(&n_s, 1)] = mine[q];
        __syncthreads();
        const int n = n_s;
        const float l2 = log2f(a.s);
        unsigned long long *out = P.keys + ((long long)r * P.S + part) * P.k;
        lp_rank<LP_THREADS>(list, n, P.k, [&](int i, unsigned long long key) {
            if (P.S == 1) lp_top(P, r, i, key, a.m, l2);
            else out[i] = key;
        });
        for (int i = n + tid; i < P.k; i += LP_THREADS) {
            if (P.S == 1) lp_top(P, r, i, 0ull, a.m, l2);
            else out[i] = 0ull;
        }
    }
}
#define LP_KERNEL(name, T, TOP) \
    extern "C" __global__ void __launch_bounds__(LP_THREADS) name(const __grid_constant__ LpParams P) { logprobs_body<T, TOP>(P); }
LP_KERNEL(logprobs_f32, float, false)
LP_KERNEL(logprobs_f16, __half, false)
LP_KERNEL(logprobs_bf16, __nv_bfloat16, false)
LP_KERNEL(logprobs_top_f32, float, true)
LP_KERNEL(logprobs_top_f16, __half, true)
LP_KERNEL(logprobs_top_bf16, __nv_bfloat16, true)

// A CTA a row: the parts' sums, and the k best of their S sorted lists.  The
// k-th best list head bounds the k-th best key from below, so at most k
// lists matter and k x k keys are kept.
// type: 0 f32, 1 f16, 2 bf16.
extern "C" __global__ void __launch_bounds__(LP_THREADS) logprobs_join(const __grid_constant__ LpParams P, int type) {
    __shared__ LpSum sum_s[LP_THREADS / 32];
    __shared__ int cnt_s[LP_THREADS / 32];
    __shared__ unsigned long long list[LP_KMAX * LP_KMAX];
    __shared__ unsigned long long bound_s;
    __shared__ int n_s;
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = blockIdx.x;
    LpSum a = {-INFINITY, 0.f, 0.f};
    int above = 0;
    for (int s = tid; s < P.S; s += LP_THREADS) {
        const float4 p = P.part[(long long)r * P.S + s];
        a = lp_join(a, {p.x, p.y, p.z});
        above += __float_as_int(p.w);
    }
    if (tid == 0) {
        n_s = 0;
        bound_s = 0ull;
    }
    a = lp_warp(a);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) above += __shfl_xor_sync(SB_FULL, above, o);
    if (lane == 0) {
        sum_s[warp] = a;
        cnt_s[warp] = above;
    }
    __syncthreads();
    a = sum_s[0];
    above = cnt_s[0];
#pragma unroll
    for (int w = 1; w < LP_THREADS / 32; w++) {
        a = lp_join(a, sum_s[w]);
        above += cnt_s[w];
    }
    const int tok = P.tok ? P.tok[r] : -1;
    const bool given = tok >= 0 && tok < P.V;
    if (tid == 0) {
        float xt = 0.f;
        if (given) {
            const long long at = r * P.stride + tok;
            xt = type == 0 ? static_cast<const float *>(P.x)[at]
                           : type == 1 ? lp_f(static_cast<const __half *>(P.x)[at]) : lp_f(static_cast<const __nv_bfloat16 *>(P.x)[at]);
        }
        lp_finish(P, r, a, above, xt, given);
    }
    if (P.k == 0) return;
    const unsigned long long *keys = P.keys + (long long)r * P.S * P.k;
    if (P.S >= P.k)
        for (int s = tid; s < P.S; s += LP_THREADS) {
            const unsigned long long me = keys[(long long)s * P.k];
            int rk = 0;
            for (int j = 0; j < P.S; j++) {
                const unsigned long long o = keys[(long long)j * P.k];
                rk += o > me || (o == me && j < s);
            }
            if (rk == P.k - 1) bound_s = me;
        }
    __syncthreads();
    const unsigned long long bound = bound_s;
    for (int i = tid; i < P.S * P.k; i += LP_THREADS) {
        const unsigned long long key = keys[i];
        if (key && key >= bound) list[atomicAdd(&n_s, 1)] = key;
    }
    __syncthreads();
    const int n = n_s;
    const float l2 = log2f(a.s);
    lp_rank<LP_THREADS>(list, n, P.k, [&](int i, unsigned long long key) { lp_top(P, r, i, key, a.m, l2); });
    for (int i = n + tid; i < P.k; i += LP_THREADS) lp_top(P, r, i, 0ull, a.m, l2);
}

// ---------------------------------------------------------------- gradient
// d logits[v] = (g_logp (1[v = tok] - p_v) - g_entropy p_v (ln p_v + H)) / temperature,
// p_v = e^(x_v - lse).  Bound: HBM, one read and one write.  lse log2(e) is
// held as two floats: its rounding alone would be 1e-6 of every p.
struct LpGradParams {
    const void *x;
    void *dx;
    long long stride, dstride;
    int R, V, S;
    float c, inv_temp;
    const int *tok;
    const float *lse, *entropy, *g_logp, *g_entropy;
};
template <typename T> SB_DEV T lp_to(float v);
template <> SB_DEV float lp_to<float>(float v) { return v; }
template <> SB_DEV __half lp_to<__half>(float v) { return __float2half_rn(v); }
template <> SB_DEV __nv_bfloat16 lp_to<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T>
SB_DEV void logprobs_grad_body(const LpGradParams &P) {
    constexpr int N = LpVec<T>::N;
    const int r = blockIdx.x / P.S, part = blockIdx.x % P.S, tid = threadIdx.x;
    const T *x = static_cast<const T *>(P.x) + r * P.stride;
    T *dx = static_cast<T *>(P.dx) + r * P.dstride;
    const int lead = (int)(((uintptr_t)x & 15) / sizeof(T));
    const bool same = (((uintptr_t)x ^ (uintptr_t)dx) & 15) == 0;  // else the vectors of dx would straddle
    const int nv = (int)(((long long)lead + P.V + N - 1) / N);
    const int v0 = (int)((long long)nv * part / P.S), v1 = (int)((long long)nv * (part + 1) / P.S);
    const int tok = P.tok ? P.tok[r] : -1;
    const bool given = tok >= 0 && tok < P.V;
    const float lse = P.lse[r], H = P.g_entropy ? P.entropy[r] : 0.f;
    const float gl = given && P.g_logp ? P.g_logp[r] * P.inv_temp : 0.f, ge = P.g_entropy ? P.g_entropy[r] * P.inv_temp : 0.f;
    const bool none = lse == -INFINITY;
    constexpr float L2E = 1.4426950408889634f, L2E_LO = 1.925963033500e-08f;
    const float hi = none ? 0.f : lse * L2E, lo = none ? 0.f : fmaf(lse, L2E, -hi) + lse * L2E_LO;
    const float a0 = gl + ge * H, a1 = ge * LP_LN2;  // dx = -p (a0 + a1 d), d = log2 p
    auto grad = [&](float v, int id) {
        const float d = fmaxf(fmaf(v, P.c, -hi) - lo, -200.f);
        const float p = none ? 0.f : lp_exp2(d);
        const float g = -p * fmaf(a1, d, a0);
        return id == tok && !none ? g + gl : g;
    };
    for (int b = v0; b < v1; b += LP_THREADS * LP_U) {
        uint4 raw[LP_U];
#pragma unroll
        for (int u = 0; u < LP_U; u++) {
            const int j = b + u * LP_THREADS + tid, e0 = j * N - lead;
            if (same && j < v1 && e0 >= 0 && e0 + N <= P.V) raw[u] = *reinterpret_cast<const uint4 *>(x + e0);
        }
#pragma unroll
        for (int u = 0; u < LP_U; u++) {
            const int j = b + u * LP_THREADS + tid, e0 = j * N - lead;
            if (j >= v1) break;
            if (same && e0 >= 0 && e0 + N <= P.V) {
                const T *h = reinterpret_cast<const T *>(&raw[u]);
                uint4 o;
                T *w = reinterpret_cast<T *>(&o);
#pragma unroll
                for (int e = 0; e < N; e++) w[e] = lp_to<T>(grad(lp_f(h[e]), e0 + e));
                *reinterpret_cast<uint4 *>(dx + e0) = o;
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
