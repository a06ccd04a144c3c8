// serve_rotary.cuh -- rotary positions of query and key rows at a position
// per row, with the key / value write into paged memory.
//
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t),  t = pos * f_i
//
// for pair i of the first `dim` values of a head: (i, i + dim / 2) in the
// half layout, (2 i, 2 i + 1) in the pair layout; the rest of the head is
// copied.  The inverse turns by -t: the gradient of the rotation.
//
// The angle at a far position needs more bits than FP32 has (pos 10^6 x f 1
// leaves 0.06 rad of error), and tables cost reads and a length limit.  So a
// frequency is held as a 64-bit fixed-point fraction of a turn, F = f / 2 pi
// x 2^64: pos * F modulo 2^64 is the fraction of the last turn from one integer
// multiply, off by pos times what F is off (the host's powl: 2^-62 of f / 2 pi,
// and half a unit of 2^-64).  Its top 32 bits as a signed fraction, rounded to
// FP32, give the angle within +-pi to 2^-25 of a half turn, and sincospif takes
// it from there.  All frequencies are a kernel parameter
// (1 KB): no table in memory.
//
// Bound: HBM, one read and one write of the rows.  A CTA takes a few tokens,
// computes their cosines and sines once into shared memory for all heads,
// and streams the rows as two 16-byte vectors of a thread: values
// [u V, u V + V) of both halves of what is turned, or of the head (pairs,
// values), so that neighbouring threads touch neighbouring vectors (16000
// tokens, 32 heads of 128 turned as pairs, BF16: 49 us, 2 V neighbours a thread
// 62; with a second unit's loads in flight, at a third fewer CTAs, 58).
// VEC = 1 serves rows whose strides, sizes or addresses are not multiples of
// 16 bytes.
#pragma once
#include <cuda_bf16.h>

#include "sb_common.cuh"

#define SB_ROT_THREADS 256
#define SB_ROT_MAX_TOK 4

// parameter block, mirrored by the host (host/sb_serve.c)
struct RotParams {
    const void *src[3];    // query, key, value rows (null: absent)
    void *dst[3];          // rotated query rows; key / value pages
    long long st[3], sh[3];   // source strides in elements: token, head
    long long dt, dh;         // query destination strides: token, head
    long long page_stride, pos_stride, head_stride;  // pages
    const int *pos;
    const long long *slots;
    long long n_slots;
    int T, heads[3], HD, dim, layout, inverse, page, tokens_per_cta;
    float mscale;
    unsigned long long turn[128];
};

template <typename T> SB_DEV float rot_f(T v);
template <> SB_DEV float rot_f<float>(float v) { return v; }
template <> SB_DEV float rot_f<__half>(__half v) { return __half2float(v); }
template <> SB_DEV float rot_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> SB_DEV T rot_t(float v);
template <> SB_DEV float rot_t<float>(float v) { return v; }
template <> SB_DEV __half rot_t<__half>(float v) { return __float2half_rn(v); }
template <> SB_DEV __nv_bfloat16 rot_t<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// one pair turned; the roundings are spelt out so that both vector widths give
// the same bits
SB_DEV float2 rot_pair(float a, float b, float2 w) {
    return make_float2(__fmaf_rn(a, w.x, -__fmul_rn(b, w.y)), __fmaf_rn(b, w.x, __fmul_rn(a, w.y)));
}
// x / d as a product with ceil(2^32 / d), exact while x d < 2^32
struct RotDiv {
    unsigned d, m;  // m = 0: divide
    SB_DEV RotDiv(unsigned div, bool small) : d(div), m(small && div > 1 ? 0xffffffffu / div + 1 : 0u) {}
    SB_DEV int operator()(int x) const { return m ? (int)__umulhi((unsigned)x, m) : (int)((unsigned)x / d); }
};
template <typename T, int V> struct alignas(sizeof(T) * V) RotVec { T v[V]; };

template <typename T, int V>
SB_DEV void rotary_body(const RotParams &P) {
    __shared__ float2 cs[SB_ROT_MAX_TOK][128];
    __shared__ int pos_s[SB_ROT_MAX_TOK];
    __shared__ long long at_s[SB_ROT_MAX_TOK];  // the slot's place in the pages, -1: none
    const int t0 = blockIdx.x * P.tokens_per_cta, nt = min(P.tokens_per_cta, P.T - t0), half = P.dim >> 1;
    if (threadIdx.x < nt) {
        pos_s[threadIdx.x] = P.pos[t0 + threadIdx.x];
        const long long slot = P.slots ? P.slots[t0 + threadIdx.x] : -1;
        at_s[threadIdx.x] = slot < 0 || slot >= P.n_slots ? -1 : slot / P.page * P.page_stride + slot % P.page * P.pos_stride;
    }
    for (int i = threadIdx.x; i < nt * half; i += SB_ROT_THREADS) {
        const int t = i / half, j = i - t * half;
        const unsigned long long ph = (unsigned long long)(long long)P.pos[t0 + t] * P.turn[j];
        float s, c;
        sincospif((float)(int)(ph >> 32) * 4.656612873077393e-10f, &s, &c);  // 2^-31: signed half turns
        cs[t][j] = make_float2(c * P.mscale, (P.inverse ? -s : s) * P.mscale);
    }
    __syncthreads();
    // units of 2 V values; rows in the order query heads, key heads, value heads
    const int U = P.HD / (2 * V), UR = half / V, H = P.heads[0] + P.heads[1] + P.heads[2], per = H * U;
    const RotDiv by_per(per, per < 32768), by_U(U, per < 32768);  // 4 per^2 < 2^32
    for (int i = blockIdx.y * SB_ROT_THREADS + threadIdx.x; i < nt * per; i += SB_ROT_THREADS * gridDim.y) {
        const int t = by_per(i), r = i - t * per;
        int h = by_U(r);
        const int u = r - h * U, pos = pos_s[t];
        const long long at = at_s[t];
        const int part = h < P.heads[0] ? 0 : h < P.heads[0] + P.heads[1] ? 1 : 2;
        if (part >= 1) h -= P.heads[0];
        if (part == 2) h -= P.heads[1];
        if (pos < 0 || (part && at < 0)) continue;  // padding, or no place in the pages
        const T *x = static_cast<const T *>(P.src[part]) + (t0 + t) * P.st[part] + h * P.sh[part];
        T *y = static_cast<T *>(P.dst[part]) + (part ? at + h * P.head_stride : (t0 + t) * P.dt + h * P.dh);
        int ia, ib;  // the two vectors: neighbouring units are neighbours in both
        bool ta, tb;
        if (P.layout == 0 && part < 2) {
            ta = tb = u < UR;
            ia = ta ? u * V : P.dim + (u - UR) * V;
            ib = ia + (ta ? half : (P.HD - P.dim) >> 1);
        } else if (V > 1) {  // pairs inside each vector, or values
            ia = u * V;
            ib = ia + (P.HD >> 1);
            ta = part < 2 && ia < P.dim;
            tb = part < 2 && ib < P.dim;
        } else {  // a pair's two values
            ia = 2 * u;
            ib = ia + 1;
            ta = tb = part < 2 && ia < P.dim;
        }
        const RotVec<T, V> a = *reinterpret_cast<const RotVec<T, V> *>(x + ia), b = *reinterpret_cast<const RotVec<T, V> *>(x + ib);
        RotVec<T, V> oa = a, ob = b;
        if constexpr (V > 1) {
            if (P.layout) {
                auto pairs = [&](RotVec<T, V> &o, const float2 *w) {
#pragma unroll
                    for (int e = 0; e < V; e += 2) {
                        const float2 r = rot_pair(rot_f<T>(o.v[e]), rot_f<T>(o.v[e + 1]), w[e / 2]);
                        o.v[e] = rot_t<T>(r.x);
                        o.v[e + 1] = rot_t<T>(r.y);
                    }
                };
                if (ta) pairs(oa, &cs[t][ia / 2]);
                if (tb) pairs(ob, &cs[t][ib / 2]);
                ta = false;
            }
        }
        if (ta) {
#pragma unroll
            for (int e = 0; e < V; e++) {
                const float2 r = rot_pair(rot_f<T>(a.v[e]), rot_f<T>(b.v[e]), cs[t][u * V + e]);
                oa.v[e] = rot_t<T>(r.x);
                ob.v[e] = rot_t<T>(r.y);
            }
        }
        *reinterpret_cast<RotVec<T, V> *>(y + ia) = oa;
        *reinterpret_cast<RotVec<T, V> *>(y + ib) = ob;
    }
}
#define SB_ROT_KERNEL(name, T, V)                                                                              \
    extern "C" __global__ void __launch_bounds__(SB_ROT_THREADS) name(const __grid_constant__ RotParams P) {   \
        rotary_body<T, V>(P);                                                                                  \
    }
SB_ROT_KERNEL(rotary_f32, float, 4)
SB_ROT_KERNEL(rotary_f16, __half, 8)
SB_ROT_KERNEL(rotary_bf16, __nv_bfloat16, 8)
SB_ROT_KERNEL(rotary_f32_any, float, 1)
SB_ROT_KERNEL(rotary_f16_any, __half, 1)
SB_ROT_KERNEL(rotary_bf16_any, __nv_bfloat16, 1)
