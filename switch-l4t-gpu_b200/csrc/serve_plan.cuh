// serve_plan.cuh -- block tables and slot maps of a batch, built on the GPU
// from request lengths (kv_plan).
//
// Request b has cache_len[b] positions in have = ceil(cache_len / page)
// pages and gets new_len[b] more, so it needs ceil((cache_len + new_len) /
// page) pages, at most the table's width.  The missing ones come from the
// free list in request order: request b's start at the sum of what the
// requests before it take.  Token i of request b sits at position p =
// cache_len[b] + i, in slot table[b][p / page] * page + p % page.
//
// Bound: latency.  The two prefix sums over B requests are a few
// microseconds on one SM and the outputs are 16 bytes a token.  So every CTA
// repeats the sums (8 B bytes of L2 reads) instead of waiting for another
// launch, and the CTAs then share out the table rows (a warp a request) and
// the tokens (a thread four neighbours, the request found by bisection in
// shared memory).  A token's page is recomputed from the sums, so no CTA
// reads what another one writes.
#pragma once
#include "sb_common.cuh"

#define SB_PLAN_THREADS 512

// exclusive sums over the block of this thread's (a, b)
SB_DEV void plan_scan2(int &a, int &b, int *wa, int *wb) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    int x = a, y = b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int p = __shfl_up_sync(SB_FULL, x, o), q = __shfl_up_sync(SB_FULL, y, o);
        if (lane >= o) { x += p; y += q; }
    }
    if (lane == 31) { wa[w] = x; wb[w] = y; }
    __syncthreads();
    int sa = 0, sb = 0;
    for (int i = 0; i < w; i++) { sa += wa[i]; sb += wb[i]; }
    a = sa + x - a;
    b = sb + y - b;
}
// pages that n positions fill; n + page - 1 < 2^32 (a 64-bit division costs 100 cycles)
SB_DEV unsigned plan_pages(unsigned n, unsigned page) { return (n + page - 1) / page; }

// dynamic shared memory: 2 (B + 1) ints
extern "C" __global__ void __launch_bounds__(SB_PLAN_THREADS)
    kv_plan(const int *__restrict__ cache_len, const int *__restrict__ new_len, int B, int page,
            const int *__restrict__ free_pages, int n_free, int *table, int table_stride, int width,
            long long *__restrict__ slots, int *__restrict__ pos, int *__restrict__ req, int T,
            int *__restrict__ cu_q, int *__restrict__ kv_len, int *__restrict__ used) {
    extern __shared__ int plan_sm[];
    __shared__ int wa[SB_PLAN_THREADS / 32], wb[SB_PLAN_THREADS / 32], lack_s;
    int *cu = plan_sm, *first = plan_sm + B + 1;
    const int tid = threadIdx.x, nthreads = blockDim.x, per = (B + nthreads - 1) / nthreads;
    if (tid == 0) lack_s = 0;
    // this thread's requests [b0, b1): tokens and pages, negative lengths as 0
    const int b0 = min(tid * per, B), b1 = min(b0 + per, B);
    int tok = 0, add = 0, lack = 0, len = 0;
    for (int b = b0; b < b1; b++) {
        const int c = max(cache_len[b], 0), n = max(new_len[b], 0);
        // unsigned until the width has cut it: lengths past the limit index nothing outside
        const unsigned have = plan_pages(c, page), need = plan_pages((unsigned)c + n, page), last = min(need, (unsigned)width);
        const int got = last > have ? (int)(last - have) : 0;
        cu[b] = n;
        first[b] = got;
        tok += n;
        add += got;
        lack += (int)(need - have) - got;
        len = c + n;
    }
    int t0 = tok, p0 = add;
    plan_scan2(t0, p0, wa, wb);
    for (int b = b0; b < b1; b++) {  // lengths turn into sums in place
        const int n = cu[b], got = first[b];
        cu[b] = t0;
        first[b] = p0;
        t0 += n;
        p0 += got;
    }
    if (b1 == B && b0 < B) {  // the thread that owns the last request (B > 0)
        cu[B] = t0;
        first[B] = p0;
    }
    if (lack) atomicAdd(&lack_s, lack);
    if (blockIdx.x == 0 && per == 1 && b0 < B) kv_len[b0] = len;
    __syncthreads();
    if (blockIdx.x == 0) {
        for (int b = tid; b <= B; b += nthreads) {
            cu_q[b] = cu[b];
            if (b < B && per > 1) kv_len[b] = max(cache_len[b], 0) + max(new_len[b], 0);
        }
        if (tid == 0) {
            const int total = first[B], taken = min(total, n_free);
            used[0] = taken;
            used[1] = total - taken + lack_s;
        }
    }
    // new entries of the tables: a warp a request
    const int lane = tid & 31, nw = gridDim.x * (nthreads / 32);
    for (int b = blockIdx.x * (nthreads / 32) + (tid >> 5); b < B; b += nw) {
        const int f = first[b], n = first[b + 1] - f;
        if (n == 0) continue;
        const unsigned have = plan_pages(max(cache_len[b], 0), page);
        for (int j = lane; j < n; j += 32)
            table[(size_t)b * table_stride + have + j] = (unsigned)(f + j) < (unsigned)n_free ? free_pages[f + j] : -1;
    }
    // tokens: four neighbours a thread
    const int total = cu[B];
    for (long long q = (long long)blockIdx.x * nthreads + tid; q * 4 < T; q += (long long)gridDim.x * nthreads) {
        const int t = (int)(q * 4);
        int b = -1;
        if (t < total) {  // the last request that starts at or before t and is not empty
            int lo = 0, hi = B;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (cu[mid] <= t) lo = mid;
                else hi = mid;
            }
            b = lo;
        }
        long long slot[4];
        int p[4], rq[4], c = -1, off = 0;
        unsigned have = 0, j = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            slot[i] = -1;
            p[i] = rq[i] = -1;
            if (t + i >= total) continue;
            bool fresh = i == 0;
            while (t + i >= cu[b + 1]) {
                b++;
                fresh = true;
            }
            if (fresh) {
                c = max(cache_len[b], 0);
                have = plan_pages(c, page);
                const unsigned at = (unsigned)c + (unsigned)(t + i - cu[b]);
                j = at / (unsigned)page;
                off = (int)(at - j * (unsigned)page);
            } else if (++off == page) {
                off = 0;
                j++;
            }
            int pg = -1;
            if (j < (unsigned)width) {
                const unsigned i_free = (unsigned)first[b] + j - have;
                if (j < have) pg = table[(size_t)b * table_stride + j];
                else if (i_free < (unsigned)n_free) pg = free_pages[i_free];
            }
            if (pg >= 0) slot[i] = (long long)pg * page + off;
            p[i] = c + (t + i - cu[b]);
            rq[i] = b;
        }
        if (t + 4 <= T && ((uintptr_t)slots & 15) == 0 && (((uintptr_t)pos | (uintptr_t)req) & 15) == 0) {
            reinterpret_cast<longlong2 *>(slots + t)[0] = make_longlong2(slot[0], slot[1]);
            reinterpret_cast<longlong2 *>(slots + t)[1] = make_longlong2(slot[2], slot[3]);
            *reinterpret_cast<int4 *>(pos + t) = make_int4(p[0], p[1], p[2], p[3]);
            *reinterpret_cast<int4 *>(req + t) = make_int4(rq[0], rq[1], rq[2], rq[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (t + i >= T) break;
                slots[t + i] = slot[i];
                pos[t + i] = p[i];
                req[t + i] = rq[i];
            }
        }
    }
}
