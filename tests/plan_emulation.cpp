// plan_emulation.cpp -- the page plan's kernel (csrc/serve_plan.cuh, its own
// source) run on the host, a fiber a thread, over arrays of exactly the sizes
// that its contract names, under the address sanitizer: any index outside
// them ends the program.  Lengths are ordinary ones, whose results are
// compared, and hostile ones, whose sums pass 2^31.  Built with -fwrapv:
// integers wrap as on the device.
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <ucontext.h>

#include <algorithm>
#include <memory>
#include <random>
#include <vector>

using std::max;
using std::min;
struct Dim { unsigned x; };
static Dim threadIdx, blockIdx, blockDim, gridDim;
struct longlong2 { long long x, y; };
struct int4 { int x, y, z, w; };
static longlong2 make_longlong2(long long x, long long y) { return {x, y}; }
static int4 make_int4(int x, int y, int z, int w) { return {x, y, z, w}; }

// every thread runs up to its next barrier, in turn
static const int MOST = 512;
static ucontext_t home, fiber[MOST];
static bool done[MOST];
static int exchange[MOST];
static void barrier() { swapcontext(&fiber[threadIdx.x], &home); }
static int shfl_up(int v, int o) {
    const unsigned t = threadIdx.x;
    exchange[t] = v;
    barrier();
    const int got = (int)(t & 31) >= o ? exchange[t - o] : v;
    barrier();
    return got;
}
static int *shared_ints;

#define __device__
#define __global__
#define __forceinline__ inline
#define __launch_bounds__(n)
#define __shared__ static
#define SB_DEV static inline
#define SB_FULL 0xffffffffu
#define __syncthreads barrier
#define __shfl_up_sync(mask, v, o) shfl_up(v, o)
#define atomicAdd(p, v) (*(p) += (v))
#include PLAN_SOURCE

struct Call {
    int B, page, n_free, width, stride, T;
    int *cache, *fresh, *pool, *table;
    long long *slots;
    int *pos, *req, *cu, *kv, *used;
};
static Call call;
static void body() {
    const Call &c = call;
    kv_plan(c.cache, c.fresh, c.B, c.page, c.pool, c.n_free, c.table, c.stride, c.width, c.slots, c.pos, c.req, c.T, c.cu, c.kv, c.used);
    done[threadIdx.x] = true;
    swapcontext(&fiber[threadIdx.x], &home);
}
static void launch(unsigned blocks, unsigned threads) {
    static std::vector<char> stacks(MOST * 65536);
    gridDim.x = blocks;
    blockDim.x = threads;
    for (blockIdx.x = 0; blockIdx.x < blocks; blockIdx.x++) {
        for (unsigned t = 0; t < threads; t++) {
            getcontext(&fiber[t]);
            fiber[t].uc_stack.ss_sp = stacks.data() + t * 65536;
            fiber[t].uc_stack.ss_size = 65536;
            fiber[t].uc_link = &home;
            done[t] = false;
            makecontext(&fiber[t], body, 0);
        }
        for (unsigned left = threads; left;) {
            left = 0;
            for (unsigned t = 0; t < threads; t++)
                if (!done[t]) {
                    threadIdx.x = t;
                    swapcontext(&home, &fiber[t]);
                    left += !done[t];
                }
        }
    }
}

int main(int argc, char **argv) {
    const int rounds = argc > 1 ? atoi(argv[1]) : 1000;
    std::mt19937 rng(1);
    const int edge[] = {0, 1, 2, 3, 15, 16, 17, 100, 0x7fffffff, 0x7ffffffe, 0x7ffffff0, 0x40000000, 0x3fffffff, -1, -0x7fffffff - 1};
    auto pick = [&](int n) { return (int)(rng() % n); };
    for (int it = 0; it < rounds; it++) {
        const bool hostile = it % 4 != 0;
        Call &c = call;
        const unsigned threads = pick(2) ? 32 : 64;
        c.B = 1 + pick(it % 50 == 0 ? 200 : 6);
        c.page = hostile ? edge[1 + pick(12)] : 1 + pick(20);
        c.width = 1 + pick(9);
        c.stride = c.width + pick(3);
        c.n_free = pick(6);
        c.T = pick(40);
        // separate allocations of exactly these sizes
        std::unique_ptr<int[]> cache(new int[c.B]), fresh(new int[c.B]), pool(new int[c.n_free]), cu(new int[c.B + 1]), kv(new int[c.B]);
        std::unique_ptr<int[]> table(new int[(c.B - 1) * c.stride + c.width]), pos(new int[c.T]), req(new int[c.T]), used(new int[2]);
        std::unique_ptr<int[]> smem(new int[2 * (c.B + 1)]);
        std::unique_ptr<long long[]> slots(new long long[c.T]);
        for (int b = 0; b < c.B; b++) {
            cache[b] = !hostile || pick(3) == 0 ? pick(40) : edge[pick(15)];
            fresh[b] = !hostile || pick(3) == 0 ? pick(12) : edge[pick(15)];
        }
        for (int i = 0; i < c.n_free; i++) pool[i] = 100 + i;
        for (int i = 0; i < (c.B - 1) * c.stride + c.width; i++) table[i] = 1000 + i;
        const std::vector<int> before(table.get(), table.get() + (c.B - 1) * c.stride + c.width);
        c.cache = cache.get(), c.fresh = fresh.get(), c.pool = pool.get(), c.table = table.get(), c.slots = slots.get(), c.pos = pos.get();
        c.req = req.get(), c.cu = cu.get(), c.kv = kv.get(), c.used = used.get(), shared_ints = smem.get();
        launch(1 + pick(3), threads);
        if (hostile) continue;
        int t = 0, at = 0, lack = 0;
        bool ok = true;
        for (int b = 0; b < c.B; b++) {
            const int have = (cache[b] + c.page - 1) / c.page, need = (cache[b] + fresh[b] + c.page - 1) / c.page;
            std::vector<int> row(before.begin() + b * c.stride, before.begin() + b * c.stride + c.width);
            for (int j = have; j < need; j++) {
                if (j >= c.width) lack++;
                else {
                    row[j] = at < c.n_free ? pool[at] : -1;
                    lack += at >= c.n_free;
                    at++;
                }
            }
            for (int j = 0; j < c.width; j++) ok &= table[b * c.stride + j] == row[j];
            ok &= cu[b] == t && kv[b] == cache[b] + fresh[b];
            for (int i = 0; i < fresh[b]; i++, t++) {
                const int p = cache[b] + i, pg = p / c.page < c.width ? row[p / c.page] : -1;
                if (t < c.T) ok &= pos[t] == p && req[t] == b && slots[t] == (pg >= 0 ? (long long)pg * c.page + p % c.page : -1);
            }
        }
        for (int i = t; i < c.T; i++) ok &= pos[i] == -1 && req[i] == -1 && slots[i] == -1;
        ok &= cu[c.B] == t && used[0] == min(at, c.n_free) && used[1] == lack;
        if (!ok) {
            printf("case %d: wrong result\n", it);
            return 1;
        }
    }
    printf("%d cases\n", rounds);
    return 0;
}
