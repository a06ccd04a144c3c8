"""Page plan, rotary positions and shared-prefix attention on the GPU against
plain implementations in 64 bits, at the sizes, masks, strides and tables
where they can go wrong."""
import math
import time

import numpy as np
import pytest
import torch

import sb200

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def half_step(t):
    return torch.finfo(t).eps / 2


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def stream():
    return torch.cuda.current_stream()


# ---------------------------------------------------------------- plan
def plan_reference(cache, new, page, free, table, width, T):
    table = [list(r) for r in table]
    at = total = lacking = 0
    slots, pos, req, cu = [], [], [], [0]
    for b, (c, n) in enumerate(zip(cache, new)):
        c, n = max(c, 0), max(n, 0)
        have, need = -(-c // page), -(-(c + n) // page)
        for j in range(have, need):
            if j >= width:
                lacking += 1
                continue
            table[b][j] = free[at] if at < len(free) else -1
            lacking += at >= len(free)
            total += at < len(free)
            at += 1
        for p in range(c, c + n):
            pg = table[b][p // page] if p // page < width else -1
            slots.append(pg * page + p % page if pg >= 0 else -1)
            pos.append(p)
            req.append(b)
        cu.append(cu[-1] + n)
    pad = lambda v: (v + [-1] * T)[:T]  # noqa: E731
    return table, pad(slots), pad(pos), pad(req), cu, [max(c, 0) + max(n, 0) for c, n in zip(cache, new)], [total, lacking]


@pytest.mark.parametrize("B,page,most_new,short,pad", [
    (1, 16, 1, 0, 0), (2, 1, 3, 0, 1), (7, 16, 40, 0, 5), (33, 24, 5, 7, 0), (64, 128, 300, 0, 3), (600, 16, 9, 11, 2), (1500, 3, 2, 0, -50),
    (16384, 8, 1, 0, 0)])
def test_kv_plan(cuda_dev, B, page, most_new, short, pad):
    rng = np.random.RandomState(B)
    cache = rng.randint(0, 5 * page + 2, B).tolist()
    new = (rng.randint(0, most_new + 1, B) if most_new > 1 else np.ones(B, int)).tolist()
    if B > 5:
        cache[3], new[2], new[4], new[B - 1] = -4, -1, 0, 0
    width = 6 + most_new // page - (1 if B == 33 else 0)
    table = np.full((B, width), -7, np.int32)
    k = 0
    for b in range(B):
        n = min(-(-max(cache[b], 0) // page), width)
        table[b, :n] = np.arange(k, k + n)
        k += n
    add = sum(-(-(max(c, 0) + max(n, 0)) // page) - -(-max(c, 0) // page) for c, n in zip(cache, new))
    free = (10 ** 6 + rng.permutation(max(add - short, 1))).astype(np.int32)
    T = max(sum(max(n, 0) for n in new) + pad, 0)
    want = plan_reference(cache, new, page, free.tolist(), table.tolist(), width, T)
    d_table = torch.full((B, width + 3), -9, dtype=torch.int32, device="cuda")  # rows wider than the table that is passed
    d_table[:, :width] = torch.from_numpy(table).cuda()
    view = d_table[:, :width]
    slots = torch.full((T + 2,), 77, dtype=torch.int64, device="cuda")
    pos, req = (torch.full((T + 2,), 77, dtype=torch.int32, device="cuda") for _ in range(2))
    cu, kv, used = i32([77] * (B + 2)), i32([77] * (B + 1)), i32([77] * 3)
    for _ in range(2):  # a second run on its own table gives the same
        sb200.kv_plan(i32(cache), i32(new), torch.from_numpy(free).cuda(), view, page, slots[:T], pos[:T], req[:T], cu, kv, used, stream=stream())
        got = view.tolist(), slots[:T].tolist(), pos[:T].tolist(), req[:T].tolist(), cu[: B + 1].tolist(), kv[:B].tolist(), used[:2].tolist()
        for name, a, b in zip(("table", "slots", "pos", "req", "cu_q", "kv_len", "used"), got, want):
            assert a == b, name
    # nothing past what was passed
    assert slots[T:].tolist() == [77, 77] and pos[T:].tolist() == [77, 77] and cu[B + 1:].tolist() == [77] and kv[B:].tolist() == [77]
    assert used[2].item() == 77 and bool((d_table[:, width:] == -9).all())


def test_kv_plan_absent_pages_and_no_free(cuda_dev):
    """A free list that is empty, or padded with -1, and a table entry that is
    not there: their tokens get no slot."""
    table = i32([[3, -1, -5], [-5, -5, -5]])
    out = lambda n, t=torch.int32: torch.zeros(n, dtype=t, device="cuda")  # noqa: E731
    slots, pos, req, cu, kv, used = out(6, torch.int64), out(6), out(6), out(3), out(2), out(2)
    sb200.kv_plan(i32([3, 0]), i32([3, 2]), i32([8, -1]), table, 2, slots, pos, req, cu, kv, used, stream=stream())
    # request 0: position 3 in its page 1 (absent), 4 and 5 in the new page 8; request 1 in the absent new page
    assert table.tolist() == [[3, -1, 8], [-1, -5, -5]]
    assert slots.tolist() == [-1, 16, 17, -1, -1, -1] and pos.tolist() == [3, 4, 5, 0, 1, -1] and used.tolist() == [2, 0]
    sb200.kv_plan(i32([0, 0]), i32([1, 0]), out(0), table, 2, slots, pos, req, cu, kv, used, stream=stream())
    assert table.tolist()[0][0] == -1 and used.tolist() == [0, 1] and slots.tolist() == [-1] * 6


# ---------------------------------------------------------------- rotary
def frequencies(dim, theta, scaling, factor, orig):
    i = np.arange(dim // 2)
    if scaling == sb200.ROPE_NTK:
        theta = theta * factor ** (dim / (dim - 2))
    f = theta ** (-2.0 * i / dim)
    m = 1.0
    if scaling == sb200.ROPE_LINEAR:
        f = f / factor
    elif scaling == sb200.ROPE_YARN:
        low = max(math.floor(dim * math.log(orig / (32 * 2 * math.pi)) / (2 * math.log(theta))), 0)
        high = min(math.ceil(dim * math.log(orig / (2 * math.pi)) / (2 * math.log(theta))), dim - 1)
        r = np.clip((i - low) / (high - low if high > low else 0.001), 0, 1)
        f, m = f / factor * r + f * (1 - r), 0.1 * math.log(factor) + 1
    elif scaling == sb200.ROPE_BANDS:
        s = np.clip((orig * f / (2 * math.pi) - 1) / 3, 0, 1)
        f = f / factor * (1 - s) + f * s
    return torch.tensor(f, device="cuda"), m


def turned(x, pos, f, m, layout, inverse=False):
    """The rotation in 64 bits, and per value the |a| + |b| of its pair."""
    d = 2 * f.numel()
    y, size = x.double().clone(), x.double().abs()
    t = pos.double()[:, None, None] * f
    c, s = torch.cos(t) * m, torch.sin(t) * m * (-1 if inverse else 1)
    ia, ib = (slice(0, d // 2), slice(d // 2, d)) if layout == sb200.ROPE_HALF else (slice(0, d, 2), slice(1, d, 2))
    a, b = x.double()[..., ia], x.double()[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    size[..., ia] = size[..., ib] = a.abs() + b.abs()
    return y, size


def rotary_bound(want, size, m, t):
    """cos and sin are off by at most 2.7e-7: the phase's 2^-25 half turns
    (9.4e-8), two ulp of sincospif (1.2e-7), the product with m (6e-8); the
    products add 1.2e-7 of |a| + |b|; then one rounding to the type: half a
    step relative to the value, for fp16 below 2^-14 half of the 2^-24 that its
    subnormals are apart."""
    return 4e-7 * m * size + half_step(t) * want.abs() + (2.0 ** -25 if t == torch.float16 else 1e-30)


@pytest.mark.parametrize("T,H,HD,dim,layout,scaling,far,kind", [
    (1, 14, 64, 64, 0, 0, 100, "f32"), (5, 3, 128, 32, 1, 3, 1 << 20, "bf16"), (130, 2, 80, 80, 0, 4, 1 << 17, "f16"),
    (33, 1, 64, 16, 1, 2, 1 << 20, "f32"), (700, 5, 256, 256, 0, 1, 1 << 30, "f32"), (3, 7, 8, 4, 0, 0, 2 ** 31 - 1, "bf16"),
    (2500, 6, 96, 48, 1, 0, 4096, "f16"), (9, 2, 6, 2, 1, 0, 50, "f32"), (41, 4, 64, 64, 1, 3, 2 ** 31 - 1, "f16")])
@pytest.mark.parametrize("odd", [False, True])
def test_rotary_rows(cuda_dev, T, H, HD, dim, layout, scaling, far, kind, odd):
    t = DT[kind]
    g = torch.Generator("cuda").manual_seed(T + H)
    extra = 1 if odd else 8  # odd: token strides that are no multiple of a vector
    x = torch.randn(T, H * HD + extra, device="cuda", generator=g).to(t)[:, : H * HD].unflatten(1, (H, HD))
    pos = torch.randint(0, far, (T,), device="cuda", generator=g).to(torch.int32)
    pos[0] = far - 1
    if T > 4:
        pos[3] = -1
    plan = sb200.Rotary(dim, theta=1e6, layout=layout, scaling=scaling, factor=16.0, orig_ctx=4096)
    f, m = frequencies(dim, 1e6, scaling, 16.0, 4096)
    for inverse in (False, True):
        y = torch.full((T, H, HD), 7.0, dtype=t, device="cuda")
        sb200.rotary(x, y, pos, plan, inverse=inverse, stream=stream())
        want, size = turned(x, pos, f, m, layout, inverse)
        live = pos >= 0
        # angles of 2^31 positions: the plan's fractions are good to 2^-54 of a turn per position (pow), the reference's product to 2^-53 of it
        slack = 2 * math.pi * far * 2.0 ** -52 * m
        err = (y.double() - want).abs()[live]
        assert bool((err <= (rotary_bound(want, size, m, t) + slack * size)[live]).all()), float(err.max())
        assert torch.equal(y[..., dim:][live], x[..., dim:][live])
        if T > 4:
            assert bool((y[3] == 7).all())  # a row of padding is left as it was
    z = x.clone()  # in place
    sb200.rotary(z, z, pos, plan, inverse=True, stream=stream())
    assert torch.equal(z[live], y[live]) and (T <= 4 or torch.equal(z[3], x[3]))


def test_rotary_inverse_is_the_gradient(cuda_dev):
    """<w, d rotary(x)> against differences of the rotation itself: it is
    linear, so a step of 1 has no error but the rounding of its values."""
    T, H, HD, dim = 3, 2, 16, 12
    g = torch.Generator("cuda").manual_seed(0)
    x, w = (torch.randn(T, H, HD, device="cuda", generator=g) for _ in range(2))
    pos, plan = i32([5, 1000, 77777]), sb200.Rotary(dim, theta=1e4, layout=sb200.ROPE_PAIRS, scaling=sb200.ROPE_YARN, factor=4.0, orig_ctx=512)
    grad, y0, y1 = (torch.empty_like(x) for _ in range(3))
    sb200.rotary(w, grad, pos, plan, inverse=True, stream=stream())
    sb200.rotary(x, y0, pos, plan, stream=stream())
    for t, h, i in ((0, 0, 0), (1, 1, 7), (2, 0, 11), (2, 1, 15)):
        z = x.clone()
        z[t, h, i] += 1.0
        sb200.rotary(z, y1, pos, plan, stream=stream())
        diff = float(((y1 - y0).double() * w.double()).sum())
        assert abs(diff - float(grad[t, h, i])) < 64 * 2.0 ** -24 * 8  # a few values of size <= 8, each off by a few half steps


@pytest.mark.parametrize("kind,page,HD,dim", [("f32", 16, 64, 64), ("f16", 1, 128, 64), ("bf16", 24, 80, 40), ("f16", 7, 10, 6)])
def test_rotary_kv(cuda_dev, kind, page, HD, dim):
    t, T, NH, NKV = DT[kind], 61, 6, 2
    g = torch.Generator("cuda").manual_seed(page)
    qkv = torch.randn(T, NH + 2 * NKV, HD, device="cuda", generator=g).to(t)
    q, k, v = qkv.split([NH, NKV, NKV], 1)
    n_pages = -(-T // page) + 2
    pool = torch.full((n_pages, page, 2, NKV, HD), 5.0, dtype=t, device="cuda")  # keys and values side by side
    kc, vc = pool[:, :, 0], pool[:, :, 1]
    slots = torch.randperm(n_pages * page, device="cuda", generator=g)[:T].contiguous()
    pos = torch.randint(0, 9000, (T,), device="cuda", generator=g).to(torch.int32)
    slots[4], slots[5], pos[6] = -1, n_pages * page, -1  # no slot, a slot outside the pool, padding
    q_out = torch.full((T, NH, HD), 5.0, dtype=t, device="cuda")
    plan = sb200.Rotary(dim, theta=1e5)
    sb200.rotary_kv(q, q_out, k, v, pos, slots, plan, sb200.KvPages(kc, vc), stream=stream())
    f, m = frequencies(dim, 1e5, 0, 1.0, 0)
    live = pos >= 0
    want, size = turned(q, pos, f, m, 0)
    assert bool(((q_out.double() - want).abs() <= rotary_bound(want, size, m, t))[live].all()) and bool((q_out[6] == 5).all())
    stored = live & (slots >= 0) & (slots < n_pages * page)
    want, size = turned(k, pos, f, m, 0)
    at = slots[stored]
    got = kc[at // page, at % page].double()
    assert bool(((got - want[stored]).abs() <= rotary_bound(want, size, m, t)[stored]).all())
    assert torch.equal(vc[at // page, at % page], v[stored])
    left = torch.ones(n_pages * page, dtype=torch.bool, device="cuda")
    left[at] = False
    left = left.view(n_pages, page)
    assert bool((pool[left] == 5).all())  # every other place is as it was


@pytest.mark.parametrize("kind,layout", [("f32", 0), ("bf16", 1), ("f16", 0)])
def test_rotary_kv_in_place(cuda_dev, kind, layout):
    """Queries turned where they are, beside keys and values of one product:
    the bits of a call with its own output."""
    t, T, NH, NKV, HD = DT[kind], 37, 6, 2, 64
    g = torch.Generator("cuda").manual_seed(3)
    qkv = torch.randn(T, NH + 2 * NKV, HD, device="cuda", generator=g).to(t)
    before = qkv.clone()
    q, k, v = qkv.split([NH, NKV, NKV], 1)
    kc, vc, kc2, vc2 = (torch.zeros(4, 16, NKV, HD, dtype=t, device="cuda") for _ in range(4))
    pos, slots = torch.arange(T, device="cuda", dtype=torch.int32) + 900, torch.randperm(64, device="cuda", generator=g)[:T]
    plan, q_out = sb200.Rotary(32, layout=layout), torch.empty(T, NH, HD, dtype=t, device="cuda")
    sb200.rotary_kv(q, q_out, k, v, pos, slots, plan, sb200.KvPages(kc, vc), stream=stream())
    sb200.rotary_kv(q, q, k, v, pos, slots, plan, sb200.KvPages(kc2, vc2), stream=stream())
    assert torch.equal(q, q_out) and torch.equal(kc, kc2) and torch.equal(vc, vc2)
    assert torch.equal(qkv[:, NH:], before[:, NH:])


# ---------------------------------------------------------------- attention
class Batch:
    """Inputs of a call with sentinels and garbage wherever nothing may be
    read or written, and its result in 64 bits."""

    def __init__(self, kind, NH, NKV, HD, P, lens, rows=None, page=16, seed=0, pad=0, peak=1.0, pool=None):
        self.t, self.NH, self.NKV, self.HD, self.P, self.page = DT[kind], NH, NKV, HD, P, page
        g = torch.Generator("cuda").manual_seed(seed)
        B = len(lens)
        self.rows = rows or [1] * B
        self.lens = lens
        self.T = sum(self.rows) + pad
        pp = -(-P // page)
        need = [-(-n // page) for n in lens]
        n_pages = pp + sum(need) + 3
        perm = torch.randperm(n_pages, device="cuda", generator=g).to(torch.int32)
        self.ptable = perm[:pp].contiguous() if P else None
        self.table = torch.full((B, max(need + [1]) + 1), -1, dtype=torch.int32, device="cuda")
        at = pp
        for b, n in enumerate(need):
            self.table[b, :n] = perm[at: at + n]
            self.table[b, n:] = 10 ** 9  # never a page
            at += n
        shape = (n_pages, page, NKV, HD) if pool is None else pool
        self.k, self.v = (torch.full(shape, float("nan"), dtype=self.t, device="cuda")[:n_pages] for _ in range(2))
        real = lambda *s: (torch.randn(*s, device="cuda", generator=g) * peak).to(self.t)  # noqa: E731
        self.places = []  # per request, then the prefix: pages and places of its positions
        for b, n in list(enumerate(lens)) + [(-1, P)]:
            i = torch.arange(n, device="cuda")
            tab = self.table[b] if b >= 0 else self.ptable
            pg = tab[i // page].long() if n else i
            self.k[pg, i % page], self.v[pg, i % page] = real(n, NKV, HD), real(n, NKV, HD)
            self.places.append((pg, i % page))
        self.q = real(self.T, NH, HD)
        self.cu = i32(np.concatenate([[0], np.cumsum(self.rows)]).tolist())
        self.kv_len = i32(lens)
        self.scale = HD ** -0.5
        self.kv = sb200.KvPages(self.k, self.v)

    def want(self):
        """out, lse, and out of |v|: the size that rounding works on."""
        T, G = self.T, self.NH // self.NKV
        out = torch.zeros(T, self.NH, self.HD, dtype=torch.float64, device="cuda")
        size, lse = out.clone(), torch.full((T, self.NH), -math.inf, dtype=torch.float64, device="cuda")
        pg, pl = self.places[-1]
        kp, vp = self.k[pg, pl].double(), self.v[pg, pl].double()
        r = 0
        for b, n in enumerate(self.rows):
            pg, pl = self.places[b]
            k, v = torch.cat([kp, self.k[pg, pl].double()]), torch.cat([vp, self.v[pg, pl].double()])
            for i in range(n):
                sees = self.P + max(min(self.lens[b] - n + i + 1, self.lens[b]), 0)
                if sees:
                    q = self.q[r].double().view(self.NKV, G, self.HD)
                    s = torch.einsum("hgd,khd->hgk", q, k[:sees]) * self.scale
                    w = torch.softmax(s, -1)
                    lse[r] = torch.logsumexp(s, -1).flatten()
                    out[r] = torch.einsum("hgk,khd->hgd", w, v[:sees]).reshape(self.NH, self.HD)
                    size[r] = torch.einsum("hgk,khd->hgd", w, v[:sees].abs()).reshape(self.NH, self.HD)
                r += 1
        return out, lse, size

    def run(self, own=True, max_q=None, out=None, lse=None, ws=None, **kw):
        out = torch.full_like(self.q, 7.0) if out is None else out
        lse = torch.full((self.T, self.NH), 7.0, device="cuda") if lse is None else lse
        max_kv = max(self.lens) if own else 0
        max_q = max_q or max(max(self.rows), 1)
        ragged = self.rows != [1] * len(self.lens) or self.T != len(self.lens) or max_q > 1
        n = sb200.attn_prefix_ws(self.q, self.kv, self.P, len(self.lens), max_q=max_q, max_kv=max_kv)
        if ws is None:  # NaN: a part that is read before it is written shows
            ws = torch.full((n // 4 + 4,), float("nan"), device="cuda")
        sb200.attn_prefix(self.q, out, self.kv, self.ptable, self.P, self.kv, self.table, self.kv_len, self.scale, ws,
                          cu_q=self.cu if ragged else None, max_q=max_q, max_kv=max_kv, lse=lse, stream=stream(), **kw)
        return out, lse

    def check(self, got=None, want=None):
        """16-bit types: half a step of each weight (on |v|), half a step of the
        result, and 6e-5 for the FP32 part (scores of size 10 off by 2^-20,
        20 to 300 truncated sums of 2^-23).  FP32: 2e-5 (scores: 130 terms of
        2^-24 on sums of |q k| up to 60).  lse: the same score error."""
        out, lse = got or self.run()
        wo, wl, size = want or self.want()
        n = sum(self.rows)
        u = half_step(self.t) if self.t != torch.float32 else 0.0
        err = (out[:n].double() - wo[:n]).abs()
        bound = u * (size[:n] + wo[:n].abs()) + (6e-5 if u else 2e-5) * size[:n] + (2.0 ** -24 if self.t == torch.float16 else 1e-30)
        assert bool((err <= bound).all()), (float(err.max()), float((err / bound).max()))
        fin = torch.isfinite(wl[:n])
        assert torch.equal(fin, torch.isfinite(lse[:n])) and bool((lse[:n][~fin] == -math.inf).all())
        assert bool(((lse[:n].double() - wl[:n]).abs()[fin] <= 6e-5 + 2.0 ** -22 * wl[:n].abs()[fin]).all())
        assert bool((out[n:] == 7).all()) and bool((lse[n:] == 7).all())  # padding is left as it was


KINDS = ["f32", "f16", "bf16"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("NH,NKV,HD,P,lens,page", [
    (14, 2, 64, 300, [64, 1, 0, 33], 16),       # the Qwen heads; a request without positions of its own
    (12, 12, 64, 1, [1], 16),                   # one position each
    (1, 1, 8, 0, [1], 1),                       # the smallest call
    (4, 4, 64, 0, [0, 5, 0], 16),               # rows that see nothing
    (8, 1, 128, 129, [127, 128, 129, 1000], 24),
    (6, 2, 80, 65, [17, 63], 7),                # odd head size, pages that end inside a tile
    (32, 8, 128, 2050, [300] * 3, 64),
    (9, 3, 40, 700, [5, 2], 1024),
    (20, 1, 64, 100, [50, 70], 32),             # more than 16 heads on one key head
])
def test_attn_prefix_single_rows(cuda_dev, kind, NH, NKV, HD, P, lens, page):
    Batch(kind, NH, NKV, HD, P, lens, page=page, seed=P + HD).check()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("NH,NKV,HD,P,lens,rows,page,pad", [
    (14, 2, 64, 200, [40, 9, 0, 130], [3, 9, 0, 33], 16, 5),   # causal among a request's rows; an empty one; padding
    (4, 1, 128, 0, [70, 1], [70, 1], 32, 0),                   # no prefix: plain causal prefill
    (2, 2, 64, 77, [3, 300], [5, 2], 16, 1),                   # more rows than positions: the first rows see only the prefix
    (2, 2, 32, 0, [2, 0], [4, 3], 8, 0),                       # and without a prefix nothing
    (8, 2, 96, 1500, [65, 64, 63], [17, 16, 15], 48, 0),
])
def test_attn_prefix_many_rows(cuda_dev, kind, NH, NKV, HD, P, lens, rows, page, pad):
    b = Batch(kind, NH, NKV, HD, P, lens, rows=rows, page=page, seed=P + HD, pad=pad)
    want = b.want()
    b.check(want=want)
    b.check(got=b.run(max_q=1), want=want)  # max_q sizes the launch only
    b.check(got=b.run(max_q=200), want=want)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("NH,NKV,HD,P,lens,rows,page", [
    (8, 2, 64, 0, [400, 130, 1], [300, 129, 1], 16),
    (4, 1, 128, 200, [513, 0, 77], [513, 0, 60], 24),
    (14, 2, 64, 333, [257, 700], [256, 255], 64)])
def test_attn_prefix_rows_of_a_prompt(cuda_dev, kind, NH, NKV, HD, P, lens, rows, page):
    """A prompt's own rows: hundreds a request, each with its own limit."""
    Batch(kind, NH, NKV, HD, P, lens, rows=rows, page=page, seed=53).check()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("NH,NKV,HD,P,lens,rows,T", [
    (14, 2, 64, 40, [20, 9, 30], [3, 4, 2], 6),      # the second request's last row and the third's are not there
    (4, 2, 128, 0, [70, 60, 90], [30, 40, 20], 50),  # row tiles of 64
    (4, 2, 64, 300, [200, 90], [150, 60], 140),      # a prefix of 256-row tiles
    (4, 2, 64, 0, [5, 2, 9], [4, 6, 2], 8)])         # more rows than positions
def test_attn_prefix_rows_past_the_last(cuda_dev, kind, NH, NKV, HD, P, lens, rows, T):
    """Fewer rows than the requests have together (as the page plan lists
    fewer tokens than there are): those that are there see what they would
    see among all of them."""
    b = Batch(kind, NH, NKV, HD, P, lens, rows=rows, seed=41)
    wo, wl, size = b.want()
    b.q, b.T = b.q[:T].contiguous(), T
    out, lse = b.run()
    b.rows = [T]
    b.check(got=(out, lse), want=(wo[:T], wl[:T], size[:T]))


@pytest.mark.parametrize("kind", KINDS)
def test_attn_prefix_rows_of_no_request(cuda_dev, kind):
    """Row offsets that do not start at 0: the rows before the first request
    mean nothing, but no part outside the workspace is read for them, and the
    others are right."""
    b = Batch(kind, 14, 2, 64, 1000, [40, 300, 170], rows=[2, 1, 3], seed=43)
    wo, wl, size = b.want()
    b.run()
    ws = torch.full((sb200.attn_prefix_ws(b.q, b.kv, 1000, 2, max_q=3, max_kv=300) // 4 + 4,), float("nan"), device="cuda")
    out, lse = torch.full_like(b.q, 7.0), torch.full((b.T, 14), 7.0, device="cuda")
    sb200.attn_prefix(b.q, out, b.kv, b.ptable, 1000, b.kv, b.table[1:], b.kv_len[1:], b.scale, ws, cu_q=b.cu[1:], max_q=3, max_kv=300,
                      lse=lse, stream=stream())
    b.rows = [4]
    b.check(got=(out[2:], lse[2:]), want=(wo[2:], wl[2:], size[2:]))


@pytest.mark.parametrize("kind", KINDS)
def test_attn_prefix_large_batch(cuda_dev, kind):
    """Many row tiles on one key head, a long prefix cut into ranges, ragged
    own lengths."""
    lens = [(i * 37) % 200 for i in range(150)]
    Batch(kind, 14, 2, 64, 3001, lens, page=16, seed=1).check()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("B,NH,NKV,HD,P,page", [
    (128, 1, 1, 64, 1, 16), (129, 2, 1, 128, 127, 7), (64, 8, 2, 80, 128, 24), (257, 1, 1, 128, 129, 1), (33, 16, 2, 64, 1300, 64),
    (40, 14, 2, 40, 700, 700), (20, 32, 2, 128, 5000, 128)])
def test_attn_prefix_many_rows_a_key_head(cuda_dev, kind, B, NH, NKV, HD, P, page):
    """More than 16 query rows of a key head (16-bit types: the tcgen05
    kernel): one row tile full, over, or partly filled; one key, a tile less
    one, a tile, one more; a negative scale."""
    lens = [(i * 5) % 9 for i in range(B)]
    b = Batch(kind, NH, NKV, HD, P, lens, page=page, seed=B + P)
    want = b.want()
    b.check(want=want)
    b.scale = -b.scale
    b.check()


@pytest.mark.parametrize("kind", KINDS)
def test_attn_prefix_growing_scores(cuda_dev, kind):
    """Keys whose scores rise along the prefix: the maximum that a row's parts
    are held against moves again and again, and a first part of low scores is
    scaled down to nothing."""
    b = Batch(kind, 16, 1, 64, 2000, [3] * 10, seed=21)
    b.q = b.q.abs()
    b.k[b.places[-1]] = (torch.linspace(-2, 2, 2000, device="cuda")[:, None, None] + 0.1 * b.k[b.places[-1]].float()).to(b.t)
    out, lse = b.run()
    wo, wl, size = b.want()
    # scores up to 64 x 0.8 x 2 / 8 = 13 either way, on |q k| sums of 100: 2^-24 x 70 terms x 100 / 8 = 5e-5, twice (key, query)
    u = half_step(b.t) if b.t != torch.float32 else 0.0
    assert bool(((out.double() - wo).abs() <= u * (size + wo.abs()) + 2e-4 * size + 2.0 ** -24).all())
    assert bool(((lse.double() - wl).abs() <= 2e-4).all())


@pytest.mark.parametrize("kind", KINDS)
def test_attn_prefix_peaked_scores(cuda_dev, kind):
    """Scores of size 60: the running maximum moves far from tile to tile.
    Their FP32 rounding grows with them, so only values of the formula count
    here: weights that sum to 1 on values of 1."""
    b = Batch(kind, 4, 2, 64, 500, [100, 37], seed=3)
    b.q *= 8
    for pg, pl in b.places:
        b.v[pg, pl] = 1.0
    out, lse = b.run()
    assert bool(((out.double() - 1).abs() <= 4 * half_step(b.t) + 1e-5).all())
    wl = b.want()[1]
    # |q k| sums reach 64 x 8 x 3: 130 terms of 2^-24 of that, times the scale
    assert bool(((lse.double() - wl).abs() <= 130 * 2.0 ** -24 * 1536 * b.scale + 2.0 ** -21 * wl.abs()).all())


@pytest.mark.parametrize("kind,size", [("bf16", 1e6), ("bf16", 3e3), ("f16", 1e4), ("f32", 1e6), ("f32", 1e10)])
@pytest.mark.parametrize("B,NH,NKV,HD,P,scale", [
    (40, 8, 2, 64, 600, 0.125), (3, 4, 2, 64, 300, 0.125), (60, 8, 2, 128, 0, 0.09), (5, 100, 2, 128, 300, 0.09), (40, 8, 2, 64, 600, -0.125),
    (40, 8, 2, 128, 300, math.log(2.0))])
def test_attn_prefix_far_scores(cuda_dev, kind, size, B, NH, NKV, HD, P, scale):
    """Scores from 2^24 to far past 2^31: FP32 holds them to 2^-19 of what
    their products add up to (HD + 2 terms, truncated), so a row whose best
    score leads by 30 and twice that much is its value; lse is that score."""
    b = Batch(kind, NH, NKV, HD, P, [(i * 37) % 90 + 2 for i in range(B)], seed=3, peak=size)
    b.scale = scale
    out, lse = b.run()
    assert bool(torch.isfinite(out.float()).all()) and bool(torch.isfinite(lse).all())
    G, clear = NH // NKV, 0
    for r in range(B):
        k, v = (torch.cat([x[b.places[-1]], x[b.places[r]]]).double().transpose(0, 1) for x in (b.k, b.v))
        q = b.q[r].double().view(NKV, G, HD)
        s = torch.einsum("hgd,hkd->hgk", q, k) * scale
        off = 2.0 ** -19 * abs(scale) * torch.einsum("hgd,hkd->hgk", q.abs(), k.abs()).amax(-1)
        two = torch.topk(s, 2, -1)
        ok = two.values[..., 0] - two.values[..., 1] > 30 + 2 * off
        want = torch.gather(v[:, None].expand(-1, G, -1, -1), 2, two.indices[..., :1, None].expand(-1, -1, 1, HD))[:, :, 0]
        got = out[r].double().view(NKV, G, HD)
        assert bool(((got - want).abs()[ok] <= 2.0 ** -20 * want.abs()[ok]).all())  # the weight 1, and its own division
        assert bool(((lse[r].double().view(NKV, G) - two.values[..., 0]).abs()[ok] <= off[ok] + 2.0 ** -22 * two.values[..., 0].abs()[ok]).all())
        clear += int(ok.sum())
    assert clear > 0.9 * B * NH


@pytest.mark.parametrize("kind", KINDS)
def test_attn_prefix_missing_pages(cuda_dev, kind):
    """A page number outside the pool: its positions are skipped, as if they
    were not there; a request whose pages are all missing sees the prefix."""
    _missing_pages(Batch(kind, 6, 2, 64, 100, [70, 40, 33], page=16, seed=5))
    _missing_pages(Batch(kind, 100, 2, 64, 100, [70, 40, 33], page=16, seed=6))  # 150 rows a key head


def _missing_pages(b):
    missing = [(0, 1), (1, 0), (1, 1), (1, 2), (2, 2)]
    for r, j in missing:
        keep = b.places[r][0] != int(b.table[r, j])
        b.places[r] = (b.places[r][0][keep], b.places[r][1][keep])
        b.table[r, j] = [-1, 10 ** 6, -2 ** 31, b.k.shape[0], -1][(r + j) % 5]
    b.ptable[2] = -1
    i = torch.arange(100, device="cuda")
    b.places[-1] = tuple(x[i // 16 != 2] for x in b.places[-1])
    lens, P = b.lens, b.P
    got = b.run()
    b.lens, b.P = [len(p[0]) for p in b.places[:-1]], len(b.places[-1][0])
    want = b.want()
    b.lens, b.P = lens, P
    b.check(got=got, want=want)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("NH,NKV,HD,rows,page", [(4, 2, 64, 1, 16), (8, 2, 128, 1, 32), (12, 2, 64, 2, 8), (4, 2, 128, 6, 64)])
def test_attn_prefix_missing_pages_among_many(cuda_dev, kind, NH, NKV, HD, rows, page):
    """Enough keys that whole pages come by boxes, with pages missing all
    along: tiles that are copied otherwise and boxes take the same places in
    turn."""
    B = 40
    b = Batch(kind, NH, NKV, HD, 700, [1000 + 13 * i for i in range(B)], rows=[rows] * B, page=page, seed=47)
    gone = torch.rand(b.table.shape, generator=torch.Generator().manual_seed(5)) < 0.2
    lens = list(b.lens)
    for r in range(B):
        j = torch.arange(lens[r], device="cuda") // page
        gone[r, int(j[-rows]):] = False  # the rows' own positions, so that their limits cut what is there
        keep = ~gone[r].cuda()[j]
        b.places[r] = tuple(x[keep] for x in b.places[r])
        b.table[r][gone[r].cuda()] = -1
    first = torch.arange(b.ptable.numel(), device="cuda")
    b.ptable[first % 4 == 1] = -1
    at = torch.arange(700, device="cuda")
    b.places[-1] = tuple(x[at // page % 4 != 1] for x in b.places[-1])
    got = b.run()
    b.lens, b.P = [len(p[0]) for p in b.places[:-1]], len(b.places[-1][0])
    b.check(got=got, want=b.want())


@pytest.mark.parametrize("kind", KINDS)
def test_attn_prefix_only_one_side(cuda_dev, kind):
    """No own positions at all (max_kv 0), or no prefix: the other side's
    arguments may be absent; nothing on both sides gives zeros."""
    b = Batch(kind, 4, 2, 64, 333, [0, 0], seed=7)
    want = b.want()
    out, lse = torch.full_like(b.q, 7.0), torch.full((2, 4), 7.0, device="cuda")
    ws = torch.empty(sb200.attn_prefix_ws(b.q, b.kv, 333, 2), dtype=torch.uint8, device="cuda")
    sb200.attn_prefix(b.q, out, b.kv, b.ptable, 333, None, None, None, b.scale, ws, lse=lse, stream=stream())
    b.check(got=(out, lse), want=want)
    c = Batch(kind, 4, 2, 64, 0, [90, 31], seed=8)
    out, lse = torch.full_like(c.q, 7.0), torch.full((2, 4), 7.0, device="cuda")
    ws = torch.empty(sb200.attn_prefix_ws(c.q, c.kv, 0, 2, max_kv=90), dtype=torch.uint8, device="cuda")
    sb200.attn_prefix(c.q, out, None, None, 0, c.kv, c.table, c.kv_len, c.scale, ws, max_kv=90, lse=lse, stream=stream())
    c.check(got=(out, lse))
    sb200.attn_prefix(c.q, out, c.kv, None, 0, c.kv, None, None, c.scale, None, lse=lse, stream=stream())
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    for one in (dict(prefix=c.kv, kv=None), dict(prefix=None, kv=c.kv)):  # one of the pools says the type; a row behind the last request
        out, lse = torch.full_like(c.q, 7.0), torch.full((2, 4), 7.0, device="cuda")
        sb200.attn_prefix(c.q, out, prefix_table=None, prefix_len=0, table=None, kv_len=None, scale=c.scale, ws=None, cu_q=i32([0, 1]),
                          lse=lse, stream=stream(), **one)
        assert bool((out[0] == 0).all()) and bool((lse[0] == -math.inf).all())
        assert bool((out[1] == 7).all()) and bool((lse[1] == 7).all())


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_attn_prefix_strides_and_lengths(cuda_dev, kind):
    """Query and output rows inside wider ones, keys and values side by side,
    pages in order (no prefix table), negative and too long lengths."""
    t, g = DT[kind], torch.Generator("cuda").manual_seed(9)
    NH, NKV, HD, page, P, lens = 4, 2, 64, 16, 40, [20, 16]
    b = Batch(kind, NH, NKV, HD, P, lens, page=page, seed=9)
    pool = torch.full((8, NKV, page, 2, HD), float("nan"), dtype=t, device="cuda").permute(0, 2, 1, 3, 4)
    k, v = pool[..., 0, :], pool[..., 1, :]
    table, at = i32([[5, 3, 10 ** 6], [6, 4, 7]]), 0
    for r, n in list(enumerate(lens)) + [(-1, P)]:
        i = torch.arange(n, device="cuda")
        pg = table[r][i // page].long() if r >= 0 else i // page
        k[pg, i % page], v[pg, i % page] = b.k[b.places[r]], b.v[b.places[r]]
    wide = torch.full((2, NH + 3, HD + 8), 7.0, dtype=t, device="cuda")
    q, out = wide[:, :NH, :HD], torch.full((2, NH + 1, HD), 7.0, dtype=t, device="cuda")
    q.copy_(b.q)
    kv = sb200.KvPages(k, v)
    ws = torch.empty(sb200.attn_prefix_ws(q, kv, P, 2, max_kv=20), dtype=torch.uint8, device="cuda")
    lse = torch.full((2, NH), 7.0, device="cuda")
    # request 0's length is cut to max_kv = 20, as the 20 that it has
    sb200.attn_prefix(q, out[:, :NH], kv, None, P, kv, table, i32([10 ** 9, 16]), b.scale, ws, max_kv=20, lse=lse, stream=stream())
    b.check(got=(out[:, :NH], lse))
    assert bool((out[:, NH:] == 7).all())
    sb200.attn_prefix(q, out[:, :NH], kv, None, P, kv, table, i32([-3, 16]), b.scale, ws, max_kv=20, lse=lse, stream=stream())
    b.lens = [0, 16]
    b.places[0] = tuple(x[:0] for x in b.places[0])
    b.check(got=(out[:, :NH], lse))


def test_attn_prefix_offsets_past_32_bits(cuda_dev):
    """Pages whose elements lie past 2^32 bytes and 2^31 elements."""
    free, _ = torch.cuda.mem_get_info()
    if free < 24 << 30:
        pytest.skip("needs 24 GB of device memory")
    NKV, HD, page = 2, 64, 16
    big = torch.empty(2, 2_200_000_000, dtype=torch.float16, device="cuda")
    stride = 2_200_000_000 // 4 // 8 * 8
    k, v = (x.as_strided((4, page, NKV, HD), (stride, NKV * HD, HD, 1)) for x in big)
    b = Batch("f16", 4, NKV, HD, 20, [30], page=page, seed=11)
    table = i32([[3, 2, -1]])
    for r, n in ((0, 30), (-1, 20)):
        i = torch.arange(n, device="cuda")
        pg = table[0][i // page].long() if r == 0 else i32([3, 1])[i // page].long()
        at = i % page
        if r:
            pg, at = i32([1, 0])[i // page].long(), at
        k[pg, at], v[pg, at] = b.k[b.places[r]], b.v[b.places[r]]
    kv, lse = sb200.KvPages(k, v), torch.empty(1, 4, device="cuda")
    out, ws = torch.empty_like(b.q), torch.empty(sb200.attn_prefix_ws(b.q, kv, 20, 1, max_kv=30), dtype=torch.uint8, device="cuda")
    sb200.attn_prefix(b.q, out, kv, i32([1, 0]), 20, kv, table, b.kv_len, b.scale, ws, max_kv=30, lse=lse, stream=stream())
    b.check(got=(out, lse))


@pytest.mark.parametrize("kind", KINDS)
def test_attn_prefix_repeats_and_replays(cuda_dev, kind):
    """The same bits on every run (no sums in an order of arrival), on another
    stream, and from a captured graph whose lengths change between replays."""
    lens = [50, 0, 200, 31]
    b = Batch(kind, 14, 2, 64, 1000, lens, rows=[2, 1, 4, 3], page=16, seed=13)
    out, lse = b.run()
    ws = torch.empty(sb200.attn_prefix_ws(b.q, b.kv, 1000, 4, max_q=4, max_kv=200), dtype=torch.uint8, device="cuda")
    o2, l2 = torch.zeros_like(out), torch.zeros_like(lse)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            b.run(out=o2, lse=l2, ws=ws)
    side.synchronize()
    assert torch.equal(out, o2) and torch.equal(lse, l2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.run(out=o2, lse=l2, ws=ws)
    for change in ([20, 0, 200, 31], [50, 0, 3, 0]):
        b.kv_len.copy_(i32(change))
        o2.fill_(9)
        graph.replay()
        places, was = list(b.places), b.lens
        b.lens, b.places = change, [tuple(x[:n] for x in p) for p, n in zip(places, change)] + [places[-1]]
        want = b.want()
        b.lens, b.places = was, places
        b.check(got=(o2, l2), want=want)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("NH,NKV,HD,page,P", [
    (4, 1, 128, 16, 130),   # a row group of 4: the 8-row tiles
    (12, 1, 64, 8, 130),    # of 12: the 16-row tiles, two pages a warp's tile
    (1, 1, 24, 32, 0),      # a head of a fifth of a box, one row
    (2, 1, 72, 64, 40),     # half the second box
    (3, 1, 96, 24, 40),     # pages that only an 8-position box divides
    (16, 1, 128, 128, 0),
])
def test_attn_prefix_many_own_keys(cuda_dev, kind, NH, NKV, HD, page, P):
    """Enough keys that whole pages come as boxes; ends inside a page, pages
    that are not there between ones that are, other rows behind the last."""
    lens = [(i * 211) % 1100 + (i % 3 == 0) * 16 for i in range(36)]
    b = Batch(kind, NH, NKV, HD, P, lens, page=page, seed=HD + page, pad=1)
    b.lens = lens = [max(lens)] + lens[1:]
    b.kv_len = i32(lens)
    drop = [(r, j) for r in (1, 2, 5) for j in (0, 3) if j * page < lens[r]]
    # request 0 claims as many positions as the longest, its table has pages outside the pool for all
    b.table[0] = 10 ** 9
    b.places[0] = tuple(x[:0] for x in b.places[0])
    for r, j in drop:
        keep = b.places[r][0] != int(b.table[r, j])
        b.places[r] = tuple(x[keep] for x in b.places[r])
        b.table[r, j] = -1
    got = b.run()
    b.lens = [len(p[0]) for p in b.places[:-1]]
    b.check(got=got)
    assert sb200.tc_error() == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("B,NH,NKV,HD", [(3, 4, 2, 64), (70, 8, 2, 128), (300, 2, 2, 64)])
def test_attn_prefix_pools_of_their_own(cuda_dev, kind, B, NH, NKV, HD):
    """Prefix and requests in pools of different page sizes and layouts."""
    lens = [(i * 29) % 150 for i in range(B)]
    b = Batch(kind, NH, NKV, HD, 500, lens, page=16, seed=B)
    page, pp = 48, 11  # 500 positions in 11 pages of 48, heads outside
    pool = torch.full((2, pp + 2, NKV, page, HD), float("nan"), dtype=b.t, device="cuda").transpose(2, 3)
    table, i = torch.randperm(pp + 2, device="cuda")[:pp].to(torch.int32), torch.arange(500, device="cuda")
    for x, y in zip(pool, (b.k, b.v)):
        x[table[i // page].long(), i % page] = y[b.places[-1]]
    kv = sb200.KvPages(pool[0], pool[1])
    out, lse = torch.full_like(b.q, 7.0), torch.full((B, NH), 7.0, device="cuda")
    ws = torch.full((sb200.attn_prefix_ws(b.q, kv, 500, B, max_kv=max(lens)) // 4 + 1,), float("nan"), device="cuda")
    sb200.attn_prefix(b.q, out, kv, table, 500, b.kv, b.table, b.kv_len, b.scale, ws, max_kv=max(lens), lse=lse, stream=stream())
    b.check(got=(out, lse))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("B", [3, 40])
def test_attn_prefix_scale_of_zero(cuda_dev, kind, B):
    """All keys alike: the mean of what a row sees, also where a tile's end is masked."""
    b = Batch(kind, 8, 2, 64, 200, [(i * 7) % 40 for i in range(B)], seed=21)
    b.scale = 0.0
    b.check()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_attn_prefix_two_at_once(cuda_dev, kind):
    """Two streams, then two captured graphs side by side, each call with its
    own workspace and outputs: the bits of one alone."""
    bs = [Batch(kind, 8, 2, 64, 900, [(i * 31) % (90 + s) for i in range(40)], seed=s) for s in (31, 32)]
    alone = [b.run() for b in bs]
    torch.cuda.synchronize()
    outs = [(torch.zeros_like(o), torch.zeros_like(x)) for o, x in alone]
    wss = [torch.empty(sb200.attn_prefix_ws(b.q, b.kv, 900, 40, max_kv=max(b.lens)), dtype=torch.uint8, device="cuda") for b in bs]
    streams = [torch.cuda.Stream() for _ in bs]
    graphs = []

    def both():
        for b, s, o, w in zip(bs, streams, outs, wss):
            with torch.cuda.stream(s):
                for _ in range(4):
                    b.run(out=o[0], lse=o[1], ws=w)
    both()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for a, o in zip(alone, outs) for x, y in zip(a, o))
    for b, s, o, w in zip(bs, streams, outs, wss):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=s):
            b.run(out=o[0], lse=o[1], ws=w)
        o[0].zero_()
    torch.cuda.synchronize()
    for _ in range(4):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for a, o in zip(alone, outs) for x, y in zip(a, o))


def test_attn_prefix_workspace_too_small(cuda_dev):
    b = Batch("f16", 14, 2, 64, 1000, [50, 20])
    n = sb200.attn_prefix_ws(b.q, b.kv, 1000, 2, max_kv=50)
    assert n > 0
    for ws in (None, torch.empty(n - 1, dtype=torch.uint8, device="cuda"), torch.empty(n + 17, dtype=torch.uint8, device="cuda")[16:]):
        with pytest.raises(sb200.SbError, match="workspace"):
            sb200.attn_prefix(b.q, torch.empty_like(b.q), b.kv, b.ptable, 1000, b.kv, b.table, b.kv_len, b.scale, ws, max_kv=50)


@pytest.mark.parametrize("kind", KINDS)
def test_attn_prefix_one_workspace_for_several_sizes(cuda_dev, kind):
    """The largest answer among the sizes that run serves them all, in any
    order."""
    sizes = [(70, 900, 200), (64, 900, 200), (8, 900, 200), (1, 900, 1500), (40, 0, 1500), (64, 900, 30), (3, 40, 3)]
    bs = [Batch(kind, 16, 4, 128, P, [(i * 31) % S + 1 for i in range(B)], seed=B) for B, P, S in sizes]
    most = max(sb200.attn_prefix_ws(b.q, b.kv, b.P, len(b.lens), max_kv=max(b.lens)) for b in bs)
    ws = torch.full((most,), 0xFF, dtype=torch.uint8, device="cuda")
    for b in bs + bs[::-1]:
        b.check(got=b.run(ws=ws))


@pytest.mark.parametrize("kind,NH,NKV,HD,B,P,S,page,skip", [
    ("f32", 4, 2, 64, 60, 0, 900, 16, 1),       # decode rows, boxes
    ("f32", 8, 1, 128, 5, 0, 90, 24, 0),        # the lanes' copies
    ("f16", 8, 2, 64, 60, 0, 900, 16, 1),
    ("bf16", 8, 2, 128, 60, 0, 900, 32, 1),
    ("f16", 12, 1, 64, 60, 0, 900, 16, 1),      # 16 rows
    ("bf16", 8, 2, 128, 40, 16000, 0, 64, 1),   # the prefix on tcgen05, boxes
    ("f16", 8, 2, 64, 40, 16000, 0, 24, 0)])    # and the loaders' copies
def test_attn_prefix_wait_timeout_recovers(cuda_dev, kind, NH, NKV, HD, B, P, S, page, skip):
    """Failure detection without a GPU fault: the test hook makes the loaders
    of keys stop before a tile, the bounded wait for it runs out, what was
    asked for drains, and the rows are NaN.  The next call with the hook off
    is right before the flag is read, and the flag is there once."""
    b = Batch(kind, NH, NKV, HD, P, [S] * B, page=page, seed=51)
    assert sb200.tc_error() == 0
    sb200.check(sb200.lib().sb_attn_set_test_skip(skip))
    try:
        t0 = time.time()
        out, lse = b.run(own=S > 0)
        torch.cuda.synchronize()
        assert time.time() - t0 < 30
    finally:
        sb200.check(sb200.lib().sb_attn_set_test_skip(-1))
    assert bool(torch.isnan(out.float()).all()) and bool(torch.isnan(lse).all())
    b.check(got=b.run(own=S > 0))
    assert sb200.tc_error() != 0
    assert sb200.tc_error() == 0
    b.check(got=b.run(own=S > 0))


def test_attn_prefix_wait_timeout_with_rows_left(cuda_dev):
    """More rows than the launch was sized for: a CTA that gave up at its
    first rows takes the others up no more, and all are NaN."""
    b = Batch("f16", 14, 2, 64, 0, [900] * 20, rows=[4] * 20, seed=52)
    sb200.check(sb200.lib().sb_attn_set_test_skip(1))
    try:
        out, lse = b.run(max_q=1)
        torch.cuda.synchronize()
    finally:
        sb200.check(sb200.lib().sb_attn_set_test_skip(-1))
    assert sb200.tc_error() != 0
    assert bool(torch.isnan(out.float()).all()) and bool(torch.isnan(lse).all())
    b.check(got=b.run(max_q=1))
    assert sb200.tc_error() == 0


def test_attn_prefix_reads_an_engine_cache(cuda_dev, qwen_weights):
    """A prompt that an engine has prefilled, as the shared prefix of a batch:
    the same attention as the single-sequence kernel on the same cache."""
    Q = sb200.QWEN
    eng = sb200.Engine(sb200.MODEL_QWEN, qwen_weights, 256)
    ids = sb200.synth_ids(100, Q["V"], 3)
    eng.begin(ids, 1)
    eng.prefill(99)
    ptr, nbytes, NL, ctx, width = eng.kv_cache()
    torch.cuda.synchronize()

    class Memory:
        __cuda_array_interface__ = {"shape": (2, NL, ctx // 16, 16, 2, 64), "typestr": "<f4", "data": (ptr, False), "version": 3}
    cache = torch.as_tensor(Memory(), device="cuda")
    for layer in (0, 23):
        kv = sb200.KvPages(cache[0, layer], cache[1, layer])
        g = torch.Generator("cuda").manual_seed(layer)
        q = torch.randn(5, 14, 64, device="cuda", generator=g)
        out = torch.empty_like(q)
        ws = torch.empty(sb200.attn_prefix_ws(q, kv, 99, 5), dtype=torch.uint8, device="cuda")
        sb200.attn_prefix(q, out, kv, None, 99, None, None, None, 0.125, ws, stream=stream())
        part, tickets = torch.zeros(2 * 7 * 7 * 66, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
        one = torch.empty(14 * 64, device="cuda")
        for r in range(5):
            sb200.attn_decode(q[r].contiguous(), cache[0, layer], cache[1, layer], one, 99, 14, 2, 64, 128, 0.125, part, tickets)
            torch.testing.assert_close(out[r].flatten(), one, rtol=1e-5, atol=2e-6)
    eng.close()
