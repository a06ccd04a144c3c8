"""Log probabilities, entropy, rank, alternatives and their gradient on the
GPU against plain implementations in 64 bits, and a serving step of all batch
operators together."""
import math

import numpy as np
import pytest
import torch

import sb200

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def stream():
    return torch.cuda.current_stream()


def run(x, tok, k=0, temperature=1.0):
    R, V = x.shape
    got = {n: torch.full((R,), 77.0, device="cuda") for n in ("logp", "entropy", "lse")}
    got["rank"] = torch.full((R,), 77, dtype=torch.int32, device="cuda")
    top = {}
    if k:
        top = dict(top_ids=torch.full((R, k), 77, dtype=torch.int32, device="cuda"), top_logp=torch.full((R, k), 77.0, device="cuda"))
    ws = torch.full((sb200.logprobs_ws(x, k),), 0xFF, dtype=torch.uint8, device="cuda")
    sb200.logprobs(x, tok, ws, temperature=temperature, stream=stream(), **got, **top)
    return got | top


def reference(x, tok, k, temperature):
    y = x.double() / temperature
    lse = torch.logsumexp(y, -1)
    none = lse == -math.inf
    logs = y - lse[:, None]
    p = torch.exp(logs)
    entropy = -torch.where(p > 0, p * logs, torch.zeros_like(p)).sum(-1)
    V = x.shape[1]
    given = (tok >= 0) & (tok < V)
    at = tok.long().clamp(0, V - 1)[:, None]
    mine, ids = x.float().gather(1, at), torch.arange(V, device="cuda")
    logp = torch.where(none, torch.full_like(lse, -math.inf), logs.gather(1, at)[:, 0])
    rank = ((x.float() > mine) | ((x.float() == mine) & (ids < at))).sum(-1)
    order = torch.sort(x.float() + 0.0, dim=-1, descending=True, stable=True).indices[:, :k]
    listed = x.float().gather(1, order) > -math.inf
    inf = torch.full_like(order, 1).double() * -math.inf
    return dict(lse=lse, entropy=torch.where(none, torch.zeros_like(lse), entropy), logp=torch.where(given, logp, torch.zeros_like(lse)),
                rank=torch.where(given, rank, torch.full_like(rank, -1)), top_ids=torch.where(listed, order, torch.full_like(order, -1)),
                top_logp=torch.where(listed, logs.gather(1, order), inf))


def check(x, tok, k, temperature=1.0):
    """lse: its sum is off by (V / 256 + 16) half steps of FP32 in the longest
    chain, 2^-22 of each exponential and the products' half step of |x| /
    temperature; logp the same, entropy the same times ln V (its terms)."""
    got, want = run(x, tok, k, temperature), reference(x, tok, k, temperature)
    V = x.shape[1]
    big = torch.where(torch.isfinite(x), x, torch.zeros_like(x)).double().abs().amax(-1) / temperature
    bound = (V / 256 + 16) * 2.0 ** -24 + 2.0 ** -21 + 2.0 ** -22 * big
    for n in ("lse", "logp", "entropy", "top_logp"):
        if n not in got:
            continue
        a, b = got[n].double(), want[n]
        fin = torch.isfinite(b)
        assert torch.equal(a[~fin], b[~fin]), n
        lim = (bound if a.dim() == 1 else bound[:, None].expand_as(a)) * (1 + math.log(V) if n == "entropy" else 2)
        assert bool(((a - b).abs()[fin] <= lim[fin]).all()), (n, float((a - b).abs()[fin].max()))
    for n in ("rank", "top_ids"):
        if n in got:
            assert torch.equal(got[n].long(), want[n]), n
    return got


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("R,V,k,temperature,odd", [
    (1, 1, 1, 1.0, 0), (3, 5, 5, 0.5, 1), (2, 64, 64, 1.0, 3), (5, 1000, 20, 0.7, 1), (1, 151936, 20, 0.7, 0), (7, 50257, 5, 1.3, 0),
    (2, 151936, 64, 1.0, 5), (700, 777, 1, 1.0, 2), (40, 30001, 24, 1.0, 7), (33, 4099, 25, 2.0, 1), (1500, 129, 0, 1.0, 0), (4, 65536, 0, 1.0, 0)])
def test_logprobs(cuda_dev, kind, R, V, k, temperature, odd):
    g = torch.Generator("cuda").manual_seed(R + V)
    x = (torch.randn(R, V + odd, device="cuda", generator=g) * 3).to(DT[kind])[:, :V]  # odd: rows at any 2-byte place
    tok = torch.randint(0, V, (R,), device="cuda", generator=g).to(torch.int32)
    if R > 3:
        tok[1], tok[2] = -1, V
        x[3, V // 2:] = -math.inf
        tok[3] = V - 1  # a masked choice
    check(x, tok, k, temperature)


@pytest.mark.parametrize("kind", list(DT))
def test_logprobs_ties_and_orders(cuda_dev, kind):
    """Equal, rising and falling logits, signed zeros: the list is cut on the
    way, and equal values go by id."""
    V, t = 20011, DT[kind]
    ramp = torch.arange(V, device="cuda", dtype=torch.float32) / V * 8 - 4
    zero = torch.zeros(V, device="cuda")
    zero[1::2] = -0.0
    step = (torch.arange(V, device="cuda") // 100).float() / 16
    x = torch.stack([torch.full((V,), 2.5, device="cuda"), ramp, ramp.flip(0), zero, step, step.flip(0)]).to(t)
    tok = torch.tensor([V - 1, 0, 17, 4, 9000, V // 2], dtype=torch.int32, device="cuda")
    for k in (1, 24, 64):
        check(x, tok, k)
    for r in range(x.shape[0]):  # one row: cut into parts
        check(x[r: r + 1].contiguous(), tok[r: r + 1].contiguous(), 64)
    check(x.repeat(200, 1), tok.repeat(200), 64)  # many rows: a CTA a row


@pytest.mark.parametrize("R", [1, 1300])
def test_logprobs_masked_rows(cuda_dev, R):
    """Rows with no choice, one, and fewer than k."""
    V = 5000
    x = torch.full((R, V), -math.inf, device="cuda")
    tok = torch.zeros(R, dtype=torch.int32, device="cuda")
    check(x, tok, 20)
    x[:, V - 1] = 3.0
    check(x, tok, 20)
    got = check(x, tok + V - 1, 20)
    # the one choice's exponential 2^d, d = x c less its rounding, and its log2 are each off by at most 2^-22: ln p by 2^-21
    assert bool((got["logp"].abs() <= 2.0 ** -21).all()) and bool((got["entropy"].abs() <= 2.0 ** -21).all()) and bool((got["rank"] == 0).all())
    x[:, 100:110] = 3.0
    check(x, tok + 105, 20)


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("R", [1, 700])
def test_logprobs_lowest_value_masks(cuda_dev, kind, R):
    """Masks of the type's lowest value: weight 0 beside other choices; alone
    they are equal choices, and -inf beside them still has weight 0."""
    V, t = 3001, DT[kind]
    low = torch.finfo(t).min
    x = torch.full((R, V), low, dtype=t, device="cuda")
    tok = torch.full((R,), 2000, dtype=torch.int32, device="cuda")
    grad, one = torch.empty_like(x), torch.ones(R, device="cuda")
    for n, ids in ((V, [0, 1, 2, 3, 4]), (V - V // 2, [1500, 1501, 1502, 1503, 1504])):
        got = run(x, tok, 5)
        # equal choices: ln n to the FP32 sum's (n / 256 + 16) half steps and 2^-22 of the logarithm
        for name in ("logp", "entropy", "top_logp"):
            assert bool(((got[name].double().abs() - math.log(n)).abs() <= 2.0 ** -18).all()), name
        assert bool((got["top_ids"] == torch.tensor(ids, device="cuda")).all()) and bool((got["rank"] == 2000 - ids[0]).all())
        sb200.logprobs_grad(x, tok, got["lse"], got["entropy"], one, one, grad, stream=stream())
        # lse = lowest + ln n rounds to the lowest value itself: a probability there means nothing, but nothing is NaN
        assert not bool(torch.isnan(grad).any())
        x[:, : V // 2] = -math.inf
    x[:, 10] = 1.5
    x[:, 2999] = -0.5
    # two choices of size 1 are left
    want = reference(x, tok - 1990, 5, 1.0)
    got = run(x, tok - 1990, 5)
    for name in ("lse", "logp", "entropy"):
        assert bool(((got[name].double() - want[name]).abs() <= 2.0 ** -20).all()), name
    assert torch.equal(got["top_ids"].long(), want["top_ids"]) and torch.equal(got["rank"].long(), want["rank"])
    sb200.logprobs_grad(x, tok - 1990, got["lse"], got["entropy"], one, one, grad, stream=stream())
    want = gradient(x, tok - 1990, one, one, 1.0)
    # values of size 1, one rounding each and 2^-20 of the exponentials
    assert bool(((grad.double() - want).abs() <= torch.finfo(t).eps / 2 * want.abs() + 2.0 ** -19).all())


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("R", [1, 700])
@pytest.mark.parametrize("mask,temperature,offset", [
    (-1e9, 1.0, 0.0), (-1e10, 1.0, 0.0), (-3e15, 0.7, 0.0), (-9e29, 1.0, 0.0), (-9e29, 1e-8, 0.0), (-1e4, 1e-8, 0.0),
    (-6e4, 1e-8, 20.0), (-6e4, 3e-5, 20.0), (-6e4, 1e-6, -20.0), (-1e30, 1.0, 7e5), (-1e30, 1.0, 7.5e5), (0.0, 1.0, 3e10)])
def test_logprobs_large_products(cuda_dev, kind, R, mask, temperature, offset):
    """Maxima whose product with 1 / temperature has no bits left for the
    choices (masks of -1e10 that fill a thread's share of the row, tiny
    temperatures, offsets): as exact as without them."""
    V, k, t = 9001, 5, DT[kind]
    if max(abs(mask), abs(offset)) > torch.finfo(t).max:
        pytest.skip("not a value of this type")
    g = torch.Generator("cuda").manual_seed(V)
    # steps of a type's last place around the offset, apart by some units of the temperature
    step = max(abs(offset) * torch.finfo(t).eps, 2 * temperature)
    x = (offset + step * torch.randint(-6, 1, (R, V), device="cuda", generator=g)).to(t)
    x[0, : V // 2] = mask
    x[-1, V // 3: V // 3 * 2] = mask
    if R > 1:
        x[1] = mask  # every choice
        x[2, ::2] = mask
    tok = torch.randint(0, V, (R,), device="cuda", generator=g).to(torch.int32)
    got = run(x, tok, k, temperature)
    top = x.amax(-1).double()  # differences to it, as a quotient of 1e30 holds no ln V in 64 bits either
    y = (x.double() - top[:, None]) / temperature
    want = reference(y, tok, k, 1.0) | {n: w for n, w in reference(x, tok, k, 1.0).items() if n in ("rank", "top_ids")}
    low = want["lse"].clone()
    want["lse"] += top / temperature
    base = (V / 256 + 16) * 2.0 ** -24 + 2.0 ** -21
    spread = -y.gather(1, tok.long()[:, None])[:, 0]
    seen = torch.where(low[:, None] - y < 700, -y, torch.zeros_like(y)).amax(-1)
    lim = dict(lse=base + 2.0 ** -22 * want["lse"].abs(), logp=2 * base + 2.0 ** -21 * (spread + math.log(V)),
               entropy=(2 * base + 2.0 ** -21 * (seen + 1)) * (1 + math.log(V)),
               top_logp=(torch.full_like(low, 2 * base + 2.0 ** -21 * (math.log(V) + 1)))[:, None] + 2.0 ** -21 * want["top_logp"].abs())
    for n, b in lim.items():
        err = (got[n].double() - want[n]).abs()
        # finite values whose quotient passes FP32 are -inf there
        big = want[n].abs() > 3.4e38
        assert bool((err <= b)[~big].all()), (n, float((err / b)[~big].max()))
        assert bool((got[n][big].abs() > 3.4e38).all()), n
    for n in ("rank", "top_ids"):
        assert torch.equal(got[n].long(), want[n]), n


def test_logprobs_nan_and_inf(cuda_dev):
    """A NaN or +inf makes its own row's sums NaN, no other row's."""
    x = torch.randn(6, 3001, device="cuda")
    tok = torch.arange(6, dtype=torch.int32, device="cuda")
    clean = run(x, tok, 5)
    x[1, 2000], x[4, 7] = math.nan, math.inf
    got = run(x, tok, 5)
    for n in ("lse", "logp", "entropy"):
        assert torch.isnan(got[n][[1, 4]]).all(), n
        assert torch.equal(got[n][[0, 2, 3, 5]], clean[n][[0, 2, 3, 5]]), n
    assert torch.equal(got["top_ids"][[0, 2, 3, 5]], clean["top_ids"][[0, 2, 3, 5]])


def test_logprobs_some_outputs(cuda_dev):
    """Any output may be absent; without tokens lse, entropy and the
    alternatives remain."""
    x = torch.randn(3, 40000, device="cuda")
    full = run(x, torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda"), 7)
    ws = torch.empty(sb200.logprobs_ws(x, 7), dtype=torch.uint8, device="cuda")
    lse, ids = torch.empty(3, device="cuda"), torch.empty(3, 7, dtype=torch.int32, device="cuda")
    sb200.logprobs(x, None, ws, lse=lse, stream=stream())
    sb200.logprobs(x, None, ws, top_ids=ids, stream=stream())
    assert torch.allclose(lse, full["lse"], rtol=1e-6) and torch.equal(ids, full["top_ids"])
    with pytest.raises(sb200.SbError, match="workspace"):
        sb200.logprobs(x, None, None, lse=lse)
    with pytest.raises(sb200.SbError, match="tokens"):
        sb200.logprobs(x, None, ws, logp=lse)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_logprobs_workspace_for_smaller_batches(cuda_dev, kind):
    """One workspace, asked for at the largest sizes, for every smaller batch,
    vocabulary and number of alternatives (fewer rows are cut into more
    parts)."""
    g = torch.Generator("cuda").manual_seed(2)
    x = torch.randn(1300, 20001, device="cuda", generator=g).to(DT[kind])
    tok = torch.randint(0, 3000, (1300,), device="cuda", generator=g).to(torch.int32)
    ws = torch.full((sb200.logprobs_ws(x, 20),), 0xFF, dtype=torch.uint8, device="cuda")
    for R, V, k in ((1300, 20001, 20), (592, 20001, 20), (591, 20001, 20), (300, 20001, 20), (149, 20001, 20), (7, 20001, 20), (1, 20001, 20),
                    (40, 3000, 20), (591, 9000, 5), (3, 20001, 1)):
        assert sb200.logprobs_ws(x[:R, :V], k) <= ws.numel()
        want = run(x[:R, :V], tok[:R], k)
        got = {n: torch.zeros_like(v) for n, v in want.items()}
        sb200.logprobs(x[:R, :V], tok[:R], ws, stream=stream(), **got)
        assert all(torch.equal(got[n], want[n]) for n in got), (R, V, k)


def gradient(x, tok, gl, ge, temperature):
    y = x.double() / temperature
    logs = torch.log_softmax(y, -1)
    p = torch.exp(logs)
    plogp = torch.where(p > 0, p * logs, torch.zeros_like(p))
    h = -plogp.sum(-1, keepdim=True)
    V = x.shape[1]
    given = (tok >= 0) & (tok < V)
    gl = torch.where(given, gl.double(), torch.zeros_like(gl.double()))[:, None]
    hot = torch.zeros_like(p).scatter_(1, tok.long().clamp(0, V - 1)[:, None], gl)
    return (hot - gl * p - ge.double()[:, None] * (plogp + p * h)) / temperature


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("R,V,temperature,odd", [(1, 1, 1.0, 0), (3, 129, 0.7, 1), (2, 151936, 1.0, 0), (300, 5001, 1.4, 0), (17, 50257, 1.0, 4)])
def test_logprobs_gradient(cuda_dev, kind, R, V, temperature, odd):
    """Against the formula: p is off by what lse is off (check() above; half a
    step of FP32 of lse itself) and 2^-22 of the exponential, then one
    rounding to the type."""
    g = torch.Generator("cuda").manual_seed(V)
    t = DT[kind]
    x = (torch.randn(R, V + odd, device="cuda", generator=g) * 2).to(t)[:, :V]
    tok = torch.randint(0, V, (R,), device="cuda", generator=g).to(torch.int32)
    if R > 2:
        tok[1] = -1
        x[2, : V // 2] = -math.inf
    gl, ge = (torch.randn(R, device="cuda", generator=g) for _ in range(2))
    f = run(x, tok, 0, temperature)
    want = gradient(x, tok, gl, ge, temperature)
    big = torch.where(torch.isfinite(x), x, torch.zeros_like(x)).double().abs().amax(-1) / temperature
    rel = (V / 256 + 16) * 2.0 ** -24 + 2.0 ** -20 + 2.0 ** -21 * (big + math.log(V) + 1)
    p = torch.softmax(x.double() / temperature, -1)
    size = p * (gl.double().abs()[:, None] + ge.double().abs()[:, None] * (2 * math.log(V) + 2 * big[:, None] + 2)) / temperature
    hot = torch.zeros_like(p).scatter_(1, tok.long().clamp(0, V - 1)[:, None], gl.double().abs()[:, None] / temperature)
    bound = rel[:, None] * size + 2.0 ** -23 * hot + torch.finfo(t).eps / 2 * want.abs() + (2.0 ** -25 if t == torch.float16 else 1e-37)
    same = torch.empty(R, V + odd, dtype=t, device="cuda")[:, :V]     # rows placed as the logits'
    other = torch.empty(R, V + 1 - odd % 2, dtype=t, device="cuda")[:, :V]  # and not
    for grad in (same, other):
        grad.fill_(7)
        sb200.logprobs_grad(x, tok, f["lse"], f["entropy"], gl, ge, grad, temperature=temperature, stream=stream())
        err = (grad.double() - want).abs()
        assert bool((err <= bound).all()), float((err / bound).max())
    z = x.clone() if odd == 0 else x
    sb200.logprobs_grad(z, tok, f["lse"], f["entropy"], gl, ge, z, temperature=temperature, stream=stream())
    assert torch.equal(z, same)  # in place


def test_logprobs_gradient_against_differences(cuda_dev):
    """Central differences of the forward call: with h = 2^-5 their own error
    is h^2 / 6 of a third derivative below 2, the sums' rounding 2^-20 / h."""
    R, V, h = 2, 37, 2.0 ** -5
    g = torch.Generator("cuda").manual_seed(1)
    x = torch.randn(R, V, device="cuda", generator=g)
    tok = torch.tensor([3, 30], dtype=torch.int32, device="cuda")
    gl, ge = torch.tensor([1.0, -0.5], device="cuda"), torch.tensor([0.7, 1.0], device="cuda")
    f, grad = run(x, tok, 0, 0.8), torch.empty_like(x)
    sb200.logprobs_grad(x, tok, f["lse"], f["entropy"], gl, ge, grad, temperature=0.8, stream=stream())
    for v in (0, 3, 17, 30, 36):
        vals = []
        for s in (h, -h):
            z = x.clone()
            z[:, v] += s
            r = run(z, tok, 0, 0.8)
            vals.append((gl * r["logp"]).double() + (ge * r["entropy"]).double())
        diff = (vals[0] - vals[1]) / (2 * h)
        assert bool(((diff - grad[:, v].double()).abs() < h * h / 6 * 2 / 0.8 ** 3 * 1.7 + 2.0 ** -20 / h).all())


def test_logprobs_gradient_parts(cuda_dev):
    """One weight alone, none, and a row of masked choices."""
    x = torch.randn(3, 1000, device="cuda")
    x[1] = -math.inf
    tok = torch.tensor([5, 6, 7], dtype=torch.int32, device="cuda")
    f = run(x, tok)
    w = torch.tensor([1.0, 2.0, -3.0], device="cuda")
    both, a, b, none = (torch.empty_like(x) for _ in range(4))
    call = lambda gl, ge, out: sb200.logprobs_grad(x, tok, f["lse"], f["entropy"], gl, ge, out, stream=stream())  # noqa: E731
    call(w, w, both), call(w, None, a), call(None, w, b), call(None, None, none)
    assert bool((both[1] == 0).all()) and bool((a[1] == 0).all()) and bool((b[1] == 0).all()) and bool((none == 0).all())
    # two values of each size, each sum rounded once, the exponents' 2^-20 apart
    assert bool(((both - a - b).abs() <= 2.0 ** -19 * (a.abs() + b.abs()) + 1e-9).all())


def gradient_bound(x, gl, ge, temperature, want, tok):
    """As in test_logprobs_gradient, with the choices' spread instead of their
    size: c (x - m) is rounded relative to itself and the product of the
    maximum is the same in every term."""
    y, V = x.double() / temperature, x.shape[1]
    p = torch.softmax(y, -1)
    seen = p > 0
    top = y.amax(-1)
    spread = torch.where(seen, top[:, None] - y, torch.zeros_like(y)).amax(-1)
    rel = (V / 256 + 16) * 2.0 ** -24 + 2.0 ** -20 + 2.0 ** -21 * (spread + math.log(V) + 1)
    size = p * (gl.double().abs()[:, None] + ge.double().abs()[:, None] * (2 * math.log(V) + 2 * spread[:, None] + 2)) / temperature
    hot = torch.zeros_like(p).scatter_(1, tok.long()[:, None], gl.double().abs()[:, None] / temperature)
    least = {torch.float16: 2.0 ** -25, torch.float32: 1e-37, torch.bfloat16: 1e-37}[x.dtype]
    # a power of two below 2^-126 is flushed to 0: there the whole value is missing, p times the same factor
    flushed = 2.0 ** -126 * (gl.double().abs() + ge.double().abs() * (2 * math.log(V) + 2 * spread + 2)) / temperature
    return rel[:, None] * size + flushed[:, None] + 2.0 ** -23 * hot + torch.finfo(x.dtype).eps / 2 * want.abs() + least


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("mask,temperature,weight", [(-9e29, 1e-4, 4.0), (-1e22, 1e-8, 1.0), (-9e29, 1.0, 1e10), (-1e4, 1.0, 1.0), (-9e29, 1e-8, 1e-3)])
def test_logprobs_gradient_large_finite_masks(cuda_dev, kind, mask, temperature, weight):
    """Masks far below the choices, between the type's lowest value and
    ordinary logits: their probability is 0, and so is their gradient, also
    where the entropy's weight times the exponent passes FP32."""
    R, V, t = 3, 20001, DT[kind]
    g = torch.Generator("cuda").manual_seed(3)
    x = (torch.randn(R, V, device="cuda", generator=g) * 2 * temperature).to(t)
    x[0, : V // 2] = mask
    x[1, V // 3:] = mask
    x[2, ::2] = mask
    tok = torch.tensor([V - 1, 5, 7], dtype=torch.int32, device="cuda")
    gl, ge = torch.tensor([1.0, -0.5, 0.25], device="cuda"), torch.tensor([weight, -weight, weight], device="cuda")
    f = run(x, tok, 0, temperature)
    want, grad = gradient(x, tok, gl, ge, temperature), torch.full_like(x, 7)
    sb200.logprobs_grad(x, tok, f["lse"], f["entropy"], gl, ge, grad, temperature=temperature, stream=stream())
    assert not bool(torch.isnan(grad).any())
    assert bool((grad[x == x.new_tensor(mask)] == 0).all())
    bound = gradient_bound(x, gl, ge, temperature, want, tok)
    assert bool(((grad.double() - want).abs() <= bound).all()), float(((grad.double() - want).abs() / bound).max())


@pytest.mark.parametrize("R,V", [(2, 20001), (700, 3001)])
@pytest.mark.parametrize("offset,temperature", [(1e4, 1.0), (-1e4, 1.0), (0.0, 1e-3), (3e4, 0.5), (300.0, 1.0)])
def test_logprobs_gradient_offset(cuda_dev, R, V, offset, temperature):
    """A common offset of a row, or a temperature that makes one, changes no
    probability: the gradient is as exact as without, and what the token and
    the choices get adds up to nothing.  (Logits in steps of 2^-9, so that the
    offset is exact.)"""
    g = torch.Generator("cuda").manual_seed(V)
    x = torch.round(torch.randn(R, V, device="cuda", generator=g) * 2 * 512) / 512
    x = x + offset
    tok = torch.randint(0, V, (R,), device="cuda", generator=g).to(torch.int32)
    gl, ge = (torch.randn(R, device="cuda", generator=g) for _ in range(2))
    f = run(x, tok, 0, temperature)
    for a, b in ((gl, ge), (gl, None), (None, ge)):
        zero = torch.zeros_like(gl)
        want = gradient(x, tok, zero if a is None else a, zero if b is None else b, temperature)
        bound = gradient_bound(x, zero if a is None else a, zero if b is None else b, temperature, want, tok)
        grad = torch.full_like(x, 7)
        sb200.logprobs_grad(x, tok, f["lse"], f["entropy"], a, b, grad, temperature=temperature, stream=stream())
        assert bool(((grad.double() - want).abs() <= bound).all()), float(((grad.double() - want).abs() / bound).max())
        assert bool((grad.double().sum(-1).abs() <= bound.sum(-1)).all())
        z = x.clone()
        sb200.logprobs_grad(z, tok, f["lse"], f["entropy"], a, b, z, temperature=temperature, stream=stream())
        assert torch.equal(z, grad)  # in place


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("R,temperature", [(1, 1.0), (700, 1.0), (3, 0.5)])
def test_logprobs_gradient_equal_lowest_values(cuda_dev, kind, R, temperature):
    """A row of the type's lowest value (every choice masked that way): n equal
    choices of probability 1 / n, as the forward call has them."""
    V, t = 3001, DT[kind]
    x = torch.full((R, V), torch.finfo(t).min, dtype=t, device="cuda")
    tok = torch.full((R,), 2000, dtype=torch.int32, device="cuda")
    g = torch.Generator("cuda").manual_seed(R)
    gl, ge = (torch.randn(R, device="cuda", generator=g) for _ in range(2))
    for _ in range(2):
        f = run(x, tok, 0, temperature)
        p = (x > -math.inf).double()
        p /= p.sum(-1, keepdim=True)
        H = -torch.log(p.amax(-1, keepdim=True))  # = - ln p of every choice: the entropy's gradient is 0
        want = torch.where(p > 0, -gl.double()[:, None] * p, torch.zeros_like(p))
        want.scatter_add_(1, tok.long()[:, None], gl.double()[:, None])
        want /= temperature
        grad = torch.full_like(x, 7)
        sb200.logprobs_grad(x, tok, f["lse"], f["entropy"], gl, ge, grad, temperature=temperature, stream=stream())
        # p to (n / 256 + 16) half steps and 2^-20; the entropy's terms, of size ln n p, cancel to as much
        bound = 2.0 ** -17 * p * (gl.double().abs()[:, None] + ge.double().abs()[:, None] * (2 * H + 2)) / temperature
        bound += 2.0 ** -23 * want.abs() + torch.finfo(t).eps / 2 * want.abs() + (2.0 ** -25 if t == torch.float16 else 1e-37)
        assert bool(((grad.double() - want).abs() <= bound).all()), float(((grad.double() - want).abs() / bound).max())
        x[:, : V // 2] = -math.inf


def test_logprobs_gradient_takes_the_given_lse(cuda_dev):
    """The softmax may go over more than these logits (a vocabulary cut over
    several calls): an lse that is not the row's own is taken as it is."""
    g = torch.Generator("cuda").manual_seed(11)
    x = torch.round(torch.randn(4, 30000, device="cuda", generator=g) * 512) / 512 + 5000.0
    tok, one = torch.tensor([3, 17, -1, 9], dtype=torch.int32, device="cuda"), torch.ones(4, device="cuda")
    f = run(x, tok)
    half = x[:, :15000].contiguous()
    grad = torch.empty_like(half)
    sb200.logprobs_grad(half, tok, f["lse"], None, one, None, grad, stream=stream())
    p = torch.exp(half.double() - f["lse"].double()[:, None])
    want = -p
    want[torch.tensor([0, 1, 3]), torch.tensor([3, 17, 9])] += 1
    want[2] = 0
    # c x - lse log2(e): a half step of FP32 of 7213 is 2^-12
    assert bool(((grad.double() - want).abs() <= 2.0 ** -12 * p + 2.0 ** -23 * want.abs()).all())


def test_logprobs_repeats_and_replays(cuda_dev):
    x = torch.randn(5, 60001, device="cuda").half()
    tok = torch.arange(5, dtype=torch.int32, device="cuda")
    a = run(x, tok, 33)
    k = a["top_ids"].shape[1]
    out = {n: torch.zeros_like(v) for n, v in a.items()}
    ws = torch.empty(sb200.logprobs_ws(x, k), dtype=torch.uint8, device="cuda")
    sb200.logprobs(x, tok, ws, stream=stream(), **out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sb200.logprobs(x, tok, ws, stream=stream(), **out)
    for _ in range(2):
        for v in out.values():
            v.fill_(3)
        graph.replay()
        assert all(torch.equal(out[n], a[n]) for n in a)
    x.copy_(torch.randn(5, 60001, device="cuda"))
    graph.replay()
    b = run(x, tok, 33)
    assert all(torch.equal(out[n], b[n]) for n in b)


# ---------------------------------------------------------------- all together
@pytest.mark.parametrize("kind,NH,NKV,HD,page", [("f32", 14, 2, 64, 16), ("f16", 8, 2, 128, 24), ("bf16", 6, 6, 64, 1)])
def test_serving_steps_together(cuda_dev, kind, NH, NKV, HD, page):
    """Three requests behind one prompt: the prompt's own plan and cache write,
    a step of ragged continuations, then decode steps that grow past page
    ends, each plan -> rotary with the cache write -> attention -> head
    product -> log probabilities, against one attention layer in 64 bits
    over the whole sequences."""
    t, V, P, B = DT[kind], 997, 37, 3
    g = torch.Generator("cuda").manual_seed(HD)
    C = NH * HD
    steps = [[5, 1, 9], [1, 1, 1], [1, 0, 20], [1, 1, 1]]
    n_pages, W = 80, 64
    kc, vc = (torch.full((n_pages, page, NKV, HD), float("nan"), dtype=t, device="cuda") for _ in range(2))
    kv, plan = sb200.KvPages(kc, vc), sb200.Rotary(HD, theta=1e4)
    head = (torch.randn(V, C, device="cuda", generator=g) * C ** -0.5)
    f = torch.tensor([1e4 ** (-2.0 * i / HD) for i in range(HD // 2)], dtype=torch.float64, device="cuda")
    e32 = lambda n, ty=torch.int32: torch.full((n,), 99, dtype=ty, device="cuda")  # noqa: E731
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    free = torch.randperm(n_pages, device="cuda", generator=g).to(torch.int32)
    at = 0

    def plan_step(cache, new, table, T):
        nonlocal at
        n = cache.numel()
        o = dict(slots=e32(T, torch.int64), pos=e32(T), req=e32(T), cu_q=e32(n + 1), kv_len=e32(n), used=e32(2))
        sb200.kv_plan(cache, new, free[at:].contiguous(), table, page, stream=stream(), **o)
        taken, lacking = o["used"].tolist()
        assert lacking == 0
        at += taken
        return o

    def turn(x, pos):  # 64 bits, half layout
        a = pos.double()[:, None, None] * f
        u, w = x.double()[..., : HD // 2], x.double()[..., HD // 2:]
        return torch.cat([u * torch.cos(a) - w * torch.sin(a), w * torch.cos(a) + u * torch.sin(a)], -1)

    rows = lambda T: (torch.randn(T, NH + 2 * NKV, HD, device="cuda", generator=g)).to(t)  # noqa: E731
    # the prompt: one request of its own
    ptable = torch.full((1, W), -1, dtype=torch.int32, device="cuda")
    x = rows(P)
    q, k, v = x.split([NH, NKV, NKV], 1)
    o = plan_step(i32([0]), i32([P]), ptable, P)
    sb200.rotary_kv(q, torch.empty(P, NH, HD, dtype=t, device="cuda"), k, v, o["pos"], o["slots"], plan, kv, stream=stream())
    u = torch.finfo(t).eps / 2
    full_k = [turn(k, o["pos"]).to(t).double()] * B  # what the pages hold: rounded once
    full_v = [v.double()] * B
    table = torch.full((B, W), -1, dtype=torch.int32, device="cuda")
    cache = i32([0] * B)
    for new in steps:
        T = sum(new) + 2  # two rows of padding
        x = rows(T)
        q, k, v = x.split([NH, NKV, NKV], 1)
        o = plan_step(cache, i32(new), table, T)
        pos = torch.where(o["pos"] >= 0, o["pos"] + P, o["pos"])
        qr, out = torch.zeros(T, NH, HD, dtype=t, device="cuda"), torch.zeros(T, NH, HD, dtype=t, device="cuda")
        sb200.rotary_kv(q, qr, k, v, pos, o["slots"], plan, kv, stream=stream())
        most = int(o["kv_len"].max())
        ws = torch.empty(sb200.attn_prefix_ws(qr, kv, P, B, max_q=max(new), max_kv=most), dtype=torch.uint8, device="cuda")
        sb200.attn_prefix(qr, out, kv, ptable[0], P, kv, table, o["kv_len"], HD ** -0.5, ws, cu_q=o["cu_q"], max_q=max(new), max_kv=most,
                          stream=stream())
        live = sum(new)
        logits = torch.empty(T, V, device="cuda")
        h = out.flatten(1).float().contiguous()
        sb200.check(sb200.lib().sb_gemv_multi_f32(head.data_ptr(), h.data_ptr(), None, logits.data_ptr(), C, V, T, stream().cuda_stream))
        tok = torch.where(o["req"] >= 0, torch.randint(0, V, (T,), device="cuda", generator=g).to(torch.int32), -1).to(torch.int32)
        lp, ids = torch.empty(T, device="cuda"), torch.empty(T, 3, dtype=torch.int32, device="cuda")
        ws = torch.empty(sb200.logprobs_ws(logits, 3), dtype=torch.uint8, device="cuda")
        sb200.logprobs(logits, tok, ws, logp=lp, top_ids=ids, stream=stream())
        r = 0
        for b, n in enumerate(new):
            p = P + int(cache[b]) + torch.arange(n, device="cuda")
            full_k[b] = torch.cat([full_k[b], turn(k[r: r + n], p).to(t).double()])
            full_v[b] = torch.cat([full_v[b], v[r: r + n].double()])
            for i in range(n):
                sees = P + int(cache[b]) + i + 1
                qd = turn(q[r: r + 1], p[i: i + 1])[0].view(NKV, NH // NKV, HD)
                w = torch.softmax(torch.einsum("hgd,khd->hgk", qd, full_k[b][:sees]) * HD ** -0.5, -1)
                want = torch.einsum("hgk,khd->hgd", w, full_v[b][:sees]).reshape(-1)
                size = torch.einsum("hgk,khd->hgd", w, full_v[b][:sees].abs()).reshape(-1)
                # query rounded once (scores of size |q k| off by half a step: 12 of it), keys at worst to the other
                # neighbour (the same again), weights and result rounded once
                err = (out[r].flatten().double() - want).abs()
                assert bool((err <= (26 * u + 2e-5) * size + u * want.abs()).all()), (b, i, float((err / size).max()))
                logs = torch.log_softmax(head.double() @ out[r].flatten().double(), -1)
                assert abs(float(lp[r]) - float(logs[int(tok[r])])) < 1e-4  # FP32 product of C <= 1024 terms of size 1 / 32
                best = torch.sort(logs, descending=True).values[:3]
                assert bool(((logs[ids[r].long()] - best).abs() < 1e-4).all())
                r += 1
        assert bool((out[live:] == 0).all()) and lp[live:].tolist() == [0.0, 0.0]
        cache = o["kv_len"]
