"""The operators for a batch of requests that share a prompt, as cases to measure.

Four operators, in the order in which a serving or scoring step calls them:

  plan      block tables, slot map, positions and row offsets from request lengths
  rotary    rotary positions of query and key rows, with the cache write through the slot map
  attn      attention of a batch over a shared prefix (read once for all) and each request's own pages
  logprobs  log probability, entropy and rank of given tokens, the top alternatives, and the gradient

`run` computes them in their plain form (elementary torch operations in 32 bits, angles in 64) where `own` is
false, and through the framework's public entry points where it is true.
"""
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
DEV = "cuda"


def _sb():
    """The framework's Python binding (its package folder is no Python identifier)."""
    here = os.path.join(os.getcwd(), "switch-l4t-gpu_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    import sb200
    return sb200


# ---------------------------------------------------------------- cases
def listed():
    return [
        # one decode step of a small batch: a new token each, the call is all latency
        dict(name="plan-decode-8", op="plan", B=8, page=16, max_cache=2048, max_new=1, width=129, short=False),
        # a prefill of many requests of ragged length whose free list runs out before the last one
        dict(name="plan-prefill-256", op="plan", B=256, page=16, max_cache=4096, max_new=2048, width=400, short=True),
        # one token of the Qwen heads (14 query, 2 key/value heads of 64), FP32 activations and cache
        dict(name="rotary-token", op="rotary", kind="kv", type="f32", T=1, NH=14, NKV=2, HD=64, dim=64, layout="half",
             scaling="none", far=8192, page=16, inverse=False),
        # a prefill of ragged requests with the cache write; neighbouring pairs, half of the head, scaled for 32 times
        # the trained context
        dict(name="rotary-prefill-scaled", op="rotary", kind="kv", type="bf16", T=8191, NH=32, NKV=8, HD=128, dim=64,
             layout="pairs", scaling="yarn", far=1000000, page=64, inverse=False),
        # the gradient of the query rotation: the inverse rotation of the incoming gradient
        dict(name="rotary-gradient", op="rotary", kind="rows", type="f32", T=4099, NH=14, NKV=2, HD=64, dim=64,
             layout="half", scaling="bands", far=131072, page=16, inverse=True),
        # a few requests behind a short system prompt on the engines' FP32 cache: latency
        dict(name="attn-few-f32", op="attn", type="f32", B=4, nq=1, NH=14, NKV=2, HD=64, P=300, S=64, page=16),
        # a serving batch of the GPT-2 heads, FP32
        dict(name="attn-serve-f32", op="attn", type="f32", B=48, nq=1, NH=12, NKV=12, HD=64, P=1000, S=777, page=16),
        # scoring many continuations of a long prompt: up to 33 rows a request, causal among themselves
        dict(name="attn-score-f16", op="attn", type="f16", B=32, nq=33, NH=14, NKV=2, HD=64, P=4001, S=129, page=32),
        # a large serving batch behind a very long prompt
        dict(name="attn-serve-bf16", op="attn", type="bf16", B=256, nq=1, NH=32, NKV=8, HD=128, P=16000, S=500, page=64),
        # the alternatives of one answer token over the Qwen vocabulary
        dict(name="logprobs-one", op="logprobs", type="f32", R=1, V=151936, k=20, temperature=0.7, grad=False),
        # a scoring batch over the odd GPT-2 vocabulary in half precision, with five alternatives
        dict(name="logprobs-score", op="logprobs", type="f16", R=1056, V=50257, k=5, temperature=1.0, grad=False),
        # a training batch over the Qwen vocabulary: forward, then the gradient of log probability and entropy
        dict(name="logprobs-train", op="logprobs", type="bf16", R=2048, V=151936, k=0, temperature=1.0, grad=True),
    ]


HEADS = [(14, 2, 64), (12, 12, 64), (32, 8, 128), (16, 1, 128), (6, 2, 64), (20, 4, 80), (24, 3, 96), (8, 8, 32)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "rotary", "attn", "attn", "logprobs"])
    caps = {o: max(_cost(c) for c in listed() if c["op"] == o) for o in ("plan", "rotary", "attn", "logprobs")}
    while True:
        if op == "plan":
            page = rng.choice([1, 8, 16, 24, 32, 64, 128])
            c = dict(op=op, B=_log(rng, 1, 512), page=page, max_cache=_log(rng, 1, 8192), max_new=_log(rng, 1, 2048),
                     short=rng.random() < 0.3)
            c["width"] = (c["max_cache"] + c["max_new"]) // page + 2
        elif op == "rotary":
            NH, NKV, HD = rng.choice(HEADS)
            c = dict(op=op, kind=rng.choice(["kv", "kv", "rows"]), type=rng.choice(list(TYPES)), T=_log(rng, 1, 16384), NH=NH,
                     NKV=NKV, HD=HD, dim=rng.choice([HD, HD // 2, HD // 4]), layout=rng.choice(["half", "pairs"]),
                     scaling=rng.choice(["none", "linear", "ntk", "yarn", "bands"]), far=_log(rng, 4096, 1 << 20),
                     page=rng.choice([1, 16, 24, 64]), inverse=False)
            c["inverse"] = c["kind"] == "rows" and rng.random() < 0.5
        elif op == "attn":
            NH, NKV, HD = rng.choice(HEADS)
            c = dict(op=op, type=rng.choice(list(TYPES)), B=_log(rng, 1, 256), nq=rng.choice([1, 1, 1, _log(rng, 2, 64)]), NH=NH,
                     NKV=NKV, HD=HD, P=rng.choice([0] + 7 * [_log(rng, 1, 32768)]), S=_log(rng, 1, 4096), page=rng.choice([16, 24, 32, 64, 128]))
            c["S"] = max(c["S"], c["nq"])
        else:
            c = dict(op=op, type=rng.choice(list(TYPES)), R=_log(rng, 1, 2048), V=_log(rng, 1000, 151936), k=rng.choice([0, 1, 5, 20, 64]),
                     temperature=rng.choice([1.0, 0.7, 1.3]), grad=rng.random() < 0.4)
        if _cost(c) <= caps[op]:
            return c


def _cost(c):
    """One figure for a case's work: its bytes, and 300 FLOP counted as a byte (about the ratio of this card's rates)."""
    w = work(c)
    return w["bytes"] + w["flops"] / 300.0


# ---------------------------------------------------------------- lengths (a part of the case, the same for each seed)
def _ragged(n, lo, hi, odd):
    """n lengths in [lo, hi], the first hi and the second lo."""
    return [hi if i == 0 else lo if i == 1 else lo + (i * 7919 + odd) % (hi - lo + 1) for i in range(n)]


def _plan_lengths(c):
    new = [1] * c["B"] if c["max_new"] == 1 else _ragged(c["B"], 0, c["max_new"], 31)
    cache = _ragged(c["B"], 0, c["max_cache"], 57)
    return cache, new


def _attn_lengths(c):
    """Rows of each request and its own positions (those of its rows among them); where there are more than two, the second is a
    place of the batch that no request fills."""
    rows = [1] * c["B"] if c["nq"] == 1 else _ragged(c["B"], 1, c["nq"], 5)
    kv = [max(n, s) for n, s in zip(rows, _ragged(c["B"], 1, c["S"], 11))]
    if c["B"] > 2:
        kv[1] = 0
        if c["nq"] > 1:
            rows[1] = 0
    return rows, kv


def _split_rows(T):
    """T rows as requests of at most 97 tokens."""
    got = []
    while sum(got) < T:
        got.append(min(T - sum(got), 1 + (len(got) * 41) % 97))
    return got


# ---------------------------------------------------------------- work
def work(case):
    c = case
    if c["op"] == "plan":
        cache, new = _plan_lengths(c)
        p, T = c["page"], sum(new)
        add = sum(-(-(a + n) // p) - -(-a // p) for a, n in zip(cache, new))
        return {"bytes": 16.0 * T + 16.0 * c["B"] + 8.0 * add, "flops": 0}
    if c["op"] == "rotary":
        e, rows = SIZE[c["type"]], c["T"] * c["HD"]
        heads = c["NH"] + (2 * c["NKV"] if c["kind"] == "kv" else 0)
        turned = c["T"] * (c["NH"] + (c["NKV"] if c["kind"] == "kv" else 0)) * c["dim"]
        return {"bytes": 2.0 * rows * heads * e + c["T"] * (12.0 if c["kind"] == "kv" else 4.0), "flops": 3.0 * turned}
    if c["op"] == "attn":
        rows, kv = _attn_lengths(c)
        e, T = SIZE[c["type"]], sum(rows)
        seen = sum(n * c["P"] + sum(max(0, s - n + i + 1) for i in range(n)) for n, s in zip(rows, kv))
        held = c["P"] + sum(kv)
        return {"bytes": 2.0 * T * c["NH"] * c["HD"] * e + 2.0 * held * c["NKV"] * c["HD"] * e, "flops": 4.0 * seen * c["NH"] * c["HD"]}
    e, n = SIZE[c["type"]], c["R"] * c["V"]
    # the gradient needs the logits a second time: they are far larger than what the card keeps near
    return {"bytes": float(n * e * (3 if c["grad"] else 1) + c["R"] * (16 + 8 * c["k"])), "flops": float(n * (10 if c["grad"] else 5))}


# ---------------------------------------------------------------- inputs
def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _offsets(v):
    return torch.cat([torch.zeros(1, dtype=torch.int32, device=DEV), torch.cumsum(_ints(v), 0).to(torch.int32)])


def _frequencies(c):
    """Radians a position of each pair and the factor on cosine and sine, in 64 bits on the host."""
    d, theta, orig, factor = c["dim"], 1e6, 4096, 32.0
    kind = c["scaling"]
    if kind == "ntk":
        theta = theta * factor ** (d / (d - 2.0))
    f = [theta ** (-2.0 * i / d) for i in range(d // 2)]
    scale = 1.0
    if kind == "linear":
        f = [x / factor for x in f]
    elif kind == "yarn":
        # pairs that turn often over the trained context stay, slow ones are stretched, those between are blended
        at = [d * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(theta)) for turns in (32.0, 1.0)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), d - 1)
        ramp = [min(max((i - lo) / (hi - lo if hi > lo else 0.001), 0.0), 1.0) for i in range(d // 2)]
        f = [x / factor * r + x * (1 - r) for x, r in zip(f, ramp)]
        scale = 0.1 * math.log(factor) + 1.0
    elif kind == "bands":
        # by wavelength: short ones stay, long ones are stretched, a linear blend between
        lo, hi, g = 1.0, 4.0, []
        for x in f:
            turns = orig * x / (2 * math.pi)
            s = min(max((turns - lo) / (hi - lo), 0.0), 1.0)
            g.append(x / factor * (1 - s) + x * s)
        f = g
    return f, scale


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 1000003 + 17)
    rand = lambda *s, t=torch.float32: torch.randn(*s, generator=g, device=DEV).to(t)  # noqa: E731
    s = {"case": c}
    if c["op"] == "plan":
        cache, new = _plan_lengths(c)
        p, W = c["page"], c["width"]
        have = [-(-a // p) for a in cache]
        add = sum(-(-(a + n) // p) - h for a, n, h in zip(cache, new, have))
        pool = torch.randperm(sum(have) + add + 8, generator=g, device=DEV).to(torch.int32)
        first = _offsets(have)
        col = torch.arange(W, device=DEV, dtype=torch.int32)[None]
        held = pool[(first[:-1, None] + col).clamp(max=pool.numel() - 1).long()]
        s["table"] = torch.where(col < _ints(have)[:, None], held, -1).contiguous()
        s["free"] = pool[sum(have):].contiguous()
        if c["short"]:
            s["free"] = s["free"][: max(1, add - add // 8)].contiguous()
        s["cache"], s["new"] = _ints(cache), _ints(new)
        T = sum(new) + 3  # three rows of padding behind the last request
        s["slots"] = torch.empty(T, dtype=torch.int64, device=DEV)
        s["pos"], s["req"] = (torch.empty(T, dtype=torch.int32, device=DEV) for _ in range(2))
        s["cu_q"], s["kv_len"] = torch.empty(c["B"] + 1, dtype=torch.int32, device=DEV), torch.empty(c["B"], dtype=torch.int32, device=DEV)
        s["used"] = torch.empty(2, dtype=torch.int32, device=DEV)
    elif c["op"] == "rotary":
        t, T, HD = TYPES[c["type"]], c["T"], c["HD"]
        # query, key and value rows come out of one product, side by side
        s["qkv"] = rand(T, c["NH"] + 2 * c["NKV"], HD, t=t)
        s["q"], s["k"], s["v"] = s["qkv"].split([c["NH"], c["NKV"], c["NKV"]], 1)
        lens = _split_rows(T)
        start = torch.randint(0, max(1, c["far"] - 97), (len(lens),), generator=g, device=DEV, dtype=torch.int32)
        off = _offsets(lens)
        req = torch.searchsorted(off[1:].contiguous(), torch.arange(T, device=DEV, dtype=torch.int32), right=True)
        s["pos"] = (start[req] + torch.arange(T, device=DEV, dtype=torch.int32) - off[req]).to(torch.int32)
        s["q_out"] = torch.empty(T, c["NH"], HD, dtype=t, device=DEV)
        pages = -(-T // c["page"]) + 3
        s["slots"] = torch.randperm(pages * c["page"], generator=g, device=DEV)[:T].contiguous()
        s["kc"], s["vc"] = (torch.zeros(pages, c["page"], c["NKV"], HD, dtype=t, device=DEV) for _ in range(2))
        f, s["scale"] = _frequencies(c)
        s["freq"] = torch.tensor(f, dtype=torch.float64, device=DEV)
    elif c["op"] == "attn":
        t, p, P = TYPES[c["type"]], c["page"], c["P"]
        rows, kv = _attn_lengths(c)
        T = sum(rows)
        pp, W = max(1, -(-P // p)), -(-max(kv) // p)
        n_pages = pp + sum(-(-x // p) for x in kv) + 2
        perm = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
        s["ptable"] = perm[:pp].contiguous()
        first = pp + _offsets([-(-x // p) for x in kv])
        col = torch.arange(W, device=DEV, dtype=torch.int32)[None]
        held = perm[(first[:-1, None] + col).clamp(max=n_pages - 1).long()]
        s["table"] = torch.where(col < _ints([-(-x // p) for x in kv])[:, None], held, -1).contiguous()
        s["kc"], s["vc"] = (rand(n_pages, p, c["NKV"], c["HD"], t=t) for _ in range(2))
        s["q"] = rand(T, c["NH"], c["HD"], t=t)
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(T, c["NH"], device=DEV)
        s["kv_len"], s["cu_q"] = _ints(kv), _offsets(rows)
        s["max_kv"], s["max_q"] = max(kv), max(rows)
        s["scale"] = c["HD"] ** -0.5
    else:
        R, V, k = c["R"], c["V"], c["k"]
        # logits of a language model: a wide bulk and a few likely tokens
        x = torch.randn(R, V, generator=g, device=DEV)
        x.mul_(2.0)
        hot = torch.randint(0, V, (R, 32), generator=g, device=DEV)
        x.scatter_add_(1, hot, torch.rand(R, 32, generator=g, device=DEV) * 12.0)
        s["logits"] = x.to(TYPES[c["type"]])
        del x
        s["tokens"] = torch.where(torch.rand(R, generator=g, device=DEV) < 0.7, hot[:, 0], torch.randint(0, V, (R,), generator=g, device=DEV)).to(torch.int32)
        if R > 2:
            s["tokens"][1] = -1  # a row without a token
            s["logits"][2, : V // 3] = -math.inf  # a row whose choices are restricted
            s["tokens"][2] = V - 1
        for n in ("logp", "entropy", "lse"):
            s[n] = torch.empty(R, device=DEV)
        s["rank"] = torch.empty(R, dtype=torch.int32, device=DEV)
        s["top_ids"], s["top_logp"] = torch.empty(R, k, dtype=torch.int32, device=DEV), torch.empty(R, k, device=DEV)
        if c["grad"]:
            s["g_logp"], s["g_entropy"] = rand(R), rand(R) * 0.01
            s["grad"] = torch.empty_like(s["logits"])
    if own:  # the handles and workspaces that a program keeps
        sb = _sb()
        if c["op"] == "rotary":
            s["rotary"] = sb.Rotary(c["dim"], theta=1e6, layout={"half": sb.ROPE_HALF, "pairs": sb.ROPE_PAIRS}[c["layout"]],
                                    scaling={"none": sb.ROPE_PLAIN, "linear": sb.ROPE_LINEAR, "ntk": sb.ROPE_NTK,
                                             "yarn": sb.ROPE_YARN, "bands": sb.ROPE_BANDS}[c["scaling"]], factor=32.0, orig_ctx=4096)
            s["kv"] = sb.KvPages(s["kc"], s["vc"])
        elif c["op"] == "attn":
            s["kv"] = sb.KvPages(s["kc"], s["vc"])
            n = sb.attn_prefix_ws(s["q"], s["kv"], P, len(kv), max_q=s["max_q"], max_kv=s["max_kv"])
            s["ws"] = torch.empty(n, dtype=torch.uint8, device=DEV)
        elif c["op"] == "logprobs":
            s["ws"] = torch.empty(sb.logprobs_ws(s["logits"], c["k"]), dtype=torch.uint8, device=DEV)
    return s


# ---------------------------------------------------------------- one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return {"plan": _own_plan, "rotary": _own_rotary, "attn": _own_attn, "logprobs": _own_logprobs}[op](state)
    return {"plan": _plain_plan, "rotary": _plain_rotary, "attn": _plain_attn, "logprobs": _plain_logprobs}[op](state)


def _own_plan(s):
    sb = _sb()
    sb.kv_plan(s["cache"], s["new"], s["free"], s["table"], s["case"]["page"], s["slots"], s["pos"], s["req"], s["cu_q"],
               s["kv_len"], s["used"], stream=torch.cuda.current_stream())
    return {n: s[n] for n in ("table", "slots", "pos", "req", "cu_q", "kv_len", "used")}


def _plain_plan(s):
    p, W, B = s["case"]["page"], s["case"]["width"], s["case"]["B"]
    cache, new, free = s["cache"].long(), s["new"].long(), s["free"].long()
    have, need = (cache + p - 1) // p, (cache + new + p - 1) // p
    last = need.clamp(max=W)
    add = (last - have).clamp(min=0)
    first = torch.cumsum(add, 0) - add
    col = torch.arange(W, device=DEV)[None]
    i = first[:, None] + col - have[:, None]
    fresh = torch.where(i < free.numel(), free[i.clamp(0, free.numel() - 1)], -1)
    table = torch.where((col >= have[:, None]) & (col < last[:, None]), fresh, s["table"].long())
    cu = torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV), torch.cumsum(new, 0)])
    t = torch.arange(s["slots"].numel(), device=DEV)
    live = t < cu[B]
    req = torch.searchsorted(cu[1:].contiguous(), t, right=True).clamp(max=B - 1)
    pos = cache[req] + t - cu[req]
    page = torch.where(pos // p < W, table[req, (pos // p).clamp(max=W - 1)], -1)
    slots = torch.where(live & (page >= 0), page * p + pos % p, -1)
    total = add.sum()
    taken = total.clamp(max=free.numel())
    used = torch.stack([taken, (need - have).sum() - taken])
    off = torch.full((), -1, device=DEV)
    return {"table": table.int(), "slots": slots, "pos": torch.where(live, pos, off).int(), "req": torch.where(live, req, off).int(),
            "cu_q": cu.int(), "kv_len": (cache + new).int(), "used": used.int()}


def _own_rotary(s):
    sb, c = _sb(), s["case"]
    if c["kind"] == "rows":
        sb.rotary(s["q"], s["q_out"], s["pos"], s["rotary"], inverse=c["inverse"], stream=torch.cuda.current_stream())
        return {"q": s["q_out"]}
    sb.rotary_kv(s["q"], s["q_out"], s["k"], s["v"], s["pos"], s["slots"], s["rotary"], s["kv"], stream=torch.cuda.current_stream())
    return {"q": s["q_out"], "k": s["kc"], "v": s["vc"]}


def _turn(x, cos, sin, c):
    """x [T, H, HD] with its first `dim` values turned, in 32 bits."""
    d = c["dim"]
    y = x.float()
    head, rest = y[..., :d], y[..., d:]
    if c["layout"] == "half":
        a, b = head[..., : d // 2], head[..., d // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = head[..., 0::2], head[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, rest], -1).to(x.dtype)


def _plain_rotary(s):
    c = s["case"]
    angle = s["pos"].double()[:, None] * s["freq"]
    cos, sin = (torch.cos(angle) * s["scale"]).float()[:, None], (torch.sin(angle) * s["scale"]).float()[:, None]
    if c["inverse"]:
        sin = -sin
    q = _turn(s["q"], cos, sin, c)
    if c["kind"] == "rows":
        return {"q": q}
    s["kc"].flatten(0, 1)[s["slots"]] = _turn(s["k"], cos, sin, c)
    s["vc"].flatten(0, 1)[s["slots"]] = s["v"]
    return {"q": q, "k": s["kc"], "v": s["vc"]}


def _own_attn(s):
    _sb().attn_prefix(s["q"], s["out"], s["kv"], s["ptable"], s["case"]["P"], s["kv"], s["table"], s["kv_len"], s["scale"], s["ws"],
                      cu_q=s["cu_q"] if s["case"]["nq"] > 1 else None, max_q=s["max_q"], max_kv=s["max_kv"], lse=s["lse"],
                      stream=torch.cuda.current_stream())
    return {"out": s["out"], "lse": s["lse"]}


def _plain_attn(s):
    c = s["case"]
    p, P, NKV, HD, B = c["page"], c["P"], c["NKV"], c["HD"], c["B"]
    G, T = c["NH"] // NKV, s["q"].shape[0]
    pos = torch.arange(P, device=DEV)
    page = s["ptable"].long()[pos // p]
    kp, vp = s["kc"][page, pos % p].float(), s["vc"][page, pos % p].float()  # [P, NKV, HD]
    q = s["q"].float().view(T, NKV, G, HD)
    # the shared prefix: one product for all rows of a key head
    sp = torch.matmul(q.permute(1, 0, 2, 3).reshape(NKV, T * G, HD), kp.permute(1, 2, 0)) * s["scale"]
    sp = sp.view(NKV, T, G, P).permute(1, 0, 2, 3)
    # each request's own positions, padded to the longest
    S, n = s["table"].shape[1] * p, s["max_q"]
    own_pos = torch.arange(S, device=DEV)
    pages = s["table"].long().clamp(min=0)[:, own_pos // p]
    ks, vs = s["kc"][pages, own_pos % p].float(), s["vc"][pages, own_pos % p].float()  # [B, S, NKV, HD]
    cu = s["cu_q"].long()
    count = cu[1:] - cu[:-1]
    i = torch.arange(n, device=DEV)
    row = (cu[:-1, None] + i).clamp(max=T - 1)
    qs = q[row].permute(0, 2, 1, 3, 4).reshape(B, NKV, n * G, HD)
    ss = torch.matmul(qs, ks.permute(0, 2, 3, 1)) * s["scale"]
    sees = s["kv_len"].long()[:, None] - count[:, None] + i + 1  # [B, n] positions that row i of a request sees
    seen = (own_pos[None, None] < sees[..., None]) & (own_pos[None, None] < s["kv_len"].long()[:, None, None])
    ss = ss.view(B, NKV, n, G, S).masked_fill(~seen[:, None, :, None], -math.inf)
    # back to rows, joined with the prefix under one softmax
    t = torch.arange(T, device=DEV)
    b = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    ss = ss[b, :, t - cu[b]]  # [T, NKV, G, S]
    both = torch.cat([sp, ss], -1)
    del sp, ss
    m = both.amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    e = torch.exp(both - m)
    del both
    l = e.sum(-1, keepdim=True)
    w = e / torch.where(l > 0, l, torch.ones_like(l))
    del e
    o = torch.matmul(w[..., :P].permute(1, 0, 2, 3).reshape(NKV, T * G, P), vp.permute(1, 0, 2)).view(NKV, T, G, HD).permute(1, 0, 2, 3)
    ws = torch.zeros(B, n, NKV, G, S, device=DEV)
    ws[b, t - cu[b]] = w[..., P:]
    os_ = torch.matmul(ws.permute(0, 2, 1, 3, 4).reshape(B, NKV, n * G, S), vs.permute(0, 2, 1, 3)).view(B, NKV, n, G, HD)
    o = o + os_[b, :, t - cu[b]]
    return {"out": o.reshape(T, c["NH"], HD).to(s["q"].dtype), "lse": (m + torch.log(l)).reshape(T, c["NH"])}


def _own_logprobs(s):
    sb, c = _sb(), s["case"]
    at = torch.cuda.current_stream()
    sb.logprobs(s["logits"], s["tokens"], s["ws"], logp=s["logp"], entropy=s["entropy"], lse=s["lse"], rank=s["rank"],
                top_ids=s["top_ids"] if c["k"] else None, top_logp=s["top_logp"] if c["k"] else None, temperature=c["temperature"], stream=at)
    out = {n: s[n] for n in ("logp", "entropy", "lse", "rank", "top_ids", "top_logp")}
    if c["grad"]:
        sb.logprobs_grad(s["logits"], s["tokens"], s["lse"], s["entropy"], s["g_logp"], s["g_entropy"], s["grad"],
                         temperature=c["temperature"], stream=at)
        out["grad"] = s["grad"]
    return out


def _plain_logprobs(s):
    c = s["case"]
    raw = s["logits"].float()
    x = raw / c["temperature"]
    V = c["V"]
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(-1, keepdim=True)
    lse = m + torch.log(total)
    p = e / total
    del e
    entropy = torch.where(p > 0, p * (lse - x), torch.zeros_like(x)).sum(-1)
    tok = s["tokens"].long()
    given = (tok >= 0) & (tok < V)
    at = tok.clamp(0, V - 1)[:, None]
    logp = torch.where(given, (x.gather(1, at) - lse)[:, 0], torch.zeros_like(entropy))
    ids = torch.arange(V, device=DEV)[None]
    mine = raw.gather(1, at)
    rank = ((raw > mine) | ((raw == mine) & (ids < at))).sum(-1)
    rank = torch.where(given, rank, torch.full_like(rank, -1))
    # value first, then the lower id: both in one whole number
    k = c["k"]
    bits = (raw + 0.0).view(torch.int32).long()
    key = torch.where(bits >= 0, bits, -1 - (bits & 0x7FFFFFFF)) * (1 << 20) + (V - 1 - ids)
    top = torch.topk(key, k, -1).values if k else key[:, :0]
    top_ids = V - 1 - (top & ((1 << 20) - 1))
    out = {"logp": logp, "entropy": entropy, "lse": lse[:, 0], "rank": rank.int(), "top_ids": top_ids.int(),
           "top_logp": x.gather(1, top_ids) - lse}
    del raw, bits, key
    if c["grad"]:
        hot = torch.where(given, s["g_logp"], torch.zeros_like(s["g_logp"]))[:, None]
        d = p * (-hot - s["g_entropy"][:, None] * torch.where(p > 0, x - lse + entropy[:, None], torch.zeros_like(x)))
        d.scatter_add_(1, at, hot)
        out["grad"] = (d / c["temperature"]).to(s["logits"].dtype)
    return out


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"plan": _exact_plan, "rotary": _exact_rotary, "attn": _exact_attn, "logprobs": _exact_logprobs}[case["op"]](s)


def _exact_plan(s):
    return None  # whole numbers


def _exact_rotary(s):
    """Each pair as a complex number times e^(i angle)."""
    c = s["case"]
    d = c["dim"]
    sign = -1.0 if c["inverse"] else 1.0
    angle = s["pos"].to(torch.float64)[:, None, None] * s["freq"]
    z = torch.polar(torch.full_like(angle, s["scale"]), sign * angle)

    def turned(x):
        y = x.to(torch.float64).clone()
        if c["layout"] == "half":
            w = torch.complex(y[..., : d // 2].contiguous(), y[..., d // 2: d].contiguous()) * z
            y[..., : d // 2], y[..., d // 2: d] = w.real, w.imag
        else:
            w = torch.view_as_complex(y[..., :d].reshape(*y.shape[:-1], d // 2, 2).contiguous()) * z
            y[..., :d] = torch.view_as_real(w).flatten(-2)
        return y

    q = turned(s["q"])
    if c["kind"] == "rows":
        return {"q": q}
    out = {"q": q}
    for name, pages, new in (("k", s["kc"], turned(s["k"])), ("v", s["vc"], s["v"].to(torch.float64))):
        flat = pages.to(torch.float64).reshape(-1, c["NKV"], c["HD"])
        flat.index_copy_(0, s["slots"], new)
        out[name] = flat.view(pages.shape)
    return out


def _exact_attn(s):
    """Request by request, key head by key head, over its positions laid out in order."""
    c = s["case"]
    if work(c)["flops"] > 4e12:
        return None
    D = torch.float64
    p, P, NKV = c["page"], c["P"], c["NKV"]
    G = c["NH"] // NKV
    out = torch.zeros(s["q"].shape, dtype=D, device=DEV)
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=D, device=DEV)
    cu, kv = s["cu_q"].tolist(), s["kv_len"].tolist()
    flat = [x.reshape(-1, NKV, c["HD"]) for x in (s["kc"], s["vc"])]
    where = lambda table, n: (table.long()[:, None] * p + torch.arange(p, device=DEV)).reshape(-1)[:n]  # noqa: E731
    shared = where(s["ptable"], P)
    shared = [x[shared].to(D) for x in flat]
    for b in range(c["B"]):
        n = cu[b + 1] - cu[b]
        if n == 0:
            continue
        mine = where(s["table"][b, : -(-kv[b] // p)], kv[b])
        k, v = (torch.cat([x, y[mine].to(D)]) for x, y in zip(shared, flat))
        if not k.shape[0]:
            continue
        q = s["q"][cu[b]: cu[b + 1]].to(D).view(n, NKV, G, c["HD"])
        score = torch.einsum("nhgd,khd->nhgk", q, k) * s["scale"]
        last = P + max(kv[b] - n, 0) if kv[b] >= n else P + kv[b] - n
        sees = last + 1 + torch.arange(n, device=DEV)
        score = score.masked_fill(torch.arange(k.shape[0], device=DEV) >= sees.view(n, 1, 1, 1).clamp(min=P), -math.inf)
        top = torch.logsumexp(score, -1)
        w = torch.where(torch.isinf(top)[..., None], torch.zeros_like(score), torch.exp(score - top[..., None]))
        out[cu[b]: cu[b + 1]] = torch.einsum("nhgk,khd->nhgd", w, v).reshape(n, c["NH"], c["HD"])
        lse[cu[b]: cu[b + 1]] = top.reshape(n, c["NH"])
    return {"out": out, "lse": lse}


def _exact_logprobs(s):
    """Some rows at a time: logsumexp and its derivative."""
    c = s["case"]
    D, R, V = torch.float64, c["R"], c["V"]
    got = {n: torch.empty(R, dtype=D, device=DEV) for n in ("logp", "entropy", "lse")}
    got["rank"] = got["top_ids"] = None
    got["top_logp"] = torch.empty(R, c["k"], dtype=D, device=DEV)
    if c["grad"]:
        got["grad"] = torch.empty(R, V, dtype=D, device=DEV)
    for r in range(0, R, 64):
        x = s["logits"][r: r + 64].to(D) / c["temperature"]
        top = torch.logsumexp(x, -1)
        logs = x - top[:, None]
        p = torch.exp(logs)
        plogp = torch.where(p > 0, p * logs, torch.zeros_like(p))
        tok = s["tokens"][r: r + 64].long()
        given = (tok >= 0) & (tok < V)
        pick = logs.gather(1, tok.clamp(0, V - 1)[:, None])[:, 0]
        got["lse"][r: r + 64], got["entropy"][r: r + 64] = top, -plogp.sum(-1)
        got["logp"][r: r + 64] = torch.where(given, pick, torch.zeros_like(pick))
        if c["k"]:
            got["top_logp"][r: r + 64] = torch.sort(logs, -1, descending=True).values[:, : c["k"]]
        if c["grad"]:
            d = s["g_entropy"][r: r + 64].to(D)[:, None] * (p * plogp.sum(-1, keepdim=True) - plogp)
            gl = torch.where(given, s["g_logp"][r: r + 64].to(D), torch.zeros_like(top))[:, None]
            d = d - gl * p
            d.scatter_add_(1, tok.clamp(0, V - 1)[:, None], gl)
            got["grad"][r: r + 64] = d / c["temperature"]
    return got
