"""The batch operators (page plan, rotary, shared-prefix attention, log
probabilities) where no GPU is needed: refusals of bad arguments, the layout of
the structs that the binding mirrors, and the rotary frequencies."""
import ctypes
import decimal
import math
import os
import subprocess

import numpy as np
import pytest
import torch

import sb200

ERR_ARG = 9001


def _pages(**kw):
    p = sb200._KvPages(0x10000, 0x20000, 16 * 2 * 64, 2 * 64, 64, sb200.F16, 8, 16, 2, 64)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def _plan(dim=64, **kw):
    r = sb200._RotaryPlan()
    args = dict(layout=0, theta=1e4, scaling=0, factor=1.0, orig=0)
    args.update(kw)
    rc = sb200.lib().sb_rotary_plan_init(ctypes.byref(r), dim, args["layout"], args["theta"], args["scaling"], args["factor"], args["orig"])
    return rc, r


def test_struct_sizes():
    assert ctypes.sizeof(sb200._KvPages) == 64
    assert ctypes.sizeof(sb200._RotaryPlan) == 128 * 8 + 16


def test_rotary_plan_refusals():
    nan = float("nan")
    for bad in (dict(dim=0), dict(dim=63), dict(dim=258), dict(layout=2), dict(theta=1.0), dict(theta=nan), dict(scaling=5),
                dict(scaling=1, factor=0.5), dict(scaling=1, factor=nan), dict(scaling=3, factor=4.0), dict(dim=2, scaling=2, factor=2.0)):
        assert _plan(**bad)[0] == ERR_ARG, bad
    assert sb200.lib().sb_rotary_plan_init(None, 64, 0, 1e4, 0, 1.0, 0) == ERR_ARG


@pytest.mark.parametrize("dim", [2, 32, 64, 128, 256])
def test_rotary_plan_frequencies(dim):
    """turn = f / 2 pi as a 64-bit fraction; f from pow in double: 2 ulp of
    double relative, and the fraction's own half unit."""
    for theta in (1e4, 1e6):
        rc, r = _plan(dim, theta=theta)
        assert rc == 0 and r.mscale == 1.0
        for i in range(dim // 2):
            f = theta ** (-2.0 * i / dim) / (2 * math.pi)
            assert abs(r.turn[i] / 2.0 ** 64 - f) <= 4 * 2.0 ** -53 * f + 2.0 ** -64
    if dim > 2:
        for i in range(dim // 2):
            base = 1e6 ** (-2.0 * i / dim)
            turns = 4096 * base / (2 * math.pi)
            got = {s: _plan(dim, theta=1e6, scaling=s, factor=8.0, orig=4096)[1].turn[i] / 2.0 ** 64 * 2 * math.pi for s in (1, 2, 3, 4)}
            assert got[1] == pytest.approx(base / 8, rel=1e-12)
            assert got[2] == pytest.approx((1e6 * 8.0 ** (dim / (dim - 2.0))) ** (-2.0 * i / dim), rel=1e-12)
            for s, keep in ((3, 32.0), (4, 4.0)):
                # the kept and the stretched ends, and between them in between
                assert base / 8 * (1 - 1e-12) <= got[s] <= base * (1 + 1e-12)
                if s == 4 and turns >= keep:
                    assert got[s] == pytest.approx(base, rel=1e-12)
                if s == 4 and turns <= 1.0:
                    assert got[s] == pytest.approx(base / 8, rel=1e-12)
        assert _plan(dim, scaling=3, factor=8.0, orig=4096)[1].mscale == pytest.approx(0.1 * math.log(8.0) + 1.0, rel=1e-6)


def test_rotary_plan_yarn_ends():
    """dim 64, theta 1e4, trained on 2048: pair 0 turns 326 times (kept), the
    last pair 0.04 times (divided), one in the middle is blended."""
    r = _plan(64, theta=1e4, scaling=3, factor=4.0, orig=2048)[1]
    f = lambda i: r.turn[i] / 2.0 ** 64 * 2 * math.pi  # noqa: E731
    base = lambda i: 1e4 ** (-2.0 * i / 64)  # noqa: E731
    assert f(0) == pytest.approx(base(0), rel=1e-12) and f(31) == pytest.approx(base(31) / 4, rel=1e-12)
    assert base(14) / 4 < f(14) < base(14)


def test_kv_plan_refusals():
    L, p = sb200.lib(), 0x1000
    ok = dict(B=2, page=16, n_free=4, stride=8, width=8, T=4, cl=p, nl=2 * p, fp=p, tb=3 * p, sl=4 * p, po=5 * p, rq=6 * p, cq=7 * p, kl=8 * p, us=9 * p)

    def call(**kw):
        a = dict(ok, **kw)
        return L.sb_kv_plan(a["cl"], a["nl"], a["B"], a["page"], a["fp"], a["n_free"], a["tb"], a["stride"], a["width"], a["sl"], a["po"],
                            a["rq"], a["T"], a["cq"], a["kl"], a["us"], None)
    for bad in (dict(B=0), dict(B=16385), dict(page=0), dict(n_free=-1), dict(fp=None), dict(width=0), dict(stride=7), dict(T=-1),
                dict(sl=None), dict(po=None), dict(rq=None), dict(cl=None), dict(nl=None), dict(tb=None), dict(cq=None), dict(kl=None),
                dict(us=None), dict(kl=p), dict(kl=2 * p), dict(cq=p), dict(T=2 ** 31 - 2)):
        assert call(**bad) == ERR_ARG, bad


def test_rotary_refusals():
    L, p = sb200.lib(), 0x1000
    _, r = _plan(64)
    ref = ctypes.byref(r)
    ok = dict(x=p, y=p, type=1, T=3, H=2, HD=64, pos=p, plan=ref, yt=128, yh=64)

    def call(**kw):
        a = dict(ok, **kw)
        return L.sb_rotary(a["x"], 128, 64, a["y"], a["yt"], a["yh"], a["type"], a["T"], a["H"], a["HD"], a["pos"], a["plan"], 0, None)
    for bad in (dict(type=3), dict(T=-1), dict(H=0), dict(HD=62), dict(HD=65), dict(x=None), dict(y=None), dict(pos=None), dict(plan=None),
                dict(plan=ctypes.byref(sb200._RotaryPlan())), dict(x=p + 1),
                dict(yt=256), dict(yh=72)):  # in place with other strides
        assert call(**bad) == ERR_ARG, bad

    def kv(pages, **kw):
        a = dict(dict(q=p, o=p, k=p, v=p, pos=p, slots=p, T=2, NH=4), **kw)
        return L.sb_rotary_kv(a["q"], 256, 64, a["o"], 256, 64, a["k"], 128, 64, a["v"], 128, 64, a["T"], a["NH"], a["pos"], a["slots"], ref,
                              None if pages is None else ctypes.byref(pages), None)
    for pages in (None, _pages(k=None), _pages(type=7), _pages(n_pages=0), _pages(page=0), _pages(NKV=0), _pages(HD=32),
                  _pages(page_stride=-1)):
        assert kv(pages) == ERR_ARG
    for bad in (dict(q=None), dict(o=None), dict(k=None), dict(v=None), dict(pos=None), dict(slots=None), dict(NH=0), dict(k=p + 1)):
        assert kv(_pages(), **bad) == ERR_ARG, bad


def test_attn_prefix_refusals():
    L, p = sb200.lib(), 0x1000
    ok = dict(q=p, q_row=256, q_head=64, out=p, lse=p, T=3, NH=4, cu=p, B=2, max_q=2, pre=_pages(), pt=p, P=64, kv=_pages(), tb=p, stride=4,
              kl=p, max_kv=64, scale=0.125, ws=p, wsb=1 << 30)

    def call(**kw):
        a = dict(ok, **kw)
        ref = lambda x: None if x is None else ctypes.byref(x)  # noqa: E731
        return L.sb_attn_prefix(a["q"], a["q_row"], a["q_head"], a["out"], 256, 64, a["lse"], a["T"], a["NH"], a["cu"], a["B"], a["max_q"],
                                ref(a["pre"]), a["pt"], a["P"], ref(a["kv"]), a["tb"], a["stride"], a["kl"], a["max_kv"], a["scale"],
                                a["ws"], a["wsb"], None)
    for bad in (dict(pre=None), dict(kv=None), dict(pre=_pages(type=5)), dict(kv=_pages(type=0)), dict(kv=_pages(NKV=1)),
                dict(kv=_pages(HD=32)), dict(NH=3), dict(NH=0), dict(T=-1), dict(B=-1), dict(max_q=0), dict(P=-1), dict(max_kv=-1),
                dict(cu=None), dict(cu=None, T=2), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=3e38), dict(pre=None, kv=None, P=0, max_kv=0),
                dict(kv=_pages(page=2 ** 31 - 1), stride=0),  # the table's width in 64 bits
                dict(q=None), dict(out=None),
                dict(q=p + 8), dict(q_row=252), dict(q_head=60), dict(lse=p + 2), dict(tb=None), dict(kl=None), dict(stride=3),
                dict(pt=None, P=129), dict(pre=_pages(HD=136), kv=_pages(HD=136)), dict(pre=_pages(HD=12), kv=_pages(HD=12)),
                dict(pre=_pages(k=0x10008)), dict(kv=_pages(pos_stride=132)), dict(kv=_pages(v=0x20004))):
        assert call(**bad) == ERR_ARG, bad
    n = ctypes.c_size_t()
    assert L.sb_attn_prefix_ws(1, 3, 2, 4, 2, 64, 2, 64, 64, None) == ERR_ARG
    assert L.sb_attn_prefix_ws(9, 3, 2, 4, 2, 64, 2, 64, 64, ctypes.byref(n)) == ERR_ARG
    assert L.sb_attn_prefix_ws(1, 3, 2, 4, 3, 64, 2, 64, 64, ctypes.byref(n)) == ERR_ARG
    assert L.sb_attn_prefix_ws(1, 0, 0, 4, 2, 64, 2, 64, 64, ctypes.byref(n)) == 0 and n.value == 0


def test_logprobs_refusals():
    L, p, n = sb200.lib(), 0x1000, ctypes.c_size_t()
    ok = dict(x=p, stride=100, type=0, R=2, V=100, temp=1.0, tok=p, logp=p, rank=p, k=5, ids=p, top=p)

    def call(**kw):
        a = dict(ok, **kw)
        return L.sb_logprobs(a["x"], a["stride"], a["type"], a["R"], a["V"], a["temp"], a["tok"], a["logp"], p, p, a["rank"], a["k"], a["ids"],
                             a["top"], p, 1 << 30, None)
    for bad in (dict(type=4), dict(R=-1), dict(V=0), dict(V=4), dict(k=-1), dict(k=65), dict(temp=0.0), dict(temp=-1.0),
                dict(temp=float("nan")), dict(temp=1e-45), dict(temp=9e-9), dict(tok=None), dict(ids=None, top=None), dict(x=None), dict(x=p + 2),
                dict(stride=99)):
        assert call(**bad) == ERR_ARG, bad
    assert L.sb_logprobs_ws(0, 2, 100, 101, ctypes.byref(n)) == ERR_ARG and L.sb_logprobs_ws(0, 2, 100, 5, None) == ERR_ARG

    def grad(**kw):
        a = dict(dict(x=p, xs=100, type=0, R=2, V=100, temp=1.0, tok=p, lse=p, ent=p, gl=p, ge=p, g=0x9000, gs=100), **kw)
        return L.sb_logprobs_grad(a["x"], a["xs"], a["type"], a["R"], a["V"], a["temp"], a["tok"], a["lse"], a["ent"], a["gl"], a["ge"], a["g"],
                                  a["gs"], None)
    for bad in (dict(type=3), dict(V=0), dict(temp=0.0), dict(temp=9e-9), dict(tok=None), dict(x=None), dict(lse=None), dict(ent=None), dict(g=None),
                dict(xs=99), dict(gs=99), dict(g=0x9001), dict(g=p, xs=100, gs=104)):
        assert grad(**bad) == ERR_ARG, bad


def test_binding_refuses_wrong_tensors():
    """Types, shapes, layouts and devices that a kernel would misread."""
    h = torch.zeros(4, 2, 64, dtype=torch.float16)
    pages = torch.zeros(3, 16, 2, 64, dtype=torch.float16)
    i32, i64 = torch.zeros(8, dtype=torch.int32), torch.zeros(8, dtype=torch.int64)
    plan = sb200.Rotary(64)
    kv = sb200.KvPages(pages, pages.clone())
    bad = [
        lambda: sb200.KvPages(pages, pages.float()),
        lambda: sb200.KvPages(pages, pages[:2]),
        lambda: sb200.KvPages(pages.transpose(2, 3), pages.transpose(2, 3)),
        lambda: sb200.KvPages(pages.double(), pages.double()),
        lambda: sb200.Rotary(63),
        lambda: sb200.rotary(h, h.float(), i32, plan),
        lambda: sb200.rotary(h, h, i64, plan),
        lambda: sb200.rotary(h, h, i32[:3], plan),
        lambda: sb200.rotary(h, h, i32, plan),  # CPU tensors
        lambda: sb200.rotary_kv(h, h, h, h, i32, i32, plan, kv),
        lambda: sb200.rotary_kv(h, h, h[:, :1], h[:, :1], i32, i64, plan, kv),
        lambda: sb200.rotary_kv(h, h, h, h, i32, i64, plan, kv),
        lambda: sb200.attn_prefix(h, h, kv, i32, 16, kv, i32.view(4, 2), i32, 0.125, None, max_kv=33),
        lambda: sb200.attn_prefix(h, h, kv, i32, 16, kv, i32.view(4, 2), i64, 0.125, None, max_kv=32),
        lambda: sb200.attn_prefix(h, h, kv, i32[:1], 17, None, None, None, 0.125, None),
        lambda: sb200.attn_prefix(h, h, None, None, 0, None, None, None, 0.125, None),
        lambda: sb200.attn_prefix(h, h, kv, i32, 16, None, None, None, 0.125, None),
        lambda: sb200.kv_plan(i32, i32, i32, i32.view(2, 4), 16, i64, i32, i32, i32, i32, i32),
        lambda: sb200.kv_plan(i32[:2], i32, i32, i32.view(2, 4), 16, i32, i32, i32, i32, i32, i32),
        lambda: sb200.logprobs(h[0].t(), i32, None),
        lambda: sb200.logprobs(h[0], i64, None),
        lambda: sb200.logprobs(h[0], i32, None, lse=torch.zeros(1)),
        lambda: sb200.logprobs(h[0], i32, None, top_ids=torch.zeros(2, 3, dtype=torch.int32), top_logp=torch.zeros(2, 4)),
        lambda: sb200.logprobs_grad(h[0], i32, torch.zeros(2), None, None, None, h[0].float()),
    ]
    assert sb200._ws(torch.zeros(8))[1] == 32 and sb200._ws(None) == (None, 0)
    bad.append(lambda: sb200._ws(torch.zeros(8)[::2]))  # its bytes are not in one piece
    for i, f in enumerate(bad):
        with pytest.raises(sb200.SbError):
            f()
            pytest.fail(f"call {i} was accepted")


def test_fixed_point_phase_against_double():
    """pos x turn modulo 2^64 is the phase of the last turn: to 1e-9 turns of
    a quotient taken in 128-bit integers at positions up to 2^31 - 1."""
    r = _plan(64, theta=1e6)[1]
    for i in (0, 5, 17, 31):
        f = np.longdouble(1e6) ** np.longdouble(-2.0 * i / 64) / (2 * np.longdouble("3.14159265358979323846264338327950288"))
        for pos in (1, 8191, 1048575, 2 ** 31 - 1):
            want = (f * pos) % 1
            got = np.longdouble((pos * r.turn[i]) % 2 ** 64) / np.longdouble(2.0 ** 64)
            d = abs(float(got - want))
            assert min(d, 1 - d) < pos * 2.0 ** -52  # pow in double: half an ulp of f <= 1/6


def test_rotary_kv_in_place_needs_one_set_of_strides():
    L, p = sb200.lib(), 0x1000
    _, r = _plan(64)
    pages = _pages()
    for tok, head in ((512, 64), (256, 128)):
        assert L.sb_rotary_kv(p, 256, 64, p, tok, head, 2 * p, 128, 64, 3 * p, 128, 64, 2, 4, 4 * p, 5 * p, ctypes.byref(r),
                              ctypes.byref(pages), None) == ERR_ARG


def test_attn_test_skip_refusals():
    L = sb200.lib()
    assert L.sb_attn_set_test_skip(-2) == ERR_ARG and L.sb_attn_set_test_skip(1 << 30) == ERR_ARG
    assert L.sb_attn_set_test_skip(3) == 0 and L.sb_attn_set_test_skip(-1) == 0


def test_kv_plan_indexes_nothing_outside(tmp_path):
    """The kernel's own source on the host, under the address sanitizer:
    hostile lengths (sums past 2^31, pages of 2^31 - 1) stay inside the
    tables, and ordinary ones give the plan."""
    here = os.path.dirname(os.path.abspath(__file__))
    text = open(os.path.join(here, "..", "switch-l4t-gpu_b200", "csrc", "serve_plan.cuh")).read()
    for was, now in (('#include "sb_common.cuh"\n', ""), ("extern __shared__ int plan_sm[];", "int *plan_sm = shared_ints;")):
        assert text.count(was) == 1
        text = text.replace(was, now)
    source, binary = tmp_path / "plan.inc", tmp_path / "plan"
    source.write_text(text)
    build = ["g++", "-std=c++17", "-O1", "-g", "-fwrapv", "-w", f'-DPLAN_SOURCE="{source}"', os.path.join(here, "plan_emulation.cpp"), "-o", str(binary)]
    probe = tmp_path / "probe.cpp"
    probe.write_text("int main() { return 0; }\n")
    if subprocess.run(["g++", "-fsanitize=address", str(probe), "-o", str(tmp_path / "probe")], capture_output=True).returncode:
        pytest.skip("no address sanitizer")
    subprocess.run(build + ["-fsanitize=address"], check=True)
    env = dict(os.environ, ASAN_OPTIONS="detect_stack_use_after_return=0:detect_leaks=0")
    run = subprocess.run([str(binary), "3000"], capture_output=True, text=True, env=env, timeout=120)
    assert run.returncode == 0 and run.stdout == "3000 cases\n", (run.stdout + run.stderr)[-3000:]


@pytest.mark.parametrize("dim,theta,factor,orig", [(64, 1e6, 8.0, 4096), (128, 1e4, 3.7, 2048), (80, 500000.0, 32.0, 8192), (6, 1.5, 2.0, 100)])
def test_rotary_plan_frequencies_in_long_double(dim, theta, factor, orig):
    """Against 50 digits: powl, a product or quotient or four of a blend, each
    within 2^-64 relative, and the fraction's own half unit."""
    D, pi = decimal.Decimal, decimal.Decimal("3.14159265358979323846264338327950288419716939937510")
    with decimal.localcontext() as ctx:
        ctx.prec = 50
        th, k = D(theta), D(factor)
        for scaling in range(5):
            rc, r = _plan(dim, theta=theta, scaling=scaling, factor=factor, orig=orig)
            assert rc == 0
            lo = max(math.floor(dim * math.log(orig / (64 * math.pi)) / (2 * math.log(theta))), 0)
            hi = min(math.ceil(dim * math.log(orig / (2 * math.pi)) / (2 * math.log(theta))), dim - 1)
            for i in range(dim // 2):
                base = th * k ** (D(dim) / D(dim - 2)) if scaling == 2 else th
                f = base ** (D(-2 * i) / D(dim))
                if scaling == 1:
                    f /= k
                if scaling == 3:
                    ramp = min(max(D(i - lo) / (D(hi - lo) if hi > lo else D("0.001")), D(0)), D(1))
                    f = f / k * ramp + f * (1 - ramp)
                if scaling == 4:
                    s = min(max((orig * f / (2 * pi) - 1) / 3, D(0)), D(1))
                    f = f / k * (1 - s) + f * s
                turns = f / (2 * pi) * D(2) ** 64
                # the blends: s is off by up to 4 relative units of a number of turns up to 4, and multiplies f
                assert abs(D(int(r.turn[i])) - turns) <= turns * D(2) ** (-62 if scaling != 4 else -60) + D("0.51"), (scaling, i)
