"""What the operators on caches in pages refuse, on the CPU: the public entry points by exceptions before anything is launched, the C
entry points by their codes, sizes of workspaces, and properties of the built kernels."""
import re

import pytest
import torch

import build
import slotattn_hip as A
import slotpage_hip as P
import slotrope_hip as R
import slotscan_lib as L

BF, F, I32, I64 = torch.bfloat16, torch.float32, torch.int32, torch.int64
z = lambda *s, dt=BF: torch.zeros(*s, dtype=dt)
i32 = lambda *x: torch.tensor(x, dtype=I32)
SHAPE, DTYPE, NULL, ALIGN = 1, 2, 3, 4
X = 1 << 20                                              # an aligned address that is never read


def _state(R=3, M=2, Pn=4):
    return z(R, dt=I32), z(R, M, dt=I32), z(Pn + 1, dt=I32)


@pytest.mark.parametrize("kw,err", [
    ({}, RuntimeError),                                               # CPU tensors: no silent fallback
    (dict(new=z(3, dt=I64)), ValueError), (dict(new=z(2, dt=I32)), ValueError), (dict(new=z(6, dt=I32)[::2]), ValueError),
    (dict(lens=z(3, dt=I64)), ValueError), (dict(lens=z(4, dt=I32)), ValueError),
    (dict(table=z(3, 2, dt=I64)), ValueError), (dict(table=z(3, dt=I32)), ValueError), (dict(table=z(2, 3, dt=I32).t()), ValueError),
    (dict(table=z(1, 2, dt=I32).expand(3, 2)), ValueError),           # rows that share memory
    (dict(table=z(3, 0, dt=I32)), ValueError),
    (dict(free=z(0, dt=I32)), ValueError), (dict(free=z(5, 1, dt=I32)), ValueError), (dict(free=z(5, dt=I64)), ValueError),
    (dict(page=0), ValueError), (dict(page=8), ValueError), (dict(page=48), ValueError), (dict(page=8192), ValueError), (dict(page=-16), ValueError),
    (dict(N=-1), ValueError),
])
def test_page_extend_and_trim_refuse(kw, err):
    lens, table, free = _state()
    a = dict(new=z(3, dt=I32), lens=lens, table=table, free=free, page=16, N=4)
    a.update(kw)
    with pytest.raises(err, match="page_extend"):
        P.page_extend(**a)
    if "N" not in kw:
        a.pop("N")
        a["keep"] = a.pop("new")
        with pytest.raises(err, match="page_trim"):
            P.page_trim(**a)


def _rope(**kw):
    a = dict(q=z(5, 4, 64), k=z(5, 2, 64), v=z(5, 2, 64), wq=None, wk=None, freqs=R.frequencies(64), pos=z(5, dt=I32), slots=z(5, dt=I64),
             kpages=z(3, 2, 16, 64), vpages=z(3, 2, 16, 64))
    a.update(kw)
    return R.qk_rope_pages(**a)


_both = z(3, 2, 2, 16, 64)


@pytest.mark.parametrize("kw,err", [
    ({}, RuntimeError),
    (dict(q=z(1, 5, 4, 64)), ValueError), (dict(k=z(4, 2, 64)), ValueError), (dict(k=z(5, 2, 128)), ValueError),
    (dict(v=z(5, 3, 64)), ValueError), (dict(v=z(5, 2, 64, dt=F)), ValueError), (dict(k=z(5, 2, 64, dt=F), v=z(5, 2, 64, dt=F)), NotImplementedError),
    (dict(q=z(5, 4, 64, dt=torch.float64), k=z(5, 2, 64, dt=torch.float64)), NotImplementedError),
    (dict(wq=z(63)), ValueError), (dict(freqs=R.frequencies(64).float()), ValueError), (dict(freqs=R.frequencies(64)[:5]), NotImplementedError),
    (dict(pos=z(5, dt=I64)), ValueError), (dict(pos=z(4, dt=I32)), ValueError), (dict(slots=z(5, dt=I32)), ValueError), (dict(slots=z(10, dt=I64)[::2]), ValueError),
    (dict(kpages=z(3, 2, 16, 64, dt=F), vpages=z(3, 2, 16, 64, dt=F)), NotImplementedError),
    (dict(kpages=z(3, 3, 16, 64), vpages=z(3, 3, 16, 64)), ValueError), (dict(vpages=z(2, 2, 16, 64)), ValueError),
    (dict(kpages=z(3, 2, 24, 64), vpages=z(3, 2, 24, 64)), ValueError), (dict(kpages=z(0, 2, 16, 64), vpages=z(0, 2, 16, 64)), ValueError),
    (dict(kpages=_both[:, 0], vpages=_both[:, 0]), ValueError),       # one cache for both
    (dict(kpages=z(1, 2, 16, 64).expand(3, 2, 16, 64)), ValueError),  # pages that share memory
    (dict(kpages=z(3, 2, 16, 128)[..., ::2]), ValueError),
    (dict(q=z(5, 4, 64).requires_grad_()), RuntimeError),
])
def test_qk_rope_pages_refuses(kw, err):
    with pytest.raises(err, match="qk_rope_pages"):
        _rope(**kw)


def _attend(**kw):
    a = dict(q=z(5, 4, 64), kpages=z(3, 2, 16, 64), vpages=z(3, 2, 16, 64), table=z(2, 3, dt=I32), starts=i32(0, 2, 5), ends=i32(2, 9))
    a.update(kw)
    return A.attend_pages(**a)


@pytest.mark.parametrize("kw,err", [
    ({}, RuntimeError),
    (dict(q=z(1, 5, 4, 64)), ValueError), (dict(q=z(5, 3, 64)), ValueError), (dict(q=z(5, 4, 128)), ValueError),
    (dict(q=z(5, 4, 64, dt=F), kpages=z(3, 2, 16, 64, dt=F), vpages=z(3, 2, 16, 64, dt=F)), NotImplementedError),
    (dict(q=z(5, 4, 64, dt=torch.float16)), NotImplementedError),
    (dict(q=z(5, 4, 96), kpages=z(3, 2, 16, 96), vpages=z(3, 2, 16, 96)), NotImplementedError),
    (dict(vpages=z(4, 2, 16, 64)), ValueError), (dict(kpages=z(3, 2, 8, 64), vpages=z(3, 2, 8, 64)), ValueError),
    (dict(kpages=z(3, 2, 17, 64), vpages=z(3, 2, 17, 64)), ValueError), (dict(kpages=z(3, 2, 64), vpages=z(3, 2, 64)), ValueError),
    (dict(kpages=z(3, 2, 16, 128)[..., ::2]), ValueError),            # rows that are not contiguous: a pool is not copied
    (dict(table=z(2, 3, dt=I64)), ValueError), (dict(table=z(6, dt=I32)), ValueError), (dict(table=z(3, 2, dt=I32).t()), ValueError),
    (dict(starts=i32(0, 2)), ValueError), (dict(starts=torch.tensor([0, 2, 5])), ValueError), (dict(ends=i32(1)), ValueError), (dict(ends=z(2)), ValueError),
    (dict(most=-1), ValueError), (dict(window=0), ValueError), (dict(cap=0.0), ValueError), (dict(cap=float("nan")), ValueError), (dict(scale=0.0), ValueError),
    (dict(slopes=z(4)), ValueError), (dict(slopes=z(2, dt=F)), ValueError), (dict(slopes=z(4, dt=F).requires_grad_()), NotImplementedError),
    (dict(prefix=i32(1)), ValueError), (dict(prefix=torch.tensor([1, 2])), ValueError),
    (dict(q=z(5, 4, 64).requires_grad_()), RuntimeError), (dict(kpages=z(3, 2, 16, 64).requires_grad_()), RuntimeError),
])
def test_attend_pages_refuses(kw, err):
    with pytest.raises(err, match="attend_pages"):
        _attend(**kw)


def _extend_c(**o):
    a = dict(new=X, lens=X, table=X, tsr=4, free=X, R=3, M=4, P=9, page=16, N=8, starts=X, ends=X, slots=X, pos=X)
    a.update(o)
    return L.lib().slotpage_extend(a["new"], a["lens"], a["table"], a["tsr"], a["free"], a["R"], a["M"], a["P"], a["page"], a["N"], a["starts"], a["ends"],
                                   a["slots"], a["pos"], None)


@pytest.mark.parametrize("o,code", [
    (dict(R=0), SHAPE), (dict(M=0), SHAPE), (dict(P=-1), SHAPE), (dict(page=8), SHAPE), (dict(page=24), SHAPE), (dict(page=8192), SHAPE), (dict(page=0), SHAPE),
    (dict(tsr=3), SHAPE), (dict(R=1 << 25), SHAPE), (dict(P=1 << 30), SHAPE), (dict(M=1 << 27, tsr=1 << 27), SHAPE), (dict(N=-1), SHAPE), (dict(N=1 << 30), SHAPE),
    (dict(new=None), NULL), (dict(lens=None), NULL), (dict(table=None), NULL), (dict(free=None), NULL), (dict(starts=None), NULL), (dict(ends=None), NULL),
    (dict(slots=None), NULL), (dict(pos=None), NULL),
])
def test_extend_codes(o, code):
    assert _extend_c(**o) == code and L.lib().slotscan_last_error()


@pytest.mark.parametrize("o,code", [(dict(R=0), SHAPE), (dict(page=20), SHAPE), (dict(tsr=1), SHAPE), (dict(keep=None), NULL), (dict(free=None), NULL)])
def test_trim_codes(o, code):
    a = dict(keep=X, lens=X, table=X, tsr=4, free=X, R=3, M=4, P=9, page=16)
    a.update(o)
    assert L.lib().slotpage_trim(a["keep"], a["lens"], a["table"], a["tsr"], a["free"], a["R"], a["M"], a["P"], a["page"], None) == code
    assert L.lib().slotscan_last_error()


@pytest.mark.parametrize("o,code", [
    (dict(N=0), SHAPE), (dict(Hq=0), SHAPE), (dict(D=96), SHAPE), (dict(rot=24), SHAPE), (dict(P=0), SHAPE), (dict(page=8), SHAPE), (dict(page=48), SHAPE),
    (dict(dt=5), DTYPE), (dict(q=None), NULL), (dict(v=None), NULL), (dict(pos=None), NULL), (dict(slots=None), NULL), (dict(qo=None), NULL), (dict(kp=None), NULL),
    (dict(vp=None), NULL), (dict(kp=X + 8), ALIGN), (dict(v=X + 2), ALIGN), (dict(st=130), ALIGN), (dict(kst=66), ALIGN),
])
def test_rope_pages_codes(o, code):
    a = dict(q=X, k=X, v=X, st=512, dt=1, f=X, rot=64, pos=X, slots=X, N=4, Hq=4, Hk=2, D=64, P=3, page=16, qo=X, kp=X, vp=X, kst=64)
    a.update(o)
    s = (64, a["st"])
    assert L.lib().slotrope_pages(a["q"], *s, a["k"], *s, a["v"], *s, a["dt"], None, None, 0, a["f"], a["rot"], 0, a["pos"], a["slots"], a["N"], a["Hq"], a["Hk"],
                                  a["D"], a["P"], a["page"], 1e-6, a["qo"], a["kp"], 2048, 1024, a["kst"], a["vp"], 2048, 1024, 64, None) == code
    assert L.lib().slotscan_last_error()


@pytest.mark.parametrize("o,code", [
    (dict(N=0), SHAPE), (dict(R=0), SHAPE), (dict(M=0), SHAPE), (dict(P=0), SHAPE), (dict(page=8), SHAPE), (dict(page=40), SHAPE), (dict(Hq=3), SHAPE), (dict(D=80), SHAPE),
    (dict(most=0), SHAPE), (dict(window=0), SHAPE), (dict(cap=-1.0), SHAPE), (dict(scale=0.0), SHAPE), (dict(ksp=1 << 31), SHAPE), (dict(ksp=-8), SHAPE), (dict(tsr=-1), SHAPE),
    (dict(M=1 << 27), SHAPE), (dict(qst=1 << 25), SHAPE), (dict(dt=0), DTYPE), (dict(q=None), NULL), (dict(k=None), NULL), (dict(table=None), NULL),
    (dict(starts=None), NULL), (dict(ends=None), NULL), (dict(out=None), NULL), (dict(ws=None, M=4096, window=1 << 20), NULL), (dict(out=X + 8), ALIGN), (dict(ws=X + 4), ALIGN), (dict(k=X + 2), ALIGN),
    (dict(ksp=2044), ALIGN),
])
def test_attend_pages_codes(o, code):
    a = dict(q=X, qst=256, k=X, ksp=2048, v=X, dt=1, table=X, tsr=4, starts=X, ends=X, N=4, R=4, M=4, P=9, page=16, Hq=4, Hk=2, D=64, most=1, scale=0.125, window=100, cap=0.0,
             ws=X, out=X)
    a.update(o)
    assert L.lib().slotattn_pages(a["q"], 64, a["qst"], a["k"], a["ksp"], 1024, 64, a["v"], 2048, 1024, 64, a["dt"], a["table"], a["tsr"], a["starts"], a["ends"], a["N"], a["R"],
                                  a["M"], a["P"], a["page"], a["Hq"], a["Hk"], a["D"], a["most"], a["scale"], a["window"], a["cap"], None, None, a["ws"], a["out"], None) == code
    assert L.lib().slotscan_last_error()


def test_attend_pages_workspace():
    """Nothing where a row has few keys and a workgroup takes each unit; at most two pieces a worker otherwise; 0 for what the call refuses."""
    ws = L.lib().slotattn_pages_workspace
    none = 2 ** 31 - 1
    assert ws(4, 4, 8, 16, 4, 2, 64, 1, none, 0) == 0
    few, many = ws(32, 32, 512, 16, 12, 4, 128, 1, none, 0), ws(4096, 2, 512, 16, 12, 4, 128, 4096, none, 0)
    assert 1024 * 2 * 16 * 130 * 4 <= few < 1024 * 2 * 16 * 130 * 4 + 4096 and 512 * 2 * 128 * 130 * 4 <= many < 512 * 2 * 128 * 130 * 4 + 65536
    assert ws(32, 32, 512, 16, 12, 4, 128, 1, 64, 0) == 0             # a window leaves few keys
    for bad in ((0, 1, 1, 16, 1, 1, 64, 1, 1, 0), (1, 0, 1, 16, 1, 1, 64, 1, 1, 0), (1, 1, 0, 16, 1, 1, 64, 1, 1, 0), (1, 1, 1, 16, 3, 2, 64, 1, 1, 0),
                (1, 1, 1, 16, 1, 1, 64, 0, 1, 0), (1, 1, 1, 16, 1, 1, 64, 1, 0, 0)):
        assert ws(*bad) == 0


def test_counted_waits_have_no_scratch_accesses_between():
    """pages_few waits for its direct global -> LDS loads by counts of the vector-memory operations behind them; a spill's accesses would
    not make a wait too short, but each would wait for loads that are not needed yet."""
    kern = {k: d for k, d in build.resource_report("slotattn_few.hip").items() if "pages_few" in k}
    assert len(kern) == 64, sorted(kern)
    for k, d in kern.items():
        assert d["ScratchSize [bytes/lane]"] == "0", f"{k} uses scratch: {d}"
