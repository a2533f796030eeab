"""What the attention and the preparation of its operands refuse, on the CPU: the public entry points by exceptions before
anything is launched, the C entry points by their codes, and properties of the built kernels."""
import ctypes
import re

import pytest
import torch

import build
import slotattn_hip as A
import slotrope_hip as R
import slotscan_lib as L

BF, F = torch.bfloat16, torch.float32
z = lambda *s, dt=BF: torch.zeros(*s, dtype=dt)
i32 = lambda *x: torch.tensor(x, dtype=torch.int32)


def _qkv(B=2, Hq=4, Hk=2, Tq=5, Tk=5, D=64, dt=BF):
    return z(B, Hq, Tq, D, dt=dt), z(B, Hk, Tk, D, dt=dt), z(B, Hk, Tk, D, dt=dt)


@pytest.mark.parametrize("args,kw,err", [
    (_qkv(), {}, RuntimeError),                                       # CPU tensors: no silent fallback
    (_qkv(dt=F), {}, NotImplementedError),
    (_qkv(D=96), {}, NotImplementedError),
    (_qkv(Hq=3), {}, ValueError),
    (_qkv(Tq=6), {}, ValueError),                                     # more queries than keys
    ((z(2, 4, 5), *_qkv()[1:]), {}, ValueError),
    ((*_qkv()[:2], z(2, 2, 4, 64)), {}, ValueError),
    ((_qkv(B=1)[0], *_qkv()[1:]), {}, ValueError),
    ((*_qkv()[:2], _qkv(dt=torch.float16)[2]), {}, NotImplementedError),
    (_qkv(), dict(window=0), ValueError),
    (_qkv(), dict(window=-3), ValueError),
    (_qkv(), dict(cap=0.0), ValueError),
    (_qkv(), dict(cap=-1.0), ValueError),
    (_qkv(), dict(cap=float("nan")), ValueError),
    (_qkv(), dict(cap=float("inf")), ValueError),
    (_qkv(), dict(scale=0.0), ValueError),
    (_qkv(), dict(scale=float("nan")), ValueError),
    (_qkv(), dict(slopes=z(4)), ValueError),
    (_qkv(), dict(slopes=z(2, dt=F)), ValueError),
    (_qkv(), dict(slopes=z(4, dt=F).requires_grad_()), NotImplementedError),
    (_qkv(), dict(prefix=i32(1)), ValueError),
    (_qkv(), dict(prefix=torch.tensor([1, 2])), ValueError),
    (_qkv(), dict(docs=torch.zeros(2, 4, dtype=torch.int32)), ValueError),
    (_qkv(), dict(docs=torch.zeros(2, 5, dtype=torch.int64)), ValueError),
])
def test_attend_refuses(args, kw, err):
    with pytest.raises(err, match="attend"):
        A.attend(*args, **kw)


@pytest.mark.parametrize("args,kw,err", [
    ((*_qkv(), i32(1, 2)), {}, RuntimeError),
    ((*_qkv(), torch.tensor([1, 2])), {}, ValueError),
    ((*_qkv(), i32(1)), {}, ValueError),
    ((*_qkv(), i32(1, 0, 2)[::2]), {}, ValueError),                   # not contiguous
    ((*_qkv(Tk=0), i32(0, 0)), {}, ValueError),                       # a cache without rows
    ((*_qkv(), i32(1, 2)), dict(window=0), ValueError),
    ((_qkv()[0].requires_grad_(), *_qkv()[1:], i32(1, 2)), {}, RuntimeError),
])
def test_attend_cache_refuses(args, kw, err):
    with pytest.raises(err, match="attend_cache"):
        A.attend_cache(*args, **kw)


FR = R.frequencies(64)


@pytest.mark.parametrize("args,kw,err", [
    ((*_qkv()[:2], None, None, FR), {}, RuntimeError),
    ((*_qkv(D=80)[:2], None, None, FR), {}, NotImplementedError),
    ((*_qkv(dt=torch.float64)[:2], None, None, FR), {}, NotImplementedError),
    ((_qkv()[0], _qkv(Tk=6)[1], None, None, FR), {}, ValueError),
    ((_qkv()[0], z(2, 0, 5, 64), None, None, FR), {}, ValueError),
    ((*_qkv()[:2], z(63), None, FR), {}, ValueError),
    ((*_qkv()[:2], None, z(64, dt=torch.float64), FR), {}, ValueError),
    ((*_qkv()[:2], None, None, FR.float()), {}, ValueError),
    ((*_qkv()[:2], None, None, FR[:5]), {}, NotImplementedError),
    ((*_qkv()[:2], None, None, R.frequencies(128)), {}, NotImplementedError),
    ((*_qkv()[:2], None, None, FR.clone().requires_grad_()), {}, NotImplementedError),
    ((*_qkv()[:2], None, None, FR), dict(positions=torch.arange(4)), ValueError),
    ((*_qkv()[:2], None, None, FR), dict(positions=torch.arange(5.0)), ValueError),
])
def test_qk_rope_refuses(args, kw, err):
    with pytest.raises(err, match="qk_rope"):
        R.qk_rope(*args, **kw)


def _cache_args(**over):
    q, k, v = _qkv()
    a = dict(q=q, k=k, v=v, wq=None, wk=None, freqs=FR, lens=i32(5, 5), kcache=z(2, 2, 9, 64), vcache=z(2, 2, 9, 64))
    a.update(over)
    return a


@pytest.mark.parametrize("over,err", [
    ({}, RuntimeError),
    (dict(v=z(2, 2, 4, 64)), ValueError),
    (dict(v=z(2, 2, 5, 64, dt=F)), ValueError),
    (dict(kcache=z(2, 2, 9, 64, dt=F)), NotImplementedError),
    (dict(vcache=z(2, 2, 8, 64)), ValueError),
    (dict(kcache=z(3, 2, 9, 64), vcache=z(3, 2, 9, 64)), ValueError),
    (dict(kcache=z(2, 1, 9, 64).expand(2, 2, 9, 64)), ValueError),    # rows that share memory
    (dict(vcache=z(2 * 2 * 9 * 64).as_strided((2, 2, 9, 64), (64, 576, 64, 1))), ValueError),
    (dict(kcache=z(2, 2, 9, 65)[..., :64]), ValueError),              # rows that are not aligned
    (dict(kcache=z(2, 2, 64, 9).transpose(2, 3)), ValueError),
    (dict(lens=torch.tensor([5, 5])), ValueError),
    (dict(wk=z(64).requires_grad_()), RuntimeError),
])
def test_qk_rope_cache_refuses(over, err):
    with pytest.raises(err, match="qk_rope_cache"):
        R.qk_rope_cache(**_cache_args(**over))


@pytest.mark.parametrize("shape,order", [((2, 3, 9, 64), (0, 1, 2, 3)), ((2, 9, 3, 64), (0, 2, 1, 3)), ((9, 2, 3, 64), (1, 2, 0, 3)),
                                         ((2, 9, 2, 3, 64), None)])
def test_layouts_of_a_cache(shape, order):
    c = z(*shape)
    c = c[:, :, 0].transpose(1, 2) if order is None else c.permute(order)
    assert R._apart(c) and L.in_place(c) and c.shape == (2, 3, 9, 64)


P = 1 << 20


def _fwd(**o):
    a = dict(q=P, qs=(512, 64, 128), k=P, ks=(512, 64, 128), v=P, vs=(512, 64, 128), dt=1, B=1, Tq=4, Tk=4, Hq=2, Hk=2, D=64, scale=0.1, causal=1,
             W=5, cap=0.0, slopes=None, docs=None, prefix=None, lens=None, ws=None, out=P, res=None, lse=None)
    a.update(o)
    return L.lib().slotattn_fwd(a["q"], *a["qs"], a["k"], *a["ks"], a["v"], *a["vs"], a["dt"], a["B"], a["Tq"], a["Tk"], a["Hq"], a["Hk"], a["D"],
                                a["scale"], a["causal"], a["W"], a["cap"], a["slopes"], a["docs"], a["prefix"], a["lens"], a["ws"], a["out"],
                                a["res"], a["lse"], None)


def _bwd(**o):
    a = dict(q=P, st=128, dt=1, B=1, Tq=4, Tk=4, Hq=2, Hk=2, D=64, out=P, res=P, lse=P, do=P, dost=128, ws=None, delta=P, dq=P, dk=P, dv=P)
    a.update(o)
    s = (512, 64, a["st"])
    return L.lib().slotattn_bwd(a["q"], *s, P, *s, P, *s, a["dt"], a["B"], a["Tq"], a["Tk"], a["Hq"], a["Hk"], a["D"], 0.1, 1, 5, 0.0, None, None,
                                None, a["out"], a["res"], a["lse"], a["do"], 512, 64, a["dost"], a["ws"], a["delta"], a["dq"], a["dk"], a["dv"],
                                None)


SHAPE, DTYPE, NULL, ALIGN = 1, 2, 3, 4


@pytest.mark.parametrize("over,code", [
    (dict(B=0), SHAPE), (dict(Tq=0), SHAPE), (dict(Tk=0), SHAPE), (dict(Hq=3), SHAPE), (dict(D=32), SHAPE), (dict(W=0), SHAPE),
    (dict(Tq=5), SHAPE), (dict(cap=-1.0), SHAPE), (dict(cap=float("nan")), SHAPE), (dict(scale=0.0), SHAPE), (dict(Tk=1 << 30), SHAPE),
    (dict(B=1 << 31), SHAPE), (dict(ks=(512, 64, 1 << 25)), SHAPE), (dict(vs=(512, 64, -128)), SHAPE), (dict(lens=P, docs=P), SHAPE),
    (dict(lens=P, causal=0), SHAPE), (dict(dt=0), DTYPE), (dict(dt=9), DTYPE), (dict(k=None), NULL), (dict(out=None), NULL),
    (dict(q=P + 2), ALIGN), (dict(ks=(512, 64, 132)), ALIGN), (dict(out=P + 8), ALIGN), (dict(docs=P + 4), ALIGN),
    (dict(Tq=1, Tk=9000, W=9000), NULL),                              # split keys without a workspace
])
def test_attention_forward_codes(over, code):
    assert _fwd(**over) == code and L.lib().slotscan_last_error()


@pytest.mark.parametrize("over,code", [
    (dict(B=0), SHAPE), (dict(Tq=5), SHAPE), (dict(st=1 << 25), SHAPE), (dict(dost=-8), SHAPE), (dict(dt=0), DTYPE), (dict(q=None), NULL),
    (dict(res=None), NULL), (dict(lse=None), NULL), (dict(dv=None), NULL), (dict(delta=None), NULL), (dict(dq=P + 8), ALIGN), (dict(dost=129), ALIGN),
])
def test_attention_backward_codes(over, code):
    assert _bwd(**over) == code and L.lib().slotscan_last_error()


def test_documents_codes_and_sizes():
    f = L.lib().slotattn_docs
    assert f(None, 1, 5, P, None) == NULL and f(P, 0, 5, P, None) == SHAPE and f(P, 70000, 5, P, None) == SHAPE and f(P, 1, 5, P + 4, None) == ALIGN
    assert L.lib().slotattn_docs_bytes(3, 65) == 3 * 2 * (64 * 4 + 8) and L.lib().slotattn_docs_bytes(0, 5) == 0


def test_counted_waits_have_no_scratch_accesses_between():
    """attn_split and attn_dkv wait for their direct global -> LDS loads by counts of the vector-memory operations behind
    them; a spill's accesses would not make a wait too short, but each would wait for loads that are not needed yet."""
    for src, name, n in (("slotattn.hip", "attn_split", 16), ("slotattn.hip", "attn_fwd", 32), ("slotattn_bwd.hip", "attn_dkv", 16)):
        rep = build.resource_report(src)
        kern = {k: d for k, d in rep.items() if re.search(name, k)}
        assert len(kern) == n, sorted(rep)
        for k, d in kern.items():
            assert d["ScratchSize [bytes/lane]"] == "0", f"{k} uses scratch: {d}"


def _rope(**o):
    a = dict(q=P, st=128, k=P, dt=1, wq=P, wk=P, wt=1, f=P, rot=64, pos=None, B=1, T=4, Hq=2, Hk=2, D=64, qo=P, ko=P)
    a.update(o)
    s = (512, 64, a["st"])
    return L.lib().slotrope_fwd(a["q"], *s, a["k"], *s, a["dt"], a["wq"], a["wk"], a["wt"], a["f"], a["rot"], 0, a["pos"], 0, 0, a["B"], a["T"],
                                a["Hq"], a["Hk"], a["D"], 1e-6, a["qo"], a["ko"], None)


@pytest.mark.parametrize("over,code", [
    (dict(B=0), SHAPE), (dict(T=0), SHAPE), (dict(Hq=0), SHAPE), (dict(D=96), SHAPE), (dict(rot=8), SHAPE), (dict(rot=80), SHAPE),
    (dict(rot=-16), SHAPE), (dict(dt=3), DTYPE), (dict(wt=3), DTYPE), (dict(q=None), NULL), (dict(f=None), NULL), (dict(ko=None), NULL),
    (dict(q=P + 8), ALIGN), (dict(st=130), ALIGN), (dict(wq=P + 4), ALIGN), (dict(qo=P + 4), ALIGN),
])
def test_preparation_codes(over, code):
    assert _rope(**over) == code and L.lib().slotscan_last_error()


@pytest.mark.parametrize("over,code", [(dict(S=0), SHAPE), (dict(lens=None), NULL), (dict(kc=None), NULL), (dict(kc=P + 2), ALIGN), (dict(v=None), NULL),
                                       (dict(cst=68), ALIGN), (dict(dt=7), DTYPE)])
def test_preparation_into_caches_codes(over, code):
    a = dict(v=P, dt=1, lens=P, S=9, kc=P, cst=128)
    a.update(over)
    s, c = (512, 64, 128), (1152, 64, a["cst"])
    assert L.lib().slotrope_cache(P, *s, P, *s, a["v"], *s, a["dt"], None, None, 0, P, 64, 0, a["lens"], 1, 4, 2, 2, 64, a["S"], 1e-6, P, a["kc"], *c,
                                  P, *c, None) == code
    assert L.lib().slotscan_last_error()


@pytest.mark.parametrize("over,code", [(dict(ws=None), NULL), (dict(dq=None), NULL), (dict(ws=P + 4), ALIGN), (dict(dk=P + 8), ALIGN)])
def test_preparation_backward_codes(over, code):
    a = dict(ws=P, dq=P, dk=P, dwq=P, dwk=P)
    a.update(over)
    s = (512, 64, 128)
    got = L.lib().slotrope_bwd(P, *s, P, *s, 1, P, P, 1, P, 64, 0, None, 0, 0, 1, 4, 2, 2, 64, 1e-6, P, *s, P, *s, a["ws"], a["dq"], a["dk"], a["dwq"],
                               a["dwk"], None)
    assert got == code, got
