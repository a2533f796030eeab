"""Infinities and NaN in several places at once (slotattn_hip): what a row does not see stays out of it also where it sees one.

The reference forms every query from its visible keys alone, cut out of the tensors, and every key's gradients from those of the
queries that see it; where that is finite the result has to be within the bound, where it is not the result is not, and an output's
infinities keep their sign."""
import pytest
import torch

from attn_cases import U, attn_inputs
from oracle import attn_oracle as AO

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import slotattn_hip as A

BF, HF = torch.bfloat16, torch.float16
NAN, INF = float("nan"), float("inf")


def _reference(q, k, v, do, ok, b, u):
    """(value, bound) of out, dq (Hq, Tq, D) and dk, dv (Hk, Tk, D) of sequence b; ok (Tq, Tk)."""
    Hq, Tq, D = q.shape[1:]
    Hk, Tk = k.shape[1:3]
    z = lambda h, t: [torch.zeros(h, t, D, dtype=torch.float64) for _ in range(2)]
    res = dict(out=z(Hq, Tq), dq=z(Hq, Tq), dk=z(Hk, Tk), dv=z(Hk, Tk))
    for i in range(Tq):
        for h in range(Hq):
            x = h // (Hq // Hk)
            see = ok[i].nonzero().flatten()
            row, up = q[b:b + 1, h:h + 1, i:i + 1], None if do is None else do[b:b + 1, h:h + 1, i:i + 1]
            # a score of -inf has no weight and adds nothing that is rounded: the bounds are those of the other keys
            score = k[b, x, see].double() @ row[0, 0, 0].double()
            weight = see[score != -INF]
            for which, keys in ((0, see), (1, weight)):
                if not len(keys):
                    continue
                if bool((score.isnan() | (score == INF)).any()):      # its softmax is NaN at every key
                    for n in ("out", "dq"):
                        res[n][which][h, i] = NAN
                    for n in ("dk", "dv"):
                        res[n][which][x, keys] += NAN
                    continue
                one = AO.attention(row, k[b:b + 1, x:x + 1, keys], v[b:b + 1, x:x + 1, keys], causal=False, u=u, scale=D ** -0.5, dout=up)
                for n, got in one.items():
                    if n in ("out", "dq"):
                        res[n][which][h, i] = got[which][0, 0, 0]
                    else:
                        res[n][which][x, keys] += got[which][0, 0]
    return res


def _same(got, ref, bound, name):
    got = got.detach().cpu().double()
    fine = ref.isfinite()
    assert bool(got[fine].isfinite().all()), f"{name}: {int((~got[fine].isfinite()).sum())} values should be finite"
    assert not bool(got[~fine].isfinite().any()), f"{name}: {int(got[~fine].isfinite().sum())} values should not be finite"
    off, b = (got - ref)[fine].abs(), bound[fine]
    assert bool((off <= b).all()), f"{name}: worst {float((off / b).max()):.3g}x its bound"
    if name == "out":
        inf = ref.isinf()
        assert torch.equal(got[inf], ref[inf]), name


# tensor, token, column, value: some seen by the later rows, some by the last ones alone, in one column and in several
PLACES = {
    "values": [("v", 0, 3, NAN), ("v", 63, 5, NAN), ("v", 100, 5, INF), ("v", 129, 9, -INF), ("v", -1, 3, NAN)],
    "infinite": [("v", 2, 7, INF), ("v", 40, 7, -INF), ("v", -1, 1, INF), ("v", 90, 7, NAN)],
    "last": [("v", -1, 11, INF), ("v", -2, 12, NAN)],
    "keys": [("k", 1, 2, NAN), ("v", 50, 4, NAN), ("k", 120, 0, INF), ("v", -1, 6, NAN)],
    "weightless": [("k", 4, 0, -INF), ("v", 30, 8, NAN), ("k", 70, 0, -INF), ("k", -1, 3, NAN)],
    "queries": [("q", 0, 1, NAN), ("q", 66, 2, INF), ("do", 90, 3, NAN), ("do", -1, 4, INF), ("q", -2, 5, NAN)],
    "upstream": [("do", 10, 3, INF), ("do", 31, 4, NAN), ("do", 64, 3, NAN), ("do", -1, 3, -INF)],
    "all": [("q", 12, 0, INF), ("k", 33, 1, NAN), ("v", 47, 2, INF), ("do", 80, 3, NAN), ("v", 101, 4, NAN), ("k", -1, 5, INF), ("do", -1, 6, INF)],
}


def _poisoned(places, xs):
    q, k, v, do = (x.clone() for x in xs)
    q[..., 0] = q[..., 0].abs() + 0.5                    # the sign of a score with an infinite key is known
    t = dict(q=q, k=k, v=v, do=do)
    Tk = k.shape[2]
    for n, at, col, val in places:
        x = t[n]
        at = at if at < 0 else at - (Tk - x.shape[2])    # places by the keys' positions
        if -x.shape[2] <= at < x.shape[2]:
            x[:, :, at, col] = val
    return q, k, v, do


@pytest.mark.parametrize("places", PLACES)
@pytest.mark.parametrize("B,Hq,Hk,Tq,Tk,D,dt,opt", [
    (1, 2, 1, 150, 150, 64, BF, {}), (1, 2, 2, 150, 150, 128, HF, dict(window=45)), (2, 2, 2, 140, 140, 64, BF, dict(docs=True)),
    (1, 2, 1, 130, 170, 128, BF, dict(prefix=20)), (1, 1, 1, 128, 128, 64, HF, dict(causal=False, window=30)),
    (130, 2, 2, 131, 131, 64, BF, {})])
def test_every_place(places, B, Hq, Hk, Tq, Tk, D, dt, opt):
    print("places", places, B, Hq, Hk, Tq, Tk, D, opt, flush=True)
    xs = _poisoned(PLACES[places], attn_inputs(B, Hq, Hk, Tq, Tk, D, dt, 51))
    o = dict(opt)
    if o.pop("docs", False):
        o["docs"] = (torch.arange(Tk) // 47).int().expand(B, Tk).clone()
        o["docs"][:, Tk - 9:] = -1
    if "prefix" in o:
        o["prefix"] = torch.full((B,), o["prefix"], dtype=torch.int32)
    ok, _ = AO.visible(B, Tq, Tk, **o)
    leaves = [x.cuda().requires_grad_() for x in xs[:3]]
    out = A.attend(*leaves, **{n: x.cuda() if torch.is_tensor(x) else x for n, x in o.items()})
    got = dict(zip(("out", "dq", "dk", "dv"), [out, *torch.autograd.grad(out, leaves, xs[3].cuda())]))
    for b in {0, B - 1}:
        ref = _reference(*xs, ok[b % ok.shape[0]], b, U[dt])
        for n, x in got.items():
            _same(x[b], *ref[n], n)


@pytest.mark.parametrize("places", ["values", "infinite", "last", "keys", "weightless"])
@pytest.mark.parametrize("B,Hq,Hk,Tq,Tk,D,dt,lens,opt", [
    (2, 8, 2, 3, 700, 128, BF, (700, 150), {}), (1, 4, 4, 5, 1500, 64, HF, (1404,), dict(window=1300)), (3, 6, 2, 1, 200, 64, BF, (131, 1, 200), {}),
    (1, 2, 1, 40, 300, 64, BF, (170,), dict(prefix=70, window=60))])
def test_every_place_of_a_cache(places, B, Hq, Hk, Tq, Tk, D, dt, lens, opt):
    print("cache places", places, B, Hq, Hk, Tq, Tk, D, opt, flush=True)
    q, k, v, _ = attn_inputs(B, Hq, Hk, Tq, Tk, D, dt, 52)
    q, k, v, _ = _poisoned([], (q, k, v, q))
    for b in range(B):                                   # places by each sequence's length
        for n, at, col, val in PLACES[places]:
            if -lens[b] <= at < lens[b]:
                (k if n == "k" else v)[b, :, at % lens[b], col] = val
    o = dict(opt)
    if "prefix" in o:
        o["prefix"] = torch.full((B,), o["prefix"], dtype=torch.int32)
    n = torch.tensor(lens, dtype=torch.int32)
    ok, _ = AO.visible(B, Tq, Tk, lens=n, **o)
    with torch.no_grad():
        out = A.attend_cache(q.cuda(), k.cuda(), v.cuda(), n.cuda(), **{m: x.cuda() if torch.is_tensor(x) else x for m, x in o.items()})
    for b in range(B):
        _same(out[b], *_reference(q, k, v, None, ok[b], b, U[dt])["out"], "out")


@pytest.mark.parametrize("Tq,Tk,D,dt,opt", [(5, 5, 64, BF, {}), (2, 898, 128, HF, {}), (9, 73, 128, HF, dict(prefix=7)), (20, 1044, 64, BF, {}), (150, 150, 128, BF, {})])
def test_rows_beside_rows_that_are_lost(Tq, Tk, D, dt, opt):
    """A query that is NaN, or a key that makes the later rows NaN, beside rows that keep a finite part; and a value that those do not
    see at the key of the lost query's place in its tile."""
    print("lost rows", Tq, Tk, D, opt, flush=True)
    q, k, v, do = _poisoned([("v", Tk - Tq, 3, NAN), ("v", -2, 5, INF), ("v", -2, 2, -INF)], attn_inputs(2, 1, 1, Tq, Tk, D, dt, 53))
    q[0, 0, Tq - 2, 7] = NAN
    k[1, :, Tk - 2, 7] = NAN
    o = dict(opt)
    if "prefix" in o:
        o["prefix"] = torch.full((2,), o["prefix"], dtype=torch.int32)
    ok, _ = AO.visible(2, Tq, Tk, **o)
    leaves = [x.cuda().requires_grad_() for x in (q, k, v)]
    out = A.attend(*leaves, **{m: x.cuda() if torch.is_tensor(x) else x for m, x in o.items()})
    got = dict(zip(("out", "dq", "dk", "dv"), [out, *torch.autograd.grad(out, leaves, do.cuda())]))
    for b in range(2):
        ref = _reference(q, k, v, do, ok[b % len(ok)], b, U[dt])
        for n, x in got.items():
            _same(x[b], *ref[n], n)
