"""Infinities and NaN in places that a query does not see leave its output and gradients as they are (slotattn_hip): the
rows next to them against the float64 oracle on the clean inputs, with the oracle's bounds."""
import pytest
import torch

from attn_cases import U, attn_inputs, near
from oracle import attn_oracle as AO

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import slotattn_hip as A

BF, HF = torch.bfloat16, torch.float16
NAN, INF = float("nan"), float("inf")
ints = lambda *x: torch.tensor(x, dtype=torch.int32)


def _poison(xs, at, values):
    """Clones with values in the tokens `at` (a slice, an index or a mask (B, T))."""
    xs = [x.clone() for x in xs]
    for x, v in zip(xs, values):
        if torch.is_tensor(at):
            x.transpose(1, 2)[at] = v
        else:
            x[:, :, at] = v
    return xs


def _run(q, k, v, do, o):
    qg, kg, vg = (x.cuda().requires_grad_() for x in (q, k, v))
    out = A.attend(qg, kg, vg, **{n: x.cuda() if torch.is_tensor(x) else x for n, x in o.items()})
    return [x.cpu() for x in (out, *torch.autograd.grad(out, (qg, kg, vg), do.cuda()))]


SHAPES = [(2, 4, 2, 230, 230, 128, BF, {}), (1, 2, 2, 200, 200, 64, HF, dict(cap=20.0)),
          (1, 3, 1, 330, 330, 64, BF, dict(slopes=0.5 ** torch.arange(1, 4), window=90)),
          (1, 2, 1, 40, 900, 128, BF, {}), (40, 8, 4, 140, 140, 64, BF, {})]
_ids = lambda c: "B{}Hq{}Hk{}Tq{}Tk{}D{}".format(*c[:6])


@pytest.mark.parametrize("values", [(NAN,) * 4, (INF, -INF, INF, -INF)], ids=["nan", "inf"])
@pytest.mark.parametrize("shape", SHAPES, ids=_ids)
def test_other_documents_and_padding(shape, values):
    """One document and the padded tokens hold nothing finite, in q, k, v and in the gradient of the output."""
    B, Hq, Hk, Tq, Tk, D, dt, opt = shape
    print("nonfinite documents", _ids(shape), values, flush=True)
    clean = attn_inputs(B, Hq, Hk, Tq, Tk, D, dt, 21)
    ids = torch.arange(Tk).expand(B, Tk).mul(5).div(Tk, rounding_mode="floor").int().clone()     # five documents
    ids[:, Tk - 25:] = -1
    ids[0, 3:9] = -4
    o = dict(opt, docs=ids)
    ref = AO.attention(*clean[:3], dout=clean[3], u=U[dt], **o)
    bad = (ids < 0) | (ids == 2)
    x = clean
    q, do = _poison((x[0], x[3]), bad[:, Tk - Tq:], (values[0], values[3]))
    k, v = _poison(x[1:3], bad, values[1:3])
    got = _run(q, k, v, do, o)
    for name, g in zip(("out", "dq", "dk", "dv"), got):
        b = bad[:, Tk - Tq:] if name in ("out", "dq") else bad
        pick = lambda y: y.transpose(1, 2)[~b]
        near(pick(g), *(pick(y) for y in ref[name]), name)
        pad = (ids < 0)[:, ids.shape[1] - b.shape[1]:]
        assert bool((g.transpose(1, 2)[pad] == 0).all()), name       # padding: nothing, whatever it holds


@pytest.mark.parametrize("shape", SHAPES, ids=_ids)
@pytest.mark.parametrize("which", ["k", "v", "both"])
def test_later_tokens(shape, which):
    """Keys and values that only later queries see; what those queries give is the formula's NaN."""
    B, Hq, Hk, Tq, Tk, D, dt, opt = shape
    print("nonfinite later", _ids(shape), which, flush=True)
    q, k, v, do = attn_inputs(B, Hq, Hk, Tq, Tk, D, dt, 22)
    ref = AO.attention(q, k, v, dout=do, u=U[dt], **opt)
    j = Tk - Tq // 3                                     # the first bad key; queries from t see it
    t = j - (Tk - Tq)
    kb, vb = _poison((k, v), slice(j, j + 1), (NAN if which != "v" else 0.5, INF if which == "both" else NAN if which == "v" else 0.5))
    if which == "v":
        kb = k
    if which == "k":
        vb = v
    out, dq, _, _ = _run(q, kb, vb, do, opt)
    seen = torch.zeros(Tq, dtype=torch.bool)
    seen[t:t + opt.get("window", Tq)] = True
    for name, g in (("out", out), ("dq", dq)):
        near(g[:, :, ~seen], *(x[:, :, ~seen] for x in ref[name]), name)
        assert bool(g[:, :, seen].isnan().all()), name


def test_gradient_of_unseen_queries():
    """A query with a bad gradient reaches the keys that it sees and no others."""
    B, Hq, Hk, T, D, W = 1, 4, 2, 400, 128, 50
    q, k, v, do = attn_inputs(B, Hq, Hk, T, T, D, BF, 23)
    ref = AO.attention(q, k, v, dout=do, window=W, u=U[BF])
    bad = do.clone()
    bad[:, :, 200] = NAN
    got = _run(q, k, v, bad, dict(window=W))
    seen = torch.zeros(T, dtype=torch.bool)
    seen[200 - W + 1:201] = True
    for name, g in zip(("out", "dq", "dk", "dv"), got):
        s = seen if name[1] in "kv" else torch.zeros(T, dtype=torch.bool)
        if name == "dq":
            s = s.clone()
            s[200] = True
        near(g[:, :, ~s], *(x[:, :, ~s] for x in ref[name]), name)
        assert bool(g[:, :, s].isnan().all()), name


@pytest.mark.parametrize("case", [(2, 8, 2, 4, 700, 128, BF, (700, 130), {}), (3, 4, 4, 3, 300, 64, HF, (2, 64, 299), dict(cap=30.0)),
                                  (70, 4, 4, 130, 200, 64, BF, tuple(range(131, 201)), {}),
                                  (1, 16, 1, 5, 1500, 64, BF, (1400,), dict(window=256))], ids=_ids)
def test_cache_newest_token(case):
    """The newest token's key and value are seen by its own query alone."""
    B, Hq, Hk, T, S, D, dt, lens, opt = case
    print("nonfinite cache", case[:6], flush=True)
    q, k, v, _ = attn_inputs(B, Hq, Hk, T, S, D, dt, 24)
    lens = ints(*lens)
    ref = AO.attention(q, k, v, lens=lens, u=U[dt], **opt)["out"]
    for b in range(B):
        k[b, :, lens[b] - 1:], v[b, :, lens[b] - 1:] = NAN, INF
    with torch.no_grad():
        out = A.attend_cache(q.cuda(), k.cuda(), v.cuda(), lens.cuda(), **opt).cpu()
    near(out[:, :, :-1], *(x[:, :, :-1] for x in ref), "out")
    assert bool(out[:, :, -1].isnan().all())


@pytest.mark.parametrize("T,D,where", [(2000, 128, "v"), (700, 64, "k"), (2000, 64, "q"), (700, 128, "do")])
def test_one_early_value(T, D, where):
    """A single value that many rows see: they may be anything there, those before it and another document are as they were."""
    print("one value", T, D, where, flush=True)
    xs = dict(zip(("q", "k", "v", "do"), attn_inputs(2, 4, 2, T, T, D, BF, 25)))
    docs = torch.zeros(2, T, dtype=torch.int32)
    docs[:, T - 300:] = 1
    ref = AO.attention(xs["q"], xs["k"], xs["v"], dout=xs["do"], docs=docs, u=U[BF])
    xs[where] = xs[where].clone()
    xs[where][:, :, 70, 3] = NAN
    got = dict(zip(("out", "dq", "dk", "dv"), _run(*xs.values(), dict(docs=docs))))
    clean = torch.ones(T, dtype=torch.bool)
    clean[70:T - 300] = False
    later = torch.arange(T) >= T - 300
    for name, g in got.items():
        keep = clean.clone()
        if name in ("dk", "dv"):                         # earlier keys are seen by the queries that it reaches
            keep = later.clone()
            if where in ("q", "do"):
                keep |= (torch.arange(T) > 70)
        elif where in ("q", "do"):
            keep = torch.ones(T, dtype=torch.bool)
            keep[70] = name == "out" and where == "do"
        near(g[:, :, keep], *(x[:, :, keep] for x in ref[name]), name)
    seen = {"v": ("out", slice(70, T - 300), 3), "k": ("out", slice(70, T - 300), slice(None)), "q": ("out", slice(70, 71), slice(None)),
            "do": ("dq", slice(70, 71), slice(None))}[where]
    assert bool(got[seen[0]][:, :, seen[1], seen[2]].isnan().all())
