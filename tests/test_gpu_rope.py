"""GPU parity of the query and key preparation (slotrope_hip) against the float64 oracle (oracle/attn_oracle.py)."""
import pytest
import torch

from attn_cases import U
from oracle import attn_oracle as AO

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import slotrope_hip as R

BF, HF, F = torch.bfloat16, torch.float16, torch.float32
CASES = [  # B, Hq, Hk, T, D, rot, pairs, dtype, gain dtypes, positions
    (1, 1, 1, 1, 64, 64, False, BF, (BF, BF), None),
    (2, 12, 4, 37, 128, 128, False, BF, (BF, BF), None),
    (3, 5, 3, 130, 64, 32, True, F, (F, F), "b"),
    (2, 6, 2, 65, 128, 16, False, HF, (HF, None), "t"),
    (2, 4, 4, 33, 128, 64, True, HF, (None, None), "far"),
    (1, 3, 1, 50, 64, 64, False, F, (None, BF), "far"),
    (2, 2, 7, 40, 128, 0, False, BF, (F, BF), None),
    (1, 2, 2, 3000, 64, 48, False, BF, (F, F), None),
    (70, 33, 3, 1, 128, 128, True, F, (F, F), "b"),
]


def _pos(kind, B, T):
    if kind is None:
        return None
    if kind == "t":
        return torch.arange(5, 5 + T, dtype=torch.int32)
    g = torch.Generator().manual_seed(4)
    if kind == "b":
        return torch.randint(-3, 5000, (B, T), generator=g)
    return torch.randint(2 ** 23, 2 ** 24, (B, T), generator=g)


def _inputs(B, Hq, Hk, T, D, dt, wt):
    g = torch.Generator().manual_seed(21)
    r = lambda *s: torch.randn(*s, generator=g)
    heads = lambda n: (2 * r(B, T, n, D)).to(dt).transpose(1, 2)
    ws = [None if t is None else (1 + 0.3 * r(D)).to(t) for t in wt]
    return heads(Hq), heads(Hk), ws, (r(B, T, Hq, D).to(dt).transpose(1, 2), r(B, T, Hk, D).to(dt).transpose(1, 2))


def _close(got, ref, scale, u, name):
    """One rounding of the result, and 32-bit steps (norm, gain, sine and cosine, two products): 2^-20 of the row's size."""
    off = (got.detach().cpu().double() - ref).abs()
    bound = u * ref.abs() * 1.01 + 2.0 ** -20 * scale + (2.0 ** -25 if u == 2.0 ** -11 else 0.0)
    assert bool((off <= bound).all()), f"{name}: worst {float((off / bound).max()):.3g}x its bound"


@pytest.mark.parametrize("case", CASES, ids=lambda c: "B{}Hq{}Hk{}T{}D{}r{}{}".format(*c[:7]))
def test_rope_matches_oracle(case):
    B, Hq, Hk, T, D, rot, pairs, dt, wt, kind = case
    print("rope", case, flush=True)
    q, k, ws, dys = _inputs(B, Hq, Hk, T, D, dt, wt)
    pos = _pos(kind, B, T)
    freqs = R.frequencies(rot)
    p2 = torch.arange(T).unsqueeze(0) if pos is None else pos.reshape(-1, T)
    leaves = [None if x is None else x.cuda().requires_grad_() for x in (q, k, *ws)]
    outs = R.qk_rope(*leaves, freqs.cuda(), positions=None if pos is None else pos.cuda(), interleaved=pairs)
    grads = iter(torch.autograd.grad(outs, [x for x in leaves if x is not None], [d.cuda() for d in dys]))
    gr = [None if x is None else next(grads) for x in leaves]
    for i, (x, w, dy) in enumerate(zip((q, k), ws, dys)):
        y, dx, dw, dwa = AO.rope(x, w, freqs, p2, interleaved=pairs, dy=dy)
        size = y.abs().amax(-1, keepdim=True)
        assert outs[i].dtype == dt and outs[i].shape == x.shape
        _close(outs[i], y, size, U[dt], "out%d" % i)
        rr = torch.rsqrt(x.double().square().mean(-1, keepdim=True) + 1e-6)
        gsize = (dy.double().abs().amax(-1, keepdim=True) * 4 * rr * (1 if w is None else w.double().abs().max()))
        _close(gr[i], dx, gsize, U[dt], "dx%d" % i)
        if w is not None:                                # a sum of n products in 32 bits, pairwise by lanes: at most 2^-14 of its absolute sum
            _close(gr[2 + i], dw, dwa * 2.0 ** 6, U[w.dtype], "dw%d" % i)
            assert gr[2 + i].dtype == w.dtype
    with torch.no_grad():
        again = R.qk_rope(*leaves, freqs.cuda(), positions=None if pos is None else pos.cuda(), interleaved=pairs)
    assert all(torch.equal(a, b) for a, b in zip(again, outs))


@pytest.mark.parametrize("T,S,lens,dt", [(1, 9, (1, 9, 4), BF), (6, 40, (3, 6, 40), HF), (4, 5, (0, 5, 8), F), (300, 310, (10, 310, 299), BF)])
def test_rope_cache_writes_its_rows_alone(T, S, lens, dt):
    B, Hq, Hk, D = 3, 6, 2, 64
    q, k, ws, (_, v) = _inputs(B, Hq, Hk, T, D, dt, (BF, BF))
    freqs = R.frequencies(D)
    g = torch.Generator().manual_seed(9)
    kc, vc = (torch.randn(B, S, Hk, D, generator=g).to(dt).transpose(1, 2) for _ in range(2))
    kg, vg = kc.cuda(), vc.cuda()
    n = torch.tensor(lens, dtype=torch.int32)
    with torch.no_grad():
        out = R.qk_rope_cache(q.cuda(), k.cuda(), v.cuda(), *(w.cuda() for w in ws), freqs.cuda(), n.cuda(), kg, vg)
    pos = n.long().unsqueeze(-1) - T + torch.arange(T)
    yq, yk = (AO.rope(x, w, freqs, pos) for x, w in zip((q, k), ws))
    _close(out, yq, yq.abs().amax(-1, keepdim=True), U[dt], "q")
    wk, wv, wrote = kc.double(), vc.clone(), torch.zeros(B, S, dtype=torch.bool)
    for b in range(B):
        for t in range(T):
            p = int(pos[b, t])
            if 0 <= p < S:
                wk[b, :, p], wv[b, :, p], wrote[b, p] = yk[b, :, t], v[b, :, t], True
    assert torch.equal(vg.cpu(), wv)
    m = wrote.view(B, 1, S, 1).expand(B, Hk, S, D)
    assert torch.equal(kg.cpu()[~m], kc[~m])
    _close(kg[m.cuda()], wk[m], 8.0, U[dt], "k")


def test_gain_gradients_are_reproducible():
    q, k, ws, dys = _inputs(2, 4, 2, 500, 128, BF, (F, F))
    res = []
    for _ in range(2):
        leaves = [x.cuda().requires_grad_() for x in (q, k, *ws)]
        outs = R.qk_rope(*leaves, R.frequencies(128, device="cuda"))
        res.append(torch.autograd.grad(outs, leaves, [d.cuda() for d in dys]))
    assert all(torch.equal(a, b) for a, b in zip(*res))
