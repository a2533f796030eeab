"""GPU parity of the attention of any range (slotattn_hip) against the float64 oracle (oracle/attn_oracle.py) on the same
16-bit inputs, with the oracle's bounds on the rounding errors, value by value."""
import pytest
import torch

from attn_cases import U, attn_inputs, near
from oracle import attn_oracle as AO

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import slotattn_hip as A

BF, HF = torch.bfloat16, torch.float16
ints = lambda *x: torch.tensor(x, dtype=torch.int32)


def _docs(B, T, kind, seed=3):
    g = torch.Generator().manual_seed(seed)
    if kind == "runs":                                   # runs of a few to a hundred tokens, a padded end
        ids = torch.cat([torch.full((int(n),), i) for i, n in enumerate(torch.randint(1, 100, (B * T,), generator=g))])[:B * T]
        ids = ids.reshape(B, T).clone()
        ids[:, T - T // 10:] = -1
        return ids.int()
    if kind == "mixed":                                  # any order, paddings between
        return torch.randint(-1, 4, (B, T), generator=g).int()
    if kind == "pad":                                    # the first sequence is padding alone
        ids = torch.zeros(B, T, dtype=torch.int32)
        ids[0] = -7
        return ids
    return torch.full((B, T), 2 ** 31 - 1, dtype=torch.int32)


CASES = [  # B, Hq, Hk, Tq, Tk, D, dtype, options
    (1, 1, 1, 1, 1, 64, BF, {}),
    (2, 3, 1, 5, 5, 128, BF, {}),
    (1, 2, 2, 64, 64, 64, HF, {}),
    (2, 6, 2, 65, 65, 128, BF, {}),
    (1, 4, 2, 127, 127, 128, HF, dict(cap=30.0)),
    (1, 2, 1, 300, 300, 128, BF, dict(cap=50.0, causal=False)),
    (2, 2, 2, 129, 129, 64, BF, dict(window=1)),
    (1, 4, 4, 260, 260, 64, BF, dict(window=33)),
    (1, 2, 2, 200, 200, 128, HF, dict(window=70, causal=False)),
    (2, 4, 2, 190, 190, 128, BF, dict(slopes=True)),
    (1, 3, 3, 150, 150, 64, HF, dict(slopes=True, causal=False, cap=20.0)),
    (2, 4, 2, 260, 260, 128, BF, dict(docs="runs")),
    (2, 2, 1, 200, 200, 64, BF, dict(docs="mixed", causal=False)),
    (2, 2, 2, 100, 100, 64, HF, dict(docs="pad")),
    (1, 2, 2, 70, 70, 64, BF, dict(docs="one")),
    (2, 2, 2, 210, 210, 128, BF, dict(prefix=ints(0, 131))),
    (3, 2, 1, 140, 140, 64, BF, dict(prefix=ints(1, 500, 64), window=20, cap=10.0)),
    (2, 2, 2, 330, 330, 64, BF, dict(prefix=ints(90, 3), docs="runs", window=50, slopes=True)),
    (1, 4, 2, 100, 333, 128, BF, dict(window=150)),      # the newest queries of longer keys
    (2, 2, 1, 40, 700, 64, HF, dict(docs="runs")),
    (2, 8, 2, 7, 900, 128, BF, dict(cap=50.0)),          # few rows: split keys
    (1, 32, 1, 3, 600, 64, BF, dict(slopes=True, prefix=ints(40), window=100)),
    (2, 4, 4, 33, 1100, 128, HF, dict(causal=False, window=200)),
    (1, 2, 2, 128, 4200, 64, BF, {}),                    # more than 64 key tiles
    (1, 1, 1, 60, 60, 64, BF, dict(cap=0.5, scale=1.0)),  # scores far past their cap
    (1, 2, 1, 70, 70, 128, BF, dict(scale=-0.05)),
]


def _ids(c):
    return "B{}Hq{}Hk{}Tq{}Tk{}D{}".format(*c[:6]) + ("f16" if c[6] == HF else "") + "".join("-" + k for k in c[7])


def _options(B, Hq, Tk, o):
    o = dict(o)
    if "docs" in o:
        o["docs"] = _docs(B, Tk, o["docs"])
    if o.get("slopes"):
        o["slopes"] = 2.0 ** (-8.0 * torch.arange(1, Hq + 1) / Hq)
    return o


def _gpu(o):
    return {k: x.cuda() if torch.is_tensor(x) else x for k, x in o.items()}


@pytest.mark.parametrize("case", CASES, ids=_ids)
def test_attend_matches_oracle(case):
    B, Hq, Hk, Tq, Tk, D, dt, opt = case
    print("attend", _ids(case), flush=True)
    q, k, v, do = attn_inputs(B, Hq, Hk, Tq, Tk, D, dt, 11)
    o = _options(B, Hq, Tk, opt)
    ref = AO.attention(q, k, v, dout=do, u=U[dt], **o)
    qg, kg, vg = (x.cuda().requires_grad_() for x in (q, k, v))
    out = A.attend(qg, kg, vg, **_gpu(o))
    assert out.dtype == dt and out.shape == q.shape
    got = [out] + list(torch.autograd.grad(out, (qg, kg, vg), do.cuda()))
    for name, x in zip(("out", "dq", "dk", "dv"), got):
        near(x, *ref[name], name)
    with torch.no_grad():
        assert torch.equal(A.attend(qg, kg, vg, **_gpu(o)), out)      # without the backward's sums: the same values


CACHE = [  # B, Hq, Hk, T, S, D, dtype, lens, options
    (4, 6, 2, 1, 700, 128, BF, (1, 64, 65, 700), {}),
    (3, 4, 4, 1, 300, 64, HF, (0, 257, 1000), dict(cap=30.0)),        # nothing yet; a length past the cache
    (2, 8, 1, 5, 512, 128, BF, (3, 512), dict(window=100)),           # padding on the left
    (2, 40, 1, 2, 200, 64, BF, (2, 199), dict(slopes=True)),          # more rows than a tile
    (2, 2, 2, 300, 2000, 64, BF, (150, 1999), dict(window=77, prefix=ints(10, 1500))),
    (2, 4, 2, 200, 260, 128, HF, (260, 201), dict(cap=50.0)),
    (70, 4, 4, 130, 200, 64, BF, tuple(range(100, 170)), {}),         # enough tiles for whole-tile rows
    (1, 2, 1, 1, 20000, 128, BF, (19990,), dict(window=4096)),
    (1, 1, 1, 9, 4, 64, BF, (4,), {}),                                # more new tokens than rows
]


@pytest.mark.parametrize("case", CACHE, ids=lambda c: "B{}Hq{}Hk{}T{}S{}D{}".format(*c[:6]))
def test_attend_cache_matches_oracle(case):
    B, Hq, Hk, T, S, D, dt, lens, opt = case
    print("attend_cache", case[:6], opt, flush=True)
    q, k, v, _ = attn_inputs(B, Hq, Hk, T, S, D, dt, 12)
    o = _options(B, Hq, S, opt)
    lens = ints(*lens)
    ref = AO.attention(q, k, v, lens=lens, u=U[dt], **o)
    for b in range(B):                                   # what lies behind a sequence is never read
        k[b, :, max(int(lens[b]), 0):], v[b, :, max(int(lens[b]), 0):] = float("nan"), float("inf")
    with torch.no_grad():
        out = A.attend_cache(q.cuda(), k.cuda(), v.cuda(), lens.cuda(), **_gpu(o))
    near(out, *ref["out"], "out")


def test_operand_layouts():
    """Slices of a fused projection, head-major tensors, shared (expanded) heads and odd strides: the same values."""
    B, H, T, D = 2, 4, 150, 64
    q, k, v, do = (x.cuda() for x in attn_inputs(B, H, H, T, T, D, BF, 13))
    want = None
    fused = torch.cat([x.transpose(1, 2) for x in (q, k, v)], 2)
    wide = torch.zeros(B, H, T, D + 3, device="cuda", dtype=BF)
    for i, (a, b, c, g) in enumerate([
            (q, k, v, do), tuple(x.contiguous() for x in (q, k, v, do)),
            (*(x.transpose(1, 2) for x in fused.split([H, H, H], 2)), do),
            tuple(wide.clone()[..., :D].copy_(x) for x in (q, k, v, do)),
            tuple(torch.empty(x.numel() + 1, device="cuda", dtype=BF)[1:].view(x.shape).copy_(x) for x in (q, k, v, do))]):
        a, b, c = (x.detach().requires_grad_() for x in (a, b, c))
        out = A.attend(a, b, c, window=40)
        got = [out] + list(torch.autograd.grad(out, (a, b, c), g))
        want = want or got
        for x, y in zip(got, want):
            assert torch.equal(x, y), i
    k1 = k[:, :1].detach().requires_grad_()              # one head for all by expansion: its gradient is the heads' sum
    out = A.attend(q, k1.expand(B, H, T, D), v)
    dk = torch.autograd.grad(out, k1, do)[0]
    assert dk.shape == k1.shape
    assert torch.equal(out, A.attend(q, k[:, :1].expand(B, H, T, D).contiguous(), v))


def test_empty_calls():
    e = lambda *s: torch.zeros(*s, device="cuda", dtype=BF, requires_grad=True)
    for B, Tq, Tk in ((0, 5, 5), (2, 0, 5), (2, 0, 0)):
        q, k, v = e(B, 2, Tq, 64), e(B, 2, Tk, 64), e(B, 2, Tk, 64)
        out = A.attend(q, k, v)
        assert out.shape == q.shape
        out.sum().backward()
        assert q.grad.shape == q.shape
    with torch.no_grad():
        assert A.attend_cache(e(2, 2, 0, 64), e(2, 2, 4, 64), e(2, 2, 4, 64), ints(0, 1).cuda()).shape == (2, 2, 0, 64)
