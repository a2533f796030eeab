"""Caps of any size (slotattn_hip): a cap far above the scores leaves them as they are, in rows beside capped ones, too.  The
bounds count a capped score's error relative to the score, not to the cap."""
import pytest
import torch

from attn_cases import U, attn_inputs, near
from oracle import attn_oracle as AO

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import slotattn_hip as A

BF, HF = torch.bfloat16, torch.float16


def _grads(q, k, v, do, **o):
    leaves = [x.cuda().requires_grad_() for x in (q, k, v)]
    out = A.attend(*leaves, **o)
    return [out, *torch.autograd.grad(out, leaves, do.cuda())]


@pytest.mark.parametrize("cap", [900.0, 1e4, 1e6, 1e8, 1e15, 1e30])
@pytest.mark.parametrize("D,dt", [(128, BF), (64, HF)])
def test_far_caps(cap, D, dt):
    print("far cap", cap, D, flush=True)
    q, k, v, do = attn_inputs(2, 4, 2, 150, 150, D, dt, 71)
    ref = AO.attention(q, k, v, dout=do, cap=cap, u=U[dt], strict=True)
    for name, x in zip(("out", "dq", "dk", "dv"), _grads(q, k, v, do, cap=cap)):
        near(x, *ref[name], name)


@pytest.mark.parametrize("cap", [900.0, 1e6, 1e30])
def test_far_caps_over_a_cache(cap):
    q, k, v, _ = attn_inputs(3, 8, 2, 1, 900, 128, HF, 72)
    lens = torch.tensor([900, 3, 400], dtype=torch.int32)
    ref = AO.attention(q, k, v, lens=lens, cap=cap, u=U[HF], strict=True)["out"]
    with torch.no_grad():
        near(A.attend_cache(*(x.cuda() for x in (q, k, v, lens)), cap=cap), *ref, "out")


def test_small_scores_beside_capped_ones():
    """One query of every 32 has scores past the cap: its neighbours' are as exact as without it."""
    cap = 1e6
    q, k, v, do = attn_inputs(1, 2, 2, 200, 200, 128, BF, 73)
    q = q.clone()
    q[:, :, 5::32] *= 2.0 ** 20
    ref = AO.attention(q, k, v, dout=do, cap=cap, u=U[BF], strict=True)
    got = _grads(q, k, v, do, cap=cap)
    far = torch.zeros(200, dtype=torch.bool)
    far[5::32] = True
    for name, x in zip(("out", "dq"), got):
        near(x[:, :, ~far], *(y[:, :, ~far] for y in ref[name]), name)


@pytest.mark.parametrize("cap,scale", [(1e-30, 1e30), (1e-6, 1.0), (1e30, 1e-6), (1e30, 1e20), (1e20, 1e20)])
def test_ends_of_the_range(cap, scale):
    """Extreme caps and scales: the score's magnitude alone decides what comes out."""
    q, k, v, do = attn_inputs(1, 2, 1, 70, 70, 64, BF, 74)
    ref = AO.attention(q, k, v, dout=do, cap=cap, scale=scale, u=U[BF], strict=True)["out"]
    out = A.attend(q.cuda(), k.cuda(), v.cuda(), cap=cap, scale=scale)
    assert bool(out.isfinite().all())
    near(out, *ref, "out")


def _whole(B, Hq, Hk, Tq, Tk, D, dt, seed):
    """Queries and keys of small whole numbers: their products are exact, the largest ones often met several times."""
    g = torch.Generator().manual_seed(seed)
    r = lambda h, t: torch.randint(-2, 3, (B, h, t, D), generator=g).to(dt)
    return r(Hq, Tq), r(Hk, Tk), torch.randn(B, Hk, Tk, D, generator=g).to(dt)


@pytest.mark.parametrize("scale", [1e4, 1e7, 3e8, 1e12, -1e20, 1e27])
@pytest.mark.parametrize("B,Hq,Hk,Tq,Tk,D,dt,lens,opt", [
    (1, 2, 1, 150, 150, 64, BF, None, {}), (70, 4, 2, 140, 140, 64, HF, None, dict(window=60)), (2, 2, 2, 130, 130, 128, HF, None, {}),
    (2, 8, 2, 1, 900, 128, BF, (900, 333), {}), (1, 4, 4, 3, 5000, 64, HF, (4800,), {}), (1, 2, 2, 70, 70, 64, BF, None, dict(cap=1e30))])
def test_scores_of_any_size(scale, B, Hq, Hk, Tq, Tk, D, dt, lens, opt):
    """Scores far past the range in which a 32-bit number resolves their differences: the largest share the weight.  The scores are
    exact, so the bounds are the probabilities' rounding and the result's alone."""
    print("far scores", scale, B, Hq, Hk, Tq, Tk, D, flush=True)
    if "cap" in opt and scale < 0:
        scale = -scale
    q, k, v = _whole(B, Hq, Hk, Tq, Tk, D, dt, 75)
    n = None if lens is None else torch.tensor(lens, dtype=torch.int32)
    with torch.no_grad():
        x = [y.cuda() for y in (q, k, v)]
        out = A.attend(*x, scale=scale, **opt) if n is None else A.attend_cache(*x, n.cuda(), scale=scale, **opt)
    want, size = (AO.attention(q, k, y, lens=n, scale=scale, window=opt.get("window"))["out"][0] for y in (v, v.abs()))
    near(out, want, 1.02 * U[dt] * (size + want.abs()) + 2.0 ** -20, "out")
