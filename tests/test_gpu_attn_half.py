"""fp16's short range (slotattn_hip): the gradients are as exact for a small or a large upstream gradient as for one of about 1,
at every query and key by itself, and small probabilities keep their share."""
import pytest
import torch

from attn_cases import U, attn_inputs, near
from oracle import attn_oracle as AO

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import slotattn_hip as A

HF = torch.float16


def _grads(q, k, v, do, **o):
    leaves = [x.cuda().requires_grad_() for x in (q, k, v)]
    out = A.attend(*leaves, **{n: x.cuda() if torch.is_tensor(x) else x for n, x in o.items()})
    return dict(zip(("out", "dq", "dk", "dv"), [out, *torch.autograd.grad(out, leaves, do.cuda())]))


def _check(q, k, v, do, **o):
    ref = AO.attention(q, k, v, dout=do, u=U[HF], strict=True, **o)
    for name, x in _grads(q, k, v, do, **o).items():
        near(x, *ref[name], name)


@pytest.mark.parametrize("size", [1e3, 1.0, 1e-2, 1e-3])
@pytest.mark.parametrize("B,Hq,Hk,T,D,opt", [(1, 2, 1, 2048, 64, {}), (1, 2, 2, 1500, 128, dict(cap=30.0)), (70, 4, 2, 130, 128, dict(window=40))])
def test_upstream_of_any_size(size, B, Hq, Hk, T, D, opt):
    print("upstream", size, B, Hq, Hk, T, D, flush=True)
    q, k, v, do = attn_inputs(B, Hq, Hk, T, T, D, HF, 61)
    _check(q, k, v, (do.float() * size).to(HF), **opt)


@pytest.mark.parametrize("T,D", [(700, 64), (500, 128)])
def test_rows_of_unlike_size(T, D):
    """Upstream gradients that grow, shrink and jump from query to query."""
    q, k, v, do = attn_inputs(1, 4, 2, T, T, D, HF, 62)
    t = torch.arange(T)
    for e in (8.0 * t / T - 4, 4 - 8.0 * t / T, 6.0 * (t % 2) - 3, 8.0 * (t // 100 % 2) - 4):
        _check(q, k, v, (do.float() * (10.0 ** e).view(1, 1, T, 1)).to(HF))


@pytest.mark.parametrize("D", [64, 128])
def test_gradient_of_a_value_that_is_hardly_read(D):
    """Probabilities of about e^-12 / T under an upstream gradient of 1,000: the value's gradient is of ordinary size."""
    q, k, v, do = (x.clone() for x in attn_inputs(1, 2, 2, 900, 900, D, HF, 63))
    q[..., 0], k[..., 0] = 4.0, 0.0
    k[:, :, 7:300:50, 0] = -3.0 * D ** 0.5
    _check(q, k, v, (1000.0 * do.float()).clamp(-6e4, 6e4).to(HF))


def test_gradients_past_the_range_of_scores():
    """dP past fp16's largest number, whose gradients are not."""
    q, k, v, do = attn_inputs(1, 2, 2, 400, 400, 64, HF, 64)
    _check((0.02 * q.float()).to(HF), (0.02 * k.float()).to(HF), (100 * v.float()).to(HF), (500 * do.float()).to(HF))


@pytest.mark.parametrize("B,Hq,Hk,Tq,Tk,D", [(1, 2, 1, 3000, 3000, 64), (1, 2, 2, 2500, 2500, 128), (2, 4, 2, 1, 3000, 64), (1, 8, 1, 40, 2000, 128)])
def test_many_small_probabilities_beside_a_large_one(B, Hq, Hk, Tq, Tk, D):
    """Keys at 2^-26 of a row's largest probability, thousands of them, whose values are not the largest one's."""
    print("small probabilities", B, Hq, Hk, Tq, Tk, D, flush=True)
    q, k, v, do = attn_inputs(B, Hq, Hk, Tq, Tk, D, HF, 65)
    q, k, v = ((0.25 * x.float()).to(HF) for x in (q, k, v))
    q[..., 0], k[..., 0] = 8.0, 0.0
    k[:, :, 3, 0] = 18.0 * D ** 0.5 / 8.0
    v = v + 1.0
    v[:, :, 3] = 0.0
    _check(q, k, v, do)
