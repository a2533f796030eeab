"""CPU checks of the attention oracle: against autograd of plain float64 expressions, against differences, and the window
oracle as a special case."""
import numpy as np
import pytest
import torch

from attn_cases import attn_inputs
from oracle import attn_oracle as AO
from oracle import window_oracle as WO


@pytest.mark.parametrize("opt", [dict(), dict(cap=2.0, window=9), dict(causal=False, slopes=torch.tensor([0.5, 0.1])),
                                 dict(docs=torch.tensor([[0] * 7 + [1] * 10 + [-1] * 4], dtype=torch.int32), prefix=torch.tensor([3]))])
def test_attention_gradients_by_autograd_and_differences(opt):
    q, k, v, do = (x.double() for x in attn_inputs(1, 2, 1, 21, 21, 8, torch.float32, 5))
    res = AO.attention(q, k, v, dout=do, **opt)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    f = lambda a, b, c: (AO.attention(a, b, c, **opt)["out"][0] * do).sum()
    gr = torch.autograd.grad(f(*leaves), leaves)
    h = 1e-5
    for i, (name, g) in enumerate(zip(("dq", "dk", "dv"), gr)):
        assert torch.allclose(res[name][0], g, rtol=1e-10, atol=1e-12), name
        step = torch.randn(leaves[i].shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64)
        at = lambda s: f(*(x.detach() + (s * h * step if j == i else 0) for j, x in enumerate(leaves)))
        assert abs(float((at(1) - at(-1)) / (2 * h) - (g * step).sum())) < 1e-6


def test_window_is_the_band_alone():
    q, k, v, do = attn_inputs(2, 4, 2, 40, 40, 8, torch.float32, 6)
    n = lambda x: x.numpy()
    out, _ = WO.window_forward(n(q), n(k), n(v), 7)
    grads = WO.window_backward(n(q), n(k), n(v), 7, n(do))
    res = AO.attention(q, k, v, window=7, dout=do)
    for name, want in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        assert np.abs(res[name][0].numpy() - want).max() < 1e-10, name


def test_rows_that_see_nothing_are_zero():
    q, k, v, do = attn_inputs(2, 1, 1, 6, 6, 8, torch.float32, 7)
    res = AO.attention(q, k, v, docs=torch.full((2, 6), -1, dtype=torch.int32), dout=do)
    assert all(float(res[n][0].abs().max()) == 0.0 for n in res)
    ok, _ = AO.visible(1, 4, 5, lens=torch.tensor([2]))
    assert ok.sum().item() == 1 + 2 and not ok[0, :2].any()


@pytest.mark.parametrize("pairs", [False, True])
def test_rope_gradient_by_autograd(pairs):
    g = torch.Generator().manual_seed(8)
    x = torch.randn(2, 3, 5, 16, generator=g, dtype=torch.float64).requires_grad_()
    w = torch.randn(16, generator=g, dtype=torch.float64).requires_grad_()
    dy = torch.randn(2, 3, 5, 16, generator=g, dtype=torch.float64)
    freqs = 10.0 ** -torch.arange(4, dtype=torch.float64)
    pos = torch.arange(5).unsqueeze(0) + 100
    y, dx, dw, _ = AO.rope(x.detach(), w.detach(), freqs, pos, interleaved=pairs, dy=dy)
    out = AO.rope(x, w, freqs, pos, interleaved=pairs)
    assert torch.equal(out, y)
    for a, b in zip((dx, dw), torch.autograd.grad(out, (x, w), dy)):
        assert torch.allclose(a, b, rtol=1e-10, atol=1e-12)
    assert torch.allclose(out.square().sum(-1)[..., 0], (AO.rope(x, w, freqs, pos * 0, interleaved=pairs)).square().sum(-1)[..., 0])
