"""Operands, upstream gradients and caches of one sequence, head or token that are cut out of odd buffers: the same values as
from tensors of their own (slotattn_hip, slotrope_hip)."""
import pytest
import torch

from attn_cases import attn_inputs

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import slotattn_hip as A
    import slotrope_hip as R

BF = torch.bfloat16


def _cut(x, n):
    """x (1, H, T, D) as one row of a buffer whose rows are n elements longer; where n is odd, too."""
    buf = torch.zeros(2, x.numel() + n, device="cuda", dtype=x.dtype)
    y = buf[:, :x.numel()].unflatten(1, x.shape[1:]).split(1)[0]
    y.copy_(x)
    return y


@pytest.mark.parametrize("n", [4, 3])
@pytest.mark.parametrize("Tq,Tk", [(50, 50), (1, 70)])
def test_one_sequence_of_an_odd_buffer(n, Tq, Tk):
    q, k, v, do = (x.cuda() for x in attn_inputs(1, 4, 2, Tq, Tk, 64, BF, 96))
    want = got = None
    for cut in (lambda x: x, lambda x: _cut(x.contiguous(), n)):
        leaves = [cut(x).detach().requires_grad_() for x in (q, k, v)]
        out = A.attend(*leaves)
        want, got = got, [out, *torch.autograd.grad(out, leaves, cut(do))]
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    fr, w = R.frequencies(64, device="cuda"), torch.ones(64, device="cuda", dtype=BF)
    kk = k[:, :, :Tq]
    for cut in (lambda x: x, lambda x: _cut(x.contiguous(), n)):
        leaves = [cut(x).detach().requires_grad_() for x in (q, kk)]
        outs = R.qk_rope(*leaves, w, w, fr)
        want, got = got, [*outs, *torch.autograd.grad(outs, leaves, [cut(do), cut(kk)])]
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("n", [4, 3])
def test_caches_of_one_sequence(n):
    """In place: a cache's row of an odd buffer is written and read where it is."""
    q, k, v, _ = (x.cuda() for x in attn_inputs(1, 4, 2, 1, 1, 64, BF, 97))
    kc, vc, *_ = (x.cuda() for x in attn_inputs(1, 2, 2, 30, 30, 64, BF, 98))
    lens = torch.tensor([30], dtype=torch.int32, device="cuda")
    fr = R.frequencies(64, device="cuda")
    want = got = None
    with torch.no_grad():
        for cut in (lambda x: x.contiguous(), lambda x: _cut(x.contiguous(), n)):
            c = [cut(kc), cut(vc)]
            qn = R.qk_rope_cache(cut(q), cut(k), cut(v), None, None, fr, lens, *c)
            want, got = got, [qn, *(x.clone() for x in c), A.attend_cache(cut(qn), *c, lens)]
    assert all(torch.equal(a, b) for a, b in zip(want, got))
