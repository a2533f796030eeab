"""What autograd has to know of the caches that the preparation writes (slotrope_hip, slotattn_hip)."""
import pytest
import torch

from attn_cases import attn_inputs

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import slotattn_hip as A
    import slotrope_hip as R

BF = torch.bfloat16


def _write(kc, vc, n, T=1):
    q, k, v, _ = (x.cuda() for x in attn_inputs(2, 4, 2, T, T, 64, BF, 95))
    with torch.no_grad():
        return R.qk_rope_cache(q, k, v, None, None, R.frequencies(64, device="cuda"), torch.full((2,), n, dtype=torch.int32, device="cuda"), kc, vc)


def test_a_write_to_caches_that_a_backward_needs():
    """The backward of an attention over the caches' tensors raises after a later write to them, as torch's own operations do."""
    q, k, v, do = (x.cuda() for x in attn_inputs(2, 4, 2, 20, 20, 64, BF, 94))
    q.requires_grad_()
    before = k._version, v._version
    out = A.attend(q, k, v)
    _write(k, v, 7)
    assert k._version > before[0] and v._version > before[1]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward(do)
    out = A.attend(q, k, v)                              # of the caches as they are now
    out.backward(do)
    assert bool(q.grad.isfinite().all())


def test_views_of_a_buffer_and_inference_tensors():
    """A cache that is a view marks its base; caches made in inference mode have no versions, and take writes all the same."""
    buf = torch.zeros(2, 9, 2, 2, 64, device="cuda", dtype=BF)
    n = buf._version
    _write(buf[:, :, 0].transpose(1, 2), buf[:, :, 1].transpose(1, 2), 9)
    assert buf._version > n and bool(buf[:, 8].any())
    with torch.inference_mode():
        c = [torch.zeros(2, 2, 9, 64, device="cuda", dtype=BF) for _ in range(2)]
        _write(*c, 9)
    assert bool(c[0][:, :, 8].any()) and bool(c[1][:, :, 8].any())
    _write(*c, 8)
    assert bool(c[0][:, :, 7].any())
    with torch.inference_mode():                         # and ordinary ones there
        _write(buf[:, :, 0].transpose(1, 2), buf[:, :, 1].transpose(1, 2), 5)
    assert bool(buf[:, 4].any())


@pytest.mark.parametrize("B,Tq,Tk", [(0, 5, 5), (2, 0, 5), (2, 0, 0)])
def test_no_query_gives_zero_gradients(B, Tq, Tk):
    z = lambda h, t: torch.full((B, h, t, 64), float("nan"), device="cuda", dtype=BF, requires_grad=True)
    leaves = [z(4, Tq), z(2, Tk), z(2, Tk)]
    out = A.attend(*leaves)
    assert out.shape == leaves[0].shape
    for x, g in zip(leaves, torch.autograd.grad(out, leaves, torch.zeros_like(out))):
        assert g.shape == x.shape and not bool(g.any())
