"""What else the attention and the preparation of its operands refuse or take, on the CPU."""
import pytest
import torch
from torch.autograd import forward_ad

import slotattn_hip as A
import slotrope_hip as R
import slotscan_lib as L

BF = torch.bfloat16
z = lambda *s, dt=BF: torch.zeros(*s, dtype=dt)
P = 1 << 20


@pytest.mark.parametrize("kw", [dict(cap=1e30, scale=1e-7), dict(cap=1e7, scale=-1e-30)])
def test_caps_beyond_the_scale(kw):
    """A cap so far above the scale that their quotient leaves 32 bits."""
    with pytest.raises(ValueError, match="cap"):
        A.attend(z(1, 2, 3, 64), z(1, 2, 3, 64), z(1, 2, 3, 64), **kw)
    s = (512, 64, 128)
    assert L.lib().slotattn_fwd(P, *s, P, *s, P, *s, 1, 1, 4, 4, 2, 2, 64, kw["scale"], 1, 5, kw["cap"], None, None, None, None, None, P, None, None,
                                None) == 1


def _calls(q, k, v, w):
    """The four entry points on these operands."""
    fr, n = R.frequencies(64), torch.tensor([3, 3], dtype=torch.int32)
    c = [z(2, 2, 4, 64) for _ in range(2)]
    return [lambda: A.attend(q, k, v), lambda: A.attend_cache(q, k, v, n), lambda: R.qk_rope(q, k, w, None, fr),
            lambda: R.qk_rope_cache(q, k, v, w, None, fr, n, *c)]


@pytest.mark.parametrize("which,at", [(0, 0), (0, 1), (0, 2), (0, 3), (1, 0), (1, 1), (1, 2), (1, 3), (2, 0), (2, 1), (2, 3), (3, 2), (3, 3)])
def test_forward_mode_derivatives(which, at):
    """A dual tensor is refused by every entry point: none of them forms its tangent."""
    xs = [z(2, 4, 3, 64), z(2, 2, 3, 64), z(2, 2, 3, 64), z(64)]
    with torch.no_grad(), forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="GPU tensors only"):                  # without one: the call goes on
            _calls(*xs)[at]()
        xs[which] = forward_ad.make_dual(xs[which], torch.ones_like(xs[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            _calls(*xs)[at]()
