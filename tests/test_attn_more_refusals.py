"""What else the attention and the preparation of its operands refuse or take, on the CPU."""
import pytest
import torch

import slotattn_hip as A
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
