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


def _views():
    """Views whose dimensions of size 1 have strides of their own, and the rows' alignment (elements) of each."""
    wide = torch.arange(4 * 644, dtype=torch.float32).to(BF).view(4, 644)
    yield wide[:, :640].unflatten(1, (2, 5, 64)).split(1)[0]                          # one sequence of rows of 644
    yield wide[:1, :640].view(1, 5, 2, 64).transpose(1, 2)
    yield torch.arange(5 * 2 * 3 * 65.0).to(BF).as_strided((2, 1, 5, 64), (960, 3, 64, 1))
    yield torch.arange(4096.0).to(BF).as_strided((2, 3, 1, 64), (640, 64, 1 << 26, 1))  # one token, far from the next
    yield torch.arange(4096.0).to(BF).as_strided((1, 1, 1, 64), (7, 5, 3, 1))


@pytest.mark.parametrize("i", range(5))
def test_strides_of_single_items_do_not_matter(i):
    """A dimension of size 1 has no stride that could be odd: the rows are read where they are."""
    x = list(_views())[i]
    y = L.rows(x)
    p, *s = L.strided(y)
    assert p % 16 == 0 and all(v % 8 == 0 and 0 <= v < 1 << 25 for v in s), s
    flat = y.as_strided((y.shape[0], y.shape[1], y.shape[2], 64), (*s, 1))
    assert torch.equal(flat, x)
    if x.data_ptr() % 16 == 0:
        assert L.in_place(x) and y is x


@pytest.mark.parametrize("x", [z(2, 2, 5, 65)[..., :64], z(2 * 2 * 5 * 64 + 1)[1:].view(2, 2, 5, 64), z(2, 2, 64, 5).transpose(2, 3),
                               z(1, 2, 5, 64).expand(3, 2, 5, 64), z(2, 5, 2, 64).transpose(1, 2), z(3, 2, 8, 64)[:, :, ::2], z(2, 2, 5, 1).expand(2, 2, 5, 64)])
def test_rows_are_aligned(x):
    y = L.rows(x)
    assert L.in_place(y) and torch.equal(x, y)


def test_constants_may_ask_for_gradients_where_none_are_formed():
    """Slopes and frequencies are constants: refused where autograd is on and would miss them, and only there."""
    q, k, n = z(2, 4, 3, 64), z(2, 2, 3, 64), torch.tensor([3, 3], dtype=torch.int32)
    s, fr = z(4, dt=torch.float32).requires_grad_(), R.frequencies(64).requires_grad_()
    calls = [lambda: A.attend(q, k, k, slopes=s), lambda: A.attend_cache(q, k, k, n, slopes=s), lambda: R.qk_rope(q, k, None, None, fr),
             lambda: R.qk_rope_cache(q, k, k, None, None, fr, n, z(2, 2, 9, 64), z(2, 2, 9, 64))]
    for f in calls:
        with pytest.raises((NotImplementedError, RuntimeError), match="constants|no backward"):
            f()
        with torch.no_grad(), pytest.raises(RuntimeError, match="GPU tensors only"):
            f()


def _pair(a, b):
    q, n = z(2, 4, 3, 64), torch.tensor([3, 3], dtype=torch.int32)
    with torch.no_grad():
        R.qk_rope_cache(q, a[:, :, :3].contiguous(), a[:, :, :3].contiguous(), None, None, R.frequencies(64), n, a, b)


@pytest.mark.parametrize("kind", range(5))
def test_caches_that_share_memory_with_each_other(kind):
    buf = z(2, 2, 12, 64)
    far = z(2 * 2 * 9 * 128)
    a, b = [(buf, buf), (buf[:, :, :9], buf[:, :, 3:]), (buf[:, :, :9], buf[:, :, 1:10]),
            (far.as_strided((2, 2, 9, 64), (2304, 1152, 128, 1)), far.as_strided((2, 2, 9, 64), (2304, 1152, 128, 1), 32)),
            (far.as_strided((2, 2, 9, 64), (2304, 1152, 128, 1)), far.as_strided((2, 2, 9, 64), (1152, 576, 64, 1)))][kind]
    with pytest.raises(ValueError, match="share memory"):
        _pair(a, b)


@pytest.mark.parametrize("kind", range(6))
def test_caches_side_by_side_in_one_buffer(kind):
    a, b = [z(2, 2, 2, 9, 64).unbind(0), z(2, 2, 2, 9, 64).unbind(1), z(2, 2, 2, 9, 64).unbind(2), z(2, 9, 2, 2, 64).transpose(1, 3).unbind(2),
            z(2, 9, 2, 128).transpose(1, 2).split(64, 3), (z(2, 2, 18, 64)[:, :, :9], z(2, 2, 18, 64)[:, :, 9:])][kind]
    with pytest.raises(RuntimeError, match="GPU tensors only"):       # taken, as far as a CPU tensor is
        _pair(a, b)


@pytest.mark.parametrize("at", [4, 8])
def test_workspace_of_the_backward_is_aligned(at):
    s = (512, 64, 128)
    assert L.lib().slotattn_bwd(P, *s, P, *s, P, *s, 1, 1, 4, 4, 2, 2, 64, 0.1, 1, 5, 0.0, None, None, None, P, P, P, P, *s, P + at, P, P, P, P,
                                None) == 4
