"""Seeded inputs of the attention and preparation tests (CPU tensors)."""
import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def attn_inputs(B, Hq, Hk, Tq, Tk, D, dtype, seed, gain=1.4):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    heads = lambda x: x.to(dtype).transpose(1, 2)        # token-major, seen as (B, H, T, D)
    return heads(gain * r(B, Tq, Hq, D)), heads(gain * r(B, Tk, Hk, D)), heads(r(B, Tk, Hk, D)), heads(r(B, Tq, Hq, D))


def near(got, ref, bound, name):
    got = got.detach().cpu().double()
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    assert bool(torch.isfinite(got).all()), f"{name} is not finite"
    off = (got - ref).abs()
    bad = off > bound
    assert not bool(bad.any()), f"{name}: {int(bad.sum())} of {bad.numel()} values past their bound, worst {float((off / bound.clamp_min(1e-30)).max()):.3g}x"
