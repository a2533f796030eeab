"""Exact attention of any range on MI355X (include/slotattn.h): where a layer's short window (slotwin_hip) and the slot read
are not enough -- packed documents, long windows, prompts read both ways, capped or biased scores, a cache of keys.

    attend(q, k, v, scale=None, causal=True, window=None, cap=None, slopes=None, docs=None, prefix=None) -> (B, Hq, Tq, D)
        q (B, Hq, Tq, D), k, v (B, Hk, Tk, D), Hq a multiple of Hk (query head h reads key/value head h // (Hq // Hk)).  The
        queries are the last Tq <= Tk of the keys' positions.  For query position i and key j:
            s = scale <q, k>  (default 1 / sqrt(D));   cap: s = cap tanh(s / cap);   slopes (Hq,): s -= slopes[h] |i - j|
        then the softmax over the visible keys: 0 <= i - j < window (causal) or |i - j| < window (not; None: no bound), and
        whatever the band says the first prefix[b] keys of the row; with docs (B, Tk) of all these only keys of the query's
        own document (so that a prefix reaches the row's first documents alone), a negative id being padding.  A query that
        sees nothing, or scores of -inf alone, gets 0.  Autograd gives dq, dk, dv; slopes are constants.
    attend_cache(q, kcache, vcache, lens, scale=None, window=None, cap=None, slopes=None, prefix=None) -> (B, Hq, T, D)
        the serving form, forward only and causal: q holds the newest T of each sequence's lens[b] tokens, whose keys and
        values (the new ones included) are the first lens[b] rows of kcache, vcache (B, Hk, S, D).  What lies behind them
        is not read.  A query of negative position (lens[b] < T) gets 0.

bf16 or fp16, D in {64, 128}; docs, prefix (B,) and lens (B,) int32, slopes fp32.  Scores, softmax statistics and sums are
fp32; the probabilities and score gradients are rounded to the operands' type for their products.  The gradients take the
probabilities from the rows' fp32 log-sum-exp, which moves them by about 2^-24 of the row's largest score (fine for scores
up to tens of thousands, no longer for millions).  What a query does not see never reaches its row, infinities and NaN
included.  Operands may be any views whose rows are contiguous and 16-byte aligned (others are copied: a cache should not
need that); results and gradients are token-major, seen as (B, H, T, D).  Gradients are bitwise reproducible; there is no
second derivative and no forward-mode one.  No CPU path: a missing library raises.
"""
import torch
from torch.autograd.function import once_differentiable

import slotscan_lib as L
from slotrope_hip import _same_device, check_caches, check_lens

_TYPES = (torch.bfloat16, torch.float16)
_D = (64, 128)
_NO_WINDOW = 2 ** 31 - 1


def _check(q, k, v, scale, window, cap, slopes, prefix, what):
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise ValueError(f"{what}: expected q (B, Hq, Tq, D) and k, v (B, Hk, Tk, D); got {tuple(q.shape)}, {tuple(k.shape)}, "
                         f"{tuple(v.shape)}")
    if k.shape[1] < 1 or q.shape[1] < 1 or q.shape[1] % k.shape[1]:
        raise ValueError(f"{what}: the query heads must be a multiple of the key/value heads")
    if q.dtype not in _TYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise NotImplementedError(f"{what} computes in bf16 or fp16, all operands alike (got {q.dtype}, {k.dtype}, {v.dtype})")
    if q.shape[3] not in _D:
        raise NotImplementedError(f"{what} needs D in {_D} (got {q.shape[3]})")
    if window is not None and int(window) < 1:
        raise ValueError(f"{what}: window must be >= 1 or None (got {window})")
    if cap is not None and not 1e-30 <= float(cap) <= 1e30:
        raise ValueError(f"{what}: cap must be in [1e-30, 1e30] or None (got {cap})")
    if scale is not None and not 1e-30 <= abs(scale) <= 1e30:
        raise ValueError(f"{what}: |scale| must be in [1e-30, 1e30] (got {scale})")
    if cap is not None and float(cap) > 1e36 * (q.shape[3] ** -0.5 if scale is None else abs(scale)):
        raise ValueError(f"{what}: cap must be at most 1e36 |scale| (got {cap}, scale {scale})")
    if slopes is not None:
        if slopes.shape != (q.shape[1],) or slopes.dtype != torch.float32:
            raise ValueError(f"{what}: slopes must be fp32 ({q.shape[1]},) (got {slopes.dtype}, {tuple(slopes.shape)})")
        if slopes.requires_grad and torch.is_grad_enabled():
            raise NotImplementedError(f"{what}: the slopes are constants (no gradient)")
    L.check_tangents(what, q, k, v, slopes)
    if prefix is not None and (prefix.dtype != torch.int32 or prefix.shape != (q.shape[0],)):
        raise ValueError(f"{what}: prefix must be int32 ({q.shape[0]},) (got {prefix.dtype}, {tuple(prefix.shape)})")


def _documents(docs, B, T):
    ws = torch.empty(L.lib().slotattn_docs_bytes(B, T), device=docs.device, dtype=torch.uint8)
    L.check(L.lib().slotattn_docs(L.ptr(docs), B, T, L.ptr(ws), L.stream_of(docs.device)), "slotattn_docs")
    return ws


def _launch_fwd(q_, k_, v_, opts, slopes, dws, prefix, lens, keep):
    """out (B, Tq, Hq, D) and, to keep for a backward, what rounding took from it and lse; on the current device."""
    scale, causal, window, cap = opts
    B, Hq, Tq, D = q_.shape
    Hk, Tk = k_.shape[1:3]
    dev, lib = q_.device, L.lib()
    out = torch.empty(B, Tq, Hq, D, device=dev, dtype=q_.dtype)
    res = torch.empty_like(out) if keep else None
    lse = torch.empty(B, Hq, Tq, device=dev, dtype=torch.float32) if keep else None
    n = lib.slotattn_fwd_workspace(B, Tq, Tk, Hq, Hk, D, causal, window, dws is not None, prefix is not None,
                                   lens is not None)
    ws = torch.empty(n, device=dev, dtype=torch.uint8) if n else None
    rc = lib.slotattn_fwd(*L.strided(q_), *L.strided(k_), *L.strided(v_), L._TYPE_CODES[q_.dtype], B, Tq, Tk, Hq, Hk, D, scale,
                          causal, window, cap, L.ptr(slopes), L.ptr(dws), L.ptr(prefix), L.ptr(lens), L.ptr(ws), L.ptr(out),
                          L.ptr(res), L.ptr(lse), L.stream_of(dev))
    L.check(rc, "slotattn_fwd")
    return out, res, lse


class _Attend(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, opts, slopes, docs, prefix):
        q_, k_, v_ = L.rows(q), L.rows(k), L.rows(v)
        with L.on(q.device):
            dws = None if docs is None else _documents(docs, k.shape[0], k.shape[2])
            out, res, lse = _launch_fwd(q_, k_, v_, opts, slopes, dws, prefix, None, True)
        ctx.save_for_backward(q_, k_, v_, out, res, lse, slopes, dws, prefix)
        ctx.opts = opts
        return out.transpose(1, 2)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q_, k_, v_, out, res, lse, slopes, dws, prefix = ctx.saved_tensors
        scale, causal, window, cap = ctx.opts
        B, Hq, Tq, D = q_.shape
        Hk, Tk = k_.shape[1:3]
        dev, dt, lib = q_.device, q_.dtype, L.lib()
        do = L.rows(dout)
        dq = torch.empty(B, Tq, Hq, D, device=dev, dtype=dt)
        dk, dv = (torch.empty(B, Tk, Hk, D, device=dev, dtype=dt) for _ in range(2))
        delta = torch.empty_like(lse)
        n = lib.slotattn_bwd_workspace(B, Tq, Tk, Hq, Hk, D, causal, window, prefix is not None)
        ws = torch.empty(n, device=dev, dtype=torch.uint8) if n else None
        with L.on(dev):
            rc = lib.slotattn_bwd(*L.strided(q_), *L.strided(k_), *L.strided(v_), L._TYPE_CODES[dt], B, Tq, Tk, Hq, Hk, D, scale,
                                  causal, window, cap, L.ptr(slopes), L.ptr(dws), L.ptr(prefix), L.ptr(out), L.ptr(res), L.ptr(lse),
                                  *L.strided(do), L.ptr(ws), L.ptr(delta), L.ptr(dq), L.ptr(dk), L.ptr(dv), L.stream_of(dev))
        L.check(rc, "slotattn_bwd")
        return dq.transpose(1, 2), dk.transpose(1, 2), dv.transpose(1, 2), None, None, None, None


def _opts(q, scale, causal, window, cap):
    return (q.shape[3] ** -0.5 if scale is None else float(scale), int(bool(causal)),
            _NO_WINDOW if window is None else min(int(window), _NO_WINDOW), 0.0 if cap is None else float(cap))


def attend(q, k, v, scale=None, causal=True, window=None, cap=None, slopes=None, docs=None, prefix=None):
    """Attention over the visible keys (see the module docstring)."""
    _check(q, k, v, scale, window, cap, slopes, prefix, "attend")
    B, Hq, Tq, D = q.shape
    Tk = k.shape[2]
    if Tq > Tk:
        raise ValueError(f"attend: the queries are the last of the keys' positions: {Tq} queries, {Tk} keys")
    if docs is not None:
        if docs.shape != (B, Tk) or docs.dtype != torch.int32:
            raise ValueError(f"attend: docs must be int32 ({B}, {Tk}) (got {docs.dtype}, {tuple(docs.shape)})")
        docs = docs.contiguous()
    _same_device("attend", q, k, v, slopes, docs, prefix)
    if B * Tq == 0:
        return q * 0 + k[:, :0].sum() + v[:, :0].sum()   # no query: an empty result, and zeros as the gradients
    slopes, prefix = (None if x is None else x.contiguous() for x in (slopes, prefix))
    opts = _opts(q, scale, causal, window, cap)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _Attend.apply(q, k, v, opts, slopes, docs, prefix)
    with L.on(q.device):
        dws = None if docs is None else _documents(docs, B, Tk)
        return _launch_fwd(L.rows(q), L.rows(k), L.rows(v), opts, slopes, dws, prefix, None, False)[0].transpose(1, 2)


def attend_cache(q, kcache, vcache, lens, scale=None, window=None, cap=None, slopes=None, prefix=None):
    """Causal attention of the newest tokens over a cache of ragged lengths (see the module docstring)."""
    what = "attend_cache"
    _check(q, kcache, vcache, scale, window, cap, slopes, prefix, what)
    check_caches(kcache, vcache, q, kcache.shape[1], what)
    check_lens(lens, q.shape[0], what)
    if torch.is_grad_enabled() and (q.requires_grad or kcache.requires_grad or vcache.requires_grad):
        raise RuntimeError(f"{what} has no backward: call it under torch.no_grad()")
    _same_device(what, q, kcache, vcache, lens, slopes, prefix)
    if q.shape[0] * q.shape[2] == 0:
        return torch.empty_like(q)
    slopes, prefix = (None if x is None else x.contiguous() for x in (slopes, prefix))
    with L.on(q.device):
        return _launch_fwd(L.rows(q), L.rows(kcache), L.rows(vcache), _opts(q, scale, True, window, cap), slopes, None, prefix, lens,
                           False)[0].transpose(1, 2)
