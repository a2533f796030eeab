"""Head norm and position rotation of queries and keys on MI355X (include/slotrope.h), one kernel each way: what a layer
does to its projected queries and keys before the attention (slotattn_hip, slotwin_hip).

    qk_rope(q, k, wq, wk, freqs, positions=None, eps=1e-6, interleaved=False) -> (q', k')
        q (B, Hq, T, D), k (B, Hk, T, D).  Every head's row is normed by its root mean square and scaled by the gain wq or
        wk (D,; None: no gain), then its first 2 len(freqs) values are rotated: pair i -- (i, i + len(freqs)), or with
        `interleaved` (2 i, 2 i + 1) -- by the angle position * freqs[i].  positions (T,) or (B, T), int32 or int64;
        None: 0 .. T - 1.  Autograd gives dq, dk, dwq, dwk; frequencies and positions are constants.
    qk_rope_cache(q, k, v, wq, wk, freqs, lens, kcache, vcache, eps=1e-6, interleaved=False) -> q'
        the serving form, forward only: the T tokens are the newest of lens[b] (int32 (B,), the new ones included), token
        t at position lens[b] - T + t; the prepared keys and the values are written into rows `position` of kcache, vcache
        (B, Hk, S, D), everything else in them stays.  A token of negative position or of one past the cache writes nothing,
        so that first prompts of unlike lengths may be padded on the left.  Later calls may not: the padding's positions
        would be those of earlier tokens, whose rows it would overwrite.  The caches share no memory with each other or with the operands.
    qk_rope_pages(q, k, v, wq, wk, freqs, pos, slots, kpages, vpages, eps=1e-6, interleaved=False) -> q'
        the serving form over a cache in pages (slotpage_hip), forward only: q (N, Hq, D), k, v (N, Hk, D) are packed tokens of many
        sequences, pos and slots (N,) int32 and int64 their positions and places as page_extend gives them.  Token i's prepared key and
        its value are written into row slots[i] % page of page slots[i] // page of kpages, vpages (P, Hk, page, D); a slot outside
        of the pages (-1) writes nothing.  q' (N, Hq, D) is written whole.  Slots of one call are different.
    frequencies(rot, theta=10000.0, device=None) -> (rot / 2,) float64: theta^(-2 i / rot)

bf16, fp16 or fp32 rows (q, k, v and the caches alike), D in {64, 128}, 2 len(freqs) a multiple of 16 up to D; freqs are
float64, so that a far position keeps its angle.  Sums are fp32, results rounded once; the gains' gradients are summed in
a fixed order; there is no second derivative and no forward-mode one.  Operands may be any views whose rows are contiguous
and 16-byte aligned, such as slices of one fused projection (others are copied); results are token-major, seen as
(B, H, T, D).  No CPU path: a missing library raises.
"""
import torch
from torch.autograd.function import once_differentiable

import slotscan_lib as L

_D = (64, 128)


def frequencies(rot, theta=10000.0, device=None):
    """The rot / 2 angular frequencies theta^(-2 i / rot), float64."""
    return float(theta) ** (-2.0 * torch.arange(rot // 2, device=device, dtype=torch.float64) / rot)


def _check(q, k, wq, wk, freqs, what):
    if q.dim() != 4 or k.dim() != 4 or q.shape[0] != k.shape[0] or q.shape[2:] != k.shape[2:]:
        raise ValueError(f"{what}: expected q (B, Hq, T, D) and k (B, Hk, T, D); got {tuple(q.shape)}, {tuple(k.shape)}")
    _check_rows(q, k, wq, wk, freqs, what)


def _check_rows(q, k, wq, wk, freqs, what):
    if q.shape[1] < 1 or k.shape[1] < 1:
        raise ValueError(f"{what}: needs at least one head of queries and of keys")
    if q.dtype not in L._TYPE_CODES or k.dtype != q.dtype:
        raise NotImplementedError(f"{what} takes bf16, fp16 or fp32 queries and keys of one type (got {q.dtype}, {k.dtype})")
    D = q.shape[-1]
    if D not in _D:
        raise NotImplementedError(f"{what} needs D in {_D} (got {D})")
    if freqs.dim() != 1 or freqs.dtype != torch.float64:
        raise ValueError(f"{what}: freqs must be a float64 vector (got {freqs.dtype}, {tuple(freqs.shape)})")
    if freqs.numel() % 8 or 2 * freqs.numel() > D:
        raise NotImplementedError(f"{what} rotates a multiple of 16 values, at most D (got 2 x {freqs.numel()})")
    if freqs.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError(f"{what}: the frequencies are constants")
    for w in (wq, wk):
        if w is not None and (w.shape != (D,) or w.dtype not in L._TYPE_CODES):
            raise ValueError(f"{what}: a gain must be ({D},), bf16, fp16 or fp32 (got {tuple(w.shape)}, {w.dtype})")
    L.check_tangents(what, q, k, wq, wk, freqs)


def _same_device(what, *ts):
    d = ts[0].get_device()                               # (numbers compare faster than devices)
    if d >= 0:
        for t in ts:
            if t is not None and t.get_device() != d:
                break
        else:
            return
    dev = ts[0].device
    for t in ts:
        if t is not None and t.device != dev:
            raise ValueError(f"{what}: every tensor must be on one device (got {dev} and {t.device})")
    if dev.type != "cuda":
        raise RuntimeError(f"{what} runs on GPU tensors only (no CPU path in this package)")


def _vec(x):
    x = x.contiguous()
    return x.clone() if x.data_ptr() % 16 else x


def _gains(wq, wk):
    """Both gains in one type, 16-byte aligned."""
    if wq is not None and wk is not None and wq.dtype != wk.dtype:
        wq, wk = wq.float(), wk.float()
    w = wq if wq is not None else wk
    return (None if wq is None else _vec(wq)), (None if wk is None else _vec(wk)), 0 if w is None else L._TYPE_CODES[w.dtype]


def _launch_fwd(q_, k_, wq_, wk_, wt, freqs, positions, eps, inter):
    B, Hq, T, D = q_.shape
    Hk = k_.shape[1]
    qo = torch.empty(B, T, Hq, D, device=q_.device, dtype=q_.dtype)
    ko = torch.empty(B, T, Hk, D, device=q_.device, dtype=q_.dtype)
    if B * T:
        with L.on(q_.device):
            rc = L.lib().slotrope_fwd(*L.strided(q_), *L.strided(k_), L._TYPE_CODES[q_.dtype], L.ptr(wq_), L.ptr(wk_), wt,
                                      L.ptr(freqs), 2 * freqs.numel(), inter, *_pos(positions), B, T, Hq, Hk, D, eps, L.ptr(qo),
                                      L.ptr(ko), L.stream_of(q_.device))
        L.check(rc, "slotrope_fwd")
    return qo.transpose(1, 2), ko.transpose(1, 2)


def _pos(p):
    """Pointer, whether 64 bits, stride of a row of the positions."""
    if p is None:
        return None, 0, 0
    return p.data_ptr(), int(p.dtype == torch.int64), p.stride(0) if p.dim() == 2 else 0


class _Rope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, wq, wk, freqs, positions, eps, inter):
        q_, k_ = L.rows(q), L.rows(k)
        wq_, wk_, wt = _gains(wq, wk)
        ctx.save_for_backward(q_, k_, wq_, wk_, freqs, positions)
        ctx.meta = (wt, eps, inter, None if wq is None else wq.dtype, None if wk is None else wk.dtype)
        return _launch_fwd(q_, k_, wq_, wk_, wt, freqs, positions, eps, inter)

    @staticmethod
    @once_differentiable
    def backward(ctx, dqo, dko):
        q_, k_, wq_, wk_, freqs, positions = ctx.saved_tensors
        wt, eps, inter, tq, tk = ctx.meta
        B, Hq, T, D = q_.shape
        Hk, dev, dt = k_.shape[1], q_.device, q_.dtype
        dq = torch.empty(B, T, Hq, D, device=dev, dtype=dt)
        dk = torch.empty(B, T, Hk, D, device=dev, dtype=dt)
        want = [w is not None and ctx.needs_input_grad[2 + i] for i, w in enumerate((wq_, wk_))]
        dw = [torch.zeros_like(w) if n and not B * T else torch.empty_like(w) if n else None for n, w in zip(want, (wq_, wk_))]
        if B * T:
            dqo, dko = L.rows(dqo), L.rows(dko)
            with L.on(dev):
                ws = torch.empty(L.lib().slotrope_bwd_workspace(B, T, Hq, Hk, D), device=dev, dtype=torch.uint8) if any(want) else None
                rc = L.lib().slotrope_bwd(*L.strided(q_), *L.strided(k_), L._TYPE_CODES[dt], L.ptr(wq_), L.ptr(wk_), wt, L.ptr(freqs),
                                          2 * freqs.numel(), inter, *_pos(positions), B, T, Hq, Hk, D, eps, *L.strided(dqo),
                                          *L.strided(dko), L.ptr(ws), L.ptr(dq), L.ptr(dk), L.ptr(dw[0]), L.ptr(dw[1]),
                                          L.stream_of(dev))
            L.check(rc, "slotrope_bwd")
        dw = [None if d is None else d.to(t) for d, t in zip(dw, (tq, tk))]
        return dq.transpose(1, 2), dk.transpose(1, 2), dw[0], dw[1], None, None, None, None


def qk_rope(q, k, wq, wk, freqs, positions=None, eps=1e-6, interleaved=False):
    """Normed and rotated queries and keys (see the module docstring)."""
    _check(q, k, wq, wk, freqs, "qk_rope")
    B, _, T, _ = q.shape
    if positions is not None:
        if positions.dtype not in (torch.int32, torch.int64) or tuple(positions.shape) not in ((T,), (B, T)):
            raise ValueError(f"qk_rope: positions must be ({T},) or ({B}, {T}), int32 or int64 (got {tuple(positions.shape)}, {positions.dtype})")
        if positions.stride(-1) != 1:
            positions = positions.contiguous()
    _same_device("qk_rope", q, k, wq, wk, freqs, positions)
    freqs = freqs.contiguous()
    if torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in (q, k, wq, wk)):
        return _Rope.apply(q, k, wq, wk, freqs, positions, float(eps), int(bool(interleaved)))
    return _launch_fwd(L.rows(q), L.rows(k), *_gains(wq, wk), freqs, positions, float(eps), int(bool(interleaved)))


def check_caches(kcache, vcache, like, Hk, what):
    """The shape, type and layout of a pair of caches (B, Hk, S, D) that are read or written in place."""
    B, D = like.shape[0], like.shape[3]
    if kcache.dim() != 4 or vcache.shape != kcache.shape or kcache.shape[0] != B or kcache.shape[1] != Hk or kcache.shape[3] != D \
            or kcache.shape[2] < 1:
        raise ValueError(f"{what}: expected caches ({B}, {Hk}, S, {D}), S >= 1; got {tuple(kcache.shape)}, {tuple(vcache.shape)}")
    if kcache.dtype != like.dtype or vcache.dtype != like.dtype:
        raise NotImplementedError(f"{what}: the caches must have the queries' type {like.dtype} (got {kcache.dtype}, {vcache.dtype})")


def _apart(c, steps=()):
    """Whether no two rows of c (B, H, S, D) share memory: every dimension steps over all that the closer ones reach.  steps:
    further dimensions, as (stride, size)."""
    st, size = c.stride(), c.shape
    reach = size[3]
    for s, n in sorted([(st[0], size[0]), (st[1], size[1]), (st[2], size[2]), *steps]):
        if n > 1:
            if s < reach:
                return False
            reach += s * (n - 1)
    return True


def _overlap(a, b):
    """Whether two caches of one shape share memory.  Where the memory that they reach over does not meet they do not; where it does
    they may lie side by side, as two parts of one buffer with the same strides; anything else counts as sharing."""
    d, n, st, size = b.data_ptr() - a.data_ptr(), a.element_size(), a.stride(), a.shape
    if d < 0:
        return _overlap(b, a)
    if d >= n * (1 + (size[0] - 1) * st[0] + (size[1] - 1) * st[1] + (size[2] - 1) * st[2] + (size[3] - 1) * st[3]) or not a.numel():
        return False
    same = all(st[i] == b.stride(i) for i in range(3) if size[i] > 1)
    return not (same and d % n == 0 and _apart(a, [(d // n, 2)]))


def check_lens(lens, B, what):
    if lens.dtype != torch.int32 or lens.shape != (B,) or not lens.is_contiguous():
        raise ValueError(f"{what}: lens must be a contiguous int32 ({B},) (got {lens.dtype}, {tuple(lens.shape)})")


def qk_rope_cache(q, k, v, wq, wk, freqs, lens, kcache, vcache, eps=1e-6, interleaved=False):
    """Prepared queries of the newest tokens, their keys and values written into the caches (see the module docstring)."""
    what = "qk_rope_cache"
    _check(q, k, wq, wk, freqs, what)
    B, Hq, T, D = q.shape
    Hk = k.shape[1]
    if v.shape != k.shape or v.dtype != k.dtype:
        raise ValueError(f"{what}: v must have k's shape and type (got {tuple(v.shape)}, {v.dtype})")
    check_caches(kcache, vcache, q, Hk, what)
    check_lens(lens, B, what)
    L.check_tangents(what, v, kcache, vcache)
    if torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in (q, k, v, wq, wk, kcache, vcache)):
        raise RuntimeError(f"{what} has no backward: call it under torch.no_grad()")
    _check_written(kcache, vcache, what)
    _same_device(what, q, k, v, wq, wk, freqs, lens, kcache, vcache)
    q_, k_, v_ = L.rows(q), L.rows(k), L.rows(v)
    wq_, wk_, wt = _gains(wq, wk)
    freqs = freqs.contiguous()
    qo = torch.empty(B, T, Hq, D, device=q.device, dtype=q.dtype)
    if B * T:
        with L.on(q.device):
            rc = L.lib().slotrope_cache(*L.strided(q_), *L.strided(k_), *L.strided(v_), L._TYPE_CODES[q.dtype], L.ptr(wq_), L.ptr(wk_),
                                        wt, L.ptr(freqs), 2 * freqs.numel(), int(bool(interleaved)), L.ptr(lens), B, T, Hq, Hk, D,
                                        kcache.shape[2], float(eps), L.ptr(qo), *L.strided(kcache), *L.strided(vcache),
                                        L.stream_of(q.device))
        L.check(rc, what)
        _written(kcache, vcache)
    return qo.transpose(1, 2)


def _check_written(kcache, vcache, what):
    n, d = kcache.numel() * kcache.element_size(), kcache.data_ptr() - vcache.data_ptr()
    if kcache.is_contiguous() and vcache.is_contiguous() and (d >= n or -d >= n) and not (kcache.data_ptr() | vcache.data_ptr()) % 16 \
            and kcache.shape[2] * kcache.shape[3] < 1 << 25:
        return                                           # the common case (2 us less)
    for c in (kcache, vcache):
        if not _apart(c) or not L.in_place(c):
            raise ValueError(f"{what}: a cache is written in place: its rows must be contiguous, 16-byte aligned and apart")
    if _overlap(kcache, vcache):
        raise ValueError(f"{what}: the two caches share memory")


def _written(*xs):
    """Raises the versions of tensors that a kernel wrote."""
    try:
        torch._C._increment_version(xs)
    except RuntimeError:                                 # inference tensors have none
        torch._C._increment_version([x for x in xs if not x.is_inference()])


def check_pools(kpages, vpages, like, Hk, what):
    """The shape, type and layout of the pages (P, Hk, page, D) of the keys and values, which are read or written in place."""
    if kpages.dim() != 4 or vpages.shape != kpages.shape or kpages.shape[1] != Hk or kpages.shape[3] != like.shape[2]:
        raise ValueError(f"{what}: expected pages (P, {Hk}, page, {like.shape[2]}); got {tuple(kpages.shape)}, {tuple(vpages.shape)}")
    check_page(kpages.shape[2], what)
    if kpages.dtype != like.dtype or vpages.dtype != like.dtype:
        raise NotImplementedError(f"{what}: the pages must have the queries' type {like.dtype} (got {kpages.dtype}, {vpages.dtype})")


def check_page(page, what):
    if page < 16 or page > 4096 or page & (page - 1):
        raise ValueError(f"{what}: a page must hold a power of two of tokens, 16 to 4096 (got {page})")


def check_ints(x, shape, dtype, what, name):
    if x.dtype is not dtype or x.shape != shape or not x.is_contiguous():
        raise ValueError(f"{what}: {name} must be a contiguous {str(dtype)[6:]} {shape} (got {x.dtype}, {tuple(x.shape)})")


def qk_rope_pages(q, k, v, wq, wk, freqs, pos, slots, kpages, vpages, eps=1e-6, interleaved=False):
    """Prepared queries of packed tokens, their keys and values written into the pages (see the module docstring)."""
    what = "qk_rope_pages"
    if q.dim() != 3 or k.dim() != 3 or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
        raise ValueError(f"{what}: expected q (N, Hq, D) and k (N, Hk, D); got {tuple(q.shape)}, {tuple(k.shape)}")
    _check_rows(q, k, wq, wk, freqs, what)
    if v.shape != k.shape or v.dtype != k.dtype:
        raise ValueError(f"{what}: v must have k's shape and type (got {tuple(v.shape)}, {v.dtype})")
    N, Hq, D = q.shape
    Hk = k.shape[1]
    check_pools(kpages, vpages, q, Hk, what)
    check_ints(pos, (N,), torch.int32, what, "pos")
    check_ints(slots, (N,), torch.int64, what, "slots")
    L.check_tangents(what, v, kpages, vpages)
    if torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in (q, k, v, wq, wk, kpages, vpages)):
        raise RuntimeError(f"{what} has no backward: call it under torch.no_grad()")
    P, page = kpages.shape[0], kpages.shape[2]
    if not P:
        raise ValueError(f"{what}: there are no pages to write into")
    _check_written(kpages, vpages, what)
    _same_device(what, q, k, v, wq, wk, freqs, pos, slots, kpages, vpages)
    q_, k_, v_ = L.tokens(q), L.tokens(k), L.tokens(v)
    wq_, wk_, wt = _gains(wq, wk)
    freqs = freqs.contiguous()
    qo = torch.empty(N, Hq, D, device=q.device, dtype=q.dtype)
    if N:
        L.call(L.lib().slotrope_pages, what, q.device, *L.by_head(q_), *L.by_head(k_), *L.by_head(v_), L._TYPE_CODES[q.dtype], L.ptr(wq_),
               L.ptr(wk_), wt, freqs.data_ptr(), 2 * freqs.numel(), int(bool(interleaved)), pos.data_ptr(), slots.data_ptr(), N, Hq, Hk, D,
               P, page, float(eps), qo.data_ptr(), *L.strided(kpages), *L.strided(vpages))
        _written(kpages, vpages)
    return qo
