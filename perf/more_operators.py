"""Serving from caches in pages, as cases for measuring its operators' time and outputs.

A case is a dict of plain values; `op` names the entry point:
    pages         page_extend and page_trim: pages handed out to the rows whose sequences grow, with the packed batch's starts,
                  positions and slots, and the same pages taken back, as after guessed tokens that are rejected
    rope_pages    qk_rope_pages: the norm of every query and key head of a packed batch with the position rotation, keys and
                  values written into the pages by their slots
    attend_pages  attend_pages: a packed batch's queries -- one token of a sequence, a few, or a prompt's -- against the
                  sequences' pages

Every case is a batch of R rows; the lengths are ragged and follow from the case alone.  Tokens are packed, (N, heads, D),
the last `pad` of them belonging to no row.  Where `own` is false, run() computes the operators with elementary torch
operations in 32 bits (the angles of the rotation in 64), rounded once at the end.
"""
import math
import os
import random
import sys

import torch

own = False

_PKG = os.path.join(os.getcwd(), "smal-memory-llm_amd")
EPS = 1e-6
THETA = 10000.0
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
GAIN = 1.4           # rows of normed queries and keys: scores of a standard deviation of 2


def listed():
    # ones: share of the rows with one new token, the others have new_lo to new_hi of them; idle: share of rows without any
    rows = dict(ones=0.0, idle=0.0, new_lo=1, new_hi=1, pad=0)
    step = dict(rows, ones=1.0)
    pg = dict(op="pages")
    ro = dict(op="rope_pages", pairs=False, tokens=False)
    at = dict(op="attend_pages", window=0, cap=0.0, slopes=False, prefix=0, tokens=False)
    return [
        # one generated token of 256 sequences: every 16th of them needs a page
        dict(step, **pg, name="pages_step", R=256, ctx_lo=1, ctx_hi=8000, page=16, spare=100, mix=1),
        # prompts and continuations of 64 sequences, some of which have no room
        dict(rows, **pg, name="pages_prompt", R=64, idle=0.1, new_lo=16, new_hi=2048, ctx_lo=1, ctx_hi=2000, page=64, spare=-40, mix=2,
             pad=64),
        # one generated token of 128 sequences: latency
        dict(step, **ro, name="write_step", R=128, ctx_lo=1, ctx_hi=2000, page=64, Hq=12, Hk=4, D=128, rot=128, dtype="bf16", mix=3),
        # twelve prompts of unlike lengths side by side
        dict(rows, **ro, name="write_prompt", R=12, new_lo=200, new_hi=1500, ctx_lo=0, ctx_hi=0, page=16, Hq=6, Hk=6, D=64, rot=64,
             dtype="f16", mix=4, pad=100),
        # one token of four short sequences: the smallest, latency
        dict(step, **at, name="attend_tiny", R=4, ctx_lo=50, ctx_hi=500, page=16, Hq=6, Hk=2, D=64, dtype="f16", mix=5),
        # one token of 32 sequences of up to 8,192 with capped scores: the pages' bytes
        dict(step, **dict(at, cap=50.0), name="attend_step", R=32, ctx_lo=1024, ctx_hi=8191, page=64, Hq=12, Hk=4, D=128, dtype="bf16",
             mix=6),
        # one token of one very long sequence: the work has to be split over its length
        dict(step, **at, name="attend_far", R=1, ctx_lo=131071, ctx_hi=131071, page=256, Hq=12, Hk=4, D=128, dtype="bf16", mix=7),
        # one token of many sequences under a sliding window, small pages
        dict(step, **dict(at, window=1024), name="attend_many", R=256, ctx_lo=64, ctx_hi=4000, page=16, Hq=12, Hk=4, D=128, dtype="bf16",
             mix=8),
        # guessed tokens of sixteen sequences being verified
        dict(rows, **dict(at, tokens=True), name="attend_guess", R=16, new_lo=2, new_hi=8, ctx_lo=500, ctx_hi=16000, page=32, Hq=12, Hk=4,
             D=128, dtype="bf16", mix=9),
        # sequences that generate beside prompts that are read
        dict(rows, **at, name="attend_mixed", R=60, ones=0.93, new_lo=300, new_hi=1200, ctx_lo=200, ctx_hi=4000, page=16, Hq=12, Hk=4,
             D=128, dtype="bf16", mix=10),
        # odd lengths, a bias that falls with the distance, half precision, padding behind the last token
        dict(rows, **dict(at, slopes=True, prefix=1), name="attend_slopes", R=5, new_lo=100, new_hi=700, ctx_lo=1, ctx_hi=900, page=32,
             Hq=6, Hk=6, D=64, dtype="f16", mix=11, pad=37),
        # two first prompts of 4,096 tokens: the largest
        dict(rows, **at, name="attend_prompt", R=2, new_lo=4096, new_hi=4096, ctx_lo=0, ctx_hi=0, page=64, Hq=12, Hk=4, D=128, dtype="bf16",
             mix=12),
    ]


def _log(rng, lo, hi):
    if lo < 1:
        return rng.randint(lo, hi)
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["pages", "rope_pages", "attend_pages", "attend_pages", "attend_pages"])
    c = dict(op=op, page=rng.choice([16, 16, 32, 64, 128, 256]), mix=rng.randrange(1 << 20), idle=rng.choice([0.0, 0.0, 0.1]),
             pad=rng.choice([0, 0, rng.randrange(1, 100)]))
    kind = rng.choice(["step", "step", "guess", "mixed", "prompt"])
    c["ones"] = dict(step=1.0, guess=0.0, mixed=0.9, prompt=0.0)[kind]
    top = dict(step=1, guess=rng.choice([2, 4, 9]), mixed=_log(rng, 16, 1500), prompt=_log(rng, 2, 3000))[kind]
    c["new_lo"], c["new_hi"] = max(1, top // 4), top
    c["ctx_hi"] = 0 if kind == "prompt" and rng.random() < 0.5 else _log(rng, 8, 30000)
    c["ctx_lo"] = c["ctx_hi"] // 8
    big = kind in ("mixed", "prompt")
    if op == "pages":
        c["R"] = _log(rng, 1, 32 if big else 2000)
        c["spare"] = rng.choice([0, 50, 1000, -10, -100])
        return c
    Hk = rng.choice([1, 2, 4, 4, 6, 8])
    c.update(Hk=Hk, Hq=Hk * rng.choice([1, 1, 2, 3, 4]), D=rng.choice([64, 128, 128]), dtype=rng.choice(["bf16", "bf16", "f16"]),
             tokens=rng.random() < 0.3)
    if op == "rope_pages":
        c.update(pairs=rng.random() < 0.4, rot=rng.choice([16, 32, 64, c["D"], c["D"]]), dtype=rng.choice(["bf16", "bf16", "f16", "f32"]))
        c["ctx_hi"] = min(c["ctx_hi"], 4000)
        c["ctx_lo"] = c["ctx_hi"] // 8
        c["R"] = _log(rng, 1, max(1, min(256, 100000 // (c["ctx_hi"] + top), 8000 // top)))
        return c
    c.update(window=rng.choice([0, 0, _log(rng, 8, 2048)]), cap=rng.choice([0.0, 0.0, 30.0]), slopes=rng.random() < 0.25,
             prefix=rng.choice([0, 0, 0, 1]))
    cost = c["Hq"] * c["D"] * (top + c["ctx_hi"]) * (top if kind != "mixed" else max(1, top // 8))
    c["R"] = _log(rng, 1, max(1, min(256, 800000 // Hk // (c["ctx_hi"] + top), 12 * 128 * 2 * 4096 * 2048 // cost)))
    return c


# ---- inputs -------------------------------------------------------------------------------------------------


def _rows(c):
    """(tokens that a sequence has, new ones) of every row, by the case alone."""
    rng = random.Random(c["mix"])
    out = []
    for r in range(c["R"]):
        new = 1 if rng.random() < c["ones"] else _log(rng, c["new_lo"], c["new_hi"])
        if rng.random() < c["idle"] and r:
            new = 0
        out.append((_log(rng, c["ctx_lo"], c["ctx_hi"]), new))
    return out


def _prefixes(c):
    """First tokens of every row that its later ones are read with both ways."""
    rng = random.Random(c["mix"] + 1)
    return [rng.randrange(0, max(1, (ctx + new) // 2)) for ctx, new in _rows(c)]


def _up(n, page):
    return -(-n // page)


def prepare(case, seed):
    c = case
    dev = torch.device("cuda:0")
    gen = torch.Generator(device=dev).manual_seed(int(seed) * 7919 + 17)
    ints = lambda x: torch.tensor(x, device=dev, dtype=torch.int32)
    rows, page = _rows(c), c["page"]
    tokens = sum(n for _, n in rows)
    s = dict(case=c, N=tokens + c["pad"])
    # pages in no order, as a pool that has been in use for long hands them out
    held = [_up(ctx + (n if c["op"] != "pages" else 0), page) for ctx, n in rows]
    M = max(max(_up(ctx + n, page) for ctx, n in rows), 1) + 3
    left = max(0, sum(_up(ctx + n, page) - _up(ctx, page) for ctx, n in rows) + c["spare"]) if c["op"] == "pages" else 5
    P = sum(held) + left
    ids = torch.randperm(P, device=dev, generator=gen).to(torch.int32)
    at = torch.arange(M, device=dev) + ints([sum(held[:r]) for r in range(len(held))]).unsqueeze(-1)
    s["table"] = torch.where(torch.arange(M, device=dev) < ints(held).unsqueeze(-1), ids[at.clamp(max=P - 1)], -1).to(torch.int32)
    if c["op"] == "pages":
        s["new"], s["before"] = ints([n for _, n in rows]), ints([ctx for ctx, _ in rows])
        s["lens"] = s["before"].clone()
        s["free"] = torch.cat((ints([left]), ids[sum(held):], ids[:sum(held)]))
        return s
    dt = TYPES[c["dtype"]]
    rn = lambda *sh: torch.randn(*sh, device=dev, generator=gen)
    N, Hq, Hk, D = s["N"], c["Hq"], c["Hk"], c["D"]
    # a page holds its heads one after another, or its tokens
    pool = lambda gain: (gain * rn(P, page, Hk, D)).to(dt).transpose(1, 2) if c["tokens"] else (gain * rn(P, Hk, page, D)).to(dt)
    s["starts"] = ints([sum(n for _, n in rows[:r]) for r in range(len(rows) + 1)])
    s["ends"] = ints([ctx + n if n else 0 for ctx, n in rows])
    s["rows"] = rows
    if c["op"] == "rope_pages":
        qkv = rn(N, Hq + 2 * Hk, D).to(dt)
        s["q"], s["k"], s["v"] = qkv.split([Hq, Hk, Hk], dim=1)
        s["wq"], s["wk"] = ((1.0 + 0.2 * rn(D)).to(dt) for _ in range(2))
        s["freqs"] = THETA ** (-2.0 * torch.arange(c["rot"] // 2, device=dev, dtype=torch.float64) / c["rot"])
        s["pos"] = ints(sum((list(range(ctx, ctx + n)) for ctx, n in rows), []) + [-1] * c["pad"])
        row = torch.repeat_interleave(torch.arange(len(rows), device=dev), ints([n for _, n in rows]))
        p = s["pos"][:tokens].long()
        s["slots"] = torch.full((N,), -1, device=dev, dtype=torch.int64)
        s["slots"][:tokens] = s["table"][row, p // page].long() * page + p % page
        s["kp"], s["vp"] = pool(1.0), pool(1.0)
        return s
    s["q"] = (GAIN * rn(N, Hq, D)).to(dt)
    s["kp"], s["vp"] = pool(GAIN), pool(1.0)
    s["most"] = max(n for _, n in rows)
    # slopes as a geometric series over the heads
    s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, Hq + 1, device=dev, dtype=torch.float32) / Hq) if c["slopes"] else None
    s["prefix"] = ints(_prefixes(c)) if c["prefix"] else None
    return s


# ---- the plain forms ----------------------------------------------------------------------------------------


def _plain_extend(new, lens, table, free, page, N):
    R, M = table.shape
    dev = new.device
    new, have, n = new.long().clamp_min(0), lens.long(), free[0].long()
    ends = torch.cumsum(new, 0)
    pages = lambda x: (x + page - 1) // page
    ok = (new > 0) & (ends <= N) & (have + new <= M * page)
    need = torch.where(ok, pages(have + new) - pages(have), 0)
    off = torch.cumsum(need, 0) - need
    got = ok & ((need == 0) | (off + need <= n))
    col, first = torch.arange(M, device=dev), pages(have).unsqueeze(-1)
    mine = got.unsqueeze(-1) & (col >= first) & (col < first + need.unsqueeze(-1))
    src = n - 1 - off.unsqueeze(-1) - (col - first)
    table.copy_(torch.where(mine, free[1:][src.clamp(0, free.numel() - 2)], table))
    free[0] -= torch.where(got, need, 0).sum().int()
    starts = torch.cat((ends.new_zeros(1), ends)).clamp_max(N)
    i = torch.arange(N, device=dev)
    r = torch.searchsorted(starts[1:].contiguous(), i, right=True)
    held = got[r.clamp_max(R - 1)] & (r < R)
    r = r.clamp_max(R - 1)
    p = torch.where(held, have[r] + i - starts[r], 0)
    slots = torch.where(held, table[r, p // page].long() * page + p % page, -1)
    after = torch.where(got, have + new, 0)
    lens.copy_(torch.where(got, after, have))
    return [starts.int(), after.int(), slots, torch.where(held, p, -1).int()]


def _plain_trim(keep, lens, table, free, page):
    M = table.shape[1]
    pages = lambda x: (x + page - 1) // page
    have, n = lens.long(), free[0].long()
    keep = torch.minimum(keep.long().clamp_min(0), have)
    count = pages(have) - pages(keep)
    off = torch.cumsum(count, 0) - count
    col, first = torch.arange(M, device=lens.device), pages(keep).unsqueeze(-1)
    mine = (col >= first) & (col < first + count.unsqueeze(-1))
    total = count.sum()
    # one place behind the buffer for everything that stays
    to = torch.where(mine, n + total - off.unsqueeze(-1) - (col - first), free.numel())
    free.copy_(torch.cat((free, free[:1])).scatter(0, to.flatten(), table.flatten())[:-1])
    free[0] += total.int()
    table.masked_fill_(mine, -1)
    lens.copy_(keep)


def _plain_rope(x, w, freqs, pos, pairs):
    """Rows of x (N, H, D) normed, scaled by w and rotated by the angles pos (N,) times freqs; in 32 bits."""
    x = x.float()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
    ang = pos.double().unsqueeze(-1) * freqs
    cos, sin = torch.cos(ang).float().unsqueeze(1), torch.sin(ang).float().unsqueeze(1)
    r = 2 * freqs.numel()
    t, rest = y[..., :r], y[..., r:]
    if pairs:
        a, b = t[..., 0::2], t[..., 1::2]
        t = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = t[..., : r // 2], t[..., r // 2:]
        t = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((t, rest), -1)


def _plain_attend(c, s, rows, n, most):
    """Outputs of the n new tokens of each of `rows` (their numbers): (rows, n, Hq, D), in 32 bits; `most` keys at most."""
    dev, D, page = s["q"].device, c["D"], c["page"]
    rep, np = c["Hq"] // c["Hk"], _up(most, page)
    r = torch.tensor(rows, device=dev)
    end, first = s["ends"][r].long(), s["starts"][r].long()
    ids = s["table"][r, :np].long().clamp_min(0)
    keys = lambda x: x[ids].float().transpose(1, 2).flatten(2, 3).repeat_interleave(rep, dim=1)      # (rows, Hq, keys, D)
    t = torch.arange(n, device=dev)
    q = s["q"][first.unsqueeze(-1) + t].float().transpose(1, 2)
    i, j = (end.unsqueeze(-1) - n + t).unsqueeze(-1), torch.arange(np * page, device=dev)
    x = q @ keys(s["kp"]).transpose(-1, -2) * D ** -0.5
    if c["cap"]:
        x = c["cap"] * torch.tanh(x / c["cap"])
    if s["slopes"] is not None:
        x = x - s["slopes"].view(-1, 1, 1) * (i - j).abs().unsqueeze(1)
    ok = (i - j >= 0) & (i - j < (c["window"] or 1 << 40))
    if s["prefix"] is not None:
        ok = ok | (j < s["prefix"][r].view(-1, 1, 1))
    ok = (ok & (j < end.view(-1, 1, 1))).unsqueeze(1)
    x = x.masked_fill(~ok, -1e30)
    p = torch.exp(x - x.amax(-1, keepdim=True)) * ok
    return (p @ keys(s["vp"]) / p.sum(-1, keepdim=True).clamp_min(1e-30)).transpose(1, 2)


def _run_plain(s):
    c = s["case"]
    if c["op"] == "pages":
        outs = _plain_extend(s["new"], s["lens"], s["table"], s["free"], c["page"], s["N"])
        _plain_trim(s["before"], s["lens"], s["table"], s["free"], c["page"])
        return outs + [s["lens"], s["table"], s["free"]]
    dt = TYPES[c["dtype"]]
    if c["op"] == "rope_pages":
        q, k = (_plain_rope(s[x], s[w], s["freqs"], s["pos"], c["pairs"]).to(dt) for x, w in (("q", "wq"), ("k", "wk")))
        n = s["N"] - c["pad"]                                         # the last tokens belong to no row
        at, row = s["slots"][:n] // c["page"], s["slots"][:n] % c["page"]
        s["kp"][at, :, row] = k[:n]
        s["vp"][at, :, row] = s["v"][:n]
        return [q, s["kp"], s["vp"]]
    out = torch.zeros(s["q"].shape, device=s["q"].device, dtype=torch.float32)
    # rows of one token together, as many as their keys in 32 bits allow; the others one by one
    ones = [r for r, (_, n) in enumerate(s["rows"]) if n == 1]
    many = max(1, (1 << 29) // (max([sum(s["rows"][r]) for r in ones] + [1]) * c["Hq"] * c["D"]))
    groups = [ones[i: i + many] for i in range(0, len(ones), many)] + [[r] for r, (_, n) in enumerate(s["rows"]) if n > 1]
    at = 0
    begin = []
    for _, n in s["rows"]:
        begin.append(at)
        at += n
    for g in groups:
        n = s["rows"][g[0]][1]
        o = _plain_attend(c, s, g, n, max(sum(s["rows"][r]) for r in g))
        if len(g) == 1:
            out[begin[g[0]]: begin[g[0]] + n] = o[0]
        else:
            out[s["starts"][torch.tensor(g, device=out.device)].long()] = o[:, 0]
    return [out.to(dt)]


def _run_own(s):
    if _PKG not in sys.path:
        sys.path.insert(1, _PKG)
    c = s["case"]
    if c["op"] == "pages":
        import slotpage_hip as P
        step = P.page_extend(s["new"], s["lens"], s["table"], s["free"], c["page"], s["N"])
        P.page_trim(s["before"], s["lens"], s["table"], s["free"], c["page"])
        return [step.starts, step.ends, step.slots, step.pos, s["lens"], s["table"], s["free"]]
    if c["op"] == "rope_pages":
        import slotrope_hip as R
        q = R.qk_rope_pages(s["q"], s["k"], s["v"], s["wq"], s["wk"], s["freqs"], s["pos"], s["slots"], s["kp"], s["vp"], eps=EPS,
                            interleaved=c["pairs"])
        return [q, s["kp"], s["vp"]]
    import slotattn_hip as A
    return [A.attend_pages(s["q"], s["kp"], s["vp"], s["table"], s["starts"], s["ends"], most=s["most"], window=c["window"] or None,
                           cap=c["cap"] or None, slopes=s["slopes"], prefix=s["prefix"])]


def run(state):
    with torch.no_grad():
        return (_run_own if own else _run_plain)(state)


# ---- the work -----------------------------------------------------------------------------------------------


def _pairs(c):
    """Visible pairs of a query and a key of one head, and the keys that any query of a row sees, over the batch."""
    W = c["window"] or 1 << 40
    pre = _prefixes(c) if c["prefix"] else [0] * c["R"]
    pairs = keys = 0
    for (ctx, n), p in zip(_rows(c), pre):
        end = ctx + n
        if not n:
            continue
        for i in range(ctx, end):
            lo = max(0, i - W + 1)
            pairs += i + 1 - lo + min(p, lo) + max(0, min(p, end) - (i + 1))
        low = max(0, ctx - W + 1)
        keys += end - low + min(p, low)
    return pairs, keys


def work(case):
    """Each input read once, each output written once; the products of the visible pairs."""
    c = case
    rows = _rows(c)
    N = sum(n for _, n in rows) + c["pad"]
    if c["op"] == "pages":
        new = sum(_up(ctx + n, c["page"]) - _up(ctx, c["page"]) for ctx, n in rows)
        return dict(bytes=12 * N + 28 * c["R"] + 24 * new, flops=8 * N)
    e = 4 if c["dtype"] == "f32" else 2
    q, kv = N * c["Hq"] * c["D"] * e, N * c["Hk"] * c["D"] * e
    if c["op"] == "rope_pages":
        return dict(bytes=2 * q + 4 * kv + 2 * c["D"] * e + 12 * N, flops=(q + kv) // e * 8)
    pairs, keys = _pairs(c)
    return dict(bytes=2 * q + 2 * keys * c["Hk"] * c["D"] * e + 4 * _up(keys, c["page"]), flops=4 * c["Hq"] * c["D"] * pairs)


# ---- the definition, whole numbers by walking the rows and the rest in 64 bits --------------------------------


def _exact_pages(c, s):
    page, N = c["page"], s["N"]
    new, lens, table, free = (s[x].tolist() for x in ("new", "before", "table", "free"))
    left, starts, ends, slots, pos, out_of_pages = free[0], [0], [], [-1] * N, [-1] * N, False
    for r, n in enumerate(new):
        at = sum(new[:r])
        starts.append(min(at + n, N))
        have = lens[r]
        fits = n > 0 and at + n <= N and have + n <= len(table[r]) * page
        want = _up(have + n, page) - _up(have, page) if fits else 0
        out_of_pages = out_of_pages or want > left
        if not fits or (want and out_of_pages):
            ends.append(0)
            continue
        mine = [x for x in table[r] if x >= 0][: _up(have, page)]
        for _ in range(want):
            mine.append(free[left])
            left -= 1
        for t in range(n):
            pos[at + t] = have + t
            slots[at + t] = mine[(have + t) // page] * page + (have + t) % page
        ends.append(have + n)
    dev = s["new"].device
    # the pages come back in the order in which they went
    ints = lambda x, dt=torch.int32: torch.tensor(x, device=dev, dtype=dt)
    return [ints(starts), ints(ends), ints(slots, torch.int64), ints(pos), s["before"].clone(), s["table"].clone(), s["free"].clone()]


def _exact_rope(c, x, w, turn):
    x = x.double()
    y = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w.double()
    r = c["rot"]
    z = torch.complex(y[..., 0:r:2], y[..., 1:r:2]) if c["pairs"] else torch.complex(y[..., : r // 2], y[..., r // 2: r])
    z = z * turn
    t = torch.view_as_real(z).flatten(-2) if c["pairs"] else torch.cat((z.real, z.imag), -1)
    return torch.cat((t, y[..., r:]), -1)


def _exact_attend(c, s):
    dev, page, D, rep = s["q"].device, c["page"], c["D"], c["Hq"] // c["Hk"]
    out = torch.zeros(s["q"].shape, device=dev, dtype=torch.float64)
    W = c["window"] or 1 << 40
    pre = _prefixes(c) if c["prefix"] else [0] * c["R"]
    at = 0
    for r, (ctx, n) in enumerate(_rows(c)):
        if not n:
            continue
        end = ctx + n
        ids = s["table"][r, : _up(end, page)].long()
        away = torch.arange(ctx, end, device=dev).view(-1, 1) - torch.arange(end, device=dev).view(1, -1)
        sees = ((away >= 0) & (away < W)) | (torch.arange(end, device=dev) < pre[r])
        for h in range(c["Hk"]):
            k, v = (x[ids, h].reshape(-1, D)[:end].double() for x in (s["kp"], s["vp"]))
            for g in range(h * rep, (h + 1) * rep):
                sc = torch.matmul(s["q"][at: at + n, g].double(), k.t()) / math.sqrt(D)
                if c["cap"]:
                    sc = c["cap"] * torch.tanh(sc / c["cap"])
                if s["slopes"] is not None:
                    sc = sc - s["slopes"][g].double() * away.abs()
                sc = torch.where(sees, sc, float("-inf"))
                out[at: at + n, g] = torch.exp(sc - torch.logsumexp(sc, -1, keepdim=True)) @ v
        at += n
    return [out]


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "pages":
        return _exact_pages(c, s)
    with torch.no_grad():
        if c["op"] == "attend_pages":
            return _exact_attend(c, s)
        turn = torch.polar(torch.ones((), device=s["q"].device, dtype=torch.float64), s["pos"].double().unsqueeze(-1) * s["freqs"]).unsqueeze(1)
        q, k = (_exact_rope(c, s[x], s["w" + x], turn) for x in "qk")
        kp, vp = s["kp"].double(), s["vp"].double()
        at = 0
        for r, (ctx, n) in enumerate(s["rows"]):
            for p0 in range(ctx // c["page"] * c["page"], ctx + n, c["page"]):
                lo, hi = max(p0, ctx), min(p0 + c["page"], ctx + n)
                if hi <= lo:
                    continue
                i = int(s["table"][r, p0 // c["page"]])
                t = slice(at + lo - ctx, at + hi - ctx)
                kp[i, :, lo - p0: hi - p0] = k[t].transpose(0, 1)
                vp[i, :, lo - p0: hi - p0] = s["v"][t].double().transpose(0, 1)
            at += n
        return [q, kp, vp]
