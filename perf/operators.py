"""The exact attention beside the slot memory, as cases for measuring its operators' time and outputs.

A case is a dict of plain values; `op` names the entry point:
    rope          qk_rope: the norm of every query and key head with the position rotation in the same pass
    rope_cache    qk_rope_cache: the same for a sequence's newest tokens, keys and values written into a cache
    attend        attend: attention whose scores may be capped by a tanh, may get a bias that falls with the distance,
                  and are masked by causality, a window, documents and a prefix
    attend_cache  attend_cache: the newest tokens' queries against a cache of ragged lengths

`train` runs the forward and the backward against given upstream gradients, otherwise the forward alone without autograd.
Where `own` is false, run() computes the operators with elementary torch operations in 32 bits (the angles of the rotation
in 64), rounded once at the end.  Tensors are token-major, (B, T, heads, D) seen as (B, heads, T, D), as a layer's
projection leaves them; queries and keys of `rope` are slices of one projection's output.
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
    at = dict(op="attend", causal=True, window=0, cap=0.0, slopes=False, docs=0, prefix=0)
    ca = dict(op="attend_cache", window=0, cap=0.0, slopes=False)
    return [
        # a training step's queries and keys, a quarter of one GPU's batch: the memory's bandwidth
        dict(name="rope_train", op="rope", B=8, T=2048, Hq=12, Hk=4, D=128, rot=128, pairs=False, dtype="bf16", train=True),
        # a small model in 32 bits, half of each head rotated, neighbouring pairs, an odd length
        dict(name="rope_odd", op="rope", B=3, T=333, Hq=6, Hk=2, D=64, rot=32, pairs=True, dtype="f32", train=True),
        # one generated token of 32 sequences: latency
        dict(name="write_step", op="rope_cache", B=32, T=1, Hq=12, Hk=4, D=128, rot=128, pairs=False, S=2048, dtype="bf16",
             train=False),
        # two prompts of different lengths, padded on the left
        dict(name="write_prompt", op="rope_cache", B=2, T=1000, Hq=6, Hk=6, D=64, rot=64, pairs=False, S=1024, dtype="f16",
             train=False),
        # the smallest training shape of the tests: latency
        dict(at, name="attend_small", B=2, T=128, Hq=6, Hk=6, D=64, dtype="bf16", train=True),
        # one long document with capped scores: the largest
        dict(at, name="attend_long", B=1, T=8192, Hq=12, Hk=4, D=128, cap=50.0, dtype="bf16", train=True),
        # packed documents under a sliding window, the last tokens of each row padding
        dict(at, name="attend_packed", B=4, T=2048, Hq=12, Hk=4, D=128, window=512, docs=7, dtype="bf16", train=True),
        # a bias that falls with the distance, an odd length, half precision
        dict(at, name="attend_slopes", B=3, T=1111, Hq=6, Hk=6, D=64, slopes=True, dtype="f16", train=True),
        # prompts read both ways before their continuation: evaluation, so the forward alone
        dict(at, name="attend_prefix", B=4, T=2000, Hq=12, Hk=4, D=128, cap=30.0, prefix=5, dtype="bf16", train=False),
        # one generated token of 32 sequences of up to 8,192: the caches' bytes
        dict(ca, name="cache_step", B=32, T=1, Hq=12, Hk=4, D=128, S=8192, cap=50.0, lens=3, dtype="bf16", train=False),
        # one generated token of one very long sequence: the work has to be split over its length
        dict(ca, name="cache_long", B=1, T=1, Hq=12, Hk=4, D=128, S=131072, lens=0, dtype="bf16", train=False),
        # a chunk of four prompts being read, under a sliding window
        dict(ca, name="cache_chunk", B=4, T=256, Hq=12, Hk=4, D=128, S=4096, window=1024, lens=2, dtype="f16", train=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "rope_cache", "attend", "attend", "attend", "attend_cache", "attend_cache"])
    Hk = rng.choice([1, 2, 4, 4, 6, 8])
    c = dict(op=op, Hk=Hk, Hq=Hk * rng.choice([1, 1, 2, 3, 4]), D=rng.choice([64, 128, 128]),
             dtype=rng.choice(["bf16", "bf16", "f16"]))
    if op in ("rope", "rope_cache"):
        c.update(rot=rng.choice([16, 32, 64, c["D"], c["D"]]), pairs=rng.random() < 0.4, train=False)
        if op == "rope":
            c["dtype"] = rng.choice(["bf16", "bf16", "f16", "f32"])
            c["T"] = _log(rng, 1, 8192)
            c["B"] = _log(rng, 1, max(1, min(64, 200000 // (c["T"] * c["Hq"]))))
            c["train"] = rng.random() < 0.7
        else:
            c["T"] = rng.choice([1, 1, 2, 5, _log(rng, 1, 2048)])
            c["S"] = c["T"] + _log(rng, 1, 4096)
            c["B"] = _log(rng, 1, max(1, min(64, 20000 // c["T"], 200000 // c["S"])))
        return c
    c.update(cap=rng.choice([0.0, 0.0, 30.0, 50.0]), slopes=rng.random() < 0.25)
    if op == "attend":
        c.update(causal=rng.random() < 0.85, train=rng.random() < 0.6, docs=rng.choice([0, 0, 1 + rng.randrange(1000)]),
                 prefix=rng.choice([0, 0, 0, 1 + rng.randrange(1000)]))
        # (one visible key has no gradient of its score: training rows have several)
        c["T"] = _log(rng, 24 if c["train"] else 1, 4096)
        c["B"] = _log(rng, 1, max(1, min(32, 12 * 8192 * 8192 // 4 // (c["T"] * max(c["T"], 256) * c["Hq"]))))
    else:
        c.update(train=False, lens=1 + rng.randrange(1000))
        c["T"] = rng.choice([1, 1, 1, 2, 4, _log(rng, 1, 512)])
        c["S"] = max(c["T"], _log(rng, 16, 65536))
        c["B"] = _log(rng, 1, max(1, min(64, 262144 // c["S"], 4000000 // (c["T"] * c["S"]))))
    c["window"] = rng.choice([0, 0, _log(rng, 8, 2048)])
    return c


# ---- inputs -------------------------------------------------------------------------------------------------


def _documents(c):
    """Lengths of the documents of every row and of its padding, by the case alone: ragged, of about a quarter row."""
    rng = random.Random(c["docs"])
    rows = []
    for _ in range(c["B"]):
        left, row = c["T"] - c["T"] // 32, []
        while left > 0:
            row.append(min(left, _log(rng, max(1, c["T"] // 16), max(1, c["T"] // 2))))
            left -= row[-1]
        rows.append((row, c["T"] // 32))
    return rows


def _prefixes(c):
    rng = random.Random(c["prefix"])
    return [rng.randrange(0, max(1, c["T"] // 2)) for _ in range(c["B"])]


def _lengths(c):
    """Tokens of every sequence, the newest ones included, by the case alone."""
    if c["op"] == "rope_cache":
        rng = random.Random(c["S"])
        return [rng.randint(max(1, c["T"] // 2), c["S"]) if c["T"] > 16 else rng.randint(c["T"], c["S"]) for _ in range(c["B"])]
    rng = random.Random(c["lens"])
    return [c["S"] if not c["lens"] else rng.randint(max(c["T"], c["S"] // 8), c["S"]) for _ in range(c["B"])]


def prepare(case, seed):
    c = case
    dev = torch.device("cuda:0")
    gen = torch.Generator(device=dev).manual_seed(int(seed) * 7919 + 13)
    dt = TYPES[c["dtype"]]
    rn = lambda *s: torch.randn(*s, device=dev, generator=gen)
    B, T, Hq, Hk, D, op = (c[x] for x in ("B", "T", "Hq", "Hk", "D", "op"))
    s = dict(case=c)
    heads = lambda x: x.transpose(1, 2)
    ints = lambda x: torch.tensor(x, device=dev, dtype=torch.int32)
    if op in ("rope", "rope_cache"):
        qkv = rn(B, T, Hq + 2 * Hk, D).to(dt)
        s["q"], s["k"], s["v"] = (heads(x) for x in qkv.split([Hq, Hk, Hk], dim=2))
        s["wq"], s["wk"] = ((1.0 + 0.2 * rn(D)).to(dt) for _ in range(2))
        s["freqs"] = THETA ** (-2.0 * torch.arange(c["rot"] // 2, device=dev, dtype=torch.float64) / c["rot"])
        if op == "rope":
            s["leaves"] = [s[x] for x in ("q", "k", "wq", "wk")]
            if c["train"]:
                s["up"] = [heads(rn(B, T, h, D).to(dt)) for h in (Hq, Hk)]
                for x in s["leaves"]:
                    x.requires_grad_()
        else:
            s["kc"], s["vc"] = (heads(rn(B, c["S"], Hk, D).to(dt)) for _ in range(2))
            s["lens"] = ints(_lengths(c))
        return s
    s["q"] = heads((GAIN * rn(B, T, Hq, D)).to(dt))
    # slopes as a geometric series over the heads
    s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, Hq + 1, device=dev, dtype=torch.float32) / Hq) if c["slopes"] else None
    n = T if op == "attend" else c["S"]
    s["k"], s["v"] = heads((GAIN * rn(B, n, Hk, D)).to(dt)), heads(rn(B, n, Hk, D).to(dt))
    if op == "attend_cache":
        s["lens"] = ints(_lengths(c))
        return s
    s["docs"] = s["prefix"] = None
    if c["docs"]:
        s["docs"] = ints([sum(([i] * n for i, n in enumerate(row)), []) + [-1] * pad for row, pad in _documents(c)])
    if c["prefix"]:
        s["prefix"] = ints(_prefixes(c))
    if c["train"]:
        s["up"] = [heads(rn(B, T, Hq, D).to(dt))]
        s["leaves"] = [s[x] for x in ("q", "k", "v")]
        for x in s["leaves"]:
            x.requires_grad_()
    return s


# ---- the plain forms, in 32 bits ----------------------------------------------------------------------------


def _plain_rope(x, w, freqs, pos, pairs):
    """Rows of x (B, H, T, D) normed, scaled by w and rotated by the angles pos (B or 1, T) times freqs; in 32 bits."""
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


def _visible(c, pos, Tk, docs, prefix, lens):
    """Which of the Tk keys each query sees, (B or 1, 1, Tq, Tk); pos (B or 1, Tq): the queries' positions."""
    i, j = pos.unsqueeze(-1), torch.arange(Tk, device=pos.device)
    far = i - j if c.get("causal", True) else (i - j).abs()
    ok = (far >= 0) & (far < (c["window"] or Tk + 1))
    if prefix is not None:
        ok = ok | (j < prefix.view(-1, 1, 1))
    if docs is not None:
        ok = ok & (docs.unsqueeze(-1) == docs.unsqueeze(-2)) & (docs >= 0).unsqueeze(-1)
    if lens is not None:
        ok = ok & (j < lens.view(-1, 1, 1)) & (i >= 0)
    return ok.unsqueeze(1)


def _plain_attend(c, q, k, v, slopes, docs, prefix, lens):
    B, Hq, Tq, D = q.shape
    Tk, rep = k.shape[2], Hq // k.shape[1]
    t = torch.arange(Tq, device=q.device).unsqueeze(0)
    pos = t if lens is None else lens.unsqueeze(-1) - Tq + t
    q, k, v = q.float(), k.float().repeat_interleave(rep, dim=1), v.float().repeat_interleave(rep, dim=1)
    s = q @ k.transpose(-1, -2) * D ** -0.5
    if c["cap"]:
        s = c["cap"] * torch.tanh(s / c["cap"])
    if slopes is not None:
        s = s - slopes.view(-1, 1, 1) * (pos.unsqueeze(-1) - torch.arange(Tk, device=q.device)).abs().unsqueeze(1)
    ok = _visible(c, pos, Tk, docs, prefix, lens)
    s = s.masked_fill(~ok, -1e30)
    p = torch.exp(s - s.amax(-1, keepdim=True).detach()) * ok
    return p @ v / p.sum(-1, keepdim=True).clamp_min(1e-30)


def _pos(c, lens, dev):
    t = torch.arange(c["T"], device=dev).unsqueeze(0)
    return t if lens is None else lens.unsqueeze(-1) - c["T"] + t


def _run_plain(s):
    c = s["case"]
    op, dt = c["op"], TYPES[c["dtype"]]
    if op == "rope":
        pos = _pos(c, None, s["q"].device)
        return [_plain_rope(s[x], s[w], s["freqs"], pos, c["pairs"]).to(dt) for x, w in (("q", "wq"), ("k", "wk"))]
    if op == "rope_cache":
        pos = _pos(c, s["lens"], s["q"].device)
        q, k = (_plain_rope(s[x], s[w], s["freqs"], pos, c["pairs"]).to(dt) for x, w in (("q", "wq"), ("k", "wk")))
        # a padding token repeats the newest one's write
        b = torch.arange(c["B"], device=pos.device).unsqueeze(-1)
        t = torch.where(pos >= 0, torch.arange(c["T"], device=pos.device), c["T"] - 1)
        s["kc"][b, :, pos.gather(1, t)] = k[b, :, t]
        s["vc"][b, :, pos.gather(1, t)] = s["v"][b, :, t]
        return [q, s["kc"], s["vc"]]
    return [_plain_attend(c, s["q"], s["k"], s["v"], s["slopes"], s.get("docs"), s.get("prefix"), s.get("lens")).to(dt)]


def _run_own(s):
    if _PKG not in sys.path:
        sys.path.insert(1, _PKG)
    import slotattn_hip as A
    import slotrope_hip as R
    c = s["case"]
    op = c["op"]
    if op == "rope":
        return list(R.qk_rope(s["q"], s["k"], s["wq"], s["wk"], s["freqs"], eps=EPS, interleaved=c["pairs"]))
    if op == "rope_cache":
        q = R.qk_rope_cache(s["q"], s["k"], s["v"], s["wq"], s["wk"], s["freqs"], s["lens"], s["kc"], s["vc"], eps=EPS,
                            interleaved=c["pairs"])
        return [q, s["kc"], s["vc"]]
    kw = dict(window=c["window"] or None, cap=c["cap"] or None, slopes=s["slopes"])
    if op == "attend":
        return [A.attend(s["q"], s["k"], s["v"], causal=c["causal"], docs=s["docs"], prefix=s["prefix"], **kw)]
    return [A.attend_cache(s["q"], s["k"], s["v"], s["lens"], **kw)]


def run(state):
    s = state
    call = _run_own if own else _run_plain
    if not s["case"]["train"]:
        with torch.no_grad():
            return call(s)
    outs = call(s)
    return [o.detach() for o in outs] + list(torch.autograd.grad(outs, s["leaves"], s["up"]))


# ---- the work -----------------------------------------------------------------------------------------------


def _pairs(c):
    """Visible pairs of a query and a key of one head, over the batch."""
    T = c["T"]
    W = c["window"] or 1 << 40

    def causal(at, n, low):                 # queries at `at` .. `at + n - 1`, keys from `low` up to each of them
        return sum(min(i + 1 - low, W) for i in range(max(at, low), at + n))

    if c["op"] == "attend_cache":
        return sum(causal(n - T, T, 0) for n in _lengths(c))
    rows = _documents(c) if c["docs"] else [([T], 0)] * c["B"]
    pre = _prefixes(c) if c["prefix"] else [0] * c["B"]
    total = 0
    for (row, _), p in zip(rows, pre):
        low = 0
        for n in row:
            # one query's keys: those of its window, and those of the prefix that are in its document
            lo = lambda i: max(low, i - W + 1)
            hi = lambda i: i + 1 if c["causal"] else min(low + n, i + W)
            end = min(p, low + n)
            total += sum(hi(i) - lo(i) + max(0, min(end, lo(i)) - low) + max(0, end - max(hi(i), low)) for i in range(low, low + n))
            low += n
    return total


def work(case):
    """Each input read once, each output written once; the products of the visible pairs."""
    c = case
    B, T, Hq, Hk, D = (c[x] for x in ("B", "T", "Hq", "Hk", "D"))
    e = 4 if c["dtype"] == "f32" else 2
    both = 2 if c["train"] else 1
    q, kv = B * T * Hq * D * e, B * T * Hk * D * e
    if c["op"] == "rope":
        # the backward reads the inputs again beside the upstream gradients
        return dict(bytes=(2 + (3 if c["train"] else 0)) * (q + kv) + both * 4 * D * e, flops=(q + kv) // e * (8 if not c["train"] else 24))
    if c["op"] == "rope_cache":
        return dict(bytes=2 * q + 4 * kv + 2 * D * e, flops=(q + kv) // e * 8)
    pairs = _pairs(c)
    if c["op"] == "attend_cache":
        W = c["window"] or 1 << 40
        rows = sum(min(n, W + T - 1) for n in _lengths(c))
        return dict(bytes=2 * q + 2 * rows * Hk * D * e, flops=4 * Hq * D * pairs)
    return dict(bytes=both * (2 * q + 2 * kv), flops=(14 if c["train"] else 4) * Hq * D * pairs)


# ---- the definition in 64 bits ------------------------------------------------------------------------------


def _turn(c, freqs, pos):
    return torch.polar(torch.ones((), device=freqs.device, dtype=torch.float64), pos.double().unsqueeze(-1) * freqs)


def _as_complex(c, x):
    r = c["rot"]
    return torch.complex(x[..., 0:r:2], x[..., 1:r:2]) if c["pairs"] else torch.complex(x[..., : r // 2], x[..., r // 2: r])


def _from_complex(c, z, rest):
    t = torch.view_as_real(z).flatten(-2) if c["pairs"] else torch.cat((z.real, z.imag), -1)
    return torch.cat((t, rest), -1)


def _exact_rope(c, x, w, turn):
    x, w = x.detach().double(), w.detach().double()
    y = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w
    return _from_complex(c, _as_complex(c, y) * turn, y[..., c["rot"]:])


def _exact_rope_grad(c, x, w, turn, up):
    x, w, up = x.detach().double(), w.detach().double(), up.double()
    g = _from_complex(c, _as_complex(c, up) * turn.conj(), up[..., c["rot"]:])       # back through the rotation
    rms = (x.square().mean(-1, keepdim=True) + EPS).sqrt()
    u = x / rms
    return (g * w - u * (g * w * u).mean(-1, keepdim=True)) / rms, (g * u).sum((0, 1, 2))


def _exact_sees(c, s, b, dev):
    """Visibility of one sequence, (Tq, Tk), and the distances."""
    cache = c["op"] == "attend_cache"
    n = _lengths(c)[b] if cache else c["T"]
    i = torch.arange(n - c["T"], n, device=dev).view(-1, 1)
    j = torch.arange(c["S"] if cache else c["T"], device=dev).view(1, -1)
    away = i - j
    W = c["window"] or 1 << 40
    ok = ((away >= 0) & (away < W)) if c.get("causal", True) else (away.abs() < W)
    if c.get("prefix"):
        ok |= j < _prefixes(c)[b]
    if c.get("docs"):
        row, pad = _documents(c)[b]
        doc = torch.repeat_interleave(torch.arange(len(row) + 1, device=dev), torch.tensor(row + [pad], device=dev))
        ok &= (doc.view(-1, 1) == doc.view(1, -1)) & (doc < len(row)).view(1, -1)
    return ok & (j < n), away.abs().double()


def _exact_attend(c, s):
    B, T, Hq, Hk, D = (c[x] for x in ("B", "T", "Hq", "Hk", "D"))
    dev, rep, train = s["q"].device, Hq // Hk, c["train"]
    z = lambda x: torch.zeros(x.shape, device=dev, dtype=torch.float64)
    out = z(s["q"])
    dq, dk, dv = (z(s[x]) for x in "qkv") if train else (None,) * 3
    with torch.no_grad():
        for b in range(B):
            ok, away = _exact_sees(c, s, b, dev)
            n = _lengths(c)[b] if c["op"] == "attend_cache" else T
            ok, away = ok[:, :n], away[:, :n]
            for h in range(Hq):
                q, k, v = s["q"][b, h].double(), s["k"][b, h // rep, :n].double(), s["v"][b, h // rep, :n].double()
                sc = torch.matmul(q, k.t()) / math.sqrt(D)
                th = torch.tanh(sc / c["cap"]) if c["cap"] else None
                if c["cap"]:
                    sc = c["cap"] * th
                if s["slopes"] is not None:
                    sc = sc - s["slopes"][h].double() * away
                sc = torch.where(ok, sc, float("-inf"))
                p = torch.where(ok, torch.exp(sc - torch.logsumexp(sc, -1, keepdim=True)), 0.0)
                o = out[b, h] = p @ v
                if train:
                    up = s["up"][0][b, h].double()
                    dv[b, h // rep] += p.t() @ up
                    ds = p * (up @ v.t() - (up * o).sum(-1, keepdim=True)) / math.sqrt(D)
                    if c["cap"]:
                        ds = ds * (1.0 - th * th)
                    dq[b, h] = ds @ k
                    dk[b, h // rep] += ds.t() @ q
                del sc, p
    return [out, dq, dk, dv] if train else [out]


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] in ("attend", "attend_cache"):
        return _exact_attend(c, s)
    with torch.no_grad():
        turn = _turn(c, s["freqs"], _pos(c, s.get("lens"), s["q"].device)).unsqueeze(1)
        outs = [_exact_rope(c, s[x], s["w" + x], turn) for x in "qk"]
        if c["op"] == "rope":
            if c["train"]:
                (dq, dwq), (dk, dwk) = (_exact_rope_grad(c, s[x], s["w" + x], turn, u) for x, u in zip("qk", s["up"]))
                outs += [dq, dk, dwq, dwk]
            return outs
        kc, vc = s["kc"].double(), s["vc"].double()
        for b, n in enumerate(_lengths(c)):
            m = min(n, c["T"])
            kc[b, :, n - m: n], vc[b, :, n - m: n] = outs[1][b, :, c["T"] - m:], s["v"][b, :, c["T"] - m:].double()
        return [outs[0], kc, vc]
