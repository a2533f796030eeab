"""Attention over a cache in pages against the float64 oracle on each sequence by itself, within the oracle's bounds; everything in
the pool that no query sees is NaN."""
import pytest
import torch

from attn_cases import U, near
from oracle import attn_oracle as AO
from oracle import page_oracle as PO
from page_cases import pool, starts_of

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import slotattn_hip as A

BF, HF = torch.bfloat16, torch.float16


def queries(N, Hq, D, dt, seed, gain=1.4):
    return (gain * torch.randn(N, Hq, D, generator=torch.Generator().manual_seed(seed))).to(dt)


def reference(q, k, v, table, news, ends, u, **o):
    """(value, bound) of every row, packed; rows of 0 where nothing is seen."""
    out, bound, at = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64), 0
    prefix = o.pop("prefix", None)
    for r, (n, end) in enumerate(zip(news, ends)):
        if n:
            m = max(min(end, table.shape[1] * k.shape[2]), 1)
            kk, vv = (PO.dense(x, table[r], m) for x in (k, v))
            ref, b = AO.attention(q[at: at + n].transpose(0, 1).unsqueeze(0), kk, vv, lens=torch.tensor([end]),
                                  prefix=None if prefix is None else prefix[r: r + 1], u=u, **o)["out"]
            out[at: at + n], bound[at: at + n] = ref[0].transpose(0, 1), b[0].transpose(0, 1)
        at += n
    return out, bound


def run(news, ctxs, page, Hq, Hk, D, dt, seed, pad=0, by_token=False, most=None, ends=None, spare=1, **o):
    ends = [c + n for c, n in zip(ctxs, news)] if ends is None else ends
    M = max(PO.up(max(e, 1), page) for e in ends) + spare
    k, v, table = pool([max(e, 0) for e in ends], M, page, Hk, D, dt, seed, by_token=by_token)
    q = queries(sum(news) + pad, Hq, D, dt, seed + 1)
    if o.get("slopes"):
        o["slopes"] = 0.5 ** torch.arange(1, Hq + 1)
    if o.get("prefix"):
        o["prefix"] = torch.tensor([(7 * r) % (e + 1) for r, e in enumerate(ends)], dtype=torch.int32)
    og = {x: y.cuda() if torch.is_tensor(y) else y for x, y in o.items()}
    got = A.attend_pages(q.cuda(), k.cuda(), v.cuda(), table.cuda(), starts_of(news).cuda(), torch.tensor(ends, dtype=torch.int32).cuda(), most=most, **og)
    ref, bound = reference(q, k, v, table, news, ends, U[dt], **o)
    near(got, ref, bound, f"out {news} {ctxs}")
    assert got.shape == q.shape and got.is_contiguous() and got.dtype == dt
    return got


@pytest.mark.parametrize("Hq,Hk,D,dt", [(6, 2, 128, BF), (4, 4, 64, HF), (5, 1, 64, BF), (12, 4, 128, HF), (32, 2, 64, BF), (40, 1, 128, BF)])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("o", [{}, dict(cap=20.0, window=40), dict(slopes=True, prefix=True), dict(cap=5.0, slopes=True, window=1)])
def test_one_token_each(Hq, Hk, D, dt, page, o):
    ctxs = [0, 1, 14, 15, 16, 31, 33, 63, 64, 127, 300, 700]
    for most in (1, None):
        run([1] * 12, ctxs, page, Hq, Hk, D, dt, 1, most=most, **o)


@pytest.mark.parametrize("Hq,Hk,D,dt,page", [(6, 2, 128, BF, 16), (4, 4, 64, HF, 32), (3, 1, 128, HF, 256), (8, 2, 64, BF, 64)])
@pytest.mark.parametrize("o", [{}, dict(cap=20.0, window=70), dict(slopes=True), dict(prefix=True, window=33), dict(cap=50.0, prefix=True, slopes=True)])
def test_prompts_and_tokens_mixed(Hq, Hk, D, dt, page, o):
    run([1, 0, 130, 1, 5, 43, 0, 1], [200, 30, 0, 77, 60, 301, 0, 0], page, Hq, Hk, D, dt, 2, pad=9, by_token=page == 32, **o)


@pytest.mark.parametrize("n,ctx", [(1, 3000), (2, 2999), (9, 5000), (500, 0), (257, 1400), (1000, 37)])
@pytest.mark.parametrize("D,dt", [(128, BF), (64, HF)])
def test_one_sequence(n, ctx, D, dt):
    """Few rows and many keys, many rows and few keys: shared out over many workgroups and joined."""
    for most in (n, None):
        run([n], [ctx], 16, 6, 2, D, dt, 3, most=most)


def test_rows_without_room_or_keys():
    """A row that was given no room (ends 0), and one with fewer tokens than queries: 0 for queries of negative position."""
    got = run([3, 4, 2, 6], [0] * 4, 16, 4, 2, 64, BF, 4, pad=5, ends=[0, 9, 0, 2])
    assert not bool(got[:3].any()) and not bool(got[7:9].any()) and not bool(got[9:13].any()) and not bool(got[15:].any())
    assert bool(got[13:15].any())


def test_a_table_that_is_full_and_lengths_past_it():
    run([1, 7], [63, 57], 16, 2, 2, 64, BF, 5, spare=0)
    k, v, table = pool([64, 64], 4, 16, 2, 64, BF, 6)
    q = queries(4, 4, 64, BF, 7)
    ends = [70, 2 ** 31 - 1]                             # the second's positions are far from all keys, which it sees nevertheless
    got = A.attend_pages(q.cuda(), k.cuda(), v.cuda(), table.cuda(), starts_of([2, 2]).cuda(), torch.tensor(ends, dtype=torch.int32).cuda())
    ref, bound = reference(q, k, v, table, [2, 2], [70, (1 << 30) - 1], U[BF])
    near(got, ref, bound, "out")


def test_pages_that_are_not_there_are_not_seen():
    """A page number outside of the pool: its keys do not count, for tokens, chunks and rows that have no other page."""
    for bad in (-1, 10 ** 6, 2 ** 31 - 1, -2 ** 31):
        for news, most in (([1, 1, 1], 1), ([1, 40, 90], None)):
            ends = [130, 100, 100]
            k, v, table = pool(ends, 9, 16, 2, 64, HF, 8)
            table[0, 2] = bad
            table[1, 0] = table[1, 5] = bad
            table[2, :] = bad
            q = queries(sum(news), 4, 64, HF, 9)
            got = A.attend_pages(q.cuda(), k.cuda(), v.cuda(), table.cuda(), starts_of(news).cuda(), torch.tensor(ends, dtype=torch.int32).cuda(), most=most)
            at = 0
            for r, n in enumerate(news):
                kk, vv = (PO.dense(x, table[r], ends[r]) for x in (k, v))
                there = torch.tensor([0 <= int(table[r, j // 16]) < k.shape[0] for j in range(ends[r])])
                ref, bound = _masked(q[at: at + n], kk, vv, there, U[HF])
                near(got[at: at + n], ref, bound, f"row {r}")
                at += n
            assert not bool(got[sum(news[:2]):].any())


def _masked(q, k, v, there, u):
    """Causal attention of the newest tokens over those keys that are there."""
    n, Hq, D = q.shape
    end, rep = k.shape[2], Hq // k.shape[1]
    ref, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for i in range(n):
        keep = there & (torch.arange(end) <= end - n + i)
        m = int(keep.sum())
        if m:
            a, b = AO.attention(q[i: i + 1].transpose(0, 1).unsqueeze(0), k[:, :, keep], v[:, :, keep], lens=torch.tensor([m]), u=u)["out"]
            ref[i: i + 1], bound[i: i + 1] = a[0].transpose(0, 1), b[0].transpose(0, 1)
    return ref, bound


@pytest.mark.parametrize("news,ctxs", [([1, 1, 2], [500, 90, 300]), ([1, 200, 50], [700, 100, 333])])
@pytest.mark.parametrize("prefix", [2 ** 31 - 1, 2 ** 31 - 20, 400, -5])
def test_prefixes_of_any_number(news, ctxs, prefix):
    """A prefix past all keys beside a window: every key is seen; a negative one is none."""
    ends = [c + n for c, n in zip(ctxs, news)]
    k, v, table = pool(ends, 60, 16, 2, 64, BF, 12)
    q = queries(sum(news), 4, 64, BF, 13)
    pre = torch.full((3,), prefix, dtype=torch.int32)
    ref, bound = reference(q, k, v, table, news, ends, U[BF], window=37, prefix=pre.long())
    for most in (max(news), None):
        got = A.attend_pages(q.cuda(), k.cuda(), v.cuda(), table.cuda(), starts_of(news).cuda(), torch.tensor(ends, dtype=torch.int32).cuda(), most=most,
                             window=37, prefix=pre.cuda())
        near(got, ref, bound, f"out {prefix}")


@pytest.mark.parametrize("Hq,Hk,dt,page", [(6, 2, BF, 16), (4, 4, HF, 64), (12, 1, BF, 32)])
@pytest.mark.parametrize("o", [{}, dict(cap=20.0, window=70), dict(slopes=True, prefix=True), dict(prefix=True, window=33)])
def test_units_of_about_one_length(Hq, Hk, dt, page, o):
    """Units that run whole, a workgroup each; rows without tokens and without earlier keys between them."""
    news = [(37 * r) % 41 + 5 for r in range(60)]
    ctxs = [(53 * r) % 200 for r in range(60)]
    news[3] = news[30] = news[59] = 0
    run(news, ctxs, page, Hq, Hk, 128, dt, 14, pad=3, by_token=page == 32, **o)
    run([128] * 7, [0] * 7, page, Hq, Hk, 128, dt, 15, **o)


def test_replays_follow_the_lengths_from_alike_rows_to_unlike_ones():
    """One captured call whose rows are alike, unlike and alike again: what is whole and what is shared out is decided on the GPU."""
    sets = [([40] * 30, [100] * 30), ([1] * 29 + [1171], [900] + [3] * 28 + [500]), ([40] * 30, [0] * 30)]
    ends = [[c + n for c, n in zip(ctxs, news)] for news, ctxs in sets]
    most = [max(e[r] for e in ends) for r in range(30)]
    k, v, table = pool(most, max(PO.up(e, 16) for e in most), 16, 2, 128, BF, 16)
    q = queries(1200, 6, 128, BF, 17)
    kc, vc, tc, qc = k.cuda(), v.cuda(), table.cuda(), q.cuda()
    starts, end = starts_of(sets[0][0]).cuda(), torch.tensor(ends[0], dtype=torch.int32).cuda()
    call = lambda: A.attend_pages(qc, kc, vc, tc, starts, end)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for (news, _), e in zip(sets, ends):
        starts.copy_(starts_of(news))
        end.copy_(torch.tensor(e, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        ref, bound = reference(q, k, v, table, news, e, U[BF])
        near(out, ref, bound, f"replay {news[-1]}")
        assert torch.equal(out, call())
