"""Attention over a cache in pages where batches outgrow the sizes of the other tests: more rows than a wave has lanes, than a workgroup has threads
and than the join has workgroups, negative scales, scores past 2^22, caps far above the scores."""
import pytest
import torch

from attn_cases import U, near
from oracle import page_oracle as PO
from page_cases import pool, starts_of
from test_gpu_attn_pages import BF, HF, queries, reference, run

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import slotattn_hip as A

ints = lambda x: torch.tensor(x, dtype=torch.int32).cuda()


def ragged(R, longest, seed, empty=7):
    """Numbers of tokens (0 or 1) and lengths of R rows, one row far longer than the others."""
    g = torch.Generator().manual_seed(seed)
    news = [int(r % empty != 2) for r in range(R)]
    ctxs = torch.randint(0, 60, (R,), generator=g).tolist()
    ctxs[R // 3], news[R // 3] = longest, 1
    return news, ctxs


@pytest.mark.parametrize("R,longest,Hq,Hk,D,dt", [(65, 1500, 4, 2, 64, BF), (200, 300, 6, 2, 128, HF), (1100, 900, 4, 2, 64, HF), (1100, 40, 3, 1, 128, BF)])
@pytest.mark.parametrize("o", [{}, dict(window=30), dict(prefix=True, slopes=True)])
def test_many_rows_of_one_token(R, longest, Hq, Hk, D, dt, o):
    """Few rows each, and more of them than lanes (65, 200), than threads of the plan's workgroup and than two for each workgroup of the join (1,100); both
    as a token each and as a batch of any lengths."""
    news, ctxs = ragged(R, longest, R)
    for most in (1, None):
        print("rows", R, most, o, flush=True)
        run(news, ctxs, 16, Hq, Hk, D, dt, 21, pad=3, most=most, **o)


@pytest.mark.parametrize("first", [0, 4000])
def test_more_rows_than_64_a_lane(first):
    """4,200 rows, nearly all of them without tokens."""
    news, ctxs = [0] * 4200, [0] * 4200
    for r in [*range(first, first + 150), 4199]:
        news[r], ctxs[r] = 1, (31 * r) % 90
    news[77], ctxs[77] = 1, 1200
    for most in (1, None):
        run(news, ctxs, 16, 4, 2, 64, BF, 22, most=most)


@pytest.mark.parametrize("R,n", [(1100, 1), (350, 130)])
@pytest.mark.parametrize("o", [{}, dict(cap=30.0, window=33)])
def test_more_whole_units_than_threads(R, n, o):
    """Alike rows whose units run whole, more of them than the plan's workgroup has threads: with a token each, and in several tiles of rows."""
    run([n] * R, [(3 * r) % 20 + 40 for r in range(R)], 16, 2 if n > 1 else 4, 1, 128, BF, 23, **o)


@pytest.mark.parametrize("Hq,Hk,D,dt", [(6, 2, 128, BF), (4, 1, 64, HF)])
@pytest.mark.parametrize("news,ctxs", [([1, 3, 2], [700, 90, 2100]), ([1], [5000]), ([1, 200, 37], [400, 90, 0])])
@pytest.mark.parametrize("o", [dict(scale=-0.1), dict(scale=-0.1, slopes=True, window=150), dict(scale=-0.2, cap=20.0)])
def test_negative_scales(Hq, Hk, D, dt, news, ctxs, o):
    """The smallest products have the largest weights."""
    for most in (max(news), None):
        k, v, table = pool([c + n for c, n in zip(ctxs, news)], 330, 16, Hk, D, dt, 24)
        q = queries(sum(news), Hq, D, dt, 25)
        opt, ends = dict(o), [c + n for c, n in zip(ctxs, news)]
        if opt.get("slopes"):
            opt["slopes"] = 0.5 ** torch.arange(1, Hq + 1)
        og = {a: b.cuda() if torch.is_tensor(b) else b for a, b in opt.items()}
        got = A.attend_pages(q.cuda(), k.cuda(), v.cuda(), table.cuda(), starts_of(news).cuda(), ints(ends), most=most, **og)
        ref, bound = reference(q, k, v, table, news, ends, U[dt], strict=True, **opt)
        near(got, ref, bound, "out")


@pytest.mark.parametrize("Hq,Hk,D,dt", [(6, 2, 128, BF), (4, 1, 64, HF)])
@pytest.mark.parametrize("scale", [3.0, 12.0])
def test_caps_far_above_some_scores(Hq, Hk, D, dt, scale):
    """A cap of 100: scores of 2 % of it and of several times it in one tile."""
    for news, ctxs, most in (([1, 2], [900, 40], 2), ([1, 90], [300, 60], None)):
        ends = [c + n for c, n in zip(ctxs, news)]
        k, v, table = pool(ends, 64, 16, Hk, D, dt, 26)
        q = queries(sum(news), Hq, D, dt, 27)
        got = A.attend_pages(q.cuda(), k.cuda(), v.cuda(), table.cuda(), starts_of(news).cuda(), ints(ends), most=most, scale=scale, cap=100.0)
        ref, bound = reference(q, k, v, table, news, ends, U[dt], scale=scale, cap=100.0, strict=True)
        near(got, ref, bound, "out")


@pytest.mark.parametrize("Hq,Hk,D,dt", [(6, 2, 128, BF), (4, 1, 64, HF)])
@pytest.mark.parametrize("scale", [1e4, 1e7, -3e8, 1e27])
@pytest.mark.parametrize("o", [{}, dict(window=60), dict(cap=1e30)])
def test_scores_of_any_size(Hq, Hk, D, dt, scale, o):
    """Queries and keys of small whole numbers: their products are exact and the largest share the weight, so the bounds are the probabilities' rounding
    (in one part at most) and the result's alone."""
    if "cap" in o and scale < 0:
        scale = -scale
    for news, ctxs, most in (([1, 3], [1400, 40], 3), ([1], [4000], 1), ([1, 150, 40], [300, 60, 0], None)):
        ends = [c + n for c, n in zip(ctxs, news)]
        k, v, table = pool(ends, 260, 16, Hk, D, dt, 28)
        g = torch.Generator().manual_seed(29)
        k = torch.randint(-2, 3, k.shape, generator=g).to(dt)
        q = torch.randint(-2, 3, (sum(news), Hq, D), generator=g).to(dt)
        got = A.attend_pages(q.cuda(), k.cuda(), v.cuda(), table.cuda(), starts_of(news).cuda(), ints(ends), most=most, scale=scale, **o)
        want, size = (reference(q, k, y, table, news, ends, U[dt], scale=scale, window=o.get("window"))[0] for y in (v, v.abs()))
        near(got, want, 1.02 * U[dt] * (size + want.abs()) + 2.0 ** -20, "out")


@pytest.mark.parametrize("news,ctxs", [([1, 1, 2], [500, 90, 300]), ([1, 200, 50], [700, 100, 333]), ([1], [3000])])
@pytest.mark.parametrize("window", [None, 37])
def test_the_least_prefix_is_none(news, ctxs, window):
    """-2^31, of which nothing can be taken: as any other negative prefix."""
    ends = [c + n for c, n in zip(ctxs, news)]
    k, v, table = pool(ends, 200, 16, 2, 64, BF, 30)
    q = queries(sum(news), 4, 64, BF, 31)
    ref, bound = reference(q, k, v, table, news, ends, U[BF], window=window)
    for most in (max(news), None):
        got = A.attend_pages(q.cuda(), k.cuda(), v.cuda(), table.cuda(), starts_of(news).cuda(), ints(ends), most=most, window=window,
                             prefix=ints([-2 ** 31] * len(news)))
        near(got, ref, bound, "out")


@pytest.mark.parametrize("Hq,Hk,D,dt,page", [(6, 2, 128, BF, 16), (4, 1, 64, HF, 128)])
@pytest.mark.parametrize("news,ctxs,most", [([1, 1, 1, 1], [5000, 900, 64, 2777], 1), ([3, 1, 6], [4000, 2500, 30], 6), ([200, 1, 40, 300], [3000, 2000, 1500, 0], None),
                                            ([1], [9000], 1), ([128] * 6, [2500] * 6, None)])
@pytest.mark.parametrize("window,prefix", [(1, 1), (33, 65), (200, 300), (64, 900)])
def test_a_prefix_far_before_the_window(Hq, Hk, D, dt, page, news, ctxs, most, window, prefix):
    """Most keys lie between the two and are nobody's; they hold NaN here, but for those in the tiles at both ends."""
    ends = [c + n for c, n in zip(ctxs, news)]
    k, v, table = pool(ends, PO.up(max(ends), page) + 1, page, Hk, D, dt, 32)
    for r, (n, end) in enumerate(zip(news, ends)):
        for j in range(-(-prefix // 64) * 64, (end - n - window + 1) // 64 * 64):
            k[table[r, j // page], :, j % page] = v[table[r, j // page], :, j % page] = float("nan")
    q = queries(sum(news), Hq, D, dt, 33)
    pre = torch.full((len(news),), prefix, dtype=torch.int32)
    got = A.attend_pages(q.cuda(), k.cuda(), v.cuda(), table.cuda(), starts_of(news).cuda(), ints(ends), most=most, window=window, prefix=pre.cuda())
    ref, bound = reference(q, k, v, table, news, ends, U[dt], window=window, prefix=pre.long())
    near(got, ref, bound, "out")
