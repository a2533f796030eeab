"""The operators on caches in pages used together, as a server uses them: prompts packed beside generated tokens, steps captured in a graph and
replayed while sequences grow, guessed tokens taken back, rows that wait for pages; and each at what its own tests leave: two streams, two
graphs, far offsets, values that are not finite, bounds that the host got wrong."""
import pytest
import torch

from attn_cases import U, near
from oracle import attn_oracle as AO
from oracle import page_oracle as PO
from page_cases import pool, starts_of
from test_gpu_attn_pages import queries, reference, run

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import slotattn_hip as A
    import slotpage_hip as P
    import slotrope_hip as R

BF, HF = torch.bfloat16, torch.float16
ints = lambda *x: torch.tensor(x, dtype=torch.int32)


class Server:
    """Sequences on pages, and every token's projection kept for the dense reference."""

    def __init__(self, R_, M, pages, page, Hq, Hk, D, dt, seed, **opt):
        self.page, self.Hq, self.Hk, self.D, self.dt, self.opt = page, Hq, Hk, D, dt, opt
        self.g = torch.Generator().manual_seed(seed)
        self.wq, self.wk = ((1 + 0.2 * torch.randn(D, generator=self.g)).to(dt).cuda() for _ in range(2))
        self.freqs = R.frequencies(D, device="cuda")
        self.lens, self.table, self.free = P.page_state(R_, M, pages)
        nan = lambda: torch.full((pages, Hk, page, D), float("nan"), device="cuda", dtype=dt)
        self.kp, self.vp = nan(), nan()
        self.seen = [torch.empty(0, Hq + 2 * Hk, D, dtype=dt) for _ in range(R_)]

    def tokens(self, n):
        return torch.randn(n, self.Hq + 2 * self.Hk, self.D, generator=self.g).to(self.dt)

    def step(self, new, x, N, most=None):
        """One layer's step: (the step's layout, its output)."""
        s = P.page_extend(new, self.lens, self.table, self.free, self.page, N)
        q, k, v = x.split([self.Hq, self.Hk, self.Hk], 1)
        q1 = R.qk_rope_pages(q, k, v, self.wq, self.wk, self.freqs, s.pos, s.slots, self.kp, self.vp)
        return s, A.attend_pages(q1, self.kp, self.vp, self.table, s.starts, s.ends, most=most, **self.opt)

    def check(self, new, x, out, taken):
        """Every row's output against the oracle over its whole sequence; rows that were not taken: 0."""
        at, out = 0, out.cpu()
        for r, n in enumerate(new):
            if n and taken[r]:
                self.seen[r] = torch.cat((self.seen[r], x[at: at + n]))
                full = self.seen[r].cuda()
                T = full.shape[0]
                q, k, v = (y.transpose(0, 1).unsqueeze(0) for y in full.split([self.Hq, self.Hk, self.Hk], 1))
                q1, k1 = R.qk_rope(q, k, self.wq, self.wk, self.freqs)
                ref, bound = AO.attention(q1[:, :, T - n:].cpu(), k1.cpu(), v.cpu(), u=U[self.dt], **self.opt)["out"]
                near(out[at: at + n], ref[0].transpose(0, 1), bound[0].transpose(0, 1), f"row {r} of {T} tokens")
            elif n:
                assert not bool(out[at: at + n].any())
            at += n
        assert not bool(out[at:].any())


@pytest.mark.parametrize("page,Hq,Hk,D,dt,opt", [(16, 6, 2, 128, BF, dict(cap=30.0)), (64, 4, 4, 64, HF, dict(window=50)), (32, 8, 1, 64, BF, {})])
@torch.no_grad()
def test_prompts_steps_guesses_and_rows_that_wait(page, Hq, Hk, D, dt, opt):
    s = Server(5, 400 // page + 2, 700 // page + 4, page, Hq, Hk, D, dt, 3, **opt)
    gone = []
    for new in ([70, 3, 0, 130, 0], [1, 1, 20, 1, 0], [1, 1, 1, 1, 1], [5, 1, 4, 1, 9], [1, 0, 1, 1, 1], [0, 0, 0, 300, 90], [1, 1, 1, 250, 1], [1, 1, 1, 1, 1]):
        print("step", new, flush=True)
        x, before = s.tokens(sum(new) + 3), s.lens.clone()
        step, out = s.step(ints(*new).cuda(), x.cuda(), sum(new) + 3, most=max(new))
        taken = (step.ends > 0).tolist()
        s.check(new, x, out, taken)
        gone.append(not all(t or not n for t, n in zip(taken, new)))
        if new == [5, 1, 4, 1, 9]:                       # guesses: one token of the first row and two of the third stay, the last row ends
            keep = before + ints(1, 1, 2, 1, -100).cuda()
            P.page_trim(keep, s.lens, s.table, s.free, page)
            for r, n in enumerate(keep.clamp_min(0).tolist()):
                s.seen[r] = s.seen[r][:n]
            assert s.lens.tolist() == keep.clamp_min(0).tolist()
    assert any(gone)                                     # some row had to wait
    P.page_trim(torch.zeros(5, dtype=torch.int32).cuda(), s.lens, s.table, s.free, page)
    assert sorted(s.free.tolist()[1:]) == list(range(700 // page + 4)) and s.free[0].item() == 700 // page + 4


@torch.no_grad()
def test_a_captured_step_is_replayed_while_sequences_grow():
    """Extension, preparation and attention in one graph over static buffers; the eager work and the synchronizations of a program between the
    replays; every replay against the oracle."""
    s = Server(4, 12, 40, 16, 6, 2, 64, BF, 5)
    new, N = ints(60, 17, 1, 90), 168
    x = s.tokens(N)
    step, out = s.step(new.cuda(), x.cuda(), N)
    s.check(new.tolist(), x, out, [True] * 4)
    static_new, static_x = ints(1, 1, 1, 1).cuda(), s.tokens(6).cuda()
    state = [y.clone() for y in (s.lens, s.table, s.free, s.kp, s.vp)]
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s.step(static_new, static_x, 6, most=1)          # warm: the libraries' first calls
        for y, z in zip((s.lens, s.table, s.free, s.kp, s.vp), state):
            y.copy_(z)
        with torch.cuda.graph(graph, stream=side):
            gstep, gout = s.step(static_new, static_x, 6, most=1)
    torch.cuda.current_stream().wait_stream(side)
    for new in ([1, 1, 1, 1], [1, 0, 1, 1], [0, 1, 1, 1], [1, 1, 1, 1], [1, 1, 1, 0]):
        x = s.tokens(6)
        static_new.copy_(ints(*new))
        static_x.copy_(x)
        graph.replay()
        s.check(new, x, gout, (gstep.ends > 0).tolist())
        torch.cuda.synchronize()
        static_x.normal_()                               # eager work between


@torch.no_grad()
def test_two_graphs_and_two_streams():
    """Two calls with workspaces captured apart and replayed in turn, and the same two on two streams at once."""
    k, v, table = pool([5000, 3000, 4100], 320, 16, 2, 128, BF, 7)
    kc, vc, tc = k.cuda(), v.cuda(), table.cuda()
    sets = []
    for news, ends, most, seed in (([1, 1, 1], [5000, 3000, 4100], 1, 8), ([300, 2, 40], [4000, 2900, 4100], None, 9)):
        q = queries(sum(news), 6, 128, BF, seed)
        sets.append((q.cuda(), starts_of(news).cuda(), ints(*ends).cuda(), most, reference(q, k, v, table, news, ends, U[BF])))
    call = lambda z: A.attend_pages(z[0], kc, vc, tc, z[1], z[2], most=z[3])
    eager = [call(z) for z in sets]
    for o, z in zip(eager, sets):
        near(o, *z[4], "out")
    graphs = []
    for z in sets:
        g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side), torch.cuda.graph(g, stream=side):
            o = call(z)
        torch.cuda.current_stream().wait_stream(side)
        graphs.append((g, o))
    for _ in range(3):
        for g, o in graphs:
            o.fill_(7.0)
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (g, o), e in zip(graphs, eager):
            assert torch.equal(o, e)
    streams = [torch.cuda.Stream() for _ in sets]
    outs = [[], []]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    for _ in range(8):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[i].append(call(sets[i]))
    torch.cuda.synchronize()
    for i, e in enumerate(eager):
        assert all(torch.equal(o, e) for o in outs[i])   # the same bits, whatever runs beside


@pytest.mark.parametrize("news,ctxs", [([5, 40, 1], [100, 300, 7]), ([9], [4000]), ([1, 70, 3], [3000, 0, 2500])])
@pytest.mark.parametrize("Hq,Hk", [(6, 2), (12, 1)])
def test_a_bound_that_is_too_small_changes_no_result(news, ctxs, Hq, Hk):
    """Rows with more tokens than `most` says."""
    for most in (0, 1, 3):
        run(news, ctxs, 16, Hq, Hk, 64, BF, 11, pad=2, most=most)


@pytest.mark.parametrize("news,most", [([3, 1, 2], 3), ([3, 40, 70], None)])
@pytest.mark.parametrize("D,dt,o", [(128, BF, {}), (64, HF, dict(window=20, cap=10.0)), (64, BF, dict(slopes=True))])
@pytest.mark.parametrize("long", [0, 2600])
def test_values_that_are_not_finite_stay_with_the_rows_that_see_them(news, most, D, dt, o, long):
    """An infinity or a NaN in a sequence's last token reaches its last row alone; one in its first token the rows whose window holds it."""
    ctxs = [90 + long, 30 + long, 0]
    ends = [c + n for c, n in zip(ctxs, news)]
    M = PO.up(max(ends), 16)
    k, v, table = pool(ends, M, 16, 2, D, dt, 13)
    clean = [x.clone() for x in (k, v)]
    put = lambda x, r, j, val: x[int(table[r, j // 16])].__setitem__((slice(None), j % 16, 5), val)
    put(v, 0, ends[0] - 1, float("inf"))
    put(k, 1, ends[1] - 1, float("nan"))
    put(v, 2, 0, float("nan"))
    q = queries(sum(news), 4, D, dt, 14)
    opt = dict(o)
    if opt.get("slopes"):
        opt["slopes"] = 0.5 ** torch.arange(1, 5)
    og = {a: b.cuda() if torch.is_tensor(b) else b for a, b in opt.items()}
    got = A.attend_pages(q.cuda(), k.cuda(), v.cuda(), table.cuda(), starts_of(news).cuda(), ints(*ends).cuda(), most=most, **og).cpu().double()
    ref, bound = reference(q, *clean, table, news, ends, U[dt], **opt)
    s = starts_of(news).tolist()
    sees = torch.zeros(sum(news), dtype=torch.bool)
    sees[s[1] - 1] = sees[s[2] - 1] = True
    W = opt.get("window") or 1 << 30
    sees[s[2]: s[3]] = torch.arange(ctxs[2], ends[2]) < W
    near(got[~sees], ref[~sees], bound[~sees], "rows that do not see it")
    assert bool(torch.isnan(got[s[2] - 1]).all()), "a NaN among the scores"
    bad = torch.zeros(D, dtype=torch.bool)
    bad[5] = True
    assert bool((got[s[1] - 1][:, bad] == float("inf")).all()), "an infinity with a weight"
    near(got[s[1] - 1][:, ~bad], ref[s[1] - 1][:, ~bad], bound[s[1] - 1][:, ~bad], "the other columns of that row")
    for i in range(s[2], s[3]):
        if sees[i]:
            assert bool(torch.isnan(got[i][:, bad]).all())
            near(got[i][:, ~bad], ref[i][:, ~bad], bound[i][:, ~bad], "the other columns of the rows that see a NaN value")


@pytest.mark.parametrize("news,ctxs,most", [([900], [0], None), ([1, 3], [6000, 9000], 3), ([1], [900], 1)])
@pytest.mark.parametrize("dt", [BF, HF])
def test_a_nan_that_every_row_sees_costs_one_pass(news, ctxs, most, dt):
    """The rows keep their sums: the column with the NaN is NaN, the others are as without it."""
    ends = [c + n for c, n in zip(ctxs, news)]
    k, v, table = pool(ends, PO.up(max(ends), 32), 32, 2, 128, dt, 17)
    clean = v.clone()
    for r in range(len(news)):
        v[table[r, 0], :, 0, 77] = float("nan")
    q = queries(sum(news), 6, 128, dt, 18)
    got = A.attend_pages(q.cuda(), k.cuda(), v.cuda(), table.cuda(), starts_of(news).cuda(), ints(*ends).cuda(), most=most).cpu().double()
    ref, bound = reference(q, k, clean, table, news, ends, U[dt])
    bad = torch.arange(128) == 77
    assert bool(torch.isnan(got[..., bad]).all())
    near(got[..., ~bad], ref[..., ~bad], bound[..., ~bad], "the other columns")


def test_offsets_past_32_bits():
    """A pool of more than 2^32 bytes: its last pages are written and read."""
    page, Hk, D, n = 64, 4, 128, 70000                   # 65,536 bytes a page and pool
    kp, vp = (torch.zeros(n, Hk, page, D, device="cuda", dtype=BF) for _ in range(2))
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(200, 12 + 2 * Hk, D, generator=g).to(BF).cuda()
    q, k, v = qkv.split([12, Hk, Hk], 1)
    lens, table, free = P.page_state(2, 5, n)
    free.copy_(torch.cat((ints(n), torch.arange(n, dtype=torch.int32))))                 # the last page leaves first
    with torch.no_grad():
        s = P.page_extend(ints(130, 70).cuda(), lens, table, free, page, 200)
        assert s.slots.max().item() == n * page - 1 and s.slots.min().item() == (n - 5) * page and table[0].tolist() == [n - 1, n - 2, n - 3, -1, -1]
        q1 = R.qk_rope_pages(q, k, v, None, None, R.frequencies(D, device="cuda"), s.pos, s.slots, kp, vp)
        _, k1 = R.qk_rope(q.transpose(0, 1).unsqueeze(0), k.transpose(0, 1).unsqueeze(0), None, None, R.frequencies(D, device="cuda"), positions=s.pos)
        assert torch.equal(kp[n - 1, :, :64], k1[0][:, :64]) and torch.equal(vp[n - 4, :, :64], v[130:194].transpose(0, 1))
        assert not bool(kp[0].any()) and not bool(kp[(n - 1) * 65536 % (1 << 32) // 65536].any())
        small_k, small_v = kp[n - 5:].cpu(), vp[n - 5:].cpu()
        ts = torch.where(table >= 0, table - (n - 5), -1).cpu()
        for most in (None, 1):                           # both ways that such rows may take
            got = A.attend_pages(q1, kp, vp, table, s.starts, s.ends, most=most)
            ref, bound = reference(q1.cpu(), small_k, small_v, ts, [130, 70], [130, 70], U[BF])
            near(got, ref, bound, "out")


def test_rows_and_pages_of_any_stride():
    """Queries that are slices of a wider projection, pages that are parts of a wider pool, a table between other columns; rows that are not
    aligned are copied where they are few, and refused where they are the pool's."""
    news, ctxs = [1, 9, 30], [200, 77, 0]
    ends = [c + n for c, n in zip(ctxs, news)]
    k, v, table = pool(ends, 16, 16, 2, 64, HF, 21)
    q = queries(40, 6, 64, HF, 22)
    ref, bound = reference(q, k, v, table, news, ends, U[HF])
    wide = torch.full((k.shape[0], 2, 3, 16, 64), float("nan"), dtype=HF, device="cuda")
    wide[:, 0, :2], wide[:, 1, :2] = k.cuda(), v.cuda()
    wt = torch.full((3, 40), 2 ** 31 - 1, dtype=torch.int32, device="cuda")
    wt[:, 7:23] = table.cuda()
    for qg in (torch.cat((q, q), 1).cuda()[:, 6:], torch.cat((q, q), 2).cuda()[..., :64], torch.cat((q[..., :1], q), 2).cuda()[..., 1:],
               q.transpose(0, 1).contiguous().cuda().transpose(0, 1)):
        got = A.attend_pages(qg, wide[:, 0, :2], wide[:, 1, :2], wt[:, 7:23], starts_of(news).cuda(), ints(*ends).cuda())
        near(got, ref, bound, "out")


def test_empty_batches():
    k, v, table = pool([20], 2, 16, 2, 64, BF, 23)
    kc, vc, tc = k.cuda(), v.cuda(), table.cuda()
    none = torch.empty(0, 4, 64, device="cuda", dtype=BF)
    assert A.attend_pages(none, kc, vc, tc, ints(0, 0).cuda(), ints(0).cuda()).shape == (0, 4, 64)
    q = queries(3, 4, 64, BF, 24).cuda()
    for args in ((kc[:0], vc[:0], tc, ints(0, 3).cuda(), ints(3).cuda()), (kc, vc, tc[:0], ints(0).cuda(), torch.empty(0, dtype=torch.int32, device="cuda")),
                 (kc, vc, tc[:, :0], ints(0, 3).cuda(), ints(3).cuda()), (kc, vc, tc, ints(0, 0).cuda(), ints(0).cuda())):
        for most in (None, 1):
            out = A.attend_pages(q, *args, most=most)
            assert out.shape == (3, 4, 64) and not bool(out.any())
    with torch.no_grad():
        version = kc._version
        out = R.qk_rope_pages(none, none[:, :2], none[:, :2], None, None, R.frequencies(64, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda"),
                              torch.empty(0, dtype=torch.int64, device="cuda"), kc, vc)
        assert out.shape == (0, 4, 64) and kc._version == version


def test_starts_that_make_no_sense_stay_in_bounds():
    """Starts that fall, pass the batch or are negative: whatever comes out, only the output is written."""
    k, v, table = pool([200, 100, 300], 20, 16, 2, 64, BF, 25)
    kc, vc, tc = k.cuda(), v.cuda(), table.cuda()
    q = queries(64, 4, 64, BF, 26).cuda()
    for starts in ([0, 64, 0, 64], [-5, 10, 2 ** 31 - 1, 3], [64, 64, 64, 64], [30, 10, 50, 20], [-2 ** 31, 2 ** 31 - 1, -1, 64]):
        for ends in ([200, 100, 300], [2 ** 31 - 1, -1, 5]):
            for most in (None, 1):
                print("starts", starts, ends, most, flush=True)
                out = A.attend_pages(q, kc, vc, tc, ints(*starts).cuda(), ints(*ends).cuda(), most=most)
                torch.cuda.synchronize()
                assert out.shape == q.shape
    assert torch.equal(kc.cpu().nan_to_num(7), k.nan_to_num(7)) and torch.equal(tc.cpu(), table)
