"""What the entry points over caches in pages write, by the C-ABI with buffers of the caller: the output, the workspace and the state, and nothing around
them, whatever starts, ends and tables hold; and no result depends on what the workspace held before."""
import pytest
import torch

from page_cases import pool, starts_of
from test_gpu_attn_pages import BF, HF, queries

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import slotscan_lib as L

ints = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
NONE = 2 ** 31 - 1
EDGE = 4096                                              # bytes around each buffer


class Guarded:
    """n bytes between two edges that hold a pattern."""

    def __init__(self, n, fill):
        self.all = torch.full((n + 2 * EDGE,), 0x5a, dtype=torch.uint8, device="cuda")
        self.body = self.all[EDGE: EDGE + n]
        self.body.fill_(fill)

    def ptr(self):
        return self.body.data_ptr()

    def intact(self):
        return bool((self.all[:EDGE] == 0x5a).all()) and bool((self.all[EDGE + self.body.numel():] == 0x5a).all())


def attend(q, k, v, table, starts, ends, most, dt, fill, window=NONE, prefix=None):
    (N, Hq, D), (P, Hk, page, _), (R, M) = q.shape, k.shape, table.shape
    lib = L.lib()
    out = Guarded(2 * N * Hq * D, fill)
    n = lib.slotattn_pages_workspace(N, R, M, page, Hq, Hk, D, most, window, prefix is not None)
    ws = Guarded(n, fill)
    L.call(lib.slotattn_pages, "slotattn_pages", q.device, *L.by_head(q), *L.strided(k), *L.strided(v), L._TYPE_CODES[dt], table.data_ptr(), M, starts.data_ptr(),
           ends.data_ptr(), N, R, M, P, page, Hq, Hk, D, most, D ** -0.5, window, 0.0, None, None if prefix is None else prefix.data_ptr(),
           ws.ptr() if n else None, out.ptr())
    torch.cuda.synchronize()
    assert out.intact() and ws.intact()
    return out.body.view(dt).view(N, Hq, D)


@pytest.mark.parametrize("starts", [[0, 64, 0, 64], [-5, 10, NONE, 3], [64, 64, 64, 64], [30, 10, 50, 20], [-2 ** 31, NONE, -1, 64], [0, 20, 21, 64]])
@pytest.mark.parametrize("ends", [[200, 100, 300], [NONE, -1, 5], [5000, 64, 0]])
@pytest.mark.parametrize("D,dt", [(64, HF), (128, BF)])
def test_only_the_output_and_the_workspace_are_written(starts, ends, D, dt):
    k, v, table = (x.cuda() for x in pool([200, 100, 300], 20, 16, 2, D, dt, 25))
    before = [x.clone() for x in (k, v, table)]
    q = queries(64, 4, D, dt, 26).cuda()
    for wide in (20, 80):                                # one workgroup a unit where rows have few keys, shares else
        t = torch.full((3, wide), -1, dtype=torch.int32, device="cuda")
        t[:, :20] = table
        for most in (1, 5, 64):
            print("starts", starts, ends, wide, most, flush=True)
            attend(q, k, v, t, ints(starts), ints(ends), most, dt, 0xff)
            attend(q, k, v, t, ints(starts), ints(ends), most, dt, 0x7f, window=40, prefix=ints([3, -1, NONE]))
    for x, y in zip((k, v, table), before):
        assert torch.equal(x.nan_to_num(7) if x.is_floating_point() else x, y.nan_to_num(7) if y.is_floating_point() else y)


@pytest.mark.parametrize("news,ctxs,most", [([1] * 70, [(31 * r) % 400 for r in range(70)], 1), ([1, 3, 0, 2], [9000, 100, 4, 2000], 3), ([1, 200, 0, 40, 5], [700, 90, 3, 0, 60], 245),
                                            ([40] * 30, [100] * 30, 40), ([1] * 6, [50] * 6, 1)])
@pytest.mark.parametrize("Hq,Hk,D,dt", [(6, 2, 128, BF), (4, 2, 64, HF)])
def test_what_the_workspace_held_before_does_not_matter(news, ctxs, most, Hq, Hk, D, dt):
    ends = [c + n for c, n in zip(ctxs, news)]
    k, v, table = (x.cuda() for x in pool(ends, max(-(-e // 16) for e in ends) + 1, 16, Hk, D, dt, 34))
    q = queries(sum(news) + 3, Hq, D, dt, 35).cuda()
    outs = [attend(q, k, v, table, starts_of(news).cuda(), ints(ends), most, dt, fill) for fill in (0, 0xff, 0x7f, 0x01)]
    assert all(torch.equal(o, outs[0]) for o in outs[1:]) and bool(outs[0].isfinite().all())


@pytest.mark.parametrize("R,M,P,N", [(3, 5, 11, 40), (1100, 3, 900, 3000), (5000, 2, 700, 9000)])
def test_tables_write_their_state_and_outputs_alone(R, M, P, N):
    g = torch.Generator().manual_seed(R)
    lib, i32 = L.lib(), torch.int32
    lens, table, free = Guarded(4 * R, 0), Guarded(4 * R * M, 0xff), Guarded(4 * (1 + P), 0)
    free.body.view(i32).copy_(torch.cat((torch.tensor([P]), torch.randperm(P, generator=g))).int())
    starts, ends, slots, pos = Guarded(4 * (R + 1), 0x7f), Guarded(4 * R, 0x7f), Guarded(8 * N, 0x7f), Guarded(4 * N, 0x7f)
    dev = lens.all.device
    for step in range(6):
        new = torch.randint(-2, 9 if step % 2 else 60, (R,), generator=g).int().cuda()
        new[::5] = NONE if step == 4 else 1
        L.call(lib.slotpage_extend, "slotpage_extend", dev, new.data_ptr(), lens.ptr(), table.ptr(), M, free.ptr(), R, M, P, 16, N, starts.ptr(), ends.ptr(), slots.ptr(), pos.ptr())
        keep = torch.randint(-5, 60, (R,), generator=g).int().cuda()
        if step == 3:                                    # nonsense: lengths past the table and below 0, pages that are not there
            lens.body.view(i32)[::2] = NONE
            lens.body.view(i32)[1::2] = -7
            table.body.view(i32)[::3] = 1 << 30
            free.body.view(i32)[0] = NONE
        L.call(lib.slotpage_trim, "slotpage_trim", dev, keep.data_ptr(), lens.ptr(), table.ptr(), M, free.ptr(), R, M, P, 16)
        torch.cuda.synchronize()
        assert all(x.intact() for x in (lens, table, free, starts, ends, slots, pos)), step
        assert 0 <= int(free.body.view(i32)[0]) <= P
        written = slots.body.view(torch.int64)
        assert bool(((written >= -1) & (written < P * 16)).all())
