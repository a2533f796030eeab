"""Preparation of packed tokens into pages: equal, bit for bit, to the preparation into rows at the same positions, which has tests
against the oracle of its own; everything else in the pages stays."""
import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import slotrope_hip as R

BF, HF, F = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("N,Hq,Hk,D,dt,rot,pairs,page,by_token", [
    (1, 1, 1, 64, BF, 64, False, 16, False), (37, 6, 2, 128, BF, 128, False, 16, True), (300, 4, 4, 64, HF, 32, True, 64, False),
    (129, 3, 1, 128, F, 64, True, 32, True), (2000, 12, 4, 128, HF, 128, False, 4096, False)])
def test_pages_hold_what_the_rows_preparation_gives(N, Hq, Hk, D, dt, rot, pairs, page, by_token):
    print("rope pages", N, Hq, Hk, D, dt, flush=True)
    g = torch.Generator().manual_seed(N)
    qkv = torch.randn(N, Hq + 2 * Hk, D, generator=g).to(dt).cuda()
    q, k, v = qkv.split([Hq, Hk, Hk], 1)                 # slices of one projection, no copies
    wq, wk = ((1 + 0.2 * torch.randn(D, generator=g)).to(dt).cuda() for _ in range(2))
    P = -(-N // page) + 3
    slots = torch.randperm(P * page, generator=g)[:N]
    slots[::7] = torch.tensor([-1, P * page, -2 ** 63, 2 ** 63 - 1])[torch.arange(len(slots[::7])) % 4]
    pos = torch.randint(-3, 1 << 20, (N,), generator=g).int()
    pos[0] = 2 ** 31 - 1
    pool = lambda: torch.randn(P, page, Hk, D, generator=g).to(dt).cuda().transpose(1, 2) if by_token else torch.randn(P, Hk, page, D, generator=g).to(dt).cuda()
    kp, vp = pool(), pool()
    wantk, wantv = kp.clone(), vp.clone()
    freqs = R.frequencies(rot, device="cuda")
    with torch.no_grad():
        q1, k1 = R.qk_rope(q.transpose(0, 1).unsqueeze(0), k.transpose(0, 1).unsqueeze(0), wq, wk, freqs, positions=pos.cuda(), interleaved=pairs)
        version = kp._version
        got = R.qk_rope_pages(q, k, v, wq, wk, freqs, pos.cuda(), slots.cuda(), kp, vp, interleaved=pairs)
    assert kp._version > version and vp._version > 0
    ok = (slots >= 0) & (slots < P * page)
    at, row = (slots[ok] // page).cuda(), (slots[ok] % page).cuda()
    ok = ok.cuda()
    wantk[at, :, row] = k1[0].transpose(0, 1)[ok]
    wantv[at, :, row] = v[ok]
    torch.cuda.synchronize()
    assert torch.equal(got, q1[0].transpose(0, 1)) and got.is_contiguous()
    assert torch.equal(kp, wantk) and torch.equal(vp, wantv)
