"""Rows whose keys are split over waves and workgroups (slotattn_hip): parts of very different size meet, at every row alike."""
import pytest
import torch

from attn_cases import U, attn_inputs, near
from oracle import attn_oracle as AO

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import slotattn_hip as A

BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("B,Hq,Hk,T,S,D,dt", [(24, 8, 2, 1, 700, 128, BF), (40, 4, 4, 2, 300, 64, HF), (1, 32, 1, 3, 5000, 64, BF)])
def test_waves_with_unlike_maxima(B, Hq, Hk, T, S, D, dt):
    """The two waves of a workgroup take every other 32 keys: scores of one wave's keys far above the other's, either way
    about, so that a part weighted by anything but the rows' common maximum is far off; and every repetition gives the same."""
    print("unlike waves", B, Hq, Hk, T, S, D, flush=True)
    q, k, v, _ = attn_inputs(B, Hq, Hk, T, S, D, dt, 91)
    even = (torch.arange(S) // 32 % 2 == 0).view(1, 1, S, 1)
    first = (torch.arange(B) % 2 == 0).view(B, 1, 1, 1)
    k = torch.where(even == first, 3 * k, 0.3 * k).to(dt)
    lens = torch.tensor([S - 13 * b % (S // 2) for b in range(B)], dtype=torch.int32)
    ref = AO.attention(q, k, v, lens=lens, u=U[dt])["out"]
    args = [x.cuda() for x in (q, k, v, lens)]
    with torch.no_grad():
        out = A.attend_cache(*args)
        near(out, *ref, "out")
        for _ in range(20):
            assert torch.equal(A.attend_cache(*args), out)
