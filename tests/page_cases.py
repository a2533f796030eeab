"""Seeded inputs of the tests of caches in pages (CPU tensors)."""
import torch

from oracle import page_oracle as PO


def pool(rows, M, page, Hk, D, dt, seed, gain=1.4, by_token=False, stale=float("nan")):
    """Keys and values of sequences of `rows` tokens, on pages in no order of a pool that holds `stale` everywhere else: (kpages,
    vpages, table)."""
    g = torch.Generator().manual_seed(seed)
    held = [PO.up(n, page) for n in rows]
    P = sum(held) + 2
    ids = torch.randperm(P, generator=g).tolist()
    table = torch.full((len(rows), M), -1, dtype=torch.int32)
    # (pages that hold their tokens one after another, or their heads)
    new = lambda: torch.full((P, page, Hk, D), stale).to(dt).transpose(1, 2) if by_token else torch.full((P, Hk, page, D), stale).to(dt)
    k, v = new(), new()
    for r, n in enumerate(rows):
        for i in range(held[r]):
            p = ids.pop()
            table[r, i] = p
            m = min(page, n - i * page)
            k[p, :, :m] = (gain * torch.randn(Hk, m, D, generator=g)).to(dt)
            v[p, :, :m] = torch.randn(Hk, m, D, generator=g).to(dt)
    return k, v, table


def starts_of(news):
    s = [0]
    for n in news:
        s.append(s[-1] + n)
    return torch.tensor(s, dtype=torch.int32)
