"""Page tables of a cache in pages on MI355X (include/slotpage.h): the memory of many growing sequences handed out and taken back
on the GPU, and a step's packed batch laid out from the requests' lengths alone.  qk_rope_pages (slotrope_hip) writes such a cache,
attend_pages (slotattn_hip) reads it.

The state belongs to the caller and may be captured in graphs; all of it is int32 on the GPU:
    lens (R,)     tokens of each row's sequence
    table (R, M)  the pages of each row in the sequence's order (rows may be strided)
    free (1 + P,) free[0] = n free pages, free[1: n + 1] a stack of them

    page_state(R, M, P, device) -> (lens, table, free)
        no tokens, no pages held (-1), all P pages free; the first to leave is page 0.
    page_extend(new, lens, table, free, page, N) -> PageStep(starts, ends, slots, pos)
        gives row r its new[r] tokens (int32 (R,)) of this step and the pages that they need; lens, table and free change in place.
            starts (R + 1,) int32  row r's tokens of the packed batch of N are starts[r] .. starts[r + 1] - 1
            ends (R,) int32        the row's tokens, the new ones included; 0 where it has no new ones or no room
            slots (N,) int64       each token's place in the pages, page number * page + row; -1: none
            pos (N,) int32         its position in the sequence; -1: none
        A row has room when its tokens fit into the batch, into M pages and -- with those of the rows before it -- into the free pages;
        a row without room keeps what it has and waits, and no later row that needs a page overtakes it.  N is the host's: at
        least the sum of new, tokens behind it belong to no row.
    page_trim(keep, lens, table, free, page)
        cuts every row to its first keep[r] tokens (int32 (R,); 0: the row is free, its length or more: nothing changes) and puts the
        pages behind them back, -1 in their place.  Trimming to the lengths before an extension undoes it, order included: the way back
        from guessed tokens.

`page` is a power of two, 16 to 4096.  Whatever the state holds, nothing outside of it is read or written.  No CPU path: a missing library
raises.
"""
from collections import namedtuple

import torch

import slotscan_lib as L
from slotrope_hip import _same_device, _written, check_ints, check_page

PageStep = namedtuple("PageStep", "starts ends slots pos")


def check_table(table, what):
    (R, M), (sr, sm) = table.shape, table.stride()
    if table.dtype is not torch.int32 or M > 1 and sm != 1 or R > 1 and sr < M:
        raise ValueError(f"{what}: table must be int32 (R, M) with contiguous rows that are apart (got {table.dtype}, "
                         f"{tuple(table.shape)}, strides {table.stride()})")


def table_rows(table):
    """Pointer and row stride."""
    return table.data_ptr(), table.stride(0) if table.shape[0] > 1 else table.shape[1]


def page_state(R, M, P, device="cuda"):
    """Lengths, table and free pages of an unused cache (see the module docstring)."""
    i32 = dict(device=device, dtype=torch.int32)
    # P on top of P - 1, ..., 0: the count, and the stack with page 0 on its top
    return torch.zeros(R, **i32), torch.full((R, M), -1, **i32), torch.arange(P, -1, -1, **i32)


def _check(counts, name, lens, table, free, page, what):
    if table.dim() != 2 or table.shape[0] < 1 or table.shape[1] < 1:
        raise ValueError(f"{what}: table must be (R, M), R and M >= 1 (got {tuple(table.shape)})")
    R, M = table.shape
    check_table(table, what)
    check_ints(lens, (R,), torch.int32, what, "lens")
    check_ints(counts, (R,), torch.int32, what, name)
    if free.dim() != 1 or free.shape[0] < 1:
        raise ValueError(f"{what}: free must be (1 + P,) (got {tuple(free.shape)})")
    check_ints(free, (free.shape[0],), torch.int32, what, "free")
    check_page(page, what)
    _same_device(what, counts, lens, table, free)
    return R, M, free.shape[0] - 1


def page_extend(new, lens, table, free, page, N):
    """New tokens and their pages for every row (see the module docstring)."""
    what = "page_extend"
    page, N = int(page), int(N)
    if N < 0:
        raise ValueError(f"{what}: N must be >= 0 (got {N})")
    R, M, P = _check(new, "new", lens, table, free, page, what)
    dev, i32 = table.device, torch.int32
    slots, pos, starts, ends = torch.empty(3 * N + 2 * R + 1, device=dev, dtype=i32).split_with_sizes((2 * N, N, R + 1, R))   # one allocation
    slots = slots.view(torch.int64)
    L.call(L.lib().slotpage_extend, what, dev, new.data_ptr(), lens.data_ptr(), *table_rows(table), free.data_ptr(), R, M, P, page, N,
           starts.data_ptr(), ends.data_ptr(), slots.data_ptr(), pos.data_ptr())
    _written(lens, table, free)
    return PageStep(starts, ends, slots, pos)


def page_trim(keep, lens, table, free, page):
    """Rows cut short and their pages put back (see the module docstring)."""
    what = "page_trim"
    page = int(page)
    R, M, P = _check(keep, "keep", lens, table, free, page, what)
    L.call(L.lib().slotpage_trim, what, table.device, keep.data_ptr(), lens.data_ptr(), *table_rows(table), free.data_ptr(), R, M, P, page)
    _written(lens, table, free)
