/* C-ABI of the page tables of a cache in pages (MI355X, gfx950), part of libslotscan.so.
 *
 * A cache in pages holds the keys and values of many sequences in P pages of `page` tokens each (slotrope_pages writes them,
 * slotattn_pages reads them).  The state, all int32 on the device and the caller's:
 *     lens (R)       tokens of each row's sequence
 *     table (R, M)   the pages of each row, in the sequence's order (rows t_sr elements apart); behind a row's last page: anything
 *                    (slotpage_trim leaves -1)
 *     free (1 + P)   free[0] = n, the number of free pages, free[1 .. n] a stack of them (its top is free[n])
 *
 * slotpage_extend gives every row r the new[r] tokens of this step (a negative count is 0) and the pages that they need:
 *     starts (R + 1) the rows' tokens in the packed batch of N: row r has starts[r] .. starts[r + 1] - 1 (running sums of new, N at most)
 *     ends (R)       lens[r] + new[r], which is lens[r] from here on; 0 for a row without new tokens or without room
 *     pos, slots (N) a token's position in its sequence, and table[r][pos / page] page + pos % page: its place in the pages;
 *                    -1 for tokens behind the last row's and those of a row without room (slots also where the table holds no page)
 * A row has room when its tokens end within N, lens[r] >= 0 and lens[r] + new[r] <= M page, and the pages that it and the rows before
 * it ask for are there (a row that needs none always has them): no row overtakes one that waits.  A row without room
 * keeps its lens and its pages.  Pages leave the stack from its top, in the order of rows and tokens.
 *
 * slotpage_trim cuts every row to its first min(lens[r], keep[r]) tokens (0: the row is free) and puts the pages behind them back, the first row's
 * first one on top: trimming to the lengths before an extension undoes it, the stack's order included.
 *
 * page a power of two in [16, 4096]; R <= 2^24, P and M page < 2^30.
 * Nothing outside the state is read or written whatever it holds; calls on one state must be ordered by the caller.
 * Conventions as in slotscan.h (device pointers, caller-allocated, launched on `stream`, 0 or a SLOTSCAN_ERR_* code). */
#ifndef SLOTPAGE_H
#define SLOTPAGE_H
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define SLOTPAGE_MIN 16
#define SLOTPAGE_MAX 4096
int slotpage_extend(const int32_t* new_, int32_t* lens, int32_t* table, int64_t t_sr, int32_t* free_, int64_t R, int64_t M,
                    int64_t P, int64_t page, int64_t N, int32_t* starts, int32_t* ends, int64_t* slots, int32_t* pos,
                    void* stream);
int slotpage_trim(const int32_t* keep, int32_t* lens, int32_t* table, int64_t t_sr, int32_t* free_, int64_t R, int64_t M,
                  int64_t P, int64_t page, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* SLOTPAGE_H */
