// The few-row kernels of the attention over pages, as its entry point launches them.
#pragma once
#include "slot_attn_pages.h"

#define FG 1024                                      // waves that share all units at D = 128: four a CU, whose rings fill the LDS (64: twice as many)
#define FS 4                                         // tiles of one of them at least
#define FW 4                                         // waves that share one unit

namespace slotattn_few {
// Tiles of QR = 16 or 32 rows; G workers with equal shares (0: a workgroup a unit, `tiles` of them a key/value head)
void launch(const slotattn::PagedArgs& a, int dtype, int D, bool cap, int QR, int G, int tiles, hipStream_t st);
}
