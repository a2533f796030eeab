// The few-row kernels of the attention over pages, as its entry point launches them.
#pragma once
#include "slot_attn_pages.h"

#define FG 1024                                      // waves that share all units: four a CU, whose rings fill the LDS
#define FS 4                                         // tiles of one of them at least
#define FW 4                                         // waves that share one unit

namespace slotattn_few {
// G workers with equal shares (0: a workgroup a unit, `tiles` of 32 rows a key/value head)
void launch(const slotattn::PagedArgs& a, int dtype, int D, bool cap, int G, int tiles, hipStream_t st);
}
