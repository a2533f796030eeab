"""How the attention over pages shares its work out, on the CPU: the arithmetic that its kernels run, compiled for the host from their header."""
import os
import subprocess

import build

_PRELUDE = """
#include <cstdio>
#include <cstdlib>
#include <cstdint>
#include <climits>
#include "slot_attn_pages.h"
using namespace slotattn;
#define CHECK(x) do { if (!(x)) { printf("line %d: %s\\n", __LINE__, #x); exit(1); } } while (0)
static uint64_t state = 1;
static int rnd(int lo, int hi) {                     // in [lo, hi]
    state = state * 6364136223846793005ull + 1442695040888963407ull;
    return (int)(lo + (int64_t)((state >> 33) % ((uint64_t)((int64_t)hi - lo) + 1)));
}
"""


def _run(tmp_path, body):
    src, out = str(tmp_path / "shares.cpp"), str(tmp_path / "shares")
    with open(src, "w") as f:
        f.write(_PRELUDE + body)
    r = subprocess.run([build.HIPCC, "--offload-host-only", "-x", "hip", "-std=c++17", "-O1", "-ftrapv", "-I", build.CSRC, "-I", os.path.join(build.ROOT, "include"),
                        src, "-o", out], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([out], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr


def test_entries_that_nobody_wrote_name_no_piece_outside(tmp_path):
    """The join of few rows finds what the workspace held before where rows that share tokens ask for more tiles than are handed out: whatever it is, the
    rows that it reads, (2 me + 1) and 2 (me + z) for z < parts, are among the two of each worker."""
    _run(tmp_path, """
int main() {
    const int odd[] = {0, 1, 2, 3, -1, -2, 1023, 1024, 1025, 2048, INT_MAX, INT_MAX - 1, INT_MIN, INT_MIN + 1, 0x7fc00000, (int)0xcdcdcdcd};
    const int G[] = {1, 2, 7, 1024, 2048};
    auto look = [&](Piece p, int g) {
        const int n = p.there(g);
        if (n < 2) return;
        CHECK(p.me >= 0 && 2ll * p.me + 1 < 2ll * g && 2ll * ((int64_t)p.me + n - 1) < 2ll * g && n == p.parts);
    };
    for (int g : G) {
        for (int m : odd) for (int n : odd) look({m, n}, g);
        for (int i = 0; i < 200000; i++) look({rnd(-3, g + 3), rnd(-3, g + 3)}, g), look({rnd(INT_MIN / 2, INT_MAX / 2), rnd(0, g)}, g);
        for (int m = 0; m < g; m++) CHECK((Piece{m, g - m}.there(g) == g - m));      // what the workers write counts whole
        CHECK((Piece{0, 1}.there(g) == 1));
    }
}
""")
