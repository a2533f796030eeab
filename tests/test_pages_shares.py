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


def test_shares_count_the_tiles_that_are_visited(tmp_path):
    """With a prefix and a window far behind it, the tiles between them cost nothing and are nobody's: a unit's number of tiles is that of the tiles in which
    one of its rows sees a key, its parts visit them all once, each as many as its share has, and four waves of a workgroup visit them, too."""
    _run(tmp_path, """
#include <vector>
#include <algorithm>
template <int STEP> void look(const PagedArgs& a, const Seq& x, int p0, int p1) {
    std::vector<int> want;                            // the first keys of tiles that somebody sees
    const int lo = std::max(0, std::max(p0, 0) - a.W + 1), hi = std::min(x.klen, p1 + 1), pre = p1 >= 0 ? std::min(x.pre, x.klen) : 0;
    for (int j = 0; j < x.klen; j += STEP)
        if ((lo < hi && j < hi && j + STEP > lo) || j < pre) want.push_back(j);
    const Reach<STEP> all(a, x, p0, p1);
    CHECK(all.tiles() == (int)want.size());
    const int n = std::max(1, all.tiles());
    std::vector<int> got;
    for (int ka = 0; ka < n;) {
        const int kb = std::min(n, ka + rnd(1, std::max(1, n / 3)));
        Reach<STEP> part = all;
        part.upto(kb);
        Steps<STEP, 1> s;
        s.enter(part, ka);
        const size_t before = got.size();
        while (s.next()) got.push_back(s.j);
        CHECK(want.empty() ? got.empty() : (int)(got.size() - before) == kb - ka && got[before] == all.key(ka));
        ka = kb;
    }
    CHECK(got == want);
    got.clear();
    for (int w = 0; w < 4; w++) {
        Steps<STEP, 4> s;
        s.enter(all, w);
        while (s.next()) got.push_back(s.j);
    }
    std::sort(got.begin(), got.end());
    CHECK(got == want);
    Reach<STEP> far = all;                            // a bound past every tile
    far.upto(0xffffff);
    CHECK(far.hi == all.hi);
}
int main() {
    for (int i = 0; i < 20000; i++) {
        PagedArgs a{};
        a.shift = rnd(4, 8);
        a.M = rnd(1, 4000 >> a.shift);
        a.N = 1000;
        const int end = rnd(0, 3) ? rnd(0, a.M << a.shift) : rnd(0, 9000), n = rnd(1, rnd(0, 1) ? 3 : 400);
        a.W = rnd(0, 3) ? rnd(1, rnd(0, 1) ? 40 : 2000) : 1 << 30;
        const Seq x = make_seq(a, 5, 5 + n, end, rnd(0, 3) ? rnd(-3, rnd(0, 1) ? 100 : 5000) : rnd(0, 1) ? INT_MIN : INT_MAX);
        const int p0 = x.end - x.n + rnd(0, x.n - 1), p1 = std::min(x.end - 1, p0 + rnd(0, 40));
        look<32>(a, x, p0, p1);
        look<64>(a, x, p0, p1);
        // no unit has more tiles than the number that all units of a sequence of few rows have
        const int most = std::max(1, Reach<32>(a, x, x.end - x.n, x.end - 1).tiles());
        CHECK((Reach<32>(a, x, p0, p1).tiles() <= most));
    }
    // the far ends: no sum leaves 32 bits (an overflow traps)
    for (int pre : {INT_MIN, -1, 0, 1, 1 << 29, INT_MAX})
        for (int W : {1, 2, 1 << 29, 1 << 30})
            for (int end : {INT_MIN, 0, 1, 1 << 29, (1 << 30) - 1, INT_MAX}) {
                PagedArgs a{};
                a.shift = 12; a.M = 0x3fffffff >> 12; a.N = 1 << 20; a.W = W;
                const Seq x = make_seq(a, 0, 1 << 20, end, pre);
                for (int p0 : {x.end - x.n, x.end - 1}) {
                    Reach<64> r(a, x, p0, x.end - 1);
                    CHECK(r.tiles() >= 0 && r.tiles() <= (1 << 24) && r.key(0xffffff - 1) >= 0);
                    r.upto(0xffffff);
                    Steps<64, 4> s;
                    s.enter(r, std::max(0, r.tiles() - 2));
                    for (int i = 0; i < 3 && s.next(); i++) CHECK(s.j >= 0 && s.j < x.klen);
                }
            }
}
""")


def test_equal_shares_meet_end_to_end(tmp_path):
    _run(tmp_path, """
int main() {
    for (int i = 0; i < 3000; i++) {
        const int G = rnd(1, 2048), total = rnd(G, rnd(0, 1) ? 20000 : 0x3fffffff);
        const Shares s(total, G);
        CHECK(s.begin(0) == 0 && s.begin(G) == total && s.owner(0) == 0 && s.owner(total - 1) == G - 1);
        for (int k = 0; k < 20; k++) {
            const int w = rnd(0, G - 1);
            CHECK(s.begin(w) < s.begin(w + 1) && s.owner(s.begin(w)) == w && s.owner(s.begin(w + 1) - 1) == w);
        }
    }
}
""")
