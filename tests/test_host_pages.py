"""CPU checks of what the attention over pages enqueues at sizes that no other test reaches: the library runs against the stand-in for the HIP runtime
(hip_stub.c), which records launches instead of executing them."""
import json
import subprocess
import sys

import pytest

import slotscan_lib as L
from test_host_streams import stub                       # noqa: F401 (a fixture)

_BODY = """
import ctypes, json, sys
stub = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
stub.stub_log.restype = ctypes.c_char_p
lib = ctypes.CDLL(sys.argv[2])
vp, i64, i32, f32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float
lib.slotattn_pages.argtypes = [vp, i64, i64] + [vp, i64, i64, i64] * 2 + [i32, vp, i64, vp, vp] + [i64] * 9 + [f32, i64, f32] + [vp] * 5
lib.slotattn_pages_workspace.argtypes = [i64] * 9 + [i32]
lib.slotattn_pages_workspace.restype = ctypes.c_size_t
N, R, M, page, Hq, Hk, D, most = map(int, sys.argv[3:])
p = 1 << 20
rc = lib.slotattn_pages(p, D, Hq * D, p, Hk * page * D, page * D, D, p, Hk * page * D, page * D, D, 1, p, M, p, p, N, R, M, 9, page, Hq, Hk, D, most,
                        0.125, 2 ** 31 - 1, 0.0, None, None, p, p, None)
log = [l.split() for l in stub.stub_log().decode().splitlines()]
print(json.dumps([rc, lib.slotattn_pages_workspace(N, R, M, page, Hq, Hk, D, most, 2 ** 31 - 1, 0),
                  [[l[2], int(l[4]), int(l[5])] for l in log if l[1] == "launch"]]))
"""


def _launches(stub, *sizes):
    r = subprocess.run([sys.executable, "-c", _BODY, stub, L.LIB_PATH] + [str(x) for x in sizes], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr[-2000:]
    rc, ws, log = json.loads(r.stdout.splitlines()[-1])
    return rc, ws, [([k for k in ("pages_plan", "pages_many", "pages_few", "pages_join_few", "pages_join") if k in name][0], x, y) for name, x, y in log]


@pytest.mark.parametrize("R,Hk,few", [(32, 4, True), (1 << 22, 128, True), (1 << 23, 128, False), (1 << 24, 64, False), (1 << 24, 128, False), (1 << 24, 256, False)])
def test_pairs_of_row_and_head_stay_in_32_bits(stub, R, Hk, few):
    """The join of few rows numbers the (row, head) pairs, and their pieces, in 32 bits: from 2^30 on the rows take the way of many."""
    rc, ws, log = _launches(stub, 16, R, 64, 64, Hk, Hk, 64, 1)
    assert rc == 0
    if few:
        assert [x[0] for x in log] == ["pages_few", "pages_join_few"] and ws >= R * Hk * 8
    else:
        assert [x[0] for x in log] == ["pages_plan", "pages_many", "pages_join"] and ws < 1 << 30
    assert all(0 < x < 1 << 31 and 0 < y < 1 << 16 for _, x, y in log)
