"""That the sizes of test_linear_walk_gpu.py lead to what they are there for (recorded on the CPU, nothing runs): in every mode each
bf16 tile kernel with more tiles than workgroups, and among those reductions of two, three and five or more steps."""
import ctypes
import re

import pytest

from sirius_amd._lib import LaunchStat, check, lib
from test_linear_choice import PRE, W, X, Y
from test_linear_walk_gpu import GATED, SIZES
from test_recorded_launches import BF16, rec  # noqa: F401


def walks(rec, mode, M, K, N):  # noqa: F811
    """(tile, steps) of the launches of one call in which workgroups walk."""
    rec.begin()
    L, h = lib(), rec.ctx
    if mode == "fwd":
        check(L.tch_linear_fwd(h, BF16, X, K, W, Y, N, None, 0, None, 0, None, 0, M, K, N))
    elif mode == "dgrad":
        check(L.tch_linear_dgrad(h, BF16, X, K, W, Y, N, 0, None, 0, None, 0, M, K, N))
    elif mode == "gated_fwd":
        check(L.tch_gated_linear_fwd(h, BF16, X, K, W, Y, N, None, 4, None, 0, M, K, N))
    else:
        check(L.tch_linear_dgrad_gated(h, BF16, X, K, W, PRE, 2 * N, Y, None, 2 * N, None, None, 0, 4, M, K, N))
    check(L.tch_program_end_record(h))
    launches, n = (LaunchStat * 2)(), ctypes.c_int64()
    check(L.tch_program_launches(rec.progs[-1], launches, 2, ctypes.byref(n)))
    out = set()
    for r in launches[:n.value]:
        kind, bm, bn = re.match(r"linear_(\w+)_kernel<\w+,\w+,(\d+)x(\d+)", r.name.decode()).groups()
        rows = round(r.flops / ((4 if mode == "gated_fwd" else 2) * N * K))
        cols = int(bn) // (2 if mode == "gated_fwd" else 1)
        if kind == "tile" and -(-rows // int(bm)) * -(-N // cols) > r.workgroups:
            out.add((f"{bm}x{bn}", -(-K // 64)))
    return out


@pytest.mark.parametrize("mode", ["fwd", "dgrad", "gated_fwd", "gated_dgrad"])
def test_what_the_sizes_reach(rec, mode):  # noqa: F811
    got = set()
    for size in GATED if mode == "gated_fwd" else SIZES:
        found = walks(rec, mode, *size)
        assert found, size
        got |= found
    steps = {tile: {s for t, s in got if t == tile} for tile in ("256x256", "256x128", "128x128", "128x64")}
    assert {2, 3} <= steps["256x256"] and max(steps["256x256"]) >= 5
    assert {1, 2, 3} <= steps["256x128"] and max(steps["256x128"]) >= 5
    assert {1, 3} <= steps["128x128"] and max(steps["128x128"]) >= 5
    assert max(steps["128x64"]) >= 5
