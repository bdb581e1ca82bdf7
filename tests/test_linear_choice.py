"""Which kernel a linear layer's sizes lead to (recorded on the CPU, nothing runs), and that the sizes of the GPU tests reach every
kernel of every operator and type."""
import ctypes
import re

import pytest

from sirius_amd._lib import check, lib
from test_linear_edges_gpu import SHAPES as EDGES
from test_linear_gpu import BWD_SHAPES, SHAPES
from test_recorded_launches import BF16, F32, Recorder, address, dtypes, rec  # noqa: F401

X, W, Y, PRE, LOW, WS = (address(1000 * i) for i in range(1, 7))   # 250 GB apart
KERNELS = {BF16: {"rows 16x16", "split 32x32", "split 32x64", "split 64x64", "tile 128x64", "tile 128x128", "tile 256x128", "tile 256x256"},
           F32: {"rows 16x16", "split 32x32", "split 32x64", "split 64x64", "tile 128x64"}}


def launch(rec, op, dtype, M, K, N):  # noqa: F811
    rec.begin()
    L, h = lib(), rec.ctx
    if op == "fwd":
        check(L.tch_linear_fwd(h, dtype, X, K, W, Y, N, None, 0, None, 0, None, 0, M, K, N))
    elif op == "dgrad":
        check(L.tch_linear_dgrad(h, dtype, X, K, W, Y, N, 0, None, 0, None, 0, M, K, N))
    elif op == "gated_fwd":
        check(L.tch_gated_linear_fwd(h, dtype, X, K, W, Y, N, None, 4, None, 0, M, K, N))
    else:
        check(L.tch_linear_dgrad_gated(h, dtype, X, K, W, PRE, 2 * N, Y, None, 2 * N, None, None, 0, 4, M, K, N))
    out = []
    for name, groups, _ in rec.end():
        kind, mode, tile = re.match(r"linear_(\w+)_kernel<\w+,(\w+),(\d+x\d+)", name).groups()
        assert mode == op
        out.append((f"{kind} {tile}", groups))
    return out


@dtypes
@pytest.mark.parametrize("op", ["fwd", "dgrad", "gated_fwd", "gated_dgrad"])
def test_every_kernel_is_reached_and_tested(rec, op, dtype):  # noqa: F811
    want = set(KERNELS[dtype])
    if op == "gated_fwd":
        want.discard("rows 16x16")
    all_launches = [launch(rec, op, dtype, M, K, N) for M, K, N in SHAPES + EDGES + [(m, n, k) for m, k, n in BWD_SHAPES]]
    assert {kernel for launches in all_launches for kernel, _ in launches} == want
    assert max(len(launches) for launches in all_launches) == 2     # rows behind the last whole round


def test_choice(rec):  # noqa: F811
    """Both sides of the rule, at sizes that were measured."""
    assert launch(rec, "fwd", BF16, 1, 4096, 4096) == [("rows 16x16", 256)]
    assert launch(rec, "fwd", BF16, 512, 8192, 1024)[0][0] == "split 32x64"
    assert launch(rec, "fwd", BF16, 1024, 1024, 1024)[0][0] == "split 64x64"
    assert launch(rec, "fwd", BF16, 512, 4096, 4096) == [("tile 128x64", 256)]
    assert launch(rec, "fwd", BF16, 512, 8192, 8192) == [("tile 128x128", 256)]
    assert launch(rec, "fwd", BF16, 4096, 1024, 4096) == [("tile 256x256", 256)]
    assert launch(rec, "fwd", F32, 2048, 1024, 2048) == [("tile 128x64", 512)]
    assert launch(rec, "fwd", F32, 1568, 1024, 4096) == [("tile 128x64", 768), ("split 32x32", 128)]
    assert launch(rec, "fwd", F32, 512, 2048, 1024) == [("split 32x64", 256)]


def test_weight_gradients_are_cut_to_whole_rounds(rec):  # noqa: F811
    def wgrad(M, K, N, low):
        rec.begin()
        need = lib().tch_linear_wgrad_workspace_bytes(M, K, N)
        check(lib().tch_linear_wgrad(rec.ctx, X, None, Y, LOW if low else None, W, None, 0, M, K, N, WS, need))
        return rec.end()
    for M, K, N, tiles in ((1803, 5120, 3312, 260), (2319, 3976, 8736, 560)):
        (name, groups, _), (add, parts, _) = wgrad(M, K, N, True)
        assert "256x256" in name and "sum" in add and groups == 256 and parts == tiles % 256 * 32
    assert len(wgrad(2048, 2048, 8192, True)) == len(wgrad(2048, 2048, 8192, False)) == 1          # 256 whole tiles
