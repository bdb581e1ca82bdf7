"""The derivative passes with a bias gradient at the C ABI, without a GPU: what is refused, and how the rows are cut."""
import ctypes

import pytest

from sirius_amd._lib import check, lib
from test_linear_refusals import A, B, BF16, C, D, F32, refused
from test_recorded_launches import address, rec  # noqa: F401

ODD = ctypes.c_void_p(0x10002)


def at(byte):
    return ctypes.c_void_p(0x100000 + byte)


def test_refused():
    def act_bwd(dbias=D, ws=None, ws_bytes=0, M=64, N=64, act=4, dz=C):
        return refused("tch_act_bwd_bias", None, BF16, A, N, B, N, dz, None, N, dbias, 0, act, M, N, ws, ws_bytes)
    act_bwd(act=5)
    act_bwd(M=-1)
    act_bwd(N=4)
    assert "4-byte" in act_bwd(dbias=ODD)
    assert "4-byte" in act_bwd(ws=ODD)
    far = [address(1000 * i) for i in range(1, 6)]
    need = lib().tch_act_bwd_workspace_bytes(BF16, 9000, 4096, 0)
    assert need > 0
    assert "workspace" in refused("tch_act_bwd_bias", None, BF16, far[0], 4096, far[1], 4096, far[2], None, 4096, far[3], 0, 4, 9000, 4096, far[4], need - 1)
    assert "overlaps" in refused("tch_act_bwd_bias", None, BF16, far[0], 4096, far[1], 4096, far[2], None, 4096, far[3], 0, 4, 9000, 4096, far[1], need)
    assert "overlaps" in act_bwd(dz=at(0), dbias=at(64))
    assert "low part" in refused("tch_gated_act_bwd_bias", None, F32, A, 64, B, 128, C, D, 128, None, 0, None, 0, 4, 4, 64, None, 0)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("gated", [0, 1])
def test_rows_are_cut_for_the_chip(rec, dtype, gated):  # noqa: F811
    """The launches' grids cover all columns and rows, and the workspace their sums."""
    E = 8 if dtype == BF16 else 4
    X, Z, O, S, W = (address(1000 * i) for i in range(1, 6))
    for M, N in ((1, 8), (16, 64), (17, 64), (1023, 2736), (8192, 4096), (100_003, 16), (5, 66_000), (2_000_000, 64)):
        need = lib().tch_act_bwd_workspace_bytes(dtype, M, N, gated)
        for ws in (W, None):
            rec.begin()
            args = (S, 0) if not gated else (None, 0, S, 0)
            fn = lib().tch_gated_act_bwd_bias if gated else lib().tch_act_bwd_bias
            check(fn(rec.ctx, dtype, X, N, Z, N * (1 + gated), O, None, N * (1 + gated), *args, 4, M, N, ws, need if ws else 0))
            launches = rec.end()
            name, groups, _ = launches[0]
            assert name.startswith("act_bwd_sum_kernel")
            chunks = N // E
            lanes = min(1 << max(chunks - 1, 0).bit_length(), 32 if ws else 8)
            col_blocks = -(-chunks // lanes)
            blocks = groups // col_blocks
            assert groups == col_blocks * blocks and blocks <= 1024
            assert need == 0 if ws and blocks == 1 else not ws or need == blocks * N * (1 + gated) * 4
            assert len(launches) == 1 + (blocks > 1) and (ws or blocks == 1)
            if blocks > 1:
                assert launches[1][:2] == ("act_bwd_bias_kernel", -(-N * (1 + gated) // 32))
    assert lib().tch_act_bwd_workspace_bytes(dtype, 4096, 4 if E == 8 else 2, gated) == 0
    assert lib().tch_act_bwd_workspace_bytes(2, 8, 8, 0) == 0 and lib().tch_act_bwd_workspace_bytes(dtype, 0, 8, 0) == 0
