"""What the 8-bit activations refuse at the C ABI and in the wrapper, without a GPU."""
import ctypes

import pytest
import torch

BF16, F32 = 1, 0
A, B, C, D = (ctypes.c_void_p(0x1000000 * i) for i in range(1, 5))
ODD = ctypes.c_void_p(0x1000008)


def last():
    from sirius_amd._lib import lib
    return (lib().tch_last_error() or b"").decode()


def pack(dtype=BF16, x=A, ldx=64, data=B, scales=C, format=0, h=None, ldh=0, act=0, M=4, width=64):
    from sirius_amd._lib import lib
    return lib().tch_pack8(None, dtype, x, ldx, data, scales, format, h, ldh, act, M, width)


def unpack(dtype=BF16, data=B, scales=C, format=0, x=A, ldx=64, M=4, width=64):
    from sirius_amd._lib import lib
    return lib().tch_unpack8(None, dtype, data, scales, format, x, ldx, M, width)


@pytest.mark.parametrize("change", [
    dict(dtype=2), dict(format=2), dict(format=-1), dict(M=-1), dict(M=1 << 31), dict(width=0), dict(width=60), dict(dtype=F32, width=62), dict(M=1 << 30, width=1 << 10, ldx=1 << 10),
    dict(x=None), dict(data=None), dict(scales=None), dict(x=ODD), dict(data=ODD), dict(ldx=56), dict(ldx=68), dict(h=D, ldh=56), dict(h=ODD, ldh=64),
    dict(act=9, h=D, ldh=64), dict(data=A), dict(scales=A), dict(scales=B), dict(h=B, ldh=64), dict(h=A, ldh=128)], ids=str)
def test_pack(change):
    assert pack(**change) == -22 and "pack8" in last()


@pytest.mark.parametrize("change", [dict(dtype=2), dict(format=2), dict(M=-1), dict(width=4), dict(x=None), dict(data=None), dict(scales=None), dict(x=ODD),
                                    dict(data=ODD), dict(ldx=32), dict(x=B), dict(x=C)], ids=str)
def test_unpack(change):
    assert unpack(**change) == -22 and "unpack8" in last()


def test_no_rows_is_no_error():
    assert pack(M=0, x=None, data=None, scales=None) == 0 and unpack(M=0, x=None, data=None, scales=None) == 0


def test_wrapper():
    from sirius_amd import ops
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8)  # noqa: E731
    with pytest.raises(ValueError, match="format"):
        ops.Packed8(u8(4, 64), u8(4, 2), "int4")
    for data, scales in ((u8(4, 64), u8(4, 3)), (u8(4, 65), u8(4, 2)), (u8(64), u8(2)), (u8(4, 64).char(), u8(4, 2)), (u8(64, 4).t(), u8(4, 2)), (u8(4, 64), u8(3, 2))):
        with pytest.raises(AssertionError):
            ops.Packed8(data, scales)
    p = ops.Packed8.empty(3, 70, "e4m3", device="cpu")
    assert p.scales.shape == (3, 3) and p.nbytes() == 219 and tuple(p.shape) == (3, 70)


def act(dtype=BF16, dy=A, lddy=64, data=B, scales=C, format=0, dz=D, dz_low=None, lddz=64, h=None, ldh=0, dbias=None, accumulate=0, gated=0, act=4, M=4, N=64,
        ws=None, ws_bytes=0):
    from sirius_amd._lib import lib
    return lib().tch_act_bwd_packed(None, dtype, dy, lddy, data, scales, format, dz, dz_low, lddz, h, ldh, dbias, accumulate, gated, act, M, N, ws, ws_bytes)


@pytest.mark.parametrize("change", [
    dict(dtype=2), dict(format=2), dict(format=-1), dict(act=7), dict(M=-1), dict(N=60), dict(N=0), dict(dy=None), dict(data=None), dict(scales=None), dict(dz=None),
    dict(dtype=F32, dz_low=ctypes.c_void_p(0x5000000)), dict(dy=ODD), dict(data=ODD), dict(dz=ODD), dict(lddy=56), dict(gated=1), dict(h=ODD, ldh=64), dict(h=D, ldh=64),
    dict(dz=B), dict(dz=C), dict(h=B, ldh=64), dict(h=A, ldh=64), dict(dbias=B), dict(M=1 << 30, N=1024, lddy=1024, lddz=1024)], ids=str)
def test_derivatives(change):
    assert act(**change) == -22 and "act_bwd" in last()


def test_weight_gradient_wrapper():
    from sirius_amd import ops
    packed, dy = ops.Packed8.empty(16, 64, device="cpu"), torch.zeros(16, 32, dtype=torch.bfloat16)
    assert ops.linear_wgrad_packed_workspace_bytes(packed, dy) >= 4
    assert ops.linear_wgrad_packed_workspace_bytes(ops.Packed8.empty(0, 64, device="cpu"), dy[:0]) >= 4

    class Here:
        handle = None

        class stream:
            device = torch.device("cpu")
    with pytest.raises(AssertionError, match="workspace"):
        ops.linear_wgrad_packed(Here, packed, dy, torch.zeros(32, 64))
    with pytest.raises(AssertionError, match="workspace"):
        ops.linear_wgrad_packed(Here, packed, dy, torch.zeros(32, 64), workspace=torch.zeros(2, dtype=torch.uint8))


@pytest.mark.parametrize("which", ["data", "scales"])
def test_a_workspace_over_what_is_kept(which):
    """The weight gradient's own part of the workspace comes behind the fetched input: it is not over the kept numbers either."""
    from sirius_amd import ops

    class Here:
        handle = None

        class stream:
            device = torch.device("cpu")
    dy = torch.zeros(16, 32, dtype=torch.bfloat16)
    need = ops.linear_wgrad_packed_workspace_bytes(ops.Packed8.empty(16, 64, device="cpu"), dy)
    room = torch.zeros(need + 1024, dtype=torch.uint8)
    data, scales = torch.zeros(16, 64, dtype=torch.uint8), torch.zeros(16, 2, dtype=torch.uint8)
    if which == "data":
        data = room[need - 16:need - 16 + 1024].view(16, 64)
    else:
        scales = room[need - 16:need + 16].view(16, 2)
    with pytest.raises(AssertionError, match=f"overlaps packed {which}"):
        ops.linear_wgrad_packed(Here, ops.Packed8(data, scales), dy, torch.zeros(32, 64), workspace=room[:need])
