"""What the rotary positions refuse, and how their frequencies are made, without a GPU."""
import ctypes
import math

import pytest
import torch

BF16, F32 = 1, 0
A, B, C, D = (ctypes.c_void_p(0x100000 * i) for i in range(1, 5))


def call(dtype=BF16, x=A, ldx=128, y=B, ldy=128, freqs=C, positions=None, wide=1, start=0, seq=4, rows=4, heads=2, head_dim=64, rot=64, layout=0):
    from sirius_amd._lib import lib
    rc = lib().tch_rotary(None, dtype, x, ldx, y, ldy, freqs, positions, wide, start, seq, rows, heads, head_dim, rot, layout, 1.0, 0)
    return rc, (lib().tch_last_error() or b"").decode()


@pytest.mark.parametrize("change", [
    dict(dtype=2), dict(rows=-1), dict(rows=1 << 31), dict(heads=0), dict(head_dim=0), dict(heads=1 << 20, head_dim=1 << 12, rot=64), dict(rot=0),
    dict(rot=7), dict(rot=66), dict(head_dim=8192, heads=1, rot=4098, ldx=8192, ldy=8192), dict(seq=0), dict(seq=1 << 31), dict(start=1 << 41), dict(x=None),
    dict(y=None), dict(freqs=None), dict(ldx=127), dict(ldy=64), dict(ldx=-128), dict(x=ctypes.c_void_p(0x100001)), dict(dtype=F32, x=ctypes.c_void_p(0x100002)),
    dict(freqs=ctypes.c_void_p(0x300004)), dict(positions=ctypes.c_void_p(0x400004)), dict(y=ctypes.c_void_p(0x100010)), dict(y=A, ldy=256), dict(freqs=B),
    dict(positions=B)], ids=str)
def test_refused(change):
    rc, message = call(**change)
    assert rc == -22 and "rotary" in message


def test_no_rows_is_no_error():
    assert call(rows=0, x=None, y=None, freqs=None)[0] == 0


def test_wrapper_refuses():
    from sirius_amd import ops
    with pytest.raises(ValueError, match="layout"):
        ops.rotary_fwd(None, torch.zeros(1, 64), None, None, 64, layout="quarter")
    with pytest.raises(AssertionError, match="whole heads"):
        ops.rotary_fwd(None, torch.zeros(1, 65), None, None, 64)
    for bad in (dict(rot=7), dict(rot=0), dict(rot=8, factor=0.0), dict(rot=8, base=-1.0), dict(rot=8, trained=0), dict(rot=8, trained=8, slow=4.0, fast=4.0)):
        with pytest.raises(ValueError):
            ops.rotary_freqs(**bad)


def test_frequencies():
    from sirius_amd import ops
    f = ops.rotary_freqs(64)
    for i in range(32):
        assert abs(f[i].item() - 10000.0 ** (-i / 32)) <= 2.0 ** -50 * f[i].item()
    assert torch.equal(ops.rotary_freqs(64, factor=4.0), f / 4.0)
    g = ops.rotary_freqs(64, factor=4.0, trained=2048, slow=1.0, fast=32.0)
    for i in range(32):
        turns = 2048 * f[i].item() / (2 * math.pi)
        share = min(max((turns - 1.0) / 31.0, 0.0), 1.0)
        assert abs(g[i].item() - f[i].item() * (share + (1 - share) / 4.0)) <= 2.0 ** -50 * f[i].item()
    assert g[0] == f[0] and g[-1] == f[-1] / 4.0


@pytest.mark.parametrize("seq", [0, -4])
def test_a_length_that_is_none_is_not_taken_for_one(seq, monkeypatch):
    from sirius_amd import ops

    class Here:
        handle = None

        class stream:
            device = torch.device("cpu")
    monkeypatch.setattr(ops, "_matrix", lambda ctx, name, t, *more: (A if name == "x" else B, 128, 4))
    monkeypatch.setattr(ops, "_p", lambda t: None if t is None else C)
    x = torch.zeros(4, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="length of a sequence"):
        ops.rotary_fwd(Here, x, x, torch.zeros(32, dtype=torch.float64), 64, seq=seq)


@pytest.mark.parametrize("ld", [0, 8, 128])
@pytest.mark.parametrize("dtype,shift", [(BF16, 16), (BF16, -16), (F32, 64), (F32, 256)], ids=str)
def test_one_row_over_another(ld, dtype, shift):
    """A single row needs no distance to the next one, 0 among them: two of them that overlap are refused all the same."""
    rc, message = call(dtype=dtype, ldx=ld, ldy=ld, y=ctypes.c_void_p(0x100000 + shift), rows=1, seq=1)
    assert rc == -22 and "overlaps" in message
