"""Data gradients with a low part at the C ABI, without a GPU: what is refused, and that the GPU tests' sizes reach every kernel."""
import ctypes
import re

from sirius_amd._lib import check, lib
from test_linear_choice import KERNELS, LOW, W, X, Y
from test_linear_gpu import SHAPES
from test_linear_refusals import A, B, C, D, F32, ODD, refused
from test_linear_walk_gpu import SIZES
from test_recorded_launches import BF16, rec  # noqa: F401


def test_refused():
    def at(byte):
        return ctypes.c_void_p(0x100000 + byte)

    def dgrad(dtype=BF16, dy=A, low=D, lddy=64, w=B, dx=C, dx_low=None, lddx=32, act=0, pre=None, ldp=0, res=None, ldr=0, M=4, K=64, N=32):
        return refused("tch_linear_dgrad_low", None, dtype, dy, low, lddy, w, dx, dx_low, lddx, act, pre, ldp, res, ldr, M, K, N)
    assert "low part" in dgrad(dtype=F32)
    assert "low part" in dgrad(dtype=F32, low=None, dx_low=D)
    dgrad(dx_low=ODD)
    assert "overlaps" in dgrad(dx=at(0), dx_low=at(0))
    assert "overlaps" in dgrad(low=at(0), lddy=128, dx_low=at(96), lddx=128)
    dgrad(low=ODD)
    dgrad(dy=None)
    assert "pre-activations" in dgrad(act=4)
    assert "overlaps" in dgrad(low=at(0), dx=at(16), lddx=64)
    assert "overlaps" in dgrad(low=at(0), dx=at(0), lddx=64, N=64)


def test_every_kernel_is_reached(rec):  # noqa: F811
    got = set()
    for M, K, N in SHAPES[:-1] + SIZES:
        rec.begin()
        check(lib().tch_linear_dgrad_low(rec.ctx, BF16, X, LOW, K, W, Y, None, N, 0, None, 0, None, 0, M, K, N))
        for name, _, _ in rec.end():
            kind, tile = re.match(r"linear_(\w+)_kernel<bf16,dgrad_low,(\d+x\d+)", name).groups()
            got.add(f"{kind} {tile}")
    assert got == KERNELS[BF16]
