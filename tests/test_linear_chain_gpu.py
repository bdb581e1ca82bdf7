"""A chain of bf16 layers that are not gated: the data gradient of a layer ends in the derivative of the activation in front, and keeps
what rounding takes off it, so that every gradient behind is that of the unrounded one.  Bounds as in test_linear_gpu.py; a value in two
parts is left 2^-16 off."""
import math

import pytest
import torch

from test_linear_dgrad_low_gpu import near_unrounded
from test_linear_gpu import BF16, F32, SHAPES, Framed, half_step, near, product, rnd, slope, value
from test_linear_walk_gpu import SIZES, normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,K,N", SHAPES[:-1] + SIZES)
def test_low_part_of_a_data_gradient(ctx, M, K, N):
    """In every kernel, with a low part of the incoming gradient and without: dx and its low part hold the unrounded gradient, dx by
    itself the rounded one, and nothing around either is written."""
    from sirius_amd import ops
    w, dy, low, res = normal(N, K, seed=2, std=1 / math.sqrt(K)), normal(M, K, seed=1), normal(M, K, seed=3), normal(M, N, seed=4)
    pre = normal(M, N, seed=5, std=2.0)
    s = slope(pre.double(), "gelu")
    for dy_low, act, residual in ((None, "gelu", None), (low, "gelu", res), (None, "none", res)):
        v, e = product(dy, w)
        if dy_low is not None:
            v, e = v + dy_low.double() @ w.double().t(), 2 * (e + product(dy_low, w)[1])
        dx, dx_low, alone = Framed(M, N, BF16, True), Framed(M, N, BF16, True), torch.empty(M, N, dtype=BF16, device="cuda")
        kw = dict(act=act, pre=pre if act != "none" else None, residual=residual, dy_low=dy_low)
        ops.linear_dgrad(ctx, dy, w, dx.view, dx_low=dx_low.view, **kw)
        ref, tol = v, e
        if act != "none":
            ref, tol = v * s, (e + 2.0 ** -23 * v.abs()) * s.abs() + 2.0 ** -19 * (v.abs() + e)
        if residual is not None:
            ref = ref + residual.double()
            tol = tol + 2.0 ** -23 * ref.abs()
        near(dx.view.double() + dx_low.view.double(), ref, tol + 2.0 ** -16 * (ref.abs() + tol), "dx and its low part")
        dx.check("dx")
        dx_low.check("dx_low")
        ops.linear_dgrad(ctx, dy, w, alone, **kw)
        # (the products' order may differ: the kernel is chosen by its time, and a low part has kernels of its own)
        near(alone, ref, tol + half_step(BF16) * (ref.abs() + tol), "dx alone")


def test_low_parts_of_values_that_are_not_finite(ctx):
    from sirius_amd import ops
    dy, wt = torch.ones(3, 8, dtype=BF16, device="cuda"), torch.zeros(16, 8, dtype=BF16, device="cuda")
    wt[0, 0], wt[1, 0], wt[2, 0], wt[3, 0] = math.inf, -math.inf, math.nan, 3e38
    dx, low = torch.empty(3, 16, dtype=BF16, device="cuda"), torch.empty(3, 16, dtype=BF16, device="cuda")
    ops.linear_dgrad(ctx, dy, wt, dx, dx_low=low)
    assert bool((dx[:, 0] == math.inf).all() and (dx[:, 1] == -math.inf).all() and dx[:, 2].isnan().all())
    assert bool((low[:, :3] == 0).all()) and bool(low.isfinite().all())


@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("M,C,F", [(5, 72, 40), (130, 264, 520), (1100, 512, 1544), (2100, 520, 2056)])
def test_block(ctx, M, C, F, act):
    """Two layers, an activation between them and the block's residual, forward and back."""
    from sirius_amd import ops
    u = half_step(BF16)
    x, dy = rnd(M, C, dtype=BF16, seed=1), rnd(M, C, dtype=BF16, seed=6)
    w, wd = rnd(F, C, dtype=BF16, seed=3, std=1 / math.sqrt(C)), rnd(C, F, dtype=BF16, seed=4, std=1 / math.sqrt(F))
    bias = rnd(F, dtype=F32, seed=5)

    def new(*shape, dtype=BF16):
        return torch.empty(shape, dtype=dtype, device="cuda")
    h, pre, y, dpre, dpre_low, dx = new(M, F), new(M, F), new(M, C), new(M, F), new(M, F), new(M, C)
    dw, db, dwd = new(F, C, dtype=F32), new(F, dtype=F32), new(C, F, dtype=F32)
    ws, wsd = (new(ops.linear_bwd_workspace_bytes(*a), dtype=torch.uint8) for a in ((x, F), (h, C)))
    ops.linear_fwd(ctx, x, w, h, bias=bias, act=act, pre=pre)
    ops.linear_fwd(ctx, h, wd, y, residual=x)
    ops.linear_dgrad(ctx, dy, wd.t().contiguous(), dpre, act=act, pre=pre, dx_low=dpre_low)
    ops.linear_wgrad(ctx, h, dy, dwd, workspace=wsd)
    ops.linear_bwd(ctx, dpre, x, w.t().contiguous(), dx, dw, dbias=db, residual=dy, workspace=ws, dy_low=dpre_low)
    z, e = product(x, w)
    z, e = z + bias.double(), e + 2.0 ** -23 * (z.abs() + bias.abs().double())
    near(pre, z, e + u * (z.abs() + e), "pre")
    ref, tol = value(z, act), 1.2 * e + 2.0 ** -20 * z.abs()
    near(h, ref, tol + u * (ref.abs() + tol), "h")
    v, ev = product(h, wd)
    ref = v + x.double()
    near(y, ref, ev + u * (ref.abs() + ev) + 2.0 ** -23 * ref.abs(), "y")
    ref = dy.double().t() @ h.double()
    near(dwd, ref, (M + 64) * 2.0 ** -23 * (dy.double().abs().t() @ h.double().abs()) + 1e-30, "dw_down")
    v, ev = product(dy, wd.t())
    s = slope(pre.double(), act)
    exact, extra = v * s, (ev + 2.0 ** -23 * v.abs()) * s.abs() + 2.0 ** -19 * (v.abs() + ev)
    near_unrounded(dx, exact, extra, w, "dx", dy)
    off = extra + 2.0 ** -16 * (exact.abs() + extra)
    sums = (2 * M + 64) * 2.0 ** -23
    near(dw, exact.t() @ x.double(), off.t() @ x.double().abs() + sums * (exact.abs().t() @ x.double().abs()) + 1e-30, "dw")
    near(db, exact.sum(0), off.sum(0) + sums * exact.abs().sum(0) + 1e-30, "db")
