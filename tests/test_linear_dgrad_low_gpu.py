"""Data gradients of bf16 layers whose gradient comes with a low part: those of the unrounded gradient.  Bounds as in
test_linear_gpu.py."""
import math

import pytest
import torch

from test_linear_gpu import BF16, BWD_SHAPES, SHAPES, Framed, half_step, near, rnd, slope, value
from test_linear_walk_gpu import SIZES, normal

pytestmark = pytest.mark.gpu


def near_unrounded(dx, dpre, extra, w, what, residual=None):
    """dx = dpre w (+ residual), dpre in fp64 with what it may be off: rounded to bf16 twice (2^-16 left of it), and dx once."""
    u, n = half_step(BF16), dpre.shape[1]
    wd, size = w.double(), dpre.abs() + extra
    ref = dpre @ wd
    tol = (extra + 2.0 ** -16 * size) @ wd.abs() + (2 * n + 8) * 2.0 ** -23 * (1 + u) * (size @ wd.abs())
    if residual is not None:
        ref = ref + residual.double()
        tol = tol + 2.0 ** -23 * ref.abs()
    near(dx, ref, tol + u * (ref.abs() + tol), what)


@pytest.mark.parametrize("M,K,N", BWD_SHAPES)
def test_data_gradients_of_backward_passes(ctx, M, K, N):
    """linear_bwd and gated_linear_bwd with dpre_low: dx is that of the unrounded gradient, as dw is."""
    from sirius_amd import ops
    x, w = rnd(M, K, dtype=BF16, seed=1), rnd(N, K, dtype=BF16, seed=2, std=1 / math.sqrt(K))
    dy, pre, res = rnd(M, N, dtype=BF16, seed=3), rnd(M, N, dtype=BF16, seed=4, std=2.0), rnd(M, K, dtype=BF16, seed=5)
    dx, dpre, low, dw = torch.empty_like(x), torch.empty_like(dy), torch.empty_like(dy), torch.empty(N, K, device="cuda")
    for act, residual in (("silu", None), ("gelu_tanh", res)):
        ops.linear_bwd(ctx, dy, x, w.t().contiguous(), dx, dw, act=act, pre=pre, dpre=dpre, residual=residual, dpre_low=low)
        near_unrounded(dx, dy.double() * slope(pre.double(), act), 2.0 ** -19 * dy.double().abs(), w, act, residual)
    wg, gu = rnd(2 * N, K, dtype=BF16, seed=6, std=1 / math.sqrt(K)), rnd(M, 2 * N, dtype=BF16, seed=7, std=2.0)
    dpre, low, dw = torch.empty_like(gu), torch.empty_like(gu), torch.empty(2 * N, K, device="cuda")
    ops.gated_linear_bwd(ctx, dy, x, wg.t().contiguous(), dx, dw, gu, dpre, dpre_low=low)
    d, g, up = dy.double(), gu[:, :N].double(), gu[:, N:].double()
    exact = torch.cat([d * up * slope(g, "silu"), d * value(g, "silu")], 1)
    extra = torch.cat([2.0 ** -19 * (d * up).abs(), 2.0 ** -20 * (d * g).abs()], 1) + 2.0 ** -22 * exact.abs()
    near_unrounded(dx, exact, extra, wg, "gated")
    # a gradient that comes with its low part already
    ops.linear_bwd(ctx, dpre, x, wg.t().contiguous(), dx, dw, dy_low=low, residual=res)
    near_unrounded(dx, exact, extra, wg, "chained", res)


@pytest.mark.parametrize("M,K,N", SHAPES[:-1] + SIZES)
def test_every_kernel(ctx, M, K, N):
    """A low part as large as the high one, in every kernel, where workgroups walk several tiles too; columns of wider tensors, with an
    activation's derivative and a residual in the epilogue and without."""
    from sirius_amd import ops
    u = half_step(BF16)
    w = normal(N, K, seed=2, std=1 / math.sqrt(K))
    dy, low = Framed(M, K, BF16, True, normal(M, K, seed=1)), Framed(M, K, BF16, True, normal(M, K, seed=3))
    v = dy.view.double() @ w.double().t() + low.view.double() @ w.double().t()
    e = (2 * K + 8) * 2.0 ** -23 * ((dy.view.double().abs() + low.view.double().abs()) @ w.double().abs().t())
    dx = Framed(M, N, BF16, True)
    ops.linear_dgrad(ctx, dy.view, w, dx.view, dy_low=low.view)
    near(dx.view, v, e + u * (v.abs() + e), "plain")
    dx.check("plain")
    pre, res = normal(M, N, seed=5, std=2.0), normal(M, N, seed=4)
    ops.linear_dgrad(ctx, dy.view, w, dx.view, act="silu", pre=pre, residual=res, dy_low=low.view)
    s = slope(pre.double(), "silu")
    ref = v * s + res.double()
    tol = (e + 2.0 ** -23 * v.abs()) * s.abs() + 2.0 ** -19 * (v.abs() + e) + 2.0 ** -23 * ref.abs()
    near(dx.view, ref, tol + u * (ref.abs() + tol), "dx")
    dx.check("dx")
    want = dx.view.clone()
    dx.view.copy_(pre)      # in place of the pre-activations
    ops.linear_dgrad(ctx, dy.view, w, dx.view, act="silu", pre=dx.view, residual=res, dy_low=low.view)
    assert torch.equal(dx.view, want)


def test_refusals(ctx):
    from sirius_amd import ops
    dy, w, dx = rnd(4, 64, dtype=BF16, seed=1), rnd(32, 64, dtype=BF16, seed=2), torch.empty(4, 32, dtype=BF16, device="cuda")
    for call in (lambda: ops.linear_dgrad(ctx, dy, w, dx, dy_low=dy.float()),
                 lambda: ops.linear_dgrad(ctx, dy.float(), w.float(), dx.float(), dy_low=dy.float()),
                 lambda: ops.linear_dgrad(ctx, dy, w, dx, dy_low=dy[:3]),
                 lambda: ops.linear_dgrad(ctx, dy, w, dx, dy_low=torch.zeros(4, 128, dtype=BF16, device="cuda")[:, :64])):
        with pytest.raises(AssertionError):
            call()
