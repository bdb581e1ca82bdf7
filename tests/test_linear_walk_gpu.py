"""The linear layers' persistent kernels where a workgroup walks several output tiles: the next tile's operands are requested ahead of
an epilogue and waited for behind its stores.  Every mode and tile, reductions of one, two, three and more steps, last tiles that
are ragged on every side, with everything an epilogue can read and write and with nothing of it, against fp64 under the bounds that
test_linear_gpu.py derives."""
import math

import pytest
import torch

from test_linear_gpu import BF16, F32, Framed, half_step, near, product, slope, value

pytestmark = pytest.mark.gpu

# rows, reduction, outputs; test_linear_walk.py holds what they lead to: each tile, walked, by steps of 64 reduction elements
SIZES = [(6489, 104, 3776), (5768, 192, 4256), (5526, 216, 4488), (5601, 328, 4408), (99334, 144, 136),
         (17076, 64, 440), (8300, 96, 1888), (14023, 136, 1048), (16658, 328, 808),
         (2333, 56, 3264), (783, 192, 8224), (1405, 304, 5424), (87298, 304, 8)]
GATED = [(2000, 104, 6312), (1961, 160, 6312), (1961, 320, 6312), (100417, 96, 72),
         (13249, 40, 272), (10287, 80, 808), (1169, 136, 6680), (15109, 328, 528),
         (305, 16, 8264), (269, 176, 10008), (284, 272, 8720), (81969, 304, 8)]


def normal(*shape, seed, std=1.0, dtype=BF16):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + sum(shape))
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


@pytest.mark.parametrize("M,K,N", SIZES)
def test_forward(ctx, M, K, N):
    from sirius_amd import ops
    u = half_step(BF16)
    x, w, bias, res = normal(M, K, seed=1), normal(N, K, seed=2, std=1 / math.sqrt(K)), normal(N, seed=3, dtype=F32), normal(M, N, seed=4)
    z0, e = product(x, w)
    y = Framed(M, N, BF16, True)
    ops.linear_fwd(ctx, x, w, y.view)
    near(y.view, z0, e + u * (z0.abs() + e), "plain")
    y.check("plain")
    pre = Framed(M, N, BF16, True)
    ops.linear_fwd(ctx, x, w, y.view, bias=bias, act="gelu_tanh", residual=res, pre=pre.view)
    e += 2.0 ** -23 * (z0.abs() + bias.abs().double())
    z = z0 + bias.double()
    near(pre.view, z, e + u * (z.abs() + e), "pre")
    ref = value(z, "gelu_tanh") + res.double()
    tol = 1.2 * e + 2.0 ** -20 * z.abs() + 2.0 ** -23 * ref.abs()
    near(y.view, ref, tol + u * (ref.abs() + tol), "y")
    y.check("y")
    pre.check("pre")


@pytest.mark.parametrize("M,K,N", SIZES)
def test_data_gradient(ctx, M, K, N):
    from sirius_amd import ops
    u = half_step(BF16)
    dy, w = normal(M, K, seed=1), normal(N, K, seed=2, std=1 / math.sqrt(K))
    v, e = product(dy, w)
    dx = Framed(M, N, BF16, True)
    ops.linear_dgrad(ctx, dy, w, dx.view)
    near(dx.view, v, e + u * (v.abs() + e), "plain")
    dx.check("plain")
    pre, res = normal(M, N, seed=5, std=2.0), normal(M, N, seed=4)
    ops.linear_dgrad(ctx, dy, w, dx.view, act="silu", pre=pre, residual=res)
    s = slope(pre.double(), "silu")
    ref = v * s + res.double()
    tol = (e + 2.0 ** -23 * v.abs()) * s.abs() + 2.0 ** -19 * (v.abs() + e) + 2.0 ** -23 * ref.abs()
    near(dx.view, ref, tol + u * (ref.abs() + tol), "dx")
    dx.check("dx")


@pytest.mark.parametrize("M,K,N", SIZES)
def test_data_gradient_through_a_gate(ctx, M, K, N):
    from sirius_amd import ops
    u = half_step(BF16)
    dy, w, pre = normal(M, K, seed=1), normal(N, K, seed=2, std=1 / math.sqrt(K)), normal(M, 2 * N, seed=5, std=2.0)
    v, e = product(dy, w)
    g, up = pre[:, :N].double(), pre[:, N:].double()
    s, a = slope(g, "silu"), value(g, "silu")
    ea = 2.0 ** -20 * g.abs()
    exact = ((slice(0, N), v * up * s, (e * s.abs() + 2.0 ** -19 * (v.abs() + e)) * up.abs()), (slice(N, 2 * N), v * a, e * a.abs() + ea * (v.abs() + e)))
    dpre = Framed(M, 2 * N, BF16, True)
    ops.linear_dgrad_gated(ctx, dy, w, pre, dpre.view, act="silu")
    for cols, ref, tol in exact:
        tol = tol + 2.0 ** -22 * ref.abs()
        near(dpre.view[:, cols], ref, tol + u * (ref.abs() + tol), "dpre")
    dpre.check("dpre")
    low, h, h_low = Framed(M, 2 * N, BF16, True), Framed(M, N, BF16, True), Framed(M, N, BF16, True)
    ops.linear_dgrad_gated(ctx, dy, w, pre, dpre.view, act="silu", h=h.view, dpre_low=low.view, h_low=h_low.view)
    for cols, ref, tol in exact:
        tol = tol + 2.0 ** -22 * ref.abs()
        near(dpre.view[:, cols].double() + low.view[:, cols].double(), ref, tol + 2.0 ** -16 * (ref.abs() + tol), "dpre and its low part")
    near(h.view.double() + h_low.view.double(), a * up, ea * up.abs() + (2.0 ** -23 + 2.0 ** -16) * (a * up).abs(), "h and its low part")
    for f, what in ((dpre, "dpre"), (low, "dpre_low"), (h, "h"), (h_low, "h_low")):
        f.check(what)


@pytest.mark.parametrize("M,K,F", GATED)
def test_gated_forward(ctx, M, K, F):
    from sirius_amd import ops
    u = half_step(BF16)
    x, w, bias = normal(M, K, seed=1), normal(2 * F, K, seed=2, std=1 / math.sqrt(K)), normal(2 * F, seed=3, dtype=F32)
    z0, e0 = product(x, w)

    def check(h, z, e):
        g, up, eg, eu = z[:, :F], z[:, F:], e[:, :F], e[:, F:]
        a = value(g, "silu")
        ref = a * up
        tol = (1.2 * eg + 2.0 ** -20 * g.abs()) * (up.abs() + eu) + a.abs() * eu + 2.0 ** -23 * ref.abs()
        near(h.view, ref, tol + u * (ref.abs() + tol), "h")
        h.check("h")
    h, pre = Framed(M, F, BF16, True), Framed(M, 2 * F, BF16, True)
    ops.gated_linear_fwd(ctx, x, w, h.view, act="silu")
    check(h, z0, e0)
    ops.gated_linear_fwd(ctx, x, w, h.view, bias=bias, act="silu", pre=pre.view)
    z, e = z0 + bias.double(), e0 + 2.0 ** -23 * (z0.abs() + bias.abs().double())
    check(h, z, e)
    near(pre.view, z, e + u * (z.abs() + e), "pre")
    pre.check("pre")
