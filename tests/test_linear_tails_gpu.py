"""Activations and their slopes where they are small, against fp64, relative to their size.

u = torch.finfo(t).eps / 2, r = 2^-24 (one fp32 rounding).  bf16 GELU (erf): the normal distribution's integral is
exp(-z^2 / 2) t Q(t).  z^2, its product with the constant and the constant itself are off by r each at most (2.5 r for the three:
the constant by less than half of it), which the exponential makes 2.5 r z^2 / 2; the exponential and the reciprocal of the hardware 2 r
each; t = 1 / (1 + a |z|) is 3 r off and changes t Q(t) by 2.3 times that; Horner's six steps 6 r of sum |c| t^k <= 1.8 Q; the
polynomial itself 12 r; the products 4 r: (40 + 1.5 z^2) r covers them.  fp32: what rounding takes off z^2 / 2 goes back, the exponential is good
to 2 r, a division 1 r: 12 r without the polynomial's 2.7e-9 (0.05 r).  GELU (tanh) and SiLU, z sigmoid(x): x is 5 r off and
its product with log2(e) 2 r more, which the exponential makes 7 r |x|; 8 r for the rest.  A slope, cdf + z density, has these errors of
each of its two terms.  Above -12.5 nothing here is subnormal in bf16."""
import math

import pytest
import torch

from test_linear_gpu import BF16, F32, half_step, near, value

pytestmark = pytest.mark.gpu

R = 2.0 ** -24
LEFT = {"gelu": -12.5, "gelu_tanh": -9.0, "silu": -80.0}


def relative(z, act, dtype):
    if act == "gelu":
        return (40 + 1.5 * z * z) * R if dtype == BF16 else torch.full_like(z, 12 * R)
    x = z if act == "silu" else 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
    return (8 + 7 * x.abs()) * R


def slope_terms(z, act):
    """What the slope is the sum of."""
    if act == "gelu":
        return 0.5 * torch.special.erfc(-z / math.sqrt(2)), z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    a, b = 2 * math.sqrt(2 / math.pi), 0.044715
    x, dx = (z, torch.ones_like(z)) if act == "silu" else (a * (z + b * z ** 3), a * (1 + 3 * b * z * z))
    return torch.sigmoid(x), z * torch.sigmoid(x) * torch.sigmoid(-x) * dx


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("act", list(LEFT))
@pytest.mark.parametrize("rows", [1, 200])
def test_values(ctx, rows, act, dtype):
    """A layer that hands its bias on: products with zero weights."""
    from sirius_amd import ops
    n, u = 4096, half_step(dtype)
    z = torch.linspace(LEFT[act], -2.0 ** -10, n, dtype=torch.float64).float().cuda()
    x, w = torch.ones(rows, 8, dtype=dtype, device="cuda"), torch.zeros(n, 8, dtype=dtype, device="cuda")
    y = torch.empty(rows, n, dtype=dtype, device="cuda")
    ops.linear_fwd(ctx, x, w, y, bias=z, act=act)
    zd = z.double()
    ref, rel = value(zd, act), relative(zd, act, dtype)
    for row in (y[0], y[-1]):
        near(row, ref, (u + rel * (1 + u)) * ref.abs(), act)
    h = torch.empty(rows, n, dtype=dtype, device="cuda")
    up = torch.full((n,), 0.75, device="cuda")
    ops.gated_linear_fwd(ctx, x, torch.zeros(2 * n, 8, dtype=dtype, device="cuda"), h, bias=torch.cat([z, up]), act=act)
    for row in (h[0], h[-1]):
        near(row, 0.75 * ref, (u + (rel + R) * (1 + u)) * 0.75 * ref.abs(), f"gated {act}")


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("act", list(LEFT))
@pytest.mark.parametrize("rows", [1, 200])
def test_gradients(ctx, rows, act, dtype):
    """The derivative's pass and the epilogue of a data gradient, of a gradient of one; in bf16 with their low parts, which leave
    2^-16 of a value."""
    from sirius_amd import ops
    n, u = 1024, half_step(dtype)
    z = torch.linspace(LEFT[act], -2.0 ** -6, n, dtype=torch.float64).to(dtype).cuda()
    pre = torch.cat([z, torch.full_like(z, 0.75)]).expand(rows, 2 * n).contiguous()
    zd = z.double()
    ref, rel = value(zd, act), relative(zd, act, dtype)
    cdf, rest = slope_terms(zd, act)
    off = (rel + 4 * R) * (cdf.abs() + rest.abs())
    one = torch.ones(rows, n, dtype=dtype, device="cuda")
    dy, wt = torch.zeros(rows, 8, dtype=dtype, device="cuda"), torch.ones(n, 8, dtype=dtype, device="cuda")
    dy[:, 3] = 1
    low = dtype == BF16
    left = 2.0 ** -16 if low else u     # of what is stored in two parts, in one

    def parts(cols):
        return [torch.empty(rows, cols, dtype=dtype, device="cuda") for _ in range(2 if low else 1)] + [None] * (not low)

    def whole(t, t_low):
        return t.double() + (t_low.double() if low else 0)
    for epilogue in (False, True):
        dpre, dpre_low = parts(2 * n)
        h, h_low = parts(n)
        if epilogue:
            ops.linear_dgrad_gated(ctx, dy, wt, pre, dpre, act=act, h=h, dpre_low=dpre_low, h_low=h_low)
            for row in whole(h, h_low)[[0, -1]]:
                near(row, 0.75 * ref, (left + rel + 2 * R) * 0.75 * ref.abs(), "h")
        else:
            ops.gated_act_bwd(ctx, one, pre, dpre, act, h=h, dpre_low=dpre_low)
            for row in h[[0, -1]]:
                near(row, 0.75 * ref, (u + rel * (1 + u) + 2 * R) * 0.75 * ref.abs(), "h")
        for row in whole(dpre, dpre_low)[[0, -1]]:
            near(row[:n], 0.75 * (cdf + rest), left * 0.75 * (cdf + rest).abs() + 0.75 * (1 + left) * off, "dg")
            near(row[n:], ref, (left + rel + 2 * R) * ref.abs(), "du")
    dx = torch.empty(rows, n, dtype=dtype, device="cuda")
    ops.linear_dgrad(ctx, dy, wt, dx, act=act, pre=pre[:, :n])
    for row in dx[[0, -1]]:
        near(row, cdf + rest, u * (cdf + rest).abs() + (1 + u) * off, "dx")
